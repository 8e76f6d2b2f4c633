"""The gated delta rule with its outputs in the values' place, and beside the inputs in one buffer: the bits of a call whose
outputs lie apart."""
import numpy as np
import pytest

from ops_cases import act, upload

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("lens,step", [([1] * 5, True), ([1] * 40, True), ([70, 1, 0, 200, 64], False), ([300, 129] * 8, False)],
                         ids=["step", "steps", "chunk", "chunks"])
def test_outputs_over_the_values_and_in_one_buffer(sc, ops, cuda, lens, step, dtype):
    S, heads, N, n = 64, 16, sum(lens), len(lens)
    rng = np.random.default_rng(N + n)
    q, k, v = (act(rng.standard_normal((N, heads * S)), dtype)[0] for _ in range(3))
    gates = [upload(sc, x.astype(np.float32)) for x in (-rng.random((N, heads)), rng.random((N, heads)))]
    M = (rng.standard_normal((n, S, heads, S)) * 0.3).astype(np.float32)
    cu = None if step else upload(sc, np.cumsum([0, *lens]).astype(np.int64))
    row, b = heads * S, v.dtype.itemsize
    found = []
    for place in ("apart", "v", "fused"):
        state = upload(sc, M)
        states = ops.gdn_states(state, n_seqs=n, v_heads=heads, state_size=S)
        kw = dict(k_heads=heads, n_seqs=n, tokens=N, cu=cu, scale=S ** -0.5, l2norm=True)
        make = ops.GdnStep if step else ops.GdnChunk
        if place == "fused":   # a row's queries, keys, values and outputs next to each other
            whole = upload(sc, np.concatenate([q, k, v, np.zeros_like(v)], 1))
            at = [whole.ptr + i * row * b for i in range(4)]
            make(states, *at[:3], *gates, at[3], dtype, q_ld=4 * row, k_ld=4 * row, v_ld=4 * row, out_ld=4 * row, **kw).launch()
        else:
            bufs = [upload(sc, x) for x in (q, k, v)]
            out = bufs[2] if place == "v" else upload(sc, np.zeros_like(v))
            make(states, *bufs, *gates, out, dtype, **kw).launch()
        sc.device_sync()
        got = whole.numpy()[:, 3 * row:] if place == "fused" else out.numpy()
        found.append((np.ascontiguousarray(got), state.numpy()))
    for got, state in found[1:]:
        assert np.array_equal(got.view(np.uint8), found[0][0].view(np.uint8)) and np.array_equal(state.view(np.uint8), found[0][1].view(np.uint8))


@pytest.mark.parametrize("heads,head_ld,key_ld", [(4, 68, 3 * 68 + 64), (4, 63 * 72 + 64, 72), (1, 64 * 64, 72), (1, 68, 64)])
@pytest.mark.parametrize("step", [True, False], ids=["step", "chunk"])
def test_states_with_room_between(sc, ops, cuda, step, heads, head_ld, key_ld):
    """Heads or keys apart by more than their rows, to the last float: the packed states' bits, and the room between untouched."""
    S, n, N = 64, 3, 3 if step else 100
    rng = np.random.default_rng(heads + key_ld)
    q, k, v = (upload(sc, rng.standard_normal((N, heads * S)).astype(np.float32)) for _ in range(3))
    gates = [upload(sc, x.astype(np.float32)) for x in (-rng.random((N, heads)), rng.random((N, heads)))]
    cu = None if step else upload(sc, np.array([0, 70, 70, 100], np.int64))
    M = rng.standard_normal((n, heads, S, S)).astype(np.float32)   # [head][key][value]
    each = (heads - 1) * head_ld + (S - 1) * key_ld + S
    flat = np.full((n, each + 4), 7, np.float32)
    at = (np.arange(heads) * head_ld)[:, None, None] + (np.arange(S) * key_ld)[:, None] + np.arange(S)
    flat[:, at] = M
    found = []
    for packed in (True, False):
        state = upload(sc, M if packed else flat)
        if packed:
            states = ops.gdn_states(state, n_seqs=n, v_heads=heads, state_size=S, layout="prefill")
        else:
            states = ops.GdnStates([state.ptr + 4 * i * (each + 4) for i in range(n)], heads, S, 0, head_ld, key_ld, keep=state)
        out = upload(sc, np.zeros((N, heads * S), np.float32))
        make = ops.GdnStep if step else ops.GdnChunk
        make(states, q, k, v, *gates, out, "f32", k_heads=heads, n_seqs=n, tokens=N, cu=cu, scale=S ** -0.5, l2norm=True).launch()
        sc.device_sync()
        got = state.numpy()
        if not packed:
            rest = np.ones(got.shape, bool)
            rest[:, at] = False
            assert (got[rest] == 7).all()
            got = np.ascontiguousarray(got[:, at])
        found.append((out.numpy(), got))
    assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(*found))
