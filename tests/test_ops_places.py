"""Where the gated delta rule's outputs may lie: what would let one workgroup write what another still reads is refused
before any HIP call, and what does not is not."""
import ctypes as C

import pytest

FAKE = 1 << 40   # stands for device addresses: every request below is refused before they are used


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


# q, k, v and out of 5 rows of 8 heads of 64 f32 values (2 KiB a row) in one buffer, by their first bytes and strides
ROW = 8 * 64 * 4


def _said(sc, ops, step, *, q, k, v, out, ld, out_ld=None, tokens=5, state_offset=0):
    a = ops.GdnDesc(k_heads=8, v_heads=8, state_size=64, n_seqs=tokens if step else 1, tokens=tokens, cu=None if step else FAKE,
                    dtype=sc.SC_DTYPE_F32, q=FAKE + q, k=FAKE + k, v=FAKE + v, out=FAKE + out, q_ld=ld // 4, k_ld=ld // 4, v_ld=ld // 4,
                    out_ld=(out_ld or ld) // 4, g=FAKE, beta=FAKE, gate_ld=8, scale=0.1, l2norm=1, eps=1e-6, state=FAKE,
                    state_offset=state_offset, state_head_ld=64, state_key_ld=512)
    code = sc.lib.sc_gdn_step_async(C.byref(a), None) if step else sc.lib.sc_gdn_chunk_async(C.byref(a), FAKE, 1 << 40, None)
    assert code != sc.SC_OK   # no GPU here: what is not refused fails when it is launched
    return code, sc.last_error()


MIB = 1 << 20
OVERLAPS = [
    dict(q=0, k=MIB, v=2 * MIB, out=0, ld=ROW), dict(q=0, k=MIB, v=2 * MIB, out=MIB, ld=ROW),               # q or k itself
    dict(q=0, k=MIB, v=2 * MIB, out=4 * ROW + 16, ld=ROW), dict(q=ROW - 16, k=MIB, v=2 * MIB, out=0, ld=ROW, tokens=1),
    dict(q=0, k=MIB, v=2 * MIB, out=2 * MIB + ROW, ld=ROW), dict(q=0, k=MIB, v=2 * MIB + ROW, out=2 * MIB, ld=ROW),   # a row off v
    dict(q=0, k=MIB, v=2 * MIB, out=2 * MIB, ld=ROW, out_ld=ROW + 16),                                        # v by another stride
    dict(q=0, k=ROW, v=2 * ROW, out=16, ld=3 * ROW), dict(q=0, k=ROW, v=2 * ROW, out=2 * ROW + 16, ld=3 * ROW),   # a fused row's parts
    dict(q=0, k=ROW, v=2 * ROW, out=3 * ROW - 16 + 2 * 4 * ROW, ld=4 * ROW),
]
APART = [
    dict(q=0, k=MIB, v=2 * MIB, out=2 * MIB, ld=ROW),                              # v itself
    dict(q=0, k=MIB, v=2 * MIB, out=5 * ROW, ld=ROW), dict(q=5 * ROW, k=MIB, v=2 * MIB, out=0, ld=ROW),   # end to end
    dict(q=0, k=ROW, v=2 * ROW, out=3 * ROW, ld=4 * ROW),                          # side by side
    dict(q=0, k=ROW, v=2 * ROW, out=2 * ROW, ld=3 * ROW), dict(q=3 * ROW, k=ROW, v=2 * ROW, out=0, ld=4 * ROW),
]


@pytest.mark.parametrize("step", [True, False], ids=["step", "chunk"])
@pytest.mark.parametrize("at", range(len(OVERLAPS)))
def test_outputs_over_inputs_are_refused(sc, ops, step, at):
    code, why = _said(sc, ops, step, **OVERLAPS[at])
    assert code == sc.SC_EINVAL and "out must not overlap" in why, why


@pytest.mark.parametrize("step", [True, False], ids=["step", "chunk"])
@pytest.mark.parametrize("at", range(len(APART)))
def test_outputs_beside_inputs_are_not(sc, ops, step, at):
    if sc.device_count() > 0:
        pytest.skip("the addresses are none: only where nothing can be launched")
    code, why = _said(sc, ops, step, **APART[at])
    assert code == sc.SC_EHIP and "overlap" not in why, why


def test_a_batch_without_tokens_has_no_rows(sc, ops):
    a = ops.GdnDesc(k_heads=8, v_heads=8, state_size=64, n_seqs=1, tokens=0, cu=FAKE, dtype=sc.SC_DTYPE_F32, q=FAKE, k=FAKE, v=FAKE,
                    out=FAKE, q_ld=512, k_ld=512, v_ld=512, out_ld=512, g=FAKE, beta=FAKE, gate_ld=8, scale=0.1, l2norm=1, eps=1e-6,
                    state=FAKE, state_offset=0, state_head_ld=64, state_key_ld=512)
    assert sc.lib.sc_gdn_chunk_async(C.byref(a), FAKE, 1 << 40, None) == sc.SC_OK


STRIDES = [(68, 7 * 68 + 64), (64, 512), (64 * 64, 64), (63 * 72 + 64, 72), (1 << 40, 64), (64, 1 << 40)]   # heads, keys
STRIDES_REFUSED = [(68, 7 * 68 + 60), (63 * 72 + 60, 72), (128, 512), (1 << 62, 64), (64, 1 << 62), ((1 << 40) + 4, 64)]


def _strides(sc, ops, step, v_heads, head_ld, key_ld, offset=0):
    n = 5
    a = ops.GdnDesc(k_heads=v_heads, v_heads=v_heads, state_size=64, n_seqs=n if step else 1, tokens=n, cu=None if step else FAKE,
                    dtype=sc.SC_DTYPE_F32, q=FAKE, k=FAKE, v=FAKE + MIB, out=FAKE + 2 * MIB, q_ld=512, k_ld=512, v_ld=512, out_ld=512,
                    g=FAKE, beta=FAKE, gate_ld=8, scale=0.1, l2norm=1, eps=1e-6, state=FAKE, state_offset=offset, state_head_ld=head_ld,
                    state_key_ld=key_ld)
    code = sc.lib.sc_gdn_step_async(C.byref(a), None) if step else sc.lib.sc_gdn_chunk_async(C.byref(a), FAKE, 1 << 40, None)
    return code, sc.last_error()


@pytest.mark.parametrize("step", [True, False], ids=["step", "chunk"])
@pytest.mark.parametrize("v_heads,head_ld,key_ld", [(8, *x) for x in STRIDES] + [(1, 64, 64), (1, 4096, 72), (1, 68, 64)])
def test_states_apart_are_taken(sc, ops, step, v_heads, head_ld, key_ld):
    if sc.device_count() > 0:
        pytest.skip("the addresses are none: only where nothing can be launched")
    code, why = _strides(sc, ops, step, v_heads, head_ld, key_ld)
    assert code == sc.SC_EHIP, why


@pytest.mark.parametrize("step", [True, False], ids=["step", "chunk"])
@pytest.mark.parametrize("head_ld,key_ld", STRIDES_REFUSED)
def test_states_that_meet_are_refused(sc, ops, step, head_ld, key_ld):
    code, why = _strides(sc, ops, step, 8, head_ld, key_ld)
    assert code == sc.SC_EINVAL and "state strides" in why, why
    assert _strides(sc, ops, step, 8, 64, 512, 1 << 62)[0] == sc.SC_EINVAL
