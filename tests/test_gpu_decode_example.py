"""A conversation through the operators and a hand-off (examples/decode_after_handoff.py) against the 64-bit
implementation, token by token; and the calls of a token replayed from a HIP graph."""
import ctypes as C
import sys
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

GEO = dict(n_layers=8, qsa_interval=4, n_head_kv=2, head_dim=128, page_size=4, ssm_state_size=64, ssm_k_heads=2,
           ssm_v_heads=4, ssm_conv_channels=256)
HEADS, PROMPT, NEW = 6, 150, 5


@pytest.fixture(scope="module")
def example():
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "strata-concurrent_amd" / "examples"))
    import decode_after_handoff
    return decode_after_handoff


def test_a_conversation(sc, example, cuda):
    """f32 inputs, f16 caches: a key or value is its f32 rotation rounded once (2^-11 of itself), which moves a score by
    at most 2^-11 scale |q| |k| and an output by twice that of max |v|, and 2^-11 |v| of its own; the recurrent layers
    stay in 32 bits through chunks, carve and steps (2^-21 sqrt(S T))."""
    from oracle import sc_ops as plain
    geo = sc.geometry(**GEO)
    S, share, D = geo.ssm_state_size, geo.ssm_v_heads // geo.ssm_k_heads, geo.head_dim
    before, new = example.Inputs(geo, PROMPT, HEADS, 1), example.Inputs(geo, NEW, HEADS, 2)
    conv = example.Conversation(geo, HEADS, PROMPT + NEW)
    outs = conv.prompt(before)
    dec = conv.decoder(new)
    attn, gdn = [], []
    for t in range(NEW):
        dec.token(t)
        attn.append([b.numpy().astype(np.float64) for b in dec.attn_out])
        gdn.append([b.numpy().astype(np.float64) for b in dec.gdn_out])
    inv_freq = conv.inv_freq.numpy()
    for i in range(geo.n_gdn):
        x = {n: np.concatenate([before.gdn[i][n], new.gdn[i][n]]) for n in before.gdn[i]}
        for h in range(geo.ssm_v_heads):
            want, _ = plain.delta_rule(np.zeros((S, S)), x["q"][:, h // share], x["k"][:, h // share], x["v"][:, h], x["g"][:, h],
                                       x["beta"][:, h], S ** -0.5, True, 1e-6)
            got = np.concatenate([outs[i][:, h], [gdn[t][i][h] for t in range(NEW)]])
            assert np.abs(got - want).max() <= 2.0 ** -21 * np.sqrt(S * (PROMPT + NEW)) * np.abs(want).max(), (i, h)
    for j in range(geo.n_qsa):
        x = {n: np.concatenate([before.attn[j][n], new.attn[j][n]]) for n in before.attn[j]}
        k = np.stack([plain.rotate(x["k"][t], t, inv_freq, example.ROT, "halves") for t in range(PROMPT + NEW)])
        for t in range(NEW):
            q = plain.rotate(x["q"][PROMPT + t], PROMPT + t, inv_freq, example.ROT, "halves")
            for h in range(HEADS):
                c = h // (HEADS // geo.n_head_kv)
                keys, values = k[:PROMPT + t + 1, c], x["v"][:PROMPT + t + 1, c]
                want, _ = plain.attention(q[h], keys, values, D ** -0.5)
                e = 2.0 ** -11 * D ** -0.5 * np.abs(keys * q[h]).sum(-1).max() + 2.0 ** -18
                assert (np.abs(attn[t][j][h] - want) <= (2 * e + 2.0 ** -11) * np.abs(values).max()).all(), (j, t, h)


def _hip(sc):
    """The HIP runtime that the library is linked with: its names are found through the library."""
    return C.CDLL(sc.lib._name)


def test_a_token_from_a_graph(sc, example, cuda):
    """The calls of a new token captured once and replayed for each token, with eager work and waits between the replays,
    give the bits that eager calls give."""
    geo = sc.geometry(**GEO)
    before, new = example.Inputs(geo, PROMPT, HEADS, 1), example.Inputs(geo, NEW, HEADS, 2)
    hip = _hip(sc)
    got = []
    for graphed in (False, True):
        conv = example.Conversation(geo, HEADS, PROMPT + NEW)
        conv.prompt(before)
        dec = conv.decoder(new)
        graph, run = C.c_void_p(), C.c_void_p()
        stream = sc.Stream()
        if graphed:
            handle = C.c_void_p(stream.handle)
            assert hip.hipStreamBeginCapture(handle, 2) == 0   # relaxed
            for call in dec.calls:
                call.launch(stream)
            assert hip.hipStreamEndCapture(handle, C.byref(graph)) == 0
            assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
        rows = []
        for t in range(NEW):
            dec.feed(t)
            sc.device_sync()
            if graphed:
                assert hip.hipGraphLaunch(run, handle) == 0
            else:
                for call in dec.calls:
                    call.launch(stream)
            stream.sync()
            rows += [b.numpy() for b in (*dec.attn_out, *dec.gdn_out)]
        rows += [b.numpy() for b in conv.slot.buffers()]
        got.append(rows)
        if graphed:
            assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(*got))


def test_a_prompt_from_a_graph(sc, example, cuda):
    """The chunk form and an append of many tokens, captured and replayed from the same state, give the eager bits."""
    import sc_ops as ops
    geo = sc.geometry(**GEO)
    S, KH, VH, H, D = geo.ssm_state_size, geo.ssm_k_heads, geo.ssm_v_heads, geo.n_head_kv, geo.head_dim
    x, T = example.Inputs(geo, 700, HEADS, 3), 700
    hip, stream = _hip(sc), sc.Stream()
    handle = C.c_void_p(stream.handle)
    cu, pos = example._up(np.array([0, T], np.int64)), example._up(np.zeros(1, np.int64))
    inv_freq = example._up((1e4 ** (-np.arange(0, 64, 2) / 64)).astype(np.float32))
    k, v = (sc.DeviceBuffer((T, H, D), "uint16") for _ in range(2))
    state, out, q_out = (sc.DeviceBuffer(s, "float32") for s in ((VH, S, S), (T, VH, S), (T, HEADS, D)))
    a, g = x.attn[0], x.gdn[0]
    cache = ops.kv_cache(k, v, n_pages=T, n_head_kv=H, head_dim=D, page_size=1, table_ld=T)
    calls = [ops.RopeAppend(cache, example._up(a["k"]), example._up(a["v"]), "f32", n_seqs=1, tokens=T, cu=cu, pos0=pos,
                            inv_freq=inv_freq, rot_dim=64, q=example._up(a["q"]), q_out=q_out, n_head=HEADS),
             ops.GdnChunk(ops.gdn_states(state, n_seqs=1, v_heads=VH, state_size=S), *(example._up(g[n]) for n in ("q", "k", "v", "g", "beta")),
                          out, "f32", k_heads=KH, n_seqs=1, tokens=T, cu=cu, scale=S ** -0.5, l2norm=True)]
    buffers = (k, v, q_out, state, out)

    def once(run):
        for b in buffers:
            b.fill(0)
        sc.device_sync()
        run()
        stream.sync()
        return [b.numpy() for b in buffers]

    want = once(lambda: [c.launch(stream) for c in calls])
    graph, run = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(handle, 2) == 0
    for c in calls:
        c.launch(stream)
    assert hip.hipStreamEndCapture(handle, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    for _ in range(3):
        got = once(lambda: hip.hipGraphLaunch(run, handle))
        assert all(np.array_equal(p.view(np.uint8), q.view(np.uint8)) for p, q in zip(want, got))
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
