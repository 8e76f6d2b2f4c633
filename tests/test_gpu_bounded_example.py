"""A conversation with a bounded cache (examples/bounded_conversation.py) against the 64-bit implementation, token by token: a
prompt with a picture, the mass of its last queries, evictions, a hand-off of the shortened slot, new tokens; and the calls of
a token and of an eviction replayed from HIP graphs."""
import ctypes as C
import sys
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

GEO = dict(n_layers=8, qsa_interval=4, n_head_kv=2, head_dim=128, page_size=4, ssm_state_size=64, ssm_k_heads=2,
           ssm_v_heads=4, ssm_conv_channels=512)
HEADS, GRID, NEW, KEEP, EVERY, LAST = 6, (7, 9), 9, 40, 3, 8
PROMPT = 50 + GRID[0] * GRID[1] + 37


@pytest.fixture(scope="module")
def example():
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "strata-concurrent_amd" / "examples"))
    import bounded_conversation
    return bounded_conversation


def _started(sc, example):
    geo = sc.geometry(**GEO)
    before, new = example.Inputs(geo, PROMPT, HEADS, 1), example.Inputs(geo, NEW, HEADS, 2)
    pos = example.positions(5, 50, GRID, 37)
    b = example.Bounded(geo, HEADS, KEEP, PROMPT, EVERY)
    return geo, before, new, pos, b


def test_a_conversation(sc, example, cuda):
    """f32 inputs, f16 caches: a key or value is its f32 rotation rounded once (2^-11 of itself), which moves a score by at most
    2^-11 scale sum |q k| =: e, an attention output by 2 e max |v| and 2^-11 of its values, a weight by 2 e of itself.  The
    recurrent layers stay in 32 bits; their inputs, sums of 4 products and a silu, are off by 2^-20 of their largest, which moves
    a query or key of unit length by sqrt(S) 2^-20 and an output by as much a token at most: 2^-19 sqrt(S T) with the chunks' own
    2^-21 sqrt(S T).  Which cells are kept is exact for the masses that the device holds."""
    from oracle import sc_ops as plain
    geo, before, new, pos, b = _started(sc, example)
    S, share, D, H, G = geo.ssm_state_size, geo.ssm_v_heads // geo.ssm_k_heads, geo.head_dim, geo.n_head_kv, HEADS // geo.n_head_kv
    KH, W = geo.ssm_k_heads, geo.ssm_d_conv
    outs = b.prompt(before, pos, LAST)
    inv_freq = b.inv_freq.numpy()
    where = np.concatenate([pos, np.broadcast_to(pos.max() + 1 + np.arange(NEW), (3, NEW))], 1)
    keys = [np.stack([plain.rotate_axes(np.concatenate([x["k"], y["k"]])[t], where[:, t], b.axis, inv_freq, example.ROT, "halves")
                      for t in range(PROMPT + NEW)]) for x, y in zip(before.attn, new.attn)]
    queries = [np.stack([plain.rotate_axes(np.concatenate([x["q"], y["q"]])[t], where[:, t], b.axis, inv_freq, example.ROT, "halves")
                         for t in range(PROMPT + NEW)]) for x, y in zip(before.attn, new.attn)]
    values = [np.concatenate([x["v"], y["v"]]).astype(np.float64) for x, y in zip(before.attn, new.attn)]
    held = [[list(range(PROMPT)) for _ in range(H)] for _ in range(geo.n_qsa)]       # the token in each cell
    mass = [[np.zeros(PROMPT) for _ in range(H)] for _ in range(geo.n_qsa)]

    def attend(j, h, i, t, tokens):
        """A query's weights over tokens, and how far a score may be off."""
        k, q = keys[j][tokens, h], queries[j][t, i]
        return plain.attention_mass(q, k, D ** -0.5), 2.0 ** -11 * D ** -0.5 * np.abs(k * q).sum(-1).max() + 2.0 ** -18

    def check_mass(j, off):
        got = b.mass[j].numpy().reshape(H, -1)
        for h in range(H):
            n = len(held[j][h])
            assert (np.abs(got[h, :n] - mass[j][h]) <= off[h] * mass[j][h] + 2.0 ** -100).all(), (j, h)
            assert not got[h, n:].any()
        return got

    off = np.zeros((geo.n_qsa, H))   # how far masses may be off, of themselves
    for j in range(geo.n_qsa):
        for h in range(H):
            for r in range(LAST):
                t = PROMPT - LAST + r
                for i in range(h * G, (h + 1) * G):
                    p, e = attend(j, h, i, t, held[j][h][:t + 1])
                    mass[j][h][:t + 1] += p
                    off[j, h] = max(off[j, h], 2.01 * e)
        check_mass(j, off[j])

    def evict(calls):
        was = [m.numpy().reshape(H, -1).copy() for m in b.mass]
        n, total = b.cells, b.tokens
        b.evict(calls)
        sc.device_sync()
        for j in range(geo.n_qsa):
            for h in range(H):
                place = plain.evict(was[j][h, :n], held[j][h], total, KEEP, example.SINKS, example.RECENT)
                held[j][h], mass[j][h] = [held[j][h][c] for c in place], mass[j][h][place]
                assert np.array_equal(b.born[j].numpy().reshape(H, -1)[h, :len(place)], held[j][h]), (j, h)
            check_mass(j, off[j])
        assert b.left.numpy()[0] == b.known.numpy()[0] == b.cells

    evict(b.evictions())
    assert b.cells == KEEP
    b.hand_off()
    dec, cut = example.Decoder(b, new), b.evictions()
    steps = []
    for t in range(NEW):
        dec.token(t, int(where[0, PROMPT + t]))
        sc.device_sync()
        steps.append([o.numpy().astype(np.float64) for o in dec.gdn_out])
        for j in range(geo.n_qsa):
            got = dec.attn_out[j].numpy().astype(np.float64)
            for h in range(H):
                held[j][h].append(PROMPT + t)
                mass[j][h] = np.append(mass[j][h], 0.0)
                for i in range(h * G, (h + 1) * G):
                    p, e = attend(j, h, i, PROMPT + t, held[j][h])
                    v = values[j][held[j][h], h]
                    assert (np.abs(got[i] - p @ v) <= (2 * e + 2.0 ** -11) * np.abs(v).max()).all(), (j, t, i)
                    mass[j][h] += p
                    off[j, h] = max(off[j, h], 2.01 * e)
            check_mass(j, off[j])
        if (t + 1) % EVERY == 0:
            evict(cut)
            assert b.cells == KEEP
    for i in range(geo.n_gdn):
        x = {n: np.concatenate([before.gdn[i][n], new.gdn[i][n]]) for n in before.gdn[i]}
        y, _ = plain.short_conv(np.zeros((W - 1, geo.ssm_conv_channels)), x["x"], b.taps[i].numpy().reshape(-1, W), None, True)
        q, k, v = y[:, :KH * S].reshape(-1, KH, S), y[:, KH * S:2 * KH * S].reshape(-1, KH, S), y[:, 2 * KH * S:].reshape(-1, geo.ssm_v_heads, S)
        for h in range(geo.ssm_v_heads):
            want, _ = plain.delta_rule(np.zeros((S, S)), q[:, h // share], k[:, h // share], v[:, h], x["g"][:, h], x["beta"][:, h], S ** -0.5, True,
                                       1e-6)
            got = np.concatenate([outs[i][:, h], [s[i][h] for s in steps]])
            assert np.abs(got - want).max() <= 2.0 ** -19 * np.sqrt(S * (PROMPT + NEW)) * np.abs(want).max(), (i, h)


def test_tokens_and_evictions_from_graphs(sc, example, cuda):
    """The calls of a token and of an eviction captured once and replayed, with eager work and waits between the replays, leave
    the bits that eager calls leave: outputs, caches, states, histories, masses and numbers."""
    hip, got = C.CDLL(sc.lib._name), []
    for graphed in (False, True):
        geo, before, new, pos, b = _started(sc, example)
        b.prompt(before, pos, LAST)
        b.evict(b.evictions())
        sc.device_sync()
        dec, cut, stream = example.Decoder(b, new), b.evictions(), sc.Stream()
        handle, graphs = C.c_void_p(stream.handle), []
        if graphed:
            for calls in (dec.calls, cut):
                graph, run = C.c_void_p(), C.c_void_p()
                assert hip.hipStreamBeginCapture(handle, 2) == 0   # relaxed
                for call in calls:
                    call.launch(stream)
                assert hip.hipStreamEndCapture(handle, C.byref(graph)) == 0
                assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
                graphs.append((graph, run))
        rows = []
        for t in range(NEW):
            dec.feed(t, int(pos.max()) + 1 + t)
            sc.device_sync()
            if graphed:
                assert hip.hipGraphLaunch(graphs[0][1], handle) == 0
            else:
                for call in dec.calls:
                    call.launch(stream)
            stream.sync()
            if t % 2:
                if graphed:
                    assert hip.hipGraphLaunch(graphs[1][1], handle) == 0
                    b.evict([], stream)
                else:
                    b.evict(cut, stream)
                stream.sync()
            rows += [x.numpy() for x in (*dec.attn_out, *dec.gdn_out, b.left, b.known)]
        rows += [x.numpy() for x in (*b.slot.buffers(), *b.mass, *b.born)]
        got.append(rows)
        for graph, run in graphs:
            assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    assert all(np.array_equal(p.view(np.uint8), q.view(np.uint8)) for p, q in zip(*got))
