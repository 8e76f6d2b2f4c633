"""sc_attn_mass_async where a workgroup takes several turns of a batch's cells, up to 16 columns: keys and pages asked for a turn
ahead, sums carried from turn to turn, turns that no row sees left out.  Tolerances as in test_gpu_mass.py, the sums over the
cells of a turn after the other in 32 bits among them: a carried sum is rounded once a turn, three of them 3 2^-24."""
import ctypes as C

import numpy as np
import pytest

from ops_cases import Cache, act, upload

pytestmark = pytest.mark.gpu

H, D, PS, SEQS, MOST, UNIT = 2, 64, 8, 24, 8200, 128


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


@pytest.fixture(scope="module")
def plain():
    from oracle import sc_ops
    return sc_ops


@pytest.fixture(scope="module", params=["f16", "int8"])
def made(request, sc, ops, plain, cuda):
    """The batch's cache, its lengths, and each sequence's keys in 64 bits [H][cells][D] with the cells that are resident."""
    rng = np.random.default_rng(17)
    table_ld = -(-MOST // PS)
    cache = Cache(sc, ops, rng, request.param, H, D, PS, SEQS, table_ld, missing=0.02)
    lens = [MOST, 0, 1, 129, 8191, *(int(x) for x in rng.integers(300, MOST, SEQS - 5))]
    K = cache.values("k").reshape(cache.n_pages, H, PS, D)
    keys, there = [], []
    for s, t in enumerate(lens):
        page = cache.table[s]
        ok = (page >= 0) & (page < cache.n_pages)
        rows = K[np.where(ok, page, 0)].transpose(1, 0, 2, 3).reshape(H, -1, D)[:, :t]
        keys.append(rows)
        there.append(np.repeat(ok, PS)[:t])
    return cache, lens, keys, there


def _weights(keys, there, q, ends, window, scale, lse):
    """One head's weights over the cells [begin, ends), and how far a score may be off; the log of the sum."""
    n, p = len(there), np.zeros(len(there))
    see = there & (np.arange(n) < ends)
    if window:
        see &= np.arange(n) >= ends - window
    if not see.any():
        return p, 0.0, -np.inf
    s = scale * (keys[see] @ q)
    e = 2.0 ** -19 * scale * (np.abs(keys[see]) @ np.abs(q)).max()
    own = np.log(np.exp(s - s.max()).sum()) + s.max()
    p[see] = np.exp(s - (own if lse is None else lse))
    return p, e, own


@pytest.mark.parametrize("given", [True, False], ids=["given", "formed"])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("rows,window", [(1, 0), (4, 0), (2, 1500)])
def test_several_turns(sc, ops, made, given, dtype, rows, window):
    cache, lens, keys, there = made
    rng, G = np.random.default_rng(rows + window), 3
    heads = H * G
    q, q64 = act(rng.standard_normal((SEQS * rows, heads, D)) * 1.5, dtype)
    scale = float(np.float32(D ** -0.5 * (0.5 if cache.fmt == "int8" else 1.0)))
    decay, old = 0.75, rng.random((SEQS, H, MOST)).astype(np.float32) / 100
    want, near = np.zeros((SEQS, H, MOST)), np.zeros((SEQS, H, MOST))
    lse = np.full((SEQS * rows, heads), -np.inf, np.float32)
    for s, t in enumerate(lens):
        for r in range(rows):
            for i in range(heads):
                ends, h = t - rows + 1 + r, i // G
                _, _, own = _weights(keys[s][h], there[s], q64[s * rows + r, i], ends, window, scale, None)
                lse[s * rows + r, i] = own
                p, e, _ = _weights(keys[s][h], there[s], q64[s * rows + r, i], ends, window, scale,
                                   float(lse[s * rows + r, i]) if given else None)
                want[s, h, :t] += p
                near[s, h, :t] += p * (2 * e + 2.0 ** -20 + (rows * G + 3) * 2.0 ** -24) + 2.0 ** -120
    mass, dlse = upload(sc, old), upload(sc, lse) if given else None
    call = ops.AttnMass(cache.c, upload(sc, q), mass, dtype, n_seqs=SEQS, n_head=heads, rows=rows, lens=upload(sc, np.array(lens, np.int64)),
                        max_len=MOST, scale=scale, window=window, lse=dlse, decay=decay)
    # a workgroup has several turns: the workspace of sums that are formed holds a reference and a sum a part and column
    desc = ops.AttnMassDesc(**{n: getattr(call.desc, n) for n, _ in ops.AttnMassDesc._fields_})
    desc.lse = None
    parts = ops.lib.sc_attn_mass_workspace_bytes(C.byref(cache.c), C.byref(desc)) // (SEQS * H * rows * G * 8) - 1
    assert parts * 2 < -(-MOST // UNIT), parts
    call.launch()
    sc.device_sync()
    got = mass.numpy()
    for s, t in enumerate(lens):
        was = decay * old[s, :, :t].astype(np.float64)
        off = np.abs(got[s, :, :t] - (was + want[s, :, :t]))
        assert (off <= near[s, :, :t] + 2.0 ** -23 * (was + want[s, :, :t])).all(), (s, off.max())
        assert np.array_equal(got[s, :, t:].view(np.uint32), old[s, :, t:].view(np.uint32)), s
