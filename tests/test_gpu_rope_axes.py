"""sc_rope_axes_append_async against the 64-bit implementation of the same operator.

What may differ is what sc_rope_append_async's may (tests/test_gpu_rope_append.py): 2^-21 (|a| + |b|) for a pair, and the
rounding to the type that holds it."""
import numpy as np
import pytest

from ops_cases import SENTINEL, Cache, act, between_rows_untouched, strided, upload

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


@pytest.fixture(scope="module")
def plain():
    from oracle import sc_ops
    return sc_ops


def _freq(rot):
    return (1e7 ** (-np.arange(0, rot, 2, dtype=np.float64) / max(rot, 1))).astype(np.float32)


CASES = [
    # fmt, act, H, D, ps, n_head, rot, pairs, pairs of each axis, by turns, rows of each sequence, first cells
    ("f16", "f32", 2, 256, 4, 24, 64, "halves", (11, 11, 10), True, [1], [4093]),
    ("f16", "f16", 2, 256, 4, 24, 256, "neighbours", (44, 42, 42), False, [1, 1, 1], [0, 131070, 7]),
    ("f16", "f32", 1, 64, 1, 1, 64, "halves", (16, 8, 8), False, [5, 0, 130], [0, 3, 61]),
    ("int8", "f16", 4, 128, 16, 4, 32, "neighbours", (0, 16), False, [33, 64, 1], [15, 16, 40000]),
    ("int8", "f32", 2, 128, 5, 0, 128, "halves", (1, 2, 3, 58), True, [600], [1]),
    ("f16", "f16", 3, 64, 3, 6, 8, "halves", (4,), False, [11], [5]),
    ("f16", "f32", 1, 256, 16, 3, 256, "halves", (32, 32, 32, 32), True, [513], [100]),
    ("f16", "f16", 1, 64, 4, 2, 0, "halves", (), False, [3], [0]),
]


def _positions(rng, A, N):
    """Positions of any sign, small and far."""
    pos = rng.integers(0, 5000, (A, N))
    far = rng.random((A, N))
    return np.where(far < 0.1, -pos, np.where(far > 0.9, pos + 1000000, pos)).astype(np.int64)


@pytest.mark.parametrize("case", CASES, ids=[f"{c[0]}-{c[1]}-{c[2]}x{c[3]}-p{c[4]}-r{c[6]}{c[7][0]}-{len(c[8])}axes" for c in CASES])
def test_append_against_64_bits(sc, ops, plain, cuda, case):
    fmt, dtype, H, D, ps, heads, rot, pairs, of, turns, lens, cell0 = case
    print(f"axes append {case}", flush=True)
    rng = np.random.default_rng(len(lens) * 1000 + D + rot)
    n, N, ld, A = len(lens), sum(lens), max((p + t - 1) // ps + 1 for p, t in zip(cell0, lens)), max(len(of), 1)
    axis = ops.axis_of_pairs(of, turns)
    table = np.full((n, ld), -1, np.int32)
    used = [(s, p) for s in range(n) for p in range(cell0[s] // ps, (cell0[s] + lens[s] - 1) // ps + 1) if lens[s]]
    n_pages = len(used) + 2
    for (s, p), phys in zip(used, rng.permutation(n_pages)):
        table[s, p] = phys if rng.random() < 0.95 else -1
    cache = Cache(sc, ops, rng, fmt, H, D, ps, n, ld, table=table, n_pages=n_pages, fill="sentinel")
    k, k64 = act(rng.standard_normal((N, H, D)), dtype)
    v, v64 = act(rng.standard_normal((N, H, D)) * 3, dtype)
    q, q64 = act(rng.standard_normal((N, max(heads, 1), D)), dtype)
    pos, pad, row, qrow = _positions(rng, A, N), 24, H * D, max(heads, 1) * D
    wide = np.full((A, N + 3), 1 << 62, np.int64)
    wide[:, :N] = pos
    dk, dv, dq = strided(sc, k, row + pad), strided(sc, v, row + 2 * pad), strided(sc, q, qrow + pad)
    dout = strided(sc, np.zeros_like(q), qrow + 2 * pad)
    freq = _freq(rot)
    ops.RopeAxesAppend(cache.c, dk, dv, dtype, n_seqs=n, tokens=N, cu=upload(sc, np.cumsum([0, *lens]).astype(np.int64)),
                       pos0=upload(sc, np.array(cell0, np.int64)), inv_freq=upload(sc, freq) if rot else None, rot_dim=rot, pairs=pairs,
                       axis=axis, pos=upload(sc, wide), pos_ld=N + 3, n_axes=A, q=dq if heads else None, q_out=dout if heads else None,
                       n_head=heads, k_ld=row + pad, v_ld=row + 2 * pad, q_ld=qrow + pad, q_out_ld=qrow + 2 * pad).launch()
    sc.device_sync()

    def near(x, turned):   # 2^-21 (|a| + |b|) of each value's pair, below 2^-20 of the head's largest
        return 2.0 ** -20 * np.abs(x).max(-1, keepdims=True) * (1 if turned and rot else 0) + 2.0 ** -60

    half = 2.0 ** -11 if dtype == "f16" else 2.0 ** -24
    got_q = dout.numpy()
    assert between_rows_untouched(got_q, qrow)
    written = np.zeros(n_pages * H * ps, bool)
    want = {c: {} for c in "kv"}
    for s, first, rows in plain.rows_of(np.cumsum([0, *lens]), n, N):
        for t in range(first, first + rows):
            if heads:
                w = plain.rotate_axes(q64[t], pos[:, t], axis, freq, rot, pairs)
                g = got_q[t, :qrow].reshape(-1, D).astype(np.float64)
                assert (np.abs(g - w) <= near(w, True) + half * np.abs(w) + (2.0 ** -25 if dtype == "f16" else 0)).all(), (s, t)
            for h in range(H):
                r = plain.pool_row(table, s, cell0[s] + t - first, h, H, ps, n_pages, ld)
                if r >= 0:
                    written[r] = True
                    want["k"][r] = plain.rotate_axes(k64[t, h], pos[:, t], axis, freq, rot, pairs)
                    want["v"][r] = v64[t, h]
    for c in "kv":
        got = cache.dev[c].numpy().reshape(-1, D)
        assert (got[~written].view(np.uint8) == SENTINEL).all()
        idx = np.array(sorted(want[c]), np.int64)
        w = np.stack([want[c][r] for r in idx])
        if fmt == "f16":
            assert (np.abs(got[idx].astype(np.float64) - w) <= near(w, c == "k") + 2.0 ** -11 * np.abs(w) + 2.0 ** -25).all()
            continue
        scales = cache.dev[c + "s"].numpy().reshape(-1, D // 64)
        assert (scales[~written].view(np.uint8) == SENTINEL).all()
        step = scales[idx].view(np.float16).astype(np.float64).repeat(64, -1)
        top = np.abs(w).reshape(len(idx), -1, 64).max(-1).repeat(64, -1)
        assert (np.abs(step - top / 127) <= 2.0 ** -10.9 * top / 127 + 2.0 ** -25).all()
        assert (np.abs(plain.dequant(got[idx], scales[idx]) - w) <= 0.5001 * step + 2.0 ** -11 * top + near(w, True)).all()


@pytest.mark.parametrize("fmt", ["f16", "int8"])
def test_one_position_on_every_axis_is_the_append(sc, ops, cuda, fmt):
    """Where all axes say the cell, the caches and queries have sc_rope_append_async's bits; without cu too."""
    H, D, heads, n, ps = 2, 128, 4, 9, 4
    rng = np.random.default_rng(2)
    k, q = rng.standard_normal((n, H, D)).astype(np.float32), rng.standard_normal((n, heads, D)).astype(np.float32)
    cell0 = rng.integers(0, 40, n).astype(np.int64)
    kw = dict(n_seqs=n, tokens=n, pos0=upload(sc, cell0), inv_freq=upload(sc, _freq(D)), rot_dim=D, n_head=heads)
    got = []
    for axes in (False, True):
        cache = Cache(sc, ops, np.random.default_rng(4), fmt, H, D, ps, n, 10, fill="sentinel")
        dk, out = upload(sc, k), upload(sc, np.zeros_like(q))
        if axes:
            op = ops.RopeAxesAppend(cache.c, dk, dk, "f32", q=upload(sc, q), q_out=out, axis=ops.axis_of_pairs((24, 20, 20), True), n_axes=3,
                                    pos=upload(sc, np.stack([cell0] * 3)), **kw)
        else:
            op = ops.RopeAppend(cache.c, dk, dk, "f32", q=upload(sc, q), q_out=out, **kw)
        op.launch()
        sc.device_sync()
        got.append([out.numpy(), *(b.numpy() for b in cache.dev.values())])
    assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(*got))


def test_rows_outside_their_batch_and_cells_outside_the_table(sc, ops, cuda):
    """A row past the last sequence is left as it was; a cell before 0 or past the table is not written, its query is turned."""
    H, D, ps, ld = 1, 64, 4, 2
    rng = np.random.default_rng(3)
    cache = Cache(sc, ops, rng, "f16", H, D, ps, 3, ld, table=None, n_pages=6, fill="sentinel")
    k = rng.standard_normal((7, H, D)).astype(np.float32)
    out, dk = upload(sc, np.full((7, 1, D), 9.0, np.float32)), upload(sc, k)
    ops.RopeAxesAppend(cache.c, dk, dk, "f32", n_seqs=3, tokens=7, cu=upload(sc, np.array([0, 2, 4, 6])),
                       pos0=upload(sc, np.array([-1, 7, 1 << 40])), inv_freq=upload(sc, _freq(8)), rot_dim=8, axis=[0, 1, 1, 0], n_axes=2,
                       pos=upload(sc, rng.integers(0, 90, (2, 7))), q=dk, q_out=out, n_head=1).launch()
    sc.device_sync()
    got = cache.dev["v"].numpy().reshape(3, ld * ps, D)
    assert np.array_equal(got[0, 0], k[1, 0].astype(np.float16)) and np.array_equal(got[1, 7], k[2, 0].astype(np.float16))
    rest = np.ones(got.shape[:2], bool)
    rest[0, 0] = rest[1, 7] = False
    assert (got[rest].view(np.uint8) == SENTINEL).all()
    q = out.numpy()[:, 0]
    assert (q[6] == 9.0).all()
    assert np.array_equal(q[:6, 8:], k[:6, 0, 8:])
