"""sc_rope_append_async against the 64-bit implementation of the same operator.

What may differ is derived: an angle is formed in 64 bits and rounded to 32 within [-pi, pi] (2^-22.3 at most), its sine
and cosine are within 2 units of 2^-24, the two products and their sum within 3: below 2^-21 (|a| + |b|) for a pair.  An
f16 value adds half a unit of its 11 bits; an int8 value half a step of its scale, and 2^-11 of the largest value where
the scale's own rounding lets the largest code saturate."""
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
    # fmt, act, H, D, ps, n_head, rot, pairs, rows of each sequence, first positions
    ("f16", "f32", 2, 256, 4, 24, 64, "halves", [1], [4093]),
    ("f16", "f16", 2, 256, 4, 24, 256, "neighbours", [1, 1, 1], [0, 131070, 7]),
    ("f16", "f32", 1, 64, 1, 1, 64, "halves", [5, 0, 130], [0, 3, 61]),
    ("f16", "f32", 4, 128, 16, 4, 32, "neighbours", [33, 64, 1], [15, 16, 40000]),
    ("f16", "f16", 2, 256, 4, 0, 8, "halves", [7], [2]),
    ("f16", "f32", 3, 64, 3, 6, 0, "halves", [11], [5]),
    ("int8", "f32", 2, 256, 4, 24, 64, "halves", [700, 1], [3, 65533]),
    ("int8", "f16", 1, 64, 8, 16, 64, "neighbours", [1] * 70, list(range(0, 700, 10))),
    ("int8", "f32", 4, 128, 1, 32, 128, "halves", [3, 9], [0, 1]),
    ("int8", "f32", 2, 128, 5, 2, 0, "halves", [600], [1]),
    ("f16", "f16", 2, 64, 4, 5, 32, "neighbours", [511, 2], [9, 0]),
    ("f16", "f32", 1, 256, 16, 3, 256, "halves", [512], [100]),
]


@pytest.mark.parametrize("packed", [True, False], ids=["packed", "strided"])
@pytest.mark.parametrize("case", CASES, ids=[f"{c[0]}-{c[1]}-{c[2]}x{c[3]}-p{c[4]}-r{c[6]}{c[7][0]}-{len(c[8])}" for c in CASES])
def test_append_against_64_bits(sc, ops, plain, oracle, cuda, case, packed):
    fmt, dtype, H, D, ps, heads, rot, pairs, lens, pos0 = case
    print(f"append {case}", flush=True)
    rng = np.random.default_rng(len(lens) * 1000 + D + rot)
    n, N, ld = len(lens), sum(lens), max((p + t - 1) // ps + 1 for p, t in zip(pos0, lens))
    # only the pages that are written lie in the pool
    table = np.full((n, ld), -1, np.int32)
    used = [(s, p) for s in range(n) for p in range(pos0[s] // ps, (pos0[s] + lens[s] - 1) // ps + 1) if lens[s]]
    n_pages = len(used) + 2
    for (s, p), phys in zip(used, rng.permutation(n_pages)):
        table[s, p] = phys if rng.random() < 0.95 else -1
    cache = Cache(sc, ops, rng, fmt, H, D, ps, n, ld, table=table, n_pages=n_pages, fill="sentinel")
    k, k64 = act(rng.standard_normal((N, H, D)), dtype)
    v, v64 = act(rng.standard_normal((N, H, D)) * 3, dtype)
    q, q64 = act(rng.standard_normal((N, max(heads, 1), D)), dtype)
    pad = 0 if packed else 24
    row, qrow = H * D, max(heads, 1) * D
    dk, dv, dq = strided(sc, k, row + pad), strided(sc, v, row + 2 * pad), strided(sc, q, qrow + pad)
    dout = strided(sc, np.zeros_like(q), qrow + 2 * pad)
    cu = None if lens == [1] * n and packed else upload(sc, np.cumsum([0, *lens]).astype(np.int64))
    freq = _freq(rot)
    op = ops.RopeAppend(cache.c, dk, dv, dtype, n_seqs=n, tokens=N, cu=cu, pos0=upload(sc, np.array(pos0, np.int64)),
                        inv_freq=upload(sc, freq) if rot else None, rot_dim=rot, pairs=pairs, q=dq if heads else None,
                        q_out=dout if heads else None, n_head=heads, k_ld=row + pad, v_ld=row + 2 * pad, q_ld=qrow + pad,
                        q_out_ld=qrow + 2 * pad)
    op.launch()
    sc.device_sync()

    def near(x, turned):   # 2^-21 (|a| + |b|) of each value's pair, below 2^-20 of the head's largest
        return 2.0 ** -20 * np.abs(x).max(-1, keepdims=True) * (1 if turned and rot else 0) + 2.0 ** -60

    half = 2.0 ** -11 if dtype == "f16" else 2.0 ** -24
    got_q = dout.numpy()
    assert packed or between_rows_untouched(got_q, qrow)
    written = np.zeros(n_pages * H * ps, bool)
    want = {c: {} for c in "kv"}
    for s, first, rows in plain.rows_of(None if cu is None else np.cumsum([0, *lens]), n, N):
        for t in range(rows):
            pos = pos0[s] + t
            if heads:
                w = plain.rotate(q64[first + t], pos, freq, rot, pairs)
                g = got_q[first + t, :qrow].reshape(-1, D).astype(np.float64)
                assert (np.abs(g - w) <= near(w, True) + half * np.abs(w) + (2.0 ** -25 if dtype == "f16" else 0)).all(), (s, t)
            for h in range(H):
                r = plain.pool_row(table, s, pos, h, H, ps, n_pages, ld)
                if r >= 0:
                    written[r] = True
                    want["k"][r] = plain.rotate(k64[first + t, h], pos, freq, rot, pairs)
                    want["v"][r] = v64[first + t, h]
    for c in "kv":
        got = cache.dev[c].numpy().reshape(-1, D)
        assert (got[~written].view(np.uint8) == SENTINEL).all()
        idx = np.array(sorted(want[c]), np.int64)
        if not len(idx):
            continue
        w = np.stack([want[c][r] for r in idx])
        if fmt == "f16":
            if c == "v":
                assert np.array_equal(got[idx], w.astype(np.float16))
            assert (np.abs(got[idx].astype(np.float64) - w) <= near(w, c == "k") + 2.0 ** -11 * np.abs(w) + 2.0 ** -25).all()
            continue
        scales = cache.dev[c + "s"].numpy().reshape(-1, D // 64)
        assert (scales[~written].view(np.uint8) == SENTINEL).all()
        if c == "v" or not rot:   # values as they came: the same codes and scales as the carve's rule
            codes, sb = oracle.q8_rows(w.astype(np.float32))
            assert np.array_equal(got[idx], codes) and np.array_equal(scales[idx], sb)
        step = scales[idx].view(np.float16).astype(np.float64).repeat(64, -1)
        top = np.abs(w).reshape(len(idx), -1, 64).max(-1).repeat(64, -1)
        assert (np.abs(step - top / 127) <= 2.0 ** -10.9 * top / 127 + 2.0 ** -25).all()
        assert (np.abs(plain.dequant(got[idx], scales[idx]) - w) <= 0.5001 * step + 2.0 ** -11 * top + near(w, True)).all()


def test_values_that_are_no_numbers(sc, ops, oracle, cuda):
    """Infinities, NaN, the largest and the smallest values go where they belong, by the carve's rules."""
    H, D, ps, N = 2, 256, 4, 6
    x = np.random.default_rng(5).standard_normal((N, H, D)).astype(np.float32)
    x[0, 0, 3], x[0, 1, 64:128], x[1, 0, 9], x[1, 1] = np.nan, np.nan, np.inf, 0.0
    x[2, 0, 70], x[2, 1, :5], x[3, 0], x[4, 0] = -np.inf, 70000.0, x[3, 0] * 1e-6, -0.0
    for fmt in ("f16", "int8"):
        print(fmt, flush=True)
        cache = Cache(sc, ops, np.random.default_rng(1), fmt, H, D, ps, 1, 4, table=None, n_pages=4, fill="sentinel")
        dx = upload(sc, x)
        ops.RopeAppend(cache.c, dx, dx, "f32", n_seqs=1, tokens=N, cu=upload(sc, np.array([0, N])), pos0=upload(sc, np.array([5]))).launch()
        want = Cache(sc, ops, np.random.default_rng(1), fmt, H, D, ps, 1, 4, table=None, n_pages=4, fill="sentinel")
        d = want.dev
        f16 = fmt == "f16"
        sc.check(sc.lib.sc_kv_append_async(dx.ptr, dx.ptr, N, 5, None, ps, d["k"].ptr if f16 else None, d["v"].ptr if f16 else None,
                                           None if f16 else d["k"].ptr, None if f16 else d["v"].ptr, None if f16 else d["ks"].ptr,
                                           None if f16 else d["vs"].ptr, None, None, None), "append")
        sc.device_sync()
        for c in d:
            assert np.array_equal(cache.dev[c].numpy().view(np.uint8), d[c].numpy().view(np.uint8)), (fmt, c)


def test_rows_outside_their_batch_and_cells_outside_the_table(sc, ops, cuda):
    """A row past the last sequence, a position before 0 and one past the table write no cell; queries are turned anyway
    where a row belongs to a sequence."""
    H, D, ps, ld = 1, 64, 4, 2
    rng = np.random.default_rng(3)
    cache = Cache(sc, ops, rng, "f16", H, D, ps, 3, ld, table=None, n_pages=6, fill="sentinel")
    k = rng.standard_normal((7, H, D)).astype(np.float32)
    out = upload(sc, np.full((7, 1, D), 9.0, np.float32))
    dk = upload(sc, k)
    ops.RopeAppend(cache.c, dk, dk, "f32", n_seqs=3, tokens=7, cu=upload(sc, np.array([0, 2, 4, 6])),
                   pos0=upload(sc, np.array([-1, 7, 1 << 40])), inv_freq=upload(sc, _freq(8)), rot_dim=8, q=dk, q_out=out,
                   n_head=1).launch()
    sc.device_sync()
    got = cache.dev["v"].numpy().reshape(3, ld * ps, D)
    assert np.array_equal(got[0, 0], k[1, 0].astype(np.float16)) and np.array_equal(got[1, 7], k[2, 0].astype(np.float16))
    rest = np.ones(got.shape[:2], bool)
    rest[0, 0] = rest[1, 7] = False
    assert (got[rest].view(np.uint8) == SENTINEL).all()
    q = out.numpy()[:, 0]
    assert (q[6] == 9.0).all()
    assert np.array_equal(q[:6, 8:], k[:6, 0, 8:])


def test_queries_in_place_and_on_another_stream(sc, ops, cuda):
    """q_out may be q; a call waits for the work before it on its own stream."""
    H, D, N = 2, 128, 300
    rng = np.random.default_rng(8)
    q = rng.standard_normal((N, 4, D)).astype(np.float32)
    k = rng.standard_normal((N, H, D)).astype(np.float32)
    cu, pos0, freq = upload(sc, np.array([0, N])), upload(sc, np.array([17])), upload(sc, _freq(D))
    dk, got = upload(sc, k), []
    for place in ("apart", "in place"):
        cache = Cache(sc, ops, rng, "f16", H, D, 4, 1, 80, table=None, n_pages=80, fill="sentinel")
        staged, dq = upload(sc, q), upload(sc, np.zeros_like(q))
        out = dq if place == "in place" else upload(sc, np.zeros_like(q))
        stream = sc.Stream()
        sc.device_sync()
        sc.delay_async(2000, stream)
        sc.check(sc.lib.sc_copy_device_async(dq.ptr, staged.ptr, q.nbytes, stream.handle), "copy")
        ops.RopeAppend(cache.c, dk, dk, "f32", n_seqs=1, tokens=N, cu=cu, pos0=pos0, inv_freq=freq, rot_dim=D, q=dq, q_out=out,
                       n_head=4).launch(stream)
        stream.sync()
        got.append((out.numpy(), cache.dev["k"].numpy()))
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])
