"""sc_attn_decode_async where a few cells outweigh the rest, and where what little the rest weighs is what counts.

What may differ is derived, in the output's own size.  A score's error e (a sum of D products in 32 bits: 2^-19 of the sum of
the products' magnitudes) moves its weight by that much of itself, and so at most moves the sum of the weights; weights
carried as two rounded f16 parts keep 2^-23 of themselves, sums in 32 bits of either sign 2^-21.  So a value is within
2 (e + 2^-20) of sum_j w_j |v_j| / sum_j w_j: small where the cells that weigh much have small values."""
import numpy as np
import pytest

from ops_cases import Cache, act, upload

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


def _run(sc, ops, cache, q, lens, max_len, window=0):
    n, heads, D = q.shape
    out, lse = upload(sc, np.full_like(q, 7)), upload(sc, np.full((n, heads), 7, np.float32))
    ops.AttnDecode(cache.c, upload(sc, q), out, "f16" if q.dtype == np.float16 else "f32", n_seqs=n, n_head=heads,
                   lens=upload(sc, np.array(lens, np.int64)), max_len=max_len, scale=D ** -0.5, window=window, lse=lse).launch()
    sc.device_sync()
    return out.numpy(), lse.numpy()


def _rows(cache, n):
    """[n][kv heads][D] of an identity cache's one sequence, in 64 bits."""
    pages = -(-n // cache.ps)
    at = lambda x: x.reshape(cache.n_pages, cache.H, cache.ps, -1)[:pages].transpose(0, 2, 1, 3).reshape(pages * cache.ps, cache.H, -1)[:n]  # noqa: E731
    return at(cache.values("k")), at(cache.values("v"))


def _check(cache, q, n, got, lse, half=0.0):
    k, v = _rows(cache, n)
    q64, G, D = q[0].astype(np.float64), q.shape[1] // cache.H, q.shape[2]
    for i in range(q.shape[1]):
        s = (k[:, i // G] @ q64[i]) * D ** -0.5
        w = np.exp(s - s.max())
        want, size = w @ v[:, i // G] / w.sum(), w @ np.abs(v[:, i // G]) / w.sum()
        e = 2.0 ** -20 + 2.0 ** -19 * D ** -0.5 * np.abs(k[:, i // G] * q64[i]).sum(-1).max()
        tol = 2 * e * size + half * np.abs(want)
        worst = (np.abs(got[0, i] - want) / tol).max()
        assert worst <= 1, (i, worst, (np.abs(got[0, i] - want) / size).max(), e)
        assert abs(lse[0, i] - (s.max() + np.log(w.sum()))) <= e + 2.0 ** -22 * abs(s.max() + np.log(w.sum()))


def _put(cache):
    for name in cache.dev:
        cache.dev[name].upload(cache.host[name])


def _sink(sc, ops, rng, fmt, H, D, heads, n, nats, at=0):
    """Cells whose first value of a key is what a query's first value meets only in cell `at`, `nats` above the rest there, with
    no value at all."""
    cache = Cache(sc, ops, rng, fmt, H, D, 4, 1, -(-n // 4), table=None, n_pages=-(-n // 4))
    q = (rng.standard_normal((1, heads, D)) * 0.5).astype(np.float32)
    q[0, :, 0] = 8.0
    k = cache.host["k"].reshape(-1, H, 4, D).transpose(0, 2, 1, 3).reshape(-1, H, D)
    v = cache.host["v"].reshape(-1, H, 4, D).transpose(0, 2, 1, 3).reshape(-1, H, D)
    k[:, :, 0], k[at], v[at] = 0, 0, 0
    high = nats * D ** 0.5 / 8.0
    if fmt == "f16":
        k[at, :, 0] = high
    else:
        k[at, :, 0] = 127
        ks = cache.host["ks"].reshape(-1, H, 4, D // 64).transpose(0, 2, 1, 3).reshape(-1, H, D // 64)
        ks[at, :, 0] = np.float16(high / 127).view(np.uint16)
        cache.host["ks"] = np.ascontiguousarray(ks.reshape(-1, 4, H, D // 64).transpose(0, 2, 1, 3)).reshape(-1, D // 64)
    for c, x in (("k", k), ("v", v)):
        cache.host[c] = np.ascontiguousarray(x.reshape(-1, 4, H, D).transpose(0, 2, 1, 3)).reshape(-1, D)
    _put(cache)
    return cache, q


SINKS = [("f16", 2, 256, 24), ("int8", 2, 256, 24), ("f16", 1, 64, 4), ("int8", 1, 128, 3), ("f16", 2, 128, 40)]


@pytest.mark.parametrize("n,at", [(5, 0), (32, 3), (33, 32), (300, 0), (8192, 0), (8192, 5000)])
@pytest.mark.parametrize("nats", [4, 11, 14, 20, 40])
@pytest.mark.parametrize("case", SINKS, ids=[f"{c[0]}-{c[1]}x{c[2]}-{c[3]}" for c in SINKS])
def test_a_cell_that_outweighs_the_rest(sc, ops, cuda, case, nats, n, at):
    fmt, H, D, heads = case
    print(f"sink {case} {nats} nats, {n} cells, cell {at}", flush=True)
    cache, q = _sink(sc, ops, np.random.default_rng(n + nats), fmt, H, D, heads, n, nats, at)
    got, lse = _run(sc, ops, cache, q, [n], -(-n // 4) * 4)
    _check(cache, q, n, got.astype(np.float64), lse)


def test_a_batch_of_sinks_with_one_part_each(sc, ops, cuda):
    """Enough sequences for one workgroup each: the wave that has the sink has most of the other cells too."""
    rng = np.random.default_rng(3)
    n, seqs = 2000, 160
    cache, q = _sink(sc, ops, rng, "f16", 2, 128, 16, n, 14)
    table = upload(sc, np.tile(np.arange(500, dtype=np.int32), (seqs, 1)))
    cache.c.table, cache.c.table_ld = table.data_ptr(), 500
    qs = np.repeat(q, seqs, 0) * (1 + np.arange(seqs, dtype=np.float32)[:, None, None] / 1024)
    got, lse = _run(sc, ops, cache, qs, [n] * seqs, n)
    for s in range(0, seqs, 13):
        _check(cache, qs[s:s + 1], n, got[s:s + 1].astype(np.float64), lse[s:s + 1])


@pytest.mark.parametrize("nats", [0, 9])
def test_blocks_of_other_sizes(sc, ops, cuda, nats):
    """int8 values whose blocks' scales are far apart, in a cell and from cell to cell, some of them zero."""
    rng = np.random.default_rng(4)
    n, H, D, heads = 1000, 2, 256, 24
    cache, q = _sink(sc, ops, rng, "int8", H, D, heads, n, nats)
    size = np.exp2(rng.integers(-12, 3, (len(cache.host["v"]), D // 64)) - np.array([0, 12, 6, 0]))
    size[rng.random(size.shape) < 0.05] = 0
    cache.host["vs"] = (size * (1 + rng.random(size.shape))).astype(np.float16).view(np.uint16)
    _put(cache)
    got, lse = _run(sc, ops, cache, q, [n], 1000)
    _check(cache, q, n, got.astype(np.float64), lse)


@pytest.mark.parametrize("fmt", ["f16", "int8"])
def test_values_that_are_all_one(sc, ops, cuda, fmt):
    """What is left out of a weight shows on either side: each result is one within 2^-20 (a few roundings), and their mean, of
    roundings of either sign, within 2^-24."""
    rng = np.random.default_rng(5)
    n, H, D, heads = 5, 2, 64, 512
    cache = Cache(sc, ops, rng, fmt, H, D, 4, 1, 2, table=None, n_pages=2)
    if fmt == "f16":
        cache.host["v"][:] = 1
    else:
        cache.host["v"][:], cache.host["vs"][:] = 64, np.float16(1 / 64).view(np.uint16)
    _put(cache)
    got, _ = _run(sc, ops, cache, rng.standard_normal((1, heads, D)).astype(np.float32), [n], 8)
    off = got[0, :, 0].astype(np.float64) - 1
    assert np.abs(off).max() <= 2.0 ** -20 and abs(off.mean()) <= 2.0 ** -24, (np.abs(off).max(), off.mean())


@pytest.mark.parametrize("nats", [0, 12, 30, 60])
def test_infinite_values_that_are_attended(sc, ops, cuda, nats):
    """A weight that is not zero times an infinity is an infinity, however little it weighs; of either sign together, or times
    a value that is no number, none.  The other values are what they are without it."""
    rng = np.random.default_rng(6)
    n, H, D, heads = 200, 2, 128, 8
    cache, q = _sink(sc, ops, rng, "f16", H, D, heads, n, nats)
    clean, _ = _run(sc, ops, cache, q, [n], 200)
    v = cache.host["v"].reshape(-1, H, 4, D)
    v[7, :, 1, 3], v[31, :, 2, 5], v[40, :, 0, 9], v[2, :, 3, 9], v[11, :, 0, 100] = np.inf, -np.inf, np.inf, -np.inf, np.nan
    cache.dev["v"].upload(cache.host["v"])
    got, _ = _run(sc, ops, cache, q, [n], 200)
    assert (got[0, :, 3] == np.inf).all() and (got[0, :, 5] == -np.inf).all()
    assert np.isnan(got[0, :, 9]).all() and np.isnan(got[0, :, 100]).all()
    cache.host["v"].reshape(-1, H, 4, D)[..., [3, 5, 9, 100]] = 0   # what is left
    rest = np.delete(np.arange(D), [3, 5, 9, 100])
    k, v = _rows(cache, n)
    for i in range(heads):
        s = (k[:, i // 4] @ q[0, i].astype(np.float64)) * D ** -0.5
        w = np.exp(s - s.max())
        e = 2.0 ** -20 + 2.0 ** -19 * D ** -0.5 * np.abs(k[:, i // 4] * q[0, i]).sum(-1).max()
        tol = 2 * e * (w @ np.abs(v[:, i // 4]) / w.sum())
        assert (np.abs(got[0, i] - w @ v[:, i // 4] / w.sum()) <= tol)[rest].all()
        assert (np.abs(clean[0, i] - w @ v[:, i // 4] / w.sum()) <= tol)[rest].all()


def test_scales_that_are_infinite(sc, ops, cuda):
    """int8 rows with an infinite scale: codes that are not zero are infinities of their sign, zeros are no numbers."""
    rng = np.random.default_rng(7)
    n, H, D, heads = 100, 1, 64, 4
    cache, q = _sink(sc, ops, rng, "int8", H, D, heads, n, 3)
    cache.host["vs"].reshape(-1, 4)[9, 2] = 0x7C00
    codes = rng.integers(1, 127, D).astype(np.int8)
    codes[1::2] *= -1
    codes[10] = 0
    cache.host["v"].reshape(-1, 4, D)[9, 2] = codes
    _put(cache)
    got, _ = _run(sc, ops, cache, q, [n], 100)
    want = np.where(codes == 0, np.nan, np.where(codes > 0, np.inf, -np.inf))
    assert np.array_equal(got[0], np.tile(want, (heads, 1)).astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("size", [2.0 ** 3, 2.0 ** 17, 2.0 ** 24, 2.0 ** 60])
def test_scores_beyond_all_measure(sc, ops, cuda, size):
    """Scores so far apart that only the largest counts, up to where a step of 32 bits is more than any weight's range; and the
    same upside down, where the first cell is the largest.  Which cell that is no score's error changes: 2^-19 of its value."""
    rng = np.random.default_rng(9)
    n, H, D, heads = 150, 1, 64, 3
    cache = Cache(sc, ops, rng, "f16", H, D, 4, 1, 38, table=None, n_pages=38)
    cache.host["k"][:] = 0
    cache.host["k"].reshape(-1, 4, D)[:, :, 0] = (256 * np.arange(152)).reshape(-1, 4)
    _put(cache)
    q = np.zeros((1, heads, D), np.float32)
    q[0, :, 0] = [size, -size, 0]
    got, lse = _run(sc, ops, cache, q, [n], 152)
    v = cache.values("v")
    assert (np.abs(got[0, 0] - v[n - 1]) <= 2.0 ** -19 * np.abs(v[n - 1])).all() and (np.abs(got[0, 1] - v[0]) <= 2.0 ** -19 * np.abs(v[0])).all()
    assert abs(lse[0, 0] / (256 * (n - 1) * size * D ** -0.5) - 1) < 2.0 ** -22 and lse[0, 1] == 0
    assert np.abs(got[0, 2] - v[:n].mean(0)).max() < 2.0 ** -19


@pytest.mark.parametrize("fmt", ["f16", "int8"])
def test_queries_and_keys_of_many_sizes(sc, ops, cuda, fmt):
    """A value of a query a million times smaller than its largest, where the keys are as much larger: the products count."""
    rng = np.random.default_rng(8)
    n, H, D, heads = 90, 1, 128, 8
    cache = Cache(sc, ops, rng, fmt, H, D, 4, 1, 23, table=None, n_pages=23)
    q = rng.standard_normal((1, heads, D)).astype(np.float32)
    if fmt == "f16":
        k = cache.host["k"].astype(np.float32) / 16
        k[:, 0] = rng.uniform(-60000, 60000, len(k))
        cache.host["k"] = k.astype(np.float16)
        q[0, :, 0] = 1.37 * 2.0 ** -16
    else:
        cache.host["ks"][:, 0] = np.float16(500).view(np.uint16)
        cache.host["ks"][:, 1] = np.float16(0.001).view(np.uint16)
        q[0, :, :64] *= 2.0 ** -16
    _put(cache)
    got, lse = _run(sc, ops, cache, q, [n], 92)
    _check(cache, q, n, got.astype(np.float64), lse)


@pytest.mark.parametrize("fmt", ["f16", "int8"])
def test_infinite_queries(sc, ops, cuda, fmt):
    """An infinite value of a query makes every score an infinity of its key's sign: nothing is left where they are all negative,
    no number where one is positive; values next to it that f16 does not hold change nothing."""
    rng = np.random.default_rng(10)
    n, H, D, heads = 40, 1, 64, 3
    cache = Cache(sc, ops, rng, fmt, H, D, 4, 1, 10, table=None, n_pages=10)
    cache.host["k"][:, 5] = -1 - np.arange(40) % 3
    cache.host["k"][:, 6] = 1
    _put(cache)
    q = (rng.standard_normal((1, heads, D)) * 1e6).astype(np.float32)
    q[0, 0, 5], q[0, 1, 5], q[0, 2, 5] = np.inf, -np.inf, 1
    got, lse = _run(sc, ops, cache, q, [n], 40)
    assert (got[0, 0] == 0).all() and lse[0, 0] == -np.inf
    assert np.isnan(got[0, 1]).all() and np.isfinite(got[0, 2]).all()


@pytest.mark.parametrize("fmt", ["f16", "int8"])
def test_few_cells_as_32_bits_have_them(sc, ops, cuda, fmt):
    """The root of the mean squared error of 5 cells' outputs, relative to sum w |v| / sum w.  A weight's parts: its score's sum and
    scaling (a score of one: 2^-23.6), the difference from the reference (at most 4: 2^-24.3), the exponential (2^-24.7), its two f16
    parts (2^-25), together 2^-23.1, of five cells with weights of like size half as much; 2^-23.5 leaves the rest to the sums."""
    rng = np.random.default_rng(11)
    n, H, D, heads = 5, 2, 64, 1024
    cache = Cache(sc, ops, rng, fmt, H, D, 4, 1, 2, table=None, n_pages=2)
    q = rng.standard_normal((1, heads, D)).astype(np.float32)
    got, _ = _run(sc, ops, cache, q, [n], 8)
    k, v = _rows(cache, n)
    off = []
    for i in range(heads):
        s = (k[:, i // 512] @ q[0, i].astype(np.float64)) * D ** -0.5
        w = np.exp(s - s.max())
        off.append((got[0, i] - w @ v[:, i // 512] / w.sum()) / (w @ np.abs(v[:, i // 512]) / w.sum()))
    rms = np.sqrt(np.mean(np.square(off)))
    assert rms <= 2.0 ** -23.5, np.log2(rms)


@pytest.mark.parametrize("n,at", [(1, 0), (200, 0), (200, 150)])
@pytest.mark.parametrize("fmt", ["f16", "int8"])
def test_small_logs_of_sums(sc, ops, cuda, fmt, n, at):
    """lse where one cell has nearly all the weight and a score near zero.  The score is one product and exact but for its scaling
    (three roundings), which is of its own size, as the end's two roundings are: 2^-22 of it.  The exponential is within 2^-23
    of itself, its mantissa's logarithm within 2^-24, the difference from the reference within 2^-24: 2^-22 together."""
    rng = np.random.default_rng(12)
    H, D, heads = 2, 256, 512
    cache = Cache(sc, ops, rng, fmt, H, D, 4, 1, 50, table=None, n_pages=50)
    k = np.zeros((n, H), np.float32)
    k[:], k[at] = -100, 1
    rows = cache.host["k"].reshape(50, H, 4, D)
    rows[:] = 0
    if fmt == "int8":
        cache.host["ks"][:] = cache.host["vs"][:] = np.float16(1).view(np.uint16)
    for c in range(n):
        rows[c // 4, :, c % 4, 3] = k[c]
    _put(cache)
    q = np.zeros((1, heads, D), np.float32)
    q[0, :, 3] = 8 + rng.random(heads) * 8
    q[0, :, 3] *= np.where(rng.random(heads) < 0.5, 1, -1) if n == 1 else 1
    _, lse = _run(sc, ops, cache, q, [n], n)
    want = q[0, :, 3].astype(np.float64) * D ** -0.5   # the others' weights are below e^-50
    off = np.abs(lse[0] - want)
    assert (off <= 2.0 ** -22 * np.abs(want) + 2.0 ** -22).all(), (off / (2.0 ** -22 * np.abs(want) + 2.0 ** -22)).max()
