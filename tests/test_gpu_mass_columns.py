"""Columns of sc_attn_mass_async that have no weight to give: those past the last query head of the last row, and queries whose
attention saw nothing (a log of -inf), whatever their values and the keys'.  Tolerances as in test_gpu_mass.py."""
import numpy as np
import pytest

from ops_cases import Cache, act, upload

pytestmark = pytest.mark.gpu

# rows, query heads, head size, act, cache; one kv head.  Up to 16 columns, and more of them, the last tile partly filled
SHAPES = [(1, 5, 64, "f32", "f16"), (2, 5, 128, "f16", "int8"), (4, 5, 64, "f16", "f16"), (3, 7, 64, "f32", "f16"), (4, 5, 128, "f16", "int8"),
          (3, 12, 256, "f16", "f16"), (5, 12, 256, "f32", "int8")]
IDS = ["-".join(map(str, s)) for s in SHAPES]


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


@pytest.fixture(scope="module")
def plain():
    from oracle import sc_ops
    return sc_ops


def _want(plain, K, q64, t, rows, scale, lse):
    """What each cell gets, and how far that may be off."""
    got, near, C = np.zeros(t), np.zeros(t), q64.shape[0] // rows * q64.shape[1] * rows
    for r in range(rows):
        seen = t - rows + 1 + r
        for i in range(q64.shape[1]):
            p = plain.attention_mass(q64[r, i], K[:seen], scale, float(lse[r, i]))
            e = 2.0 ** -19 * scale * np.abs(K[:seen] * q64[r, i]).sum(-1).max()
            got[:seen] += p
            near[:seen] += p * (2 * e + 2.0 ** -20 + C * 2.0 ** -24) + 2.0 ** -120
    return got, near + 2.0 ** -23 * got


def _run(sc, ops, cache, q, dtype, t, rows, heads, scale, lse):
    mass = upload(sc, np.full((1, 1, t), np.nan, np.float32))
    ops.AttnMass(cache.c, upload(sc, q), mass, dtype, n_seqs=1, n_head=heads, rows=rows, lens=upload(sc, np.array([t])), max_len=t, scale=scale,
                 lse=upload(sc, lse.astype(np.float32)), decay=0.0).launch()
    sc.device_sync()
    return mass.numpy().reshape(t)


@pytest.mark.parametrize("rows,heads,D,dtype,fmt", SHAPES, ids=IDS)
def test_an_infinite_score_under_given_sums(sc, ops, plain, cuda, rows, heads, D, dtype, fmt):
    """exp(inf - lse) is inf: a cell whose score is infinite gets that, and no column that there is none of makes it NaN."""
    t, bad, rng = 140, 37, np.random.default_rng(rows * heads)
    cache = Cache(sc, ops, rng, fmt, 1, D, 4, 1, 35)
    at = [plain.pool_row(cache.table, 0, c, 0, 1, 4, cache.n_pages, 35) for c in range(t)]
    q, q64 = act(np.abs(rng.standard_normal((rows, heads, D))) + 0.1, dtype)
    scale = float(np.float32(0.25 * D ** -0.5))
    k = cache.host["k"]
    k[at[bad]] = np.abs(k[at[bad]]) + 1 if fmt == "f16" else np.maximum(np.abs(k[at[bad]].astype(np.int16)), 1).astype(np.int8)
    K = cache.values("k")[at]
    s = scale * np.einsum("rid,cd->ric", q64, K)
    lse = np.log(np.exp(s - s.max(-1, keepdims=True)).sum(-1)) + s.max(-1)
    want, near = _want(plain, K, q64, t, rows, scale, lse.astype(np.float32))
    if fmt == "f16":
        k[at[bad], 3] = np.inf
    else:
        cache.host["ks"][at[bad]] = np.float16(np.inf).view(np.uint16)
    cache.dev["k"].upload(k)
    if fmt == "int8":
        cache.dev["ks"].upload(cache.host["ks"])
    got = _run(sc, ops, cache, q, dtype, t, rows, heads, scale, lse)
    others = np.arange(t) != bad
    assert got[bad] == np.inf, got[bad]
    assert (np.abs(got - want)[others] <= near[others]).all()


@pytest.mark.parametrize("rows,heads,D,dtype,fmt", SHAPES, ids=IDS)
def test_a_query_that_saw_nothing_gives_nothing(sc, ops, plain, cuda, rows, heads, D, dtype, fmt):
    """A log of -inf is a query without a weight (of a padded row, say): NaN and infinities in it reach no cell."""
    t, rng = 140, np.random.default_rng(rows + heads)
    cache = Cache(sc, ops, rng, fmt, 1, D, 4, 1, 35)
    at = [plain.pool_row(cache.table, 0, c, 0, 1, 4, cache.n_pages, 35) for c in range(t)]
    q, q64 = act(rng.standard_normal((rows, heads, D)), dtype)
    scale = float(np.float32(0.25 * D ** -0.5))
    K = cache.values("k")[at]
    s = scale * np.einsum("rid,cd->ric", q64, K)
    lse = np.log(np.exp(s - s.max(-1, keepdims=True)).sum(-1)) + s.max(-1)
    lse[0, 1] = lse[rows - 1, heads - 1] = lse[rows // 2, 0] = -np.inf
    want, near = _want(plain, K, q64, t, rows, scale, lse.astype(np.float32))
    q[0, 1], q[rows - 1, heads - 1], q[rows // 2, 0, 5] = np.nan, np.nan, np.inf
    got = _run(sc, ops, cache, q, dtype, t, rows, heads, scale, lse)
    assert (np.abs(got - want) <= near).all(), np.abs(got - want).max()


@pytest.mark.parametrize("rows,heads,D,dtype,fmt", [s for s in SHAPES if s[4] == "f16"], ids=[i for i, s in zip(IDS, SHAPES) if s[4] == "f16"])
def test_an_infinite_score_under_its_own_sum(sc, ops, plain, cuda, rows, heads, D, dtype, fmt):
    """The log of a sum with inf in it is inf: finite scores weigh exp(-inf) under it, the infinite one is NaN.  Where the sum is formed
    here every cell that the query sees is NaN, and none that it does not see."""
    t, bad, rng = 140, 139, np.random.default_rng(rows)
    cache = Cache(sc, ops, rng, fmt, 1, D, 4, 1, 35, missing=0.1)
    at = [plain.pool_row(cache.table, 0, c, 0, 1, 4, cache.n_pages, 35) for c in range(t)]
    if at[bad] < 0:   # the latest cell is there
        cache.table[0, 34] = next(p for p in range(cache.n_pages) if p not in cache.table[0])
        cache.t_dev.upload(cache.table)
        at = [plain.pool_row(cache.table, 0, c, 0, 1, 4, cache.n_pages, 35) for c in range(t)]
    q, q64 = act(np.abs(rng.standard_normal((rows, heads, D))) + 0.1, dtype)
    k = cache.host["k"]
    k[at[bad]] = np.abs(k[at[bad]]) + 1
    k[at[bad], 3] = np.inf
    cache.dev["k"].upload(k)
    lse = np.full((rows, heads), -np.inf)   # only the last row, the only one that sees the latest cell, has a weight
    lse[rows - 1] = np.inf
    scale = float(np.float32(0.25 * D ** -0.5))
    got = _run(sc, ops, cache, q, dtype, t, rows, heads, scale, lse)
    assert np.isnan(got[bad]) and not got[:bad].any()
    mass = upload(sc, np.zeros((1, 1, t + 3), np.float32))
    ops.AttnMass(cache.c, upload(sc, q), mass, dtype, n_seqs=1, n_head=heads, rows=rows, lens=upload(sc, np.array([t])), max_len=t, scale=scale,
                 mass_ld=t + 3).launch()
    sc.device_sync()
    got, there = mass.numpy().reshape(t + 3), np.array([r >= 0 for r in at])
    assert np.isnan(got[:t][there]).all() and not got[:t][~there].any() and not got[t:].any()
