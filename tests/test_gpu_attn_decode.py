"""sc_attn_decode_async against the 64-bit implementation of the same operator.

What may differ is derived.  A score is a sum of D products in 32 bits: its error stays below twice sqrt(256) 2^-24 = 2^-19
of the sum of the products' magnitudes, which moves a probability by that much of itself; probabilities carried as two f16
parts keep 2^-21.  So with e = 2^-19 max_j scale sum_d |q_d k_jd| + 2^-20, a value is within 2 e max |v| and lse within
e + 2^-22 |lse|; an f16 value adds half a unit of its 11 bits."""
import numpy as np
import pytest

from ops_cases import Cache, act, between_rows_untouched, strided, upload

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


@pytest.fixture(scope="module")
def plain():
    from oracle import sc_ops
    return sc_ops


def _check(plain, cache, q64, lens, window, scale, got, lse, dtype, seqs=None):
    n, heads, D = q64.shape
    K, V = cache.values("k"), cache.values("v")
    G = heads // cache.H
    for s in range(n) if seqs is None else seqs:
        L = min(max(int(lens[s]), 0), cache.ld * cache.ps)
        cells = range(max(0, L - window) if window else 0, L)
        for h in range(cache.H):
            rows = np.array([r for r in (plain.pool_row(cache.table, s, c, h, cache.H, cache.ps, cache.n_pages, cache.ld) for c in cells) if r >= 0], np.int64)
            k, v = K[rows], V[rows]
            for i in range(h * G, h * G + G):
                want, want_lse = plain.attention(q64[s, i], k, v, scale)
                e = 2.0 ** -20 + (2.0 ** -19 * scale * np.abs(k * q64[s, i]).sum(-1).max() if len(rows) else 0)
                tol = 2 * e * (np.abs(v).max() if len(rows) else 0) + (2.0 ** -11 * np.abs(want) + 2.0 ** -25 if dtype == "f16" else 0)
                assert (np.abs(got[s, i] - want) <= tol).all(), (s, i, np.abs(got[s, i] - want).max(), tol)
                if len(rows):
                    assert abs(lse[s, i] - want_lse) <= e + 2.0 ** -22 * abs(want_lse), (s, i)
                else:
                    assert lse[s, i] == -np.inf


CASES = [
    # fmt, act, H, D, heads, page size, lengths, window
    ("f16", "f32", 2, 256, 24, 4, [1], 0),
    ("f16", "f16", 2, 256, 24, 4, [0, 1, 2, 31, 32, 33, 127, 129], 0),
    ("f16", "f32", 2, 256, 24, 4, [5000, 3, 1021], 0),
    ("f16", "f32", 1, 128, 1, 1, [257, 64], 0),
    ("f16", "f16", 4, 64, 64, 16, [300, 999, 15], 0),
    ("f16", "f32", 3, 128, 9, 3, [100, 31, 1000], 0),
    ("f16", "f32", 1, 64, 40, 8, [333], 0),                 # more query heads to a kv head than a tile holds
    ("f16", "f16", 2, 128, 34, 5, [77, 500], 0),
    ("f16", "f32", 2, 256, 8, 4, [40, 900, 2000, 7], 100),
    ("int8", "f32", 2, 256, 24, 4, [0, 1, 65, 700, 4097], 0),
    ("int8", "f16", 2, 256, 24, 4, [3000, 130], 0),
    ("int8", "f32", 1, 64, 16, 1, [129, 64, 500], 0),
    ("int8", "f16", 4, 128, 8, 8, [511, 90], 33),
    ("int8", "f32", 2, 128, 2, 6, [400], 0),
]


@pytest.mark.parametrize("missing", [0.0, 0.3], ids=["whole", "holes"])
@pytest.mark.parametrize("case", CASES, ids=[f"{c[0]}-{c[1]}-{c[2]}x{c[3]}-{c[4]}-p{c[5]}-{max(c[6])}w{c[7]}" for c in CASES])
def test_attention_against_64_bits(sc, ops, plain, cuda, case, missing):
    fmt, dtype, H, D, heads, ps, lens, window = case
    print(f"attention {case} missing {missing}", flush=True)
    rng = np.random.default_rng(sum(lens) + D + heads)
    n, ld = len(lens), -(-max(lens) // ps)
    cache = Cache(sc, ops, rng, fmt, H, D, ps, n, max(ld, 1), missing=missing)
    q, q64 = act(rng.standard_normal((n, heads, D)) * 2, dtype)
    pad = 16 if missing else 0
    dq, out = strided(sc, q, heads * D + pad), strided(sc, np.zeros_like(q), heads * D + 2 * pad)
    lse = upload(sc, np.zeros((n, heads), np.float32))
    op = ops.AttnDecode(cache.c, dq, out, dtype, n_seqs=n, n_head=heads, lens=upload(sc, np.array(lens, np.int64)),
                        max_len=max(ld, 1) * ps if missing else max(max(lens), 0), scale=D ** -0.5, window=window, lse=lse, q_ld=heads * D + pad,
                        out_ld=heads * D + 2 * pad)
    op.launch()
    sc.device_sync()
    got, got_lse = out.numpy(), lse.numpy()
    assert not pad or between_rows_untouched(got, heads * D)
    _check(plain, cache, q64, lens, window, D ** -0.5, got[:, :heads * D].reshape(n, heads, D).astype(np.float64), got_lse, dtype)
    op.launch()
    sc.device_sync()
    assert np.array_equal(out.numpy().view(np.uint8), got.view(np.uint8)) and np.array_equal(lse.numpy().view(np.uint8), got_lse.view(np.uint8))


def _run(sc, ops, cache, q, dtype, lens, max_len, window=0):
    n, heads, D = q.shape
    out, lse = upload(sc, np.full_like(q, 7)), upload(sc, np.full((n, heads), 7, np.float32))
    ops.AttnDecode(cache.c, upload(sc, q), out, dtype, n_seqs=n, n_head=heads, lens=upload(sc, np.array(lens, np.int64)), max_len=max_len,
                   scale=D ** -0.5, window=window, lse=lse).launch()
    sc.device_sync()
    return out.numpy(), lse.numpy()


@pytest.mark.parametrize("fmt", ["f16", "int8"])
def test_a_long_cache_and_a_loose_bound(sc, ops, plain, cuda, fmt):
    """Many parts of one sequence, with short ones beside it, and a bound far above every length."""
    rng = np.random.default_rng(11)
    H, D, heads, ps, lens = 2, 128, 16, 4, [20011, 1, 0, 700]
    cache = Cache(sc, ops, rng, fmt, H, D, ps, len(lens), 6000)
    q, q64 = act(rng.standard_normal((len(lens), heads, D)) * 3, "f32")
    got, lse = _run(sc, ops, cache, q, "f32", lens, 24000)
    _check(plain, cache, q64, lens, 0, D ** -0.5, got.astype(np.float64), lse, "f32")


def test_many_sequences(sc, ops, plain, cuda):
    """More sequences than lanes, ragged, some empty: every one its own cells."""
    rng = np.random.default_rng(12)
    n, H, D, heads, ps = 200, 1, 64, 4, 4
    lens = rng.integers(0, 90, n)
    cache = Cache(sc, ops, rng, "f16", H, D, ps, n, 24)
    q, q64 = act(rng.standard_normal((n, heads, D)), "f32")
    got, lse = _run(sc, ops, cache, q, "f32", lens, 96)
    _check(plain, cache, q64, lens, 0, D ** -0.5, got.astype(np.float64), lse, "f32")


def test_lengths_outside_their_bounds(sc, ops, plain, cuda):
    """A negative length is an empty sequence; one past max_len counts as max_len."""
    rng = np.random.default_rng(13)
    cache = Cache(sc, ops, rng, "f16", 2, 64, 4, 3, 10)
    q, q64 = act(rng.standard_normal((3, 4, 64)), "f32")
    got, lse = _run(sc, ops, cache, q, "f32", [-5, 1 << 50, 40], 37)
    _check(plain, cache, q64, [0, 37, 37], 0, 64 ** -0.5, got.astype(np.float64), lse, "f32")


@pytest.mark.parametrize("fmt", ["f16", "int8"])
def test_what_lies_outside_a_sequence_does_not_matter(sc, ops, plain, cuda, fmt):
    """NaN and infinities in the cells past a length, before a window, in the rest of a page, in unmapped pages."""
    rng = np.random.default_rng(14)
    H, D, heads, ps, lens, window = 2, 256, 24, 4, [1, 30, 77, 0], 21
    cache = Cache(sc, ops, rng, fmt, H, D, ps, 4, 25, missing=0.2)
    cache.table[3] = -1
    cache.table[1, 9 // ps:] = -1                # nothing of its window (cells 9 to 29) is resident
    cache.t_dev.upload(cache.table)
    q, q64 = act(rng.standard_normal((4, heads, D)), "f32")
    read = set()
    for s, L in enumerate(lens):
        for c in range(max(0, L - window), L):
            read |= {plain.pool_row(cache.table, s, c, h, H, ps, cache.n_pages, 25) for h in range(H)}
    other = np.array([r for r in range(len(cache.host["k"])) if r not in read])
    for c in ("k", "v"):
        if fmt == "f16":
            cache.host[c][other] = np.where(rng.random((len(other), D)) < 0.5, np.nan, np.inf)
        else:
            cache.host[c + "s"][other] = rng.choice([0x7E00, 0x7C00, 0xFC00], (len(other), D // 64))
        for name in cache.dev:
            cache.dev[name].upload(cache.host[name])
    got, lse = _run(sc, ops, cache, q, "f32", lens, 100, window)
    clean = Cache.__new__(Cache)
    clean.__dict__.update(cache.__dict__)
    clean.host = {n: x.copy() for n, x in cache.host.items()}
    for c in ("k", "v"):
        clean.host[c if fmt == "f16" else c + "s"][other] = 0
    _check(plain, clean, q64, lens, window, D ** -0.5, got.astype(np.float64), lse, "f32")
    assert (got[1] == 0).all() and (got[3] == 0).all()


def test_large_scores_and_cells_that_weigh_nothing(sc, ops, plain, cuda):
    """Scores in the thousands (only differences count), keys of -inf weight, and a sequence all of whose scores are -inf."""
    rng = np.random.default_rng(15)
    H, D, heads, ps = 1, 64, 3, 4
    cache = Cache(sc, ops, rng, "f16", H, D, ps, 2, 20, table=None, n_pages=40)
    cache.host["k"] = (cache.host["k"].astype(np.float32) * 200).astype(np.float16)
    cache.host["k"][5, 0] = -np.inf
    cache.host["k"][80:, 0] = -np.inf
    cache.dev["k"].upload(cache.host["k"])
    q = rng.standard_normal((2, heads, D)).astype(np.float32) * 20
    q[:, :, 0] = np.abs(q[:, :, 0]) + 1
    got, lse = _run(sc, ops, cache, q, "f32", [80, 80], 80)
    K, V = cache.host["k"].astype(np.float64), cache.host["v"].astype(np.float64)
    keep = np.arange(80) != 5
    for i in range(heads):
        want, want_lse = plain.attention(q[0, i], K[:80][keep], V[:80][keep], D ** -0.5)
        e = 2.0 ** -20 + 2.0 ** -19 * np.abs(K[:80][keep] * q[0, i]).sum(-1).max() * D ** -0.5
        assert (np.abs(got[0, i] - want) <= 2 * e * np.abs(V).max()).all() and abs(lse[0, i] - want_lse) <= e + 2.0 ** -22 * abs(want_lse)
    assert (got[1] == 0).all() and (lse[1] == -np.inf).all()


def test_a_number_that_is_none_shows(sc, ops, cuda):
    """A NaN inside a sequence reaches the heads that read it, and no other sequence."""
    rng = np.random.default_rng(16)
    cache = Cache(sc, ops, rng, "f16", 2, 128, 4, 2, 40, table=None, n_pages=80)
    cache.host["k"].reshape(80, 2, 4, 128)[9, 1, 2, 77] = np.nan
    cache.host["v"].reshape(80, 2, 4, 128)[3, 0, 1, 5] = np.nan
    for c in "kv":
        cache.dev[c].upload(cache.host[c])
    got, _ = _run(sc, ops, cache, rng.standard_normal((2, 8, 128)).astype(np.float32), "f32", [160, 160], 160)
    assert np.isnan(got[0, 4:]).all() and np.isnan(got[0, :4, 5]).all()
    assert np.isfinite(np.delete(got[0, :4], 5, -1)).all() and np.isfinite(got[1]).all()


def test_row_offsets_past_32_bits(sc, ops, plain, cuda):
    """A pool whose rows pass 4 GiB: the cells of a short sequence at its very end."""
    rng = np.random.default_rng(17)
    H, D, ps, n_pages = 2, 256, 4, (1 << 32) // (2 * 4 * 256 * 2) + 8
    pools = [sc.DeviceBuffer(n_pages * H * ps * D, "uint16") for _ in range(2)]
    pages = [n_pages - 1, 0, n_pages - 3]
    small = {c: rng.standard_normal((3, H * ps * D)).astype(np.float16) for c in "kv"}
    for c, p in zip("kv", pools):
        for i, page in enumerate(pages):
            p.upload(small[c][i].view(np.uint16), page * H * ps * D)
    c = ops.kv_cache(*pools, n_pages=n_pages, n_head_kv=H, head_dim=D, page_size=ps, table=upload(sc, np.array(pages, np.int32)), table_ld=3)
    q = rng.standard_normal((1, 4, D)).astype(np.float32)
    out = upload(sc, np.zeros_like(q))
    ops.AttnDecode(c, upload(sc, q), out, "f32", n_seqs=1, n_head=4, lens=upload(sc, np.array([11])), max_len=12, scale=D ** -0.5).launch()
    sc.device_sync()
    rows = {c: x.reshape(3, H, ps, D).transpose(1, 0, 2, 3).reshape(H, 12, D)[:, :11].astype(np.float64) for c, x in small.items()}
    for i in range(4):
        want, _ = plain.attention(q[0, i], rows["k"][i // 2], rows["v"][i // 2], D ** -0.5)
        e = 2.0 ** -20 + 2.0 ** -19 * np.abs(rows["k"][i // 2] * q[0, i]).sum(-1).max() * D ** -0.5
        assert (np.abs(out.numpy()[0, i] - want) <= 2 * e * np.abs(rows["v"]).max()).all()


def test_the_parts_join(sc, ops, plain, cuda):
    """Two calls over the two halves of a cache join by their lse to the whole."""
    rng = np.random.default_rng(18)
    H, D, ps, heads = 2, 128, 4, 8
    cache = Cache(sc, ops, rng, "f16", H, D, ps, 1, 100)
    q, _ = act(rng.standard_normal((1, heads, D)), "f32")
    whole, whole_lse = _run(sc, ops, cache, q, "f32", [400], 400)
    table, parts = cache.table.copy(), []
    for half in (np.s_[:, :50], np.s_[:, 50:]):
        cache.table = np.full_like(table, -1)
        cache.table[half] = table[half]
        cache.t_dev.upload(cache.table)
        parts.append(_run(sc, ops, cache, q, "f32", [400], 400))
    w = np.exp(np.stack([p[1] for p in parts]).astype(np.float64) - whole_lse)
    assert np.abs(w.sum(0) - 1).max() < 2.0 ** -17
    joined = sum(x[..., None] * p[0] for x, p in zip(w, parts))
    assert np.abs(joined - whole).max() < 2.0 ** -16
