"""sc_attn_mass_async against the 64-bit implementation of the same operator.

What may differ is derived.  A score is a sum of D products in 32 bits: its error stays below twice sqrt(256) 2^-24 = 2^-19 of the
sum of the products' magnitudes (f32 queries' parts and the three roundings of the scale among them: 2^-22 more of the score),
which moves a weight by that much of itself; where the sum of exponentials is formed here it moves by the largest of these errors
too.  With e = 2^-19 max_j scale sum_d |q_d k_jd|, a weight is within 2 e + 2^-20 of itself.  The weights of C columns are added
with C roundings of 2^-24 at most, the old mass with two."""
import numpy as np
import pytest

from ops_cases import Cache, act, strided, upload

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


@pytest.fixture(scope="module")
def plain():
    from oracle import sc_ops
    return sc_ops


def _cells(plain, cache, s, ends, window, h):
    """The cells that a row sees, and their pool rows."""
    cells = range(max(0, ends - window) if window else 0, max(ends, 0))
    rows = [(c, plain.pool_row(cache.table, s, c, h, cache.H, cache.ps, cache.n_pages, cache.ld)) for c in cells]
    rows = [(c, r) for c, r in rows if r >= 0]
    return np.array([c for c, _ in rows], np.int64), np.array([r for _, r in rows], np.int64)


def _want(plain, cache, q64, lens, rows, window, scale, lse):
    """The weights that each cell gets, and how far they may be off."""
    n, heads, D = len(lens), q64.shape[1], q64.shape[2]
    K, G = cache.values("k"), heads // cache.H
    most = max(max(lens), 1)
    got, near = np.zeros((n, cache.H, most)), np.zeros((n, cache.H, most))
    for s, t in enumerate(lens):
        for r in range(rows):
            for h in range(cache.H):
                cells, at = _cells(plain, cache, s, t - rows + 1 + r, window, h)
                for i in range(h * G, (h + 1) * G):
                    q, row = q64[s * rows + r, i], s * rows + r
                    p = plain.attention_mass(q, K[at], scale, None if lse is None else float(lse[row, i]))
                    e = 2.0 ** -19 * scale * np.abs(K[at] * q).sum(-1).max() if len(at) else 0
                    got[s, h, cells] += p
                    near[s, h, cells] += p * (2 * e + 2.0 ** -20 + rows * G * 2.0 ** -24) + 2.0 ** -120
    return got, near


def _sums(plain, cache, q64, lens, rows, window, scale):
    """The logs of the sums of exponentials, as an attention over the same cells leaves them."""
    heads, lse = q64.shape[1], np.full(q64.shape[:2], -np.inf, np.float32)
    K, G = cache.values("k"), heads // cache.H
    for s, t in enumerate(lens):
        for r in range(rows):
            for i in range(heads):
                _, at = _cells(plain, cache, s, t - rows + 1 + r, window, i // G)
                lse[s * rows + r, i] = plain.attention(q64[s * rows + r, i], K[at], K[at], scale)[1]
    return lse


CASES = [
    # fmt, act, H, D, ps, heads, lengths, rows, window, decay, pages missing
    ("f16", "f32", 2, 256, 4, 24, [1021], 1, 0, 1.0, 0.0),
    ("f16", "f16", 1, 64, 1, 1, [1, 0, 2, 33, 128, 129], 1, 0, 0.5, 0.0),
    ("int8", "f16", 2, 256, 4, 24, [300, 31], 1, 0, 1.0, 0.1),
    ("int8", "f32", 4, 128, 16, 32, [500], 3, 0, 0.0, 0.0),
    ("f16", "f16", 2, 256, 4, 24, [260, 20], 32, 0, 1.0, 0.0),
    ("f16", "f32", 2, 128, 3, 8, [400, 3, 0, 129], 5, 70, 1.0, 0.05),
    ("int8", "f32", 1, 256, 8, 3, [700], 2, 600, 0.9, 0.0),
    ("f16", "f16", 3, 64, 5, 51, [140, 141], 60, 0, 1.0, 0.0),
    ("int8", "f16", 2, 64, 4, 64, [200], 7, 1, 1.0, 0.3),
    ("f16", "f32", 1, 64, 4, 16, [333, 64], 64, 50, 0.0, 0.0),
    ("f16", "f32", 1, 128, 4, 5, [4000], 1, 0, 1.0, 0.0),
]


@pytest.mark.parametrize("given", [True, False], ids=["given", "formed"])
@pytest.mark.parametrize("case", CASES, ids=[f"{c[0]}-{c[1]}-{c[2]}x{c[3]}-h{c[5]}-{max(c[6])}-r{c[7]}-w{c[8]}" for c in CASES])
def test_against_64_bits(sc, ops, plain, cuda, case, given):
    fmt, dtype, H, D, ps, heads, lens, rows, window, decay, missing = case
    print(f"mass {case} {given}", flush=True)
    rng = np.random.default_rng(sum(lens) + D + rows)
    n, most = len(lens), max(lens)
    cache = Cache(sc, ops, rng, fmt, H, D, ps, n, -(-most // ps) + 1, missing=missing)
    q, q64 = act(rng.standard_normal((n * rows, heads, D)) * 1.5, dtype)
    scale = float(np.float32(D ** -0.5 * (0.5 if fmt == "int8" else 1.0)))
    lse = _sums(plain, cache, q64, lens, rows, window, scale) if given else None
    ld, bound = most + 9, most + 2 if (most + 2) <= cache.ld * ps else most
    mass = rng.random((n, H, ld)).astype(np.float32) * (rows * heads / H / most)
    if decay == 0:
        mass[...] = np.nan
    dmass, row = upload(sc, mass), heads * D
    ops.AttnMass(cache.c, strided(sc, q, row + 24), dmass, dtype, n_seqs=n, n_head=heads, lens=upload(sc, np.array(lens, np.int64)), max_len=bound,
                 scale=scale, rows=rows, window=window, lse=None if lse is None else upload(sc, lse), decay=decay, q_ld=row + 24,
                 mass_ld=ld).launch()
    sc.device_sync()
    got = dmass.numpy().reshape(mass.shape)
    add, near = _want(plain, cache, q64, lens, rows, window, scale, lse)
    for s, t in enumerate(lens):
        old = 0 if decay == 0 else decay * mass[s, :, :t].astype(np.float64)
        off = np.abs(got[s, :, :t] - (old + add[s, :, :t]))
        assert (off <= near[s, :, :t] + 2.0 ** -23 * (np.abs(old) + add[s, :, :t])).all(), (s, off.max())
        assert np.array_equal(got[s, :, t:].view(np.uint32), mass[s, :, t:].view(np.uint32)), s


@pytest.mark.parametrize("fmt", ["f16", "int8"])
def test_what_attention_left_and_what_is_formed_here(sc, ops, plain, cuda, fmt):
    """The attention's own sums give what the sums formed here give; the weights of a query add up to 1."""
    H, D, heads, lens = 2, 128, 8, [1500, 7, 0, 260]
    rng, n = np.random.default_rng(3), 4
    cache = Cache(sc, ops, rng, fmt, H, D, 4, n, 380)
    q, dlens = upload(sc, rng.standard_normal((n, heads, D)).astype(np.float32)), upload(sc, np.array(lens, np.int64))
    out, lse = sc.DeviceBuffer((n, heads, D), "float32"), sc.DeviceBuffer((n, heads), "float32")
    ops.AttnDecode(cache.c, q, out, "f32", n_seqs=n, n_head=heads, lens=dlens, max_len=1520, scale=D ** -0.5, lse=lse).launch()
    got = []
    for sums in (lse, None):
        mass = upload(sc, np.zeros((n, H, 1520), np.float32))
        ops.AttnMass(cache.c, q, mass, "f32", n_seqs=n, n_head=heads, lens=dlens, max_len=1520, scale=D ** -0.5, lse=sums).launch()
        sc.device_sync()
        got.append(mass.numpy().reshape(n, H, 1520))
    assert np.abs(got[0] - got[1]).max() <= 2.0 ** -16 * got[0].max()
    for s, t in enumerate(lens):
        assert (np.abs(got[1][s].sum(-1) - (heads // H if t else 0)) <= 2.0 ** -18 * heads).all() and not got[1][s, :, t:].any()


def test_far_scores_infinities_and_garbage_outside(sc, ops, plain, cuda):
    """Scores of hundreds keep their weights' bits; what lies outside a sequence or a window is not looked at; a row whose scores
    are all -inf gives nothing, and a cell of +inf score makes NaN where the formula does."""
    H, D, ps, heads, t = 1, 64, 4, 2, 100
    rng = np.random.default_rng(7)
    cache = Cache(sc, ops, rng, "f16", H, D, ps, 3, 40)
    rows = lambda s, c: plain.pool_row(cache.table, s, c, 0, H, ps, cache.n_pages, cache.ld)  # noqa: E731
    k = cache.host["k"]
    for s in range(3):
        for c in range(t, 160):
            k[rows(s, c)] = np.nan if c % 2 else np.inf
    for c in range(t):
        k[rows(1, c)] = np.abs(k[rows(1, c)])
        k[rows(1, c), 3] = -np.inf if c < 60 else 1.0
        k[rows(2, c), 3] = -np.inf
    cache.dev["k"].upload(k)
    q = rng.standard_normal((3, heads, D)).astype(np.float32)
    q[0] *= 40
    q[1], q[2] = np.abs(q[1]), np.abs(q[2])
    q[2, :, :3] = q[2, :, 4:] = 0.0
    k2 = np.zeros((t, D), np.float16)
    k2[:, 3] = -np.inf
    for c in range(t):
        k[rows(2, c)] = k2[c]
        k[rows(2, c), :3] = k[rows(2, c), 4:] = 1.0
    cache.dev["k"].upload(k)
    dq, dlens = upload(sc, q), upload(sc, np.array([t] * 3, np.int64))
    for sums in (False, True):
        lse = None
        if sums:
            lse = sc.DeviceBuffer((3, heads), "float32")
            lse.upload(_sums(plain, cache, q.astype(np.float64), [t] * 3, 1, 0, D ** -0.5))
        mass = upload(sc, np.full((3, H, 160), 5.0, np.float32))
        ops.AttnMass(cache.c, dq, mass, "f32", n_seqs=3, n_head=heads, lens=dlens, max_len=160, scale=D ** -0.5, lse=lse, decay=0.0).launch()
        sc.device_sync()
        got = mass.numpy().reshape(3, 160)
        K = cache.values("k")
        assert (got[:, t:] == 5).all() and (got[2, :t] == 0).all() and (got[1, :60] == 0).all()
        for s in (0, 1):
            at = np.array([rows(s, c) for c in range(t)])
            want = sum(plain.attention_mass(q[s, i], K[at], D ** -0.5) for i in range(heads))
            e = max(2.0 ** -19 * D ** -0.5 * np.abs(np.where(np.isinf(K[at]), 0, K[at]) * q[s, i]).sum(-1).max() for i in range(heads))
            # the sum's log that is given is itself rounded to 2^-24 of itself
            e += 2.0 ** -23 * np.abs(_sums(plain, cache, q.astype(np.float64), [t] * 3, 1, 0, D ** -0.5)[s]).max() if sums else 0
            assert (np.abs(got[s, :t] - want) <= want * (2 * e + 2.0 ** -19) + 2.0 ** -119).all(), s
    k[rows(0, 5)] = np.inf
    cache.dev["k"].upload(k)
    q[0] = np.abs(q[0])
    mass = upload(sc, np.zeros((3, H, 160), np.float32))
    ops.AttnMass(cache.c, upload(sc, q), mass, "f32", n_seqs=3, n_head=heads, lens=dlens, max_len=160, scale=D ** -0.5).launch()
    sc.device_sync()
    assert np.isnan(mass.numpy().reshape(3, 160)[0, 5])


def test_a_long_cache_in_parts(sc, ops, plain, cuda):
    """Long sequences whose sums are formed in parts of several turns each; a batch with many workgroups."""
    for lens, H, D, rows in (([70000, 100], 1, 64, 2), ([1300] * 40, 4, 64, 1)):
        print(lens[0], flush=True)
        rng, n, heads = np.random.default_rng(5), len(lens), 2 * H
        cache = Cache(sc, ops, rng, "f16", H, D, 16, n, -(-max(lens) // 16))
        q, q64 = act(rng.standard_normal((n * rows, heads, D)), "f16")
        mass = upload(sc, np.zeros((n, H, max(lens)), np.float32))
        ops.AttnMass(cache.c, upload(sc, q), mass, "f16", n_seqs=n, n_head=heads, lens=upload(sc, np.array(lens, np.int64)), max_len=max(lens),
                     scale=D ** -0.5, rows=rows).launch()
        sc.device_sync()
        add, near = _want(plain, cache, q64, lens, rows, 0, D ** -0.5, None)
        assert (np.abs(mass.numpy().reshape(add.shape) - add) <= near + 2.0 ** -23 * add).all()


def test_lengths_outside_their_bounds(sc, ops, plain, cuda):
    H, D, heads = 1, 64, 2
    rng = np.random.default_rng(5)
    cache = Cache(sc, ops, rng, "f16", H, D, 4, 3, 10)
    q, q64 = act(rng.standard_normal((3, heads, D)), "f32")
    mass = upload(sc, np.full((3, H, 40), 2.0, np.float32))
    ops.AttnMass(cache.c, upload(sc, q), mass, "f32", n_seqs=3, n_head=heads, lens=upload(sc, np.array([-3, 1 << 40, 39])), max_len=33,
                 scale=D ** -0.5, mass_ld=40).launch()
    sc.device_sync()
    add, near = _want(plain, cache, q64, [0, 33, 33], 1, 0, D ** -0.5, None)
    got = mass.numpy().reshape(3, H, 40)
    assert (got[0] == 2).all() and (got[:, :, 33:] == 2).all()
    assert (np.abs(got[1:, :, :33] - 2 - add[1:]) <= near[1:] + 2.0 ** -22).all()


def test_the_same_bits_again_and_on_another_stream(sc, ops, cuda):
    """A call waits for the work before it on its own stream, and gives the same bits every time."""
    H, D, heads, t, rows = 2, 256, 24, 3000, 9
    rng = np.random.default_rng(8)
    cache = Cache(sc, ops, rng, "f16", H, D, 4, 1, 750)
    q, got = rng.standard_normal((rows, heads, D)).astype(np.float32), []
    for late in (False, False, True):
        staged, dq = upload(sc, q), upload(sc, np.zeros_like(q) if late else q)
        mass, stream = upload(sc, np.zeros((1, H, t), np.float32)), sc.Stream()
        sc.device_sync()
        if late:
            sc.delay_async(2000, stream)
            sc.check(sc.lib.sc_copy_device_async(dq.ptr, staged.ptr, q.nbytes, stream.handle), "copy")
        ops.AttnMass(cache.c, dq, mass, "f32", n_seqs=1, n_head=heads, rows=rows, lens=upload(sc, np.array([t])), max_len=t,
                     scale=D ** -0.5).launch(stream)
        stream.sync()
        got.append(mass.numpy())
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


@pytest.mark.parametrize("rows,heads,dtype,fmt", [(1, 4, "f32", "f16"), (3, 4, "f16", "int8"), (32, 4, "f16", "f16"), (32, 2, "f32", "f16"), (20, 2, "f16", "int8")])
def test_a_row_that_is_no_number_stays_in_what_it_sees(sc, ops, plain, cuda, rows, heads, dtype, fmt):
    """A key that is NaN in the latest cell makes NaN of the cells that the latest row sees, and of no other: neither those before
    its window, which earlier rows see, nor those that are not resident, nor those past the end."""
    H, D, ps, t, window = 1, 64, 4, 200, 20
    for given in (False, True):
        got = []
        for bad in (False, True):
            rng = np.random.default_rng(31)
            table = rng.permutation(60)[:50].astype(np.int32).reshape(1, 50)
            table[0, (t - 10) // ps] = -1
            cache = Cache(sc, ops, rng, fmt, H, D, ps, 1, 50, table=table, n_pages=60)
            q, q64 = act(rng.standard_normal((rows, heads, D)), dtype)
            lse = _sums(plain, cache, q64, [t], rows, window, D ** -0.5)
            last = plain.pool_row(table, 0, t - 1, 0, H, ps, 60, 50)
            if bad and fmt == "f16":
                x = cache.host["k"]
                x[last, 5] = np.nan
                cache.dev["k"].upload(x)
            elif bad:
                x = cache.host["ks"]
                x[last] = 0x7E00
                cache.dev["ks"].upload(x)
            if bad:
                lse[rows - 1] = np.nan
            mass = upload(sc, np.zeros((1, H, 210), np.float32))
            ops.AttnMass(cache.c, upload(sc, q), mass, dtype, n_seqs=1, n_head=heads, rows=rows, lens=upload(sc, np.array([t])), max_len=t,
                         scale=D ** -0.5, window=window, lse=upload(sc, lse) if given else None, mass_ld=210).launch()
            sc.device_sync()
            got.append(mass.numpy().reshape(210))
        clean, odd = got
        seen = np.zeros(210, bool)
        seen[t - window:t] = True
        seen[(t - 10) // ps * ps:(t - 10) // ps * ps + ps] = False
        assert np.isfinite(clean).all() and np.isnan(odd[seen]).all()
        assert np.array_equal(odd[~seen], clean[~seen]), (given, np.flatnonzero(odd[~seen] != clean[~seen]))
