"""sc_kv_evict_async against a plain implementation: which cells are kept, where they go, and that nothing else is touched.
Rows are moved, so everything is equal to the last bit."""
import numpy as np
import pytest

from ops_cases import Cache, upload

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


@pytest.fixture(scope="module")
def plain():
    from oracle import sc_ops
    return sc_ops


def _mass(rng, kind, shape):
    if kind == "spread":
        return np.exp2(rng.standard_normal(shape) * 8).astype(np.float32)
    if kind == "few":       # many equal ones
        return rng.integers(0, 3, shape).astype(np.float32)
    if kind == "none":
        return np.zeros(shape, np.float32)
    if kind == "late":      # all that is kept lies behind what is kept
        return np.broadcast_to(np.arange(shape[-1], dtype=np.float32), shape).copy()
    if kind == "bits":      # any pattern: both signs, infinities, NaN, denormals
        m = rng.integers(0, 1 << 32, shape, dtype=np.uint64).astype(np.uint32).view(np.float32)
        m[rng.random(shape) < 0.1] = np.nan
        m[rng.random(shape) < 0.05] = np.inf
        m[rng.random(shape) < 0.1] = -0.0
        m[rng.random(shape) < 0.1] = 0.0
        m[rng.random(shape) < 0.1] = -np.inf
        return m
    raise ValueError(kind)


CASES = [
    # fmt, H, D, ps, lens, keep, sinks, recent, mass, cells with numbers of their own, more tokens than cells
    ("f16", 2, 256, 4, [1021], 200, 4, 16, "spread", None, 0),
    ("f16", 1, 64, 1, [70, 64, 65, 1, 0, 63], 64, 0, 0, "few", None, 0),
    ("int8", 2, 256, 4, [513, 4, 300], 100, 2, 50, "spread", None, 0),
    ("int8", 4, 64, 16, [2000], 1, 0, 0, "spread", None, 0),
    ("int8", 1, 128, 3, [333, 334], 332, 0, 1, "few", None, 0),
    ("f16", 3, 128, 5, [5000], 4097, 0, 0, "none", None, 0),
    ("f16", 2, 64, 8, [4096, 4095, 8193], 2048, 8, 1024, "late", None, 0),
    ("f16", 1, 256, 4, [900, 901], 64, 0, 64, "spread", None, 0),
    ("f16", 2, 128, 4, [1500, 40], 700, 10, 100, "bits", None, 0),
    ("f16", 2, 64, 4, [264, 264, 260, 250], 256, 4, 32, "spread", [256, 264, 0, 250], 1000),
    ("int8", 1, 256, 7, [1029], 1024, 0, 128, "few", [1024], 31337),
    ("f16", 2, 64, 4, [300, 100], 50, 20, 30, "bits", [100, 100], 7),
    # heads of several workgroups
    ("f16", 1, 64, 16, [40000, 3, 17000, 8192], 8192, 4, 100, "spread", None, 0),
    ("int8", 2, 64, 16, [30001], 29000, 0, 0, "few", [20000], 50000),
    ("f16", 1, 64, 64, [33000, 32999], 100, 50, 50, "bits", None, 9),
    ("f16", 2, 64, 32, [25000], 12500, 0, 0, "late", None, 0),
    ("int8", 1, 64, 8, [16385], 16384, 0, 0, "none", None, 0),
    # more cells than a workgroup holds, too many heads to share them out
    ("f16", 130, 64, 64, [8300], 5000, 3, 10, "few", None, 0),
]


@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in place"])
@pytest.mark.parametrize("case", CASES, ids=[f"{c[0]}-{c[1]}x{c[2]}-p{c[3]}-{max(c[4])}to{c[5]}-{c[8]}" for c in CASES])
def test_against_the_plain_form(sc, ops, plain, cuda, case, in_place):
    fmt, H, D, ps, lens, keep, sinks, recent, kind, known, more = case
    print(f"evict {case}", flush=True)
    rng = np.random.default_rng(sum(lens) + D)
    n, most = len(lens), max(lens)
    cache = Cache(sc, ops, rng, fmt, H, D, ps, n, -(-most // ps) + 1)
    ld = most + 5
    mass = _mass(rng, kind, (n, H, ld))
    total = np.array([t + more for t in lens], np.int64)
    born = np.full((n, H, ld), -77, np.int32)
    for s in range(n):
        for h in range(H):
            if known and known[s]:   # numbers below those of the later cells, in no order
                born[s, h, :known[s]] = rng.permutation(total[s] - (lens[s] - known[s]))[:known[s]]
    dmass, dborn, dlens = upload(sc, mass), upload(sc, born), upload(sc, np.array(lens, np.int64))
    mass_out, born_out = (dmass, dborn) if in_place else (upload(sc, np.full_like(mass, 3.5)), upload(sc, np.full_like(born, -5)))
    dknown = upload(sc, np.array(known or [0] * n, np.int64))
    lens_out = dlens if in_place else upload(sc, np.full(n, -9, np.int64))
    given = known or in_place
    ops.KvEvict(cache.c, dmass, n_seqs=n, lens=dlens, max_len=most, keep=keep, sinks=sinks, recent=recent, mass_out=mass_out,
                born=dborn if given else None, born_out=born_out, ld=ld, known=dknown if given else None,
                total=upload(sc, total) if more else None, lens_out=lens_out).launch()
    sc.device_sync()
    got_mass, got_born, left = mass_out.numpy().reshape(mass.shape), born_out.numpy().reshape(born.shape), lens_out.numpy()
    want = {c: x.copy() for c, x in cache.host.items()}
    want_mass = (mass if in_place else np.full_like(mass, 3.5)).copy()
    want_born = (born if in_place else np.full_like(born, -5)).copy()
    for s, t in enumerate(lens):
        for h in range(H):
            number = np.arange(t) + total[s] - t
            if known:
                number[:known[s]] = born[s, h, :known[s]]
            place = plain.evict(mass[s, h, :t], number, int(total[s]), keep, sinks, recent)
            want_mass[s, h, :t] = 0
            want_mass[s, h, :len(place)], want_born[s, h, :len(place)] = mass[s, h, place], number[place]
            for c, cell in enumerate(place):
                if c != cell:
                    to, of = (plain.pool_row(cache.table, s, int(x), h, H, ps, cache.n_pages, cache.ld) for x in (c, cell))
                    for w in want:
                        want[w][to] = cache.host[w][of]
        assert left[s] == min(t, keep), s
    assert np.array_equal(got_mass.view(np.uint32), want_mass.view(np.uint32))
    assert np.array_equal(got_born, want_born)
    for w, x in want.items():
        assert np.array_equal(cache.dev[w].numpy().reshape(x.shape), x), w


def test_again_and_again(sc, ops, plain, cuda):
    """A cache that grows by some cells and is cut to its size, many times, holds the rows, masses and numbers that the plain
    form keeps; the workspace and the arrays are the same ones all along."""
    H, D, ps, keep, ld = 2, 64, 4, 50, 80
    rng = np.random.default_rng(11)
    cache = Cache(sc, ops, rng, "f16", H, D, ps, 2, ld // ps)
    host = {c: x.copy() for c, x in cache.host.items()}
    mass, born, total, known = np.zeros((2, H, ld), np.float32), np.zeros((2, H, ld), np.int32), np.zeros(2, np.int64), np.zeros(2, np.int64)
    dmass, dborn, dknown = upload(sc, mass), upload(sc, born), upload(sc, known)
    dlens, dtotal = upload(sc, known), upload(sc, total)
    call = ops.KvEvict(cache.c, dmass, n_seqs=2, lens=dlens, max_len=ld, keep=keep, sinks=2, recent=10, born=dborn, known=dknown, total=dtotal,
                       lens_out=dknown)
    for step in range(12):
        lens = known + rng.integers(0, 30, 2)
        total += lens - known
        for s in range(2):
            mass[s, :, :lens[s]] += rng.random((H, lens[s])).astype(np.float32)
        dmass.upload(mass), dlens.upload(lens), dtotal.upload(total)
        call.launch()
        sc.device_sync()
        for s in range(2):
            for h in range(H):
                t = lens[s]
                number = np.arange(t) + total[s] - t
                number[:known[s]] = born[s, h, :known[s]]
                place = plain.evict(mass[s, h, :t], number, int(total[s]), keep, 2, 10)
                rows = [plain.pool_row(cache.table, s, int(c), h, H, ps, cache.n_pages, cache.ld) for c in range(ld)]
                for x in host.values():
                    x[np.array(rows)[:len(place)]] = x[np.array(rows)[place]]
                kept = mass[s, h, place]
                mass[s, h, :t] = 0
                mass[s, h, :len(place)], born[s, h, :len(place)] = kept, number[place]
            known[s] = min(lens[s], keep)
        assert np.array_equal(dknown.numpy(), known) and np.array_equal(dmass.numpy().reshape(mass.shape), mass), step
        for s in range(2):
            assert np.array_equal(dborn.numpy().reshape(born.shape)[s, :, :known[s]], born[s, :, :known[s]]), step
        for w, x in host.items():
            assert np.array_equal(cache.dev[w].numpy().reshape(x.shape), x), (step, w)


def test_lengths_and_numbers_outside_their_bounds(sc, ops, cuda):
    """Negative lengths count as 0, long ones as the bound; numbers and totals that make no sense move rows within their heads."""
    H, D, ps, ld = 1, 64, 4, 40
    rng = np.random.default_rng(1)
    lens = np.array([-5, 1 << 40, 30, 40, 40], np.int64)
    cache = Cache(sc, ops, rng, "f16", H, D, ps, len(lens), ld // ps)
    mass, born = rng.random((len(lens), H, ld)).astype(np.float32), rng.integers(-(1 << 31), 1 << 31, (len(lens), H, ld)).astype(np.int32)
    out, left = upload(sc, np.full_like(mass, 2)), upload(sc, np.zeros(len(lens), np.int64))
    ops.KvEvict(cache.c, upload(sc, mass), n_seqs=len(lens), lens=upload(sc, lens), max_len=ld, keep=10, sinks=3, recent=3, mass_out=out,
                born=upload(sc, born), born_out=upload(sc, born), known=upload(sc, np.array([5, 1 << 50, -3, 40, 12], np.int64)),
                total=upload(sc, np.array([0, -7, 1 << 60, -(1 << 62), 3], np.int64)), lens_out=left).launch()
    sc.device_sync()
    assert np.array_equal(left.numpy(), [0, 10, 10, 10, 10])
    got = out.numpy().reshape(mass.shape)
    assert (got[0] == 2).all() and (got[2, :, 30:] == 2).all()
    for s in range(1, len(lens)):
        t = min(int(lens[s]), ld)
        assert (got[s, 0, 10:t] == 0).all() and set(got[s, 0, :10]) <= set(mass[s, 0, :t]) and len(set(got[s, 0, :10])) == 10


def test_pages_that_are_not_resident(sc, ops, plain, cuda):
    """A row is neither read from nor written to a page outside the pool; the others move as ever."""
    H, D, ps, n_pages, ld = 2, 64, 4, 40, 16
    rng = np.random.default_rng(9)
    table = rng.permutation(n_pages)[:ld].astype(np.int32).reshape(1, ld)
    table[0, 2], table[0, 11], table[0, 13] = -1, n_pages, 1 << 30
    cache = Cache(sc, ops, rng, "f16", H, D, ps, 1, ld, table=table, n_pages=n_pages)
    mass = rng.random((1, H, ld * ps)).astype(np.float32)
    ops.KvEvict(cache.c, upload(sc, mass), n_seqs=1, lens=upload(sc, np.array([ld * ps])), max_len=ld * ps, keep=20,
                lens_out=upload(sc, np.zeros(1, np.int64))).launch()
    sc.device_sync()
    want = {c: x.copy() for c, x in cache.host.items()}
    for h in range(H):
        for c, cell in enumerate(plain.evict(mass[0, h], np.arange(ld * ps), ld * ps, 20, 0, 0)):
            to, of = (plain.pool_row(table, 0, int(x), h, H, ps, n_pages, ld) for x in (c, cell))
            if to >= 0 and of >= 0:
                for w in want:
                    want[w][to] = cache.host[w][of]
    for w, x in want.items():
        assert np.array_equal(cache.dev[w].numpy().reshape(x.shape), x), w


def test_rows_past_4_gib(sc, ops, cuda):
    """Pools of more than 2^32 bytes: rows at both ends of them go where they belong."""
    H, D, ps, ld = 1, 256, 4, 8
    n_pages = (1 << 32) // (H * ps * D * 2) + 64
    rng = np.random.default_rng(4)
    table = np.array([[3, n_pages - 1, 1, n_pages - 9, n_pages - 2, 0, n_pages - 40, 7]], np.int32)
    pools, rows = [sc.DeviceBuffer(n_pages * H * ps * D, "uint16") for _ in range(2)], []
    for pool in pools:
        rows.append(rng.integers(0, 1 << 16, (ld, ps, D)).astype(np.uint16))
        for p, page in enumerate(table[0]):
            one = upload(sc, rows[-1][p])
            sc.check(sc.lib.sc_copy_device_async(pool.ptr + int(page) * one.nbytes, one.ptr, one.nbytes, None), "copy")
            sc.device_sync()
    mass = rng.random((1, 1, ld * ps)).astype(np.float32)
    cache = ops.kv_cache(*pools, n_pages=n_pages, n_head_kv=H, head_dim=D, page_size=ps, table=upload(sc, table), table_ld=ld)
    ops.KvEvict(cache, upload(sc, mass), n_seqs=1, lens=upload(sc, np.array([ld * ps])), max_len=ld * ps, keep=9,
                lens_out=upload(sc, np.zeros(1, np.int64))).launch()
    sc.device_sync()
    from oracle import sc_ops as plain
    place = plain.evict(mass[0, 0], np.arange(ld * ps), ld * ps, 9, 0, 0)
    for pool, x in zip(pools, rows):
        got = sc.DeviceBuffer((ld, ps, D), "uint16")
        for p, page in enumerate(table[0]):
            sc.check(sc.lib.sc_copy_device_async(got.ptr + p * ps * D * 2, pool.ptr + int(page) * ps * D * 2, ps * D * 2, None), "copy")
        sc.device_sync()
        want = x.reshape(-1, D).copy()
        want[:9] = want[place]
        assert np.array_equal(got.numpy().reshape(-1, D), want)
        pool.free()


def test_on_another_stream(sc, ops, cuda):
    """A call waits for the work before it on its own stream."""
    H, D, ps, ld = 2, 128, 4, 64
    rng = np.random.default_rng(8)
    mass, got = rng.random((1, H, ld * ps)).astype(np.float32), []
    for late in (False, True):
        cache = Cache(sc, ops, np.random.default_rng(2), "f16", H, D, ps, 1, ld)
        staged, dmass, left = upload(sc, mass), upload(sc, np.zeros_like(mass) if late else mass), upload(sc, np.zeros(1, np.int64))
        stream = sc.Stream()
        sc.device_sync()
        if late:
            sc.delay_async(2000, stream)
            sc.check(sc.lib.sc_copy_device_async(dmass.ptr, staged.ptr, mass.nbytes, stream.handle), "copy")
        ops.KvEvict(cache.c, dmass, n_seqs=1, lens=upload(sc, np.array([ld * ps])), max_len=ld * ps, keep=77, lens_out=left).launch(stream)
        stream.sync()
        got.append([dmass.numpy(), left.numpy(), *(b.numpy() for b in cache.dev.values())])
    assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(*got))


def test_two_calls_at_once(sc, ops, cuda):
    """Masses and evictions of two caches on two streams at the same time, a workspace each, leave what they leave one by one."""
    H, D, ps, t, heads = 2, 128, 4, 2000, 8
    got = []
    for together in (False, True):
        streams, outs = [sc.Stream(), sc.Stream()], []
        calls = []
        for i in range(2):
            rng = np.random.default_rng(20 + i)
            cache = Cache(sc, ops, rng, "f16", H, D, ps, 1, t // ps)
            mass, lens, left = upload(sc, np.zeros((1, H, t), np.float32)), upload(sc, np.array([t - i])), upload(sc, np.zeros(1, np.int64))
            q = upload(sc, rng.standard_normal((5, heads, D)).astype(np.float32))
            calls.append([ops.AttnMass(cache.c, q, mass, "f32", n_seqs=1, rows=5, n_head=heads, lens=lens, max_len=t, scale=D ** -0.5),
                          ops.KvEvict(cache.c, mass, n_seqs=1, lens=lens, max_len=t, keep=300 + i, lens_out=left)])
            outs.append((cache, mass, left))
        sc.device_sync()
        for a, b in zip(*calls) if together else ():
            a.launch(streams[0])
            b.launch(streams[1])
        for i in range(2) if not together else ():
            for call in calls[i]:
                call.launch(streams[i])
            streams[i].sync()
        sc.device_sync()
        got.append([x.numpy() for cache, mass, left in outs for x in (mass, left, *cache.dev.values())])
    assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(*got))


def test_nothing_to_evict_in_a_long_cache(sc, ops, cuda):
    """A bound that no sequence can pass leaves caches as they are and hands masses and numbers on."""
    H, D, ps, ld = 1, 64, 64, 320
    rng = np.random.default_rng(2)
    cache = Cache(sc, ops, rng, "f16", H, D, ps, 2, ld)
    mass, lens = rng.random((2, H, ld * ps)).astype(np.float32), np.array([ld * ps, 0], np.int64)
    out, born, left = upload(sc, np.full_like(mass, 9)), upload(sc, np.full((2, H, ld * ps), -1, np.int32)), upload(sc, np.full(2, -1, np.int64))
    ops.KvEvict(cache.c, upload(sc, mass), n_seqs=2, lens=upload(sc, lens), max_len=ld * ps, keep=ld * ps, mass_out=out, born_out=born,
                lens_out=left).launch()
    sc.device_sync()
    assert np.array_equal(left.numpy(), lens) and np.array_equal(out.numpy().reshape(mass.shape)[0], mass[0])
    assert (out.numpy().reshape(mass.shape)[1] == 9).all() and np.array_equal(born.numpy().reshape(mass.shape)[0, 0], np.arange(ld * ps))
    for w, x in cache.host.items():
        assert np.array_equal(cache.dev[w].numpy().reshape(x.shape), x)
