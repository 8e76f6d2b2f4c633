"""What the tests of the operators share: activations in their types, paged caches with their host copies."""
import numpy as np

SENTINEL = 0x5A   # bytes that no call may touch


def act(x, dtype):
    """Values as the device holds them: (what is uploaded, the same in 64 bits)."""
    y = np.asarray(x, np.float32).astype(np.float16 if dtype == "f16" else np.float32)
    return y, y.astype(np.float64)


def upload(sc, x):
    b = sc.DeviceBuffer(x.shape, x.dtype)
    b.upload(x)
    return b


def strided(sc, x, ld):
    """Rows [n][...] uploaded `ld` values apart, a sentinel between them; the buffer."""
    n = x.shape[0]
    flat = np.full((max(n, 1), ld), np.frombuffer(bytes([SENTINEL] * x.dtype.itemsize), x.dtype)[0], x.dtype)
    flat[:n, :x[0].size if n else 0] = x.reshape(n, -1)
    return upload(sc, flat)


def between_rows_untouched(got, row):
    """The values past `row` of each row still hold the sentinel."""
    return bool((got[:, row:].copy().view(np.uint8) == SENTINEL).all())


def random_tables(rng, n_seqs, table_ld, n_pages, missing=0.0):
    """Distinct physical pages for every logical page, some of them not resident (-1, or past the pool)."""
    t = rng.permutation(n_pages)[:n_seqs * table_ld].astype(np.int32).reshape(n_seqs, table_ld)
    gone = rng.random(t.shape) < missing
    return np.where(gone, np.where(rng.random(t.shape) < 0.5, -1, n_pages + 7), t).astype(np.int32)


class Cache:
    """A paged cache on the device and on the host: random rows, or sentinels."""

    def __init__(self, sc, ops, rng, fmt, H, D, ps, n_seqs, table_ld, *, table="random", n_pages=None, missing=0.0, fill="random"):
        self.fmt, self.H, self.D, self.ps, self.ld = fmt, H, D, ps, table_ld
        self.n_pages = n_pages if n_pages is not None else n_seqs * table_ld + 3
        rows = self.n_pages * H * ps
        if fmt == "f16":
            make = lambda: rng.standard_normal((rows, D)).astype(np.float16)  # noqa: E731
        else:
            make = lambda: rng.integers(-127, 128, (rows, D)).astype(np.int8)  # noqa: E731
        self.host = {"k": make(), "v": make()}
        if fmt == "int8":
            for c in ("ks", "vs"):
                self.host[c] = (0.01 + 0.02 * rng.random((rows, D // 64))).astype(np.float16).view(np.uint16)
        if fill == "sentinel":
            for x in self.host.values():
                x.view(np.uint8)[:] = SENTINEL
        self.table = random_tables(rng, n_seqs, table_ld, self.n_pages, missing) if isinstance(table, str) else table
        self.upload(sc)
        self.t_dev = None if self.table is None else upload(sc, self.table)
        self.c = ops.kv_cache(self.dev["k"], self.dev["v"], self.dev.get("ks"), self.dev.get("vs"), n_pages=self.n_pages,
                              n_head_kv=H, head_dim=D, page_size=ps, table=self.t_dev, table_ld=table_ld)

    def upload(self, sc):
        self.dev = {n: upload(sc, x) for n, x in self.host.items()}

    def values(self, which):
        """Every row in 64 bits."""
        from oracle import sc_ops as oracle
        x = self.host[which]
        return x.astype(np.float64) if self.fmt == "f16" else oracle.dequant(x, self.host[which + "s"])
