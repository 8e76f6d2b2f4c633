"""A token's row does not depend on how many others are appended with it: calls of one token, of some and of many share their
rows out differently, and leave the same bits."""
import numpy as np
import pytest

from ops_cases import Cache, act, upload

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


def _append(sc, ops, fmt, dtype, H, heads, D, rot, pairs, axes, x, cells, pos, inv_freq):
    """Appends the rows x = (q, k, v) of len(cells) sequences; queries and the caches' rows of their cells."""
    n, ps = len(cells), 4
    cache = Cache(sc, ops, np.random.default_rng(0), fmt, H, D, ps, n, 2, fill="sentinel", table=None, n_pages=2 * n)
    q, k, v = (upload(sc, a) for a in x)
    out = sc.DeviceBuffer((n, heads, D), x[0].dtype)
    kw = dict(n_seqs=n, tokens=n, pos0=upload(sc, np.asarray(cells, np.int64)), inv_freq=inv_freq, rot_dim=rot, pairs=pairs, q=q, q_out=out, n_head=heads)
    if axes:
        call = ops.RopeAxesAppend(cache.c, k, v, dtype, axis=[i % 3 for i in range(rot // 2)], n_axes=3, pos=upload(sc, np.ascontiguousarray(pos)), **kw)
    else:
        call = ops.RopeAppend(cache.c, k, v, dtype, **kw)
    call.launch()
    sc.device_sync()
    at = np.array([((2 * s + c // ps) * H + h) * ps + c % ps for s, c in enumerate(cells) for h in range(H)])
    return [out.numpy(), *(b.numpy().reshape(2 * n * H * ps, -1)[at].reshape(n, H, -1) for b in cache.dev.values())]


@pytest.mark.parametrize("axes", [False, True], ids=["one", "axes"])
@pytest.mark.parametrize("fmt,dtype,H,heads,D,rot,pairs", [
    ("f16", "f32", 2, 24, 256, 64, "halves"), ("int8", "f16", 2, 24, 256, 256, "neighbours"), ("f16", "f16", 8, 64, 128, 128, "halves"),
    ("int8", "f32", 1, 3, 64, 32, "halves"), ("f16", "f16", 3, 9, 64, 64, "neighbours")])
def test_a_row_does_not_depend_on_the_others(sc, ops, cuda, fmt, dtype, H, heads, D, rot, pairs, axes):
    rng, most = np.random.default_rng(H + D), 600
    x = [act(rng.standard_normal((most, h, D)), dtype)[0] for h in (heads, H, H)]
    cells, pos = rng.integers(0, 8, most), rng.integers(-5, 100000, (3, most))
    inv_freq = upload(sc, (1e6 ** (-np.arange(0, rot, 2) / rot)).astype(np.float32))
    few = [0, 1, 57, 149, 299, 519, 599]
    alone = {i: _append(sc, ops, fmt, dtype, H, heads, D, rot, pairs, axes, [a[i:i + 1] for a in x], cells[i:i + 1], pos[:, i:i + 1], inv_freq) for i in few}
    for n in (2, 60, 150, 300, 520, most):
        print(fmt, D, axes, n, flush=True)
        got = _append(sc, ops, fmt, dtype, H, heads, D, rot, pairs, axes, [a[:n] for a in x], cells[:n], pos[:, :n], inv_freq)
        for i in few:
            if i < n:
                for a, b in zip(got, alone[i]):
                    assert np.array_equal(a[i].view(np.uint8), b[0].view(np.uint8)), (n, i)
