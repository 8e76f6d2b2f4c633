"""sc_gdn_chunk_async where a chunk's keys differ in length: padding rows of zeros, short and long ones side by side.  What a row
writes to the state is known to 2^-22 of itself, whatever the other rows' keys are: the bounds of test_gpu_gdn_scales."""
import numpy as np
import pytest

from test_gpu_gdn import Layer
from test_gpu_gdn_scales import WIDTHS, _check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


@pytest.fixture(scope="module")
def plain():
    from oracle import sc_ops
    return sc_ops


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("eps", [1e-6, 1e-12])
@pytest.mark.parametrize("lengths", ["zeros", "long and zeros", "spread", "long", "one short", "least"])
def test_keys_of_many_lengths(sc, ops, plain, cuda, lengths, eps, width, dtype):
    S, kh, vh, n = WIDTHS[width]
    x = Layer(sc, ops, 31, S, kh, vh, [150] + [70] * (n - 1), dtype)
    x.eps = eps
    rng = np.random.default_rng(32)
    by = np.ones(x.N)
    if lengths == "spread":
        by = np.exp2(rng.uniform(-8, 8, x.N))
    if "long" in lengths:
        by[:] = 1000 / S ** 0.5
    if "zeros" in lengths:
        by[rng.random(x.N) < 0.1] = 0
        by[::64] = 0
    if lengths == "one short":
        by[7::20] = 2.0 ** -16
    if lengths == "least":
        by[:] = 2.0 ** -20 if dtype == "f16" else 2.0 ** -40
    x.k = (x.k64 * by[:, None, None]).astype(x.k.dtype)
    x.k64 = x.k.astype(np.float64)
    x.build().launch()
    sc.device_sync()
    _check(x, plain, [0, vh - 1], [0, n - 1])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_keys_as_they_are(sc, ops, plain, cuda, dtype):
    """Without the norm: keys up to a length of one, some of them a thousandth of that, some zeros."""
    x = Layer(sc, ops, 33, 128, 2, 4, [200, 64], dtype, l2norm=False)
    by = np.where(np.arange(x.N) % 3 == 1, 2.0 ** -10, 1.0) * (np.arange(x.N) % 7 != 4)
    x.k = (x.k64 * by[:, None, None]).astype(x.k.dtype)
    x.k64 = x.k.astype(np.float64)
    x.build().launch()
    sc.device_sync()
    _check(x, plain, [0, 3])
