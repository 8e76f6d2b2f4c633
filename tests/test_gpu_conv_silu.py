"""The silu of sc_conv_async over its whole range.  With one tap of 1 the sum is the row itself, so that only the silu is off: the
exponential and the reciprocal by 2^-23 each, what is left of the exponent, 1 + e, the two products by 2^-24 each, 2^-21 together, and
an f16 result by its rounding and the exponent's own, 2^-24 |v| of e^-v, beside these.  A result whose e^-v is beyond 2^126 is 0, which
is off by 88 2^-126 at most."""
import numpy as np
import pytest

from ops_cases import act, upload

pytestmark = pytest.mark.gpu

C = 8192


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


@pytest.mark.parametrize("tokens", [1, 3], ids=["step", "prompt"])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_silu(sc, ops, cuda, dtype, tokens):
    rng = np.random.default_rng(4)
    far = -(10.0 ** rng.uniform(-3, 2.3, C // 2))
    x, x64 = act(np.tile(np.concatenate([far, rng.uniform(-104, 104, C // 2)]), (tokens, 1)), dtype)
    x[:, :5] = x64[:, :5] = np.array([0.0, -0.0, 60.0, -90.0, 104.0])
    weight = np.zeros((C, 2), np.float32)
    weight[:, 1] = 1
    state, out = upload(sc, np.zeros((C, 1), np.float32)), sc.DeviceBuffer((tokens, C), x.dtype)
    ops.Conv(ops.conv_states(state, n_seqs=1, channels=C, taps=2), upload(sc, x), upload(sc, weight), out, dtype, n_seqs=1, tokens=tokens,
             cu=None if tokens == 1 else upload(sc, np.array([0, tokens]))).launch()
    sc.device_sync()
    want = x64 / (1 + np.exp(-x64))
    near = np.abs(want) * (2.0 ** -21 if dtype == "f32" else 2.0 ** -11 + 2.0 ** -24 * np.abs(x64) + 2.0 ** -21) + 88 * 2.0 ** -126
    if dtype == "f16":
        near += 2.0 ** -25   # half a step of the smallest f16 values
    assert (np.abs(out.numpy().astype(np.float64) - want) <= near).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_silu_of_no_numbers(sc, ops, cuda, dtype):
    """inf / (1 + 0) is inf, -inf / inf and what is NaN is NaN."""
    x = np.zeros((1, 8), np.float16 if dtype == "f16" else np.float32)
    x[0, :3] = np.inf, -np.inf, np.nan
    weight = np.zeros((8, 2), np.float32)
    weight[:, 1] = 1
    state, out = upload(sc, np.zeros((8, 1), np.float32)), sc.DeviceBuffer((1, 8), x.dtype)
    ops.Conv(ops.conv_states(state, n_seqs=1, channels=8, taps=2), upload(sc, x), upload(sc, weight), out, dtype, n_seqs=1, tokens=1).launch()
    sc.device_sync()
    got = out.numpy()[0]
    assert got[0] == np.inf and np.isnan(got[1:3]).all() and not got[3:].any()


@pytest.mark.parametrize("tokens", [1, 9], ids=["step", "prompt"])
def test_silu_where_no_sum_is_far(sc, ops, cuda, tokens):
    """Sums above -5.5 alone: the exponent, 8 at most, is rounded to 2^-22 and its factor to 2^-26 of it, which is 2^-22 of e^-v beside
    what the exponential, 1 + e, the reciprocal and the product leave, 2^-21.5."""
    rng = np.random.default_rng(6)
    x = rng.uniform(-5.499, 30, (tokens, C)).astype(np.float32)
    x[:, ::3] = -x[:, ::3].clip(0, 5.499)
    weight = np.zeros((C, 2), np.float32)
    weight[:, 1] = 1
    state, out = upload(sc, np.zeros((C, 1), np.float32)), sc.DeviceBuffer((tokens, C), "float32")
    ops.Conv(ops.conv_states(state, n_seqs=1, channels=C, taps=2), upload(sc, x), upload(sc, weight), out, "f32", n_seqs=1, tokens=tokens,
             cu=None if tokens == 1 else upload(sc, np.array([0, tokens]))).launch()
    sc.device_sync()
    want = x.astype(np.float64) / (1 + np.exp(-x.astype(np.float64)))
    assert (np.abs(out.numpy().astype(np.float64) - want) <= np.abs(want) * (2.0 ** -22 + 2.0 ** -21.5)).all()
