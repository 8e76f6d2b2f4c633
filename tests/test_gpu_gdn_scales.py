"""sc_gdn_chunk_async where what a chunk begins with and what it leaves differ by orders of magnitude.

What may differ is derived in the results' own size.  A column of a state is known to 2^-20 of its norm: every write to 2^-22 of
itself and sums in 32 bits of either sign over 128 keys, as for states as a whole.  An output is the product of a column of the
state at that token with the query, so it is known to 2^-19 of scale |q| times that column's norm (twice, for the product's own
sum), and an f16 value to half a unit of its 11 bits besides; products below f32's normal range may be lost, 2^-126.  A bound of the output's own size there is none: right after a token that
forgets all, the state is k u^T, and the output scale (k . q) u, whose k . q may be anything down to 0."""
import numpy as np
import pytest

from ops_cases import upload
from test_gpu_gdn import Layer

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


@pytest.fixture(scope="module")
def plain():
    from oracle import sc_ops
    return sc_ops


def _check(x, plain, heads, seqs=None):
    out, M = x.read()
    share = x.vh // x.kh
    for s in range(x.n) if seqs is None else seqs:
        lo, hi = int(x.cu[s]), int(x.cu[s + 1])
        for h in heads:
            state = x.M[s, h].astype(np.float64)
            for t in range(lo, hi):
                row = np.s_[t:t + 1]
                q = x.q64[row, h // share]
                want, state = plain.delta_rule(state, q, x.k64[row, h // share], x.v64[row, h], x.g[row, h], x.beta[row, h], x.scale,
                                               x.l2norm, x.eps)
                length = np.linalg.norm(q) / np.sqrt((q * q).sum() + x.eps) if x.l2norm else np.linalg.norm(q)
                tol = 2.0 ** -19 * x.scale * length * np.linalg.norm(state, axis=0) + 2.0 ** -126
                seen = np.ones(x.S, bool)
                if x.dtype == "f16":
                    tol = tol + 2.0 ** -11 * np.abs(want[0]) + 2.0 ** -25
                    seen = np.abs(want[0]) < 60000   # in range
                off = np.abs(out[t, h].astype(np.float64) - want[0])[seen] / tol[seen]
                assert not len(off) or off.max() <= 1, ("row", s, h, t - lo, off.max())
            err = np.linalg.norm(M[s, h] - state, axis=0) / np.linalg.norm(state, axis=0)
            assert err.max() <= 2.0 ** -20, ("state", s, h, err.max())


# one column tile a workgroup and two
WIDTHS = {"narrow": (128, 2, 4, 1), "wide": (128, 8, 16, 8), "small": (32, 2, 2, 1)}


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("by", [1e3, 1e5, 1e8])
@pytest.mark.parametrize("gate", ["first", "mid", "second", "slow", "200"])
def test_a_large_old_state(sc, ops, plain, cuda, gate, by, width, dtype):
    """A state far larger than the values, forgotten at one token, by one of -200, or at e^-0.5 a token."""
    S, kh, vh, n = WIDTHS[width]
    x = Layer(sc, ops, 21, S, kh, vh, [150] + [130] * (n - 1), dtype)
    x.M *= np.float32(by)
    at = {"first": 0, "mid": 40, "second": 100, "slow": 0, "200": 70}[gate]
    for s in range(n):
        x.g[x.cu[s] + at] = -200 if gate == "200" else -np.inf
        if gate == "slow":
            x.g[x.cu[s]:x.cu[s + 1]] = -0.5
    x.build().launch()
    sc.device_sync()
    _check(x, plain, [0, vh - 1], [0, n - 1])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("at", [17, 33, 64, 90])
def test_large_values_that_are_forgotten(sc, ops, plain, cuda, at, width, dtype):
    """Values of thousands, then a token that forgets them, then values of thousandths, in one chunk and over two."""
    S, kh, vh, n = WIDTHS[width]
    x = Layer(sc, ops, 22, S, kh, vh, [140] * n, dtype)
    for s in range(n):
        rows = slice(int(x.cu[s]), int(x.cu[s + 1]))
        size = np.where(np.arange(140) < at, 2.0 ** 11, 2.0 ** -9)[:, None, None]
        x.v[rows] = (x.v64[rows] * size).astype(x.v.dtype)
        x.v64[rows] = x.v[rows]
        x.g[int(x.cu[s]) + at] = -np.inf
    x.build().launch()
    sc.device_sync()
    _check(x, plain, [0, vh - 1], [0, n - 1])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_a_token_much_larger_than_the_state(sc, ops, plain, cuda, dtype):
    """The outputs before a token whose values are ten thousand times the rest's."""
    x = Layer(sc, ops, 23, 128, 2, 4, [200], dtype)
    x.v[50], x.v[140] = x.v[50] * 2 ** 12, x.v[140] * 2 ** 12
    x.v64[:] = x.v
    x.build().launch()
    sc.device_sync()
    _check(x, plain, [0, 3])


def test_values_over_the_whole_range(sc, ops, plain, cuda):
    """States and values from 10^-30 to 10^30, a column each, and states that fade for thousands of tokens."""
    x = Layer(sc, ops, 24, 64, 1, 2, [90, 400], "f32")
    size = np.exp2(np.linspace(-100, 100, 64))
    x.M, x.v = (x.M * size).astype(np.float32), (x.v * size).astype(np.float32)
    x.v64 = x.v.astype(np.float64)
    x.v[150:400], x.v64[150:400] = 0, 0
    x.build().launch()
    sc.device_sync()
    _check(x, plain, [0, 1])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("what", ["k", "v", "q", "beta", "g"])
def test_no_number_reaches_tokens_before_its_own(sc, ops, cuda, what, dtype):
    """What is no number, or infinite, at a token changes no bit of the tokens before the 16 that it is among."""
    def run(spoil):
        x = Layer(sc, ops, 25, 64, 1, 2, [150], dtype)
        if spoil is not None:
            getattr(x, what)[125] = spoil   # row 61 of the second chunk, in its last 16
        x.build().launch()
        sc.device_sync()
        return x.read()[0]

    clean = run(None)
    for spoil in (np.nan, np.inf) if what != "g" else (np.nan,):
        got = run(spoil)
        assert got[:112].tobytes() == clean[:112].tobytes()
        assert not np.isfinite(got[125:]).all()
