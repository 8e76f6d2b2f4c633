"""sc_conv_async against the 64-bit implementation of the same operator.

What may differ is derived.  The sum of W products and a bias in f32 has W + 1 roundings of at most 2^-24 of the sum of the
terms' sizes, M = |bias| + sum |w x|: off by (W + 1) 2^-24 M.  silu's slope is at most 1.1, and of itself it is off by 2^-21.5 of
its value: the exponential's argument v log2(e) by 2^-24 of itself, so e^-v by |v| 2^-24 + 2^-23 of itself and the quotient by
no more than that (a sigmoid moves by at most min(1, e^-v) of that), with |v| e^-v / (1 + e^-v) <= 0.28 where v > 0; where v < 0
by |v| 2^-24 of a value that is |v| e^v at most: |v|^2 e^v <= 0.55, so 2^-23 in absolute terms.  The type adds half a step.  A
history is moved, in f32, without a rounding."""
import numpy as np
import pytest

from ops_cases import SENTINEL, act, between_rows_untouched, strided, upload

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


@pytest.fixture(scope="module")
def plain():
    from oracle import sc_ops
    return sc_ops


def _near(history, x, weight, bias, want, W, silu, dtype):
    rows = np.concatenate([history, x])
    M = sum(np.abs(weight[:, j] * rows[j:j + len(x)]) for j in range(W)) + (0 if bias is None else np.abs(bias))
    e = 1.1 * (W + 1) * 2.0 ** -24 * M + (2.0 ** -21.5 * np.abs(want) + 2.0 ** -23 if silu else 0)
    return e + (2.0 ** -11 * (np.abs(want) + e) + 2.0 ** -25 if dtype == "f16" else 2.0 ** -24 * np.abs(want))


CASES = [
    # act, channels, taps, layout, rows of each sequence, bias, silu, a sequence without a slot
    ("f32", 8192, 4, "slot", [1], True, True, None),
    ("f16", 64, 4, "slot", [1] * 70, True, True, 3),
    ("f32", 8, 2, "rows", [1, 1], False, False, None),
    ("f32", 1032, 5, "slot", [1] * 5, True, True, 4),
    ("f16", 256, 3, "rows", [5, 0, 33, 1, 2, 64, 32], True, True, None),
    ("f32", 264, 4, "slot", [3, 2, 1, 0, 31, 32, 33, 4], True, True, 4),
    ("f16", 8192, 4, "slot", [97], False, True, None),
    ("f32", 2056, 5, "rows", [4, 3, 70], True, False, None),
    ("f16", 1000, 2, "slot", [0, 0, 129, 0], True, True, None),
    ("f32", 16, 4, "rows", [1] * 130 + [40] + [0] * 70 + [2], True, True, 130),
]


@pytest.mark.parametrize("case", CASES, ids=[f"{c[0]}-{c[1]}x{c[2]}-{c[3]}-{len(c[4])}" for c in CASES])
def test_against_64_bits(sc, ops, plain, cuda, case):
    dtype, C_, W, layout, lens, biased, silu, without = case
    print(f"conv {case}", flush=True)
    rng = np.random.default_rng(C_ + W)
    n, N, pad, past = len(lens), sum(lens), 24, 3
    step = lens == [1] * n
    rows = N if step else N + past   # rows past the last sequence
    x, x64 = act(rng.standard_normal((rows, C_)) * 2, dtype)
    weight, bias = (rng.standard_normal((C_, W)) / W ** 0.5).astype(np.float32), rng.standard_normal(C_).astype(np.float32)
    hist = rng.standard_normal((n, W - 1, C_)).astype(np.float32)
    ld = C_ + 4 if layout == "rows" else C_
    each = (W - 1) * ld + 8   # a history and what lies behind it
    state = np.full((n, each), 7.0, np.float32)
    for s in range(n):
        state[s, 4:4 + (W - 1) * ld] = hist[s].T.ravel() if layout == "slot" else np.pad(hist[s], ((0, 0), (0, ld - C_)), constant_values=7.0).ravel()
    dstate = upload(sc, state)
    states = ops.ConvStates([None if s == without else dstate.ptr + s * each * 4 for s in range(n)], C_, W, 4, layout, ld, keep=dstate)
    dx, dout = strided(sc, x, C_ + pad), strided(sc, np.full_like(x, 9.0), C_ + 2 * pad)
    ops.Conv(states, dx, upload(sc, weight), dout, dtype, n_seqs=n, tokens=rows, bias=upload(sc, bias) if biased else None,
             cu=None if step else upload(sc, np.cumsum([0, *lens]).astype(np.int64)), activation="silu" if silu else None,
             x_ld=C_ + pad, out_ld=C_ + 2 * pad).launch()
    sc.device_sync()
    got, after = dout.numpy(), dstate.numpy()
    assert between_rows_untouched(got, C_)
    assert (got[N:rows, :C_] == 9.0).all()
    for s, first, t in plain.rows_of(np.cumsum([0, *lens]), n, N):
        out = got[first:first + t, :C_].astype(np.float64)
        if s == without:
            assert not out.any() and np.array_equal(after[s], state[s])
            continue
        want, new = plain.short_conv(hist[s], x64[first:first + t], weight, bias if biased else None, silu)
        assert (np.abs(out - want) <= _near(hist[s].astype(np.float64), x64[first:first + t], weight.astype(np.float64),
                                            bias if biased else None, want, W, silu, dtype)).all(), s
        expect = state[s].copy()
        expect[4:4 + (W - 1) * ld] = (new.T.ravel() if layout == "slot" else np.pad(new, ((0, 0), (0, ld - C_)), constant_values=7.0).ravel())
        assert np.array_equal(after[s], expect), s


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_a_prompt_in_pieces_is_the_prompt(sc, ops, cuda, dtype):
    """A prompt in one call, in pieces of a few rows, and token by token gives the same bits, the history too."""
    C_, W, T = 264, 4, 75
    rng = np.random.default_rng(6)
    x, _ = act(rng.standard_normal((T, C_)), dtype)
    weight, bias = upload(sc, rng.standard_normal((C_, W)).astype(np.float32)), upload(sc, rng.standard_normal(C_).astype(np.float32))
    got = []
    for cuts in ([0, T], [0, 1, 3, 35, 67, 70, T], list(range(T + 1))):
        state, dx = sc.DeviceBuffer((1, C_, W - 1), "float32"), upload(sc, x)
        state.fill(0)
        out, size = upload(sc, np.zeros_like(x)), x.dtype.itemsize * C_
        states = ops.conv_states(state, n_seqs=1, channels=C_, taps=W)
        for b, e in zip(cuts, cuts[1:]):
            ops.Conv(states, dx.ptr + b * size, weight, out.ptr + b * size, dtype, n_seqs=1, tokens=e - b, bias=bias,
                     cu=None if e - b == 1 else upload(sc, np.array([0, e - b]))).launch()
        sc.device_sync()
        got.append((out.numpy(), state.numpy()))
    for o, s in got[1:]:
        assert np.array_equal(o, got[0][0]) and np.array_equal(s, got[0][1])


def test_in_place_and_on_another_stream(sc, ops, cuda):
    """A step's out may be x; a call waits for the work before it on its own stream."""
    C_, W, n = 512, 4, 9
    rng = np.random.default_rng(8)
    x, hist = rng.standard_normal((n, C_)).astype(np.float32), rng.standard_normal((n, C_, W - 1)).astype(np.float32)
    weight, got = upload(sc, rng.standard_normal((C_, W)).astype(np.float32)), []
    for place in ("apart", "in place"):
        staged, dx, state = upload(sc, x), upload(sc, np.zeros_like(x)), upload(sc, hist)
        out = dx if place == "in place" else upload(sc, np.zeros_like(x))
        stream = sc.Stream()
        sc.device_sync()
        sc.delay_async(2000, stream)
        sc.check(sc.lib.sc_copy_device_async(dx.ptr, staged.ptr, x.nbytes, stream.handle), "copy")
        ops.Conv(ops.conv_states(state, n_seqs=n, channels=C_, taps=W), dx, weight, out, "f32", n_seqs=n, tokens=n).launch(stream)
        stream.sync()
        got.append((out.numpy(), state.numpy()))
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])


def test_values_that_are_no_numbers_and_far_ones(sc, ops, cuda):
    """Infinities and NaN stay in their channel and in the rows that need them; sums far from 0 end in 0 or themselves."""
    C_, W, T = 16, 4, 12
    rng = np.random.default_rng(3)
    x = rng.standard_normal((T, C_)).astype(np.float32)
    clean = x.copy()
    x[4, 2], x[5, 3], x[6, 5] = np.nan, np.inf, -1e30
    x[:, 7], x[:, 8] = 500.0, -500.0
    weight = np.abs(rng.standard_normal((C_, W))).astype(np.float32) + 0.5
    outs = []
    for rows in (x, clean):
        out, state = upload(sc, np.zeros_like(x)), sc.DeviceBuffer((1, C_, W - 1), "float32")
        state.fill(0)
        ops.Conv(ops.conv_states(state, n_seqs=1, channels=C_, taps=W), upload(sc, rows), upload(sc, weight), out, "f32", n_seqs=1, tokens=T,
                 cu=upload(sc, np.array([0, T]))).launch()
        sc.device_sync()
        outs.append(out.numpy())
    got, want = outs
    assert np.isnan(got[4:8, 2]).all() and (got[5:9, 3] == np.inf).all() and (got[6:10, 5] == 0).all()
    assert (got[3:, 7] > 500).all() and (got[:, 8] == 0).all()
    same = np.ones((T, C_), bool)
    same[4:8, 2] = same[5:9, 3] = same[6:10, 5] = same[:, 7] = same[:, 8] = False
    assert np.array_equal(got[same], want[same])


def test_a_slots_history(sc, ops, plain, cuda):
    """The histories of two layers in decode slots advance in place, behind their states, and nothing else of the slot does."""
    geo = sc.geometry(n_layers=8, qsa_interval=4, n_head_kv=2, head_dim=128, page_size=4, ssm_state_size=64, ssm_k_heads=2, ssm_v_heads=4,
                      ssm_conv_channels=256)
    slots = [sc.new_slot(geo, geo.cells(8)) for _ in range(3)]
    rng = np.random.default_rng(5)
    C_, W, at = geo.ssm_conv_channels, geo.ssm_d_conv, geo.ssm_state_size ** 2 * geo.ssm_v_heads
    rows = [rng.standard_normal((geo.n_gdn, geo.gdn_row_floats)).astype(np.float32) for _ in slots]
    for slot, r in zip(slots, rows):
        slot.gdn.upload(r)
    weight, x = rng.standard_normal((C_, W)).astype(np.float32), rng.standard_normal((3, C_)).astype(np.float32)
    for layer in (0, geo.n_gdn - 1):
        out = upload(sc, np.zeros_like(x))
        ops.Conv(ops.slot_conv(geo, slots, layer), upload(sc, x), upload(sc, weight), out, "f32", n_seqs=3, tokens=3).launch()
        sc.device_sync()
        for s in range(3):
            hist = rows[s][layer, at:].reshape(C_, W - 1)
            want, new = plain.short_conv(hist.T, x[s:s + 1], weight, None, True)
            assert (np.abs(out.numpy()[s] - want[0]) <= _near(hist.T.astype(np.float64), x[s:s + 1].astype(np.float64), weight.astype(np.float64), None, want, W, True, "f32")[0]).all()
            rows[s][layer, at:] = new.T.ravel()
    for slot, r in zip(slots, rows):
        assert np.array_equal(slot.gdn.numpy().reshape(r.shape), r)
