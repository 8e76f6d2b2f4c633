"""sc_gdn_step_async and sc_gdn_chunk_async against the 64-bit recurrence, token by token.

What may differ is derived: a token's products with the state are sums of S terms in 32 bits, so it moves the state by about
2^-24 sqrt(S) of the state's largest value, and what earlier tokens moved only shrinks (a decay of at most one, a projection
of at most one).  Errors of T tokens add like steps of either sign, and eight times that is allowed: 2^-21 sqrt(S T) of the
largest value.  An f16 output adds half a unit of its 11 bits."""
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


class Layer:
    """The inputs of one layer's call, on the host in 64 bits and on the device, and its states."""

    def __init__(self, sc, ops, seed, S, kh, vh, lens, dtype, *, layout="slot", l2norm=True, step=False, pad=0, by=1.0, key_by=1.0,
                 gates=(-8, 0.5), state=True, extra=0):
        rng = np.random.default_rng(seed)
        self.S, self.kh, self.vh, self.lens, self.dtype, self.l2norm, self.layout = S, kh, vh, lens, dtype, l2norm, layout
        self.n, self.N = len(lens), sum(lens) + extra
        N = self.N
        self.q, self.q64 = act(rng.standard_normal((N, kh, S)) * by, dtype)
        # without the norm a key longer than one makes the state grow
        self.k, self.k64 = act(rng.standard_normal((N, kh, S)) * (key_by if l2norm else S ** -0.5), dtype)
        self.v, self.v64 = act(rng.standard_normal((N, vh, S)) * by, dtype)
        self.g = -np.exp(rng.uniform(*gates, (N, vh))).astype(np.float32)
        self.beta = (1 / (1 + np.exp(-rng.standard_normal((N, vh))))).astype(np.float32)
        M = rng.standard_normal((self.n, vh, S, S)) * 0.3 * by if state else np.zeros((self.n, vh, S, S))
        self.M = M.astype(np.float32)                     # [n][head][key][value]
        self.cu = np.cumsum([0, *lens]).astype(np.int64)
        self.sc, self.ops, self.step, self.pad = sc, ops, step, pad
        self.scale, self.eps = S ** -0.5, 1e-6

    def place(self, M):
        return np.ascontiguousarray(M.transpose(0, 2, 1, 3) if self.layout == "slot" else M)

    def build(self):
        sc, p, row, vrow = self.sc, self.pad, self.kh * self.S, self.vh * self.S
        self.d_state = upload(sc, self.place(self.M))
        self.out = strided(sc, np.full_like(self.v, 7), vrow + 3 * p)
        self.in_bufs = [strided(sc, self.q, row + p), strided(sc, self.k, row + 2 * p), strided(sc, self.v, vrow + p),
                        strided(sc, self.g, self.vh + p), strided(sc, self.beta, self.vh + p)]
        states = self.ops.gdn_states(self.d_state, n_seqs=self.n, v_heads=self.vh, state_size=self.S, layout=self.layout)
        make = self.ops.GdnStep if self.step else self.ops.GdnChunk
        return make(states, *self.in_bufs, self.out, self.dtype, k_heads=self.kh, n_seqs=self.n, tokens=self.N,
                    cu=None if self.step else upload(sc, self.cu), scale=self.scale, l2norm=self.l2norm, eps=self.eps, q_ld=row + p,
                    k_ld=row + 2 * p, v_ld=vrow + p, out_ld=vrow + 3 * p, gate_ld=self.vh + p)

    def read(self):
        """(out [tokens][heads][S], states [n][head][key][value]) as the device has them."""
        out = self.out.numpy()
        assert not self.pad or between_rows_untouched(out, self.vh * self.S)
        M = self.d_state.numpy()
        return out[:self.N, :self.vh * self.S].reshape(self.N, self.vh, self.S), M.transpose(0, 2, 1, 3) if self.layout == "slot" else M

    def check(self, plain, heads=None, seqs=None):
        out, M = self.read()
        share = self.vh // self.kh
        for s in range(self.n) if seqs is None else seqs:
            rows = slice(int(self.cu[s]), int(self.cu[s + 1]))
            for h in range(self.vh) if heads is None else heads:
                w, wM = plain.delta_rule(self.M[s, h], self.q64[rows, h // share], self.k64[rows, h // share], self.v64[rows, h],
                                         self.g[rows, h], self.beta[rows, h], self.scale, self.l2norm, self.eps)
                T = max(self.lens[s], 1)
                e = 2.0 ** -21 * np.sqrt(self.S * T)
                assert (np.abs(M[s, h] - wM) <= e * max(np.abs(wM).max(), np.abs(self.M[s, h]).max() if T == 1 else 0)).all(), \
                    (s, h, np.abs(M[s, h] - wM).max() / np.abs(wM).max(), e)
                if len(w):
                    tol = e * np.abs(w).max() + (2.0 ** -11 * np.abs(w) + 2.0 ** -25 if self.dtype == "f16" else 0)
                    assert (np.abs(out[rows, h] - w) <= tol).all(), (s, h, np.abs(out[rows, h] - w).max() / np.abs(w).max(), e)


STEPS = [(128, 16, 32, 1, "f32", "slot"), (128, 16, 32, 5, "f16", "prefill"), (128, 16, 48, 2, "f32", "slot"),
         (64, 4, 8, 3, "f16", "slot"), (32, 4, 8, 7, "f32", "prefill"), (64, 1, 1, 1, "f32", "slot"), (128, 8, 8, 70, "f32", "slot"),
         (64, 8, 16, 40, "f16", "prefill"), (128, 2, 4, 66, "f16", "slot")]   # the last three by 64 columns


@pytest.mark.parametrize("l2norm", [True, False], ids=["unit", "as-is"])
@pytest.mark.parametrize("case", STEPS, ids=[f"S{c[0]}-{c[1]}-{c[2]}-n{c[3]}-{c[4]}-{c[5]}" for c in STEPS])
def test_step_against_64_bits(sc, ops, plain, cuda, case, l2norm):
    S, kh, vh, n, dtype, layout = case
    print(f"step {case}", flush=True)
    x = Layer(sc, ops, n * S + vh, S, kh, vh, [1] * n, dtype, layout=layout, l2norm=l2norm, step=True, pad=0 if l2norm else 8)
    x.build().launch()
    sc.device_sync()
    x.check(plain)


CHUNKS = [
    # S, key heads, value heads, lengths, type, layout
    (128, 16, 32, [61], "f32", "slot"), (128, 2, 4, [1, 0, 64, 65, 127, 128, 129], "f32", "prefill"),
    (128, 2, 4, [300, 1, 15, 16, 17], "f16", "slot"), (64, 4, 8, [33, 200, 2], "f32", "slot"), (64, 2, 2, [130], "f16", "prefill"),
    (32, 4, 8, [77, 64, 3], "f32", "slot"), (32, 1, 2, [200], "f16", "prefill"), (128, 1, 3, [500, 63], "f16", "slot"),
    # enough heads for workgroups of 32 columns, and more sequences than a wave sorts
    (128, 2, 4, [1, 0, 64, 65, 127, 128, 129, 33, 3, 200, 63, 66], "f16", "slot"),
    (128, 4, 8, [1, 0, 64, 65, 127, 128, 129, 33, 3, 200, 63, 66, 2, 5, 70, 9], "f32", "prefill"),
    (64, 8, 16, [70, 64, 1, 130, 0, 17], "f16", "prefill"), (64, 8, 16, [70, 64, 1, 130, 0, 17, 65, 2, 3, 4, 5, 6, 7, 8, 9, 60], "f32", "slot"),
    (64, 1, 2, [5, 0, 66, 1, 64] * 14, "f32", "slot"), (64, 1, 4, [5, 0, 66, 1, 64] * 14, "f16", "slot"),
]


@pytest.mark.parametrize("l2norm", [True, False], ids=["unit", "as-is"])
@pytest.mark.parametrize("case", CHUNKS, ids=[f"S{c[0]}-{c[1]}-{c[2]}-n{len(c[3])}-{max(c[3])}-{c[4]}-{c[5]}" for c in CHUNKS])
def test_chunk_against_64_bits(sc, ops, plain, cuda, case, l2norm):
    S, kh, vh, lens, dtype, layout = case
    print(f"chunk {case}", flush=True)
    x = Layer(sc, ops, sum(lens) * S + vh, S, kh, vh, lens, dtype, layout=layout, l2norm=l2norm, pad=0 if l2norm else 8)
    x.build().launch()
    sc.device_sync()
    x.check(plain)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_a_long_prompt(sc, ops, plain, cuda, dtype):
    """Thousands of tokens, slow and fast decays, from an empty state: sampled heads."""
    x = Layer(sc, ops, 5, 128, 2, 4, [4099], dtype, state=False)
    x.build().launch()
    sc.device_sync()
    x.check(plain, heads=[0, 3])


@pytest.mark.parametrize("dtype,lens", [("f16", [8300]), ("f32", [9000, 3000, 1000]), ("f16", [100, 13000, 70, 4000])])
def test_prompts_of_several_pieces(sc, ops, plain, cuda, dtype, lens):
    """Prompts that go through the workspace in pieces, a piece's end inside a sequence or between two."""
    x = Layer(sc, ops, 16, 64, 1, 2, lens, dtype)
    x.build().launch()
    sc.device_sync()
    x.check(plain, heads=[1])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_a_state_as_a_whole(sc, ops, plain, cuda, dtype):
    """The error of a state in its norm: every token's write is known to 2^-22 of itself and 2^-27 of the column's largest
    value, errors of either sign in 128 keys and of some tens of tokens that the state still holds: below 2^-20."""
    x = Layer(sc, ops, 14, 128, 2, 4, [2050], dtype)
    x.v, x.v64 = act(x.v64 * np.exp2(-np.arange(128) / 16), dtype)   # columns of other sizes
    x.build().launch()
    sc.device_sync()
    _, M = x.read()
    for h in range(x.vh):
        _, want = plain.delta_rule(x.M[0, h], x.q64[:, h // 2], x.k64[:, h // 2], x.v64[:, h], x.g[:, h], x.beta[:, h], x.scale, True, x.eps)
        err = np.linalg.norm(M[0, h] - want, axis=0) / np.linalg.norm(want, axis=0)
        assert err.max() <= 2.0 ** -20, (h, err.max())


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("by", [2.0 ** -9, 2.0 ** 9])
def test_small_and_large_values(sc, ops, plain, cuda, by, dtype):
    """The rule is linear in its values and its state: results keep their accuracy whatever their size."""
    x = Layer(sc, ops, 6, 64, 2, 2, [150, 31], dtype, by=by)
    x.build().launch()
    sc.device_sync()
    x.check(plain)


def test_values_far_outside_f16(sc, ops, plain, cuda):
    """f32 values and states of 10^8 and of 10^-8, and keys whose length the norm takes out."""
    for by, key_by in ((1e8, 1e4), (1e-8, 1e-2)):
        x = Layer(sc, ops, 7, 128, 1, 2, [100, 64], "f32", by=by, key_by=key_by)
        x.q, x.q64 = act(np.asarray(x.q) / by, "f32")
        x.build().launch()
        sc.device_sync()
        x.check(plain)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_equal_keys(sc, ops, plain, cuda, dtype):
    """Every token writes to the same key: the products inside a chunk are as large as they can be."""
    x = Layer(sc, ops, 8, 64, 1, 2, [200], dtype, gates=(-12, -10))
    x.k[:], x.k64[:] = x.k[0], x.k64[0]
    x.beta[:] = 1.0
    x.build().launch()
    sc.device_sync()
    x.check(plain)


@pytest.mark.parametrize("step", [True, False], ids=["step", "chunk"])
def test_gates_at_their_ends(sc, ops, plain, cuda, step):
    """A decay of nothing and of everything, a write of nothing: the state is kept, replaced or left."""
    x = Layer(sc, ops, 9, 64, 2, 4, [1] * 5 if step else [70, 64, 5], "f32", step=step)
    x.g[:, 0], x.g[::3, 1], x.beta[:, 2] = 0.0, -np.inf, 0.0
    x.g[1::2, 3], x.beta[::2, 3] = -500.0, 1.0
    x.build().launch()
    sc.device_sync()
    x.check(plain)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("step", [True, False], ids=["step", "chunk"])
def test_values_that_are_no_numbers(sc, ops, cuda, step, dtype):
    """Infinities and NaN in a sequence's values, keys, gates or state change no bit of other heads and sequences."""
    def run(spoil):
        x = Layer(sc, ops, 15, 64, 2, 4, [1] * 5 if step else [70, 130, 64, 65, 3], dtype, step=step)
        if spoil:
            x.v[x.cu[0], 1, 3], x.k[x.cu[1] + 0, 1, 5], x.M[2, 0, 7, 9] = np.nan, np.inf, -np.inf
            x.beta[x.cu[3], 2], x.q[x.cu[4], 0, 1] = np.nan, np.inf
        x.build().launch()
        sc.device_sync()
        return x, *x.read()

    (x, a, m), (_, b, n) = run(False), run(True)
    spoiled = {(0, 1), (1, 2), (1, 3), (2, 0), (3, 2), (4, 0), (4, 1)}
    for s in range(5):
        for h in range(4):
            same = (a[x.cu[s]:x.cu[s + 1], h].tobytes() == b[x.cu[s]:x.cu[s + 1], h].tobytes(), m[s, h].tobytes() == n[s, h].tobytes())
            if (s, h) not in spoiled:
                assert same == (True, True), (s, h)
            else:
                assert not same[0] and not np.isfinite(b[x.cu[s]:x.cu[s + 1], h]).all(), (s, h)


def test_pieces_of_a_prompt(sc, ops, plain, cuda):
    """A prompt in three calls, the last tokens one by one, goes on from the state that each leaves."""
    S, kh, vh, T = 64, 2, 4, 200
    x = Layer(sc, ops, 10, S, kh, vh, [T], "f32")
    states = upload(sc, x.place(x.M))
    where = ops.gdn_states(states, n_seqs=1, v_heads=vh, state_size=S)
    out = upload(sc, np.zeros_like(x.v))
    bufs = [upload(sc, b) for b in (x.q, x.k, x.v, x.g, x.beta)]
    at = lambda b, t, w: b.ptr + 4 * t * w   # noqa: E731
    for lo, hi in ((0, 67), (67, 131), (131, 197), (197, 198), (198, 199), (199, 200)):
        ptrs = [at(b, lo, w) for b, w in zip(bufs, (kh * S, kh * S, vh * S, vh, vh))]
        kw = dict(k_heads=kh, n_seqs=1, tokens=hi - lo, scale=x.scale, l2norm=True)
        if hi - lo == 1:
            op = ops.GdnStep(where, *ptrs, at(out, lo, vh * S), "f32", **kw)
        else:
            op = ops.GdnChunk(where, *ptrs, at(out, lo, vh * S), "f32", cu=upload(sc, np.array([0, hi - lo])), **kw)
        op.launch()
        sc.device_sync()
    x.out, x.d_state = out, states
    x.out.shape = (T, vh * S)
    x.check(plain)


@pytest.mark.parametrize("step", [True, False], ids=["step", "chunk"])
def test_sequences_without_a_slot(sc, ops, plain, cuda, step):
    """A sequence whose state pointer is null gets zeros and touches nothing; rows past the batch are left."""
    S, kh, vh, lens = 128, 2, 4, [1, 1, 1] if step else [70, 33, 5]
    x = Layer(sc, ops, 11, S, kh, vh, lens, "f32", step=step, extra=0 if step else 9)
    op = x.build()
    bases = op._things[0].bases
    ptrs = bases.numpy()
    ptrs[1] = 0
    bases.upload(ptrs)
    op.launch()
    sc.device_sync()
    out, M = x.read()
    x.check(plain, seqs=[0, 2])
    assert np.array_equal(M[1], x.M[1])
    assert (out[x.cu[1]:x.cu[2]] == 0).all() and (out[sum(lens):] == 7).all()


def test_states_of_slots(sc, ops, plain, cuda):
    """A layer of decode slots: the rows of the other layers and the conv history keep every byte."""
    geo = sc.geometry(n_layers=8, ssm_state_size=64, ssm_k_heads=2, ssm_v_heads=4, ssm_conv_channels=256)
    slots = [sc.new_slot(geo, 8, fill=SENTINEL) for _ in range(3)]
    x = Layer(sc, ops, 12, 64, 2, 4, [1, 1, 1], "f32", step=True)
    layer, row, each = 3, geo.gdn_row_floats, 4 * 64 * 64
    for s, slot in enumerate(slots):
        slot.gdn.upload(x.place(x.M)[s], layer * row)
    out = upload(sc, np.zeros_like(x.v))
    ops.GdnStep(ops.slot_states(geo, slots, layer), *[upload(sc, b) for b in (x.q, x.k, x.v, x.g, x.beta)], out, "f32", k_heads=2,
                n_seqs=3, tokens=3, scale=x.scale, l2norm=True).launch()
    sc.device_sync()
    rows = [slot.gdn.numpy().reshape(-1) for slot in slots]
    for r in rows:
        rest = np.delete(r, np.s_[layer * row:layer * row + each])
        assert (rest.view(np.uint8) == SENTINEL).all()
    x.out, x.d_state = out, upload(sc, np.stack([r[layer * row:layer * row + each].reshape(64, 4, 64) for r in rows]))
    x.out.shape = (3, 4 * 64)
    x.check(plain)


@pytest.mark.parametrize("step", [True, False], ids=["step", "chunk"])
def test_the_same_every_time_and_on_another_stream(sc, ops, cuda, step):
    """Two runs agree bit for bit, and a call waits for the work before it on its own stream."""
    got = []
    for stream in (None, sc.Stream()):
        x = Layer(sc, ops, 13, 128, 2, 4, [1] * 4 if step else [333, 64], "f16", step=step)
        op = x.build()
        staged, state = upload(sc, x.place(x.M)), x.d_state
        state.fill(0xFF)
        sc.device_sync()
        if stream is not None:
            sc.delay_async(2000, stream)
        sc.check(sc.lib.sc_copy_device_async(state.ptr, staged.ptr, state.nbytes, None if stream is None else stream.handle), "copy")
        op.launch(stream)
        sc.device_sync()
        got.append(x.read())
    assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(*got))
