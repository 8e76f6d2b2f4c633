"""A conversation whose paged cache is held at a number of cells, with the operators of include/sc_ops.h around a hand-off.

The prompt has a picture in it: its tokens share positions in time and count through a grid, so positions of three axes turn
queries and keys.  Its recurrent layers run the short convolution and the gated delta rule.  One carve puts everything into a
decode slot; what the last queries attend to decides which cells are kept, and the slot is parked at that length and resumed
into another one.  Then every new token is convolved, appended behind the kept cells at its own position, attends, adds its
weights to the cells' mass, and steps the recurrent states; every few tokens the cache is cut to its size again.  The
projections around these operators are the engine's: here their results are random numbers.

    python strata-concurrent_amd/examples/bounded_conversation.py --layers 48 --prompt 8192 --keep 2048 --new 64
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import sc_handoff as sc  # noqa: E402
import sc_ops as ops  # noqa: E402

ROT, BASE, SECTIONS = 64, 1e7, (12, 10, 10)   # rotated values of a head, base of the frequencies, pairs of each axis
SINKS, RECENT = 4, 16                         # tokens that are kept whatever attends to them


def _up(x: np.ndarray) -> sc.DeviceBuffer:
    b = sc.DeviceBuffer(x.shape, x.dtype)
    b.upload(x)
    return b


def _copy(dst: int, src: int, size: int, stream=None) -> None:
    sc.check(sc.lib.sc_copy_device_async(dst, src, size, stream if stream is None else stream.handle), "copy")


def positions(first: int, words: int, grid: tuple[int, int], after: int) -> np.ndarray:
    """Positions [3][tokens] of words, a picture of grid[0] x grid[1] tokens, and words after it."""
    h, w = grid
    a = np.broadcast_to(first + np.arange(words), (3, words))
    p = first + words
    picture = p + np.stack([np.zeros(h * w, int), np.repeat(np.arange(h), w), np.tile(np.arange(w), h)])
    b = np.broadcast_to(p + max(h, w) + np.arange(after), (3, after))
    return np.ascontiguousarray(np.concatenate([a, picture, b], 1).astype(np.int64))


class Inputs:
    """What the projections of `tokens` tokens of every layer would have given, f32, the same for the same seed."""

    def __init__(self, geo: sc.Geometry, tokens: int, n_head: int, seed: int):
        rng = np.random.default_rng(seed)
        normal = lambda *shape: rng.standard_normal(shape).astype(np.float32)  # noqa: E731
        H, D, VH = geo.n_head_kv, geo.head_dim, geo.ssm_v_heads
        self.attn = [dict(q=normal(tokens, n_head, D), k=normal(tokens, H, D), v=normal(tokens, H, D)) for _ in range(geo.n_qsa)]
        self.gdn = [dict(x=normal(tokens, geo.ssm_conv_channels), g=-rng.random((tokens, VH), np.float32),
                         beta=rng.random((tokens, VH), np.float32)) for _ in range(geo.n_gdn)]


class Bounded:
    """The slot, and beside it each attention layer's masses and the numbers of the tokens that its cells hold."""

    def __init__(self, geo: sc.Geometry, n_head: int, keep: int, prompt: int, between: int):
        self.geo, self.n_head, self.keep, self.between = geo, n_head, keep, between
        # the slot's cells, which a hand-off makes fewer, and the width of the arrays beside it
        self.max_cells = self.width = geo.cells(max(prompt, keep) + between)
        self.slot = sc.new_slot(geo, self.max_cells)
        self.inv_freq = _up((BASE ** (-np.arange(0, ROT, 2) / ROT)).astype(np.float32))
        self.axis = ops.axis_of_pairs(SECTIONS, by_turns=True)
        rng = np.random.default_rng(7)
        C, W = geo.ssm_conv_channels, geo.ssm_d_conv
        self.taps = [_up((rng.standard_normal((C, W)) / W).astype(np.float32)) for _ in range(geo.n_gdn)]
        heads = (1, geo.n_head_kv, self.width)
        self.mass, self.born = ([sc.DeviceBuffer(heads, t) for _ in range(geo.n_qsa)] for t in ("float32", "int32"))
        for b in (*self.mass, *self.born):
            b.fill(0)
        one = lambda: sc.DeviceBuffer(1, "int64")  # noqa: E731
        # where the next token goes, cells and tokens so far, cells that eviction left last, and what it leaves now
        self.cell, self.len, self.total, self.known, self.left = one(), one(), one(), one(), one()
        for b in (self.cell, self.len, self.total, self.known):
            b.upload([0])
        self.cells = self.tokens = 0

    def _gdn(self, states, conv_out, x, out, **kw):
        """The delta rule over the convolution's outputs: a row's queries, keys and values lie side by side."""
        geo = self.geo
        S, KH, VH, C = geo.ssm_state_size, geo.ssm_k_heads, geo.ssm_v_heads, geo.ssm_conv_channels
        q = conv_out.ptr
        make = ops.GdnChunk if "cu" in kw else ops.GdnStep
        call = make(states, q, q + 4 * KH * S, q + 8 * KH * S, x["g"], x["beta"], out, "f32", k_heads=KH, n_seqs=1, scale=S ** -0.5, l2norm=True,
                    q_ld=C, k_ld=C, v_ld=C, **kw)
        call.keep = conv_out
        return call

    def prompt(self, x: Inputs, pos: np.ndarray, last: int) -> list[np.ndarray]:
        """The prompt's operators, the carve and the mass that its `last` queries give; the recurrent layers' outputs."""
        geo, T, n_head = self.geo, pos.shape[1], self.n_head
        H, D, S, VH, C, W = geo.n_head_kv, geo.head_dim, geo.ssm_state_size, geo.ssm_v_heads, geo.ssm_conv_channels, geo.ssm_d_conv
        cu, where = _up(np.array([0, T], np.int64)), _up(pos)
        k, v, q, rec, conv, outs, calls = [], [], [], [], [], [], []
        for layer in x.attn:
            k.append(sc.DeviceBuffer((T, H, D), "uint16"))
            v.append(sc.DeviceBuffer((T, H, D), "uint16"))
            q.append(_up(layer["q"]))
            # the prefill layout [T][H][D] is a cache with pages of one cell
            cache = ops.kv_cache(k[-1], v[-1], n_pages=T, n_head_kv=H, head_dim=D, page_size=1, table_ld=T)
            calls.append(ops.RopeAxesAppend(cache, _up(layer["k"]), _up(layer["v"]), "f32", n_seqs=1, tokens=T, cu=cu, pos0=self.cell,
                                            inv_freq=self.inv_freq, rot_dim=ROT, axis=self.axis, n_axes=3, pos=where, q=q[-1], q_out=q[-1],
                                            n_head=n_head))
        for layer, taps in zip(x.gdn, self.taps):
            rec.append(sc.DeviceBuffer((VH, S, S), "float32"))
            conv.append(sc.DeviceBuffer((W - 1, C), "float32"))
            rec[-1].fill(0), conv[-1].fill(0)
            y = sc.DeviceBuffer((T, C), "float32")
            outs.append(sc.DeviceBuffer((T, VH, S), "float32"))
            calls.append(ops.Conv(ops.conv_states(conv[-1], n_seqs=1, channels=C, taps=W, layout="rows"), _up(layer["x"]), taps, y, "f32",
                                  n_seqs=1, tokens=T, cu=cu))
            states = ops.gdn_states(rec[-1], n_seqs=1, v_heads=VH, state_size=S, layout="prefill")
            calls.append(self._gdn(states, y, {n: _up(layer[n]) for n in ("g", "beta")}, outs[-1], tokens=T, cu=cu))
        for call in calls:
            call.launch()
        plan = sc.plan_carve(geo, sc.PrefillBuffers(geo, T, k, v, rec, conv, W - 1), self.slot)
        plan.launch()
        sc.device_sync()
        plan.destroy()
        self.cells = self.tokens = T
        self.len.upload([T]), self.total.upload([T])
        for j in range(geo.n_qsa):
            ops.AttnMass(ops.slot_cache(geo, self.slot, j), q[j].ptr + 4 * (T - last) * n_head * D, self.mass[j], "f32", n_seqs=1, rows=last,
                         n_head=n_head, lens=self.len, max_len=self.max_cells, scale=D ** -0.5, mass_ld=self.width).launch()
        sc.device_sync()
        return [o.numpy() for o in outs]

    def evictions(self) -> list[ops.KvEvict]:
        """Every attention layer's eviction.  They read one array of lengths, so what they leave goes to another."""
        geo = self.geo
        return [ops.KvEvict(ops.slot_cache(geo, self.slot, j), self.mass[j], n_seqs=1, lens=self.len, max_len=self.max_cells, keep=self.keep,
                            sinks=SINKS, recent=RECENT, born=self.born[j], ld=self.width, known=self.known, total=self.total,
                            lens_out=self.left) for j in range(geo.n_qsa)]

    def evict(self, calls, stream=None) -> None:
        for call in calls:
            call.launch(stream)
        _copy(self.known.ptr, self.left.ptr, 8, stream)
        self.cells = min(self.cells, self.keep)

    def hand_off(self) -> None:
        """The slot parked at the length that it has and resumed into one with room for a bounded cache only: what it has or may keep, and
        the tokens up to the next eviction.  Calls made before are of the old slot."""
        geo = self.geo
        image = sc.PinnedBuffer(sc.image_layout(geo, self.cells)[1])
        sc.device_sync()
        sc.park_async(geo, self.slot, self.cells, image.ptr, image.nbytes)
        self.max_cells = geo.cells(max(self.cells, self.keep) + self.between)
        target = sc.new_slot(geo, self.max_cells)
        sc.resume_async(geo, image.ptr, image.nbytes, self.cells, target)
        sc.device_sync()
        self.slot = target
        image.free()


class Decoder:
    """The calls of one new token, made once: token t's inputs are copied to the same places for every t."""

    def __init__(self, b: Bounded, x: Inputs):
        geo, n_head, slot = b.geo, b.n_head, b.slot
        S, VH, D, C = geo.ssm_state_size, geo.ssm_v_heads, geo.head_dim, geo.ssm_conv_channels
        self.bounded, self.all, self.calls = b, [], []
        self.attn_out, self.gdn_out, self.pos = [], [], sc.DeviceBuffer((3, 1), "int64")

        def one(values):   # every token's rows on the device, and the place that a call reads
            whole, place = _up(values), sc.DeviceBuffer(values.shape[1:], values.dtype)
            self.all.append((whole, place))
            return place

        for j, layer in enumerate(x.attn):
            cache, q, lse = ops.slot_cache(geo, slot, j), one(layer["q"]), sc.DeviceBuffer(n_head, "float32")
            self.attn_out.append(sc.DeviceBuffer((n_head, D), "float32"))
            self.calls += [
                ops.RopeAxesAppend(cache, one(layer["k"]), one(layer["v"]), "f32", n_seqs=1, tokens=1, pos0=b.cell, inv_freq=b.inv_freq,
                                   rot_dim=ROT, axis=b.axis, n_axes=3, pos=self.pos, q=q, q_out=q, n_head=n_head),
                ops.AttnDecode(cache, q, self.attn_out[-1], "f32", n_seqs=1, n_head=n_head, lens=b.len, max_len=b.max_cells, scale=D ** -0.5,
                               lse=lse),
                ops.AttnMass(cache, q, b.mass[j], "f32", n_seqs=1, n_head=n_head, lens=b.len, max_len=b.max_cells, scale=D ** -0.5, lse=lse,
                             mass_ld=b.width)]
        for i, layer in enumerate(x.gdn):
            y = sc.DeviceBuffer((1, C), "float32")
            self.gdn_out.append(sc.DeviceBuffer((VH, S), "float32"))
            self.calls += [ops.Conv(ops.slot_conv(geo, [slot], i), one(layer["x"]), b.taps[i], y, "f32", n_seqs=1, tokens=1),
                           b._gdn(ops.slot_states(geo, [slot], i), y, {n: one(layer[n]) for n in ("g", "beta")}, self.gdn_out[-1], tokens=1)]

    def feed(self, t: int, position: int) -> None:
        b = self.bounded
        for whole, place in self.all:
            _copy(place.ptr, whole.ptr + t * place.nbytes, place.nbytes)
        self.pos.upload(np.full((3, 1), position, np.int64))
        b.cell.upload([b.cells])
        b.cells, b.tokens = b.cells + 1, b.tokens + 1
        b.len.upload([b.cells]), b.total.upload([b.tokens])

    def token(self, t: int, position: int, stream=None) -> None:
        self.feed(t, position)
        for call in self.calls:
            call.launch(stream)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=48)
    ap.add_argument("--heads", type=int, default=24)
    ap.add_argument("--prompt", type=int, default=8192)
    ap.add_argument("--keep", type=int, default=2048)
    ap.add_argument("--every", type=int, default=16)
    ap.add_argument("--new", type=int, default=64)
    a = ap.parse_args()
    geo = sc.geometry(n_layers=a.layers)
    b = Bounded(geo, a.heads, a.keep, a.prompt, a.every)
    side = int((a.prompt // 2) ** 0.5)
    pos = positions(0, a.prompt // 4, (side, side), a.prompt - a.prompt // 4 - side * side)
    t0 = time.perf_counter()
    b.prompt(Inputs(geo, a.prompt, a.heads, 1), pos, min(32, a.prompt))
    print(f"prompt of {a.prompt} tokens: operators and carve, inputs made on the host, {time.perf_counter() - t0:.2f} s", flush=True)
    b.evict(b.evictions())
    b.hand_off()
    print(f"handed off with {b.cells} cells", flush=True)
    dec, cut = Decoder(b, Inputs(geo, a.new, a.heads, 2)), b.evictions()
    spent, cuts, n_cuts = 0.0, 0.0, 0
    for t in range(a.new):
        dec.feed(t, int(pos.max()) + 1 + t)
        sc.device_sync()
        t0 = time.perf_counter()
        for call in dec.calls:
            call.launch()
        sc.device_sync()
        spent += time.perf_counter() - t0 if t else 0
        if (t + 1) % a.every == 0:
            t0 = time.perf_counter()
            b.evict(cut)
            sc.device_sync()
            cuts, n_cuts = cuts + time.perf_counter() - t0, n_cuts + 1
    if a.new > 1:
        print(f"a new token's operators in {geo.n_qsa} attention and {geo.n_gdn} recurrent layers: {spent / (a.new - 1) * 1e6:.0f} us, "
              f"{len(dec.calls)} calls; an eviction in every attention layer {cuts / max(n_cuts, 1) * 1e6:.0f} us", flush=True)


if __name__ == "__main__":
    main()
