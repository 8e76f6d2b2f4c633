"""One conversation from its prompt to its first new tokens, with the operators of include/sc_ops.h around a hand-off.

A prompt's recurrent layers run by chunks into the prefill layout and its full-attention layers write their rotated keys and
values there; one carve puts both into a decode slot; then every new token is appended, attends over the paged cache and
steps the recurrent states, in place in the slot.  The projections around these operators are the engine's: here their
results are random numbers.

    python strata-concurrent_amd/examples/decode_after_handoff.py --layers 48 --prompt 8192 --new 64
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

ROT, BASE = 64, 1e7   # rotated values of a head, base of the rotation's frequencies


def _up(x: np.ndarray) -> sc.DeviceBuffer:
    b = sc.DeviceBuffer(x.shape, x.dtype)
    b.upload(x)
    return b


class Inputs:
    """What the projections of `tokens` tokens of every layer would have given, f32, the same for the same seed."""

    def __init__(self, geo: sc.Geometry, tokens: int, n_head: int, seed: int):
        rng = np.random.default_rng(seed)
        normal = lambda *shape: rng.standard_normal(shape).astype(np.float32)  # noqa: E731
        H, D, S, KH, VH = geo.n_head_kv, geo.head_dim, geo.ssm_state_size, geo.ssm_k_heads, geo.ssm_v_heads
        self.attn = [dict(q=normal(tokens, n_head, D), k=normal(tokens, H, D), v=normal(tokens, H, D)) for _ in range(geo.n_qsa)]
        self.gdn = [dict(q=normal(tokens, KH, S), k=normal(tokens, KH, S), v=normal(tokens, VH, S),
                         g=-rng.random((tokens, VH), np.float32), beta=rng.random((tokens, VH), np.float32))
                    for _ in range(geo.n_gdn)]


class Conversation:
    def __init__(self, geo: sc.Geometry, n_head: int, max_cells: int):
        self.geo, self.n_head = geo, n_head
        self.slot = sc.new_slot(geo, geo.cells(max_cells))
        self.inv_freq = _up((BASE ** (-np.arange(0, ROT, 2) / ROT)).astype(np.float32))
        self.pos, self.len = sc.DeviceBuffer(1, "int64"), sc.DeviceBuffer(1, "int64")
        self.cells = 0

    def prompt(self, x: Inputs) -> list[np.ndarray]:
        """The prompt's operators and the carve; the recurrent layers' outputs [tokens][heads][S]."""
        geo, T = self.geo, len(x.gdn[0]["g"])
        H, D, S, KH, VH = geo.n_head_kv, geo.head_dim, geo.ssm_state_size, geo.ssm_k_heads, geo.ssm_v_heads
        cu = _up(np.array([0, T], np.int64))
        self.pos.upload([0])
        k, v, rec, outs, calls = [], [], [], [], []
        for layer in x.attn:
            k.append(sc.DeviceBuffer((T, H, D), "uint16"))
            v.append(sc.DeviceBuffer((T, H, D), "uint16"))
            # the prefill layout [T][H][D] is a cache with pages of one cell
            cache = ops.kv_cache(k[-1], v[-1], n_pages=T, n_head_kv=H, head_dim=D, page_size=1, table_ld=T)
            calls.append(ops.RopeAppend(cache, _up(layer["k"]), _up(layer["v"]), "f32", n_seqs=1, tokens=T, cu=cu, pos0=self.pos,
                                        inv_freq=self.inv_freq, rot_dim=ROT))
        for layer in x.gdn:
            rec.append(sc.DeviceBuffer((VH, S, S), "float32"))
            rec[-1].fill(0)
            outs.append(sc.DeviceBuffer((T, VH, S), "float32"))
            states = ops.gdn_states(rec[-1], n_seqs=1, v_heads=VH, state_size=S, layout="prefill")
            calls.append(ops.GdnChunk(states, *(_up(layer[n]) for n in ("q", "k", "v", "g", "beta")), outs[-1], "f32", k_heads=KH,
                                      n_seqs=1, tokens=T, cu=cu, scale=S ** -0.5, l2norm=True))
        for call in calls:
            call.launch()
        rows = min(T, geo.ssm_d_conv - 1)
        conv = [_up(np.zeros((max(rows, 1), geo.ssm_conv_channels), np.float32)) for _ in range(geo.n_gdn)]
        plan = sc.plan_carve(geo, sc.PrefillBuffers(geo, T, k, v, rec, conv, rows), self.slot)
        plan.launch()
        sc.device_sync()
        plan.destroy()
        self.cells = T
        return [o.numpy() for o in outs]

    def decoder(self, x: Inputs) -> "Decoder":
        return Decoder(self, x)


class Decoder:
    """The calls of one new token, made once: token t's inputs are copied to the same places for every t."""

    def __init__(self, conv: Conversation, x: Inputs):
        geo, n_head, slot = conv.geo, conv.n_head, conv.slot
        S, KH, VH, D = geo.ssm_state_size, geo.ssm_k_heads, geo.ssm_v_heads, geo.head_dim
        self.conv, self.all, self.calls = conv, [], []
        self.attn_out, self.gdn_out = [], []

        def one(values):   # every token's rows on the device, and the place that a call reads
            whole, place = _up(values), sc.DeviceBuffer(values.shape[1:], values.dtype)
            self.all.append((whole, place))
            return place

        for j, layer in enumerate(x.attn):
            cache, q = ops.slot_cache(geo, slot, j), one(layer["q"])
            self.attn_out.append(sc.DeviceBuffer((n_head, D), "float32"))
            self.calls.append(ops.RopeAppend(cache, one(layer["k"]), one(layer["v"]), "f32", n_seqs=1, tokens=1, pos0=conv.pos,
                                             inv_freq=conv.inv_freq, rot_dim=ROT, q=q, q_out=q, n_head=n_head))
            self.calls.append(ops.AttnDecode(cache, q, self.attn_out[-1], "f32", n_seqs=1, n_head=n_head, lens=conv.len,
                                             max_len=slot.max_cells, scale=D ** -0.5))
        for i, layer in enumerate(x.gdn):
            self.gdn_out.append(sc.DeviceBuffer((VH, S), "float32"))
            self.calls.append(ops.GdnStep(ops.slot_states(geo, [slot], i), *(one(layer[n]) for n in ("q", "k", "v", "g", "beta")),
                                          self.gdn_out[-1], "f32", k_heads=KH, n_seqs=1, tokens=1, scale=S ** -0.5, l2norm=True))

    def feed(self, t: int) -> None:
        for whole, place in self.all:
            sc.check(sc.lib.sc_copy_device_async(place.ptr, whole.ptr + t * place.nbytes, place.nbytes, None), "copy")
        self.conv.pos.upload([self.conv.cells])
        self.conv.cells += 1
        self.conv.len.upload([self.conv.cells])

    def token(self, t: int) -> None:
        self.feed(t)
        for call in self.calls:
            call.launch()


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=48)
    ap.add_argument("--heads", type=int, default=24)
    ap.add_argument("--prompt", type=int, default=8192)
    ap.add_argument("--new", type=int, default=64)
    a = ap.parse_args()
    geo = sc.geometry(n_layers=a.layers)
    conv = Conversation(geo, a.heads, a.prompt + a.new)
    t0 = time.perf_counter()
    conv.prompt(Inputs(geo, a.prompt, a.heads, 1))
    print(f"prompt of {a.prompt} tokens: operators and carve, inputs made on the host, {time.perf_counter() - t0:.2f} s", flush=True)
    dec = conv.decoder(Inputs(geo, a.new, a.heads, 2))
    dec.token(0)
    sc.device_sync()
    spent = 0.0
    for t in range(1, a.new):
        dec.feed(t)
        sc.device_sync()
        t0 = time.perf_counter()
        for call in dec.calls:
            call.launch()
        sc.device_sync()
        spent += time.perf_counter() - t0
    if a.new > 1:
        print(f"a new token's operators in {geo.n_qsa} attention and {geo.n_gdn} recurrent layers: "
              f"{spent / (a.new - 1) * 1e6:.0f} us, {len(dec.calls)} calls", flush=True)


if __name__ == "__main__":
    main()
