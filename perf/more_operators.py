"""The measured operators of a decode slot whose cache is kept bounded, and of the convolution before its recurrent layers.

`conv`   the short causal convolution over a recurrent layer's inputs, its history carried in the slot
`axes`   new tokens' keys and values written to a paged cache, turned by positions of several axes; queries turned too
`mass`   the attention weights that the latest queries give each cell, added to what the cell has had before
`evict`  the cells with the most weight kept, and moved to the front of the cache
"""
import math
import random

import numpy as np
import torch

own = False

THETA = 1e7          # base of the rotation's frequencies
BLOCK = 64           # values that share a scale in an int8 cache
F = {"f16": torch.float16, "f32": torch.float32}
# attention heads, kv heads, head size and page size of the configurations: the full-depth one
FULL = {"heads": 24, "kv": 2, "dim": 256, "page": 4}
# channels and taps of the recurrent layers' convolution
CONV = {"channels": 8192, "taps": 4}


def listed():
    return [
        # one conversation's new token in one recurrent layer: launch latency
        {"name": "conv_1", "kind": "conv", "act": "f32", "seqs": 1, "most": 1, "layout": "slot", **CONV},
        # a batch of conversations decodes, histories in their slots
        {"name": "conv_61_f16", "kind": "conv", "act": "f16", "seqs": 61, "most": 1, "layout": "slot", **CONV},
        # the chunks of eight prompts, of ragged lengths up to 2048 tokens, into the rows that a carve reads
        {"name": "conv_8x2048", "kind": "conv", "act": "f32", "seqs": 8, "most": 2048, "layout": "rows", **CONV},
        # one conversation's new token after a picture: latency
        {"name": "axes_1", "kind": "axes", "fmt": "f16", "act": "f32", "seqs": 1, "most": 1, "rot": 64, "pairs": "halves",
         "axes": 3, "order": "turns", "pos": 4093, **FULL},
        # a batch's new tokens into int8 caches
        {"name": "axes_61_int8", "kind": "axes", "fmt": "int8", "act": "f16", "seqs": 61, "most": 1, "rot": 64,
         "pairs": "halves", "axes": 3, "order": "turns", "pos": 30011, **FULL},
        # eight prompts with pictures between their words
        {"name": "axes_8x2048", "kind": "axes", "fmt": "f16", "act": "f16", "seqs": 8, "most": 2048, "rot": 128,
         "pairs": "halves", "axes": 3, "order": "runs", "pos": 6141, **FULL},
        # a short conversation's new token: its attention has left the log of its sum
        {"name": "mass_1x1021", "kind": "mass", "fmt": "f16", "act": "f32", "seqs": 1, "most": 1021, "rows": 1, "given": True, **FULL},
        # a batch's new tokens over int8 caches
        {"name": "mass_24x8190_int8", "kind": "mass", "fmt": "int8", "act": "f16", "seqs": 24, "most": 8190, "rows": 1, "given": True, **FULL},
        # the last 32 queries of two prompts, before they are handed off: many rows, no sums in hand
        {"name": "mass_2x16381_rows32", "kind": "mass", "fmt": "f16", "act": "f16", "seqs": 2, "most": 16381, "rows": 32, "given": False, **FULL},
        # a prompt of 128K cells cut to an eighth before its hand-off
        {"name": "evict_1x131072", "kind": "evict", "fmt": "f16", "seqs": 1, "most": 131072, "keep": 16384, "sinks": 4, "recent": 64,
         "again": 0, **FULL},
        # a batch whose bounded caches have grown by 16 cells since the last time
        {"name": "evict_32x2064", "kind": "evict", "fmt": "f16", "seqs": 32, "most": 2064, "keep": 2048, "sinks": 4, "recent": 128,
         "again": 2048, **FULL},
        # ragged int8 caches, some of them shorter than what is kept
        {"name": "evict_8x4090_int8", "kind": "evict", "fmt": "int8", "seqs": 8, "most": 4090, "keep": 1000, "sinks": 0, "recent": 32,
         "again": 0, **FULL},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["conv", "axes", "mass", "mass", "evict", "evict"])
    act, fmt = rng.choice(["f16", "f32"]), rng.choice(["f16", "int8"])
    kv = rng.choice([1, 2, 2, 4])
    heads = {"heads": kv * rng.choice([1, 4, 8, 12, 16]), "kv": kv, "dim": rng.choice([64, 128, 256]), "page": rng.choice([1, 4, 4, 8, 16])}
    seqs = _log(rng, 1, 64)
    if kind == "conv":
        channels = 8 * _log(rng, 8, 1536)
        most = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 8192 * 8192 // channels // seqs))
        return {"kind": kind, "act": act, "seqs": seqs, "most": most, "layout": rng.choice(["slot", "rows"]), "channels": channels,
                "taps": rng.choice([2, 3, 4, 4, 5])}
    if kind == "axes":
        most = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 8192 * 24 * 256 // (heads["heads"] * heads["dim"]) // seqs))
        return {"kind": kind, "fmt": fmt, "act": act, "seqs": seqs, "most": most,
                "rot": rng.choice([heads["dim"], heads["dim"] // 2, heads["dim"] // 4]), "pairs": rng.choice(["halves", "neighbours"]),
                "axes": rng.choice([1, 2, 3, 3, 4]), "order": rng.choice(["turns", "runs"]), "pos": _log(rng, 1, 65536) - 1, **heads}
    if kind == "mass":
        rows = 1 if rng.random() < 0.5 else _log(rng, 2, 64)
        cells = min(100_000_000 // (kv * heads["dim"]), 6_000_000_000 // (rows * heads["heads"] * heads["dim"]))
        return {"kind": kind, "fmt": fmt, "act": act, "seqs": seqs, "most": _log(rng, 1, min(131072, cells // seqs)), "rows": rows,
                "given": rng.choice([True, False]), **heads}
    most = _log(rng, 64, min(131072, 65_000_000 // (kv * heads["dim"]) // seqs))
    keep = _log(rng, 16, most)
    recent = rng.choice([0, rng.randint(0, keep // 2)])
    # the cells that an eviction before this one has left, in no order
    again = rng.choice([0, 0, rng.randint(1, most)])
    return {"kind": kind, "fmt": fmt, "seqs": seqs, "most": most, "keep": keep, "sinks": rng.choice([0, 4]), "recent": recent,
            "again": again, **heads}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _lens(case):
    """A batch's lengths: ragged up to the most, the longest among them; one sequence has the most."""
    n, most = case["seqs"], case["most"]
    r = random.Random(n * 1000003 + most)
    if case.get("again"):   # caches held at one size have grown alike
        return [most] * n
    return [most] + [max(1, int(most * (1 / 128 + 127 / 128 * r.random()))) for _ in range(n - 1)]


def _pages(case, cells):
    return -(-cells // case["page"])


def _axis(case):
    """The axis whose position turns each pair: the axes one after another in runs, or by turns as long as each has pairs left."""
    n, A = case["rot"] // 2, case["axes"]
    runs = [(i + 1) * n // A - i * n // A for i in range(A)]
    if case["order"] == "runs":
        return [a for a, k in enumerate(runs) for _ in range(k)]
    got, left = [], list(runs)
    while len(got) < n:
        for a in range(A):
            if left[a]:
                got.append(a)
                left[a] -= 1
    return got


def _positions(case, lens, first, seed):
    """Positions of every token on every axis: words have the same on all, a picture's tokens count through a grid."""
    r, A, all_ = random.Random(seed), case["axes"], []
    for n, p in zip(lens, first):
        got = np.zeros((A, 0), np.int64)
        while got.shape[1] < n:
            words = min(n, 1 + r.randrange(200))
            got = np.concatenate([got, np.broadcast_to(p + np.arange(words), (A, words))], 1)
            p += words
            h, w = 4 + r.randrange(20), 4 + r.randrange(20)
            grid = np.stack(np.meshgrid(np.arange(1), np.arange(h), np.arange(w), indexing="ij")).reshape(3, -1)
            grid = np.concatenate([grid, grid[:1]])[[0, 1, 2, 3][:A]]
            got, p = np.concatenate([got, p + grid], 1), p + max(h, w)
        all_.append(got[:, :n])
    return np.ascontiguousarray(np.concatenate(all_, 1))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    n, act, lens, kind = case["seqs"], F[case.get("act", "f32")], _lens(case), case["kind"]
    normal = lambda *shape, dtype=torch.float32, by=1.0: (torch.randn(shape, device="cuda", generator=g) * by).to(dtype)  # noqa: E731
    host = lambda x, dtype: torch.tensor(x, dtype=dtype, device="cuda")  # noqa: E731
    if kind in ("conv", "axes"):
        N = s["tokens"] = sum(lens)
        s["cu"], s["longest"] = host(np.cumsum([0, *lens]).tolist(), torch.int64), max(lens)
    if kind == "conv":
        C, W = case["channels"], case["taps"]
        s["x"], s["out"] = normal(N, C, dtype=act), torch.empty((N, C), dtype=act, device="cuda")
        s["weight"], s["bias"] = normal(C, W, by=W ** -0.5), normal(C, by=0.1)
        s["state"] = normal(*((n, C, W - 1) if case["layout"] == "slot" else (n, W - 1, C)))
        if own:
            s["op"] = _operator(s)
        return s
    H, D, ps = case["kv"], case["dim"], case["page"]
    if kind == "axes":
        # each sequence's new tokens begin at a cell of their own; its older pages lie in no pool here
        cell = [case["pos"] + 131 * i % 977 for i in range(n)]
        spans = [(p // ps, _pages(case, p + t)) for p, t in zip(cell, lens)]
    else:
        spans = [(0, _pages(case, t)) for t in lens]
    s["ld"] = max(e for _, e in spans)
    s["pages"] = sum(e - b for b, e in spans)
    phys = torch.randperm(s["pages"], device="cuda", generator=g).to(torch.int32)
    s["table"] = torch.full((n, s["ld"]), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, (b, e) in enumerate(spans):
        s["table"][i, b:e] = phys[at:at + e - b]
        at += e - b
    rows = (s["pages"], H, ps)
    if case["fmt"] == "f16":
        pool = lambda: torch.zeros(*rows, D, dtype=torch.float16, device="cuda") if kind == "axes" else normal(*rows, D, dtype=torch.float16)  # noqa: E731
        s["kc"], s["vc"] = pool(), pool()
    else:
        codes = lambda: torch.randint(-127, 128, (*rows, D), dtype=torch.int8, device="cuda", generator=g)  # noqa: E731
        scales = lambda: (0.01 + 0.02 * torch.rand((*rows, D // BLOCK), device="cuda", generator=g)).half()  # noqa: E731
        s["kc"], s["vc"], s["ks"], s["vs"] = codes(), codes(), scales(), scales()
    if kind == "axes":
        s["cell0"] = host(cell, torch.int64)
        s["axis"] = _axis(case)
        # pictures before this chunk have put positions behind cells
        s["pos_at"] = torch.from_numpy(_positions(case, lens, [c - c // 5 for c in cell], int(seed))).cuda()
        s["inv_freq"] = (THETA ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])).float().cuda()
        s["q"], s["k"], s["v"] = normal(N, case["heads"], D, dtype=act), normal(N, H, D, dtype=act), normal(N, H, D, dtype=act)
        s["q_out"] = torch.empty_like(s["q"])
    s["lens"] = host(lens, torch.int64)
    if kind == "mass":
        s["q"] = normal(n, case["rows"], case["heads"], D, dtype=act)
        # what queries before these have given
        s["mass"] = torch.rand((n, H, case["most"]), device="cuda", generator=g) * (case["rows"] * case["heads"] / H / case["most"])
        s["lse"] = _sums(s) if case["given"] else None
    if kind == "evict":
        most, again = case["most"], case["again"]
        # weights over many powers of ten, as attention leaves them, a few of them the same
        s["mass"] = torch.exp2(torch.round(normal(n, H, most, by=2.5 * 64)) / 64)
        s["mass_out"], s["lens_out"] = torch.zeros_like(s["mass"]), torch.zeros_like(s["lens"])
        s["born_out"] = torch.zeros((n, H, most), dtype=torch.int32, device="cuda")
        # after an eviction a cell's place says nothing about its age: its token's number is kept beside it
        s["known"], s["born"], s["total"] = host([min(again, t) for t in lens], torch.int64), None, s["lens"]
        if again:
            s["total"] = s["lens"] + most
            s["born"] = torch.zeros((n, H, most), dtype=torch.int32, device="cuda")
            top = 2 * most - again   # numbers below those of the cells that came since
            key = torch.rand((n, H, top), device="cuda", generator=g).argsort(-1)[..., :min(again, top)]
            s["born"][..., :key.shape[-1]] = key.to(torch.int32)
    if own:
        s["op"] = _operator(s)
    return s


# ---- the framework's operators -----------------------------------------------------------------------------------------

def _operator(s):
    """The handle that a serving program keeps for a layer: the tensors' places, the operator's workspace."""
    import sys
    from pathlib import Path
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "strata-concurrent_amd"))
    import sc_ops
    if s["kind"] == "conv":
        states = sc_ops.conv_states(s["state"], n_seqs=s["seqs"], channels=s["channels"], taps=s["taps"], layout=s["layout"])
        return sc_ops.Conv(states, s["x"], s["weight"], s["out"], s["act"], n_seqs=s["seqs"], tokens=s["tokens"],
                           cu=None if s["longest"] == 1 else s["cu"], bias=s["bias"], activation="silu")
    cache = sc_ops.kv_cache(s["kc"], s["vc"], s.get("ks"), s.get("vs"), n_pages=s["pages"], n_head_kv=s["kv"], head_dim=s["dim"],
                            page_size=s["page"], table=s["table"], table_ld=s["ld"])
    if s["kind"] == "axes":
        return sc_ops.RopeAxesAppend(cache, s["k"], s["v"], s["act"], n_seqs=s["seqs"], tokens=s["tokens"], cu=s["cu"], pos0=s["cell0"],
                                     inv_freq=s["inv_freq"], rot_dim=s["rot"], pairs=s["pairs"], axis=s["axis"], pos=s["pos_at"],
                                     pos_ld=s["tokens"], n_axes=s["axes"], q=s["q"], q_out=s["q_out"], n_head=s["heads"])
    if s["kind"] == "mass":
        return sc_ops.AttnMass(cache, s["q"], s["mass"], s["act"], n_seqs=s["seqs"], rows=s["rows"], n_head=s["heads"], lens=s["lens"],
                               max_len=s["most"], scale=s["dim"] ** -0.5, lse=s["lse"])
    return sc_ops.KvEvict(cache, s["mass"], n_seqs=s["seqs"], lens=s["lens"], max_len=s["most"], keep=s["keep"], sinks=s["sinks"],
                          recent=s["recent"], mass_out=s["mass_out"], born=s["born"], born_out=s["born_out"],
                          known=s["known"] if s["again"] else None, total=s["total"], lens_out=s["lens_out"])


def run(s):
    if own:
        s["op"].launch()
    else:
        {"conv": _conv, "axes": _axes, "mass": _mass, "evict": _evict}[s["kind"]](s)
    if s["kind"] == "conv":
        return s["out"], s["state"]
    if s["kind"] == "mass":
        return s["mass"]
    # an int8 cache comes back as the values that it stands for, in the type that the scales have
    worth = lambda c, x: c if x is None else c.view(*x.shape, BLOCK) * x[..., None]  # noqa: E731
    pools = worth(s["kc"], s.get("ks")), worth(s["vc"], s.get("vs"))
    return (s["q_out"], *pools) if s["kind"] == "axes" else (*pools, s["mass_out"], s["born_out"], s["lens_out"])


# ---- plain forms ---------------------------------------------------------------------------------------------------------

def _conv(s):
    W = s["taps"]
    hist = s["state"].transpose(1, 2) if s["layout"] == "slot" else s["state"]   # [sequences, taps - 1, channels]
    at = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["cu"], at, right=True) - 1
    local = at - s["cu"][seq]

    def before(seq, row, local):   # the rows at `local` of their sequences, the history's where that is before the first
        past = hist[seq, (local + W - 1).clamp(0, W - 2)]
        return torch.where((local < 0)[:, None], past, s["x"][row.clamp(0, s["tokens"] - 1)].float())

    y = s["bias"] + sum(s["weight"][:, W - 1 - d] * before(seq, at - d, local - d) for d in range(W))
    each, lens = torch.arange(s["seqs"], device="cuda"), s["cu"][1:] - s["cu"][:-1]
    new = torch.stack([before(each, s["cu"][1:] - d, lens - d) for d in range(W - 1, 0, -1)], 1)
    s["out"].copy_(y * torch.sigmoid(y))
    hist.copy_(new)


def _turn(x, cos, sin, rot, pairs):
    """The first `rot` values of each head turned by their pairs' angles."""
    x = x.to(cos.dtype)
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if pairs == "halves" else (x[..., :rot:2], x[..., 1:rot:2])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([a, b], -1) if pairs == "halves" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _codes(x):
    """int8 codes and f16 scales of blocks of values."""
    x = x.unflatten(-1, (-1, BLOCK))
    scale = (x.abs().amax(-1) / 127).half()
    code = torch.where(scale[..., None] > 0, (x / scale[..., None].to(x.dtype)).round().clamp(-127, 127), torch.zeros_like(x))
    return code.to(torch.int8).flatten(-2), scale


def _axes(s):
    at = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["cu"], at, right=True) - 1
    cell = s["cell0"][seq] + at - s["cu"][seq]
    page, off = s["table"][seq, cell // s["page"]].long(), cell % s["page"]
    pos = s["pos_at"][torch.tensor(s["axis"], device="cuda")].T
    angle = (pos.double() * s["inv_freq"])[:, None]   # a product in 32 bits would be off by thousandths at these positions
    cos, sin = angle.cos().float(), angle.sin().float()
    k = _turn(s["k"], cos, sin, s["rot"], s["pairs"])
    s["q_out"].copy_(_turn(s["q"], cos, sin, s["rot"], s["pairs"]))
    v = s["v"].float()
    if s["fmt"] == "f16":
        s["kc"][page, :, off], s["vc"][page, :, off] = k.half(), v.half()
    else:
        (s["kc"][page, :, off], s["ks"][page, :, off]), (s["vc"][page, :, off], s["vs"][page, :, off]) = _codes(k), _codes(v)


def _scores(s):
    """Scores [sequences, kv heads, rows, query heads of each, cells], -inf where a row does not see a cell."""
    n, H, R, G = s["seqs"], s["kv"], s["rows"], s["heads"] // s["kv"]
    page = s["table"].clamp_min(0).long()
    k = s["kc"][page].float()
    if s["fmt"] == "int8":
        k = (k.unflatten(-1, (-1, BLOCK)) * s["ks"][page].float()[..., None]).flatten(-2)
    k = k.transpose(1, 2).flatten(2, 3)[:, :, :s["most"]]
    q = s["q"].float().view(n, R, H, G, s["dim"]).transpose(1, 2).reshape(n, H, R * G, s["dim"]) * s["dim"] ** -0.5
    score = (q @ k.transpose(2, 3).contiguous()).view(n, H, R, G, -1)
    ends = s["lens"][:, None] - R + 1 + torch.arange(R, device="cuda")
    seen = torch.arange(k.shape[2], device="cuda") < ends[..., None]
    return score.masked_fill_(~seen[:, None, :, None], -math.inf)


def _sums(s):
    """The log of each query's sum of exponentials [sequences * rows, heads], -inf where it sees nothing."""
    score = _scores(s)
    top = score.amax(-1, keepdim=True).clamp_min(-1e30)
    lse = (top + (score - top).exp().sum(-1, keepdim=True).log())[..., 0]
    return lse.transpose(1, 2).reshape(s["seqs"] * s["rows"], s["heads"]).contiguous()


def _mass(s):
    n, H, R, G = s["seqs"], s["kv"], s["rows"], s["heads"] // s["kv"]
    score = _scores(s)
    if s["given"]:
        lse = s["lse"].view(n, R, H, G).transpose(1, 2)[..., None]
        p = (score - lse.clamp_min(-1e30)).exp()
    else:
        p = (score - score.amax(-1, keepdim=True).clamp_min(-1e30)).exp()
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    s["mass"] += p.sum((2, 3))


def _evict(s):
    n, H, most, keep, ps = s["seqs"], s["kv"], s["most"], s["keep"], s["page"]
    cell, lens = torch.arange(most, device="cuda"), s["lens"][:, None, None]
    born = (s["total"][:, None, None] - lens + cell).expand(n, H, most)
    if s["born"] is not None:
        born = torch.where(cell < s["known"][:, None, None], s["born"].long(), born)
    first = (born < s["sinks"]) | (born >= s["total"][:, None, None] - s["recent"])
    key = torch.where(first, torch.full_like(s["mass"], math.inf), s["mass"]).masked_fill(cell >= lens, -math.inf)
    order = key.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.zeros((n, H, most), dtype=torch.bool, device="cuda").scatter_(-1, order, True) & (cell < lens)
    over = lens > keep
    to = (over & ~kept & (cell < keep)).nonzero(as_tuple=True)
    of = (over & kept & (cell >= keep)).nonzero(as_tuple=True)

    def rows(i):
        return (s["table"][i[0], i[2] // ps].long() * H + i[1]) * ps + i[2] % ps

    dst, src = rows(to), rows(of)
    for c in ("kc", "vc", "ks", "vs"):
        if c in s:
            pool = s[c].view(-1, s[c].shape[-1])
            pool[dst] = pool[src]
    after = torch.minimum(lens, torch.full_like(lens, keep))
    s["mass_out"].copy_(torch.where(cell < after, s["mass"], torch.zeros_like(s["mass"])))
    s["born_out"].copy_(torch.where(cell < after, born, s["born_out"]))
    s["mass_out"][to], s["born_out"][to] = s["mass"][of], born[of].to(torch.int32)
    s["lens_out"].copy_(after[:, 0, 0])


# ---- 64 bits -------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    return {"conv": _conv_64, "axes": _axes_64, "mass": _mass_64, "evict": _evict_64}[case["kind"]](case, prepare(case, seed))


def _conv_64(case, s):
    W, cu, out, states = case["taps"], s["cu"].tolist(), [], []
    for i, (b, e) in enumerate(zip(cu, cu[1:])):
        hist = s["state"][i].double()
        x = torch.cat([hist.T if case["layout"] == "slot" else hist, s["x"][b:e].double()])
        y = (x.unfold(0, W, 1) * s["weight"].double()).sum(-1) + s["bias"].double()
        out.append(y / (1 + (-y).exp()))
        states.append(x[-(W - 1):].T if case["layout"] == "slot" else x[-(W - 1):])
    return torch.cat(out), torch.stack(states)


def _axes_64(case, s):
    cu, cell0, table, ps, R = s["cu"].tolist(), s["cell0"].tolist(), s["table"].cpu(), case["page"], case["rot"]
    cell = torch.cat([p + torch.arange(e - b) for p, b, e in zip(cell0, cu, cu[1:])])
    page = torch.cat([table[i, (p + torch.arange(e - b)) // ps] for i, (p, b, e) in enumerate(zip(cell0, cu, cu[1:]))]).long()
    pos = np.stack([s["pos_at"].cpu().numpy()[a] for a in s["axis"]], 1).astype(np.float64)
    angle = torch.from_numpy(pos * s["inv_freq"].double().cpu().numpy())
    turn = torch.complex(torch.cos(angle), torch.sin(angle))[:, None]

    def turned(x):   # a pair of values as a complex number
        x = x.double().cpu()
        z = x[..., :R].unflatten(-1, (2, R // 2) if case["pairs"] == "halves" else (R // 2, 2))
        z = z.movedim(-2, -1) if case["pairs"] == "halves" else z
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
        z = z.movedim(-1, -2) if case["pairs"] == "halves" else z
        return torch.cat([z.flatten(-2), x[..., R:]], -1)

    found = [turned(s["q"])]
    for x, c in ((turned(s["k"]), "k"), (s["v"].double().cpu(), "v")):
        rows = s[c + "c"].double().cpu()
        if case["fmt"] == "int8":   # the cache's values are the rounded ones by definition
            rows = rows.view(*rows.shape[:3], -1, BLOCK) * s[c + "s"].double().cpu()[..., None]
            x = x.view(*x.shape[:2], -1, BLOCK)
            step = (x.abs().max(-1, keepdim=True).values / 127).half().double()
            x = (x / step).round().clamp(-127, 127) * step
        rows[page, :, cell % ps] = x
        found.append(rows)
    return found


def _mass_64(case, s):
    mass, G, R = s["mass"].double(), case["heads"] // case["kv"], case["rows"]
    for i, n in enumerate(s["lens"].tolist()):
        cell = torch.arange(n, device="cuda")
        page, off = s["table"][i, cell // case["page"]].long(), cell % case["page"]
        k = s["kc"][page, :, off].double()   # [cells, kv heads, values]
        if case["fmt"] == "int8":
            k *= s["ks"][page, :, off].double().repeat_interleave(BLOCK, -1)
        for r in range(R):
            ends = n - R + 1 + r
            if ends <= 0:
                continue
            for h in range(case["kv"]):
                q = s["q"][i, r, h * G:(h + 1) * G].double()
                score = (k[:ends, h] @ q.T.contiguous()) / math.sqrt(case["dim"])
                p = (score - s["lse"][i * R + r, h * G:(h + 1) * G].double()).exp() if case["given"] else score.softmax(0)
                mass[i, h, :ends] += p.sum(1)
    return mass


def _evict_64(case, s):
    keep, ps, H = case["keep"], case["page"], case["kv"]
    pools = {c: s[c].reshape(-1, s[c].shape[-1]).cpu().numpy().copy() for c in ("kc", "vc", "ks", "vs") if c in s}
    table, lens, total, known = (s[x].cpu().numpy() for x in ("table", "lens", "total", "known"))
    mass, born_out = s["mass"].cpu().numpy().astype(np.float64), s["born_out"].cpu().numpy().copy()
    born = None if s["born"] is None else s["born"].cpu().numpy()
    mass_out = np.zeros_like(mass)
    for i, n in enumerate(lens.tolist()):
        for h in range(H):
            num = np.arange(n) + int(total[i]) - n
            if born is not None:
                num[:known[i]] = born[i, h, :known[i]]
            safe = (num < case["sinks"]) | (num >= total[i] - case["recent"])
            best = np.lexsort((np.arange(n), -mass[i, h, :n], ~safe))[:keep]
            late, free = np.sort(best[best >= keep]), np.setdiff1d(np.arange(min(n, keep)), best)
            place = np.arange(min(n, keep))
            place[free] = late   # the cell that each place holds now
            mass_out[i, h, :len(place)], born_out[i, h, :len(place)] = mass[i, h, place], num[place]
            row = lambda c: (table[i, c // ps].astype(np.int64) * H + h) * ps + c % ps  # noqa: E731
            for x in pools.values():
                x[row(free)] = x[row(late)]
    got = []
    for c in "kv":
        x = torch.from_numpy(pools[c + "c"]).view(s[c + "c"].shape).double()
        if case["fmt"] == "int8":
            x = x.view(*x.shape[:3], -1, BLOCK) * torch.from_numpy(pools[c + "s"]).view(*x.shape[:3], -1)[..., None].double()
        got.append(x)
    return (*got, mass_out, born_out.astype(np.int64), np.minimum(lens, keep))


# ---- what a pass cannot do without -------------------------------------------------------------------------------------

def work(case):
    size, kind, lens = {"f16": 2, "f32": 4}[case.get("act", "f32")], case["kind"], _lens(case)
    n = sum(lens)
    if kind == "conv":
        C, W = case["channels"], case["taps"]
        return {"bytes": 2 * n * C * size + 8 * case["seqs"] * C * (W - 1) + 4 * C * (W + 1), "flops": n * C * (2 * W + 5)}
    H, D, heads = case["kv"], case["dim"], case["heads"]
    row = 2 * D if case["fmt"] == "f16" else D + D // BLOCK * 2
    if kind == "axes":
        return {"bytes": n * (D * size * (2 * heads + 2 * H) + 2 * H * row + 8 * case["axes"]), "flops": n * 3 * case["rot"] * (heads + H)}
    if kind == "mass":
        R = case["rows"]
        seen = sum(max(0, t - R + 1 + r) for t in lens for r in range(R))
        return {"bytes": n * H * (row + 8) + case["seqs"] * R * heads * (D * size + 4), "flops": seen * 2 * heads * D}
    moved = 0.0
    for t in lens:
        if t > case["keep"]:
            free = max(0, case["keep"] - case["sinks"] - case["recent"])   # places that weights compete for
            rest = max(1, t - case["sinks"] - case["recent"])
            late = max(0, t - case["keep"] - case["recent"])
            moved += min(case["recent"], t - case["keep"]) + late * min(1.0, free / rest)
    return {"bytes": n * H * (8 + (4 if case["again"] else 0)) + sum(min(t, case["keep"]) for t in lens) * H * 4 + moved * H * 4 * row, "flops": n * H}
