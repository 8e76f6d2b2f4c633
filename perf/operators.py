"""The measured operators of a decode slot: what a serving engine calls between two hand-offs.

`append`  new tokens' keys and values written to a paged cache with the position rotation on the way, queries rotated too
`attn`    attention of one new token a sequence over its paged cache
`step`    the gated delta rule of one new token a sequence
`chunk`   the gated delta rule over the tokens of a prompt, or of many prompts' pieces
"""
import math
import random

import numpy as np
import torch

own = False

THETA = 1e7          # base of the rotation's frequencies
BLOCK = 64           # values that share a scale in an int8 cache
F = {"f16": torch.float16, "f32": torch.float32}
# attention heads, kv heads, head size and page size of the configurations: the full-depth one first
FULL = {"heads": 24, "kv": 2, "dim": 256, "page": 4}
# key heads, value heads and state size of the recurrent layers
GDN = {"kh": 16, "vh": 32, "size": 128}


def listed():
    return [
        # one conversation decodes: its new token's row in one layer, launch latency
        {"name": "append_1", "kind": "append", "fmt": "f16", "act": "f32", "seqs": 1, "most": 1, "rot": 64, "pairs": "halves",
         "pos": 4093, **FULL},
        # a batch of conversations decodes into int8 caches
        {"name": "append_61_int8", "kind": "append", "fmt": "int8", "act": "f16", "seqs": 61, "most": 1, "rot": 64,
         "pairs": "halves", "pos": 30011, **FULL},
        # the chunks of eight prompts, of ragged lengths up to 2048 tokens
        {"name": "append_8x2048", "kind": "append", "fmt": "f16", "act": "f32", "seqs": 8, "most": 2048, "rot": 256,
         "pairs": "neighbours", "pos": 6141, **FULL},
        # a short conversation's token
        {"name": "attn_1x1021", "kind": "attn", "fmt": "f16", "act": "f32", "seqs": 1, "most": 1021, "window": 0, **FULL},
        # one conversation at 128K: a long cache and few rows
        {"name": "attn_1x131072", "kind": "attn", "fmt": "f16", "act": "f16", "seqs": 1, "most": 131072, "window": 0, **FULL},
        # a batch at ordinary lengths over int8 caches
        {"name": "attn_32x8190_int8", "kind": "attn", "fmt": "int8", "act": "f16", "seqs": 32, "most": 8190, "window": 0, **FULL},
        # eight ragged conversations of 1K to 128K tokens
        {"name": "attn_8x131072_ragged", "kind": "attn", "fmt": "f16", "act": "f32", "seqs": 8, "most": 131072, "window": 0, **FULL},
        # one conversation's recurrent layer: latency
        {"name": "step_1", "kind": "step", "act": "f32", "seqs": 1, "layout": "slot", **GDN},
        # a batch's
        {"name": "step_64", "kind": "step", "act": "f16", "seqs": 64, "layout": "slot", **GDN},
        # the last tokens of a prompt whose beginning was cached
        {"name": "chunk_1x61", "kind": "chunk", "act": "f32", "seqs": 1, "most": 61, "layout": "slot", **GDN},
        # a prompt's chunk in one call, into the prefill layout that a carve reads
        {"name": "chunk_1x8192", "kind": "chunk", "act": "f16", "seqs": 1, "most": 8192, "layout": "prefill", **GDN},
        # pieces of many prompts, ragged
        {"name": "chunk_8x2048_f32", "kind": "chunk", "act": "f32", "seqs": 8, "most": 2048, "layout": "slot", **GDN},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["append", "attn", "attn", "step", "chunk", "chunk"])
    act = rng.choice(["f16", "f32"])
    kv = rng.choice([1, 2, 2, 4])
    heads = {"heads": kv * rng.choice([1, 4, 8, 12, 16]), "kv": kv, "dim": rng.choice([64, 128, 256]), "page": rng.choice([1, 4, 4, 8, 16])}
    size = rng.choice([64, 128, 128])
    gdn = dict(zip(("kh", "vh"), rng.choice([(16, 32), (16, 48), (4, 8), (8, 8)])), size=size, layout=rng.choice(["slot", "prefill"]))
    if kind == "append":
        seqs = _log(rng, 1, 64)
        most = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 8192 * 24 * 256 // (heads["heads"] * heads["dim"]) // seqs))
        return {"kind": kind, "fmt": rng.choice(["f16", "int8"]), "act": act, "seqs": seqs, "most": most,
                "rot": rng.choice([heads["dim"], heads["dim"] // 2, heads["dim"] // 4]), "pairs": rng.choice(["halves", "neighbours"]),
                "pos": _log(rng, 1, 65536) - 1, **heads}
    if kind == "attn":
        seqs = _log(rng, 1, 64)
        # at most the cells of the ragged batch of eight
        return {"kind": kind, "fmt": rng.choice(["f16", "int8"]), "act": act, "seqs": seqs, "most": _log(rng, 1, min(131072, 500000 // seqs)),
                "window": rng.choice([0, 0, 0, _log(rng, 16, 8192)]), **heads}
    if kind == "step":
        return {"kind": kind, "act": act, "seqs": _log(rng, 1, 64), **gdn}
    seqs = _log(rng, 1, 16)
    return {"kind": kind, "act": act, "seqs": seqs, "most": _log(rng, 2, 7000 // seqs), **gdn}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _lens(case):
    """A batch's lengths: ragged up to the most, the longest among them; one sequence has the most."""
    n, most = case["seqs"], case["most"]
    r = random.Random(n * 1000003 + most)
    return [most] + [max(1, int(most * (1 / 128 + 127 / 128 * r.random()))) for _ in range(n - 1)]


def _pages(case, cells):
    return -(-cells // case["page"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    n, act = case["seqs"], F[case["act"]]
    normal = lambda *shape, dtype=torch.float32, by=1.0: (torch.randn(shape, device="cuda", generator=g) * by).to(dtype)  # noqa: E731
    host = lambda x, dtype: torch.tensor(x, dtype=dtype, device="cuda")  # noqa: E731
    if case["kind"] in ("append", "attn"):
        H, D, ps, lens = case["kv"], case["dim"], case["page"], _lens(case)
        if case["kind"] == "append":
            # each sequence's new tokens begin at a position of its own; its older pages lie in no pool here
            pos = [case["pos"] + 131 * i % 977 for i in range(n)]
            spans = [(p // ps, _pages(case, p + t)) for p, t in zip(pos, lens)]
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
            s["kc"], s["vc"] = ((normal(*rows, D, dtype=torch.float16) if case["kind"] == "attn" else torch.zeros(*rows, D, dtype=torch.float16, device="cuda"))
                                for _ in range(2))
        else:
            codes = lambda: torch.randint(-127, 128, (*rows, D), dtype=torch.int8, device="cuda", generator=g)  # noqa: E731
            scales = lambda: (0.01 + 0.02 * torch.rand((*rows, D // BLOCK), device="cuda", generator=g)).half()  # noqa: E731
            s["kc"], s["vc"], s["ks"], s["vs"] = codes(), codes(), scales(), scales()
    if case["kind"] == "append":
        N = sum(lens)
        s["cu"] = host(np.cumsum([0, *lens]).tolist(), torch.int64)
        s["pos0"], s["tokens"] = host(pos, torch.int64), N
        s["inv_freq"] = (THETA ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])).float().cuda()
        s["q"], s["k"], s["v"] = normal(N, case["heads"], D, dtype=act), normal(N, H, D, dtype=act), normal(N, H, D, dtype=act)
        s["q_out"] = torch.empty_like(s["q"])
    elif case["kind"] == "attn":
        s["lens"] = host(lens, torch.int64)
        s["q"] = normal(n, case["heads"], D, dtype=act)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((n, case["heads"]), device="cuda")
    else:
        lens = _lens(case) if case["kind"] == "chunk" else [1] * n
        N, kh, vh, size = sum(lens), case["kh"], case["vh"], case["size"]
        s["cu"], s["tokens"], s["longest"] = host(np.cumsum([0, *lens]).tolist(), torch.int64), N, max(lens)
        s["q"], s["k"], s["v"] = normal(N, kh, size, dtype=act), normal(N, kh, size, dtype=act), normal(N, vh, size, dtype=act)
        # log decays of heads that forget within a few tokens and of heads that keep thousands
        s["g"] = -torch.exp(torch.empty((N, vh), device="cuda").uniform_(-8, 0.5, generator=g))
        s["beta"] = torch.sigmoid(normal(N, vh))
        shape = (n, size, vh, size) if case["layout"] == "slot" else (n, vh, size, size)
        s["state"] = normal(*shape, by=0.1)
        s["out"] = torch.empty_like(s["v"])
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
    if s["kind"] in ("append", "attn"):
        cache = sc_ops.kv_cache(s["kc"], s["vc"], s.get("ks"), s.get("vs"), n_pages=s["pages"], n_head_kv=s["kv"], head_dim=s["dim"],
                                page_size=s["page"], table=s["table"], table_ld=s["ld"])
        if s["kind"] == "append":
            return sc_ops.RopeAppend(cache, s["k"], s["v"], s["act"], n_seqs=s["seqs"], tokens=s["tokens"], cu=s["cu"], pos0=s["pos0"],
                                     inv_freq=s["inv_freq"], rot_dim=s["rot"], pairs=s["pairs"], q=s["q"], q_out=s["q_out"],
                                     n_head=s["heads"])
        return sc_ops.AttnDecode(cache, s["q"], s["out"], s["act"], n_seqs=s["seqs"], n_head=s["heads"], lens=s["lens"],
                                 max_len=s["most"], scale=s["dim"] ** -0.5, window=s["window"], lse=s["lse"])
    state = sc_ops.gdn_states(s["state"], n_seqs=s["seqs"], v_heads=s["vh"], state_size=s["size"], layout=s["layout"])
    make = sc_ops.GdnStep if s["kind"] == "step" else sc_ops.GdnChunk
    return make(state, s["q"], s["k"], s["v"], s["g"], s["beta"], s["out"], s["act"], k_heads=s["kh"], n_seqs=s["seqs"],
                tokens=s["tokens"], cu=s["cu"], scale=s["size"] ** -0.5, l2norm=True)


def run(s):
    if own:
        s["op"].launch()
    else:
        {"append": _append, "attn": _attn, "step": _step, "chunk": _chunk}[s["kind"]](s)
    if s["kind"] == "append":
        # an int8 cache comes back as the values that it stands for, in the type that the scales have
        worth = lambda c, x: c if x is None else c.view(*x.shape, BLOCK) * x[..., None]  # noqa: E731
        return s["q_out"], worth(s["kc"], s.get("ks")), worth(s["vc"], s.get("vs"))
    return (s["out"], s["lse"]) if s["kind"] == "attn" else (s["out"], s["state"])


# ---- plain forms ---------------------------------------------------------------------------------------------------------

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


def _places(s):
    """Each new token's position, page and place in the page."""
    at = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["cu"], at, right=True) - 1
    pos = s["pos0"][seq] + at - s["cu"][seq]
    return pos, s["table"][seq, pos // s["page"]].long(), pos % s["page"]


def _append(s):
    pos, page, off = _places(s)
    angle = (pos.double()[:, None] * s["inv_freq"])[:, None]   # a product in 32 bits would be off by thousandths at these positions
    cos, sin = angle.cos().float(), angle.sin().float()
    k = _turn(s["k"], cos, sin, s["rot"], s["pairs"])
    s["q_out"].copy_(_turn(s["q"], cos, sin, s["rot"], s["pairs"]))
    v = s["v"].float()
    if s["fmt"] == "f16":
        s["kc"][page, :, off], s["vc"][page, :, off] = k.half(), v.half()
    else:
        (s["kc"][page, :, off], s["ks"][page, :, off]), (s["vc"][page, :, off], s["vs"][page, :, off]) = _codes(k), _codes(v)


def _cells(s, name):
    """A cache as [sequences, kv heads, cells, values], with whatever the first page holds where a sequence has no page."""
    page = s["table"].clamp_min(0).long()
    x = s[name + "c"][page].float()
    if s["fmt"] == "int8":
        x = (x.unflatten(-1, (-1, BLOCK)) * s[name + "s"][page].float()[..., None]).flatten(-2)
    return x.transpose(1, 2).flatten(2, 3)


def _attn(s):
    n, H, G = s["seqs"], s["kv"], s["heads"] // s["kv"]
    k = _cells(s, "k")
    at, lens = torch.arange(k.shape[2], device="cuda"), s["lens"][:, None]
    seen = (at < lens) & (at >= (lens - s["window"] if s["window"] else 0))
    q = s["q"].float().view(n, H, G, s["dim"]) * s["dim"] ** -0.5
    score = (q @ k.transpose(2, 3).contiguous()).masked_fill(~seen[:, None, None], -math.inf)
    del k
    top = score.amax(-1, keepdim=True)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    s["out"].copy_(((p @ _cells(s, "v")) / total).view(n, H * G, s["dim"]))
    s["lse"].copy_((top + total.log()).view(n, H * G))


def _unit(x):
    return x * torch.rsqrt(x.square().sum(-1, keepdim=True) + 1e-6)


def _states(s):
    """The states as [sequences, heads, keys, values]."""
    return s["state"].transpose(1, 2) if s["layout"] == "slot" else s["state"]


def _inputs(s):
    """Queries, keys and values, each value head with its own, the first two of length one."""
    each = s["vh"] // s["kh"]
    q, k = (_unit(s[x].float()).repeat_interleave(each, 1) for x in "qk")
    return q * s["size"] ** -0.5, k, s["v"].float()


def _step(s):
    q, k, v = _inputs(s)
    S = _states(s) * s["g"].exp()[..., None, None]
    u = s["beta"][..., None] * (v - (k[..., None] * S).sum(-2))
    S = S + k[..., None] * u[..., None, :]
    _states(s).copy_(S)
    s["out"].copy_((q[..., None] * S).sum(-2))


def _chunk(s, C=64):
    n, long = s["seqs"], -(-s["longest"] // C) * C
    at = s["cu"][:-1, None] + torch.arange(long, device="cuda")
    real = at < s["cu"][1:, None]
    at = at.clamp_max(s["tokens"] - 1)

    def split(x):  # [tokens, heads, ...] as [sequences, heads, chunks, C, ...], zeros past a sequence's end
        x = (x[at] * real.view(n, long, *[1] * (x.dim() - 1))).transpose(1, 2)
        return x.reshape(n, x.shape[1], long // C, C, *x.shape[3:])

    q, k, v = (split(x) for x in _inputs(s))
    beta, G = split(s["beta"])[..., None], split(s["g"]).cumsum(-1)
    lower = torch.ones(C, C, dtype=torch.bool, device="cuda").tril()
    fade = (G[..., :, None] - G[..., None, :]).masked_fill(~lower, -math.inf).exp()
    A = (beta * (k @ k.transpose(-1, -2).contiguous()) * fade).masked_fill(torch.eye(C, dtype=torch.bool, device="cuda"), 0)
    T = torch.eye(C, device="cuda").expand_as(A).contiguous()
    for i in range(1, C):   # the inverse of 1 + A, row by row
        T[..., i, :i] = -(A[..., i, None, :i] @ T[..., :i, :i])[..., 0, :]
    U, W = T @ (beta * v), T @ (beta * G[..., None].exp() * k)
    P, q = (q @ k.transpose(-1, -2).contiguous()) * fade, q * G[..., None].exp()
    k = (k * (G[..., -1:] - G).exp()[..., None]).transpose(-1, -2).contiguous()
    S, end = _states(s).clone(), G[..., -1].exp()[..., None, None]
    out = []
    for c in range(long // C):   # the state from chunk to chunk
        u = U[:, :, c] - W[:, :, c] @ S
        out.append(q[:, :, c] @ S + P[:, :, c] @ u)
        S = end[:, :, c] * S + k[:, :, c] @ u
    _states(s).copy_(S)
    s["out"].copy_(torch.cat(out, 2).transpose(1, 2)[real])


# ---- 64 bits -------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _append_64, "attn": _attn_64}.get(case["kind"], _delta_64)(case, s)


def _append_64(case, s):
    cu, pos0, table, ps, R = s["cu"].tolist(), s["pos0"].tolist(), s["table"].cpu(), case["page"], case["rot"]
    pos = torch.cat([p + torch.arange(e - b) for p, b, e in zip(pos0, cu, cu[1:])])
    page = torch.cat([table[i, (p + torch.arange(e - b)) // ps] for i, (p, b, e) in enumerate(zip(pos0, cu, cu[1:]))]).long()
    turn = torch.polar(torch.ones((), dtype=torch.float64), pos.double()[:, None] * s["inv_freq"].double().cpu())[:, None]

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
        rows[page, :, pos % ps] = x
        found.append(rows)
    return found


def _attn_64(case, s):
    out, lse, G = [], [], case["heads"] // case["kv"]
    for i, n in enumerate(s["lens"].tolist()):
        cell = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device="cuda")
        page, off = s["table"][i, cell // case["page"]].long(), cell % case["page"]
        rows = []
        for c in "kv":
            x = s[c + "c"][page, :, off].double()   # [cells, kv heads, values]
            if case["fmt"] == "int8":
                x *= s[c + "s"][page, :, off].double().repeat_interleave(BLOCK, -1)
            rows.append(x.repeat_interleave(G, 1).transpose(0, 1) if x.numel() * G < 1 << 31 else None)
        if rows[0] is None or rows[1] is None:
            return None
        score = (rows[0] @ s["q"][i].double()[..., None])[..., 0] / math.sqrt(case["dim"])
        lse.append(score.logsumexp(-1))
        out.append((score.softmax(-1)[:, None] @ rows[1])[:, 0])
    return torch.stack(out), torch.stack(lse)


def _delta_64(case, s):
    d = torch.float64
    S = _states(s).double()
    unit = lambda x: x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
    each, out = case["vh"] // case["kh"], torch.zeros(s["out"].shape, dtype=d, device="cuda")
    q, k = (unit(s[x].double()).repeat_interleave(each, 1) for x in "qk")
    a, beta, v, last = s["g"].double().exp(), s["beta"].double(), s["v"].double(), s["tokens"] - 1
    for t in range(s["longest"]):   # token by token; a sequence that has ended keeps its state
        at = s["cu"][:-1] + t
        real = at < s["cu"][1:]
        at = at.clamp_max(last)
        kt = k[at]
        decayed = S * a[at][..., None, None]
        u = beta[at][..., None] * (v[at] - (kt[..., None, :] @ decayed)[..., 0, :])
        S = torch.where(real[:, None, None, None], decayed + kt[..., None] * u[..., None, :], S)
        o = (q[at][..., None, :] @ S)[..., 0, :] / math.sqrt(case["size"])
        out.index_add_(0, at, o * real[:, None, None])
    return out, S.transpose(1, 2) if case["layout"] == "slot" else S


# ---- what a pass cannot do without -------------------------------------------------------------------------------------

def work(case):
    size = {"f16": 2, "f32": 4}[case["act"]]
    if case["kind"] in ("append", "attn"):
        n, H, D, heads = sum(_lens(case)), case["kv"], case["dim"], case["heads"]
        row = 2 * D if case["fmt"] == "f16" else D + D // BLOCK * 2
    if case["kind"] == "append":
        return {"bytes": n * (D * size * (2 * heads + 2 * H) + 2 * H * row), "flops": n * 3 * case["rot"] * (heads + H)}
    if case["kind"] == "attn":
        n = sum(min(t, case["window"] or t) for t in _lens(case))
        return {"bytes": n * 2 * H * row + 2 * case["seqs"] * heads * D * size, "flops": n * 4 * heads * D}
    kh, vh, S = case["kh"], case["vh"], case["size"]
    n = case["seqs"] if case["kind"] == "step" else sum(_lens(case))
    return {"bytes": 8 * case["seqs"] * vh * S * S + n * (size * S * 2 * (kh + vh) + 8 * vh), "flops": n * vh * 7 * S * S}
