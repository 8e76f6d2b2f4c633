"""Plain implementations in 64 bits of the operators of include/sc_ops.h, from their formulas, for the tests.

Independent of the library: numpy only, one loop per sequence, token by token."""
from __future__ import annotations

import numpy as np

BLOCK = 64


def rows_of(cu, n_seqs: int, tokens: int):
    """[(sequence, first row, rows)] of a packed batch (cu None: one row a sequence), rows past the batch left out."""
    if cu is None:
        return [(s, s, 1) for s in range(n_seqs)]
    return [(s, int(cu[s]), max(0, min(int(cu[s + 1]), tokens) - int(cu[s]))) for s in range(n_seqs)]


def pool_row(table, s: int, cell: int, h: int, H: int, ps: int, n_pages: int, table_ld: int) -> int:
    """The pool row of a cell, or -1 where it is not resident."""
    if not 0 <= cell < table_ld * ps:
        return -1
    page = s * table_ld + cell // ps if table is None else int(table[s][cell // ps])
    return (page * H + h) * ps + cell % ps if 0 <= page < n_pages else -1


def rotate(x: np.ndarray, pos: int, inv_freq, rot: int, pairs: str) -> np.ndarray:
    """The heads [.., D] of one token turned by its position."""
    y = np.array(x, np.float64)
    if rot:
        angle = float(pos) * np.asarray(inv_freq, np.float64)
        a, b = (np.s_[..., :rot // 2], np.s_[..., rot // 2:rot]) if pairs == "halves" else (np.s_[..., :rot:2], np.s_[..., 1:rot:2])
        xa, xb = np.array(y[a]), np.array(y[b])
        y[a], y[b] = xa * np.cos(angle) - xb * np.sin(angle), xa * np.sin(angle) + xb * np.cos(angle)
    return y


def rotate_axes(x: np.ndarray, pos, axis, inv_freq, rot: int, pairs: str) -> np.ndarray:
    """The heads [.., D] of one token, each pair turned by the token's position on the pair's axis."""
    y = np.array(x, np.float64)
    for i in range(rot // 2):
        angle = float(pos[axis[i]]) * float(inv_freq[i])
        a, b = (i, i + rot // 2) if pairs == "halves" else (2 * i, 2 * i + 1)
        xa, xb = np.array(y[..., a]), np.array(y[..., b])
        y[..., a], y[..., b] = xa * np.cos(angle) - xb * np.sin(angle), xa * np.sin(angle) + xb * np.cos(angle)
    return y


def attention(q, keys, values, scale: float):
    """One head's query over its cells [n][D]: (out, lse); nothing left gives zeros and -inf."""
    q, keys, values = (np.asarray(x, np.float64) for x in (q, keys, values))
    if not len(keys):
        return np.zeros_like(q), -np.inf
    s = scale * (keys @ q)
    top = s.max()
    if top == -np.inf:
        return np.zeros_like(q), -np.inf
    p = np.exp(s - top)
    return p @ values / p.sum(), top + np.log(p.sum())


def delta_rule(state, q, k, v, g, beta, scale: float, l2norm: bool, eps: float):
    """One head over its tokens: state [S][S] (key, value), q, k, v [T][S], g, beta [T]; (out [T][S], new state)."""
    M = np.array(state, np.float64)
    q, k, v, g, beta = (np.asarray(x, np.float64) for x in (q, k, v, g, beta))
    if l2norm:
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + eps) for x in (q, k))
    out = np.zeros((len(q), M.shape[1]))
    for t in range(len(q)):
        M *= np.exp(g[t])
        M += np.outer(k[t], beta[t] * (v[t] - M.T @ k[t]))
        out[t] = scale * (M.T @ q[t])
    return out, M


def short_conv(history, x, weight, bias, silu: bool):
    """One sequence: history [taps - 1][C] (the oldest row first), x [T][C], weight [C][taps], bias [C] or None;
    (out [T][C], new history)."""
    rows = np.concatenate([np.asarray(history, np.float64), np.asarray(x, np.float64)])
    w, W, out = np.asarray(weight, np.float64), np.shape(weight)[1], np.zeros(np.shape(x))
    for t in range(len(out)):
        y = np.zeros(w.shape[0]) if bias is None else np.array(bias, np.float64)
        for j in range(W):
            y += w[:, j] * rows[t + j]
        out[t] = y / (1 + np.exp(-y)) if silu else y
    return out, rows[len(rows) - (W - 1):]


def dequant(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """int8 rows [..][D] with f16 scales (bits) [..][D / 64]."""
    s = scales.view(np.float16).astype(np.float64)
    return codes.astype(np.float64) * np.repeat(s, BLOCK, -1)


def evict(mass, born, total: int, keep: int, sinks: int, recent: int):
    """One kv head of one sequence: the mass and the token's number of each cell; the cell that each place holds afterwards
    (places below min(len(mass), keep))."""
    n = len(mass)
    if n <= keep:
        return np.arange(n)
    weight = np.array([-np.inf if np.isnan(m) else m for m in np.asarray(mass, np.float64)])
    nan = np.isnan(np.asarray(mass, np.float64))
    always = np.array([b < sinks or b >= total - recent for b in born])
    order = sorted(range(n), key=lambda c: (not always[c], nan[c], -weight[c], c) if not always[c] else (False, False, 0.0, c))
    kept = set(order[:keep])
    place = np.arange(keep)
    free = [c for c in range(keep) if c not in kept]
    place[free] = sorted(c for c in kept if c >= keep)
    return place


def attention_mass(q, keys, scale: float, lse=None):
    """The weights that one head's query gives its cells [n][D]; `lse` the log of its sum of exponentials, or formed here."""
    if not len(keys):
        return np.zeros(0)
    s = scale * (np.asarray(keys, np.float64) @ np.asarray(q, np.float64))
    if lse is not None:
        return np.zeros(len(s)) if lse == -np.inf else np.exp(s - lse)
    if s.max() == -np.inf:
        return np.zeros(len(s))
    p = np.exp(s - s.max())
    return p / p.sum()
