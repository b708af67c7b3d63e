"""Plain 64-bit restatement of the paged cache: rotation, append, attention and
the handoff, one token or row at a time (numpy)."""
from __future__ import annotations

import numpy as np


def rotate(x, position, inv_freq, interleaved=False, scale=1.0):
    """Heads ``x [..., head_dim]`` of one token turned at its position."""
    x = np.array(x, np.float64)
    f = np.asarray(inv_freq, np.float64)
    n = len(f)
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    c, s = np.cos(position * f) * scale, np.sin(position * f) * scale
    u, v = a * c - b * s, b * c + a * s
    if interleaved:
        x[..., 0:2 * n:2], x[..., 1:2 * n:2] = u, v
    else:
        x[..., :n], x[..., n:2 * n] = u, v
    return x


def tokens_of(starts, cu, tokens):
    """(token, sequence, position) of every token of a sequence in use."""
    n = len(starts)
    if cu is None:
        cu = [b * (tokens // n) for b in range(n + 1)]
    return [(t, b, int(starts[b]) + t - int(cu[b])) for b in range(n) for t in range(int(cu[b]), int(cu[b + 1])) if starts[b] >= 0]


def append(qkv, pages, tables, starts, cu, q_heads, inv_freq, interleaved=False, scale=1.0):
    """``(q, pages)`` after the append; rows of q that no sequence in use has are NaN."""
    pages = np.array(pages, np.float64)
    n_pages, size, _, heads, d = pages.shape
    x = np.asarray(qkv, np.float64).reshape(len(qkv), -1, d)
    q = np.full((len(x), q_heads, d), np.nan)
    for t, b, p in tokens_of(starts, cu, len(x)):
        turned = rotate(x[t, :q_heads + heads], p, inv_freq, interleaved, scale)
        q[t] = turned[:q_heads]
        if p // size < len(tables[b]) and 0 <= tables[b][p // size] < n_pages:
            pages[tables[b][p // size], p % size, 0] = turned[q_heads:]
            pages[tables[b][p // size], p % size, 1] = x[t, q_heads + heads:]
    return q, pages


def attend(q, pages, tables, starts, cu, causal=True, scale=None, max_seqlen=None):
    """``(out, weight, reach)``: attention of every token ``q [tokens, q_heads, d]`` (NaN for a
    token of no sequence), and what its error is measured by: the sum of
    p |v| of each output and, of each row, the most that sum_d |q_d k_d| comes to."""
    q, pages = np.asarray(q, np.float64), np.asarray(pages, np.float64)
    tokens, q_heads, d = q.shape
    n_pages, size, _, heads, _ = pages.shape
    scale = d ** -0.5 if scale is None else scale
    out, weight, reach = np.full(q.shape, np.nan), np.zeros(q.shape), np.zeros(q.shape[:2])
    n = len(starts)
    bounds = [b * (tokens // n) for b in range(n + 1)] if cu is None else cu
    for b in range(n):
        first, last = int(bounds[b]), int(bounds[b + 1])
        for t in range(first, last):
            total = 0 if starts[b] < 0 else int(starts[b]) + (t - first + 1 if causal else last - first)
            total = total if max_seqlen is None else min(total, max_seqlen)
            at = [p for p in range(total) if 0 <= tables[b][p // size] < n_pages]
            out[t] = 0
            if not at:
                continue
            rows = pages[[tables[b][p // size] for p in at], [p % size for p in at]]
            for h in range(q_heads):
                k, v = rows[:, 0, h * heads // q_heads], rows[:, 1, h * heads // q_heads]
                with np.errstate(all="ignore"):
                    s = k @ q[t, h] * scale
                    e = np.exp(s - s.max())
                    p = e / e.sum()
                    out[t, h], weight[t, h], reach[t, h] = p @ v, p @ np.abs(v), (np.abs(k) @ np.abs(q[t, h])).max()
    return out, weight, reach


def pack(pages, tables, lens):
    """``[sum(lens), 2, heads, d]`` of one layer."""
    pages = np.asarray(pages)
    size = pages.shape[1]
    rows = [pages[tables[b][p // size], p % size] for b, n in enumerate(lens) for p in range(n)]
    return np.stack(rows) if rows else np.zeros((0, *pages.shape[2:]), pages.dtype)


def unpack(packed, pages, tables, lens):
    pages, at = np.array(pages), 0
    for b, n in enumerate(lens):
        for p in range(n):
            pages[tables[b][p // pages.shape[1]], p % pages.shape[1]] = packed[at]
            at += 1
    return pages
