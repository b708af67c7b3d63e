"""Plain 64-bit restatement of the four-bit block format, of attention and
products over it, and of log-probabilities (numpy, one element or row at a time
where that is clearest)."""
from __future__ import annotations

import numpy as np

BLOCK = 32
VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def quantize(x):
    """(codes [..., k] one per element, powers [..., k / 32]) of float64 ``x``:
    the smallest power in [2^-125, 2^126] that leaves no element above 6 (1
    for a block of zeros), nearest elements, halfway to the even code; powers
    255 and codes 0 for a block that is not finite."""
    x = np.asarray(x, dtype=np.float64)
    blocks = x.reshape(*x.shape[:-1], -1, BLOCK)
    most = np.abs(blocks).max(-1)
    bad = ~np.isfinite(blocks).all(-1)
    _, e = np.frexp(np.where(bad, 1.0, most) / 6)  # most / 6 = f 2^e, f in [0.5, 1)
    e = np.where(most * 2.0 ** -(e - 1.0) <= 6, e - 1, e)  # f == 0.5
    e = np.clip(np.where(most == 0, 0, e), -125, 126)
    size = np.abs(np.where(bad[..., None], 0, blocks)) / 2.0 ** e[..., None]
    distance = np.abs(size[..., None] - VALUES)
    nearest = distance.argmin(-1)  # the lower of two
    upper = np.minimum(nearest + 1, 7)
    tie = (np.take_along_axis(distance, nearest[..., None], -1) ==
           np.take_along_axis(distance, upper[..., None], -1))[..., 0] & (upper != nearest)
    codes = np.where(tie & (nearest % 2 == 1), upper, nearest) + 8 * (np.signbit(blocks) & ~bad[..., None])
    return codes.reshape(x.shape), np.where(bad, 255, e + 127)


def values(codes, powers):
    """Float64 values of one-per-element codes and their powers."""
    codes = np.asarray(codes)
    v = np.where(codes & 8, -1.0, 1.0) * VALUES[codes & 7]
    scale = np.where(np.asarray(powers) == 255, np.nan, 2.0 ** (np.asarray(powers, dtype=np.float64) - 127))
    return (v.reshape(*codes.shape[:-1], -1, BLOCK) * scale[..., None]).reshape(codes.shape)


def rounded(x):
    """What four-bit storage makes of ``x``."""
    return values(*quantize(x))


def pack(codes):
    """Two codes a byte, the earlier in the lower half."""
    codes = np.asarray(codes)
    return (codes[..., 0::2] | codes[..., 1::2] << 4).astype(np.uint8)


def unpack(packed):
    packed = np.asarray(packed)
    return np.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], -1)


def rows(kv):
    """Cache rows [..., row bytes] of kv [..., 2, heads, head_dim]."""
    kv = np.asarray(kv, dtype=np.float64)
    heads, d = kv.shape[-2:]
    codes, powers = quantize(kv)
    lead = kv.shape[:-3]
    row = np.concatenate((pack(codes).reshape(*lead, -1), powers.astype(np.uint8).reshape(*lead, -1)), -1)
    return np.concatenate((row, np.zeros((*lead, -row.shape[-1] % 16), np.uint8)), -1)


def row_values(row, heads, d):
    """kv [..., 2, heads, d] of cache rows."""
    row = np.asarray(row)
    lead, n = row.shape[:-1], heads * d
    codes = unpack(row[..., :n]).reshape(*lead, 2, heads, d)
    return values(codes, row[..., n:n + 2 * heads * d // BLOCK].reshape(*lead, 2, heads, d // BLOCK))


def attend(q, kv, lens, causal=False, scale=None):
    """softmax(q k^T) v per row: q [B, T, Hq, D], kv [B, S, 2, Hkv, D], row b
    over lens[b] keys (fewer for earlier queries with ``causal``); a row
    without keys is zero."""
    q, kv = np.asarray(q, np.float64), np.asarray(kv, np.float64)
    b, t, hq, d = q.shape
    group = hq // kv.shape[3]
    scale = d ** -0.5 if scale is None else scale
    out = np.zeros_like(q)
    for i in range(b):
        for j in range(t):
            n = lens[i] - (t - 1 - j if causal else 0)
            if n <= 0:
                continue
            for h in range(hq):
                s = (kv[i, :n, 0, h // group] * q[i, j, h]).sum(-1) * scale
                p = np.exp(s - s.max())
                out[i, j, h] = (p[:, None] * kv[i, :n, 1, h // group]).sum(0) / p.sum()
    return out


def logprobs(logits, tokens, top):
    """(logprob, entropy, top ids, top log-probabilities) per row."""
    logits = np.asarray(logits, np.float64)
    rows, vocab = logits.shape
    lp, entropy = np.zeros(rows), np.zeros(rows)
    ids, best = np.zeros((rows, top), np.int64), np.zeros((rows, top))
    with np.errstate(all="ignore"):
        for r, x in enumerate(logits):
            m = np.nan if np.isnan(x).any() else x.max()
            if m == -np.inf:
                logs = np.full(vocab, -np.inf)
            else:
                logs = x - m - np.log(np.exp(x - m).sum())
                entropy[r] = -(np.exp(logs) * np.where(np.exp(logs) > 0, logs, 0)).sum() if not np.isnan(logs).any() else np.nan
            t = tokens[r]
            lp[r] = 0 if t < 0 else np.nan if t >= vocab else logs[t]
            order = np.argsort(-np.where(np.isnan(x), np.inf, x), kind="stable")
            order = np.concatenate((order[np.isnan(x[order])], order[~np.isnan(x[order])]))[:top]
            ids[r], best[r] = order, logs[order]
    return lp, entropy, ids, best
