"""Operators of a paged KV cache, as cases that can be timed and checked.

A case is a dict of plain values; ``op`` says which operator one pass calls:

* ``append``  the new tokens' rows of the joined q/k/v product: q and k rotated to their positions, k and v written into
  the pages their sequence's table names (``paged.append``);
* ``attend``  attention of the new tokens over the pages, themselves included (``paged.attention``): decode batches, chunks of
  prompts, and both in one call;
* ``handoff`` the live rows of every layer out of one pool into the packed handoff layout, and from there into the pages of
  another (``paged.pack_live`` + ``paged.unpack_live``).

A layer's pool is ``[n_pages, page_size, 2, kv_heads, head_dim]``; in memory a page holds its heads one after another, each
with its keys and then its values.  Position p of sequence b is row ``p % page_size`` of page ``tables[b, p // page_size]``.
Tokens lie sequence after sequence, sequence b's from ``cu[b]`` to ``cu[b + 1]``, the first of them at position
``starts[b]``.  The rotation turns pair j of the first ``2 * len(inv_freq)`` dims by position * inv_freq[j] and multiplies it by a scale;
pairs are (j, j + half) or, interleaved, (2j, 2j + 1).

Shapes are those of ``hexgen2_amd.workloads``, of ``perf/cases.py`` and ``perf/operators.py``, or generic.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}

# (q_heads, kv_heads, head_dim, dtype) of the workloads
_TINYLLAMA = (32, 4, 64, "float16")
_LLAMA2_7B = (32, 32, 128, "float16")
_LLAMA2_70B_TP8 = (8, 1, 128, "bfloat16")
_LLAMA3_8B = (32, 8, 128, "bfloat16")
_SMALL = (4, 2, 32, "float32")
_WIDE = (16, 2, 256, "bfloat16")
_GEOMETRIES = (_TINYLLAMA, _LLAMA2_7B, _LLAMA2_70B_TP8, _LLAMA3_8B)


def _kv(op, geometry, name=None, **sizes):
    q_heads, kv_heads, head_dim, dtype = geometry
    case = dict(op=op, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype)
    case.update(sizes)
    if name:
        case["name"] = name
    return case


# Sequences of an append or attend case: `chunks` of them bring chunk_lo to chunk_hi new tokens, `decodes` one token; each has
# lo to hi rows in the cache before.

def listed():
    return [
        # one decode step of the ragged Llama-3-8B batch: a token each, where the launch is the cost
        _kv("append", _LLAMA3_8B, "append-llama3-8b-decode", chunks=0, chunk_lo=0, chunk_hi=0, decodes=64, lo=128, hi=500,
            page=16, rotary=128, interleaved=False, scale=1.0, base=500000.0),
        # the second chunks of two prompts, of odd and different lengths
        _kv("append", _LLAMA2_7B, "append-llama2-7b-chunk", chunks=2, chunk_lo=433, chunk_hi=611, decodes=0, lo=512, hi=512,
            page=32, rotary=128, interleaved=False, scale=1.0, base=10000.0),
        # a long chunk far into a long context: half of each head rotated, interleaved, cosines and sines scaled
        _kv("append", _LLAMA3_8B, "append-llama3-8b-8192", chunks=1, chunk_lo=8192, chunk_hi=8192, decodes=0, lo=122893, hi=122893,
            page=64, rotary=64, interleaved=True, scale=1.1386, base=500000.0),
        # one request of the pilot's model decoding
        _kv("attend", _TINYLLAMA, "attend-tinyllama-577", chunks=0, chunk_lo=0, chunk_hi=0, decodes=1, lo=577, hi=577, page=16),
        # a ragged decode batch, one query head per KV head
        _kv("attend", _LLAMA2_7B, "attend-llama2-7b", chunks=0, chunk_lo=0, chunk_hi=0, decodes=8, lo=256, hi=2048, page=32),
        # the largest decode batch of the workloads
        _kv("attend", _LLAMA3_8B, "attend-llama3-8b", chunks=0, chunk_lo=0, chunk_hi=0, decodes=64, lo=128, hi=8192, page=16),
        # later chunks of two long prompts, on a tensor-parallel share of a large model
        _kv("attend", _LLAMA2_70B_TP8, "attend-llama2-70b-chunk", chunks=2, chunk_lo=509, chunk_hi=509, decodes=0, lo=3587,
            hi=3587, page=64),
        # a chunk of a long prompt after four others
        _kv("attend", _LLAMA3_8B, "attend-llama3-8b-chunk", chunks=1, chunk_lo=2048, chunk_hi=2048, decodes=0, lo=8192, hi=8192,
            page=64),
        # a serving step: two prompts' chunks beside the sequences that decode
        _kv("attend", _LLAMA2_70B_TP8, "attend-llama2-70b-mixed", chunks=2, chunk_lo=200, chunk_hi=700, decodes=46, lo=0, hi=4096,
            page=16),
        # a small model in 32 bits, prompts and single tokens
        _kv("attend", _SMALL, "attend-small-float32", chunks=3, chunk_lo=20, chunk_hi=90, decodes=5, lo=0, hi=300, page=16),
        # a request of the pilot's model from the prefill side's pages to the decode side's
        _kv("handoff", _TINYLLAMA, "handoff-tinyllama-512", layers=22, batch=1, lo=512, hi=512, page=16),
        # a ragged batch, every layer
        _kv("handoff", _LLAMA2_7B, "handoff-llama2-7b", layers=32, batch=8, lo=256, hi=2048, page=32),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "append", "attend", "attend", "attend", "attend", "handoff"))
    u = rng.random()
    geometry = _SMALL if u < 0.08 else _WIDE if u < 0.2 else rng.choice(_GEOMETRIES)
    if op != "handoff" and rng.random() < 0.2:
        geometry = (*geometry[:3], rng.choice(("float16", "bfloat16", "float32")))
    q_heads, kv_heads, head_dim, dtype = geometry
    page = rng.choice((16, 16, 32, 64, 128))
    row = 2 * kv_heads * head_dim
    if op == "append":
        width = q_heads * head_dim + row
        rows = _log_int(rng, 1, max(2, (48 << 20) // width // (2 if dtype == "float32" else 1)))
        chunks = 0 if rows < 8 or rng.random() < 0.4 else rng.randint(1, min(4, rows // 4))
        decodes = min(rows, rng.randint(1, 200)) if not chunks else rng.randint(0, 20)
        hi = _log_int(rng, 1, 100000)
        most = max(2, rows // max(1, chunks))
        rotary = rng.choice((head_dim, head_dim, head_dim // 2, head_dim // 4))
        return _kv(op, geometry, chunks=chunks, chunk_lo=max(1, most // 3) if chunks else 0, chunk_hi=most if chunks else 0,
                   decodes=decodes, lo=hi // rng.randint(1, 32), hi=hi, page=page, rotary=rotary,
                   interleaved=rng.random() < 0.4, scale=rng.choice((1.0, 1.0, 1.2079)),
                   base=rng.choice((10000.0, 500000.0, 1000000.0)))
    if op == "attend":
        hi = _log_int(rng, 1, 8192)
        lo = hi // rng.randint(1, 32)
        most = max(1, min(64, (1 << 28) // (row * (hi + 1)) // (2 if dtype == "float32" else 1)))
        if rng.random() < 0.55:
            return _kv(op, geometry, chunks=0, chunk_lo=0, chunk_hi=0, decodes=_log_int(rng, 1, most), lo=lo, hi=hi, page=page)
        # chunks, from a few guessed tokens to be verified to long ones, alone or beside decoding sequences
        few = rng.random() < 0.3
        chunk = rng.randint(2, 9) if few else _log_int(rng, 10, 700 if dtype != "float32" else 150)
        chunks = rng.randint(1, min(16, most)) if few else rng.randint(1, 2)
        decodes = rng.randint(1, min(40, most)) if rng.random() < 0.4 else 0
        while q_heads * (chunks + decodes) * chunk * (hi + chunk) > 1 << 30:
            hi, lo, decodes = hi // 2, lo // 2, decodes // 2
        return _kv(op, geometry, chunks=chunks, chunk_lo=max(1, chunk // 2), chunk_hi=chunk, decodes=decodes, lo=lo, hi=hi, page=page)
    layers = rng.randint(1, 40)
    hi = _log_int(rng, 1, 4096)
    batch = max(1, min(_log_int(rng, 1, 64), (1 << 30) // (layers * row * hi)))
    return _kv(op, geometry, layers=layers, batch=batch, lo=max(1, hi // rng.randint(1, 16)), hi=hi, page=page)


# ---------------------------------------------------------------- inputs ---


def _between(lo, hi, count, salt):
    """`count` lengths: part of the case, not of its inputs, so that every seed moves the same bytes."""
    g = torch.Generator().manual_seed(count * 100003 + hi * 7 + salt)
    return torch.randint(lo, hi + 1, (count,), generator=g).tolist()


def _sequences(case):
    """(new tokens, cached rows before them) of every sequence, chunks first."""
    new = _between(case["chunk_lo"], case["chunk_hi"], case["chunks"], 1) + [1] * case["decodes"]
    return new, _between(case["lo"], case["hi"], len(new), 2)


def _pool(pages, case, gen, device, layers=None):
    """A pool with rows of about unit size in every page, as earlier requests leave them."""
    h, d, p = case["kv_heads"], case["head_dim"], case["page"]
    shape = (pages, h, 2, p, d) if layers is None else (layers, pages, h, 2, p, d)
    pool = torch.empty(shape, dtype=_DTYPES[case["dtype"]], device=device)
    for part in pool.split(max(1, pages // 8)) if layers is None else pool:
        part.normal_(generator=gen)
    return pool.transpose(-2, -4)  # [.., pages, page, 2, heads, head_dim]


def _tables(lens, page, gen, device, first=0):
    """``(tables, pages of the pool)`` for sequences of these lengths, their pages in any order.  Pages before position
    `first` of a sequence are not needed by the call and all name page 0."""
    used = [(-(-n // page) - f // page) for n, f in zip(lens, first or [0] * len(lens))]
    total = sum(used) + 3
    order = torch.randperm(total - 1, generator=gen, device=device).to(torch.int32) + 1
    width = max(-(-n // page) for n in lens) + 2
    tables = torch.full((len(lens), width), -1, dtype=torch.int32, device=device)
    at = 0
    for b, (n, count) in enumerate(zip(lens, used)):
        last = -(-n // page)
        tables[b, :last - count] = 0
        tables[b, last - count:last] = order[at:at + count]
        at += count
    return tables, total


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype, page = _DTYPES[case["dtype"]], case["page"]
    hq, h, d = case["q_heads"], case["kv_heads"], case["head_dim"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device, dtype=dtype)

    state = dict(case=case)
    if case["op"] == "handoff":
        lens = _between(case["lo"], case["hi"], case["batch"], 2)
        state["lens"] = lens
        for side in ("source", "target"):
            state[side + "_tables"], pages = _tables(lens, page, gen, device)
            state[side] = _pool(pages, case, gen, device, case["layers"])
        return state
    new, starts = _sequences(case)
    lens = [n + s for n, s in zip(new, starts)]
    state["starts"] = torch.tensor(starts, dtype=torch.int32, device=device)
    state["cu"] = torch.tensor([0] + new, device=device).cumsum(0).to(torch.int32) if case["chunks"] else None
    state["max_tokens"], state["max_seqlen"] = max(new), max(lens)
    state["tables"], pages = _tables(lens, page, gen, device, starts if case["op"] == "append" else None)
    state["pages"] = _pool(pages, case, gen, device)
    if case["op"] == "append":
        state["qkv"] = normal(sum(new), (hq + 2 * h) * d)
        r = case["rotary"]
        state["inv_freq"] = 1.0 / case["base"] ** (torch.arange(0, r, 2, device=device, dtype=torch.float32) / r)
    else:
        state["q"] = normal(sum(new), hq, d).mul_(4)  # a softmax neither flat nor one-hot
    return state


# ----------------------------------------------------------- plain forms ---


def _places(state):
    """(sequence, position) of every token."""
    starts, tokens = state["starts"].long(), (state["qkv"] if "qkv" in state else state["q"]).shape[0]
    t = torch.arange(tokens, device=starts.device)
    if state["cu"] is None:
        return t, starts
    cu = state["cu"].long()
    seq = torch.searchsorted(cu[1:], t, right=True)
    return seq, starts[seq] + t - cu[seq]


def _rotate(x, cos, sin, interleaved):
    """Rotated heads ``x [tokens, heads, head_dim]`` by ``cos``, ``sin [tokens, 1, pairs]``."""
    r = 2 * cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., r:]), dim=-1)


def _plain_append(state):
    case, qkv, pages = state["case"], state["qkv"], state["pages"]
    hq, h, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    seq, pos = _places(state)
    angle = pos.double()[:, None, None] * state["inv_freq"].double()  # 32 bits lose the angles of far positions
    cos, sin = (angle.cos() * case["scale"]).float(), (angle.sin() * case["scale"]).float()
    x = qkv.float().view(-1, hq + 2 * h, d)
    turned = _rotate(x[:, :hq + h], cos, sin, case["interleaved"])
    at = state["tables"][seq, pos // page].long(), pos % page
    pages[at[0], at[1], 0] = turned[:, hq:].to(qkv.dtype)
    pages[at[0], at[1], 1] = qkv.view(-1, hq + 2 * h, d)[:, hq + h:]
    return dict(q=turned[:, :hq].to(qkv.dtype), pages=pages)


def _plain_attend(state):
    case, q, pages, tables = state["case"], state["q"], state["pages"], state["tables"]
    hq, h, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    g, b, longest, most = hq // h, tables.shape[0], state["max_seqlen"], state["max_tokens"]
    count = -(-longest // page)
    kv = pages[tables[:, :count].long()].float().flatten(1, 2)[:, :longest]  # [b, s, 2, h, d]
    k = kv[:, :, 0].permute(0, 2, 3, 1).contiguous()  # [b, h, d, s]
    v = kv[:, :, 1].permute(0, 2, 1, 3).contiguous()  # [b, h, s, d]
    seq, pos = _places(state)
    nth = pos - state["starts"].long()[seq]
    rows = torch.zeros((b, most, hq, d), device=q.device)
    rows[seq, nth] = q.float()
    rows = rows.view(b, most, h, g, d).permute(0, 2, 1, 3, 4).reshape(b, h, most * g, d)
    scores = torch.matmul(rows, k).mul_(d ** -0.5).view(b, h, most, g, longest)
    seen = state["starts"].long()[:, None] + 1 + torch.arange(most, device=q.device)  # token i sees the keys up to itself
    hidden = torch.arange(longest, device=q.device) >= seen[:, None, :, None, None]
    scores.masked_fill_(hidden, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(b, h, most * g, longest)
    out = torch.matmul(p, v).view(b, h, most, g, d).permute(0, 2, 1, 3, 4).reshape(b, most, hq, d)
    return out[seq, nth].to(q.dtype)


def _plain_handoff(state):
    case, source, target = state["case"], state["source"], state["target"]
    page, lens, device = case["page"], state["lens"], source.device
    seq = torch.repeat_interleave(torch.arange(len(lens), device=device), torch.tensor(lens, device=device))
    starts = torch.tensor([0] + lens[:-1], device=device).cumsum(0)
    pos = torch.arange(sum(lens), device=device) - starts[seq]
    packed = source[:, state["source_tables"][seq, pos // page].long(), pos % page]
    target[:, state["target_tables"][seq, pos // page].long(), pos % page] = packed
    return dict(packed=packed, pages=target)


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "handoff": _plain_handoff}[op](state)
    from hexgen2_amd import paged

    if op == "append":
        q = paged.append(state["qkv"], state["pages"], state["tables"], state["starts"], cu_tokens=state["cu"],
                         q_heads=case["q_heads"], inv_freq=state["inv_freq"], interleaved=case["interleaved"],
                         rotary_scale=case["scale"])
        return dict(q=q, pages=state["pages"])
    if op == "attend":
        return paged.attention(state["q"], state["pages"], state["tables"], state["starts"], cu_tokens=state["cu"],
                               max_tokens=state["max_tokens"], max_seqlen=state["max_seqlen"])
    packed = paged.pack_live(state["source"], state["source_tables"], state["lens"])
    paged.unpack_live(packed, state["target"], state["target_tables"], state["lens"])
    return dict(packed=packed, pages=state["target"])


# ------------------------------------------------------------------ work ---


def work(case):
    elem = 4 if case["dtype"] == "float32" else 2
    hq, h, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    row = 2 * h * d * elem
    if case["op"] == "handoff":
        return dict(bytes=4.0 * case["layers"] * sum(_between(case["lo"], case["hi"], case["batch"], 2)) * row, flops=0)
    new, starts = _sequences(case)
    if case["op"] == "append":
        # every element read once and written once; per new token three operations an element that turns
        return dict(bytes=2.0 * sum(new) * (hq * d * elem + row), flops=3.0 * sum(new) * (hq + h) * case["rotary"])
    lens = [n + s for n, s in zip(new, starts)]
    keys = sum(n * s + n * (n + 1) // 2 for n, s in zip(new, starts))
    moved = sum(lens) * row + 2.0 * sum(new) * hq * d * elem + 4 * sum(-(-n // page) for n in lens)
    return dict(bytes=moved, flops=4.0 * hq * d * keys)


# ----------------------------------------------------- the same in 64 bits ---


def _exact_append(case, state):
    hq, h, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    new, starts = _sequences(case)
    pages, x = state["pages"].double(), state["qkv"].double().view(-1, hq + 2 * h, d)
    # pairs as complex numbers, turned by a product
    j = torch.arange(case["rotary"] // 2, device=x.device)
    first, second = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + case["rotary"] // 2)
    q, at = torch.empty_like(x[:, :hq]), 0
    for b, (n, start) in enumerate(zip(new, starts)):
        pos = torch.arange(start, start + n, device=x.device, dtype=torch.float64)
        turn = torch.polar(torch.full((), case["scale"], dtype=torch.float64, device=x.device).expand(n, j.numel()),
                           torch.outer(pos, state["inv_freq"].double()))
        rows = x[at:at + n].clone()
        z = torch.complex(rows[:, :hq + h, first], rows[:, :hq + h, second]) * turn[:, None]
        rows[:, :hq + h, first], rows[:, :hq + h, second] = z.real, z.imag
        q[at:at + n] = rows[:, :hq]
        places = torch.arange(start, start + n, device=x.device)
        where = state["tables"][b].long()[places // page], places % page
        pages[where[0], where[1]] = rows[:, hq:].view(n, 2, h, d)
        at += n
    return dict(q=q, pages=pages)


def _exact_attend(case, state):
    q, page, h, d = state["q"], case["page"], case["kv_heads"], case["head_dim"]
    g, at, outs = case["q_heads"] // h, 0, []
    for b, (n, start) in enumerate(zip(*_sequences(case))):
        total = n + start
        kv = state["pages"][state["tables"][b, :-(-total // page)].long()].flatten(0, 1)[:total].double()
        limit = start + 1 + torch.arange(n, device=q.device).repeat_interleave(g)
        hidden = torch.arange(total, device=q.device)[None, :] >= limit[:, None]
        heads = []
        for i in range(h):
            rows = q[at:at + n, i * g:(i + 1) * g].double().reshape(n * g, d)
            scores = (rows @ kv[:, 0, i].t().contiguous()) * d ** -0.5
            p = torch.softmax(scores.masked_fill(hidden, -math.inf), dim=-1)
            heads.append((p @ kv[:, 1, i].contiguous()).view(n, g, d))
        outs.append(torch.cat(heads, dim=1))
        at += n
    return torch.cat(outs)


def exact(case, seed):
    if case["op"] == "handoff":
        return None  # nothing is computed: the rows come out as they went in
    state = prepare(case, seed)
    return _exact_append(case, state) if case["op"] == "append" else _exact_attend(case, state)
