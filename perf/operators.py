"""Operators of decoding in four bits and of scoring its answers, as cases that can be timed and checked.

A case is a dict of plain values; ``op`` says which operator one pass calls:

* ``store``   K/V rows into a 4-bit cache and back out of it (``fp4.store_kv`` + ``fp4.load_kv``): a prompt's rows, or
  one new row per sequence at per-sample positions;
* ``attend``  attention over a 4-bit cache (``fp4.decode_attention``): a decode step that appends each sequence's new row
  (with the stored rows read back), or several query rows per sequence over what is cached;
* ``linear``  activations of 16 or 32 bits times a 4-bit matrix (``fp4.linear``);
* ``logprobs``  log-probabilities of given tokens, the entropy and the top alternatives of each row of logits
  (``logprobs.token_logprobs``).

The 4-bit format: blocks of 32 consecutive elements share a power of two, 2^(b - 127) for the block's byte b, and an
element is sign, two exponent bits and one fraction bit: 0, 0.5, 1, 1.5, 2, 3, 4 or 6 times it; the lower half of a byte
is the element before the upper half's.  The power of a block is the smallest that leaves no element above 6; elements
go to the nearest value, halfway to the even code.  A cache is ``[batch, capacity, row]`` bytes, a row one position's
``[2][kv_heads][head_dim / 2]`` elements followed by their ``[2][kv_heads][head_dim / 32]`` powers, filled up to a
multiple of 16 bytes; a matrix ``[n, k / 2]`` elements and ``[n, k / 32]`` powers.

Shapes are those of ``hexgen2_amd.workloads`` and of ``perf/cases.py``, or generic.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

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


def listed():
    return [
        # one decode step's rows of the ragged Llama-3-8B batch: a row each, where the launch is the cost
        _kv("store", _LLAMA3_8B, "store-llama3-8b-append", batch=64, rows=1, capacity=512, ragged=True),
        # the second chunk of two prompts of odd length
        _kv("store", _LLAMA2_7B, "store-llama2-7b-chunk", batch=2, rows=611, capacity=1200, ragged=False),
        # the longest prompt of the Llama-3-8B workload
        _kv("store", _LLAMA3_8B, "store-llama3-8b-8192", batch=1, rows=8192, capacity=8192, ragged=False),
        # one request of the pilot's model decoding
        _kv("attend", _TINYLLAMA, "attend-tinyllama-577", batch=1, q_len=1, lo=577, hi=577, capacity=2048, append=True),
        # a ragged decode batch, one query head per KV head
        _kv("attend", _LLAMA2_7B, "attend-llama2-7b", batch=8, q_len=1, lo=256, hi=2048, capacity=4096, append=True),
        # the largest decode batch of the workloads
        _kv("attend", _LLAMA3_8B, "attend-llama3-8b", batch=64, q_len=1, lo=128, hi=8192, capacity=8448, append=True),
        # a later chunk of two long prompts, on a tensor-parallel share of a large model
        _kv("attend", _LLAMA2_70B_TP8, "attend-llama2-70b-chunk", batch=2, q_len=509, lo=4096, hi=4096, capacity=4128,
            append=False),
        # the joined q/k/v product of one decoding token
        dict(op="linear", rows=1, n=2560, k=2048, dtype="float16", name="linear-qkv-1"),
        # the joined gate/up product of a decode batch
        dict(op="linear", rows=64, n=22528, k=4096, dtype="bfloat16", name="linear-gate-up-64"),
        # the down product of a prompt of odd length
        dict(op="linear", rows=611, n=4096, k=11264, dtype="float16", name="linear-down-611"),
        # one decoded token's alternatives
        dict(op="logprobs", rows=1, vocab=32000, top=5, dtype="float16", masked=False, name="logprobs-step"),
        # every position of a long prompt scored, some of the vocabulary ruled out
        dict(op="logprobs", rows=8191, vocab=32000, top=20, dtype="bfloat16", masked=True, name="logprobs-prompt"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("store", "store", "attend", "attend", "attend", "linear", "linear", "logprobs", "logprobs"))
    if op in ("store", "attend"):
        u = rng.random()
        geometry = _SMALL if u < 0.08 else _WIDE if u < 0.2 else rng.choice(_GEOMETRIES)
        row = 2 * geometry[1] * geometry[2]
        if rng.random() < 0.25:
            geometry = (*geometry[:3], rng.choice(("float16", "bfloat16", "float32")))
    if op == "store":
        if rng.random() < 0.4:
            capacity = _log_int(rng, 2, 2048)
            return _kv(op, geometry, batch=_log_int(rng, 1, 200), rows=1, capacity=capacity, ragged=True)
        most = 1 << (23 if geometry[3] == "float32" else 24)
        rows = _log_int(rng, 2, max(2, min(8192, most // row)))
        batch = rng.randint(1, max(1, min(16, most // (row * rows))))
        return _kv(op, geometry, batch=batch, rows=rows, capacity=rows + rng.randint(0, 600), ragged=False)
    if op == "attend":
        hi = _log_int(rng, 1, 8192)
        lo = max(1, hi // rng.randint(1, 32))
        if rng.random() < 0.75:
            most = max(1, min(64, (1 << 29) // (row * (hi + 1))))
            return _kv(op, geometry, batch=_log_int(rng, 1, most), q_len=1, lo=lo, hi=hi,
                       capacity=hi + rng.randint(1, 600), append=rng.random() < 0.7)
        # a few query rows (guesses to be verified), or a chunk of a prompt
        q_len = rng.randint(2, 9) if rng.random() < 0.5 else _log_int(rng, 10, 700)
        hi = max(hi, q_len) if geometry[3] != "float32" else min(max(hi, q_len), 1500)
        q_len = min(q_len, hi)
        return _kv(op, geometry, batch=rng.randint(1, 2), q_len=q_len, lo=max(q_len, lo), hi=max(q_len, hi),
                   capacity=hi + rng.randint(1, 600), append=False)
    if op == "linear":
        k = 32 * _log_int(rng, 4, 350)
        n = _log_int(rng, 16, 22528)
        rows = _log_int(rng, 1, 600)
        while rows * n * k > 64 * 22528 * 4096 * 4:
            rows = max(1, rows // 2)
        return dict(op=op, rows=rows, n=n, k=k, dtype=rng.choice(("float16", "bfloat16", "bfloat16", "float32")))
    vocab = _log_int(rng, 300, 160000)
    rows = _log_int(rng, 1, max(1, min(8191, 8191 * 32000 // vocab)))
    dtype = rng.choice(("float16", "bfloat16", "float32"))
    if dtype == "float32":
        rows = max(1, rows // 2)
    return dict(op=op, rows=rows, vocab=vocab, top=rng.choice((0, 1, 5, 20, 32)), dtype=dtype, masked=rng.random() < 0.3)


# ---------------------------------------------------------------- inputs ---


def _lens(case):
    """The batch's cached lengths: part of the case, not of its inputs, so that every seed moves the same bytes."""
    if case["lo"] == case["hi"]:
        return [case["hi"]] * case["batch"]
    g = torch.Generator().manual_seed(case["batch"] * 100003 + case["hi"])
    return torch.randint(case["lo"], case["hi"] + 1, (case["batch"],), generator=g).tolist()


def _row_bytes(kv_heads, head_dim):
    return -(-2 * kv_heads * (head_dim // 2 + head_dim // 32) // 16) * 16


def _random_cache(case, gen, device):
    """A cache of random elements, with powers such that the values are of about unit size (outlying ones up to 16
    times that) and, as in a cache of earlier requests, in every row up to the capacity."""
    b, cap, h, d = case["batch"], case["capacity"], case["kv_heads"], case["head_dim"]
    codes, powers = h * d, 2 * h * d // 32
    cache = torch.zeros((b, cap, _row_bytes(h, d)), dtype=torch.uint8, device=device)
    for i in range(b):
        cache[i, :, :codes] = torch.randint(0, 256, (cap, codes), generator=gen, device=device, dtype=torch.uint8)
        shift = torch.randint(0, 40, (cap, powers), generator=gen, device=device)
        cache[i, :, codes:codes + powers] = (124 + (shift > 20).int() + (shift > 36).int() + (shift > 38).int()
                                             + (shift < 4).int() * -2).to(torch.uint8)
    return cache


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device, dtype=dtype)

    state = dict(case=case)
    op = case["op"]
    if op == "store":
        b, s, h, d = case["batch"], case["rows"], case["kv_heads"], case["head_dim"]
        state["kv"] = normal(b, s, 2, h, d)
        state["kv"][:, :, 0, :, :: 16] *= 8  # a few channels of the keys are far larger than the others
        state["cache"] = torch.zeros((b, case["capacity"], _row_bytes(h, d)), dtype=torch.uint8, device=device)
        last = case["capacity"] - s
        state["positions"] = torch.randint(0, last + 1, (b,), generator=gen, device=device, dtype=torch.int32) \
            if case["ragged"] else None
        state["bias"] = 0 if case["ragged"] else last // 2
    elif op == "attend":
        b, h, d = case["batch"], case["kv_heads"], case["head_dim"]
        state["cache"] = _random_cache(case, gen, device)
        state["q"] = normal(b, case["q_len"], case["q_heads"], d).mul_(4)  # a softmax neither flat nor one-hot
        state["kv_new"] = normal(b, 1, 2, h, d) if case["append"] else None
        state["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device=device)
    elif op == "linear":
        n, k = case["n"], case["k"]
        state["x"] = normal(case["rows"], k)
        state["codes"] = torch.randint(0, 256, (n, k // 2), generator=gen, device=device, dtype=torch.uint8)
        # weights of about 1 / sqrt(k), the power a block of them needs one of three
        low = 125 - round(math.log2(k) / 2)
        state["powers"] = torch.randint(low - 1, low + 2, (n, k // 32), generator=gen, device=device).to(torch.uint8)
    else:
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.randn((rows, vocab), generator=gen, device=device, dtype=dtype)
        # from rows that are nearly sure of a token to rows that know little
        state["logits"] = logits.mul_(torch.linspace(0.5, 4.0, rows, device=device)[:, None].to(dtype))
        if case["masked"]:
            first = torch.randint(0, vocab, (1,), generator=gen, device=device)
            out = (torch.arange(vocab, device=device) + first) % vocab < vocab // 3
            logits.masked_fill_(out[None, :], -math.inf)
        state["tokens"] = torch.randint(0, vocab, (rows,), generator=gen, device=device)
    return state


# ----------------------------------------------------------- plain forms ---


def _quantized(x):
    """``(elements, powers)`` of float32 blocks ``x [..., 32]``: their values over the power, and its exponent."""
    fraction, exponent = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = torch.where(fraction <= 0.75, exponent - 3, exponent - 2).clamp(-125, 126)
    y = x * _power(-e)
    size = y.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    return torch.round(y / step) * step, e


def _power(e):
    """2^e in float32 for whole numbers e in [-126, 127]."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _plain_encode(kv):
    """Cache rows ``[b, s, row]`` of ``kv [b, s, 2, heads, head_dim]``."""
    b, s, _, h, d = kv.shape
    y, e = _quantized(kv.float().reshape(b, s, 2 * h * d // 32, 32))
    edges = torch.tensor(_VALUES, device=kv.device)
    code = torch.bucketize(y.abs(), edges).int() + 8 * torch.signbit(y).int()
    packed = (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8).reshape(b, s, -1)
    rows = torch.cat((packed, (e + 127).to(torch.uint8).reshape(b, s, -1)), dim=-1)
    return torch.nn.functional.pad(rows, (0, _row_bytes(h, d) - rows.shape[-1]))


def _plain_values(codes, powers):
    """Float32 values of elements ``codes [..., k / 2]`` and ``powers [..., k / 32]``."""
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=codes.device)
    halves = torch.stack((codes & 15, codes >> 4), dim=-1).int()
    values = table[halves].reshape(*powers.shape, 32) * _power(powers.int() - 127)[..., None]
    return values.flatten(-2)


def _plain_decode(rows, h, d):
    """``[b, s, 2, heads, head_dim]`` float32 values of cache rows ``[b, s, row]``."""
    codes, powers = h * d, 2 * h * d // 32
    values = _plain_values(rows[..., :codes], rows[..., codes:codes + powers])
    return values.view(*rows.shape[:2], 2, h, d)


def _plain_store(state):
    case, kv, cache = state["case"], state["kv"], state["cache"]
    b, s, h, d = case["batch"], case["rows"], case["kv_heads"], case["head_dim"]
    at = torch.full((b,), state["bias"], device=kv.device) if state["positions"] is None else state["positions"].long()
    rows = at[:, None] + torch.arange(s, device=kv.device)
    seq = torch.arange(b, device=kv.device)[:, None]
    cache[seq, rows] = _plain_encode(kv)
    return _plain_decode(cache[seq, rows], h, d).to(kv.dtype)


def _plain_attend(state):
    case, q, cache, lens = state["case"], state["q"], state["cache"], state["lens"].long()
    b, t, hq, d = q.shape
    h, longest = case["kv_heads"], max(_lens(case))
    new = None
    if case["append"]:
        seq = torch.arange(b, device=q.device)
        cache[seq, lens] = _plain_encode(state["kv_new"])[:, 0]
        new = _plain_decode(cache[seq, lens][:, None], h, d).to(q.dtype)
        lens, longest = lens + 1, longest + 1
    kv = _plain_decode(cache[:, :longest], h, d)
    k = kv[:, :, 0].permute(0, 2, 3, 1).contiguous()  # [b, h, d, s]
    v = kv[:, :, 1].permute(0, 2, 1, 3).contiguous()  # [b, h, s, d]
    g = hq // h
    rows = q.float().view(b, t, h, g, d).permute(0, 2, 1, 3, 4).reshape(b, h, t * g, d)
    scores = torch.matmul(rows, k).mul_(d ** -0.5).view(b, h, t, g, longest)
    seen = lens[:, None] - t + 1 + torch.arange(t, device=q.device)  # causal: the last query row sees every key
    hidden = torch.arange(longest, device=q.device) >= seen[:, None, :, None, None]
    scores.masked_fill_(hidden, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(b, h, t * g, longest)
    out = torch.matmul(p, v).view(b, h, t, g, d).permute(0, 2, 1, 3, 4).reshape(b, t, hq, d).to(q.dtype)
    return dict(out=out, new=new) if case["append"] else dict(out=out)


def _plain_linear(state):
    weight = _plain_values(state["codes"], state["powers"])
    return torch.matmul(state["x"].float(), weight.t()).to(state["x"].dtype)


def _plain_logprobs(state):
    case = state["case"]
    x = state["logits"].float()
    u = x - x.amax(-1, keepdim=True)
    w = torch.exp(u)
    total = w.sum(-1, keepdim=True)
    log_total = torch.log(total)
    entropy = log_total[:, 0] - torch.where(w > 0, u * w, 0.0).sum(-1) / total[:, 0]
    result = dict(logprob=(u.gather(1, state["tokens"][:, None]) - log_total)[:, 0], entropy=entropy)
    if case["top"]:
        ids = torch.argsort(u, dim=-1, descending=True, stable=True)[:, :case["top"]]
        result.update(top_ids=ids, top_logprobs=u.gather(1, ids) - log_total)
    return result


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"store": _plain_store, "attend": _plain_attend, "linear": _plain_linear,
                "logprobs": _plain_logprobs}[op](state)
    from hexgen2_amd import fp4, logprobs

    if op == "store":
        kv, at = state["kv"], dict(positions=state["positions"], position_bias=state["bias"])
        fp4.store_kv(state["cache"], kv, **at)
        return fp4.load_kv(state["cache"], case["rows"], case["kv_heads"], case["head_dim"], kv.dtype, **at)
    if op == "attend":
        longest, new = max(_lens(case)), state["kv_new"]
        out = fp4.decode_attention(state["q"], state["cache"], case["kv_heads"], seqlens=state["lens"],
                                   max_seqlen=longest + int(case["append"]), kv_new=new, causal=case["q_len"] > 1)
        if new is None:
            return dict(out=out)
        return dict(out=out, new=fp4.load_kv(state["cache"], 1, case["kv_heads"], case["head_dim"], out.dtype,
                                             positions=state["lens"]))
    if op == "linear":
        return fp4.linear(state["x"], fp4.Fp4Tensor(state["codes"], state["powers"]))
    scores = logprobs.token_logprobs(state["logits"], state["tokens"], top=case["top"])
    result = dict(logprob=scores.logprob, entropy=scores.entropy)
    if case["top"]:
        result.update(top_ids=scores.top_ids, top_logprobs=scores.top_logprobs)
    return result


# ------------------------------------------------------------------ work ---


def work(case):
    elem = 4 if case["dtype"] == "float32" else 2
    op = case["op"]
    if op == "store":
        values = case["batch"] * case["rows"] * 2 * case["kv_heads"] * case["head_dim"]
        # 16-bit rows in, 4-bit rows out; 4-bit rows in, 16-bit rows out
        return dict(bytes=values * 2 * (elem + 17 / 32), flops=0)
    if op == "attend":
        lens, t = _lens(case), case["q_len"]
        hq, h, d = case["q_heads"], case["kv_heads"], case["head_dim"]
        row = 2 * h * d * 17 / 32
        moved = sum(lens) * row + 2 * len(lens) * t * hq * d * elem
        if case["append"]:
            moved += len(lens) * (2 * h * d * elem + row + 2 * h * d * elem)
        keys = sum(t * n - t * (t - 1) // 2 for n in lens) + (len(lens) if case["append"] else 0)
        return dict(bytes=moved, flops=4.0 * hq * d * keys)
    if op == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        return dict(bytes=n * k * 17 / 32 + rows * (n + k) * elem, flops=2.0 * rows * n * k)
    rows = case["rows"]
    return dict(bytes=rows * (case["vocab"] * elem + 16 + 12 * case["top"]), flops=4.0 * rows * case["vocab"])


# ----------------------------------------------------- the same in 64 bits ---


def _exact_values(codes, powers):
    """Values in 64 bits from the fields of each element: sign, exponent, fraction."""
    bits = torch.empty((*codes.shape, 2), dtype=torch.int64, device=codes.device)
    bits[..., 0], bits[..., 1] = codes % 16, codes // 16
    sign, exponent, fraction = bits // 8, bits // 2 % 4, bits % 2
    size = torch.where(exponent == 0, 0.5 * fraction, (1 + 0.5 * fraction) * torch.pow(2.0, (exponent - 1).double()))
    scale = torch.exp2(powers.double() - 127)
    signed = torch.where(sign == 1, -size, size).view(*powers.shape, 32)
    return (signed * scale[..., None]).flatten(-2)


def _exact_rounded(x):
    """What 4-bit storage makes of ``x [..., k]``, in 64 bits: every block's nearest representable values."""
    blocks = x.double().unflatten(-1, (-1, 32))
    most = blocks.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(torch.clamp(most, min=2.0 ** -140) / 6)))
    # the logarithm may fall a power to either side where the block's largest is 6 times a power of two
    scale = torch.where(most > 6 * scale, 2 * scale, torch.where(most <= 3 * scale, scale / 2, scale))
    scale = scale.clamp(2.0 ** -125, 2.0 ** 126)
    size = blocks.abs() / scale
    low = torch.zeros_like(size)
    high = torch.full_like(size, 0.5)
    odd = torch.zeros_like(size, dtype=torch.bool)  # whether the lower neighbour has an odd code
    for i, v in enumerate(_VALUES[1:], start=1):
        above = size >= v
        low = torch.where(above, v, low)
        high = torch.where(above, _VALUES[min(i + 1, 7)], high)
        odd = torch.where(above, i % 2 == 1, odd)
    up = (size - low > high - size) | ((size - low == high - size) & odd)
    return (torch.copysign(torch.where(up, high, low), blocks) * scale).flatten(-2)


def _exact_attend(case, state):
    q, h, d, t = state["q"], case["kv_heads"], case["head_dim"], case["q_len"]
    g, codes, powers = case["q_heads"] // h, h * d, 2 * h * d // 32
    outs, new = [], None
    if case["append"]:
        new = _exact_rounded(state["kv_new"])
    for b, n in enumerate(_lens(case)):
        rows = state["cache"][b, :n]
        kv = _exact_values(rows[:, :codes], rows[:, codes:codes + powers]).view(n, 2, h, d)
        if new is not None:
            kv = torch.cat((kv, new[b].view(1, 2, h, d)))
        total = kv.shape[0]
        limit = total - t + 1 + torch.arange(t, device=q.device).repeat_interleave(g)
        hidden = torch.arange(total, device=q.device)[None, :] >= limit[:, None]
        heads = []
        for i in range(h):
            rows_q = q[b, :, i * g:(i + 1) * g].double().reshape(t * g, d)
            scores = (rows_q @ kv[:, 0, i].t().contiguous()) * d ** -0.5
            p = torch.softmax(scores.masked_fill(hidden, -math.inf), dim=-1)
            heads.append((p @ kv[:, 1, i].contiguous()).view(t, g, d))
        outs.append(torch.cat(heads, dim=1))
    result = dict(out=torch.stack(outs))
    if new is not None:
        result["new"] = new
    return result


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "store":
        return _exact_rounded(state["kv"])
    if op == "attend":
        return _exact_attend(case, state)
    if op == "linear":
        x, n = state["x"].double(), case["n"]
        out = torch.empty((case["rows"], n), dtype=torch.float64, device=x.device)
        for first in range(0, n, 4096):
            part = slice(first, min(n, first + 4096))
            out[:, part] = x @ _exact_values(state["codes"][part], state["powers"][part]).t().contiguous()
        return out
    logits, tokens, top = state["logits"], state["tokens"], case["top"]
    parts = []
    for first in range(0, case["rows"], 512):
        rows = slice(first, min(case["rows"], first + 512))
        logs = torch.log_softmax(logits[rows].double(), dim=-1)
        p = logs.exp()
        entropy = -torch.where(p > 0, p * logs, 0.0).sum(-1)
        parts.append((logs.gather(1, tokens[rows, None])[:, 0], entropy, torch.sort(logs, dim=-1, descending=True)[0][:, :top]))
    logprob, entropy, best = (torch.cat(x) for x in zip(*parts))
    result = dict(logprob=logprob, entropy=entropy)
    if top:
        result.update(top_ids=None, top_logprobs=best)
    return result
