"""Paged caches against the 64-bit oracle: every head size and type, lengths at
the borders of pages, steps and partitions, chunks beside single tokens, what
the device finds in its own memory, streams and graphs."""
import itertools

import numpy as np
import pytest
import torch

from hexgen2_amd import ops, paged
from oracle import paged_oracle as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
GEOMETRIES = [(8, 2, 64), (4, 4, 128), (8, 1, 128), (6, 2, 32), (2, 1, 256), (4, 2, 16)]  # (q heads, KV heads, head_dim)


def randn(shape, seed, dtype, device, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(dtype).to(device)


def wide(t):
    return t.detach().cpu().double().numpy()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def make_pool(geometry, page, count, seed, dtype, device, order="heads"):
    """A pool of random rows, in one of several orders of its memory."""
    _, heads, d = geometry
    shape = (count, page, 2, heads, d)
    if order == "heads":
        pool = paged.kv_pages(count, page, heads, d, dtype, device)
        assert pool.shape == shape
    elif order == "rows":
        pool = torch.empty(shape, dtype=dtype, device=device)
    else:  # K and V pools apart, rows with gaps
        pool = torch.empty((2, count, page, heads + 1, d), dtype=dtype, device=device)[:, :, :, 1:].permute(1, 2, 0, 3, 4)
    pool.copy_(randn(shape, seed, dtype, device))
    return pool


def make_tables(lens, page, seed, device, spare=2):
    """Tables of shuffled pages for sequences of these lengths, and the pool's size."""
    need = [paged.pages_for(n, page) for n in lens]
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(need) + spare, generator=g).tolist()
    width = max(need + [1]) + 1
    tables, at = [], 0
    for n in need:
        tables.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return int32(tables, device), len(order)


def cu_of(new, device):
    return int32(np.concatenate(([0], np.cumsum(new))).tolist(), device)


def inv_freq_of(dim, device, base=10000.0):
    return (1.0 / base ** (torch.arange(0, dim, 2, dtype=torch.float32) / dim)).to(device)


# ---------------------------------------------------------------- append ---


def check_append(device, dtype, geometry, new, starts, page, rotary, interleaved=False, scale=1.0, uniform=False, order="heads",
                 seed=0, extra=0, base=10000.0):
    hq, h, d = geometry
    lens = [max(s + n, 0) for s, n in zip(starts, new)]
    tables, count = make_tables(lens, page, seed, device)
    pool = make_pool(geometry, page, count, seed + 1, dtype, device, order)
    qkv = randn((sum(new) + extra, (hq + 2 * h) * d), seed + 2, dtype, device)
    f = inv_freq_of(rotary, device, base) if rotary else None
    cu = None if uniform else cu_of(new, device)
    before = pool.clone()
    out = torch.full((sum(new) + extra, hq, d), 7.0, dtype=dtype, device=device)
    got = paged.append(qkv, pool, tables, int32(starts, device), q_heads=hq, cu_tokens=cu, inv_freq=f,
                       interleaved=interleaved, rotary_scale=scale, out=out)
    assert got is out
    freq = np.zeros(0) if f is None else wide(f)
    q, pages = oracle.append(wide(qkv), wide(before), tables.tolist(), starts, None if uniform else cu.tolist(), hq, freq,
                             interleaved, scale)
    # sums of two products: the angle to 2^-23 of a radian, sine and cosine to two
    # steps of fp32 each, products and sum to half a step each, then the type's rounding
    most = float(np.abs(wide(qkv)).max()) * 2 * max(scale, 1.0)
    for have, want, old in ((wide(got), q, np.full(q.shape, 7.0)), (wide(pool), pages, wide(before))):
        want = np.where(np.isnan(want), old, want)
        tol = half_step(dtype) * np.abs(want) * 1.001 + most * 2.0 ** -21
        same = want == old
        assert (np.abs(have - want) <= np.where(same, 0, tol)).all()


@pytest.mark.parametrize("dtype,geometry", itertools.product(DTYPES, GEOMETRIES))
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_of_chunks(device, dtype, geometry, interleaved):
    d = geometry[2]
    check_append(device, dtype, geometry, [5, 1, 17, 33], [0, 31, 15, 127], 16, d, interleaved)
    check_append(device, dtype, geometry, [20, 3], [7, 64], 32, d // 2, interleaved, 1.25, order="rows")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rotary,interleaved", [(0, False), (0, True), (2, False), (2, True), (6, False), (6, True), (24, False),
                                                (24, True), (64, False)])
def test_append_turns_part_of_a_head(device, dtype, rotary, interleaved):
    check_append(device, dtype, (4, 2, 64), [3, 2], [9, 30], 16, rotary, interleaved, 0.75, order="apart")


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_of_single_tokens(device, dtype):
    # one a sequence, more than a wave's and a workgroup's worth of sequences
    for n in (1, 3, 64, 65, 300):
        starts = [(17 * i) % 50 for i in range(n)]
        check_append(device, dtype, (4, 2, 64), [1] * n, starts, 16, 64, uniform=True, seed=n)
        check_append(device, dtype, (4, 2, 64), [1] * n, starts, 16, 64, seed=n + 1)
    check_append(device, dtype, (4, 2, 64), [4] * 3, [0, 15, 40], 32, 64, uniform=True)


def test_append_of_many_tokens(device):
    check_append(device, torch.bfloat16, (8, 2, 64), [700, 0, 1, 311], [0, 5, 2000, 77], 64, 64)


@pytest.mark.parametrize("position", [100000, 1 << 20, (1 << 26) - 20])
def test_append_far_positions(device, position):
    """Angles of far positions: 32 bits would be off by position * 2^-24 of a radian."""
    hq, h, d, page = 2, 1, 32, 1 << 16
    width = paged.pages_for(position + 20, page)
    tables = torch.zeros((1, width), dtype=torch.int32, device=device)
    pool = torch.zeros((1, page, 2, h, d), dtype=torch.float32, device=device)
    qkv = randn((20, (hq + 2 * h) * d), 5, torch.float32, device)
    f = inv_freq_of(d, device)
    q = paged.append(qkv, pool, tables, int32([position], device), q_heads=hq, inv_freq=f)
    x = wide(qkv).reshape(20, -1, d)
    want = np.stack([oracle.rotate(x[i], position + i, wide(f)) for i in range(20)])
    tol = 2.0 ** -24 * np.abs(want) + 2 * np.abs(x).max() * 2.0 ** -21
    assert (np.abs(wide(q) - want[:, :hq]) <= tol[:, :hq]).all()
    rows = wide(pool)[0, [(position + i) % page for i in range(20)], 0]
    assert (np.abs(rows - want[:, hq:hq + h]) <= tol[:, hq:hq + h]).all()


@pytest.mark.parametrize("uniform", [False, True])
def test_append_leaves_what_is_not_in_use(device, uniform):
    check_append(device, torch.float16, (4, 2, 64), [2, 2, 2], [5, -1, 14], 16, 64, uniform=uniform)
    if not uniform:  # tokens behind the last sequence
        check_append(device, torch.float16, (4, 2, 64), [2, 0, 3], [5, 9, 14], 16, 64, extra=5)
    assert ops.device_status(device) & ops._lib.STATUS_ERRORS == 0


def test_append_skips_and_flags_pages_outside_the_pool(device):
    geometry, page = (4, 2, 64), 16
    pool = make_pool(geometry, page, 3, 1, torch.float16, device)
    qkv = randn((4, 8 * 64), 2, torch.float16, device)
    f = inv_freq_of(64, device)
    tables = int32([[0], [3], [-1], [1]], device)
    before, starts = pool.clone(), [3, 3, 3, 16]
    ops.device_status(device)
    q = paged.append(qkv, pool, tables, int32(starts, device), q_heads=4, inv_freq=f)
    assert ops.device_status(device) == ops._lib.STATUS_PAGE | ops._lib.STATUS_APPEND_SKIPPED
    changed = (pool != before).flatten(2).any(-1)
    assert changed.nonzero().tolist() == [[0, 3]]
    want, _ = oracle.append(wide(qkv), wide(before), tables.tolist(), starts, None, 4, wide(f))
    assert np.abs(wide(q) - want).max() < 1e-2  # q is turned all the same


def test_append_in_place_and_strided(device):
    hq, h, d = 4, 2, 64
    width = (hq + 2 * h) * d
    base = randn((9, width + 24), 3, torch.bfloat16, device)
    f, starts = inv_freq_of(d, device), int32([40], device)
    tables, count = make_tables([60], 16, 1, device)
    pools = [make_pool((hq, h, d), 16, count, 2, torch.bfloat16, device) for _ in range(4)]
    want = paged.append(base[:, :width].contiguous(), pools[0], tables, starts, q_heads=hq, inv_freq=f)
    rows = base[:, :width]
    assert torch.equal(paged.append(rows, pools[1], tables, starts, q_heads=hq, inv_freq=f), want)
    odd = torch.zeros((9, width + 25), dtype=torch.bfloat16, device=device)[:, 1:width + 1]  # not aligned to a vector
    odd.copy_(rows)
    assert torch.equal(paged.append(odd, pools[2], tables, starts, q_heads=hq, inv_freq=f), want)
    q = rows[:, :hq * d].unflatten(-1, (hq, d))
    assert paged.append(rows, pools[3], tables, starts, q_heads=hq, inv_freq=f, out=q) is q
    assert torch.equal(q, want)
    assert all(torch.equal(p, pools[0]) for p in pools[1:])


# ------------------------------------------------------------- attention ---


def tolerance(dtype, want, weight, reach, d, scale=None, keys=1):
    """What rounding allows: half a step of the output's type; of the sum of p |v|:
    16-bit probabilities of up to two terms (one in tiles of many rows: half a step of the type, in
    numerator and sum apart), sums of `keys` fp32 terms taken 32 at a time,
    and scores off by (d + 2) half steps of fp32 of sum |q k| (2 of them: p and its sum)."""
    scale = d ** -0.5 if scale is None else scale
    score = reach[..., None] * scale * (d + 4) * 2.0 ** -24
    term = 0 if dtype == torch.float32 else half_step(dtype)
    sums = (keys / 16 + 40) * 2.0 ** -24
    return half_step(dtype) * np.abs(want) * 1.01 + weight * (2 * score + term + 2 * sums) + 1e-30


def check_attend(device, dtype, geometry, new, starts, page, causal=True, uniform=False, order="heads", seed=0, extra=0, sharp=2.0,
                 partition=0, max_seqlen=None, scale=None, fill=None):
    hq, h, d = geometry
    lens = [max(s + n, 0) for s, n in zip(starts, new)]
    tables, count = make_tables(lens, page, seed, device)
    pool = make_pool(geometry, page, count, seed + 1, dtype, device, order)
    if fill is not None:  # what no sequence has yet
        live = torch.zeros(pool.shape[:2], dtype=torch.bool, device=device)
        for b, n in enumerate(lens):
            for p in range(n):
                live[tables[b, p // page].long(), p % page] = True
        pool.masked_fill_(~live[:, :, None, None, None], fill)
    q = randn((sum(new) + extra, hq, d), seed + 2, dtype, device, sharp)
    cu = None if uniform else cu_of(new, device)
    out = torch.full_like(q, 7.0)
    longest = max(lens + [0]) if max_seqlen is None else max_seqlen
    got = paged.attention(q, pool, tables, int32(starts, device), max_seqlen=longest, cu_tokens=cu,
                          max_tokens=max(new), causal=causal, out=out, partition=partition, softmax_scale=scale)
    assert got is out
    want, weight, reach = oracle.attend(wide(q), wide(pool), tables.tolist(), starts, None if uniform else cu.tolist(), causal,
                                        scale)
    idle = np.isnan(want).all(axis=(1, 2))
    assert (wide(got)[idle] == 7).all()
    want = np.where(idle[:, None, None], 7.0, want)
    off = np.abs(wide(got) - want)
    tol = tolerance(dtype, want, weight, reach, d, scale, max(lens + [1]))
    assert (off <= tol).all(), (float((off / tol).max()), np.argwhere(off > tol)[:4])


@pytest.mark.parametrize("dtype,geometry", itertools.product(DTYPES, GEOMETRIES))
def test_decode_rows(device, dtype, geometry):
    check_attend(device, dtype, geometry, [1] * 9, [0, 1, 14, 15, 16, 31, 32, 100, 255], 16, uniform=True)
    check_attend(device, dtype, geometry, [1, 1, 1], [640, 0, 333], 64, order="rows", seed=5)
    check_attend(device, dtype, geometry, [1, 1, 1], [640, 0, 333], 128, order="apart", seed=6, partition=64)


@pytest.mark.parametrize("dtype,geometry", itertools.product(DTYPES, GEOMETRIES))
@pytest.mark.parametrize("causal", [True, False])
def test_chunks(device, dtype, geometry, causal):
    check_attend(device, dtype, geometry, [3, 1, 40, 2], [0, 20, 5, 99], 16, causal)
    check_attend(device, dtype, geometry, [37, 5], [0, 300], 32, causal, order="rows", partition=64)
    check_attend(device, dtype, geometry, [8, 8], [33, 0], 16, causal, uniform=True, order="apart")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("geometry", [(4, 1, 64), (4, 2, 128), (3, 3, 64), (8, 1, 128)])
def test_long_chunks(device, dtype, geometry):
    """Chunks of more rows than a tile, over keys that end inside pages and tiles."""
    check_attend(device, dtype, geometry, [150, 1, 65], [0, 200, 77], 16)
    check_attend(device, dtype, geometry, [129, 130], [63, 321], 128, order="rows")
    check_attend(device, dtype, geometry, [140, 3, 1], [250, 130, 31], 32, partition=64)
    check_attend(device, dtype, geometry, [140], [250], 32, causal=False, partition=64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1] * 4, [1, 30, 1, 90]])
def test_rows_behind_the_last_length_do_not_matter(device, dtype, new):
    """Rows of a page that were never written hold anything."""
    for fill in (float("nan"), float("inf"), -float("inf")):
        check_attend(device, dtype, (4, 2, 64), new, [0, 17, 40, 70], 32, fill=fill)


@pytest.mark.parametrize("uniform", [False, True])
def test_sequences_not_in_use(device, uniform):
    check_attend(device, torch.bfloat16, (4, 2, 64), [2, 2, 2], [5, -1, 30], 16, uniform=uniform)
    check_attend(device, torch.bfloat16, (4, 2, 64), [2, 2, 2], [5, -7, 30], 16, uniform=uniform, causal=False)
    if not uniform:
        check_attend(device, torch.float16, (4, 2, 64), [2, 0, 60], [5, 9, 30], 16, extra=7)
    assert ops.device_status(device) & ops._lib.STATUS_ERRORS == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("new", [6, 100])
def test_values_that_are_not_finite_reach_only_the_rows_that_attend_them(device, dtype, value, new):
    hq, h, d, page = 4, 2, 64, 16
    start, bad = 45, 45 + new // 2  # a value among the chunk's own keys
    tables, count = make_tables([start + new], page, 1, device)
    for where in (0, 1):  # a key's element, a value's
        pool = make_pool((hq, h, d), page, count, 2, dtype, device)
        q = randn((new, hq, d), 3, dtype, device)
        clean = paged.attention(q, pool, tables, int32([start], device), max_seqlen=start + new)
        pool[tables[0, bad // page].long(), bad % page, where, 1, 5] = value
        got = paged.attention(q, pool, tables, int32([start], device), max_seqlen=start + new)
        sees = torch.zeros((new, hq), dtype=torch.bool)
        sees[new // 2:, 2:] = True
        if where == 1 or value != value:
            want = torch.zeros((new, hq, d), dtype=torch.bool)
            want[sees] = torch.tensor([e == 5 or where == 0 for e in range(d)])
            assert torch.equal(~torch.isfinite(got.cpu()), want)
        # (a row that is taken key by key rounds apart from the tile it lies in)
        assert torch.allclose(got[~sees].float(), clean[~sees].float(), rtol=4 * torch.finfo(dtype).eps, atol=4e-3 if dtype != torch.float32 else 1e-5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 40])
def test_pages_outside_the_pool_are_not_attended(device, dtype, new):
    hq, h, d, page = 4, 2, 64, 16
    lens = [100, 90]
    tables, count = make_tables(lens, page, 1, device)
    tables[0, 2], tables[1, 5] = count, -3  # the second holds some of a chunk's own keys
    pool = make_pool((hq, h, d), page, count, 2, dtype, device)
    q = randn((2 * new, hq, d), 3, dtype, device)
    starts = [n - new for n in lens]
    ops.device_status(device)
    got = paged.attention(q, pool, tables, int32(starts, device), max_seqlen=100)
    assert ops.device_status(device) == ops._lib.STATUS_PAGE
    want, weight, reach = oracle.attend(wide(q), wide(pool), tables.tolist(), starts, None)
    assert (np.abs(wide(got) - want) <= tolerance(dtype, want, weight, reach, d, keys=100)).all()


def test_lengths_past_the_bound_are_cut_and_flagged(device):
    hq, h, d, page = 4, 2, 64, 16
    tables, count = make_tables([100, 60], page, 1, device)
    pool = make_pool((hq, h, d), page, count, 2, torch.float16, device)
    q = randn((2, hq, d), 3, torch.float16, device)
    ops.device_status(device)
    got = paged.attention(q, pool, tables, int32([99, 59], device), max_seqlen=70)
    assert ops.device_status(device) == ops._lib.STATUS_LENGTH_CLAMPED
    want, weight, reach = oracle.attend(wide(q), wide(pool), tables.tolist(), [99, 59], None, max_seqlen=70)
    assert (np.abs(wide(got) - want) <= tolerance(torch.float16, want, weight, reach, d, keys=100)).all()
    # more tokens than the bound says: the first of them are computed, the rest left as they were
    out = torch.full((40, hq, d), 7.0, dtype=torch.float16, device=device)
    q = randn((40, hq, d), 4, torch.float16, device)
    paged.attention(q, pool, tables, int32([10, 0], device), max_seqlen=80, cu_tokens=int32([0, 35, 40], device), max_tokens=16,
                    out=out)
    assert ops.device_status(device) == ops._lib.STATUS_LENGTH_CLAMPED
    want, weight, reach = oracle.attend(wide(q), wide(pool), tables.tolist(), [10, 0], [0, 35, 40])
    near = np.abs(wide(out) - want) <= tolerance(torch.float16, want, weight, reach, d, keys=100)
    assert near[:16].all() and near[35:].all() and (out[16:35] == 7).all()


@pytest.mark.parametrize("cu", [[0, 5, 3], [-2, 1, 4], [0, 2, 9], [3, 3, 4]])
def test_token_bounds_that_do_not_fit_are_not_followed(device, cu):
    """Only a sequence whose bounds lie in order inside the tokens has any."""
    hq, h, d, page = 4, 2, 64, 16
    tables, count = make_tables([40, 40], page, 1, device)
    pool = make_pool((hq, h, d), page, count, 2, torch.float16, device)
    before = pool.clone()
    qkv = randn((4, 8 * d), 3, torch.float16, device)
    paged.append(qkv, pool, tables, int32([10, 20], device), q_heads=hq, cu_tokens=int32(cu, device))
    own = {p for b in range(2) if 0 <= cu[b] <= cu[b + 1] <= 4 for p in range(cu[b + 1] - cu[b])}
    out = torch.full((4, hq, d), 7.0, dtype=torch.float16, device=device)
    q = randn((4, hq, d), 4, torch.float16, device)
    paged.attention(q, pool, tables, int32([10, 20], device), max_seqlen=40, cu_tokens=int32(cu, device), max_tokens=4, out=out)
    written = [t for b in range(2) if 0 <= cu[b] <= cu[b + 1] <= 4 for t in range(cu[b], cu[b + 1])]
    assert [t for t in range(4) if (out[t] != 7).any()] == written
    assert bool((pool != before).any()) == bool(own)
    ops.device_status(device)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_far_apart_and_all_low(device, dtype):
    """One key far above many, and rows whose scores all lie far below zero."""
    hq, h, d, page = 2, 1, 64, 64
    tables, count = make_tables([700], page, 1, device)
    pool = make_pool((hq, h, d), page, count, 2, dtype, device)
    pool[..., 0, :, 1:] *= 0
    pool[..., 0, :, 0] = -3.0
    pool[tables[0, 3].long(), 7, 0, :, 0] = 5.0
    q = torch.zeros((1, hq, d), dtype=dtype, device=device)
    q[0, 0, 0], q[0, 1, 0] = 10.0, 60000.0
    for scale in (0.125, 1.0):
        got = paged.attention(q, pool, tables, int32([699], device), max_seqlen=700, softmax_scale=scale)
        want, weight, reach = oracle.attend(wide(q), wide(pool), tables.tolist(), [699], None, scale=scale)
        assert (np.abs(wide(got) - want) <= tolerance(dtype, want, weight, reach, d, scale, 700)).all()
    pool[tables[0, 3].long(), 7, 0, :, 0] = -3.0
    got = paged.attention(q, pool, tables, int32([699], device), max_seqlen=700)
    want, weight, reach = oracle.attend(wide(q), wide(pool), tables.tolist(), [699], None)
    assert (np.abs(wide(got) - want) <= tolerance(dtype, want, weight, reach, d, keys=700)).all()


def test_attention_in_place_and_strided(device):
    hq, h, d, page = 4, 2, 64, 16
    for new in ([1, 1], [70, 3]):
        tables, count = make_tables([120, 90], page, 1, device)
        pool = make_pool((hq, h, d), page, count, 2, torch.float16, device)
        starts, cu = int32([120 - new[0], 90 - new[1]], device), cu_of(new, device)
        base = randn((sum(new), hq * d + 24), 3, torch.float16, device)
        q = base[:, :hq * d].unflatten(-1, (hq, d))
        args = dict(max_seqlen=120, cu_tokens=cu, max_tokens=max(new))
        want = paged.attention(q.contiguous(), pool, tables, starts, **args)
        assert torch.equal(paged.attention(q, pool, tables, starts, **args), want)
        odd = torch.zeros((sum(new), hq * d + 3), dtype=torch.float16, device=device)[:, 1:hq * d + 1].unflatten(-1, (hq, d))
        paged.attention(q, pool, tables, starts, out=odd, **args)
        assert torch.equal(odd, want)
        wider = torch.full((2, tables.shape[1] + 5), -1, dtype=torch.int32, device=device)
        wider[:, :tables.shape[1]] = tables
        assert torch.equal(paged.attention(q, pool, wider[:, :tables.shape[1]], starts, **args), want)
        paged.attention(q, pool, tables, starts, out=q, **args)
        assert torch.equal(q, want)


# --------------------------------------------------------------- handoff ---


@pytest.mark.parametrize("dtype,geometry", itertools.product(DTYPES, [(8, 2, 64), (4, 3, 128), (2, 1, 256), (4, 1, 16)]))
@pytest.mark.parametrize("order", ["heads", "rows", "apart"])
def test_pack_and_unpack(device, dtype, geometry, order):
    _, h, d = geometry
    lens, page, layers = [1, 0, 16, 37, 64, 15], 16, 3
    tables, count = make_tables(lens, page, 1, device)
    pools = [make_pool(geometry, page, count, 10 + i, dtype, device, order) for i in range(layers)]
    got = paged.pack_live(pools, tables, lens)
    assert got.shape == (layers, sum(lens), 2, h, d)
    for i in range(layers):
        assert np.array_equal(wide(got[i]), oracle.pack(wide(pools[i]), tables.tolist(), lens))
    # into another pool of another page size, in another order of memory
    other, size = make_tables(lens, 32, 2, device)
    target = [make_pool(geometry, 32, size, 20 + i, dtype, device, "rows") for i in range(layers)]
    want = [oracle.unpack(wide(got[i]), wide(target[i]), other.tolist(), lens) for i in range(layers)]
    paged.unpack_live([got[i] for i in range(layers)], target, other, lens)
    assert all(np.array_equal(wide(t), w) for t, w in zip(target, want))


def test_handoff_of_stacked_layers_and_large_batches(device):
    """More sequences and layers than a launch's arguments hold."""
    geometry, page, layers = (2, 1, 16), 16, 100
    lens = [(7 * i) % 40 for i in range(300)]
    tables, count = make_tables(lens, page, 1, device)
    pool = paged.kv_pages(count, page, 1, 16, torch.float16, device, layers=layers)
    pool.copy_(randn(pool.shape, 3, torch.float16, device))
    got = paged.pack_live(pool, tables, lens)
    for i in (0, 57, 99):
        assert np.array_equal(wide(got[i]), oracle.pack(wide(pool[i]), tables.tolist(), lens))
    target = torch.zeros_like(pool)
    paged.unpack_live(got, target, tables, lens)
    assert torch.equal(paged.pack_live(target, tables, lens), got)
    # rows of more than a workgroup's share
    geometry = (64, 64, 256)
    tables, count = make_tables([35, 18], 32, 1, device)
    pool = make_pool(geometry, 32, count, 3, torch.float32, device)
    got = paged.pack_live([pool], tables, [35, 18])
    assert np.array_equal(wide(got[0]), oracle.pack(wide(pool), tables.tolist(), [35, 18]))
    assert paged.pack_live([pool], tables, [0, 0]).shape == (1, 0, 2, 64, 256)


def test_handoff_flags_pages_outside_the_pool(device):
    geometry, lens = (2, 2, 32), [40, 20]
    tables, count = make_tables(lens, 16, 1, device)
    pool = make_pool(geometry, 16, count, 2, torch.bfloat16, device)
    good = paged.pack_live([pool], tables, lens)
    tables[0, 1] = count
    ops.device_status(device)
    got = paged.pack_live([pool], tables, lens)
    assert ops.device_status(device) == ops._lib.STATUS_PAGE
    good[0, 16:32] = 0
    assert torch.equal(got, good)
    before = pool.clone()
    paged.unpack_live(torch.full_like(got, 3.0), [pool], tables, lens)
    assert ops.device_status(device) == ops._lib.STATUS_PAGE
    changed = (pool != before).flatten(2).any(-1)
    assert changed.sum() == 44  # all but the 16 rows of that page


def test_handoff_meets_the_other_caches(device):
    """What a paged prefill side packs, a decode side with plain caches unpacks."""
    geometry, lens = (4, 2, 64), [33, 50]
    tables, count = make_tables(lens, 16, 1, device)
    pools = [make_pool(geometry, 16, count, 3 + i, torch.float16, device) for i in range(2)]
    packed = paged.pack_live(pools, tables, lens)
    plain = [torch.zeros((2, 64, 2, 2, 64), dtype=torch.float16, device=device) for _ in range(2)]
    ops.unpack_live(packed, plain, lens)
    again = [torch.zeros_like(p) for p in pools]
    paged.unpack_live(ops.pack_live(plain, lens), again, tables, lens)
    assert torch.equal(paged.pack_live(again, tables, lens), packed)


# -------------------------------------------------------------- together ---


def test_a_decode_over_pages_matches_plain_caches(device):
    """Prompt in two chunks, handoff, decode steps: the paged calls against
    rope_split, append_kv and decode_attention of the plain caches."""
    hq, h, d, page, dtype = 8, 2, 64, 16, torch.float16
    f = inv_freq_of(d, device)
    lens, steps = [50, 23], 5
    tables, count = make_tables([n + steps for n in lens], page, 1, device)
    pool = make_pool((hq, h, d), page, count, 2, dtype, device)
    cache = torch.zeros((2, 64, 2, h, d), dtype=dtype, device=device)
    prompt = [randn((1, n, (hq + 2 * h) * d), 10 + b, dtype, device) for b, n in enumerate(lens)]
    done = [0, 0]
    for part in (20, None):
        new = [min(part or n, n) - 0 if part else n - s for n, s in zip(lens, done)]
        qkv = torch.cat([prompt[b][0, done[b]:done[b] + new[b]] for b in range(2)])
        cu, starts = cu_of(new, device), int32(done, device)
        q = paged.append(qkv, pool, tables, starts, q_heads=hq, cu_tokens=cu, inv_freq=f)
        out = paged.attention(q, pool, tables, starts, max_seqlen=max(lens), cu_tokens=cu, max_tokens=max(new))
        done = [s + n for s, n in zip(done, new)]
    for b, n in enumerate(lens):
        q, kv = ops.rope_split(prompt[b], hq, h, d, f)
        ops.write_rows(cache, kv, b, 0)
        want = ops.decode_attention(q, cache[b:b + 1], max_seqlen=n, seqlen_bias=n, causal=True)[0, 20:]
        at = 0 if b == 0 else lens[0] - 20
        assert (out[at:at + n - 20].float() - want.float()).abs().max() < 4e-3
    for s in range(steps):
        x = randn((2, 1, (hq + 2 * h) * d), 30 + s, dtype, device)
        starts = int32([n + s for n in lens], device)
        q = paged.append(x[:, 0], pool, tables, starts, q_heads=hq, inv_freq=f)
        out = paged.attention(q, pool, tables, starts, max_seqlen=max(lens) + s + 1)
        q2, kv = ops.rope_split(x, hq, h, d, f, positions=starts)
        want = ops.decode_attention(q2, cache, max_seqlen=max(lens) + s + 1, seqlens=starts, kv_new=kv[:, 0].contiguous())
        assert (out.float() - want[:, 0].float()).abs().max() < 4e-3


@pytest.mark.parametrize("new,dtype", [([1] * 5, torch.float16), ([90, 1, 1, 70, 1], torch.bfloat16), ([1] * 5, torch.float32)])
def test_a_captured_step_replays(device, new, dtype):
    """Append, attention and handoff in one graph, replayed with other inputs
    and lengths (one sequence not in use at times) between eager work."""
    hq, h, d, page = 8, 2, 128, 16
    most = [600 + n for n in new]
    tables, count = make_tables(most, page, 1, device)
    pool = make_pool((hq, h, d), page, count, 2, dtype, device)
    f, cu = inv_freq_of(d, device), cu_of(new, device)
    qkv = randn((sum(new), (hq + 2 * h) * d), 3, dtype, device)
    starts = int32([300, 0, 17, 599, 128], device)

    def step():
        q = paged.append(qkv, pool, tables, starts, q_heads=hq, cu_tokens=cu, inv_freq=f)
        out = paged.attention(q, pool, tables, starts, max_seqlen=max(most), cu_tokens=cu, max_tokens=max(new))
        return out, paged.pack_live([pool], tables, [40] * 5)

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.current_stream().wait_stream(side)
    for n in range(4):
        qkv.copy_(randn(qkv.shape, 50 + n, dtype, device))
        starts.copy_(int32([10 * n, 600 if n else 0, 7 * n, 500 + n, -1 if n == 2 else 64], device))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), n


def test_calls_on_another_stream(device):
    hq, h, d, page = 8, 2, 128, 32
    tables, count = make_tables([500, 300], page, 1, device)
    pool = make_pool((hq, h, d), page, count, 2, torch.bfloat16, device)
    q = randn((2, hq, d), 3, torch.bfloat16, device)
    starts = int32([499, 299], device)
    want = paged.attention(q, pool, tables, starts, max_seqlen=500, partition=64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        parts = [paged.attention(q, pool, tables, starts, max_seqlen=500, partition=64) for _ in range(8)]
    here = [paged.attention(q, pool, tables, starts, max_seqlen=500, partition=64) for _ in range(8)]
    side.synchronize()
    assert all(torch.equal(t, want) for t in parts + here)


def test_pools_of_more_than_2_to_the_32_bytes(device):
    """Pages whose offsets do not fit 32 bits."""
    hq, h, d, page = 8, 1, 128, 1024
    count = (5 << 30) // (page * 2 * d * 2)
    pool = paged.kv_pages(count, page, h, d, torch.float16, device)
    pool[:8].zero_()
    tables = int32([[count - 1, 0], [count - 2, count // 2 + 1]], device)
    for b in range(2):
        for i in range(2):
            pool[tables[b, i].long()] = randn((page, 2, h, d), 3 + 2 * b + i, torch.float16, device)
    f = inv_freq_of(d, device)
    qkv = randn((2, (hq + 2 * h) * d), 9, torch.float16, device)
    starts = int32([1500, 700], device)
    q = paged.append(qkv, pool, tables, starts, q_heads=hq, inv_freq=f)
    got = paged.attention(q, pool, tables, starts, max_seqlen=2048)
    used = tables.flatten().long()
    small, local = pool[used], [[0, 1], [2, 3]]
    want, weight, reach = oracle.attend(wide(q), wide(small), local, [1500, 700], None)
    assert (np.abs(wide(got) - want) <= tolerance(torch.float16, want, weight, reach, d, keys=2048)).all()
    packed = paged.pack_live([pool], tables, [1501, 701])
    assert np.array_equal(wide(packed[0]), oracle.pack(wide(small), local, [1501, 701]))
    del pool
