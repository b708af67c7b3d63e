"""Paged attention and append over the far ends of their ranges: tiles of 256 rows over
long caches, rows of many partitions, hundreds of ragged sequences, calls at the
same time on streams and with graphs, pages that sequences share."""
import numpy as np
import pytest
import torch

from hexgen2_amd import ops, paged
from oracle import paged_oracle as oracle
from tests.test_gpu_paged import (DTYPES, check_append, check_attend, cu_of, inv_freq_of, int32, make_pool, make_tables,
                                  randn, tolerance, wide)

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]


# From 4096 keys on and 512 rows a KV head, heads of 128 take tiles of 256 rows.


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("causal", [True, False])
def test_tiles_of_256_rows(device, dtype, causal):
    check_attend(device, dtype, (8, 1, 128), [70], [4050], 64, causal, uniform=True)
    check_attend(device, dtype, (16, 2, 128), [65, 65], [4031, 70], 16, causal, uniform=True, order="rows")
    check_attend(device, dtype, (4, 1, 128), [131], [4100], 128, causal, uniform=True, partition=64)
    check_attend(device, dtype, (4, 1, 128), [129], [3968], 128, causal, uniform=True, partition=1024, order="apart")


@pytest.mark.parametrize("dtype", HALVES)
def test_tiles_of_256_rows_beside_single_tokens(device, dtype):
    check_attend(device, dtype, (8, 1, 128), [70, 1, 3, 33], [4030, 0, 1500, 4090], 64)
    check_attend(device, dtype, (8, 1, 128), [1, 0, 70], [4095, 40, 300], 32, partition=192, extra=3)
    check_attend(device, dtype, (8, 1, 128), [64, 66], [4096, -1], 64)
    check_attend(device, dtype, (8, 1, 128), [1, 64], [4096, 4000], 64, causal=False, partition=1 << 20)


@pytest.mark.parametrize("value", [float("inf"), float("nan"), -float("inf")])
@pytest.mark.parametrize("dtype", HALVES)
def test_tiles_of_256_rows_and_values_that_are_not_finite(device, dtype, value):
    """Beyond the lengths they do nothing; attended, they reach those rows alone."""
    check_attend(device, dtype, (8, 1, 128), [70, 40], [4027, 17], 64, fill=value)
    hq, h, d, page, start, new = 8, 1, 128, 64, 4050, 70
    tables, count = make_tables([start + new], page, 1, device)
    pool = make_pool((hq, h, d), page, count, 2, dtype, device)
    q = randn((new, hq, d), 3, dtype, device)
    clean = paged.attention(q, pool, tables, int32([start], device), max_seqlen=start + new)
    at = start + 50
    pool[tables[0, at // page].long(), at % page, 1, 0, 9] = value
    got = paged.attention(q, pool, tables, int32([start], device), max_seqlen=start + new)
    want = torch.ones((new, hq, d), dtype=torch.bool)
    want[50:, :, 9] = False
    assert torch.equal(torch.isfinite(got.cpu()), want)
    assert torch.allclose(got[:50].float(), clean[:50].float(), rtol=4 * torch.finfo(dtype).eps, atol=4e-3)


@pytest.mark.parametrize("dtype", HALVES)
def test_tiles_of_256_rows_skip_pages_outside_the_pool(device, dtype):
    hq, h, d, page, start, new = 8, 1, 128, 64, 4050, 70
    tables, count = make_tables([start + new], page, 1, device)
    tables[0, 3], tables[0, 63], tables[0, 64] = count, -1, 1 << 30
    pool = make_pool((hq, h, d), page, count, 2, dtype, device)
    q = randn((new, hq, d), 3, dtype, device)
    ops.device_status(device)
    got = paged.attention(q, pool, tables, int32([start], device), max_seqlen=start + new)
    assert ops.device_status(device) == ops._lib.STATUS_PAGE
    want, weight, reach = oracle.attend(wide(q), wide(pool), tables.tolist(), [start], None)
    assert (np.abs(wide(got) - want) <= tolerance(dtype, want, weight, reach, d, keys=start + new)).all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("causal", [True, False])
def test_tiles_of_heads_of_256(device, dtype, causal):
    check_attend(device, dtype, (8, 1, 256), [260], [260], 16, causal, uniform=True)
    check_attend(device, dtype, (8, 2, 256), [150, 1, 33, 9], [1001, 900, 0, 130], 32, causal, order="rows", extra=2)
    check_attend(device, dtype, (4, 4, 256), [70, 64], [2000, 127], 64, causal, order="apart", partition=192)
    for fill in (float("nan"), float("inf")):
        check_attend(device, dtype, (8, 1, 256), [100, 3], [1300, 17], 64, causal, fill=fill)


@pytest.mark.parametrize("dtype", HALVES)
def test_tiles_of_heads_of_256_and_what_they_leave_out(device, dtype):
    hq, h, d, page, start, new = 8, 1, 256, 64, 1300, 110
    tables, count = make_tables([start + new], page, 1, device)
    pool = make_pool((hq, h, d), page, count, 2, dtype, device)
    q = randn((new, hq, d), 3, dtype, device)
    clean = paged.attention(q, pool, tables, int32([start], device), max_seqlen=start + new)
    at = start + 50
    pool[tables[0, at // page].long(), at % page, 1, 0, 9] = float("nan")
    got = paged.attention(q, pool, tables, int32([start], device), max_seqlen=start + new)
    want = torch.ones((new, hq, d), dtype=torch.bool)
    want[50:, :, 9] = False
    assert torch.equal(torch.isfinite(got.cpu()), want)
    assert torch.allclose(got[:50].float(), clean[:50].float(), rtol=4 * torch.finfo(dtype).eps, atol=4e-3)
    pool[tables[0, at // page].long(), at % page, 1, 0, 9] = 0
    tables[0, 3], tables[0, 20] = count, -1
    ops.device_status(device)
    got = paged.attention(q, pool, tables, int32([start], device), max_seqlen=start + new)
    assert ops.device_status(device) == ops._lib.STATUS_PAGE
    want, weight, reach = oracle.attend(wide(q), wide(pool), tables.tolist(), [start], None)
    assert (np.abs(wide(got) - want) <= tolerance(dtype, want, weight, reach, d, keys=start + new)).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_many_partitions(device, dtype):
    """More partitions than a wave has lanes, and more keys than the most partitions
    of the length asked for hold."""
    check_attend(device, dtype, (2, 1, 16), [1, 1, 1], [20000, 0, 8191], 1024, uniform=True, partition=64)
    check_attend(device, dtype, (2, 2, 64), [2, 1], [9000, 4160], 256, partition=128)
    check_attend(device, dtype, (1, 1, 16), [1], [70000], 4096, uniform=True, partition=64)
    check_attend(device, dtype, (4, 1, 64), [40, 1], [9000, 5000], 256, partition=64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_hundreds_of_ragged_sequences(device, dtype):
    new = [1 + (i % 5 == 0) * (i % 7) for i in range(300)]
    starts = [(37 * i) % 90 - (i % 11 == 10) * 200 for i in range(300)]
    check_attend(device, dtype, (4, 2, 64), new, starts, 16, extra=2)
    check_append(device, dtype, (4, 2, 64), new, starts, 16, 64, extra=2)
    new = [0, 50, 0, 0, 17] * 26  # sequences without tokens between tiles
    check_attend(device, dtype, (4, 2, 64), new, [5] * 130, 16)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("lens", [[5000], [5000, 300]])
def test_padded_chunks(device, dtype, lens):
    """Token tensors much longer than what cu_tokens bounds: single tokens where the call
    could hold chunks alone."""
    hq, h, d, page, n = 8, 1, 128, 64, len(lens)
    tables, count = make_tables([x + 1 for x in lens], page, 1, device)
    pool = make_pool((hq, h, d), page, count, 2, dtype, device)
    q = randn((70 * n, hq, d), 3, dtype, device)
    out, cu = torch.full_like(q, 7.0), list(range(n + 1))
    paged.attention(q, pool, tables, int32(lens, device), max_seqlen=5001, cu_tokens=int32(cu, device), max_tokens=70, out=out)
    want, weight, reach = oracle.attend(wide(q), wide(pool), tables.tolist(), lens, cu)
    assert (np.abs(wide(out) - want)[:n] <= tolerance(dtype, want, weight, reach, d, keys=5001)[:n]).all()
    assert (out[n:] == 7).all()


def test_the_smallest_calls(device):
    for dtype in DTYPES:
        check_attend(device, dtype, (1, 1, 16), [1], [0], 16, uniform=True)
        check_attend(device, dtype, (1, 1, 128), [1], [0], 16)
        check_append(device, dtype, (1, 1, 16), [1], [0], 16, 2, uniform=True)
    # no keys at all: rows are zero
    q = randn((1, 4, 64), 1, torch.float16, device)
    pool = make_pool((4, 2, 64), 16, 1, 2, torch.float16, device)
    tables = int32([[0]], device)
    assert (paged.attention(q, pool, tables, int32([0], device), max_seqlen=0) == 0).all()
    assert ops.device_status(device) == ops._lib.STATUS_LENGTH_CLAMPED
    empty = torch.zeros((1, 0), dtype=torch.int32, device=device)
    assert (paged.attention(q, pool, empty, int32([-1], device), max_seqlen=0) == 0).all()
    assert ops.device_status(device) == 0
    for n in (0, 3):  # no tokens
        got = paged.attention(q[:0], pool, tables.expand(n, 1), int32([0] * n, device), max_seqlen=16)
        assert got.shape == (0, 4, 64)
        assert paged.append(randn((0, 8 * 64), 1, torch.float16, device), pool, tables.expand(n, 1), int32([0] * n, device),
                            q_heads=4).shape == (0, 4, 64)


def test_stacked_handoffs_of_changing_lengths(device):
    """One stack of pools, other lengths and packets each time, none at all among them; refusals after good calls."""
    pool = paged.kv_pages(8, 16, 2, 64, torch.float16, device, layers=3)
    pool.copy_(randn(pool.shape, 1, torch.float16, device))
    tables = int32([[0, 1, 2, 3], [4, 5, 6, 7]], device)
    for lens in ([0, 0], [5, 60], [64, 0], [5, 60], [1, 1]):
        got = paged.pack_live(pool, tables, lens)
        for i in range(3):
            assert np.array_equal(wide(got[i]), oracle.pack(wide(pool[i]), tables.tolist(), lens))
        out = torch.empty_like(got)
        assert paged.pack_live(pool, tables, lens, out=out) is out and torch.equal(out, got)
        target = torch.zeros_like(pool)
        paged.unpack_live(got, target, tables, lens)
        assert torch.equal(paged.pack_live(target, tables, lens), got)
    for bad in (torch.empty((3, 3, 2, 2, 64), dtype=torch.float16, device=device), got[:2], got.float(), got.cpu()):
        with pytest.raises(ValueError):
            paged.unpack_live(bad, pool, tables, [1, 1])
        with pytest.raises(ValueError):
            paged.pack_live(pool, tables, [1, 1], out=bad)
    for wrong in (tables.cpu(), tables.long(), tables[:1]):
        with pytest.raises(ValueError):
            paged.pack_live(pool, wrong, [1, 1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_sequences_that_share_a_prefix(device, dtype):
    """The same page in several tables, and twice in one, is read like any other."""
    hq, h, d, page = 4, 2, 64, 16
    pool = make_pool((hq, h, d), page, 6, 1, dtype, device)
    tables, starts, new = int32([[0, 1, 2], [0, 1, 3], [0, 0, 0]], device), [39, 32, 40], [1, 9, 2]
    q, cu = randn((12, hq, d), 2, dtype, device), cu_of(new, device)
    got = paged.attention(q, pool, tables, int32(starts, device), max_seqlen=48, cu_tokens=cu, max_tokens=9)
    want, weight, reach = oracle.attend(wide(q), wide(pool), tables.tolist(), starts, cu.tolist())
    assert (np.abs(wide(got) - want) <= tolerance(dtype, want, weight, reach, d, keys=48)).all()
    rows = paged.pack_live([pool], tables, [40, 41, 48])
    assert np.array_equal(wide(rows[0]), oracle.pack(wide(pool), tables.tolist(), [40, 41, 48]))


@pytest.mark.parametrize("new,partition", [([1, 1], 64), ([70, 3], 64), ([70], 1024)])
def test_split_rows_in_place(device, new, partition):
    """out may be q, or lie beside it in the same rows, where several workgroups read a row."""
    hq, h, d, page = 8, 1, 128, 64
    lens = [4130, 333][:len(new)]
    tables, count = make_tables(lens, page, 1, device)
    pool = make_pool((hq, h, d), page, count, 2, torch.bfloat16, device)
    starts, cu = int32([n - m for n, m in zip(lens, new)], device), cu_of(new, device)
    both = randn((sum(new), 2, hq, d), 3, torch.bfloat16, device)
    args = dict(max_seqlen=max(lens), cu_tokens=cu, max_tokens=max(new), partition=partition)
    want = paged.attention(both[:, 0].contiguous(), pool, tables, starts, **args)
    paged.attention(both[:, 0], pool, tables, starts, out=both[:, 1], **args)
    assert torch.equal(both[:, 1], want)
    paged.attention(both[:, 0], pool, tables, starts, out=both[:, 0], **args)
    assert torch.equal(both[:, 0], want)
    if sum(new) > 2:  # (both[1:, 0] and both[:1, 0] share nothing)
        with pytest.raises(ValueError, match="rows of q"):
            paged.attention(both[1:, 0], pool, tables, starts, out=both[:-1, 0], **args)


@pytest.mark.parametrize("new,lens,dtype", [([70], [4200], torch.bfloat16), ([70, 1], [4200, 900], torch.float16),
                                            ([1] * 3, [5000, 17, 4100], torch.float32)])
def test_captured_steps_side_by_side(device, new, lens, dtype):
    """Two graphs of split rows that replay at once on two streams, and eager calls beside them."""
    hq, h, d, page = 8, 1, 128, 64
    tables, count = make_tables(lens, page, 1, device)
    pool = make_pool((hq, h, d), page, count, 2, dtype, device)
    cu, starts = cu_of(new, device), int32([n - m for n, m in zip(lens, new)], device)
    qs = [randn((sum(new), hq, d), 3 + i, dtype, device) for i in range(3)]
    streams = [torch.cuda.Stream() for _ in range(2)]

    def step(q):
        return paged.attention(q, pool, tables, starts, max_seqlen=max(lens), cu_tokens=cu, max_tokens=max(new), partition=512)

    want = [step(q) for q in qs]
    torch.cuda.synchronize()
    graphs, held = [], []
    for q, stream in zip(qs, streams):
        with torch.cuda.stream(stream):
            step(q)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                held.append(step(q))
            graphs.append(graph)
    for _ in range(3):
        torch.cuda.synchronize()
        for t in held:
            t.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        here = step(qs[2])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([*held, here], want))


def test_two_threads_at_once(device):
    """Calls of several geometries from two host threads, each on a stream of its own."""
    import threading
    jobs = []
    for i, (geometry, new, lens) in enumerate([((8, 2, 64), [1, 1], [900, 40]), ((4, 1, 128), [40, 1], [300, 77])]):
        hq, h, d = geometry
        tables, count = make_tables(lens, 16, i, device)
        pool = make_pool(geometry, 16, count, 2, torch.float16, device)
        q, cu = randn((sum(new), hq, d), 3, torch.float16, device), cu_of(new, device)
        jobs.append((q, pool, tables, int32([n - m for n, m in zip(lens, new)], device),
                     dict(max_seqlen=max(lens), cu_tokens=cu, max_tokens=max(new))))
    want = [paged.attention(*job[:4], **job[4]) for job in jobs]
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for n in range(60):
                job = jobs[i]
                got[i].append(paged.attention(*job[:4], **{**job[4], "max_seqlen": job[4]["max_seqlen"] + n % 3}))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(len(g) == 60 and all(torch.equal(t, w) for t in g) for g, w in zip(got, want))


def test_a_step_over_two_pools_of_one_geometry(device):
    """Nothing of a call is kept for the next: other pools, tables and lengths at the same sizes."""
    geometry, page = (8, 2, 128), 32
    for seed in range(3):
        check_attend(device, torch.bfloat16, geometry, [1, 40, 2], [100 + seed, 7 * seed, 2], page, seed=seed, max_seqlen=160)
    f = inv_freq_of(128, device)
    tables, count = make_tables([64], page, 1, device)
    pools = [make_pool(geometry, page, count, 5, torch.bfloat16, device) for _ in range(2)]
    for at, pool in ((3, pools[0]), (9, pools[1]), (3, pools[1]), (9, pools[0])):
        paged.append(randn((1, 12 * 128), 7, torch.bfloat16, device), pool, tables, int32([at], device), q_heads=8, inv_freq=f)
    assert torch.equal(*pools)
