"""The workspace of attention over pages: its size as Python reports it, by what it grows, and that such a one is taken."""
import pytest
import torch

from hexgen2_amd import paged
from tests.test_gpu_paged import cu_of, int32, make_pool, make_tables, randn


def sized(hq, h, d, dtype, new, keys, device="cpu", **options):
    """attend_workspace_bytes of sequences with `new` tokens each over up to `keys` rows (none of them read)."""
    page = 1024
    pages = paged.kv_pages(1, page, h, d, dtype, device)
    tables = torch.zeros((len(new), paged.pages_for(keys, page)), dtype=torch.int32, device=device)
    q = torch.zeros((1, hq, d), dtype=dtype, device=device).expand(sum(new), hq, d) if sum(new) == 1 else \
        torch.empty((sum(new), hq, d), dtype=dtype, device=device)
    uniform = options.pop("uniform", False)
    return paged.attend_workspace_bytes(q, pages, tables, torch.zeros(len(new), dtype=torch.int32, device=device), max_seqlen=keys,
                                        cu_tokens=None if uniform else cu_of(new, device), max_tokens=max(new), **options)


def test_split_rows_have_a_workspace():
    # four rows of 32 heads in four partitions: 128 dims, a maximum and a sum each
    need = sized(32, 8, 128, torch.float16, [1] * 4, 8192, uniform=True, partition=2048)
    assert need >= 4 * 32 * 4 * (128 + 2) * 4
    assert sized(32, 8, 128, torch.float16, [1] * 4, 8192, partition=2048) == need
    assert sized(32, 8, 128, torch.float16, [1] * 4, 64, uniform=True) == 0
    assert sized(32, 8, 128, torch.bfloat16, [512], 8192, uniform=True, partition=4096) >= 512 * 32 * 2 * 130 * 4


@pytest.mark.parametrize("hq,h,d,dtype", [(32, 8, 128, torch.float32), (32, 8, 32, torch.bfloat16), (8, 1, 16, torch.float16),
                                          (32, 8, 128, torch.bfloat16), (4, 4, 256, torch.float16)])
@pytest.mark.parametrize("new", [[2048] + [1] * 63, [512] + [1] * 63, [4096], [3, 700, 1, 1, 90], [1] * 300, [9] * 40])
def test_the_workspace_grows_with_the_tokens(hq, h, d, dtype, new):
    """Every row of every token split, on both of a launch's paths, is the most that is taken, however
    long the longest sequence is; and of single tokens no more than they are."""
    for options, parts in ((dict(partition=1024), 8), ({}, 32)):
        paths = 2 if d >= 64 and dtype != torch.float32 and max(new) > 1 else 1
        assert sized(hq, h, d, dtype, new, 8192, **options) <= paths * sum(new) * hq * parts * (d + 2) * 4


def test_more_split_rows_than_a_launch_joins_are_refused():
    # 2^21 tokens of 32 heads: 2^26 rows, a wave each, are 2^32 lanes
    with pytest.raises(ValueError, match="2\\^26 split rows"):
        sized(32, 2, 16, torch.float16, [1 << 21], 256, uniform=True, partition=128)
    assert sized(32, 2, 16, torch.float16, [1 << 20], 256, uniform=True, partition=128) == (1 << 25) * 2 * 18 * 4



def test_bounds_that_attention_refuses_have_no_size():
    with pytest.raises(ValueError, match="max_seqlen"):
        sized(8, 2, 64, torch.float16, [1], -1)
    with pytest.raises(ValueError, match="multiple of 64"):
        sized(8, 2, 64, torch.float16, [1], 1000, partition=100)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,new", [(torch.float16, 64, [1, 1]), (torch.bfloat16, 128, [70, 1]), (torch.float32, 128, [5, 40]),
                                         (torch.bfloat16, 32, [90, 1])])
def test_a_workspace_of_that_size_is_taken(device, dtype, d, new):
    hq, h, page, lens = 8, 2, 64, [4200, 700]
    tables, count = make_tables(lens, page, 1, device)
    pool = make_pool((hq, h, d), page, count, 2, dtype, device)
    q, starts = randn((sum(new), hq, d), 3, dtype, device), int32([n - m for n, m in zip(lens, new)], device)
    options = dict(max_seqlen=4200, cu_tokens=cu_of(new, device), max_tokens=max(new), partition=512)
    want = paged.attention(q, pool, tables, starts, **options)
    need = paged.attend_workspace_bytes(q, pool, tables, starts, **options)
    assert need > 0
    space = torch.full((need + 64,), 255, dtype=torch.uint8, device=device)  # (all NaN, if read before it is written)
    got = paged.attention(q, pool, tables, starts, workspace=space[:need], **options)
    assert torch.equal(got, want) and (space[need:] == 255).all()
    with pytest.raises(ValueError, match="workspace"):
        paged.attention(q, pool, tables, starts, workspace=space[:need - 1], **options)
