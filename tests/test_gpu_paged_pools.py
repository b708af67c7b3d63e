"""Pools whose positions lie far apart: a row's place in its page does not fit 32 bits."""
import numpy as np
import pytest
import torch

from hexgen2_amd import paged
from oracle import paged_oracle as oracle
from tests.test_gpu_paged import cu_of, int32, inv_freq_of, randn, tolerance, wide

pytestmark = pytest.mark.gpu


def far_pool(base, dtype, page, heads, d, single):
    """Positions 2^26 elements apart: a pool stored position after position, or one page of rows with gaps."""
    memory = base.view(dtype)
    if single:
        return memory.as_strided((1, page, 2, heads, d), (0, 1 << 26, heads * d, d, 1))
    return memory.view(page, -1, 2, heads, d).transpose(0, 1)


@pytest.fixture(scope="module")
def base(device):
    memory = torch.empty(64 << 27, dtype=torch.uint8, device=device)  # 8.6 GB, of which little is written
    yield memory
    del memory
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,page", [(torch.bfloat16, 64), (torch.float16, 64), (torch.float32, 32), (torch.float32, 16)])
@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("new", [1, 12])
def test_positions_that_lie_far_apart(device, base, dtype, page, single, new):
    """Append, attention of single tokens and of chunks, and the handoff, in the last rows of such pages."""
    hq, h, d = 8, 2, 128
    pool = far_pool(base[:(page << 26) * dtype.itemsize], dtype, page, h, d, single)
    assert pool.stride(1) == 1 << 26 and pool.shape[1] == page
    used = [0] if single else [7, pool.shape[0] - 1, 1]
    rows = randn((len(used), page, 2, h, d), 3, dtype, device)
    for i, n in enumerate(used):
        pool[n] = rows[i]
    start, f = len(used) * page - 1 - new, inv_freq_of(d, device)
    tables = int32([used], device)
    qkv = randn((new, (hq + 2 * h) * d), 9, dtype, device)
    q = paged.append(qkv, pool, tables, int32([start], device), q_heads=hq, inv_freq=f)
    _, after = oracle.append(wide(qkv), wide(rows), [list(range(len(used)))], [start], None, hq, wide(f))
    small = pool[tables[0].long()]
    assert np.abs(wide(small) - after).max() <= 2 * np.abs(after).max() * torch.finfo(dtype).eps
    want, weight, reach = oracle.attend(wide(q), wide(small), [list(range(len(used)))], [start], None)
    got = paged.attention(q, pool, tables, int32([start], device), max_seqlen=start + new)
    assert (np.abs(wide(got) - want) <= tolerance(dtype, want, weight, reach, d, keys=start + new)).all()
    packed = paged.pack_live([pool], tables, [start + new])
    assert np.array_equal(wide(packed[0]), oracle.pack(wide(small), [list(range(len(used)))], [start + new]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tiles_of_256_rows_of_positions_that_lie_far_apart(device, base, dtype):
    hq, h, d, page, new, start = 16, 2, 128, 64, 70, 4050
    pool = far_pool(base, dtype, page, h, d, False)
    used = [3 * i + 5 for i in range(paged.pages_for(start + new, page))]
    rows = randn((len(used), page, 2, h, d), 3, dtype, device)
    pool[torch.tensor(used, device=device)] = rows
    q, cu = randn((new + 1, hq, d), 4, dtype, device), [0, new, new + 1]
    local = [list(range(len(used))), list(range(len(used)))[::-1]]
    tables = int32([used, used[::-1]], device)
    got = paged.attention(q, pool, tables, int32([start, 1000], device), max_seqlen=start + new, cu_tokens=cu_of([new, 1], device),
                          max_tokens=new)
    want, weight, reach = oracle.attend(wide(q), wide(rows), local, [start, 1000], cu)
    assert (np.abs(wide(got) - want) <= tolerance(dtype, want, weight, reach, d, keys=start + new)).all()
