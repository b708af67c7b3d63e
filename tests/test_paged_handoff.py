"""Handoffs whose layers overlap are refused before anything is copied."""
import ctypes

import pytest
import torch

from hexgen2_amd import _lib, paged
from tests.test_gpu_paged import int32
from tests.test_paged_host import PAGES, QKV, TABLE, pool, refused

POOL = 8 * 2 * 2 * 16 * 64 * 2  # bytes of a layer's pool
PACKED = 13 * 2 * 2 * 64 * 2    # and of its packet


def copy(name, pages, packed):
    array = lambda x: (ctypes.c_void_p * len(x))(*x)  # noqa: E731
    sides = (pages, packed) if name == "hexkv_paged_pack" else (packed, pages)
    return lambda lib: getattr(lib, name)(ctypes.byref(pool()), *map(array, sides), len(pages), TABLE, 4, 4, 2,
                                          (ctypes.c_int64 * 2)(10, 3), None)


@pytest.mark.parametrize("name", ["hexkv_paged_pack", "hexkv_paged_unpack"])
@pytest.mark.parametrize("pages,packed", [
    ([PAGES], [PAGES]), ([PAGES], [PAGES + POOL - 16]), ([PAGES], [PAGES - PACKED + 16]),
    ([PAGES, PAGES + POOL], [QKV, PAGES + POOL // 2]), ([PAGES + POOL, PAGES], [PAGES + 2 * POOL - 16, QKV]),
    ([PAGES + 4 * POOL, PAGES, PAGES + 2 * POOL], [QKV, PAGES + 3 * POOL - 16, QKV + PACKED]),
])
def test_layers_that_are_read_and_written_must_lie_apart(name, pages, packed):
    refused(copy(name, pages, packed), _lib.HEXKV_EINVAL, "overlaps")


def test_layers_that_are_written_must_lie_apart():
    refused(copy("hexkv_paged_pack", [PAGES, PAGES + POOL], [QKV, QKV]), _lib.HEXKV_EINVAL, "overlaps")
    refused(copy("hexkv_paged_pack", [PAGES, PAGES], [QKV, QKV + PACKED - 16]), _lib.HEXKV_EINVAL, "overlaps")
    refused(copy("hexkv_paged_unpack", [PAGES, PAGES + POOL, PAGES], [QKV] * 3), _lib.HEXKV_EINVAL, "overlaps")


@pytest.mark.parametrize("name", ["hexkv_paged_pack", "hexkv_paged_unpack"])
def test_overlaps_among_more_layers_than_a_launch_takes(name):
    pages = [PAGES + (i * 73 % 200) * POOL for i in range(200)]
    packed = [QKV + i * PACKED for i in range(199)]
    refused(copy(name, pages, packed + [PAGES + 150 * POOL + 16]), _lib.HEXKV_EINVAL, "overlaps")


@pytest.mark.gpu
def test_layers_side_by_side_and_on_top_of_each_other(device):
    """One allocation holds pools and packets: next to each other they are copied, a byte over they are refused."""
    memory = torch.randn(2 * POOL + 2 * PACKED, device=device).to(torch.float16)
    n, m = POOL // 2, PACKED // 2
    pages = [memory[i * n:(i + 1) * n].view(8, 2, 2, 16, 64).transpose(1, 3) for i in range(2)]
    tables, lens = int32([[3, -1, -1, -1], [7, -1, -1, -1]], device), [10, 3]
    packed = [memory[2 * n + i * m:2 * n + (i + 1) * m].view(13, 2, 2, 64) for i in range(2)]
    want = paged.pack_live(pages, tables, lens)
    paged.pack_live(pages, tables, lens, out=packed)
    assert all(torch.equal(a, b) for a, b in zip(packed, want))
    paged.unpack_live(packed, pages, tables, lens)
    assert torch.equal(paged.pack_live(pages, tables, lens), want)
    over = [packed[0], memory[2 * n - 8:2 * n - 8 + m].view(13, 2, 2, 64)]
    for out in (over, [packed[0], packed[0]]):
        with pytest.raises(ValueError, match="overlaps"):
            paged.pack_live(pages, tables, lens, out=out)
    for layers in (pages, [pages[0], pages[0]]):
        with pytest.raises(ValueError, match="overlaps"):
            paged.unpack_live(over, layers, tables, lens)
    # pools that lie in turn, page by page
    both = torch.zeros((8, 2, 2, 2, 16, 64), dtype=torch.float16, device=device)
    turn = [both[:, i].transpose(1, 3) for i in range(2)]
    paged.unpack_live(want, turn, tables, lens)
    assert torch.equal(paged.pack_live(turn, tables, lens), want)
