"""Calls of attention over pages that are refused before anything runs."""
import ctypes

import pytest

from hexgen2_amd import _lib
from tests.test_paged_host import attend_params, pool, refused, seqs


def test_launches_of_2_to_the_32_lanes_and_more_are_refused():
    # one chunk of 2^20 tokens, 32 heads on one of 128: 2^17 tiles of 256 rows (512 lanes) in 64 partitions
    p = attend_params(pool=pool(kv_heads=1, head_dim=128, pos_stride=128, kv_stride=16 * 128, head_stride=0, page_stride=2 * 16 * 128),
                      q_heads=32, q_stride=32 * 128, out_stride=32 * 128, max_tokens=1 << 20, max_seqlen=4096, partition=64, out=1 << 40,
                      seqs=seqs(batch=1, tokens=1 << 20, table_width=256, table_stride=256, cu_tokens=None))
    refused(lambda lib: lib.hexkv_paged_attend(ctypes.byref(p), None, 0, None), _lib.HEXKV_ERANGE, "2\\^32 lanes")
    p.partition = 128
    refused(lambda lib: lib.hexkv_paged_attend(ctypes.byref(p), None, 0, None), _lib.HEXKV_EWORKSPACE, "workspace")


@pytest.mark.parametrize("scale", [3.4e38, 2.4e38, 2.36e38])
def test_scales_that_no_float_holds_in_powers_of_two_are_refused(scale):
    """Scores are taken in powers of two: a scale whose product with log2(e) is infinite would make every score so."""
    refused(lambda lib: lib.hexkv_paged_attend(ctypes.byref(attend_params(softmax_scale=scale)), None, 0, None),
            _lib.HEXKV_EINVAL, "softmax_scale")
