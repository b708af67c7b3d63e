"""Infinities and NaN that split rows attend: the same result whatever the partitions."""
import numpy as np
import pytest
import torch

from hexgen2_amd import paged
from oracle import paged_oracle as oracle
from tests.test_gpu_paged import int32, make_pool, make_tables, randn, wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.bfloat16, 128), (torch.float32, 64), (torch.bfloat16, 32)])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("new", [1, 40])
def test_values_that_are_not_finite_in_split_rows(device, dtype, d, value, new):
    """A value in the first, a middle or the last of 1 to 9 partitions, attended by all rows, by some or by none."""
    hq, h, page, total = 4, 2, 64, 1100
    tables, count = make_tables([total], page, 1, device)
    pool = make_pool((hq, h, d), page, count, 2, dtype, device)
    q = randn((new, hq, d), 3, dtype, device)
    for at in (3, 500, 1050, 1070, total - 1):
        old = pool[tables[0, at // page].long(), at % page, 1, 1, 5].item()
        pool[tables[0, at // page].long(), at % page, 1, 1, 5] = value
        with np.errstate(all="ignore"):
            want = oracle.attend(wide(q), wide(pool), tables.tolist(), [total - new], None)[0]
        for partition in (1 << 20, 640, 384, 256, 192, 128):
            got = wide(paged.attention(q, pool, tables, int32([total - new], device), max_seqlen=total, partition=partition))
            odd = ~np.isfinite(want)
            assert np.array_equal(got[odd], want[odd], equal_nan=True), (at, partition)
            assert np.isfinite(got[~odd]).all()
        pool[tables[0, at // page].long(), at % page, 1, 1, 5] = old
