"""How exact the probabilities of attention over pages are: inputs whose scores are
exact in fp32, so that little but the probabilities' own rounding is left."""
import numpy as np
import pytest
import torch

from hexgen2_amd import paged
from oracle import paged_oracle as oracle
from tests.test_gpu_paged import cu_of, half_step, int32, make_tables, wide

HALVES = [torch.float16, torch.bfloat16]


def inputs(dtype, geometry, new, starts, page, seed, device="cpu"):
    """Queries and keys with one element that is not zero: every score is one product, exact in fp32."""
    hq, h, d = geometry
    g = torch.Generator().manual_seed(seed)
    tables, count = make_tables([s + n for s, n in zip(starts, new)], page, seed, device)
    pool = paged.kv_pages(count, page, h, d, dtype, device).zero_()
    pool[..., 0, :, 0] = (2 * torch.randn(pool.shape[:2] + (h,), generator=g, dtype=torch.float64)).to(dtype).to(device)
    pool[..., 1, :, :] = torch.randn(pool.shape[:2] + (h, d), generator=g, dtype=torch.float64).to(dtype).to(device)
    q = torch.zeros((sum(new), hq, d), dtype=dtype, device=device)
    q[..., 0] = (1 + torch.rand((sum(new), hq), generator=g, dtype=torch.float64)).to(dtype).to(device)
    return q, pool, tables


def tolerance(dtype, want, weight, reach, keys):
    """Half a step of the output's type, and of the sum of p |v|: two 16-bit terms a
    probability (half a step squared), sums of `keys` fp32 terms taken 16 at a time, and p's
    own error, once in the numerator and once in the sum.  That is, for scores of
    up to X in size: 3 X half steps for the scale's three roundings; of an exponent of up to 2 X log2(e) + 15 half a
    step and of exp2 two, in p and in up to six factors that bring sums to another maximum."""
    x = reach[..., None]
    p = (3 * x + 7 * (3 * x + 17)) * 2.0 ** -24
    sums = (keys / 16 + 40) * 2.0 ** -24
    return half_step(dtype) * np.abs(want) * 1.01 + weight * 2 * (p + half_step(dtype) ** 2 + sums) + 1e-30


def check(device, dtype, geometry, new, starts, page, uniform=False, partition=0, causal=True, seed=0):
    q, pool, tables = inputs(dtype, geometry, new, starts, page, seed, device)
    cu, keys = None if uniform else cu_of(new, device), max(s + n for s, n in zip(starts, new))
    got = paged.attention(q, pool, tables, int32(starts, device), max_seqlen=keys, cu_tokens=cu, max_tokens=max(new),
                          softmax_scale=1.0, partition=partition, causal=causal)
    want, weight, reach = oracle.attend(wide(q), wide(pool), tables.tolist(), starts, None if uniform else cu.tolist(), causal, 1.0)
    off = np.abs(wide(got) - want) / tolerance(dtype, want, weight, reach, keys)
    assert (off <= 1).all(), float(off.max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("geometry", [(8, 2, 64), (8, 1, 128), (2, 1, 256), (6, 2, 32), (4, 2, 16)])
def test_rows_keep_probabilities_in_two_terms(device, dtype, geometry):
    check(device, dtype, geometry, [1] * 9, [0, 1, 14, 15, 31, 32, 100, 255, 640], 16, uniform=True)
    check(device, dtype, geometry, [1, 2, 1], [640, 0, 333], 64, partition=64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("geometry", [(4, 1, 64), (4, 2, 128), (8, 1, 256)])
def test_tiles_keep_probabilities_in_two_terms(device, dtype, geometry, causal):
    more = 600 if geometry[2] == 256 else 0  # (from 2^20 query heads times keys on heads of 256 take tiles)
    check(device, dtype, geometry, [150], [250 + more], 16, uniform=True, causal=causal)
    check(device, dtype, geometry, [140, 1, 65], [250 + more, 200, 77], 32, partition=64, causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
def test_tiles_of_256_rows_keep_probabilities_in_two_terms(device, dtype):
    check(device, dtype, (8, 1, 128), [70], [4050], 64, uniform=True)
    check(device, dtype, (8, 1, 128), [70, 1, 3], [4030, 0, 1500], 64, partition=512)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("keys", [40, 700])
def test_the_tolerance_sees_a_probability_of_one_term(dtype, keys):
    """The same sums with each probability rounded once: outside of what two terms allow."""
    q, pool, tables = inputs(dtype, (8, 2, 64), [1] * 4, [keys - 1] * 4, 16, 1)
    want, weight, reach = oracle.attend(wide(q), wide(pool), tables.tolist(), [keys - 1] * 4, None, True, 1.0)
    rough = np.zeros_like(want)
    for t in range(4):
        rows = wide(pool)[[tables[t, p // 16].item() for p in range(keys)], [p % 16 for p in range(keys)]]
        for head in range(8):
            s = rows[:, 0, head // 4] @ wide(q)[t, head]
            e = np.exp(s - s.max())
            one = wide(torch.from_numpy(e * 2.0 ** 11).to(dtype)) / 2.0 ** 11
            rough[t, head] = one @ rows[:, 1, head // 4] / e.sum()
    assert (np.abs(rough - want) > tolerance(dtype, want, weight, reach, keys)).any()
