"""Rotation of far positions: paged.append turns by the exact angle, ops.rope_split (the plain caches)
by its fp32 product, so that they part by no more than that product's rounding."""
import pytest
import torch

from hexgen2_amd import ops, paged, rotary
from tests.test_gpu_paged import int32, randn

pytestmark = pytest.mark.gpu

LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}


@pytest.mark.parametrize("position", [0, 2000, 100000, 1 << 20])
@pytest.mark.parametrize("scaling", [None, LLAMA3])
def test_rotations_of_plain_and_paged_caches_part_by_the_angles_rounding(device, position, scaling):
    hq, h, d, page, n = 4, 2, 128, 1 << 14, 20
    f, scale = rotary.frequencies(d, 500000.0, scaling, device=device)
    assert scale == 1
    qkv = randn((1, n, (hq + 2 * h) * d), 3, torch.float32, device)
    tables = torch.zeros((1, paged.pages_for(position + n, page)), dtype=torch.int32, device=device)
    pool = paged.kv_pages(1, page, h, d, torch.float32, device)
    q = paged.append(qkv[0], pool, tables, int32([position], device), q_heads=hq, inv_freq=f)
    plain_q, plain_kv = ops.rope_split(qkv, hq, h, d, f, offset=position)
    rows = pool[0, torch.arange(position, position + n, device=device) % page]
    x = qkv[0].view(n, -1, d)[:, :hq + h].double()
    # the product of a position and a frequency is off by half a step of itself, sines, cosines, products and
    # sums by a few of 1
    size = torch.hypot(x[..., :d // 2], x[..., d // 2:]).repeat(1, 1, 2)
    angle = torch.arange(position, position + n, device=device, dtype=torch.float64)[:, None] * f.double()
    tol = size * (angle.repeat(1, 2)[:, None] * 2.0 ** -24 + 2.0 ** -21)
    apart = torch.cat((q - plain_q[0], rows[:, 0] - plain_kv[0, :, 0]), dim=1).double().abs()
    assert (apart <= tol).all(), float((apart / tol).max())
    assert torch.equal(rows[:, 1], plain_kv[0, :, 1])
