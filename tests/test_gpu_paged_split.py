"""Split rows that are numbered by token: chunks beside many single tokens, with and without tiles,
padded, in place and captured."""
import pytest
import torch

from hexgen2_amd import ops, paged
from tests.test_gpu_paged import check_attend, cu_of, int32, make_pool, make_tables, randn

pytestmark = pytest.mark.gpu

KINDS = [(torch.float32, (8, 2, 64)), (torch.float32, (4, 1, 128)), (torch.bfloat16, (6, 2, 32)), (torch.float16, (4, 2, 16)),
         (torch.bfloat16, (8, 2, 128)), (torch.float16, (8, 1, 64)), (torch.bfloat16, (4, 2, 256))]


@pytest.mark.parametrize("dtype,geometry", KINDS)
@pytest.mark.parametrize("causal", [True, False])
def test_chunks_beside_many_single_tokens(device, dtype, geometry, causal):
    new = [1] * 20 + [37] + [1] * 20 + [0, 3]
    starts = [(131 * i) % 900 - (i % 9 == 8) * 1000 for i in range(20)] + [700] + [(77 * i) % 1100 for i in range(20)] + [5, 250]
    check_attend(device, dtype, geometry, new, starts, 32, causal, partition=128, extra=5)
    check_attend(device, dtype, geometry, new, starts, 16, causal, partition=64)
    check_attend(device, dtype, geometry, new, starts, 64, causal)


@pytest.mark.parametrize("dtype,geometry", KINDS)
def test_they_in_place_and_captured(device, dtype, geometry):
    hq, h, d = geometry
    new = [1] * 15 + [40, 1, 9]
    lens = [100 + (211 * i) % 900 for i in range(len(new))]
    tables, count = make_tables(lens, 32, 1, device)
    pool = make_pool(geometry, 32, count, 2, dtype, device)
    cu, starts = cu_of(new, device), int32([n - m for n, m in zip(lens, new)], device)
    args = dict(max_seqlen=max(lens), cu_tokens=cu, max_tokens=max(new), partition=128)
    q = randn((sum(new), hq, d), 3, dtype, device)
    want = paged.attention(q.clone(), pool, tables, starts, **args)
    assert paged.attention(q, pool, tables, starts, out=q, **args) is q and torch.equal(q, want)
    need = paged.attend_workspace_bytes(q, pool, tables, starts, **args)
    space = torch.full((need,), 255, dtype=torch.uint8, device=device)
    held = torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            paged.attention(q, pool, tables, starts, out=held, workspace=space, **args)
    torch.cuda.current_stream().wait_stream(side)
    for n in range(3):
        q.copy_(randn(q.shape, 50 + n, dtype, device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, paged.attention(q, pool, tables, starts, **args)), n
    assert ops.device_status(device) & ops._lib.STATUS_ERRORS == 0
