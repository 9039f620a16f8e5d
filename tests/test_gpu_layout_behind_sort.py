"""Grouped GEMMs right behind the sort that makes their layout: with launches that overlap, they are on the device before it is there. Runs are
captured and replayed on other choices, so that the layout of the run before is what memory holds until then."""

import pytest
import torch

import deep_gemm
from helpers import seed_all

pytestmark = pytest.mark.gpu

EXPERTS, TOPK = 48, 4


def _choices(tokens, seed):
    gen = torch.Generator().manual_seed(seed)
    liked = torch.randn(EXPERTS, generator=gen)
    return (torch.randn(tokens, EXPERTS, generator=gen) + liked).topk(TOPK, dim=1).indices


def _replayed(tokens, sort, gemm, d):
    """The captured pair of calls on new choices, and the same calls with the device idle in between."""
    idx = _choices(tokens, 0).cuda()
    gemm(sort(idx))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gemm(sort(idx))
    for seed in range(1, 13):
        idx.copy_(_choices(tokens, seed))
        d.fill_(7.0)
        graph.replay()
        got = d.clone()
        d.fill_(7.0)
        plan = sort(idx.clone())
        torch.cuda.synchronize()
        gemm(plan)
        assert torch.equal(got, d), seed
    assert deep_gemm.device_status() == 0


@pytest.mark.parametrize('tokens', [30, 700])
def test_masked(tokens):
    seed_all(1)
    a = [deep_gemm.cast_to_fp8(torch.randn(128, 512, device='cuda').bfloat16()) for _ in range(EXPERTS)]
    scales = torch.stack([sf.t() for _, sf in a]).transpose(1, 2)
    a = (torch.stack([q.view(torch.uint8) for q, _ in a]).view(torch.float8_e4m3fn), scales)
    w = deep_gemm.cast_to_fp4(torch.randn(EXPERTS, 256, 512, device='cuda'))
    d = torch.empty(EXPERTS, 128, 256, dtype=torch.bfloat16, device='cuda')
    _replayed(tokens, lambda i: deep_gemm.moe_sort(i, EXPERTS, max_m=128),
              lambda plan: deep_gemm.m_grouped_fp8_fp4_gemm_nt_masked(a, w, d, plan[0], max(1, tokens * TOPK // EXPERTS)), d)


@pytest.mark.parametrize('tokens', [30, 700])
def test_psum(tokens):
    seed_all(2)
    rows = deep_gemm.moe_sort(_choices(tokens, 0).cuda(), EXPERTS)[2].numel()
    a = deep_gemm.cast_to_fp8(torch.randn(rows, 512, device='cuda').bfloat16())
    w = deep_gemm.cast_to_fp4(torch.randn(EXPERTS, 256, 512, device='cuda'))
    d = torch.empty(rows, 256, dtype=torch.bfloat16, device='cuda')
    _replayed(tokens, lambda i: deep_gemm.moe_sort(i, EXPERTS), lambda plan: deep_gemm.m_grouped_fp8_fp4_gemm_nt_contiguous(a, w, d, plan[0]), d)


@pytest.mark.parametrize('tokens', [30, 700])
def test_k_grouped(tokens):
    seed_all(3)
    rows = deep_gemm.moe_sort(_choices(tokens, 0).cuda(), EXPERTS)[2].numel()
    a, b = (torch.randn(rows, n, device='cuda').bfloat16() for n in (256, 128))
    d = torch.empty(EXPERTS, 256, 128, device='cuda')
    _replayed(tokens, lambda i: deep_gemm.moe_sort(i, EXPERTS), lambda plan: deep_gemm.k_grouped_bf16_gemm_tn_contiguous(a, b, d, None, plan[0]), d)
