"""The FP4 quantiser on the layouts that the grouped GEMMs read, by the arguments' defaults."""

import inspect
import re

import pytest
import torch

import deep_gemm
import oracle
from both_hosts import python_layer, quant_hosts
from deep_gemm import _api
from helpers import assert_close, seed_all

NAN = float('nan')


def test_the_default_alignment_is_that_of_the_grouped_layouts():
    assert inspect.signature(python_layer('quant_ops').cast_to_fp4).parameters['expert_alignment'].default == _api.MK_ALIGNMENT
    if deep_gemm.BACKEND == '_C':
        said = re.search(r'expert_alignment: [^=]*= (\d+)', deep_gemm.cast_to_fp4.__doc__)
        assert int(said.group(1)) == _api.MK_ALIGNMENT


def _codes(packed):
    u = packed.cpu().contiguous().view(torch.uint8)
    return torch.stack((u & 15, u >> 4), dim=-1).flatten(-2)


def _plan(sizes, extra=0):
    """moe_sort of choices that give the experts these numbers of rows."""
    idx = torch.cat([torch.full((n,), e) for e, n in enumerate(sizes)] + [torch.full((extra,), -1)])
    return deep_gemm.moe_sort(idx[torch.randperm(idx.numel())].view(-1, 1).cuda(), len(sizes))


@pytest.mark.gpu
@pytest.mark.parametrize('host', quant_hosts)
@pytest.mark.parametrize('sizes', [(100, 40), (1, 0, 300, 129, 128), (300,)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_a_plan_without_an_alignment_of_its_own(host, sizes, dtype):
    """Groups whose next multiple of 128 is not their next multiple of 256: rows in between are padding, the second group's start and what is
    behind the last group as well."""
    seed_all(len(sizes))
    plan = _plan(sizes, 20)
    rows, total = plan[2].numel(), oracle.align(int(plan[0][-1]), 256)
    valid = plan[2].cpu() >= 0
    x = torch.randn(rows, 96)
    x[~valid] = NAN
    x = x.to(dtype)
    torch.full((rows, 48), 0x5a, dtype=torch.int8, device='cuda')     # (given back at once: what a new tensor may hold)
    out, sf = host.cast_to_fp4(x.cuda(), plan[0], mn_major=True)
    code, byte, _ = oracle.cast_fp4_ref(x, -2, valid)
    got = sf.cpu().int()
    assert torch.equal(_codes(out)[:total], code[:total])
    assert torch.equal(torch.stack((got & 255, got >> 8 & 255), 1).flatten(0, 1)[:total // 32], byte[:total // 32].int())
    out, sf = host.cast_to_fp4(x.cuda(), plan[0])
    code, byte, _ = oracle.cast_fp4_ref(x, -1, valid)
    got = sf.cpu().int()
    assert torch.equal(_codes(out)[valid], code[valid])
    assert torch.equal(torch.stack((got & 255, got >> 8 & 255), -1).flatten(1)[valid][:, :3], byte[valid].int())


@pytest.mark.gpu
@pytest.mark.parametrize('host', quant_hosts)
def test_the_weight_gradient_in_fp4_as_it_is_documented(host):
    """Both sides of a weight gradient quantised down the rows of a plan, no alignment given; the padding holds NaN."""
    seed_all(6)
    plan = _plan((100, 40, 0, 257, 3), 50)
    rows, psum = plan[2].numel(), plan[0].cpu().tolist()
    valid = plan[2].cpu() >= 0
    x, dy = torch.randn(rows, 256), torch.randn(rows, 384)
    for t in (x, dy):
        t[~valid] = NAN
    a, b = (host.cast_to_fp4(t.cuda(), plan[0], mn_major=True) for t in (dy, x))
    d = torch.full((5, 384, 256), NAN, device='cuda')
    deep_gemm.k_grouped_fp8_gemm_tn_contiguous(a, b, d, None, plan[0])
    assert deep_gemm.device_status() == 0
    total = oracle.align(psum[-1], 256)
    ref = oracle.k_grouped_psum_ref(*(oracle.cast_fp4_ref(t, -2, valid)[2].float()[:total] for t in (dy, x)), psum, torch.float32)
    assert_close(d, ref, 'weight gradient')


@pytest.mark.gpu
@pytest.mark.parametrize('host', quant_hosts)
@pytest.mark.parametrize('mn_major', [False, True])
def test_a_layout_without_experts_is_refused(host, mn_major):
    """It is not the same as no layout, for which all rows count."""
    none = torch.empty(0, dtype=torch.int32, device='cuda')
    for rows in (64, 0):
        with pytest.raises(RuntimeError, match='must hold an expert'):
            host.cast_to_fp4(torch.ones(rows, 64, device='cuda'), none, mn_major=mn_major)
