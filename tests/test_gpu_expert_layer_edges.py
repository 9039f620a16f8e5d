"""Where the router's choice, the norm and SwiGLU's gradient can go wrong: sums that cancel or leave the range, numbers that are not finite, rows next to a
border of rounding. Against 64 bits on the CPU (oracle/layers.py)."""

import math

import pytest
import torch

import deep_gemm
import oracle
from both_hosts import moe_hosts
from helpers import seed_all

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
INF, NAN = math.inf, math.nan


def _routed(logits, topk, scoring='softmax', **kw):
    """The choices are those of the oracle."""
    cuda = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    idx, w = deep_gemm.moe_route(logits.cuda(), topk, scoring, **cuda)
    want, want_w = oracle.moe_route_ref(logits, topk, scoring, **kw)
    assert torch.equal(idx.cpu(), want)
    # (24 roundings of a score, 90 of a softmax's with logits that are at most 8 apart: twice that)
    assert ((w.cpu().double() - want_w).abs() <= 220 * E * want_w.abs()).all()
    return idx, w


# --------------------------------------------------------------------------------------------------------- the router
@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('size', [2, 4, 8])
def test_groups_whose_large_biases_cancel(scoring, size):
    """Scores of a group that are sums of a large positive and a large negative number, next to one another."""
    seed_all(size)
    for large in (4.0, 16.0, 64.0, 256.0, 5000.0):
        for groups, taken in ((2, 1), (8, 3)):
            one = torch.full((size,), -large)
            one[size // 2] = large
            first = torch.randn(500, 1, size)
            logits = (first + 1e-5 * torch.randn(500, groups, size)).flatten(1).contiguous()
            _routed(logits, 1, scoring, bias=one.repeat(groups), num_groups=groups, topk_groups=taken)
            _routed(logits, min(4, taken * size), scoring, bias=one.repeat(groups), num_groups=groups, topk_groups=taken, renormalize=True)


def test_groups_whose_sums_leave_the_range():
    """The largest numbers of FP32 as biases: their sums are infinite in 32 bits, and are told apart in 64."""
    seed_all(1)
    logits, lowest = torch.randn(5, 16), torch.finfo(torch.float32).min
    for scoring in ('softmax', 'sigmoid'):
        _routed(logits, 3, scoring, bias=torch.tensor([2e38] * 4 + [3e38] * 4 + [2.5e38] * 4 + [-1.0] * 4), num_groups=4, topk_groups=2)
        _routed(logits, 6, scoring, bias=torch.tensor([-3e38] * 4 + [-2e38] * 4 + [-2.5e38] * 8), num_groups=4, topk_groups=2)
        # every expert, and all but one of a group, masked by the least number
        for topk in (1, 2, 6):
            _routed(logits, topk, scoring, bias=torch.full((16,), lowest), num_groups=4, topk_groups=2)
            bias = torch.full((16,), lowest)
            bias[[9, 14]] = 0.0
            _routed(logits, topk, scoring, bias=bias, num_groups=4, topk_groups=2)
            bias[:4] = -INF
            _routed(logits, topk, scoring, bias=bias, num_groups=4, topk_groups=2)


@pytest.mark.parametrize('host', moe_hosts)
def test_a_sum_that_is_not_a_number_shows(host):
    """Weights that are divided by a sum with a NaN in it are NaN, and so are their gradients; places without a choice have the weight 0 all the same."""
    seed_all(2)
    logits = torch.randn(5, 40)
    logits[1, 7] = NAN
    logits[2, 4:] = -INF
    logits[2, 1] = NAN
    logits[3, 9] = INF
    logits[4] = -INF
    g = torch.randn(5, 6)
    for scoring in ('softmax', 'sigmoid'):
        idx, w = host.moe_route(logits.cuda(), 6, scoring, renormalize=True, scale=2.5)
        want, want_w = oracle.moe_route_ref(logits, 6, scoring, renormalize=True, scale=2.5)
        assert torch.equal(idx.cpu(), want) and torch.equal(w.isnan().cpu(), want_w.isnan())
        assert w[1].isnan().all() and w[2, :4].isnan().all() and (w[2, 4:] == 0).all() and (w[4] == 0).all()
        got = host.moe_route_grad(g.cuda(), logits.cuda(), idx, scoring, True, 2.5).cpu()
        chosen = torch.zeros(5, 40, dtype=torch.bool)
        for t in range(5):
            chosen[t, [e for e in want[t].tolist() if e >= 0]] = True
        bad = torch.tensor([False, True, True, scoring == 'softmax', False])
        assert torch.equal(got.isnan(), chosen & bad[:, None]) and (got[~chosen] == 0).all()
