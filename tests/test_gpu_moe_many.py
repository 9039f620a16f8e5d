"""The MoE row operators where there is enough work for the forms that large calls take, against sums in 64 bits on the GPU.

Tolerances as for the small calls: u = half a step of the result's type (BF16 2^-8, FP32 2^-24), e = 2^-24. A sum of k products in FP32 is within
(k + 1) e of the sum of the terms' magnitudes, rounding adds u of the value; a product has one rounding in FP32 and one to the result's type; a dot
product of H terms over at least 32 lanes passes every term through at most H / 32 + 40 additions. (Sums in 64 bits add 2^-53 each: nothing beside these.)"""

import pytest
import torch

import deep_gemm
import oracle
from both_hosts import moe_hosts
from helpers import seed_all

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
NAN = float('nan')
BUSY_WARPS = 148 * 64         # from this number of warps' work on a call takes the forms for many tokens (kBusyWarps of the kernels)


def _plan(tokens, topk, experts, seed=0, max_m=None):
    """Token t has t % (topk + 1) choices here, at random places among its topk; the others are another rank's. The same expert may be there twice.
    -> (plan, token_rows int64 [tokens, topk] on the GPU, choices int64 by rows)."""
    gen = torch.Generator().manual_seed(seed)
    here = torch.rand(tokens, topk, generator=gen).argsort(1) < (torch.arange(tokens) % (topk + 1))[:, None]
    idx = torch.where(here, torch.randint(0, experts, (tokens, topk), generator=gen), -1)
    plan, ref = deep_gemm.moe_sort(idx.cuda(), experts, max_m=max_m), oracle.moe_sort_ref(idx, experts, 256, max_m)
    for a, b in zip(plan, ref):
        assert torch.equal(a.cpu(), b)
    if max_m is None:
        live = (plan[1] >= 0).sum(1)
        assert torch.equal(live.cpu(), torch.arange(tokens) % (topk + 1))
    return plan, plan[1].long(), plan[2].reshape(-1).long()


def _warps(tokens, hidden, dtype, pieces):
    """Warps of a call that takes `pieces` of 16 bytes of a token's row in each lane."""
    units = hidden * (2 if dtype == torch.bfloat16 else 4) // 16
    return tokens * oracle.ceil_div(units, 32 * pieces)


# tokens, choices of each, hidden: whole turns, a last turn or warp with only part of the pieces, few pieces, more choices than a warp has lanes
COMBINES = [(2600, 8, 2048, torch.bfloat16), (2600, 8, 1000, torch.bfloat16), (2500, 12, 1160, torch.bfloat16), (1500, 5, 7168, torch.bfloat16),
            (9600, 4, 8, torch.bfloat16), (2600, 40, 1032, torch.bfloat16), (3001, 8, 2052, torch.float32), (2500, 3, 700, torch.float32),
            (1300, 34, 1156, torch.float32), (9500, 8, 4, torch.float32)]


@pytest.mark.parametrize('tokens,topk,hidden,dtype', COMBINES)
def test_combine_of_many_tokens(tokens, topk, hidden, dtype):
    """Every number of rows from none to all of a token's choices."""
    assert _warps(tokens, hidden, dtype, 1) >= BUSY_WARPS
    seed_all(tokens + hidden)
    plan, of, choice = _plan(tokens, topk, 24, hidden)
    rows = torch.randn(plan[2].numel(), hidden, device='cuda').to(dtype)
    rows[choice < 0] = NAN                                        # rows without a choice are not read
    weights = torch.rand(tokens, topk, device='cuda') * 2 - 0.5
    weights[of < 0] = NAN                                         # nor do the weights of choices without a row count
    for w in (None, weights):
        ref = torch.zeros(tokens, hidden, dtype=torch.float64, device='cuda')
        size = torch.zeros_like(ref)
        for j in range(topk):
            has = of[:, j] >= 0
            term = rows[of[has, j]].double() * (1.0 if w is None else w[has, j, None].double())
            ref[has] += term
            size[has] += term.abs()
        err = (topk + 1) * E * size * (1 + 2 * topk * E)
        err += HALF[dtype] * (ref.abs() + err)
        for host in moe_hosts:
            room = torch.full((tokens + 1, hidden), 7.0, dtype=dtype, device='cuda')
            out = host.moe_combine(rows, plan, w, out=room[:tokens])
            assert ((out.double() - ref).abs() <= err).all()
            assert (room[tokens] == 7).all()


@pytest.mark.parametrize('tokens,topk,hidden,dtype', COMBINES)
def test_gradient_of_many_tokens(tokens, topk, hidden, dtype):
    seed_all(tokens + hidden + 1)
    plan, of, choice = _plan(tokens, topk, 24, hidden)
    live = choice >= 0
    rows = torch.randn(plan[2].numel(), hidden, device='cuda').to(dtype)
    rows[~live] = NAN
    g = torch.randn(tokens, hidden, device='cuda').to(dtype)
    weights = torch.rand(tokens, topk, device='cuda') * 2 - 0.5
    weights[of < 0] = NAN
    out = torch.full_like(rows, 7.0)
    dy, dw = deep_gemm.moe_combine_grad(g, rows, plan, weights, out=out)
    assert (dy[~live] == 7).all()
    for j in range(topk):
        has = of[:, j] >= 0
        at, gj = of[has, j], g[has].double()
        ref = gj * weights[has, j, None].double()
        assert ((dy[at].double() - ref).abs() <= (HALF[dtype] * (1 + E) + E) * ref.abs()).all(), j
        terms = rows[at].double() * gj
        assert ((dw[has, j].double() - terms.sum(1)).abs() <= (hidden / 32 + 40) * E * terms.abs().sum(1)).all(), j
        assert (dw[~has, j] == 0).all()


@pytest.mark.parametrize('tokens,topk,hidden,dtype,max_m', [(2600, 8, 7168, torch.bfloat16, None), (9600, 3, 1000, torch.bfloat16, None), (3001, 4, 2052, torch.float32, None),
                                                            (5000, 40, 1160, torch.bfloat16, None), (9500, 2, 8, torch.bfloat16, 300), (4000, 6, 2056, torch.bfloat16, 70)])
def test_dispatch_of_many_tokens(tokens, topk, hidden, dtype, max_m):
    """Tokens without a choice here are passed over."""
    assert _warps(tokens, hidden, dtype, 4) >= BUSY_WARPS
    seed_all(hidden)
    plan, _, choice = _plan(tokens, topk, 24, hidden, max_m)
    live, pad = choice >= 0, oracle.moe_padding(plan[0].cpu(), choice.numel(), 256, max_m).cuda()
    x = torch.randn(tokens, hidden, device='cuda').to(dtype)
    for host in moe_hosts:
        for zero in (False, True):
            out = torch.full((*plan[2].shape, hidden), 7.0, dtype=dtype, device='cuda')
            flat = host.moe_dispatch(x, plan, out=out, zero_padding=zero).view(-1, hidden)
            assert torch.equal(flat[live], x[choice[live] // topk])
            assert (flat[pad] == (0.0 if zero else 7.0)).all() and (flat[~live & ~pad] == 7.0).all()


@pytest.mark.parametrize('tokens,topk,hidden', [(1500, 8, 7168), (2047, 40, 1568), (8191, 6, 512), (9600, 2, 32)])
def test_dispatch_to_fp8_of_many_tokens_in_one_launch(tokens, topk, hidden):
    """Scales written one by one where there are tokens enough to pass over those without a choice."""
    assert deep_gemm._lib.lib().dg_moe_dispatch_fp8_scratch_bytes(tokens, hidden) == 0 and tokens * oracle.ceil_div(hidden, 256) >= BUSY_WARPS
    seed_all(hidden)
    plan, _, choice = _plan(tokens, topk, 24, hidden)
    live = choice >= 0
    x = (torch.randn(tokens, hidden, device='cuda') * 3).bfloat16()
    codes, sf = deep_gemm.cast_to_fp8(x)                          # compared with 64 bits elsewhere
    data = torch.full((plan[2].numel(), hidden), 0x11, dtype=torch.uint8, device='cuda')
    scales = torch.full((sf.size(1), plan[2].numel()), 0x2222, dtype=torch.int16, device='cuda').t()
    for host in moe_hosts:
        got, got_sf = host.moe_dispatch_to_fp8(x, plan, out=(data.view(torch.float8_e4m3fn), scales))
        assert torch.equal(data[live], codes.view(torch.uint8)[choice[live] // topk]) and torch.equal(got_sf[live], sf[choice[live] // topk])
        assert (data[~live] == 0x11).all() and (got_sf[~live] == 0x2222).all()


def test_any_number_of_experts_over_a_cluster():
    """Numbers of experts that end inside a warp, on the paths with barriers between the CTAs."""
    gen = torch.Generator().manual_seed(1)
    for experts in (1, 2, 7, 31, 33, 100, 161, 511, 1000, 1023):
        idx = torch.randint(-1, experts, (6001, 3), generator=gen)
        for max_m in (None, 50):
            plan, ref = deep_gemm.moe_sort(idx.cuda(), experts, max_m=max_m), oracle.moe_sort_ref(idx, experts, 256, max_m)
            assert all(torch.equal(a.cpu(), b) for a, b in zip(plan, ref)), (experts, max_m)


def test_a_captured_run_of_many_tokens_on_other_choices():
    """Replays write the same memory: what a kernel may find there before the one in front of it is done is the plan of the run before."""
    tokens, topk, experts, h = 2300, 6, 40, 2048
    gen = torch.Generator().manual_seed(4)
    choices = lambda: torch.where(torch.rand(tokens, topk, generator=gen) < 0.7, torch.randint(0, experts, (tokens, topk), generator=gen), -1)  # noqa: E731
    assert deep_gemm._lib.lib().dg_moe_dispatch_fp8_scratch_bytes(tokens, h) > 0
    idx, x = choices().cuda(), torch.randn(tokens, h, device='cuda').bfloat16()

    def way():
        plan = deep_gemm.moe_sort(idx, experts)
        q, sf = deep_gemm.moe_dispatch_to_fp8(x, plan)
        y = deep_gemm.moe_dispatch(x, plan)
        return (*plan, q.view(torch.uint8), sf, y, deep_gemm.moe_combine(y, plan))

    way()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = way()
    for seed in range(8):
        idx.copy_(choices())
        x.copy_(torch.randn(tokens, h))
        graph.replay()
        codes, sf = deep_gemm.cast_to_fp8(x)
        choice = held[2].long()
        live = choice >= 0
        of = choice[live] // topk
        for a, b in zip(held[:3], oracle.moe_sort_ref(idx.cpu(), experts)):
            assert torch.equal(a.cpu(), b), seed
        assert torch.equal(held[3][live], codes.view(torch.uint8)[of]) and torch.equal(held[4][live], sf[of]) and torch.equal(held[5][live], x[of]), seed
        ref = x.double() * (idx >= 0).sum(1, keepdim=True)
        size = ref.abs()
        assert ((held[6].double() - ref).abs() <= (topk + 1) * E * size + HALF[torch.bfloat16] * (size + (topk + 1) * E * size)).all(), seed
