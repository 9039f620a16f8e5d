"""The router's choices -> rows of a grouped layout -> back, with gradients, against loops in 64 bits on the CPU (oracle/moe.py).

Tolerances. u = half a step of the result's type (BF16 2^-8, FP32 2^-24), e = 2^-24. A sum of k products in FP32, one fused multiply-add
each, is within k e (1 + k e) of the sum of the terms' magnitudes; rounding adds u of the value. A product w g has one rounding in FP32 and
one to the result's type. A dot product of H terms that is split over at least 32 lanes passes every term through at most
H / 32 + 40 additions, whatever the order."""

import itertools

import pytest
import torch

import deep_gemm
import oracle
from both_hosts import moe_hosts, python_layer
from helpers import seed_all

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
NAN = float('nan')


def _choices(tokens, topk, total, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.rand(tokens, total, generator=gen).topk(topk, dim=1).indices


def _sort(idx, experts, alignment=256, max_m=None, host=deep_gemm):
    plan = host.moe_sort(idx.cuda(), experts, expert_alignment=alignment, max_m=max_m)
    return plan, oracle.moe_sort_ref(idx, experts, alignment, max_m)


def _check_plan(plan, ref):
    for name, a, b in zip(('layout', 'token_rows', 'row_choices'), plan, ref):
        assert a.dtype == torch.int32 and a.shape == b.shape, name
        assert torch.equal(a.cpu(), b), name


# ------------------------------------------------------------------------------------------------------------------ sort
@pytest.mark.parametrize('host', moe_hosts)
@pytest.mark.parametrize('tokens,topk,experts', [(1, 1, 1), (1, 8, 256), (3, 2, 5), (33, 6, 64), (128, 8, 32), (1000, 4, 160), (777, 8, 1024)])
@pytest.mark.parametrize('dtype', [torch.int32, torch.int64])
def test_sort(host, tokens, topk, experts, dtype):
    idx = _choices(tokens, topk, experts, tokens).to(dtype)
    _check_plan(*_sort(idx, experts, host=host))
    _check_plan(*_sort(idx, experts, 1, host=host))
    _check_plan(*_sort(idx, experts, max_m=3, host=host))


@pytest.mark.parametrize('tokens,topk,experts,alignment', [(4095, 8, 64, 256), (4097, 1, 7, 32), (8191, 6, 160, 100), (16384, 8, 256, 256), (40000, 3, 1000, 64),
                                                           (131073, 2, 1024, 8)])
def test_sort_over_a_cluster(tokens, topk, experts, alignment):
    gen = torch.Generator().manual_seed(tokens)
    idx = torch.randint(-1, experts + 1, (tokens, topk), generator=gen)
    idx[: tokens // 3] = torch.randint(0, 1 + experts // 8, (tokens // 3, topk), generator=gen)        # long groups, and the same expert twice
    _check_plan(*_sort(idx, experts, alignment))
    _check_plan(*_sort(idx.int(), experts, max_m=70))


def test_sort_of_choices_without_an_expert():
    far = torch.tensor([[-1, 3], [4, -7], [2 ** 32 + 1, -2 ** 32], [2, 2 ** 62], [2, 2]])
    _check_plan(*_sort(far, 4))                                   # 2^32 + 1 is not expert 1
    _check_plan(*_sort(far, 4, max_m=2))                          # the third choice of expert 2 is dropped
    none = torch.full((50, 4), -1)
    _check_plan(*_sort(none, 16))
    _check_plan(*_sort(none, 16, max_m=8))
    same = torch.full((300, 8), 5)
    _check_plan(*_sort(same, 16))
    _check_plan(*_sort(same, 6, max_m=64))
    empty = torch.empty(0, 8, dtype=torch.int64)
    _check_plan(*_sort(empty, 16))
    _check_plan(*_sort(empty, 16, max_m=8))


# -------------------------------------------------------------------------------------------------------------- dispatch
LAYOUTS = [(1, 1, 1, 1, None), (1, 8, 64, 64, None), (37, 3, 8, 8, None), (300, 6, 32, 4, None), (64, 8, 16, 16, 40), (50, 2, 8, 1, 7), (20, 40, 48, 48, None)]


def _plan(tokens, topk, total, experts, max_m, alignment=256):
    idx = _choices(tokens, topk, total, tokens + topk)
    idx = torch.where(idx < experts, idx, -1)
    return _sort(idx, experts, alignment, max_m)


@pytest.mark.parametrize('host', moe_hosts)
@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('hidden,dtype', [(8, torch.bfloat16), (1000, torch.bfloat16), (2048, torch.bfloat16), (4, torch.float32), (700, torch.float32), (7168, torch.float32)])
def test_dispatch(host, layout, hidden, dtype):
    seed_all(hidden)
    plan, (psum, token_rows, row_choices) = _plan(*layout)
    x = torch.randn(layout[0], hidden, dtype=dtype)
    for zero in (False, True):
        out = torch.full((*row_choices.shape, hidden), 7.0, dtype=dtype, device='cuda')
        assert host.moe_dispatch(x.cuda(), plan, out=out, zero_padding=zero).data_ptr() == out.data_ptr()
        flat, choice = out.cpu().view(-1, hidden), row_choices.view(-1).long()
        live, pad = choice >= 0, oracle.moe_padding(psum, row_choices.numel(), 256, layout[4])
        assert torch.equal(flat[live], x[choice[live] // layout[1]])
        assert not (live & pad).any()
        assert (flat[pad] == (0.0 if zero else 7.0)).all() and (flat[~live & ~pad] == 7.0).all()
    fresh = host.moe_dispatch(x.cuda(), plan)
    assert fresh.shape == out.shape and torch.equal(fresh.cpu().view(-1, hidden)[live], flat[live])


@pytest.mark.parametrize('host', moe_hosts)
@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('hidden', [32, 288, 512, 1120, 7168])
def test_dispatch_to_fp8(host, layout, hidden):
    """Bit for bit what the quantiser makes of the dispatched rows."""
    seed_all(hidden)
    plan, (_, _, row_choices) = _plan(*layout)
    x = (torch.randn(layout[0], hidden) * 3).bfloat16()
    x[0, :32] = 0
    codes, sf, _, _ = oracle.swiglu_quant_ref(x, swiglu=False)
    choice = row_choices.view(-1).long()
    live = choice >= 0
    cols = sf.size(1)
    data = torch.full((*row_choices.shape, hidden), 0x11, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn)
    groups, per = (layout[3], layout[4]) if layout[4] else (1, row_choices.numel())
    scales = torch.full((groups, cols, per), 0x2222, dtype=torch.int16, device='cuda').transpose(1, 2)
    scales = scales if layout[4] else scales[0]
    for out in (None, (data, scales)):
        got, got_sf = host.moe_dispatch_to_fp8(x.cuda(), plan, out=out)
        assert got.dtype == torch.float8_e4m3fn and got.shape == data.shape and got_sf.dtype == torch.int16 and got_sf.shape == scales.shape
        assert got_sf.stride(-2) == 1 or per == 1
        flat, flat_sf = got.view(torch.uint8).cpu().view(-1, hidden), got_sf.cpu().contiguous().view(-1, cols)
        assert torch.equal(flat[live], codes[choice[live] // layout[1]])
        assert torch.equal(flat_sf[live], sf[choice[live] // layout[1]])
    assert (flat[~live] == 0x11).all() and (flat_sf[~live] == 0x2222).all()


@pytest.mark.parametrize('tokens,topk,experts,max_m,hidden', [(2100, 6, 16, None, 7168), (2301, 8, 40, None, 4128), (3100, 2, 7, 333, 8224), (2100, 33, 64, 130, 3200),
                                                              (5000, 1, 3, None, 65568)])
def test_dispatch_to_fp8_of_many_tokens(tokens, topk, experts, max_m, hidden):
    """Where the scales take a second launch."""
    assert deep_gemm._lib.lib().dg_moe_dispatch_fp8_scratch_bytes(tokens, hidden) > 0
    seed_all(hidden)
    idx = _choices(tokens, topk, 2 * experts, 5)
    plan, (_, _, row_choices) = _sort(torch.where(idx < experts, idx, -1), experts, max_m=max_m)
    x = (torch.randn(tokens, hidden, device='cuda') * 3).bfloat16()
    codes, sf = deep_gemm.cast_to_fp8(x)
    choice = row_choices.view(-1).long().cuda()
    live = choice >= 0
    cols = sf.size(1)
    data = torch.full((*row_choices.shape, hidden), 0x11, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn)
    groups, per = (experts, max_m) if max_m else (1, row_choices.numel())
    room = torch.full((groups, cols + 1, per + 5), 0x2222, dtype=torch.int16, device='cuda')
    scales = room[:, :cols, :per].transpose(1, 2)
    for host in moe_hosts:
        got, got_sf = host.moe_dispatch_to_fp8(x, plan, out=(data, scales if max_m else scales[0]))
        flat, flat_sf = got.view(torch.uint8).view(-1, hidden), got_sf.reshape(-1, cols)
        assert torch.equal(flat[live], codes.view(torch.uint8)[choice[live] // topk]) and torch.equal(flat_sf[live], sf[choice[live] // topk])
        assert (flat[~live] == 0x11).all() and (flat_sf[~live] == 0x2222).all() and (room[:, cols] == 0x2222).all() and (room[:, :, per:] == 0x2222).all()
        fresh, fresh_sf = host.moe_dispatch_to_fp8(x, plan)
        assert torch.equal(fresh_sf.reshape(-1, cols)[live], flat_sf[live])


def test_rows_with_strides():
    """Views of wider tensors on both sides, and one token's row broadcast to all."""
    seed_all(3)
    plan, (_, token_rows, row_choices) = _plan(45, 4, 8, 8, None)
    choice = row_choices.long()
    live, of = choice >= 0, choice[choice >= 0] // 4
    x = torch.randn(45, 1024, device='cuda', dtype=torch.bfloat16)[:, 256:512]
    out = torch.zeros(row_choices.numel(), 768, dtype=torch.bfloat16, device='cuda')
    deep_gemm.moe_dispatch(x, plan, out=out[:, 128:384])
    assert torch.equal(out[live.cuda(), 128:384], x[of.cuda()]) and (out[:, :128] == 0).all() and (out[:, 384:] == 0).all()
    one = torch.randn(1, 256, device='cuda', dtype=torch.bfloat16).expand(45, 256)
    assert (deep_gemm.moe_dispatch(one, plan)[live.cuda()] == one[0]).all()
    y = torch.randn(row_choices.numel(), 512, device='cuda')[:, 64:320]
    total = torch.zeros(45, 300, device='cuda')
    deep_gemm.moe_combine(y, plan, out=total[:, 4:260])
    ref, size = oracle.moe_combine_ref(y.cpu(), token_rows)
    assert ((total[:, 4:260].cpu().double() - ref).abs() <= 5 * E * size + E * ref.abs()).all() and (total[:, :4] == 0).all() and (total[:, 260:] == 0).all()
    plan, (_, _, row_choices) = _plan(45, 4, 8, 8, 16)
    out = torch.zeros(8, 16, 768, dtype=torch.bfloat16, device='cuda')
    deep_gemm.moe_dispatch(x, plan, out=out[..., 256:512])
    live = row_choices >= 0
    assert torch.equal(out[..., 256:512][live.cuda()], x[(row_choices[live].long() // 4).cuda()])


# --------------------------------------------------------------------------------------------------------------- combine
def _combine_bound(ref, size, topk, dtype):
    err = (topk + 1) * E * size * (1 + 2 * topk * E)
    return err + HALF[dtype] * (ref.abs() + err)


@pytest.mark.parametrize('host', moe_hosts)
@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('hidden,dtype', [(8, torch.bfloat16), (1000, torch.bfloat16), (7168, torch.bfloat16), (4, torch.float32), (2052, torch.float32)])
def test_combine(host, layout, hidden, dtype):
    seed_all(hidden + 1)
    plan, (_, token_rows, row_choices) = _plan(*layout)
    rows = torch.randn(*row_choices.shape, hidden).to(dtype)
    rows[row_choices < 0] = NAN                                   # rows without a choice are not read
    weights = torch.rand(layout[0], layout[1]) * 2 - 0.5
    weights[token_rows < 0] = NAN                                 # nor do the weights of choices without a row count
    for w in (None, weights):
        out = host.moe_combine(rows.cuda(), plan, None if w is None else w.cuda())
        assert out.dtype == dtype and out.shape == (layout[0], hidden)
        ref, size = oracle.moe_combine_ref(rows.view(-1, hidden), token_rows, w)
        assert ((out.cpu().double() - ref).abs() <= _combine_bound(ref, size, layout[1], dtype)).all()


def test_combine_passes_what_is_not_finite_on():
    plan, (_, token_rows, _) = _plan(10, 2, 4, 4, None)
    rows = torch.ones(plan[2].numel(), 64, device='cuda', dtype=torch.bfloat16)
    rows[token_rows[3, 1].item(), 5], rows[token_rows[4, 0].item(), 6] = float('inf'), NAN
    out = deep_gemm.moe_combine(rows, plan).cpu()
    assert out[3, 5] == float('inf') and torch.isnan(out[4, 6])
    out[3, 5] = out[4, 6] = 2
    assert (out == 2).all()


# -------------------------------------------------------------------------------------------------------------- gradient
@pytest.mark.parametrize('host', moe_hosts)
@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('hidden,dtype', [(8, torch.bfloat16), (1000, torch.bfloat16), (7168, torch.bfloat16), (4, torch.float32), (2052, torch.float32)])
def test_combine_grad(host, layout, hidden, dtype):
    seed_all(hidden + 2)
    plan, (psum, token_rows, row_choices) = _plan(*layout)
    rows = torch.randn(*row_choices.shape, hidden).to(dtype)
    rows[row_choices < 0] = NAN
    g = torch.randn(layout[0], hidden).to(dtype)
    weights = torch.rand(layout[0], layout[1]) * 2 - 0.5
    weights[token_rows < 0] = NAN
    ref, ref_w, size = oracle.moe_combine_grad_ref(g, rows.view(-1, hidden), token_rows, weights)
    live, pad = row_choices.view(-1) >= 0, oracle.moe_padding(psum, row_choices.numel(), 256, layout[4])
    for zero in (False, True):
        out = torch.full(rows.shape, 7.0, dtype=dtype, device='cuda')
        got, got_w = host.moe_combine_grad(g.cuda(), rows.cuda(), plan, weights.cuda(), out=out, zero_padding=zero)
        assert got.data_ptr() == out.data_ptr() and got_w.dtype == torch.float32 and got_w.shape == weights.shape
        flat = got.cpu().view(-1, hidden)
        assert ((flat[live].double() - ref[live]).abs() <= (HALF[dtype] * (1 + E) + E) * ref[live].abs()).all()
        assert (flat[pad] == (0.0 if zero else 7.0)).all() and (flat[~live & ~pad] == 7.0).all()
        assert ((got_w.cpu().double() - ref_w).abs() <= (hidden / 32 + 40) * E * size).all()
        assert (got_w.cpu()[token_rows < 0] == 0).all()
    # without `out`, and over the rows themselves: the same bits
    fresh, fresh_w = host.moe_combine_grad(g.cuda(), rows.cuda(), plan, weights.cuda())
    mine = rows.cuda()
    same, same_w = host.moe_combine_grad(g.cuda(), mine, plan, weights.cuda(), out=mine)
    assert same.data_ptr() == mine.data_ptr() and torch.equal(same_w, got_w) and torch.equal(fresh_w, got_w)
    for t in (fresh, same):
        assert torch.equal(t.cpu().view(-1, hidden)[live], flat[live])


def test_gradients_against_differences():
    """combine is linear in the rows and in the weights: <dout, combine(y + d) - combine(y)> is <dy, d> for a d of any size. FP32, and the sums
    in 64 bits: every value passes at most 40 roundings of 2^-24 of terms whose magnitudes are summed beside."""
    seed_all(11)
    plan, (_, token_rows, row_choices) = _plan(40, 4, 16, 12, None)
    h = 260
    live = (row_choices >= 0).cuda()
    rows, w, g = torch.randn(row_choices.numel(), h, device='cuda'), torch.rand(40, 4, device='cuda'), torch.randn(40, h, device='cuda')
    dy, dw = deep_gemm.moe_combine_grad(g, rows, plan, w)
    dot = lambda a, b: (a.double() * b.double())  # noqa: E731
    d = torch.randn_like(rows)
    terms = dot(g, deep_gemm.moe_combine(rows + d, plan, w)) - dot(g, deep_gemm.moe_combine(rows, plan, w))
    terms_dy = dot(dy, d)[live]
    size = dot(g, deep_gemm.moe_combine(rows, plan, w)).abs().sum() + dot(g, deep_gemm.moe_combine(rows + d, plan, w)).abs().sum() + terms_dy.abs().sum()
    slack = sum(oracle.moe_combine_ref(t.cpu(), token_rows, w.cpu())[1].cuda().mul(g.abs()).sum() for t in (rows, rows + d))
    assert (terms.sum() - terms_dy.sum()).abs() <= 40 * E * (size + slack)
    dv = torch.randn_like(w)
    terms = dot(g, deep_gemm.moe_combine(rows, plan, w + dv)) - dot(g, deep_gemm.moe_combine(rows, plan, w))
    slack = sum(oracle.moe_combine_ref(rows.cpu(), token_rows, t.cpu())[1].cuda().mul(g.abs()).sum() for t in (w, w + dv))
    assert (terms.sum() - dot(dw, dv).sum()).abs() <= 40 * E * (dot(dw, dv).abs().sum() + 4 * slack)
    # the gradient of a dispatch is the sum over a token's rows
    x = torch.randn(40, h, device='cuda')
    dx = deep_gemm.moe_combine(rows, plan)
    forward = dot(deep_gemm.moe_dispatch(x, plan), rows)[live]
    slack = oracle.moe_combine_ref(rows.cpu(), token_rows)[1].cuda().mul(x.abs()).sum()
    assert (forward.sum() - dot(dx, x).sum()).abs() <= 40 * E * slack


# -------------------------------------------------------------------------------------------------- refusals and bad plans
def test_refusals():
    plan, _ = _plan(16, 2, 4, 4, None)
    masked, _ = _plan(16, 2, 4, 4, 8)
    x = torch.zeros(16, 64, dtype=torch.bfloat16, device='cuda')
    rows = torch.zeros(plan[2].numel(), 64, dtype=torch.bfloat16, device='cuda')
    w = torch.zeros(16, 2, device='cuda')
    for host in moe_hosts:
        bad = lambda match: pytest.raises(RuntimeError, match=match)  # noqa: E731
        with bad('contiguous 2-D int32 or int64'):
            host.moe_sort(torch.zeros(4, 4, dtype=torch.int64, device='cuda').t()[:, :2], 4)
        with bad('contiguous 2-D int32 or int64'):
            host.moe_sort(torch.zeros(4, 4, device='cuda'), 4)
        with bad('num_experts must be between 1 and 1024'):
            host.moe_sort(torch.zeros(4, 4, dtype=torch.int64, device='cuda'), 1025)
        with bad('max_m must be positive'):
            host.moe_sort(torch.zeros(4, 4, dtype=torch.int64, device='cuda'), 4, max_m=0)
        with bad('expert_alignment must be positive'):
            host.moe_sort(torch.zeros(4, 4, dtype=torch.int64, device='cuda'), 4, expert_alignment=0)
        with bad('too many rows'):
            host.moe_sort(torch.zeros(4, 4, dtype=torch.int64, device='cuda'), 1024, max_m=1 << 22)
        with bad('another number of tokens'):
            host.moe_dispatch(x[:15], plan)
        with bad('row-major 2-D BF16 or FP32'):
            host.moe_dispatch(x.half(), plan)
        with bad('16-byte boundaries'):
            host.moe_dispatch(torch.zeros(16, 65, dtype=torch.bfloat16, device='cuda')[:, 1:], plan)
        with bad('16-byte boundaries'):
            host.moe_combine(torch.zeros(rows.size(0), 60, dtype=torch.bfloat16, device='cuda'), plan)
        with bad('the type, the device and the row length of x'):
            host.moe_dispatch(x, plan, out=rows.float())
        for out in (rows[1:], rows[:1].expand(rows.shape), torch.zeros(4, 8, 64, dtype=torch.bfloat16, device='cuda')):
            with bad("a row for each of the layout's"):
                host.moe_dispatch(x, plan, out=out)
        with bad("a row for each of the layout's"):
            host.moe_dispatch(x, masked, out=torch.zeros(5, 8, 64, dtype=torch.bfloat16, device='cuda')[:4].transpose(0, 1).contiguous().transpose(0, 1))
        with bad('multiple of 32'):
            host.moe_dispatch_to_fp8(torch.zeros(16, 48, dtype=torch.bfloat16, device='cuda'), plan)
        with bad('E4M3 tensor of the row length'):
            host.moe_dispatch_to_fp8(x, plan, out=(rows, rows))
        with bad('the scales of out must be int16'):
            host.moe_dispatch_to_fp8(torch.zeros(16, 128, dtype=torch.bfloat16, device='cuda'), plan,
                                     out=(torch.zeros(rows.size(0), 128, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn),
                                          torch.zeros(rows.size(0), 2, dtype=torch.int16, device='cuda')))
        with bad("a row for each of the layout's"):
            host.moe_combine(rows, masked, w)
        with bad('float32 tensor with one weight per choice'):
            host.moe_combine(rows, plan, w[:, :1])
        with bad('float32 tensor with one weight per choice'):
            host.moe_combine(rows, plan, w.bfloat16())
        with bad(r'row-major \[tokens, hidden\]'):
            host.moe_combine(rows, plan, w, out=x.t())
        with bad('the type, the device and the row length of grad_out'):
            host.moe_combine_grad(x, rows.float(), plan, w)
        with bad('three contiguous int32 tensors'):
            host.moe_dispatch(x, (plan[0].long(), *plan[1:]))
        with bad('three contiguous int32 tensors'):
            host.moe_dispatch(x, (plan[0].cpu(), *plan[1:]))
        with bad('layout, token_rows, row_choices'):
            host.moe_dispatch(x, (plan[0][:3], plan[1], masked[2]))


def test_a_plan_with_rows_outside_the_layout():
    """The kernels check what they are given: such choices have no row."""
    plan, (_, token_rows, _) = _plan(16, 2, 4, 4, None)
    rows_total = plan[2].numel()
    broken = plan[1].clone()
    broken[2, 0], broken[3, 1], broken[4, 0] = rows_total, -5, 2 ** 31 - 1
    layout = plan[0].clone()
    layout[1], layout[2] = -3, 2 ** 31 - 300
    x = torch.randn(16, 64, device='cuda')
    y = deep_gemm.moe_dispatch(x, (layout, broken, plan[2]), out=torch.zeros(rows_total, 64, device='cuda'), zero_padding=True)
    keep = (broken >= 0) & (broken < rows_total)
    out = deep_gemm.moe_combine(y, (layout, broken, plan[2]))
    assert torch.equal(out, x * keep.sum(1, keepdim=True))
    _, dw = deep_gemm.moe_combine_grad(x, y, (layout, broken, plan[2]), torch.ones(16, 2, device='cuda'), zero_padding=True)
    assert ((dw != 0) == keep).all()
    q, sf = deep_gemm.moe_dispatch_to_fp8(x.bfloat16(), (layout, broken, plan[2]))
    assert q.shape == (rows_total, 64)
    torch.cuda.synchronize()


@pytest.mark.parametrize('topk', [0, 2])
def test_no_tokens(topk):
    idx = torch.empty(0, topk, dtype=torch.int64, device='cuda')
    for max_m in (None, 4):
        plan = deep_gemm.moe_sort(idx, 4, max_m=max_m)
        x = torch.empty(0, 64, dtype=torch.bfloat16, device='cuda')
        y = deep_gemm.moe_dispatch(x, plan, zero_padding=True)
        assert y.shape == (*plan[2].shape, 64) and (y == 0).all()
        deep_gemm.moe_dispatch_to_fp8(x, plan)
        assert deep_gemm.moe_combine(y, plan).shape == (0, 64)
        dy, dw = deep_gemm.moe_combine_grad(x, y, plan, torch.empty(0, topk, device='cuda'), zero_padding=True)
        assert dy.shape == y.shape and dw.shape == (0, topk) and (dy == 0).all()


def test_zeros_spare_the_rows_that_hold_a_choice():
    """Whatever alignment is given: groups on multiples of 32, zeros up to the next multiple of 256."""
    plan, (psum, _, row_choices) = _plan(60, 3, 8, 8, None, alignment=32)
    x = torch.randn(60, 64, device='cuda')
    out = torch.full((row_choices.numel(), 64), 7.0, device='cuda')
    deep_gemm.moe_dispatch(x, plan, out=out, zero_padding=True)
    live, pad = row_choices >= 0, oracle.moe_padding(psum, row_choices.numel(), 256)
    assert torch.equal(out.cpu()[live], x.cpu()[row_choices[live].long() // 3]) and (out.cpu()[pad & ~live] == 0).all()
    assert (out.cpu()[~pad & ~live] == 7).all()
    g, w = torch.randn(60, 64, device='cuda'), torch.rand(60, 3, device='cuda')
    dy, _ = deep_gemm.moe_combine_grad(g, out, plan, w, zero_padding=True)
    assert torch.equal(dy.cpu()[live], (w.view(-1, 1) * g.repeat_interleave(3, 0)).cpu()[row_choices[live].long()]) and (dy.cpu()[pad & ~live] == 0).all()


def test_no_choices_at_all():
    idx, x = torch.empty(5, 0, dtype=torch.int64, device='cuda'), torch.randn(5, 64, device='cuda')
    for max_m in (None, 4):
        plan = deep_gemm.moe_sort(idx, 3, max_m=max_m)
        y = deep_gemm.moe_dispatch(x, plan, zero_padding=True)
        assert (y == 0).all() and (deep_gemm.moe_combine(y, plan) == 0).all()
        deep_gemm.moe_dispatch_to_fp8(x.bfloat16(), plan)
        _, dw = deep_gemm.moe_combine_grad(x, y, plan, torch.empty(5, 0, device='cuda'))
        assert dw.shape == (5, 0)


def test_tokens_without_choices():
    idx = torch.full((9, 3), -1, device='cuda')
    plan = deep_gemm.moe_sort(idx, 4)
    x = torch.randn(9, 64, device='cuda')
    y = deep_gemm.moe_dispatch(x, plan, out=torch.full((plan[2].numel(), 64), 7.0, device='cuda'), zero_padding=True)
    assert (y == 7).all() and (deep_gemm.moe_combine(y, plan, torch.ones(9, 3, device='cuda')) == 0).all()
    dy, dw = deep_gemm.moe_combine_grad(x, y, plan, torch.ones(9, 3, device='cuda'), out=y)
    assert (dy == 7).all() and (dw == 0).all()


# --------------------------------------------------------------------------------------------------- streams and graphs
def test_another_stream_and_a_captured_run():
    """The whole way there and back on a stream of its own, then captured once and replayed on other choices."""
    seed_all(5)
    experts, tokens, topk, h = 8, 50, 3, 512
    idx, x, w = _choices(tokens, topk, experts, 1).cuda(), torch.randn(tokens, h, device='cuda').bfloat16(), torch.rand(tokens, topk, device='cuda')

    def way(i, v, u):
        plan = deep_gemm.moe_sort(i, experts)
        y = deep_gemm.moe_dispatch(v, plan, zero_padding=True)
        q = deep_gemm.moe_dispatch_to_fp8(v, plan)
        out = deep_gemm.moe_combine(y, plan, u)
        return (*plan, out, *deep_gemm.moe_combine_grad(v, y, plan, u), *q)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = way(idx, x, w)
    side.synchronize()
    here = way(idx, x, w)
    for a, b in itertools.islice(zip(there, here), 4):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = way(idx, x, w)
    for seed in (2, 3):
        idx.copy_(_choices(tokens, topk, experts, seed))
        x.copy_(torch.randn(tokens, h))
        w.copy_(torch.rand(tokens, topk))
        graph.replay()
        fresh = way(idx.clone(), x.clone(), w.clone())
        live = fresh[2] >= 0
        for k, (a, b) in enumerate(zip(held, fresh)):
            if k in (4, 6, 7):
                a, b = a.view(torch.int16 if k != 6 else torch.uint8)[live], b.view(torch.int16 if k != 6 else torch.uint8)[live]
            assert torch.equal(a, b), k


def test_two_streams_at_once_and_launches_that_do_not_overlap():
    """Calls in turn on two streams, nothing waited for in between, a sort over a cluster and the scales' second launch among them; then the same
    one after the other with every launch waiting for the one in front of it."""
    sizes = ((2500, 4, 16, 2048), (64, 8, 32, 512))
    inputs = [[(_choices(t, k, e, seed).cuda(), torch.randn(t, h, device='cuda').bfloat16(), torch.rand(t, k, device='cuda')) for seed in range(4)] for t, k, e, h in sizes]

    def way(n, i, x, w):
        plan = deep_gemm.moe_sort(i, sizes[n][2])
        y = deep_gemm.moe_dispatch(x, plan, out=torch.zeros(plan[2].numel(), x.size(1), dtype=x.dtype, device='cuda'))
        q, sf = deep_gemm.moe_dispatch_to_fp8(x, plan)
        live = plan[2] >= 0
        return (*plan, y, deep_gemm.moe_combine(y, plan, w), *deep_gemm.moe_combine_grad(x, y, plan, w, out=y.clone()),
                torch.where(live[:, None], q.view(torch.uint8), 0), torch.where(live[:, None], sf, 0))

    want = [[way(n, *case) for case in inputs[n]] for n in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for k in range(4):
        for n, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[n].append(way(n, *inputs[n][k]))
    torch.cuda.synchronize()
    lib = deep_gemm._lib.lib()
    lib.dg_set_overlap_launches(0)
    try:
        alone = [[way(n, *case) for case in inputs[n]] for n in range(2)]
    finally:
        lib.dg_set_overlap_launches(1)
    for n in range(2):
        for k in range(4):
            for a, b, c in zip(want[n][k], got[n][k], alone[n][k]):
                assert torch.equal(a, b) and torch.equal(a, c)


def test_offsets_beyond_32_bits():
    """Rows behind 2^32 bytes: 600000 rows of 7168 bytes, the last expert's at the end."""
    free = torch.cuda.mem_get_info()[0]
    if free < 24 << 30:
        pytest.skip('needs 24 GB')
    max_m, h = 300000, 7168
    idx = torch.tensor([[1, 0], [1, -1], [0, 1]], device='cuda')
    plan = deep_gemm.moe_sort(idx, 2, max_m=max_m)
    x = torch.randn(3, h, device='cuda').bfloat16()
    q, sf = deep_gemm.moe_dispatch_to_fp8(x, plan)
    ref, ref_sf = deep_gemm.cast_to_fp8(x)
    assert torch.equal(q[1, :3].view(torch.uint8), ref.view(torch.uint8)) and torch.equal(sf[1, :3], ref_sf)
    del q, sf
    y = deep_gemm.moe_dispatch(x, plan)
    assert torch.equal(y[1, :3], x) and torch.equal(y[0, :2], x[[0, 2]])
    assert torch.equal(deep_gemm.moe_combine(y, plan), x * torch.tensor([[2], [1], [2]], device='cuda'))
    dy, dw = deep_gemm.moe_combine_grad(x, y, plan, torch.ones(3, 2, device='cuda'), out=y)
    assert torch.equal(dy[1, :3], x) and dw[1, 1] == 0


# ------------------------------------------------------------------------------------------------------ as they are used
# Tolerances of the two layers, worst case: every BF16 tensor on the way adds 2^-8 of its value (the GEMM's result, the gradients of the rows),
# a GEMM over K terms adds K 2^-23 of the sum of its terms' magnitudes, and each is carried on by magnitudes through what follows.
U, F = 2.0 ** -8, 2.0 ** -23


@pytest.mark.parametrize('max_m', [None, 64])
def test_an_expert_layer_forward(max_m):
    """choices -> FP8 rows -> grouped GEMM -> weighted sum, against 64 bits on the dequantised operands."""
    seed_all(21)
    tokens, topk, experts, h, n = 100, 4, 8, 512, 384
    idx = _choices(tokens, topk, experts + 4, 3)
    x = torch.randn(tokens, h).bfloat16()
    wr = torch.rand(tokens, topk)
    weights = torch.randn(experts, n, h) * h ** -0.5
    w4 = deep_gemm.cast_to_fp4(weights.cuda())
    w_values = deep_gemm.cast_from_fp4(w4, out_dtype=torch.float32).cpu().double()
    plan = deep_gemm.moe_sort(idx.cuda(), experts, max_m=max_m)
    a = deep_gemm.moe_dispatch_to_fp8(x.cuda(), plan)
    y = torch.full((*plan[2].shape, n), NAN, dtype=torch.bfloat16, device='cuda')
    if max_m:
        deep_gemm.m_grouped_fp8_fp4_gemm_nt_masked(a, w4, y, plan[0], tokens * topk // experts)
    else:
        deep_gemm.m_grouped_fp8_fp4_gemm_nt_contiguous(a, w4, y, plan[0])
    out = deep_gemm.moe_combine(y, plan, wr.cuda())
    assert deep_gemm.device_status() == 0
    x_values = oracle.swiglu_quant_ref(x, swiglu=False)[3].double()
    ref, err, size = (torch.zeros(tokens, n, dtype=torch.float64) for _ in range(3))
    for e in range(experts):
        w = ((idx == e) * wr.double()).sum(1, keepdim=True)
        value, magnitude = x_values @ w_values[e].t(), x_values.abs() @ w_values[e].abs().t()
        ref += w * value
        size += w * value.abs()
        err += w * (U * value.abs() + (1 + U) * h * F * magnitude)
    err += (topk + 1) * E * (size + err)
    err += U * (ref.abs() + err)
    assert ((out.cpu().double() - ref).abs() <= err).all()


def test_an_expert_layer_backward():
    """BF16 rows through one grouped GEMM; the result and the gradients of the input, of the experts' weights and of the routing weights against
    64 bits (the gradients by autograd) on the same BF16 values."""
    seed_all(22)
    tokens, topk, experts, h, n = 90, 3, 6, 256, 320
    idx = _choices(tokens, topk, experts + 2, 4)
    x, weights, wr = torch.randn(tokens, h).bfloat16(), (torch.randn(experts, n, h) * h ** -0.5).bfloat16(), torch.rand(tokens, topk)
    g = torch.randn(tokens, n).bfloat16()
    plan = deep_gemm.moe_sort(idx.cuda(), experts)
    rows = plan[2].numel()
    a = deep_gemm.moe_dispatch(x.cuda(), plan, zero_padding=True)
    y = torch.empty(rows, n, dtype=torch.bfloat16, device='cuda')
    deep_gemm.m_grouped_bf16_gemm_nt_contiguous(a, weights.cuda(), y, plan[0])
    out = deep_gemm.moe_combine(y, plan, wr.cuda())
    dy, dr = deep_gemm.moe_combine_grad(g.cuda(), y, plan, wr.cuda(), zero_padding=True)
    da = torch.empty(rows, h, dtype=torch.bfloat16, device='cuda')
    deep_gemm.m_grouped_bf16_gemm_nn_contiguous(dy, weights.cuda(), da, plan[0])
    dx = deep_gemm.moe_combine(da, plan)
    dw = torch.empty(experts, n, h, dtype=torch.float32, device='cuda')
    deep_gemm.k_grouped_bf16_gemm_tn_contiguous(dy, a, dw, None, plan[0])
    assert deep_gemm.device_status() == 0
    x64, w64, r64, g64 = (t.double().requires_grad_() for t in (x, weights, wr, g))
    per_expert = [((idx == e) * r64).sum(1, keepdim=True) for e in range(experts)]
    ref = sum(r * (x64 @ w64[e].t()) for e, r in enumerate(per_expert))
    ref.backward(g64.detach())
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.float64)  # noqa: E731
    err_out, err_dx, err_dw, err_dr = zeros(tokens, n), zeros(tokens, h), zeros(experts, n, h), zeros(tokens, topk)
    with torch.no_grad():
        for e, r in enumerate(per_expert):
            has = (idx == e).any(1, keepdim=True)
            value, magnitude = x64 @ w64[e].t(), x64.abs() @ w64[e].abs().t()
            y_err = U * value.abs() + (1 + U) * h * F * magnitude
            err_out += r * (y_err + (topk + 1) * E * (value.abs() + y_err))
            back, back_magnitude = (r * g64) @ w64[e], (r * g64).abs() @ w64[e].abs()
            da_err = (1 + U) * (U + F + n * F * (1 + 2 * U)) * back_magnitude + U * back.abs()
            err_dx += da_err + (topk + 1) * E * (back.abs() + da_err)
            err_dw[e] = (U + F + tokens * F * (1 + 2 * U)) * ((r * g64).abs().t() @ x64.abs())
            dr_err = (g64.abs() * y_err).sum(1, keepdim=True) + (n / 32 + 40) * E * (g64.abs() * (value.abs() + y_err)).sum(1, keepdim=True)
            err_dr += torch.where(idx == e, dr_err, 0.0)
            assert (has | (r == 0)).all()
        err_out += U * (ref.abs() + err_out)
        err_dx += U * (x64.grad.abs() + err_dx)
        for name, got, want, err in (('out', out, ref, err_out), ('dx', dx, x64.grad, err_dx), ('dw', dw, w64.grad, err_dw), ('dr', dr, r64.grad, err_dr)):
            assert ((got.cpu().double() - want).abs() <= err).all(), name


def test_both_host_layers_give_the_same_bits():
    seed_all(30)
    idx, x = _choices(200, 4, 16, 6).cuda(), torch.randn(200, 288, device='cuda').bfloat16()
    layer = python_layer('moe_ops')
    for max_m in (None, 32):
        p, q = deep_gemm.moe_sort(idx, 12, max_m=max_m), layer.moe_sort(idx, 12, max_m=max_m)
        assert all(torch.equal(a, b) for a, b in zip(p, q))
        live = p[2] >= 0
        for a, b in zip(deep_gemm.moe_dispatch_to_fp8(x, p), layer.moe_dispatch_to_fp8(x, q)):
            assert a.stride() == b.stride() and torch.equal(a.view(torch.uint8 if a.element_size() == 1 else torch.int16)[live],
                                                            b.view(torch.uint8 if b.element_size() == 1 else torch.int16)[live])
