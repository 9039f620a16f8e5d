"""SwiGLU with its input kept in 8 bits, its gradient, 8-bit operands along the rows and the way back, against the CPU oracle (oracle/layers.py), and an
expert layer's training step with all of them.

Tolerances, e = 2^-24. Everything that does not depend on the exponential is compared bit for bit. Gradient of SwiGLU, p = 1 / (1 + e^-l): the fast
exponential is within (2 + 1.173 |l|) ulp, the reciprocal within 2 ulp: p within d p, d = (2 (2 + 1.2 |l|) + 8) e. dx_r = g w l p: d and four roundings.
dx_l = g w r (p + l p (1 - p)): the terms move by d p and 3 d |l| p (1 - p carries d p too), and a few roundings. p stays at the least
normal number where it is below: it moves by at most t = 2^-126 beyond that, dx_r by t |g w l| and dx_l by t |g w r| (1 + |l|). dx is rounded to BF16 once, 2^-8 of the value.
dw: a sum whose terms pass at most H / 32 + 60 additions."""

import os
import subprocess
import sys
import textwrap

import pytest
import torch

import deep_gemm
import oracle
from both_hosts import python_layer, quant_hosts
from helpers import seed_all

pytestmark = pytest.mark.gpu

E, U = 2.0 ** -24, 2.0 ** -8
BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn
NAN, INF = float('nan'), float('inf')


def _layout(sizes, alignment=128, behind=0):
    """(rows in all, ends of the groups, bool rows that hold a value, bool rows of the padding)"""
    total, psum = oracle.make_psum_layout(list(sizes), alignment)
    live, pad = torch.zeros(total + behind, dtype=torch.bool), torch.zeros(total + behind, dtype=torch.bool)
    for size, p in zip(sizes, psum):
        live[p - size:p] = True
        pad[p:oracle.align(p, alignment)] = True
    return total + behind, psum, live, pad


def _bytes(t):
    return t.view(torch.uint8).cpu()


def _pair(x, device='cuda'):
    """The 8-bit pair of BF16 or FP32 rows, made by the oracle."""
    codes, byte, values = oracle.cast_fp8_ref(x, 1)
    sf = oracle.pack_scales(byte, 1)
    out = torch.empty_strided(sf.shape, (1, sf.size(0)), dtype=torch.int16)
    return (codes.contiguous().view(FP8).to(device), out.copy_(sf).to(device)), values


# --------------------------------------------------------------------------------------------------------------- forward
@pytest.mark.parametrize('host', quant_hosts)
@pytest.mark.parametrize('tokens,hidden', [(1, 128), (33, 256), (64, 2048), (100, 1408)])
def test_checkpoint(host, tokens, hidden):
    seed_all(tokens)
    x, w = (torch.randn(tokens, 2 * hidden) * 3).bfloat16().cuda(), torch.rand(tokens, device='cuda')
    for weights in (None, w):
        for clamp in (None, 2.0):
            (out, sf), (kept, kept_sf) = host.swiglu_apply_weight_to_fp8_with_checkpoint(x, weights, clamp_value=clamp)
            want, want_sf = deep_gemm.swiglu_apply_weight_to_fp8(x, weights, clamp_value=clamp)
            assert torch.equal(_bytes(out), _bytes(want)) and torch.equal(sf, want_sf)
            want, want_sf = deep_gemm.cast_to_fp8(x)
            assert kept.dtype == FP8 and torch.equal(_bytes(kept), _bytes(want)) and torch.equal(kept_sf, want_sf) and (kept_sf.stride(0) == 1 or tokens == 1)


@pytest.mark.parametrize('host', quant_hosts)
def test_checkpoint_of_a_layout(host):
    """Rows without a value are left as they were."""
    seed_all(1)
    rows, psum, live, _ = _layout([300, 0, 129, 1, 0], 128, behind=40)
    layout = torch.tensor(psum, dtype=torch.int32, device='cuda')
    x, w = torch.randn(rows, 1024).bfloat16().cuda(), torch.rand(rows, device='cuda')
    empty = lambda width: (torch.full((rows, width), 0x11, dtype=torch.uint8, device='cuda').view(FP8),  # noqa: E731
                           torch.full((width // 64, rows), 0x2222, dtype=torch.int16, device='cuda').t())
    out = empty(512), empty(1024)
    got = host.swiglu_apply_weight_to_fp8_with_checkpoint(x, w, layout, 3.0, out=out)
    want = deep_gemm.swiglu_apply_weight_to_fp8(x, w, layout, 3.0), deep_gemm.cast_to_fp8(x, layout)
    for (q, sf), (q0, sf0), (q1, sf1) in zip(got, out, want):
        assert q.data_ptr() == q0.data_ptr() and sf.data_ptr() == sf0.data_ptr()
        assert torch.equal(_bytes(q)[live], _bytes(q1)[live]) and torch.equal(sf.cpu()[live], sf1.cpu()[live])
        assert (_bytes(q)[~live] == 0x11).all() and (sf.cpu()[~live] == 0x2222).all()


# -------------------------------------------------------------------------------------------------------------- gradient
def _check_grad(g, x, values, w=None, clamp=None, live=None, host=deep_gemm, **kw):
    """x: what the call gets; values: FP32 of it."""
    dx, dw = host.swiglu_apply_weight_grad(g.cuda(), x, None if w is None else w.cuda(), clamp_value=clamp, **kw)
    tokens, hidden = g.shape
    assert dx.dtype == BF16 and dx.shape == (tokens, 2 * hidden)
    dl, dr, dw_ref, (g64, l, r, p, w64) = oracle.swiglu_grad_ref(g, values, w, clamp)
    live = torch.ones(tokens, dtype=torch.bool) if live is None else live
    d = (2 * (2 + 1.2 * l.abs()) + 8) * E
    silu = l.abs() * p
    tiny = 2.0 ** -126
    err_r = (g64 * w64).abs() * (silu * (d + 5 * E) + tiny * l.abs())
    err_l = (g64 * w64 * r).abs() * ((d + 6 * E) * p + (3 * d + 8 * E) * silu + tiny * (1 + l.abs()))
    for got, want, err in ((dx[:, :hidden], dl, err_l), (dx[:, hidden:], dr, err_r)):
        bound = err + U * (want.abs() + err) + 2.0 ** -130
        assert ((got.cpu().double() - want).abs() <= bound)[live].all()
    if w is None:
        assert dw is None
    else:
        size = (g64 * silu * r).abs()
        bound = (size * (d + 4 * E) + tiny * (g64 * l * r).abs()).sum(1) + (hidden / 32 + 60) * E * size.sum(1) + 2.0 ** -130
        assert dw.dtype == torch.float32 and dw.shape == w.shape
        assert ((dw.cpu().double().view(-1) - dw_ref).abs() <= bound)[live].all() and (dw.cpu().view(-1)[~live] == 0).all()
    return dx, dw


@pytest.mark.parametrize('host', quant_hosts)
@pytest.mark.parametrize('tokens,hidden', [(1, 128), (33, 256), (77, 2048), (65, 1408), (4, 4224), (320, 640)])
@pytest.mark.parametrize('kept', [False, True])
def test_gradient(host, tokens, hidden, kept):
    seed_all(hidden)
    x, g, w = (torch.randn(tokens, 2 * hidden) * 3).bfloat16(), torch.randn(tokens, hidden).bfloat16(), torch.rand(tokens, 1) * 2 - 0.5
    arg, values = _pair(x) if kept else (x.cuda(), x.float())
    for weights in (None, w):
        for clamp in (None, 2.0, 0.0):
            first = _check_grad(g, arg, values, weights, clamp, host=host)
    again = host.swiglu_apply_weight_grad(g.cuda(), arg, w.cuda(), clamp_value=0.0)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize('host', quant_hosts)
@pytest.mark.parametrize('kept', [False, True])
@pytest.mark.parametrize('sizes,alignment,behind', [([300, 0, 129, 1, 0], 128, 40), ([0, 0], 256, 33), ([31, 33, 64], 32, 5), ([1000], 256, 0)])
def test_gradient_of_a_layout(host, kept, sizes, alignment, behind):
    seed_all(alignment)
    rows, psum, live, pad = _layout(sizes, alignment, behind)
    layout = torch.tensor(psum, dtype=torch.int32, device='cuda')
    x, g, w = torch.randn(rows, 512).bfloat16(), torch.randn(rows, 256).bfloat16(), torch.rand(rows)
    arg, values = _pair(x) if kept else (x.cuda(), x.float())
    # what rows without a value hold does not matter
    g[~live], w[~live] = NAN, INF
    if kept:
        _bytes_of = arg[0].view(torch.uint8)
        _bytes_of[~live.cuda()] = 0x7F
        arg[1][~live.cuda()] = -1
    else:
        arg[~live.cuda()] = NAN
    for zero in (False, True):
        out = torch.full((rows, 512), 7.0, dtype=BF16, device='cuda')
        dx, dw = _check_grad(g, arg, values, w, 1.5, live, host, psum_num_tokens_per_expert=layout, expert_alignment=alignment, out=out, zero_padding=zero)
        assert dx.data_ptr() == out.data_ptr()
        dx = dx.cpu()
        assert (dx[pad] == (0.0 if zero else 7.0)).all() and (dx[~live & ~pad] == 7.0).all()


def test_gradient_at_the_ends():
    """Logits far out, a NaN, and the clamp's edge, where the gradient passes."""
    x = torch.tensor([-1e4, -100.0, -88.5, -40.0, -1.278, 0.0, -0.0, 1e-30, 1.5, 40.0, 100.0, 1e4] + [0.0] * 116).bfloat16()
    x = torch.cat((x, torch.linspace(-2, 2, 128).bfloat16())).view(1, 256).repeat(3, 1)
    g = torch.randn(3, 128).bfloat16()
    _check_grad(g, x.cuda(), x.float(), torch.rand(3))
    _check_grad(g, x.cuda(), x.float(), torch.rand(3), 1.5)
    x[1, 5] = NAN
    for clamp in (None, 1.0):
        dx, dw = deep_gemm.swiglu_apply_weight_grad(g.cuda(), x.cuda(), torch.ones(3, device='cuda'), clamp_value=clamp)
        # (x_r there is -1.92: the clamp cuts it off)
        assert dx[1, 5].isnan() and (dx[1, 133] == 0 if clamp else dx[1, 133].isnan())
        assert dw[1].isnan() and dx.isnan().sum() == (1 if clamp else 2) and dw.isnan().sum() == 1


def test_gradient_against_differences():
    seed_all(4)
    x, g, w = torch.randn(2, 256).bfloat16(), torch.randn(2, 128).bfloat16(), torch.rand(2)
    dx, dw = deep_gemm.swiglu_apply_weight_grad(g.cuda(), x.cuda(), w.cuda())

    def loss(x, w):
        l, r = x[:, :128], x[:, 128:]
        return float((g.double() * l * torch.sigmoid(l) * r * w[:, None]).sum())
    for t, c in ((0, 3), (1, 127), (0, 128), (1, 200)):
        step, ws = torch.zeros(2, 256, dtype=torch.float64), torch.zeros(2, dtype=torch.float64)
        step[t, c], ws[t] = 1e-5, 1e-5
        d = (loss(x.double() + step, w.double()) - loss(x.double() - step, w.double())) / 2e-5
        assert abs(d - float(dx[t, c])) <= U * abs(d) + 1e-5           # (a rounding to BF16; 1e-9 from the difference, 1e-6 from FP32)
        d = (loss(x.double(), w.double() + ws) - loss(x.double(), w.double() - ws)) / 2e-5
        assert abs(d - float(dw[t])) <= 1e-4


# ------------------------------------------------------------------------------------------------------ along the rows
@pytest.mark.parametrize('host', quant_hosts)
@pytest.mark.parametrize('rows,cols', [(1, 32), (31, 64), (32, 96), (33, 256), (64, 288), (65, 544), (200, 1120), (257, 2048)])
@pytest.mark.parametrize('kept', [False, True])
def test_cast_down_the_rows(host, rows, cols, kept):
    seed_all(rows)
    x = (torch.randn(rows, cols) * torch.exp(2 * torch.randn(1, cols))).bfloat16()
    x[:, 5] = 0
    x[:, 7] *= 1e-12
    arg, values = _pair(x) if kept else (x.cuda(), x.float())
    for floor in (1e-4, 0.0, 3.0):
        q, sf = host.cast_to_fp8(arg, mn_major=True, min_amax=floor)
        codes, byte, want = oracle.cast_fp8_ref(values, 0, floor)
        assert q.dtype == FP8 and q.shape == x.shape and torch.equal(_bytes(q), codes)
        assert sf.dtype == torch.int16 and sf.shape == ((rows + 63) // 64, cols) and torch.equal(sf.cpu(), oracle.pack_scales(byte, 0))
        for dtype in (BF16, torch.float32):
            back = host.cast_from_fp8((q, sf), dtype, mn_major=True)
            assert back.dtype == dtype and torch.equal(back.cpu(), want.to(dtype))


@pytest.mark.parametrize('host', quant_hosts)
@pytest.mark.parametrize('kept', [False, True])
@pytest.mark.parametrize('sizes,alignment,behind', [([300, 0, 129, 1, 0], 128, 40), ([0, 0], 256, 33), ([31, 33, 64], 64, 5), ([1000], 256, 0), ([5] * 70, 64, 0)])
def test_cast_of_a_layout(host, kept, sizes, alignment, behind):
    seed_all(alignment)
    rows, psum, live, pad = _layout(sizes, alignment, behind)
    layout = torch.tensor(psum, dtype=torch.int32, device='cuda')
    x = torch.randn(rows, 320).bfloat16()
    arg, values = _pair(x) if kept else (x.cuda(), x.float())
    if kept:
        arg[0].view(torch.uint8)[~live.cuda()] = 0x7F
        arg[1][~live.cuda()] = -1
    else:
        arg[~live.cuda()] = NAN
    q, sf = host.cast_to_fp8(arg, layout, alignment, mn_major=True)
    codes, byte, _ = oracle.cast_fp8_ref(values, 0, valid=live)
    written = live | pad
    assert torch.equal(_bytes(q)[written], codes[written])
    blocks = torch.nn.functional.pad(written, (0, -rows % 32)).view(-1, 32).any(1)
    got = torch.stack((sf.cpu().int() & 255, (sf.cpu().int() >> 8) & 255), 1).flatten(0, 1)[:len(blocks)]
    assert torch.equal(got[blocks], byte.int()[blocks])


def test_cast_of_groups_strides_and_offsets():
    seed_all(6)
    x = torch.randn(3, 100, 160).bfloat16().cuda()
    wide = torch.randn(3, 130, 320, device='cuda').bfloat16()
    wide[:, 20:120, 32:192] = x
    for host in quant_hosts:
        for arg in (x, wide[:, 20:120, 32:192]):
            q, sf = host.cast_to_fp8(arg, mn_major=True)
            assert q.shape == x.shape and sf.shape == (3, 2, 160)
            for i in range(3):
                q1, sf1 = host.cast_to_fp8(x[i], mn_major=True)
                assert torch.equal(_bytes(q[i]), _bytes(q1)) and torch.equal(sf[i], sf1)
            back = host.cast_from_fp8((q, sf), mn_major=True)
            assert all(torch.equal(back[i], host.cast_from_fp8((q[i], sf[i]), mn_major=True)) for i in range(3))
        # 8-bit rows of a masked layout, as the dispatch writes them, and with strides
        pairs = [host.cast_to_fp8(x[i]) for i in range(3)]
        codes = torch.zeros(3, 100, 200, dtype=torch.uint8, device='cuda')
        codes[:, :, 8:168] = torch.stack([p[0].view(torch.uint8) for p in pairs])
        scales = torch.zeros(3, 5, 130, dtype=torch.int16, device='cuda')
        scales[:, 1:4, 11:111] = torch.stack([p[1].t() for p in pairs])
        pair = codes[:, :, 8:168].view(FP8), scales[:, 1:4, 11:111].transpose(1, 2)
        q, sf = host.cast_to_fp8(pair, mn_major=True)
        back = host.cast_from_fp8(pair)
        for i in range(3):
            q1, sf1 = host.cast_to_fp8(pairs[i], mn_major=True)
            assert torch.equal(_bytes(q[i]), _bytes(q1)) and torch.equal(sf[i], sf1) and torch.equal(back[i], host.cast_from_fp8(pairs[i]))
        q, sf = host.cast_to_fp8(torch.zeros(0, 5, 32, dtype=BF16, device='cuda'), mn_major=True)
        assert q.shape == (0, 5, 32) and sf.shape == (0, 1, 32) and host.cast_from_fp8((q, sf), mn_major=True).shape == (0, 5, 32)
        q, sf = host.cast_to_fp8(torch.zeros(0, 32, dtype=BF16, device='cuda'), mn_major=True)
        assert q.shape == (0, 32) and sf.shape == (0, 32)


def test_what_is_not_finite_shows():
    x = torch.randn(64, 64).bfloat16()
    x[3, 5], x[40, 5], x[7, 9] = NAN, INF, -INF
    q, sf = deep_gemm.cast_to_fp8(x.cuda(), mn_major=True)
    byte = torch.stack((sf.cpu().int() & 255, (sf.cpu().int() >> 8) & 255), 1).flatten(0, 1)
    assert byte[0, 5] == byte[1, 5] == byte[0, 9] == 255 and (byte == 255).sum() == 3
    back = deep_gemm.cast_from_fp8((q, sf), torch.float32, mn_major=True).cpu()
    assert back[:, 5].isnan().all() and back[:32, 9].isnan().all() and not back[32:, 9].isnan().any()
    # 8-bit rows with a NaN code, a NaN scale, and values beyond FP32
    codes, sf = torch.full((64, 64), 0x38, dtype=torch.uint8), torch.full((64, 1), 0x7F7F, dtype=torch.int16)
    codes[1, 3], sf[2, 0], sf[40, 0], codes[40] = 0x7F, 0x7F | -256, 0x7F | (254 - 256) * 256, 0x7E
    q, out = deep_gemm.cast_to_fp8((codes.cuda().view(FP8), sf.cuda()), mn_major=True)
    byte = torch.stack((out.cpu().int() & 255, (out.cpu().int() >> 8) & 255), 1).flatten(0, 1)
    assert byte[0, 3] == 255 and (byte[0, 32:] == 255).all() and (byte[1, 32:] == 255).all() and (byte == 255).sum() == 65
    back = deep_gemm.cast_from_fp8((codes.cuda().view(FP8), sf.cuda()), torch.float32).cpu()
    assert back[1, 3].isnan() and back[2, 32:].isnan().all() and (back[40, 32:] == INF).all() and (back[40, :32] == 448).all()


def test_all_codes_and_scales_come_back():
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    byte = torch.arange(256, dtype=torch.int32)
    sf = torch.where(byte >= 128, byte * 257 - 65536, byte * 257).to(torch.int16)[:, None].expand(256, 4).t().contiguous().t()
    want = codes.view(FP8).double() * torch.where(byte == 255, NAN, torch.exp2((byte - 127).double()))[:, None]
    for host in quant_hosts:
        for dtype in (torch.float32, BF16):
            got = host.cast_from_fp8((codes.cuda().view(FP8), sf.cuda()), dtype).cpu()
            assert torch.equal(got.nan_to_num(7e30), want.to(torch.float32).to(dtype).nan_to_num(7e30))


@pytest.mark.parametrize('host', quant_hosts)
def test_cast_along_the_rows_with_a_least_amax(host):
    seed_all(9)
    x = (torch.randn(50, 96) * 1e-8).bfloat16()
    x[3] = 0
    for floor in (0.0, 1e-9, 1e-4, 5.0):
        q, sf = host.cast_to_fp8(x.cuda(), min_amax=floor)
        codes, byte, _ = oracle.cast_fp8_ref(x, 1, floor)
        assert torch.equal(_bytes(q), codes) and torch.equal(sf.cpu(), oracle.pack_scales(byte, 1))
    assert torch.equal(_bytes(host.cast_to_fp8(x.cuda())[0]), _bytes(host.cast_to_fp8(x.cuda(), min_amax=1e-4)[0]))
    one = torch.randn(1, 64, device='cuda').bfloat16()
    q, sf = host.cast_to_fp8(one.expand(40, 64))
    assert torch.equal(_bytes(q), _bytes(host.cast_to_fp8(one)[0]).expand(40, 64))


def test_refusals():
    x, b = torch.zeros(64, 256, device='cuda'), torch.zeros(64, 256, dtype=BF16, device='cuda')
    pair, psum = deep_gemm.cast_to_fp8(b), torch.tensor([64], dtype=torch.int32, device='cuda')
    none = torch.zeros(0, dtype=torch.int32, device='cuda')
    for host in quant_hosts:
        for arg, kw, match in ((x, {}, 'BF16'), (b.t(), {}, 'row-major'), (b[:, :40], {}, 'multiple of 32'), (b, dict(psum_num_tokens_per_expert=none), 'hold an expert'),
                               (b, dict(psum_num_tokens_per_expert=psum, expert_alignment=32), 'multiple of 64'), (b, dict(psum_num_tokens_per_expert=psum.cpu()), 'int32 vector'),
                               (b.view(1, 64, 256), dict(psum_num_tokens_per_expert=psum), '2-D x'), ((b, pair[1]), {}, 'E4M3'), ((pair[0], pair[1][:32]), {}, 'scales must be'),
                               ((pair[0], pair[1].int()), {}, 'scales must be'), ((pair[0], pair[1].contiguous()), {}, 'contiguous along MN'),
                               ((pair[0], pair[1].cpu()), {}, 'scales must be'), (b, dict(min_amax=-1.0), 'min_amax'), (b, dict(min_amax=NAN), 'min_amax')):
            with pytest.raises(RuntimeError, match=match):
                host.cast_to_fp8(arg, mn_major=True, **kw)
        with pytest.raises(RuntimeError, match='min_amax'):
            host.cast_to_fp8(b, min_amax=INF)
        with pytest.raises(RuntimeError, match='x must be a row-major 2-D BF16'):
            host.cast_to_fp8(pair)
        mn = host.cast_to_fp8(b, mn_major=True)
        for arg, kw, match in ((mn, {}, 'scales must be'), (pair, dict(mn_major=True), 'scales must be'), (pair, dict(out_dtype=torch.half), 'out_dtype'), ((b, pair[1]), {}, 'E4M3')):
            with pytest.raises(RuntimeError, match=match):
                host.cast_from_fp8(arg, **kw)
        for arg, kw, match in ((x, {}, 'BF16'), (b[:, :128], {}, 'multiple of 256'), (b, dict(clamp_value=-1.0), 'clamp_value'), (b, dict(topk_weights=x[:, 0]), 'topk_weights'),
                               (b, dict(psum_num_tokens_per_expert=psum, expert_alignment=48), 'multiple of 32'), (b, dict(psum_num_tokens_per_expert=none), 'hold an expert'),
                               (b, dict(out=(pair, pair)), 'out must hold'), (b, dict(topk_weights=torch.zeros(64)), 'topk_weights')):
            with pytest.raises(RuntimeError, match=match):
                host.swiglu_apply_weight_to_fp8_with_checkpoint(arg, **kw)
        g = b[:, :128]
        for args, kw, match in (((x, b), {}, 'grad_out must be'), ((g, x), {}, 'x must be'), ((g, b[:32]), {}, 'x must be'), ((g, (b, pair[1])), {}, 'x must be'),
                                ((g, pair[0]), {}, 'x must be'), ((g, (pair[0], pair[1][:, :2])), {}, 'scales of x'), ((g, (pair[0], pair[1].contiguous())), {}, 'scales of x'),
                                ((g[:, :64], b[:, :128]), {}, 'multiple of 128'), ((g, b), dict(clamp_value=-0.5), 'clamp_value'), ((g, b), dict(out=x), 'out must be'),
                                ((g, b), dict(out=b[:1].expand(64, 256)), 'out must be'), ((g, b), dict(topk_weights=torch.zeros(63, device='cuda')), 'topk_weights')):
            with pytest.raises(RuntimeError, match=match):
                host.swiglu_apply_weight_grad(*args, **kw)


def test_no_rows():
    b = torch.zeros(0, 256, dtype=BF16, device='cuda')
    w = torch.zeros(0, device='cuda')
    for host in quant_hosts:
        out, kept = host.swiglu_apply_weight_to_fp8_with_checkpoint(b, w)
        assert out[0].shape == (0, 128) and kept[0].shape == (0, 256) and out[1].shape == (0, 2) and kept[1].shape == (0, 4)
        for x in (b, kept):
            dx, dw = host.swiglu_apply_weight_grad(out[0].to(BF16), x, w)
            assert dx.shape == (0, 256) and dw.shape == (0,)


def test_rows_behind_32_bits():
    rows, stride = 70000, 65536
    base = torch.zeros(rows * stride, dtype=torch.uint8, device='cuda')
    kept = base.as_strided((rows, 256), (stride, 1)).view(FP8)
    x = torch.randn(rows, 256, device='cuda').bfloat16()
    out = (torch.empty(rows, 128, dtype=FP8, device='cuda'), torch.empty(2, rows, dtype=torch.int16, device='cuda').t())
    sf = torch.empty(4, rows, dtype=torch.int16, device='cuda').t()
    deep_gemm.swiglu_apply_weight_to_fp8_with_checkpoint(x, out=(out, (kept, sf)))
    want = deep_gemm.cast_to_fp8(x)
    assert torch.equal(kept.contiguous().view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(sf, want[1])
    g = torch.randn(rows, 128, device='cuda').bfloat16()
    assert torch.equal(deep_gemm.swiglu_apply_weight_grad(g, (kept, sf))[0], deep_gemm.swiglu_apply_weight_grad(g, want)[0])
    a, b = deep_gemm.cast_to_fp8((kept, sf), mn_major=True), deep_gemm.cast_to_fp8(want, mn_major=True)
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])
    assert torch.equal(deep_gemm.cast_from_fp8((kept, sf)), deep_gemm.cast_from_fp8(want))


def test_many_rows():
    """Against torch on the GPU: rows over many CTAs, an odd number of them."""
    seed_all(10)
    rows, hidden = 5003, 1408
    x, g, w = (torch.randn(rows, 2 * hidden, device='cuda') * 2).bfloat16(), torch.randn(rows, hidden, device='cuda').bfloat16(), torch.rand(rows, device='cuda')
    out, kept = deep_gemm.swiglu_apply_weight_to_fp8_with_checkpoint(x, w)
    want, want_kept = deep_gemm.swiglu_apply_weight_to_fp8(x, w), deep_gemm.cast_to_fp8(x)
    for (q, sf), (q1, sf1) in ((out, want), (kept, want_kept)):
        assert torch.equal(q.view(torch.uint8), q1.view(torch.uint8)) and torch.equal(sf, sf1)
    dx, dw = deep_gemm.swiglu_apply_weight_grad(g, kept, w)
    values = deep_gemm.cast_from_fp8(kept, torch.float32).double().requires_grad_()
    w64 = w.double().requires_grad_()
    l, r = values[:, :hidden], values[:, hidden:]
    (l * torch.sigmoid(l) * r * w64[:, None]).backward(g.double())
    # (2^-8 of the value for the rounding; a few ulp of FP32 times the terms, which are at most |g w| (1 + |l|) (1 + |r|))
    size = (g.double() * w.double()[:, None]).abs() * (1 + l.abs()) * (1 + r.abs())
    assert ((dx.double() - values.grad).abs() <= U * values.grad.abs() + 64 * E * torch.cat((size, size), 1)).all()
    assert ((dw.double() - w64.grad).abs() <= (hidden / 32 + 124) * E * (g.double() * l * r).abs().sum(1)).all()
    q, sf = deep_gemm.cast_to_fp8(kept, mn_major=True)
    part = slice(4992, 5003)                                  # the last, ragged tile
    codes, byte, _ = oracle.cast_fp8_ref(values.detach()[4992:].float().cpu(), 0)
    assert torch.equal(_bytes(q[part]), codes) and torch.equal(sf[78:].cpu(), oracle.pack_scales(byte, 0))
    back = deep_gemm.cast_from_fp8((q, sf), torch.float32, mn_major=True).double()
    amax = torch.nn.functional.pad(values.detach().abs(), (0, 0, 0, -rows % 32)).unflatten(0, (-1, 32)).amax(1).repeat_interleave(32, 0)[:rows]
    # (half a step of a code is 2^-4 of it, or 2^-10 of a scale, which is at most amax / 224)
    assert ((back - values.detach()).abs() <= 2.0 ** -4 * values.detach().abs() + 2.0 ** -10 * amax / 224 + 1e-9).all()


def test_two_streams_at_once_a_captured_run_and_both_hosts():
    seed_all(12)
    layer = python_layer('quant_ops')
    rows, psum, live, _ = _layout([200, 0, 300, 7], 256)
    layout = torch.tensor(psum, dtype=torch.int32, device='cuda')
    live = live.cuda()
    sets = [(torch.randn(rows, 1024, device='cuda').bfloat16(), torch.randn(rows, 512, device='cuda').bfloat16(), torch.rand(rows, device='cuda')) for _ in range(2)]

    def way(s, host=deep_gemm):
        x, g, w = s
        out, kept = host.swiglu_apply_weight_to_fp8_with_checkpoint(x, w, layout, 7.0, 256)
        dx, dw = host.swiglu_apply_weight_grad(g, kept, w, layout, 7.0, 256, zero_padding=True)
        a, b = host.cast_to_fp8(kept, layout, 256, mn_major=True), host.cast_to_fp8(dx, layout, 256, mn_major=True, min_amax=0.0)
        return (out[0].view(torch.uint8)[live], out[1][live], kept[0].view(torch.uint8)[live], kept[1][live], dx, dw, a[0].view(torch.uint8), a[1], b[0].view(torch.uint8), b[1],
                host.cast_from_fp8(a, mn_major=True), host.cast_from_fp8(kept)[live])
    want = [way(s) for s in sets]
    assert all(torch.equal(a, b) for a, b in zip(want[0], way(sets[0], layer)))
    streams, got = [torch.cuda.Stream() for _ in sets], [None, None]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = way(sets[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))

    def run(s):
        x, g, w = s
        out, kept = deep_gemm.swiglu_apply_weight_to_fp8_with_checkpoint(x, w, layout, 7.0, 256)
        dx, dw = deep_gemm.swiglu_apply_weight_grad(g, kept, w, layout, 7.0, 256, zero_padding=True)
        return dx, dw, *deep_gemm.cast_to_fp8(kept, layout, 256, mn_major=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(sets[0])
    for t in sets[0]:
        t.copy_(torch.rand_like(t))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8) if a.dtype == FP8 else a, b.view(torch.uint8) if b.dtype == FP8 else b) for a, b in zip(held, run(sets[0])))


FIRST = textwrap.dedent('''
    import sys
    sys.path.insert(0, %r)
    import torch
    import deep_gemm

    x, r, w = torch.randn(300, 2048, device='cuda').bfloat16(), torch.randn(300, 2048, device='cuda').bfloat16(), torch.ones(2048, device='cuda')
    logits, g = torch.randn(300, 64, device='cuda'), torch.randn(300, 4, device='cuda')


    def way():
        (q, sf), rows, h, rstd = deep_gemm.rms_norm_to_fp8(x, w, residual=r, with_rows=True)
        idx, p = deep_gemm.moe_route(logits, 4, bias=w[:64].contiguous(), num_groups=8, topk_groups=3)
        out, kept = deep_gemm.swiglu_apply_weight_to_fp8_with_checkpoint(rows, rstd)
        dx, dw = deep_gemm.swiglu_apply_weight_grad(rows[:, :1024], kept, rstd)
        mn = deep_gemm.cast_to_fp8(kept, mn_major=True)
        return [q.view(torch.uint8), sf, rows, h, rstd, idx, p, deep_gemm.moe_route_grad(g, logits, idx), out[0].view(torch.uint8), out[1], dx, dw, mn[0].view(torch.uint8), mn[1],
                deep_gemm.cast_from_fp8(mn, mn_major=True), *deep_gemm.rms_norm_grad(dx, h, w, rstd, grad_h=r)]


    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = way()
    graph.replay()
    torch.cuda.synchronize()
    with torch.inference_mode():
        inside = way()
    for a, b, c in zip(held, way(), inside):
        assert torch.equal(a, b) and torch.equal(a, c)
    print('PASS')
''') % os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'deepgemm-ascend_b200')


@pytest.mark.parametrize('python_host', ['0', '1'])
def test_a_capture_that_holds_the_first_call(python_host):
    proc = subprocess.run([sys.executable, '-c', FIRST], capture_output=True, text=True, timeout=600, env={**os.environ, 'DG_PYTHON_HOST': python_host})
    assert proc.returncode == 0 and 'PASS' in proc.stdout, proc.stderr[-3000:]


# ------------------------------------------------------------------------------------------------------ as they are used
F = 2.0 ** -23


def test_a_weight_gradient_from_what_was_kept():
    """The k-grouped GEMM of 8-bit operands along the rows against 64 bits on the values that they stand for."""
    seed_all(13)
    sizes, m, n = [70, 0, 256, 1, 300], 256, 384
    rows, psum, live, _ = _layout(sizes, 256)
    layout = torch.tensor(psum, dtype=torch.int32, device='cuda')
    dy, a = (torch.randn(rows, m) * 1e-7).bfloat16(), torch.randn(rows, n).bfloat16()
    dy[~live], a[~live] = NAN, NAN
    kept = deep_gemm.cast_to_fp8(a.cuda(), layout, 256)
    ops = deep_gemm.cast_to_fp8(dy.cuda(), layout, 256, mn_major=True, min_amax=0.0), deep_gemm.cast_to_fp8(kept, layout, 256, mn_major=True)
    d = torch.full((len(sizes), m, n), NAN, device='cuda')
    deep_gemm.k_grouped_fp8_gemm_tn_contiguous(*ops, d, None, layout)
    assert deep_gemm.device_status() == 0
    x, y = (deep_gemm.cast_from_fp8(o, torch.float32, mn_major=True).cpu().double() for o in ops)
    assert ((x - torch.where(live[:, None], dy.double(), 0.0)).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -9 * 2e-9).all()        # half a step of E4M3; its least one
    for i, (size, p) in enumerate(zip(sizes, psum)):
        want, total = x[p - size:p].t() @ y[p - size:p], x[p - size:p].abs().t() @ y[p - size:p].abs()
        assert ((d[i].cpu().double() - want).abs() <= (size * F + F) * total + 2.0 ** -140).all()


def test_an_expert_layer_in_8_bits():
    """A training step of norm, router, experts and weighted sum, every stage against 64 bits on what the stage in front of it gave; its gradients of the
    input, the experts' weights, the router's and the norm's."""
    seed_all(14)
    tokens, hidden, inner, experts, topk = 120, 256, 128, 8, 3
    dev = lambda t: t.cuda()  # noqa: E731
    x, res = torch.randn(tokens, hidden).bfloat16(), torch.randn(tokens, hidden).bfloat16()
    wn, wr = 1 + 0.1 * torch.randn(hidden), (torch.randn(experts, hidden) * hidden ** -0.5).bfloat16()
    w1, w2 = (torch.randn(experts, 2 * inner, hidden) * hidden ** -0.5).bfloat16(), (torch.randn(experts, hidden, inner) * inner ** -0.5).bfloat16()
    bias, g_out = torch.randn(experts) * 0.05, torch.randn(tokens, hidden).bfloat16()
    values = lambda pair, mn=False: deep_gemm.cast_from_fp8(pair, torch.float32, mn_major=mn).cpu().double()  # noqa: E731
    flat = lambda w: w.cuda().flatten(0, 1)  # noqa: E731

    def weights(w):
        """K-major and MN-major 8-bit weights of all experts."""
        q, sf = deep_gemm.cast_to_fp8(flat(w))
        e, n, k = w.shape
        return (q.view(e, n, k), sf.t().reshape(-1, e, n).transpose(0, 1).contiguous().transpose(1, 2)), deep_gemm.cast_to_fp8(w.cuda(), mn_major=True)
    (w1_k, w1_mn), (w2_k, w2_mn) = weights(w1), weights(w2)
    recipe = (1, 1, 32)

    # forward
    _, y, h, rstd = deep_gemm.rms_norm_to_fp8(dev(x), dev(wn), residual=dev(res), with_rows=True)
    logits = torch.empty(tokens, experts, dtype=torch.float32, device='cuda')
    deep_gemm.bf16_gemm_nt(y, dev(wr), logits)
    idx, p = deep_gemm.moe_route(logits, topk, 'sigmoid', bias=dev(bias), num_groups=4, topk_groups=2, renormalize=True, scale=1.5)
    plan = deep_gemm.moe_sort(idx, experts)
    a1 = deep_gemm.moe_dispatch_to_fp8(y, plan)
    rows = plan[2].numel()
    live = (plan[2] >= 0).cpu()
    h1 = torch.zeros(rows, 2 * inner, dtype=torch.bfloat16, device='cuda')
    deep_gemm.m_grouped_fp8_gemm_nt_contiguous(a1, w1_k, h1, plan[0], recipe=recipe)
    a2, kept = deep_gemm.swiglu_apply_weight_to_fp8_with_checkpoint(h1, None, plan[0], expert_alignment=256)
    y2 = torch.zeros(rows, hidden, dtype=torch.bfloat16, device='cuda')
    deep_gemm.m_grouped_fp8_gemm_nt_contiguous(a2, w2_k, y2, plan[0], recipe=recipe)
    out = deep_gemm.moe_combine(y2, plan, p)
    # backward
    dy2, dp = deep_gemm.moe_combine_grad(dev(g_out), y2, plan, p)
    dy2_k = deep_gemm.cast_to_fp8(dy2, plan[0], 256, min_amax=0.0)
    da2 = torch.zeros(rows, inner, dtype=torch.bfloat16, device='cuda')
    deep_gemm.m_grouped_fp8_gemm_nn_contiguous(dy2_k, w2_mn, da2, plan[0], recipe=recipe)
    dh1, _ = deep_gemm.swiglu_apply_weight_grad(da2, kept, None, plan[0], expert_alignment=256)
    dh1_k = deep_gemm.cast_to_fp8(dh1, plan[0], 256, min_amax=0.0)
    da1 = torch.zeros(rows, hidden, dtype=torch.bfloat16, device='cuda')
    deep_gemm.m_grouped_fp8_gemm_nn_contiguous(dh1_k, w1_mn, da1, plan[0], recipe=recipe)
    along = [deep_gemm.cast_to_fp8(t, plan[0], 256, mn_major=True, min_amax=0.0) for t in (dy2, a2, dh1, a1)]
    dw2, dw1 = torch.empty(experts, hidden, inner, device='cuda'), torch.empty(experts, 2 * inner, hidden, device='cuda')
    deep_gemm.k_grouped_fp8_gemm_tn_contiguous(along[0], along[1], dw2, None, plan[0])
    deep_gemm.k_grouped_fp8_gemm_tn_contiguous(along[2], along[3], dw1, None, plan[0])
    dlogits = deep_gemm.moe_route_grad(dp, logits, idx, 'sigmoid', True, 1.5)
    dy_router, dwr = torch.empty(tokens, hidden, dtype=torch.bfloat16, device='cuda'), torch.empty(experts, hidden, device='cuda')
    deep_gemm.bf16_gemm_nn(dlogits.bfloat16(), dev(wr), dy_router)
    deep_gemm.bf16_gemm_tn(dlogits.bfloat16(), y, dwr)
    dy = deep_gemm.moe_combine(da1, plan) + dy_router
    dx, dwn = deep_gemm.rms_norm_grad(dy, h, dev(wn), rstd, grad_h=dev(g_out))
    assert deep_gemm.device_status() == 0

    # every stage against 64 bits on its own inputs
    assert torch.equal(h.cpu(), (x.float() + res.float()).bfloat16())
    y64 = oracle.rms_norm_ref(h.cpu(), wn, 1e-6)[1]
    assert ((y.cpu().double() - y64).abs() <= (U + 4 * E) * y64.abs()).all()
    l64, size = y.cpu().double() @ wr.double().t(), y.cpu().double().abs() @ wr.double().abs().t()
    assert ((logits.cpu().double() - l64).abs() <= (hidden + 1) * F * size).all()
    ref_idx, ref_p = oracle.moe_route_ref(logits.cpu(), topk, 'sigmoid', bias, 4, 2, 2, True, 1.5)
    assert torch.equal(idx.cpu(), ref_idx) and ((p.cpu().double() - ref_p).abs() <= 56 * E * ref_p).all()
    groups, start = [], 0
    for end in plan[0].tolist():
        groups.append((start, end))
        start = oracle.align(end, 256)

    def grouped(got, a, w, k):
        """got[group] = a[group] @ w[expert]^T, rounded to BF16"""
        for i, (s, e) in enumerate(groups):
            want, size = a[s:e] @ w[i].t(), a[s:e].abs() @ w[i].abs().t()
            err = (k + 1) * F * size
            assert ((got.cpu().double()[s:e] - want).abs() <= err + U * (want.abs() + err) + 2.0 ** -130).all()
    w1_values, w2_values = values(w1_mn, True), values(w2_mn, True)
    from_k = lambda pair: deep_gemm.cast_from_fp8(pair, torch.float32).cpu().double()  # noqa: E731
    grouped(h1, values(a1), from_k(w1_k), hidden)
    grouped(y2, values(a2), from_k(w2_k), inner)
    want = deep_gemm.swiglu_apply_weight_to_fp8(h1, None, plan[0], expert_alignment=256)
    assert torch.equal(_bytes(a2[0])[live], _bytes(want[0])[live]) and torch.equal(a2[1].cpu()[live], want[1].cpu()[live])
    grouped(da2, values(dy2_k), w2_values.transpose(1, 2), hidden)
    grouped(da1, values(dh1_k), w1_values.transpose(1, 2), 2 * inner)
    ops = [values(t, True) for t in along]
    for d, a, b in ((dw2, ops[0], ops[1]), (dw1, ops[2], ops[3])):
        for i, (s, e) in enumerate(groups):
            want, size = a[s:e].t() @ b[s:e], a[s:e].abs().t() @ b[s:e].abs()
            assert ((d[i].cpu().double() - want).abs() <= (e - s + 1) * F * size + 2.0 ** -140).all()
    want, size = oracle.moe_route_grad_ref(dp.cpu(), logits.cpu(), idx.cpu(), 'sigmoid', True, 1.5)
    assert ((dlogits.cpu().double() - want).abs() <= 112 * E * size).all()
    _check_norm_grad(dy.cpu(), h.cpu(), wn, rstd.cpu(), g_out, dx, dwn)
    # the whole of it: the gradient of the loss <out, g_out> + <h, g_out> by differences of the same layer in 64 bits, with the choices held: the
    # 8 bits of the operands (2^-4 of each value, of either sign) leave the direction
    def loss(x64, w1_64, wr64, wn64):
        h64 = x64 + res.double()
        y64 = h64 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + 1e-6) * wn64
        s = torch.sigmoid(y64 @ wr64.t()).gather(1, idx.cpu().long())
        weight = 1.5 * s / s.sum(1, keepdim=True)
        total = h64
        for j in range(topk):
            z = torch.einsum('th,tnh->tn', y64, w1_64[idx.cpu().long()[:, j]])
            z = z[:, :inner] * torch.sigmoid(z[:, :inner]) * z[:, inner:]
            total = total + weight[:, j:j + 1] * torch.einsum('ti,thi->th', z, w2.double()[idx.cpu().long()[:, j]])
        return (total * g_out.double()).sum()
    leaves = [t.double().requires_grad_() for t in (x, w1, wr, wn)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    for got, want in zip((dx, dw1, dwr, dwn), grads):
        got = got.cpu().double()
        assert float((got * want).sum() / (got.norm() * want.norm())) > 0.995
    assert out.shape == (tokens, hidden) and torch.isfinite(out).all()


def _check_norm_grad(g, h, weight, rstd, grad_h, dx, dw):
    ref, r, hidden = oracle.rms_norm_grad_ref(g, h, weight, rstd, grad_h), rstd.double()[:, None], h.size(1)
    mean_err = (hidden / 32 + 85) * E * ref['mean_size']
    err = r * (3 * E * ref['u'] + ref['n'] * (mean_err + 4 * E * (ref['mean'] + mean_err))) + 4 * E * r * (ref['u'] + ref['n'] * ref['mean']) + E * grad_h.double().abs()
    assert ((dx.cpu().double() - ref['dx']).abs() <= err + U * (ref['dx'].abs() + err)).all()
    assert ((dw.cpu().double() - ref['dw']).abs() <= (h.size(0) + 303) * E * ref['dw_size']).all()
