"""What the router's choice, the norm, SwiGLU's gradient and the 8-bit operands along the rows refuse, in both host layers and in the C ABI, and the
oracle that their GPU tests use. Nothing here reaches a launch."""

import math

import pytest
import torch

import deep_gemm
import oracle
from both_hosts import moe_hosts, quant_hosts
from deep_gemm import _lib as L

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize('host', moe_hosts)
def test_host_tensors_are_refused_by_the_router(host):
    logits = torch.zeros(4, 16)
    with pytest.raises(RuntimeError, match='logits must be a row-major 2-D BF16 or FP32 tensor on a CUDA device'):
        host.moe_route(logits, 2)
    with pytest.raises(RuntimeError, match='logits must be'):
        host.moe_route_grad(torch.zeros(4, 2), logits, torch.zeros(4, 2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match='topk_idx must be'):
        host.moe_route_grad(torch.zeros(4, 2), logits, torch.zeros(4, 2))
    with pytest.raises(RuntimeError, match='topk_idx must be'):
        host.moe_route_grad(torch.zeros(4, 2), logits, torch.zeros(3, 2, dtype=torch.int32))


@pytest.mark.parametrize('host', quant_hosts)
def test_host_tensors_are_refused_by_the_quantisers(host):
    x, pair = torch.zeros(4, 256, dtype=BF16), (torch.zeros(4, 256).to(FP8), torch.zeros(4, 4, dtype=torch.int16))
    for call in (lambda: host.cast_to_fp8(x), lambda: host.cast_to_fp8(x, mn_major=True), lambda: host.cast_to_fp8(pair, mn_major=True), lambda: host.cast_to_fp8(pair),
                 lambda: host.cast_from_fp8(pair), lambda: host.swiglu_apply_weight_to_fp8(x), lambda: host.swiglu_apply_weight_to_fp8_with_checkpoint(x),
                 lambda: host.swiglu_apply_weight_grad(x, pair), lambda: host.rms_norm_to_fp8(x, torch.ones(256)),
                 lambda: host.rms_norm_grad(x, x, torch.ones(256), torch.ones(4))):
        with pytest.raises(RuntimeError, match='on a CUDA device'):
            call()


def _refused(rc, match):
    assert rc in (L.DG_ERR_INVALID, L.DG_ERR_UNSUPPORTED) and match in L.last_error(), L.last_error()


def test_the_c_abi_refuses_routers_out_of_range():
    lib, p = L.lib(), 0x1000
    route = lambda experts=64, topk=4, groups=1, taken=1, best=2, logits=p, idx=p: lib.dg_moe_route_launch(  # noqa: E731
        logits, 1, experts, 8, experts, topk, 0, None, groups, taken, best, 0, 1.0, idx, p, None)
    _refused(route(experts=0), 'number of experts')
    _refused(route(experts=1025), 'number of experts')
    _refused(route(topk=0), 'topk must be')
    _refused(route(topk=33), 'topk must be')
    _refused(route(experts=3, topk=4), 'topk must be')
    _refused(route(groups=0), 'number of groups')
    _refused(route(groups=33, experts=66), 'number of groups')
    _refused(route(groups=5), 'number of groups')
    _refused(route(groups=8, taken=9), 'topk_groups')
    _refused(route(groups=8, taken=0), 'topk_groups')
    _refused(route(groups=32, taken=1), 'fewer experts than topk')
    _refused(route(best=3), 'group_best')
    _refused(route(logits=None), 'logits')
    _refused(route(logits=p + 2), 'logits')
    _refused(route(idx=None), 'null pointer')
    grad = lambda topk=4, g=p, out=p: lib.dg_moe_route_grad_launch(g, p, 1, 64, 8, 64, p, 0, topk, 0, 0, 1.0, out, 64, None)  # noqa: E731
    _refused(grad(topk=33), 'topk must be')
    _refused(grad(g=None), 'null pointer')
    _refused(grad(out=p + 2), 'aligned')


def test_the_c_abi_refuses_norms_it_cannot_run():
    lib, p = L.lib(), 0x1000
    norm = lambda hidden=64, x=p, res=None, h=p, w=p, out=p, sf_stride=8, rows=None, stride=64: lib.dg_rms_norm_fp8_launch(  # noqa: E731
        x, 0, stride, res, 64, h, 64, w, 0, 1e-6, 8, hidden, out, 64, p, sf_stride, rows, 64, p, None)
    _refused(norm(hidden=48), 'multiple of 32')
    _refused(norm(hidden=0), 'multiple of 32')
    _refused(norm(hidden=16384 + 32), 'at most 16384')
    _refused(norm(x=None), 'null pointer')
    _refused(norm(res=p, h=None), 'null pointer')
    for bad in (dict(x=p + 8), dict(res=p + 2), dict(h=p + 4), dict(w=p + 8), dict(rows=p + 8), dict(stride=68)):
        _refused(norm(**bad), '16-byte')
    _refused(norm(out=p + 4), '8-byte')
    _refused(norm(sf_stride=7), 'scale column stride')
    grad = lambda g=p, g32=0, h32=0, hidden=64, nbytes=1 << 20, scratch=p, dx=p: lib.dg_rms_norm_grad_launch(  # noqa: E731
        g, g32, 64, p, h32, 64, p, 0, p, None, 0, 8, hidden, dx, 64, p, scratch, nbytes, None)
    _refused(grad(g=None), 'null pointer')
    _refused(grad(g32=1), 'FP32 gradient beside BF16 rows')
    _refused(grad(hidden=16416), 'at most 16384')
    _refused(grad(nbytes=lib.dg_rms_norm_grad_scratch_bytes(8, 64) - 1), 'scratch is too small')
    _refused(grad(scratch=None), 'null pointer')
    _refused(grad(dx=p + 8), '16-byte')


def test_the_c_abi_refuses_8_bit_rows_it_cannot_read():
    lib, p = L.lib(), 0x1000
    keep = lambda hidden=128, kept=p, kept_sf=p, stride=8, psum=None, align=128, experts=1: lib.dg_swiglu_checkpoint_launch(  # noqa: E731
        p, 256, 8, hidden, None, psum, experts, align, 0, 0.0, p, 128, p, 8, kept, 256, kept_sf, stride, None)
    _refused(keep(hidden=96), 'multiple of 64')
    _refused(keep(kept=None), 'null pointer')
    _refused(keep(kept=p + 4), '8-byte')
    _refused(keep(stride=7), 'scale column stride')
    _refused(keep(psum=p, align=48), 'multiple of 32')
    _refused(keep(psum=p, experts=0), 'multiple of 32')
    grad = lambda hidden=128, x=p, sf=p, stride=8, w=None, dw=None, dx=p, psum=None, align=128, scratch=None, nbytes=0: lib.dg_swiglu_grad_launch(  # noqa: E731
        p, 128, x, 256, sf, stride, 8, hidden, w, psum, 1, align, 0, 0.0, dx, 256, dw, 0, scratch, nbytes, None)
    _refused(grad(hidden=96), 'multiple of 64')
    _refused(grad(x=None), 'null pointer')
    _refused(grad(x=p + 4), 'boundaries')
    _refused(grad(x=p + 8, sf=None), 'boundaries')
    _refused(grad(dx=p + 8), 'boundaries')
    _refused(grad(stride=7), 'scale column stride')
    _refused(grad(dw=p), 'weights that are not there')
    _refused(grad(psum=p, align=33), 'multiple of 32')
    _refused(grad(hidden=512, w=p, dw=p), 'scratch is too small')
    _refused(grad(hidden=512, w=p, dw=p, scratch=p, nbytes=lib.dg_swiglu_grad_scratch_bytes(8, 512) - 1), 'scratch is too small')
    mn = lambda cols=64, x=p, sf=None, sf_stride=8, out=p, stride=64, psum=None, align=64, groups=1, floor=1e-4: lib.dg_quant_fp8_mn_launch(  # noqa: E731
        x, 64, 0, sf, sf_stride, 0, groups, 8, cols, psum, 1, align, floor, out, 64, 0, p, stride, 0, None)
    _refused(mn(cols=48), 'multiple of 32')
    _refused(mn(x=None), 'null pointer')
    _refused(mn(x=p + 8), '16-byte')
    _refused(mn(x=p + 4, sf=p), '8-byte')
    _refused(mn(out=p + 4), '8-byte')
    _refused(mn(stride=63), 'scale stride')
    _refused(mn(sf=p, sf_stride=7), 'scale stride')
    _refused(mn(psum=p, align=32), 'multiple of 64')
    _refused(mn(psum=p, groups=2), 'one matrix')
    for floor in (-1.0, math.inf, math.nan):
        _refused(mn(floor=floor), 'min_amax')
        _refused(lib.dg_cast_fp8_launch(p, 64, 8, 64, None, 0, 128, floor, p, 64, p, 8, None), 'min_amax')
    back = lambda cols=64, codes=p, sf=p, out=p, fp32=0, mn_major=0, stride=64: lib.dg_dequant_fp8_launch(  # noqa: E731
        codes, 64, 0, sf, stride, 0, 1, 8, cols, mn_major, out, fp32, 64, 0, None)
    _refused(back(cols=40), 'multiple of 32')
    _refused(back(sf=None), 'null pointer')
    _refused(back(codes=p + 4), '8-byte')
    _refused(back(out=p + 8), '16-byte')
    _refused(back(out=p + 16, fp32=1), '32-byte')
    _refused(back(stride=7), 'scale stride')
    _refused(back(stride=63, mn_major=1), 'scale stride')


def test_nothing_to_do_is_no_error():
    lib = L.lib()
    assert lib.dg_moe_route_launch(None, 1, 64, 0, 64, 4, 0, None, 1, 1, 2, 0, 1.0, None, None, None) == L.DG_OK
    assert lib.dg_moe_route_grad_launch(None, None, 1, 64, 0, 64, None, 0, 4, 0, 0, 1.0, None, 64, None) == L.DG_OK
    assert lib.dg_rms_norm_fp8_launch(None, 0, 64, None, 0, None, 0, None, 0, 1e-6, 0, 64, None, 64, None, 0, None, 0, None, None) == L.DG_OK
    assert lib.dg_swiglu_grad_launch(None, 0, None, 0, None, 0, 0, 128, None, None, 0, 128, 0, 0.0, None, 0, None, 0, None, 0, None) == L.DG_OK
    assert lib.dg_quant_fp8_mn_launch(None, 0, 0, None, 0, 0, 1, 0, 64, None, 0, 0, 0.0, None, 0, 0, None, 0, 0, None) == L.DG_OK
    assert lib.dg_dequant_fp8_launch(None, 0, 0, None, 0, 0, 1, 0, 64, 0, None, 0, 0, 0, None) == L.DG_OK
    assert lib.dg_rms_norm_grad_scratch_bytes(0, 64) == 0


# ------------------------------------------------------------------------------------------------------------- the oracle
def test_the_oracle_of_the_choice():
    logits = torch.tensor([[1.0, 3.0, 2.0, 3.0], [-math.inf] * 4, [-math.inf, 0.0, -math.inf, -math.inf]])
    idx, w = oracle.moe_route_ref(logits, 2)
    p = torch.softmax(logits[0].double(), 0)
    assert idx.tolist() == [[1, 3], [-1, -1], [1, -1]] and torch.equal(w[0], p[[1, 3]]) and w[1].tolist() == [0, 0] and w[2].tolist() == [1, 0]
    idx, w = oracle.moe_route_ref(logits[:1], 2, 'sigmoid', torch.tensor([9.0, 0, 0, 0]), 2, 1, renormalize=True, scale=2.0)
    s = torch.sigmoid(logits[0].double())
    assert idx.tolist() == [[0, 1]] and torch.allclose(w[0], 2 * s[:2] / s[:2].sum(), rtol=1e-15)


def test_the_oracle_of_the_choice_against_its_gradient():
    gen = torch.Generator().manual_seed(1)
    l = torch.randn(3, 7, generator=gen, dtype=torch.float64)
    idx, g = torch.tensor([[1, 5, 2], [0, -1, 6], [3, 3, 4]]), torch.randn(3, 3, generator=gen, dtype=torch.float64)
    for scoring in ('softmax', 'sigmoid'):
        for renormalize in (False, True):
            def f(x):
                s = torch.sigmoid(x) if scoring == 'sigmoid' else torch.softmax(x, 1)
                w = torch.where(idx >= 0, s.gather(1, idx.clamp(min=0)), 0.0)
                return 1.5 * (w / w.sum(1, keepdim=True) if renormalize else w)
            x = l.clone().requires_grad_()
            want = torch.autograd.grad(f(x), x, g)[0]
            got, size = oracle.moe_route_grad_ref(g, l, idx, scoring, renormalize, 1.5)
            assert (got - want).abs().max() < 1e-14 and (size >= got.abs() - 1e-14).all()


def test_the_oracle_of_the_gradients():
    gen = torch.Generator().manual_seed(2)
    randn = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    h, w, g = randn(3, 32).requires_grad_(), randn(32).requires_grad_(), randn(3, 32)
    rstd, y = oracle.rms_norm_ref(h, w, 1e-6)
    dh, dw = torch.autograd.grad(y, (h, w), g)
    ref = oracle.rms_norm_grad_ref(g, h.detach(), w.detach(), rstd.detach())
    assert (ref['dx'] - dh).abs().max() < 1e-13 and (ref['dw'] - dw).abs().max() < 1e-13
    x, w, g = (2 * randn(3, 16)).requires_grad_(), randn(3).requires_grad_(), randn(3, 8)
    l, r = x[:, :8].clamp(max=1.5), x[:, 8:].clamp(-1.5, 1.5)
    dx, dw = torch.autograd.grad(l * torch.sigmoid(l) * r * w[:, None], (x, w), g)
    dl, dr, dw_ref, _ = oracle.swiglu_grad_ref(g, x.detach(), w.detach(), 1.5)
    assert (torch.cat((dl, dr), 1) - dx).abs().max() < 1e-13 and (dw_ref - dw).abs().max() < 1e-13


def test_the_oracle_of_the_cast_agrees_with_the_rows():
    x = torch.randn(40, 96).bfloat16()
    codes, sf, _, deq = oracle.swiglu_quant_ref(x, swiglu=False)
    c, e, v = oracle.cast_fp8_ref(x, 1)
    assert torch.equal(c, codes) and torch.equal(oracle.pack_scales(e, 1), sf) and torch.equal(v, deq)
    c, e, v = oracle.cast_fp8_ref(x.t().contiguous(), 0)
    assert torch.equal(c.t(), codes) and torch.equal(oracle.pack_scales(e, 0).t(), sf) and torch.equal(v.t(), deq)


def test_entry_points_are_exported():
    for name in ('moe_route', 'moe_route_grad', 'rms_norm_to_fp8', 'rms_norm_grad', 'swiglu_apply_weight_to_fp8_with_checkpoint', 'swiglu_apply_weight_grad',
                 'cast_to_fp8', 'cast_from_fp8'):
        assert callable(getattr(deep_gemm, name)), name
