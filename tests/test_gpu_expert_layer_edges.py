"""Where the router's choice, the norm and SwiGLU's gradient can go wrong: sums that cancel or leave the range, numbers that are not finite, rows next to a
border of rounding. Against 64 bits on the CPU (oracle/layers.py)."""

import ctypes as C
import math
import os
import shutil
import subprocess
import sys

import pytest
import torch

import deep_gemm
import oracle
from both_hosts import moe_hosts, quant_hosts
from deep_gemm import _lib as L
from helpers import seed_all
from test_gpu_rms_norm import _check_grad

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
INF, NAN = math.inf, math.nan
BF16 = torch.bfloat16


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


# ------------------------------------------------------------------------------------------------- SwiGLU's gradient
@pytest.mark.parametrize('host', quant_hosts)
@pytest.mark.parametrize('clamp', [None, 7.0])
def test_gates_far_below_zero_have_no_gradient(host, clamp):
    """silu(l) and its slope are 0 in FP32 from about l = -110 on, down to the type's lowest number."""
    seed_all(3)
    far = torch.tensor([-128.0, -1e4, -1e20, -1e30, -1e37, -1e38, -3e38, torch.finfo(BF16).min])
    x, g, w = torch.randn(4, 512).bfloat16(), torch.randn(4, 256).bfloat16(), torch.rand(4) + 0.5
    x[:, 32:40] = far.bfloat16()
    x[2, :256] = torch.finfo(BF16).min
    x[3] = torch.finfo(BF16).min
    pair = deep_gemm.cast_to_fp8(x.cuda())
    # (code times scale in 64 bits: the lowest number of BF16 becomes -2^128)
    byte = torch.stack((pair[1].cpu().int() & 255, (pair[1].cpu().int() >> 8) & 255), 2).flatten(1)
    kept = pair[0].cpu().double() * torch.exp2((byte - 127).double()).repeat_interleave(32, 1)
    assert kept.min() == -2.0 ** 128
    for arg, values in ((x.cuda(), x.double()), (pair, kept)):
        dx, dw = host.swiglu_apply_weight_grad(g.cuda(), arg, w.cuda(), clamp_value=clamp)
        dx, dw = dx.cpu(), dw.cpu()
        none = values[:, :256] <= -128
        assert (dx[:, :256][none] == 0).all() and (dx[:, 256:][none] == 0).all() and torch.isfinite(dx).all()
        l, r = values[:, :256], values[:, 256:]
        if clamp:
            l, r = l.clamp(max=clamp), r.clamp(-clamp, clamp)
        terms = g.double() * l * torch.sigmoid(l) * r
        # (64 roundings, of 32 channels a lane and of each term)
        assert ((dw.double() - terms.sum(1)).abs() <= 128 * E * terms.abs().sum(1)).all() and (dw[2:] == 0).all()


def test_codes_that_are_not_numbers_show_in_the_gradient():
    """A NaN code of either sign, and the NaN scale, in both halves of the 8-bit input."""
    codes, sf = torch.full((6, 256), 0x38, dtype=torch.uint8), torch.full((4, 6), 0x7F7F, dtype=torch.int16)
    codes[0, 3], codes[1, 3], codes[2, 131], codes[3, 131] = 0x7F, 0xFF, 0x7F, 0xFF
    sf[0, 4], sf[2, 5] = -129, -129                                  # 0xFF7F: columns 32 to 63 of a half
    dx, dw = deep_gemm.swiglu_apply_weight_grad(torch.ones(6, 128, dtype=BF16, device='cuda'), (codes.cuda().view(torch.float8_e4m3fn), sf.cuda().t()), torch.ones(6, device='cuda'))
    bad = torch.zeros(6, 256, dtype=torch.bool)
    bad[:2, 3] = bad[:2, 131] = bad[2:4, 3] = True
    bad[4, 32:64] = bad[4, 160:192] = bad[5, 32:64] = True
    assert torch.equal(dx.isnan().cpu(), bad) and dw.isnan().all()


@pytest.mark.parametrize('host', quant_hosts)
def test_codes_beyond_the_range_are_infinities_whatever_lies_beside_them(host):
    """-256 x 2^120, what the lowest BF16 number becomes, in tiles whose other rows have scales near to that one and far from it."""
    for other in (247, 240, 200, 0):
        codes, byte = torch.full((64, 64), 0x30, dtype=torch.uint8), torch.full((64, 2), other, dtype=torch.int32)
        codes[5, 3], codes[5, 40], codes[9, 7] = 0xF8, 0x78, 0x77             # -256, 256, and 240, which is within
        byte[5] = byte[9] = 247
        sf = (byte[:, :1] | byte[:, 1:] << 8)
        sf = torch.where(sf >= 32768, sf - 65536, sf).to(torch.int16)
        q, out = host.cast_to_fp8((codes.cuda().view(torch.float8_e4m3fn), sf.cuda()), mn_major=True)
        first = out.cpu().int() & 255
        want = oracle.cast_fp8_ref((codes.view(torch.float8_e4m3fn).double() * torch.exp2((byte - 127).double()).repeat_interleave(32, 1)).float(), 0, 1e-4)
        assert torch.equal(first[0], want[1][0].int()) and first[0, 3] == first[0, 40] == 255 and first[0, 7] == 247
        fine = (want[1] != 255).repeat_interleave(32, 0)
        assert torch.equal(q.view(torch.uint8).cpu()[fine], want[0][fine])


# ---------------------------------------------------------------------------------------------------------- the norm
@pytest.mark.parametrize('dtype,hidden', [(BF16, 96), (BF16, 2048), (BF16, 4096), (BF16, 7168), (BF16, 8224), (torch.float32, 96), (torch.float32, 2048),
                                          (torch.float32, 4128), (torch.float32, 8224)])
@pytest.mark.parametrize('size,grad_size', [(1e-25, 1.0), (1e30, 1e10), (1e-30, 1e-5)])
def test_gradient_of_rows_far_from_one(dtype, hidden, size, grad_size):
    """rstd^2 and the products of h and its gradient leave the range of FP32, dx does not."""
    seed_all(hidden)
    for tokens in (3, 400):
        h, g = (torch.randn(tokens, hidden) * size).to(dtype), (torch.randn(tokens, hidden) * grad_size).to(dtype)
        weight = 1 + 0.1 * torch.randn(hidden)
        _check_grad(g, h, weight, oracle.rms_norm_ref(h, weight, 0.0)[0].float())


def _rows_near_a_border(count, hidden, eps):
    """BF16 rows whose 1 / sqrt(mean(h^2) + eps) lies within a few 2^-53 of the middle between two FP32 numbers, with squares whose sum depends on its order."""
    rows = (torch.randn(count, hidden) * torch.exp2(torch.randint(-14, 15, (count, hidden)).float())).bfloat16()
    spare, nothing = torch.randperm(hidden)[:10], torch.zeros((), dtype=BF16)
    rows[:, spare] = 0
    eps = float(torch.tensor(eps))
    for row, steps in zip(rows, torch.randint(-4, 5, (count,)).tolist()):
        base = math.fsum((row.double() ** 2).tolist())
        low = torch.tensor(1 / math.sqrt(base / hidden + eps))
        low = torch.nextafter(torch.nextafter(low, torch.zeros(())), torch.zeros(()))
        middle = (float(low) + float(torch.nextafter(low, torch.ones(()) * 9e9))) / 2
        left = (1 / middle ** 2 - eps) * hidden * (1 + steps * 2.0 ** -53) - base
        for c in spare:
            v = torch.tensor(math.sqrt(max(left, 0.0)), dtype=torch.float64).bfloat16()
            if float(v) ** 2 > left:
                v = torch.nextafter(v, nothing)
            row[c] = v
            left -= float(v) ** 2
    return rows


@pytest.mark.parametrize('hidden', [2048, 4096, 7168])
def test_rows_next_to_a_border_do_not_depend_on_their_number(hidden):
    """The sum of squares is made in one order, whatever the number of tokens."""
    seed_all(hidden)
    x, w = _rows_near_a_border(400, hidden, 1e-6).cuda(), torch.ones(hidden, device='cuda')
    few = torch.cat([deep_gemm.rms_norm_to_fp8(x[i:i + 100], w)[3] for i in range(0, 400, 100)])
    assert torch.equal(deep_gemm.rms_norm_to_fp8(x, w)[3], few)
    assert torch.equal(deep_gemm.rms_norm_to_fp8(x.repeat(3, 1), w)[3], few.repeat(3))


@pytest.mark.parametrize('tokens,hidden', [(4736, 3616), (4737, 3616), (5003, 4096), (5003, 4128)])
def test_gradient_on_both_sides_of_a_long_walk(tokens, hidden):
    """BF16 rows of which a CTA holds one in registers and two in shared memory."""
    seed_all(tokens + hidden)
    h, g, more = torch.randn(tokens, hidden).bfloat16(), torch.randn(tokens, hidden).bfloat16(), torch.randn(tokens, hidden).bfloat16()
    weight = torch.randn(hidden)
    _check_grad(g, h, weight, oracle.rms_norm_ref(h, weight, 1e-6)[0].float(), more)


WAITS = '''
#include "%s"
namespace dg {
void set_last_error(const char*, ...) {}
void count_kernel_launch(unsigned) {}
bool overlap_launches_enabled() { return false; }
}
extern "C" int take_status() { int code = 0; return cudaDeviceSynchronize() == cudaSuccess && dg::take_norm_status(&code) == 0 ? code : -1; }
'''


def test_a_wait_that_gives_up_is_reported(tmp_path):
    """The norm's kernels, built so that no wait for a bulk copy lasts: they let the copies land, say so, and leave NaN; the device goes on."""
    nvcc = shutil.which('nvcc') or '/usr/local/cuda/bin/nvcc'
    if not os.path.exists(nvcc):
        pytest.skip('no nvcc')
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(deep_gemm.__file__))), 'csrc')
    (tmp_path / 'waits.cu').write_text(WAITS % os.path.join(csrc, 'norm_ops.cu'))
    subprocess.run([nvcc, '-gencode', 'arch=compute_100a,code=sm_100a', '-O3', '-std=c++17', '--expt-relaxed-constexpr', '-DDG_NORM_LONGEST_WAIT_NS=0', '-Xcompiler', '-fPIC',
                    '-Xlinker', '-Bsymbolic', '-shared', '-o', str(tmp_path / 'waits.so'), str(tmp_path / 'waits.cu')], check=True, timeout=300)
    lib = C.CDLL(str(tmp_path / 'waits.so'))
    for name in ('dg_rms_norm_fp8_launch', 'dg_rms_norm_grad_launch'):
        getattr(lib, name).restype, getattr(lib, name).argtypes = L._PROTOTYPES[name]
    stream = torch.cuda.current_stream().cuda_stream
    # four, one and two tokens ahead; several groups of a CTA, and one; one turn, and many; whether the norm and its gradient have bulk copies there
    for dtype, tokens, hidden, forward, backward in ((BF16, 1100, 1056, True, False), (BF16, 1100, 16384, True, True), (torch.float32, 100, 16384, True, True),
                                                     (torch.float32, 1100, 4096, True, True), (torch.float32, 1100, 2080, True, True), (BF16, 5000, 4096, False, True)):
        x, w, fp32 = torch.randn(tokens, hidden, device='cuda').to(dtype), torch.randn(hidden, device='cuda'), int(dtype == torch.float32)
        q, sf = torch.zeros(tokens, hidden, dtype=torch.uint8, device='cuda'), torch.zeros(hidden // 64 + 1, tokens, dtype=torch.int16, device='cuda')
        rstd, h = torch.zeros(tokens, device='cuda'), torch.zeros_like(x)
        assert lib.dg_rms_norm_fp8_launch(x.data_ptr(), fp32, hidden, x.data_ptr(), hidden, h.data_ptr(), hidden, w.data_ptr(), 1, 1e-6, tokens, hidden, q.data_ptr(), hidden,
                                          sf.data_ptr(), tokens, None, 0, rstd.data_ptr(), stream) == 0
        assert lib.take_status() == (108 if forward else 0) and lib.take_status() == 0 and rstd.isnan().all() == forward and (q == 0).all() == forward
        ones = torch.ones(tokens, device='cuda')
        dx, dw, scratch = torch.zeros_like(x), torch.zeros(hidden, device='cuda'), torch.empty(148 * hidden, device='cuda')
        assert lib.dg_rms_norm_grad_launch(x.data_ptr(), fp32, hidden, x.data_ptr(), fp32, hidden, w.data_ptr(), 1, ones.data_ptr(), x.data_ptr(), hidden,
                                           tokens, hidden, dx.data_ptr(), hidden, dw.data_ptr(), scratch.data_ptr(), scratch.numel() * 4, stream) == 0
        assert lib.take_status() == (108 if backward else 0) and dw.isnan().all() == backward and (dx == 0).all() == backward
        # the library itself reports nothing, and works
        want = deep_gemm.rms_norm_to_fp8(x, w)[3]
        assert deep_gemm.device_status() == 0 and not want.isnan().any()


FIRST = '''
import sys
sys.path.insert(0, %r)
import torch
import deep_gemm
x, w, g = torch.randn(1100, 2048, device='cuda').bfloat16(), torch.ones(2048, device='cuda'), torch.randn(1100, 4096, device='cuda')
wide = torch.ones(4096, device='cuda')


def way():
    (q, sf), rows, h, rstd = deep_gemm.rms_norm_to_fp8(x, w, residual=x, with_rows=True)
    return [q.view(torch.uint8), sf, rows, h, rstd, *deep_gemm.rms_norm_grad(g, g, wide, rstd, grad_h=g)]


torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    held = way()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(held, way())) and deep_gemm.device_status() == 0
print('PASS')
'''


def test_bulk_copies_in_a_capture_that_holds_the_first_call():
    """The norm's forms that raise a limit of shared memory, in the first call of a process."""
    package = os.path.dirname(os.path.dirname(os.path.abspath(deep_gemm.__file__)))
    for host in '01':
        proc = subprocess.run([sys.executable, '-c', FIRST % package], capture_output=True, text=True, timeout=600, env={**os.environ, 'DG_PYTHON_HOST': host})
        assert proc.returncode == 0 and 'PASS' in proc.stdout, proc.stderr[-3000:]
