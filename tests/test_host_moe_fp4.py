"""What the MoE row operators and the FP4 quantiser refuse, in both host layers and in the C ABI, and the oracle that their GPU tests use.
Nothing here reaches a launch."""

import pytest
import torch

import oracle
from both_hosts import moe_hosts, quant_hosts
from deep_gemm import _lib as L


def _plan(tokens=4, topk=2, experts=3, max_m=0, dtype=torch.int32):
    rows = (experts, max_m) if max_m else (768,)
    return tuple(torch.zeros(s, dtype=dtype) for s in ((experts,), (tokens, topk), rows))


@pytest.mark.parametrize('host', moe_hosts)
def test_host_tensors_are_refused(host):
    x, idx, plan = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 2, dtype=torch.int64), _plan()
    with pytest.raises(RuntimeError, match='topk_idx must be a contiguous 2-D int32 or int64 tensor on a CUDA device'):
        host.moe_sort(idx, 3)
    with pytest.raises(RuntimeError, match='x must be a row-major 2-D BF16 or FP32 tensor on a CUDA device'):
        host.moe_dispatch(x, plan)
    with pytest.raises(RuntimeError, match='x must be a row-major 2-D BF16 tensor on a CUDA device'):
        host.moe_dispatch_to_fp8(x, plan)
    with pytest.raises(RuntimeError, match='rows must be a 2-D or 3-D BF16 or FP32 tensor on a CUDA device'):
        host.moe_combine(torch.zeros(768, 64, dtype=torch.bfloat16), plan)
    with pytest.raises(RuntimeError, match='grad_out must be a row-major 2-D BF16 or FP32 tensor on a CUDA device'):
        host.moe_combine_grad(x, torch.zeros(768, 64, dtype=torch.bfloat16), plan, torch.zeros(4, 2))


@pytest.mark.parametrize('host', quant_hosts)
def test_host_tensors_are_refused_by_the_quantiser(host):
    with pytest.raises(RuntimeError, match='x must be a row-major 2-D or 3-D BF16 or FP32 tensor on a CUDA device'):
        host.cast_to_fp4(torch.zeros(4, 64))
    with pytest.raises(RuntimeError, match='x must be a row-major 2-D or 3-D tensor of packed FP4 on a CUDA device'):
        host.cast_from_fp4((torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.int16)))


def _refused(rc, message):
    assert rc == L.DG_ERR_INVALID and message in L.last_error(), (rc, L.last_error())


def test_the_c_abi_checks_its_arguments():
    lib, p = L.lib(), 1 << 20                                     # (an address that nothing reads: every call is refused)
    sort = lambda n=8, k=2, e=4, align=256, max_m=0, rows=None, idx=p: lib.dg_moe_sort_launch(  # noqa: E731
        idx, 1, n, k, e, align, max_m, p, p, p, oracle.moe_rows(n * k, e, align) if rows is None else rows, None)
    _refused(sort(e=0), 'between 1 and 1024')
    _refused(sort(e=1025), 'between 1 and 1024')
    _refused(sort(rows=100), 'wrong number of rows')
    _refused(sort(max_m=16, rows=1024), 'wrong number of rows')
    _refused(sort(align=0, rows=0), 'alignment must be positive')
    _refused(sort(n=1 << 31, k=2), 'too many choices')
    _refused(sort(align=1 << 31, e=1, rows=1 << 31), 'too many rows')
    _refused(sort(idx=None), 'null pointer')
    copy = lambda x=p, xs=128, nbytes=128, rows=512, out=p, os=128, layout=p, e=4, align=256, zero=0, of=p, rc=p: lib.dg_moe_dispatch_launch(  # noqa: E731
        x, xs, 4, 2, nbytes, of, rc, rows, out, os, layout, e, align, 0, zero, None)
    for bad in (dict(nbytes=120), dict(x=p + 8), dict(xs=120), dict(out=p + 8), dict(os=136)):
        _refused(copy(**bad), '16-byte boundaries')
    for bad in (dict(x=None), dict(out=None), dict(of=None)):
        _refused(copy(**bad), 'null pointer')
    for bad in (dict(layout=None), dict(rc=None), dict(e=0), dict(align=0)):
        _refused(copy(zero=1, **bad), 'zeros in the padding need the layout')
    _refused(copy(rows=1 << 31), 'too many choices or rows')
    _refused(copy(zero=1, e=1024, align=1 << 22), 'too many rows')
    fp8 = lambda x=p, xs=64, hidden=64, out=p, os=64, sf=p, col=512, per=512, rc=p, scratch=None, nbytes=0: lib.dg_moe_dispatch_fp8_launch(  # noqa: E731
        x, xs, 4, 2, hidden, p, rc, 512, out, os, sf, col, 0, per, scratch, nbytes, None)
    _refused(fp8(hidden=48), 'multiple of 32')
    _refused(fp8(xs=60), 'input rows must start on 16-byte boundaries')
    _refused(fp8(os=60), 'output rows must start on 8-byte boundaries')
    _refused(fp8(col=500), 'scale column stride')
    _refused(fp8(per=0, col=0), 'scale column stride')
    _refused(fp8(sf=None), 'null pointer')
    for bad in (dict(nbytes=63), dict(scratch=p + 8, nbytes=64), dict(rc=None, nbytes=64)):
        _refused(fp8(**{'scratch': p, **bad}), 'the scratch must be')
    assert lib.dg_moe_dispatch_fp8_scratch_bytes(2047, 7168) == 0 and lib.dg_moe_dispatch_fp8_scratch_bytes(8191, 7200) == 8191 * 240
    combine = lambda y=p, ys=64, hidden=64, out=p, os=64: lib.dg_moe_combine_launch(y, 0, ys, 512, hidden, p, 4, 2, p, out, os, None)  # noqa: E731
    for bad in (dict(y=p + 2), dict(ys=60), dict(hidden=60), dict(out=p + 2), dict(os=60)):
        _refused(combine(**bad), '16-byte boundaries')
    _refused(combine(y=None), 'null pointer')
    grad = lambda g=p, gs=64, y=p, w=p, dw=p, dy=p: lib.dg_moe_combine_grad_launch(  # noqa: E731
        g, 0, gs, y, 64, 512, 64, p, None, 4, 2, w, dy, 64, dw, None, 0, 256, 0, 0, None)
    for bad in (dict(g=None), dict(y=None), dict(w=None), dict(dw=None), dict(dy=None)):
        _refused(grad(**bad), 'null pointer')
    _refused(grad(gs=60), '16-byte boundaries')
    fp4 = lambda x=p, xs=64, rows=8, cols=64, mn=0, psum=None, e=0, align=0, groups=1, out=p, os=32, sf=p, ss=64: lib.dg_quant_fp4_launch(  # noqa: E731
        x, 0, xs, 0, groups, rows, cols, mn, psum, e, align, out, os, 0, sf, ss, 0, None)
    _refused(fp4(cols=48), 'multiple of 32')
    _refused(fp4(xs=60), '16-byte boundaries')
    _refused(fp4(os=30), 'codes must start on 4-byte boundaries')
    _refused(fp4(os=36, mn=1), 'codes must start on 16-byte boundaries')
    _refused(fp4(ss=7), 'scale stride')
    _refused(fp4(mn=1, ss=63), 'scale stride')
    _refused(fp4(psum=p, e=4, align=48), 'multiple of 32')
    _refused(fp4(psum=p, e=4, align=96, mn=1), 'multiple of 64')
    _refused(fp4(psum=p, e=4, align=128, groups=2), 'one matrix')
    _refused(fp4(rows=(1 << 32) - 1, cols=1 << 13, ss=1 << 32), 'too many values')
    for bad in (dict(x=None), dict(out=None), dict(sf=None)):
        _refused(fp4(**bad), 'null pointer')
    assert lib.dg_moe_num_rows(0, 4, 256) == 0
    for choices, experts, alignment in ((1, 256, 256), (8, 4, 256), (1000, 3, 32), (65536, 256, 256), (7, 7, 1)):
        assert lib.dg_moe_num_rows(choices, experts, alignment) == oracle.moe_rows(choices, experts, alignment)


def test_no_choices_need_more_rows_than_the_bound():
    """By trying all splits of a few choices: the bound is reached and never passed."""
    def splits(n, parts):
        if parts == 1:
            yield (n,)
            return
        for a in range(n + 1):
            for rest in splits(n - a, parts - 1):
                yield (a, *rest)
    for n in range(1, 9):
        for experts in (1, 2, 3):
            for alignment in (1, 2, 3, 4):
                most = max(sum(oracle.align(c, alignment) for c in s) for s in splits(n, experts))
                assert most == oracle.moe_rows(n, experts, alignment), (n, experts, alignment)


def test_the_fp4_oracle_on_values_that_can_be_checked_by_hand():
    x = torch.zeros(1, 64)
    x[0, :9] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.3])
    x[0, 32] = 6.1                                                # one bit more than a scale of 1 allows
    code, byte, values = oracle.cast_fp4_ref(x, -1)
    assert code[0, :9].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 9]
    assert byte[0].tolist() == [127, 128] and values[0, 32] == 6.0 and code[0, 32] == 5
    code, byte, values = oracle.cast_fp4_ref(torch.tensor([[1e-30] * 32, [float('inf')] * 32, [0.0] * 32]), -1)
    assert byte[:, 0].tolist() == [25, 255, 1] and torch.isnan(values[1]).all() and (values[2] == 0).all()
    assert abs(values[0, 0].item() / 1e-30 - 1) <= 0.25
