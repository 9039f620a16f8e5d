"""Microscaled 4-bit quantisation and the way back, bit for bit against 64 bits on the CPU (oracle/quant.py: the only rounding is the one to
the code), and the products that take the result."""

import pytest
import torch

import deep_gemm
import oracle
from both_hosts import python_layer, quant_hosts
from helpers import assert_close, seed_all

pytestmark = pytest.mark.gpu


def _codes(packed):
    u = packed.cpu().contiguous().view(torch.uint8)
    return torch.stack((u & 15, u >> 4), dim=-1).flatten(-2)


def _bytes(sf, axis):
    """Packed scales -> bytes, two for each element along `axis`."""
    s = sf.cpu().to(torch.int32).movedim(axis, -1)
    return torch.stack((s & 255, (s >> 8) & 255), dim=-1).flatten(-2).to(torch.uint8).movedim(-1, axis)


def _check(x, mn_major, host=deep_gemm, on=None):
    axis = -2 if mn_major else -1
    out, sf = host.cast_to_fp4(x.cuda() if on is None else on, mn_major=mn_major)
    code, byte, values = oracle.cast_fp4_ref(x, axis)
    rows, cols = x.shape[-2:]
    blocks = byte.size(axis)
    assert out.dtype == torch.int8 and out.shape == (*x.shape[:-1], cols // 2) and out.is_contiguous() and sf.dtype == torch.int16
    got = _bytes(sf, axis)
    assert torch.equal(got.narrow(axis, 0, blocks), byte)
    assert (got.narrow(axis, blocks, got.size(axis) - blocks) == 0).all()          # behind the last block
    if mn_major:
        assert sf.shape == (*x.shape[:-2], oracle.ceil_div(rows, 64), cols) and sf.is_contiguous()
    else:
        assert sf.shape == (*x.shape[:-2], rows, oracle.ceil_div(cols, 64)) and sf.transpose(-2, -1).is_contiguous()
    finite = byte.ne(255).repeat_interleave(32, axis).narrow(axis, 0, x.size(axis))
    assert torch.equal(_codes(out)[finite], code[finite])
    for dtype in (torch.float32, torch.bfloat16):
        back = host.cast_from_fp4((out, sf), out_dtype=dtype, mn_major=mn_major)
        assert back.dtype == dtype and back.shape == x.shape
        # (a code times a scale may pass the type's range, as 4 x 2^126 does: an infinity then, on both sides)
        assert torch.equal(torch.isnan(back).cpu(), torch.isnan(values)) and torch.equal(back.cpu()[values == values], values.to(dtype)[values == values])


SHAPES = [(1, 32), (5, 64), (31, 96), (32, 256), (33, 288), (64, 2048), (65, 544), (100, 7168), (1000, 160), (2, 65568)]


@pytest.mark.parametrize('host', quant_hosts)
@pytest.mark.parametrize('mn_major', [False, True])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('rows,cols', SHAPES)
def test_round_trip(host, mn_major, dtype, rows, cols):
    seed_all(rows + cols)
    x = (torch.randn(rows, cols) * torch.exp2(torch.randint(-20, 20, (rows, cols // 32)).float()).repeat_interleave(32, 1)).to(dtype)
    x[0, :16] = 0
    x[-1, -32:] = 0
    _check(x, mn_major, host)


@pytest.mark.parametrize('mn_major', [False, True])
def test_every_tie_and_border(mn_major):
    """All halves between neighbouring codes and what lies one BF16 or FP32 step beside them, at scales from subnormal to huge; a largest
    magnitude of exactly 6 s and one step above."""
    base = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 4.0, 0.5])
    for dtype in (torch.bfloat16, torch.float32):
        step = torch.finfo(dtype).eps
        near = torch.cat([base, base * (1 + step), base * (1 - step / 2)])
        near = torch.cat([near, -near])
        blocks = []
        for k in (-133, -128, -126, -100, -1, 0, 3, 120, 124):
            for top in (6.0, 6.0 * (1 + step), 4.0, 3.0 + 1e-6):
                b = torch.zeros(64, dtype=torch.float64)
                b[:60] = near.double()
                b[(b.abs() > top)] = 0.0
                b[60] = top
                blocks.append(torch.cat([b[:31], b[60:61], b[31:62]])[:64] * 2.0 ** k)
        x = torch.stack([torch.nn.functional.pad(b, (0, 64 - b.numel())) for b in blocks]).to(dtype)
        _check(x.t().contiguous()[:, :32].contiguous() if mn_major else x, mn_major)
        _check(x if not mn_major else x.repeat(1, 1).t().contiguous()[:, -32:].contiguous(), mn_major)


@pytest.mark.parametrize('mn_major', [False, True])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_what_is_not_finite_becomes_a_scale_of_nan(mn_major, dtype):
    seed_all(4)
    x = torch.randn(96, 128).to(dtype)
    x[3, 5], x[40, 70], x[64, 127] = float('inf'), float('nan'), -float('inf')
    x[70] = torch.finfo(dtype).max
    x[71] = torch.finfo(dtype).tiny
    _check(x, mn_major)


@pytest.mark.parametrize('mn_major', [False, True])
def test_groups_and_strides(mn_major):
    seed_all(8)
    wide = torch.randn(3, 80, 512)
    for dtype in (torch.bfloat16, torch.float32):
        x = wide.to(dtype)[:, 10:77, 64:288]
        _check(x, mn_major, on=wide.to(dtype).cuda()[:, 10:77, 64:288])
        _check(x[1], mn_major, on=wide.to(dtype).cuda()[1, 10:77, 64:288])
    x = wide.bfloat16()[:, :64].contiguous()
    codes, sf = deep_gemm.cast_to_fp4(x.cuda(), mn_major=mn_major)
    # codes and scales as views of wider tensors
    room = torch.zeros(3, 64, 300, dtype=torch.int8, device='cuda')
    room[:, :, 4:260] = codes
    sf_room = torch.zeros(3, sf.size(1 if mn_major else 2) + 1, sf.size(2 if mn_major else 1) + 6, dtype=torch.int16, device='cuda')
    sf_view = sf_room[:, 1:, 6:] if mn_major else sf_room[:, 1:, 6:].transpose(1, 2)
    sf_view.copy_(sf)
    assert torch.equal(deep_gemm.cast_from_fp4((room[:, :, 4:260], sf_view), mn_major=mn_major), deep_gemm.cast_from_fp4((codes, sf), mn_major=mn_major))


@pytest.mark.parametrize('mn_major', [False, True])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_many_matrices_give_what_each_gives(mn_major, dtype):
    """Enough of them for the larger tiles of the way back, and more than a grid holds."""
    seed_all(14)
    for shape in ((600, 67, 1056), (70001, 3, 32)):
        x = torch.randn(shape, device='cuda', dtype=dtype)
        codes, sf = deep_gemm.cast_to_fp4(x, mn_major=mn_major)
        back = deep_gemm.cast_from_fp4((codes, sf), out_dtype=dtype, mn_major=mn_major)
        for g in (*range(0, 600, 37), *range(65530, 65540), shape[0] - 1):
            if g >= shape[0]:
                continue
            one, one_sf = deep_gemm.cast_to_fp4(x[g], mn_major=mn_major)
            assert torch.equal(codes[g], one) and torch.equal(sf[g], one_sf), g
            assert torch.equal(back[g], deep_gemm.cast_from_fp4((one, one_sf), out_dtype=dtype, mn_major=mn_major)), g
            if g < 74:
                _check(x[g].cpu(), mn_major)


@pytest.mark.parametrize('mn_major,alignment', [(False, 32), (False, 256), (True, 64), (True, 256)])
def test_psum_layout(mn_major, alignment):
    seed_all(alignment)
    sizes = [100, 0, 33, 1, 256, 31] + [7] * 40
    total, psum = oracle.make_psum_layout(sizes, alignment)
    rows = total + 96                                             # and rows behind the last group
    x = torch.randn(rows, 288)
    valid = torch.zeros(rows, dtype=torch.bool)
    for span in oracle.psum_valid_spans(psum, alignment):
        valid[span] = True
    x[~valid] = float('nan')
    layout = torch.tensor(psum, dtype=torch.int32, device='cuda')
    on = x.cuda()
    out, sf = deep_gemm.cast_to_fp4(on, layout, alignment, mn_major=mn_major)
    code, byte, _ = oracle.cast_fp4_ref(x, -2 if mn_major else -1, valid)
    if mn_major:
        assert torch.equal(_codes(out)[:total], code[:total])
        used = byte[:total // 32].clone()
        assert torch.equal(_bytes(sf, -2)[:total // 32], used)
    else:
        assert torch.equal(_codes(out)[valid], code[valid]) and torch.equal(_bytes(sf, -1)[valid][:, :9], byte[valid])
    # what is not to be written is left as it was
    from deep_gemm import _lib as L
    mark, mark_sf = torch.full_like(out, 0x5a), torch.full_like(sf.contiguous() if mn_major else sf.t().contiguous(), 0x1111)
    L.check(L.lib().dg_quant_fp4_launch(on.data_ptr(), 1, 288, 0, 1, rows, 288, int(mn_major), layout.data_ptr(), len(psum), alignment, mark.data_ptr(),
                                        144, 0, mark_sf.data_ptr(), mark_sf.size(1), 0, torch.cuda.current_stream().cuda_stream))
    if mn_major:
        assert (mark[total:] == 0x5a).all() and (mark_sf[oracle.ceil_div(total, 64):] == 0x1111).all()
    else:
        assert (mark[(~valid).cuda()] == 0x5a).all() and (mark_sf.t()[(~valid).cuda()] == 0x1111).all()


def test_empty_and_refused():
    for host in quant_hosts:
        for shape in ((0, 64), (4, 0, 64), (0, 4, 64), (4, 0)):
            out, sf = host.cast_to_fp4(torch.empty(shape, device='cuda'))
            assert out.shape == (*shape[:-1], shape[-1] // 2)
            assert host.cast_from_fp4((out, sf)).shape == shape
        bad = lambda match: pytest.raises(RuntimeError, match=match)  # noqa: E731
        x = torch.zeros(64, 64, device='cuda')
        with bad('BF16 or FP32'):
            host.cast_to_fp4(x.half())
        with bad('row-major'):
            host.cast_to_fp4(x.t()[:, :32])
        with bad('multiple of 32'):
            host.cast_to_fp4(x[:, :48])
        with bad('16-byte boundaries'):
            host.cast_to_fp4(torch.zeros(64, 65, device='cuda')[:, 1:])
        psum = torch.tensor([64], dtype=torch.int32, device='cuda')
        with bad('contiguous int32 vector'):
            host.cast_to_fp4(x, psum.long())
        with bad('needs a 2-D x'):
            host.cast_to_fp4(x[None], psum)
        for mn_major, alignment in ((False, 48), (True, 96), (False, 0)):
            with bad('multiple of 32'):
                host.cast_to_fp4(x, psum, alignment, mn_major=mn_major)
        codes, sf = host.cast_to_fp4(x)
        with bad('out_dtype must be bf16 or fp32'):
            host.cast_from_fp4((codes, sf), out_dtype=torch.float16)
        with bad('one byte for each 32 values'):
            host.cast_from_fp4((codes, sf[:32]))
        with bad('packed FP4'):
            host.cast_from_fp4((x, sf))
        codes, sf = host.cast_to_fp4(torch.zeros(64, 128, device='cuda'))
        with bad('contiguous along MN'):
            host.cast_from_fp4((codes, sf.contiguous()))
        with bad('4-byte boundaries'):
            host.cast_from_fp4((torch.zeros(64, 65, dtype=torch.int8, device='cuda')[:, 1:], sf))


# ---------------------------------------------------------------------------------------------------------- the products
def _values(x, axis):
    return oracle.cast_fp4_ref(x, axis)[2].float()


@pytest.mark.parametrize('m,n,k', [(1, 256, 512), (64, 384, 1024), (300, 512, 2080)])
def test_products_take_the_result_in_every_spelling(m, n, k):
    seed_all(m)
    a, b = torch.randn(m, k), torch.randn(n, k) * k ** -0.5
    ref = oracle.gemm_ref(_values(a, -1), _values(b, -1), torch.bfloat16)
    a_nt, b_nt = deep_gemm.cast_to_fp4(a.cuda()), deep_gemm.cast_to_fp4(b.cuda())
    b_nn = deep_gemm.cast_to_fp4(b.t().contiguous().cuda(), mn_major=True)
    d = torch.full((m, n), float('nan'), dtype=torch.bfloat16, device='cuda')
    deep_gemm.fp8_fp4_gemm_nt(a_nt, b_nt, d)
    assert_close(d, ref, 'nt')
    d.fill_(float('nan'))
    deep_gemm.fp8_fp4_gemm_nn(a_nt, b_nn, d)
    assert_close(d, ref, 'nn')
    if m % 32 == 0:
        a_tn = deep_gemm.cast_to_fp4(a.t().contiguous().cuda(), mn_major=True)
        d.fill_(float('nan'))
        deep_gemm.fp8_fp4_gemm_tn(a_tn, b_nn, d)
        assert_close(d, ref, 'tn')
    a8 = deep_gemm.cast_to_fp8(a.bfloat16().cuda())
    a8_values = oracle.swiglu_quant_ref(a.bfloat16(), swiglu=False)[3]
    d.fill_(float('nan'))
    deep_gemm.fp8_fp4_gemm_nt(a8, b_nt, d)
    assert_close(d, oracle.gemm_ref(a8_values, _values(b, -1), torch.bfloat16), 'fp8 x fp4')
    assert deep_gemm.device_status() == 0


def test_a_block_with_a_nan_shows_in_the_product():
    seed_all(2)
    a, b = torch.randn(64, 512), torch.randn(128, 512)
    a[5, 100], a[9, 300] = float('nan'), float('inf')
    d = torch.zeros(64, 128, dtype=torch.bfloat16, device='cuda')
    deep_gemm.fp8_fp4_gemm_nt(deep_gemm.cast_to_fp4(a.cuda()), deep_gemm.cast_to_fp4(b.cuda()), d)
    bad = torch.zeros(64, dtype=torch.bool)
    bad[[5, 9]] = True
    assert torch.isnan(d.cpu()[bad]).all() and torch.isfinite(d.cpu()[~bad]).all()


def test_the_weight_gradient_of_experts_in_fp4():
    """K holds the experts' tokens: both sides quantised down the rows, rows of the padding and behind the last group hold NaN."""
    seed_all(6)
    idx = torch.rand(200, 6).topk(3, dim=1).indices
    plan = deep_gemm.moe_sort(idx.cuda(), 5)
    rows, psum = plan[2].numel(), plan[0].cpu().tolist()
    valid = plan[2].cpu() >= 0
    x, dy = torch.randn(rows, 256), torch.randn(rows, 384)
    for t in (x, dy):
        t[~valid] = float('nan')
    a, b = (deep_gemm.cast_to_fp4(t.cuda(), plan[0], 256, mn_major=True) for t in (dy, x))
    for dtype in (torch.float32, torch.bfloat16):
        d = torch.full((5, 384, 256), float('nan'), dtype=dtype, device='cuda')
        deep_gemm.k_grouped_fp8_gemm_tn_contiguous(a, b, d, None, plan[0])
        assert deep_gemm.device_status() == 0
        total = oracle.align(psum[-1], 256)
        ref = oracle.k_grouped_psum_ref(*(oracle.cast_fp4_ref(t, -2, valid)[2].float()[:total] for t in (dy, x)), psum, dtype)
        assert_close(d, ref, 'weight gradient')


def test_another_stream_and_a_captured_run():
    seed_all(12)
    x = torch.randn(130, 512, device='cuda')
    ways = [lambda v, m=m: (*deep_gemm.cast_to_fp4(v, mn_major=m), deep_gemm.cast_from_fp4(deep_gemm.cast_to_fp4(v, mn_major=m), mn_major=m)) for m in (False, True)]
    for way in ways:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = way(x)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(there, way(x)))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = way(x)
        x.copy_(torch.randn(130, 512))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, way(x.clone())))


def test_offsets_beyond_32_bits():
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip('needs 40 GB')
    rows, cols = 600000, 7168
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device='cuda')
    x[-64:] = torch.randn(64, cols, device='cuda')
    for mn_major in (False, True):
        tail, tail_sf = deep_gemm.cast_to_fp4(x[-64:].clone(), mn_major=mn_major)
        codes, sf = deep_gemm.cast_to_fp4(x, mn_major=mn_major)
        assert torch.equal(codes[-64:], tail) and torch.equal(sf[-1:] if mn_major else sf[-64:], tail_sf)
        back = deep_gemm.cast_from_fp4((codes, sf), mn_major=mn_major)
        assert torch.equal(back[-64:], deep_gemm.cast_from_fp4((tail, tail_sf), mn_major=mn_major)) and (back[:-64].view(torch.int16).amax() == 0)
        del codes, sf, back


def test_both_host_layers_give_the_same_bits():
    seed_all(13)
    layer = python_layer('quant_ops')
    x = torch.randn(2, 70, 320, device='cuda')
    for mn_major in (False, True):
        for a, b in zip(deep_gemm.cast_to_fp4(x, mn_major=mn_major), layer.cast_to_fp4(x, mn_major=mn_major)):
            assert a.shape == b.shape and a.stride() == b.stride() and torch.equal(a, b)
