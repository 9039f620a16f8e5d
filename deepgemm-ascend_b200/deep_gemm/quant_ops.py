"""Producers of block-scaled FP8 and FP4 operands whose scale factors come out in the layout the GEMM reads.

`swiglu_apply_weight_to_fp8` mirrors the reference's third-party/tilelang_ops/swiglu_apply_weight_to_fp8.py:411-449
(same arguments, same return pair); `cast_to_fp8` is the same kernel without the SwiGLU step and has no counterpart in
the reference. Both return `(out, out_sf)` with `out` E4M3 [tokens, hidden] and `out_sf` int16 [tokens, hidden / 64]
whose stride(0) == 1: pass them to `fp8_gemm_*` / `m_grouped_fp8_gemm_*` as `(out, out_sf)` with `recipe_a=(1, 32)`
and no scale-factor transform runs. `cast_to_fp4` does the same for packed E2M1, in both majors, and `cast_from_fp4` is the way back.

`rms_norm_to_fp8` is the step in front of a product: the residual's addition, the norm and the quantiser in one pass; `rms_norm_grad` is its
gradient. For training with 8-bit operands, `swiglu_apply_weight_to_fp8_with_checkpoint` keeps the input of SwiGLU in 8 bits in the same pass,
`swiglu_apply_weight_grad` reads it, and `cast_to_fp8(mn_major=True)` turns what was kept (or BF16) into the operands of a weight gradient,
whose contraction runs down the rows:

    (a2, kept) = swiglu_apply_weight_to_fp8_with_checkpoint(h1, w, psum, expert_alignment=256)
    dh1, dw = swiglu_apply_weight_grad(da2, kept, w, psum, expert_alignment=256)
    g, a = (cast_to_fp8(t, psum, 256, mn_major=True, min_amax=0) for t in (dh1, a1))       # a1: the 8-bit rows of the first product
    k_grouped_fp8_gemm_tn_contiguous(g, a, dw1, None, psum)

Gradients pass the rounding to 8 bits as if it were not there. None of these has a counterpart in the reference.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L
from ._api import MK_ALIGNMENT, _C, _ceil_div, _host_assert, _stream_ptr


_INT_MAX = 2 ** 31 - 1


def _is_float(t):
    return t.dtype in (torch.bfloat16, torch.float32)


def _row_stride(x):
    return x.stride(0) if x.size(0) > 1 else x.size(1)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _check_rows(topk_weights, psum, tokens, device):
    if topk_weights is not None:
        _host_assert(topk_weights.dtype == torch.float32 and topk_weights.is_contiguous() and topk_weights.numel() == tokens and topk_weights.device == device,
                     'topk_weights must be a contiguous float32 tensor with one weight per token')
    if psum is not None:
        _host_assert(psum.dtype == torch.int32 and psum.dim() == 1 and psum.is_contiguous() and psum.device == device,
                     'psum_num_tokens_per_expert must be a contiguous int32 vector on the device of x')


def _check_layout(psum, expert_alignment, multiple):
    """(an empty tensor has no address, and the C ABI takes a null pointer for no layout)"""
    if psum is not None:
        _host_assert(psum.numel() > 0, 'psum_num_tokens_per_expert must hold an expert')
        _host_assert(0 < expert_alignment <= _INT_MAX and expert_alignment % multiple == 0, f'expert_alignment must be a positive multiple of {multiple}')


def _check_clamp(clamp_value):
    _host_assert(clamp_value is None or clamp_value >= 0, 'clamp_value must not be negative')


def _launch(x, hidden, swiglu, topk_weights, psum, clamp_value, expert_alignment, min_amax=None):
    tokens = x.size(0)
    with torch.cuda.device(x.device):
        return _launch_on(x, tokens, hidden, swiglu, topk_weights, psum, clamp_value, expert_alignment, min_amax)


def _launch_on(x, tokens, hidden, swiglu, topk_weights, psum, clamp_value, expert_alignment, min_amax):
    out = torch.empty((tokens, hidden), dtype=torch.float8_e4m3fn, device=x.device)
    cols = (hidden // 32 + 1) // 2
    storage = torch.empty((cols, tokens), dtype=torch.int16, device=x.device)
    if tokens:
        _check_rows(topk_weights, psum, tokens, x.device)
        if min_amax is not None:
            L.check(L.lib().dg_cast_fp8_launch(
                x.data_ptr(), _row_stride(x), tokens, hidden, _ptr(psum), psum.numel() if psum is not None else 0, int(expert_alignment), float(min_amax),
                out.data_ptr(), hidden, storage.data_ptr(), tokens, _stream_ptr(x.device)))
            return out, storage.T
        L.check(L.lib().dg_quant_fp8_launch(
            x.data_ptr(), x.stride(0), tokens, hidden, int(swiglu),
            topk_weights.data_ptr() if topk_weights is not None else None,
            psum.data_ptr() if psum is not None else None, psum.numel() if psum is not None else 0, int(expert_alignment),
            int(clamp_value is not None), float(clamp_value or 0.0), out.data_ptr(), out.stride(0),
            storage.data_ptr(), tokens, _stream_ptr(x.device)))
    return out, storage.T


def swiglu_apply_weight_to_fp8(x: torch.Tensor, topk_weights: Optional[torch.Tensor] = None,
                               psum_num_tokens_per_expert: Optional[torch.Tensor] = None,
                               clamp_value: Optional[float] = None, expert_alignment: int = 128):
    """x [tokens, 2 * hidden] BF16 -> (E4M3 [tokens, hidden], packed UE8M0 scales) of
    silu(min(x_l, clamp)) * clamp(x_r, -clamp, clamp) * weight. Rows in the padding of the psum layout are not written."""
    _host_assert(x.is_cuda and x.dim() == 2 and x.is_contiguous() and x.dtype == torch.bfloat16, 'x must be a contiguous 2-D BF16 tensor on a CUDA device')
    _host_assert(x.size(1) % 256 == 0, 'the row length of x must be a multiple of 256')
    return _launch(x, x.size(1) // 2, True, topk_weights, psum_num_tokens_per_expert, clamp_value, expert_alignment)


def swiglu_apply_weight_to_fp8_with_checkpoint(x: torch.Tensor, topk_weights: Optional[torch.Tensor] = None,
                                               psum_num_tokens_per_expert: Optional[torch.Tensor] = None, clamp_value: Optional[float] = None,
                                               expert_alignment: int = 128, out=None):
    """`swiglu_apply_weight_to_fp8(x, ...)` and, from the same pass over x, x itself in 8 bits as `cast_to_fp8(x, ...)` makes it: ((out, out_sf),
    (kept, kept_sf)) with `kept` E4M3 [tokens, 2 * hidden]. The result is that of the BF16 x; `swiglu_apply_weight_grad` takes the
    second pair. Rows of x start on 16-byte boundaries. `out`: two such pairs to write to."""
    psum, hidden, tokens = psum_num_tokens_per_expert, x.size(-1) // 2, x.size(0)
    _host_assert(x.is_cuda and x.dim() == 2 and x.stride(1) == 1 and x.dtype == torch.bfloat16, 'x must be a row-major 2-D BF16 tensor on a CUDA device')
    _host_assert(x.size(1) % 256 == 0, 'the row length of x must be a multiple of 256')
    _host_assert(max(x.shape) <= _INT_MAX, 'x is too large')
    _check_rows(topk_weights, psum, tokens, x.device)
    _check_layout(psum, expert_alignment, 32)
    _check_clamp(clamp_value)
    with torch.cuda.device(x.device):
        if out is None:
            out = tuple((torch.empty((tokens, width), dtype=torch.float8_e4m3fn, device=x.device), _empty_scales((tokens, width // 64), x.device))
                        for width in (hidden, 2 * hidden))
        ((q, sf), (kept, kept_sf)) = out
        _check_fp8_out(q, sf, x, hidden)
        _check_fp8_out(kept, kept_sf, x, 2 * hidden)
        if x.numel():
            L.check(L.lib().dg_swiglu_checkpoint_launch(
                x.data_ptr(), _row_stride(x), tokens, hidden, _ptr(topk_weights), _ptr(psum), psum.numel() if psum is not None else 0, int(expert_alignment),
                int(clamp_value is not None), float(clamp_value or 0.0), q.data_ptr(), _row_stride(q), sf.data_ptr(), _scale_stride(sf),
                kept.data_ptr(), _row_stride(kept), kept_sf.data_ptr(), _scale_stride(kept_sf), _stream_ptr(x.device)))
    return (q, sf), (kept, kept_sf)


def _scale_stride(sf):
    return sf.stride(1) if sf.size(1) > 1 else sf.size(0)


def _is_scales(sf, rows, cols):
    """int16 [rows, cols], consecutive rows contiguous"""
    return sf.dtype == torch.int16 and tuple(sf.shape) == (rows, cols) and (sf.stride(0) == 1 or rows <= 1) and (cols <= 1 or sf.stride(1) >= rows)


def _check_fp8_out(q, sf, x, width):
    _host_assert(q.dtype == torch.float8_e4m3fn and q.device == x.device and tuple(q.shape) == (x.size(0), width) and q.stride(1) == 1 and _row_stride(q) >= width and
                 sf.device == x.device and _is_scales(sf, x.size(0), _ceil_div(width, 64)),
                 'out must hold E4M3 rows on the device of x and their int16 scales, one element for 64 channels of each row, contiguous along the rows')


def swiglu_apply_weight_grad(grad_out: torch.Tensor, x, topk_weights: Optional[torch.Tensor] = None,
                             psum_num_tokens_per_expert: Optional[torch.Tensor] = None, clamp_value: Optional[float] = None, expert_alignment: int = 128,
                             out: Optional[torch.Tensor] = None, zero_padding: bool = False):
    """Gradients of `swiglu_apply_weight_to_fp8` for grad_out BF16 [tokens, hidden]: (grad_x BF16 [tokens, 2 * hidden], grad_weights float32 like
    topk_weights, or None). x is the BF16 input or the 8-bit pair that `..._with_checkpoint` (or `cast_to_fp8`) made of it. Where the clamp cuts off
    the gradient is 0. What rows without a value (the padding of a psum layout, rows behind its last group) hold does not matter; their weights
    have the gradient 0, and grad_x is not written there, but for the zeros that `zero_padding` puts into the padding. `out`: where grad_x goes, which may overlap
    nothing else. Rows of BF16 start on 16-byte boundaries, those of E4M3 on 8. A NaN in x shows here whether there is a clamp or not; the forward pass takes minima
    and maxima, and makes the clamp of it."""
    psum, is_pair = psum_num_tokens_per_expert, isinstance(x, (tuple, list))
    x, sf = x if is_pair else (x, None)
    _host_assert(grad_out.is_cuda and grad_out.dim() == 2 and grad_out.stride(1) == 1 and grad_out.dtype == torch.bfloat16,
                 'grad_out must be a row-major 2-D BF16 tensor on a CUDA device')
    tokens, hidden = grad_out.shape
    _host_assert(hidden % 128 == 0, 'the row length of grad_out must be a multiple of 128')
    _host_assert(max(tokens, 2 * hidden) <= _INT_MAX, 'grad_out is too large')
    _host_assert(x.device == grad_out.device and tuple(x.shape) == (tokens, 2 * hidden) and x.stride(1) == 1 and
                 x.dtype == (torch.float8_e4m3fn if is_pair else torch.bfloat16),
                 'x must be a row-major [tokens, 2 * hidden] tensor on the device of grad_out: BF16, or E4M3 with its scales')
    if is_pair:
        _host_assert(sf.device == x.device and _is_scales(sf, tokens, 2 * hidden // 64),
                     'the scales of x must be int16, one element for 64 channels of each row, contiguous along the rows')
    _check_rows(topk_weights, psum, tokens, x.device)
    _check_layout(psum, expert_alignment, 32)
    _check_clamp(clamp_value)
    with torch.cuda.device(x.device):
        if out is not None:
            _host_assert(out.dtype == torch.bfloat16 and out.device == x.device and tuple(out.shape) == (tokens, 2 * hidden) and out.stride(1) == 1 and
                         _row_stride(out) >= 2 * hidden, 'out must be a row-major [tokens, 2 * hidden] BF16 tensor on the device of grad_out')
        else:
            out = torch.empty((tokens, 2 * hidden), dtype=torch.bfloat16, device=x.device)
        grad_weights = torch.empty_like(topk_weights) if topk_weights is not None else None
        nbytes = L.lib().dg_swiglu_grad_scratch_bytes(tokens, hidden) if topk_weights is not None else 0
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
        if x.numel():
            L.check(L.lib().dg_swiglu_grad_launch(
                grad_out.data_ptr(), _row_stride(grad_out), x.data_ptr(), _row_stride(x), _ptr(sf), _scale_stride(sf) if is_pair else 0, tokens, hidden,
                _ptr(topk_weights), _ptr(psum), psum.numel() if psum is not None else 0, int(expert_alignment), int(clamp_value is not None),
                float(clamp_value or 0.0), out.data_ptr(), _row_stride(out), _ptr(grad_weights), int(zero_padding), _ptr(scratch), nbytes,
                _stream_ptr(x.device)))
        elif grad_weights is not None:
            grad_weights.zero_()
    return out, grad_weights


def cast_to_fp8(x, psum_num_tokens_per_expert: Optional[torch.Tensor] = None, expert_alignment: int = 128, mn_major: bool = False, min_amax: float = 1e-4):
    """x [rows, cols] BF16 -> (E4M3 [rows, cols], packed UE8M0 scales), one scale per 32 values along K, in the layout that the GEMMs read:

      mn_major=False   K runs along the row. Scales int16 [rows, ceil(cols / 64)] with consecutive rows contiguous
      mn_major=True    K runs down the rows. Scales int16 [.., ceil(rows / 64), cols]: the operands that the "NN" and "TN" spellings take with K
                       in front (both sides of a weight gradient, weights for the gradient of the activations). x may have three
                       dimensions, [groups, rows, cols], and may be E4M3 rows with their scales along the row, the pair that the K-major
                       form (or `moe_dispatch_to_fp8`, `rms_norm_to_fp8`, a SwiGLU) made: what a forward pass has kept in 8 bits

    The scale is the smallest power of two s (2^-126 or more) with max(amax, min_amax) <= 448 s; gradients want a min_amax below their own
    size, or 0. A block that holds an infinity (or, with mn_major, a NaN) gets the scale NaN. Rows in the padding of a psum layout are not
    written; with mn_major they count as zeros and are written as zeros. `expert_alignment` is a multiple of 32, or of 64 with mn_major."""
    psum = psum_num_tokens_per_expert
    if not mn_major:
        _host_assert(isinstance(x, torch.Tensor) and x.is_cuda and x.dim() == 2 and x.stride(1) == 1 and x.dtype == torch.bfloat16,
                     'x must be a row-major 2-D BF16 tensor on a CUDA device')
        _host_assert(x.size(1) % 32 == 0, 'the row length of x must be a multiple of 32')
        return _launch(x, x.size(1), False, None, psum, None, expert_alignment, min_amax)
    is_pair = isinstance(x, (tuple, list))
    x, x_sf = x if is_pair else (x, None)
    _host_assert(x.is_cuda and x.dim() in (2, 3) and x.stride(-1) == 1 and x.dtype == (torch.float8_e4m3fn if is_pair else torch.bfloat16),
                 'x must be a row-major 2-D or 3-D tensor on a CUDA device: BF16, or E4M3 with its scales')
    groups, rows, cols = x.size(0) if x.dim() == 3 else 1, x.size(-2), x.size(-1)
    _host_assert(cols % 32 == 0, 'the row length of x must be a multiple of 32')
    _host_assert(max(groups, rows, cols) <= _INT_MAX, 'x is too large')
    if is_pair:
        _check_scales(x, x_sf, groups, rows, _ceil_div(cols, 64), False)
    _check_rows(None, psum, rows, x.device)
    _check_layout(psum, expert_alignment, 64)
    _host_assert(psum is None or x.dim() == 2, 'a psum layout needs a 2-D x')
    k64 = _ceil_div(rows, 64)
    with torch.cuda.device(x.device):
        out = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
        sf = torch.empty((*x.shape[:-2], k64, cols), dtype=torch.int16, device=x.device)
        if x.numel():
            L.check(L.lib().dg_quant_fp8_mn_launch(
                x.data_ptr(), x.stride(-2) if rows > 1 else cols, x.stride(0) if groups > 1 else 0, _ptr(x_sf),
                (x_sf.stride(-1) if cols > 64 else rows) if is_pair else 0, x_sf.stride(0) if is_pair and groups > 1 else 0, groups, rows, cols,
                _ptr(psum), psum.numel() if psum is not None else 0, int(expert_alignment), float(min_amax),
                out.data_ptr(), cols, rows * cols, sf.data_ptr(), cols, k64 * cols, _stream_ptr(x.device)))
    return out, sf


def _check_scales(x, sf, groups, run, k64, mn_major):
    """`run`: the scales' length along MN"""
    along_k, along_mn = (-2, -1) if mn_major else (-1, -2)
    _host_assert(sf.dtype == torch.int16 and sf.device == x.device and sf.dim() == x.dim() and (sf.dim() == 2 or sf.size(0) == groups) and
                 sf.size(along_k) == k64 and sf.size(along_mn) == run,
                 'the scales must be packed int16 on the device of x, one byte for each 32 values along K')
    _host_assert(sf.stride(along_mn) == 1 or run <= 1, 'the scales must be contiguous along MN')


def cast_from_fp8(x, out_dtype: torch.dtype = torch.bfloat16, mn_major: bool = False):
    """The pair that `cast_to_fp8` makes (or any E4M3 operand with packed scales) -> [.., rows, cols] BF16 or FP32: the values that a product with it
    sees, code times scale. (What lies beyond FP32, such as the -2^128 that the lowest BF16 number becomes, is an infinity.)"""
    codes, sf = x
    _host_assert(codes.is_cuda and codes.dim() in (2, 3) and codes.dtype == torch.float8_e4m3fn and codes.stride(-1) == 1,
                 'x must be a row-major 2-D or 3-D E4M3 tensor on a CUDA device, with its scales')
    _host_assert(out_dtype in (torch.bfloat16, torch.float32), 'out_dtype must be bf16 or fp32')
    groups, rows, cols = codes.size(0) if codes.dim() == 3 else 1, codes.size(-2), codes.size(-1)
    _host_assert(cols % 32 == 0, 'the row length of x must be a multiple of 32')
    _host_assert(max(groups, rows, cols) <= _INT_MAX, 'x is too large')
    k64, run = _ceil_div(rows if mn_major else cols, 64), cols if mn_major else rows
    _check_scales(codes, sf, groups, run, k64, mn_major)
    with torch.cuda.device(codes.device):
        out = torch.empty(codes.shape, dtype=out_dtype, device=codes.device)
        if out.numel():
            L.check(L.lib().dg_dequant_fp8_launch(
                codes.data_ptr(), codes.stride(-2) if rows > 1 else cols, codes.stride(0) if groups > 1 else 0, sf.data_ptr(),
                sf.stride(-2 if mn_major else -1) if k64 > 1 else run, sf.stride(0) if groups > 1 else 0, groups, rows, cols, int(mn_major),
                out.data_ptr(), int(out_dtype == torch.float32), cols, rows * cols, _stream_ptr(codes.device)))
    return out


def rms_norm_to_fp8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6, with_rows: bool = False,
                    out_h: Optional[torch.Tensor] = None):
    """x [tokens, hidden] BF16 or FP32 -> ((out, out_sf), rows, h, rstd):

        h = x + residual             rounded to the type of x (x itself without a residual)
        rstd = 1 / sqrt(mean(h^2) + eps)                     float32 [tokens]
        y = h * rstd * weight        (out, out_sf): y as `cast_to_fp8` quantises it, but from FP32; rows: y in BF16 `with_rows`, else None

    weight: BF16 or FP32 [hidden]. The sum of squares is held in 64 bits: a token's results do not depend on how many others there are. `out_h`:
    where h goes with a residual, which may be `residual` or x itself. hidden is a multiple of 32, at most 16384; rows start on 16-byte boundaries.
    out_sf and rstd may share one allocation: keeping rstd keeps the scales."""
    _host_assert(x.is_cuda and x.dim() == 2 and x.stride(1) == 1 and _is_float(x), 'x must be a row-major 2-D BF16 or FP32 tensor on a CUDA device')
    tokens, hidden = x.shape
    _check_norm(x, weight, tokens, hidden)
    for name, t in (('residual', residual), ('out_h', out_h)):
        if t is not None:
            _host_assert(t.dtype == x.dtype and t.device == x.device and t.shape == x.shape and t.stride(1) == 1 and (name == 'residual' or _row_stride(t) >= hidden),
                         f'{name} must be row-major, of the type, the shape and the device of x')
    _host_assert(out_h is None or residual is not None, 'out_h needs a residual')
    with torch.cuda.device(x.device):
        q = torch.empty((tokens, hidden), dtype=torch.float8_e4m3fn, device=x.device)
        sf = _empty_scales((tokens, _ceil_div(hidden, 64)), x.device)
        rows = torch.empty((tokens, hidden), dtype=torch.bfloat16, device=x.device) if with_rows else None
        h = x if residual is None else out_h if out_h is not None else torch.empty((tokens, hidden), dtype=x.dtype, device=x.device)
        rstd = torch.empty(tokens, dtype=torch.float32, device=x.device)
        if tokens:
            L.check(L.lib().dg_rms_norm_fp8_launch(
                x.data_ptr(), int(x.dtype == torch.float32), _row_stride(x), _ptr(residual), _row_stride(residual) if residual is not None else 0,
                h.data_ptr(), _row_stride(h), weight.data_ptr(), int(weight.dtype == torch.float32), float(eps), tokens, hidden, q.data_ptr(), hidden,
                sf.data_ptr(), tokens, _ptr(rows), hidden, rstd.data_ptr(), _stream_ptr(x.device)))
    return (q, sf), rows, h, rstd


def _check_norm(x, weight, tokens, hidden):
    _host_assert(hidden > 0 and hidden % 32 == 0 and hidden <= 16384, 'the row length must be a multiple of 32, at most 16384')
    _host_assert(tokens <= _INT_MAX, 'there are too many tokens')
    _host_assert(weight.device == x.device and _is_float(weight) and weight.dim() == 1 and weight.size(0) == hidden and weight.is_contiguous(),
                 'weight must be a contiguous BF16 or FP32 vector of the row length, on the device of the rows')


def rms_norm_grad(grad_out: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor, grad_h: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None):
    """Gradients of the norm of `rms_norm_to_fp8` for grad_out [tokens, hidden] (of its y; BF16, or FP32 beside an FP32 h): (grad_x like h, grad_weight
    float32 [hidden]). grad_h: the gradient that reaches h by the residual stream, in the type of h, which is added; grad_x is the gradient
    of x and of the residual alike. `out`: where grad_x goes; it may be grad_h, h or grad_out itself."""
    _host_assert(h.is_cuda and h.dim() == 2 and h.stride(1) == 1 and _is_float(h), 'h must be a row-major 2-D BF16 or FP32 tensor on a CUDA device')
    tokens, hidden = h.shape
    _check_norm(h, weight, tokens, hidden)
    _host_assert(grad_out.device == h.device and grad_out.shape == h.shape and grad_out.stride(1) == 1 and grad_out.dtype in (h.dtype, torch.bfloat16),
                 'grad_out must be row-major, of the shape and the device of h, BF16 or of the type of h')
    _host_assert(rstd.device == h.device and rstd.dtype == torch.float32 and tuple(rstd.shape) == (tokens,) and rstd.is_contiguous(),
                 'rstd must be a contiguous float32 vector with one value per token, on the device of h')
    for name, t in (('grad_h', grad_h), ('out', out)):
        if t is not None:
            _host_assert(t.dtype == h.dtype and t.device == h.device and t.shape == h.shape and t.stride(1) == 1 and (name == 'grad_h' or _row_stride(t) >= hidden),
                         f'{name} must be row-major, of the type, the shape and the device of h')
    with torch.cuda.device(h.device):
        if out is None:
            out = torch.empty((tokens, hidden), dtype=h.dtype, device=h.device)
        grad_weight = torch.empty(hidden, dtype=torch.float32, device=h.device)
        nbytes = L.lib().dg_rms_norm_grad_scratch_bytes(tokens, hidden)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=h.device)
        L.check(L.lib().dg_rms_norm_grad_launch(
            _ptr(grad_out), int(grad_out.dtype == torch.float32), _row_stride(grad_out), _ptr(h), int(h.dtype == torch.float32), _row_stride(h), weight.data_ptr(),
            int(weight.dtype == torch.float32), _ptr(rstd), _ptr(grad_h), _row_stride(grad_h) if grad_h is not None else 0, tokens, hidden,
            out.data_ptr(), _row_stride(out), grad_weight.data_ptr(), _ptr(scratch), nbytes, _stream_ptr(h.device)))
    return out, grad_weight


def _empty_scales(shape, device):
    """Packed scales [.., rows, cols] with consecutive rows contiguous."""
    rows, cols = max(shape[-2], 1), max(shape[-1], 1)
    return torch.empty_strided(shape, (rows * cols, 1, rows)[-len(shape):], dtype=torch.int16, device=device)


def cast_to_fp4(x: torch.Tensor, psum_num_tokens_per_expert: Optional[torch.Tensor] = None, expert_alignment: int = MK_ALIGNMENT, mn_major: bool = False):
    """x [rows, cols] or [groups, rows, cols] BF16 or FP32 -> (packed E2M1 int8 [.., rows, cols / 2], packed UE8M0 scales), one scale per
    32 values along K, in the layout that the GEMMs read:

      mn_major=False   K runs along the row. Scales int16 [.., rows, ceil(cols / 64)] with consecutive rows contiguous: either operand of
                       an "NT" GEMM, the experts' weights of a grouped one
      mn_major=True    K runs down the rows. Scales int16 [.., ceil(rows / 64), cols]: the operands that the "NN" and "TN" spellings
                       take with K in front (weights for the gradient of the activations, both sides of a weight gradient)

    The scale is the smallest power of two with which the block's largest magnitude is at most 6 (2^-126 or more); values are rounded to the
    nearest code, halves to the even one. A block that holds an infinity or a NaN gets the scale NaN. Rows in the padding of a psum layout
    are not written; with mn_major they count as zeros and are written as zeros. `expert_alignment` is that of the layout, the one of `moe_sort` and
    the grouped GEMMs if it is not given: a multiple of 32, or of 64 with mn_major."""
    _host_assert(x.is_cuda and x.dim() in (2, 3) and x.stride(-1) == 1 and x.dtype in (torch.bfloat16, torch.float32),
                 'x must be a row-major 2-D or 3-D BF16 or FP32 tensor on a CUDA device')
    groups, rows, cols = x.size(0) if x.dim() == 3 else 1, x.size(-2), x.size(-1)
    _host_assert(cols % 32 == 0, 'the row length of x must be a multiple of 32')
    _host_assert(max(groups, rows, cols) < 2 ** 31, 'x is too large')
    psum = psum_num_tokens_per_expert
    if psum is not None:
        _host_assert(psum.dtype == torch.int32 and psum.dim() == 1 and psum.is_contiguous() and psum.device == x.device,
                     'psum_num_tokens_per_expert must be a contiguous int32 vector on the device of x')
        _host_assert(psum.numel() > 0, 'psum_num_tokens_per_expert must hold an expert')
        _host_assert(x.dim() == 2, 'a psum layout needs a 2-D x')
        _host_assert(0 < expert_alignment < 2 ** 31 and expert_alignment % (64 if mn_major else 32) == 0,
                     'expert_alignment must be a positive multiple of 32 (64 when mn_major)')
    with torch.cuda.device(x.device):
        out = torch.empty((*x.shape[:-1], cols // 2), dtype=torch.int8, device=x.device)
        k64, run = _ceil_div(rows if mn_major else cols, 64), cols if mn_major else rows
        sf = (torch.empty((*x.shape[:-2], k64, cols), dtype=torch.int16, device=x.device) if mn_major else
              _empty_scales((*x.shape[:-1], k64), x.device))
        if x.numel():
            L.check(L.lib().dg_quant_fp4_launch(
                x.data_ptr(), int(x.dtype == torch.float32), x.stride(-2) if rows > 1 else cols, x.stride(0) if groups > 1 else 0, groups, rows, cols,
                int(mn_major), psum.data_ptr() if psum is not None else None, psum.numel() if psum is not None else 0, int(expert_alignment),
                out.data_ptr(), cols // 2, rows * (cols // 2), sf.data_ptr(), run, k64 * run, _stream_ptr(x.device)))
    return out, sf


def cast_from_fp4(x, out_dtype: torch.dtype = torch.bfloat16, mn_major: bool = False):
    """The pair that `cast_to_fp4` makes (or the quantised weights of a GEMM) -> [.., rows, cols] BF16 or FP32: the values that a product with
    it sees, code times scale."""
    codes, sf = x
    _host_assert(codes.is_cuda and codes.dim() in (2, 3) and codes.dtype == torch.int8 and codes.stride(-1) == 1,
                 'x must be a row-major 2-D or 3-D tensor of packed FP4 on a CUDA device, with its scales')
    _host_assert(out_dtype in (torch.bfloat16, torch.float32), 'out_dtype must be bf16 or fp32')
    groups, rows, cols = codes.size(0) if codes.dim() == 3 else 1, codes.size(-2), codes.size(-1) * 2
    _host_assert(cols % 32 == 0, 'the row length of x must be a multiple of 32')
    _host_assert(max(groups, rows, cols) < 2 ** 31, 'x is too large')
    k64, run = _ceil_div(rows if mn_major else cols, 64), cols if mn_major else rows
    along_k, along_mn = (-2, -1) if mn_major else (-1, -2)
    _host_assert(sf.dtype == torch.int16 and sf.device == codes.device and sf.dim() == codes.dim() and (sf.dim() == 2 or sf.size(0) == groups) and
                 sf.size(along_k) == k64 and sf.size(along_mn) == run,
                 'the scales must be packed int16 on the device of x, one byte for each 32 values along K')
    _host_assert(sf.stride(along_mn) == 1 or run <= 1, 'the scales must be contiguous along MN')
    with torch.cuda.device(codes.device):
        out = torch.empty((*codes.shape[:-1], cols), dtype=out_dtype, device=codes.device)
        if out.numel():
            L.check(L.lib().dg_dequant_fp4_launch(
                codes.data_ptr(), codes.stride(-2) if rows > 1 else cols // 2, codes.stride(0) if groups > 1 else 0, sf.data_ptr(),
                sf.stride(along_k) if k64 > 1 else run, sf.stride(0) if groups > 1 else 0, groups, rows, cols, int(mn_major),
                out.data_ptr(), int(out_dtype == torch.float32), cols, rows * cols, _stream_ptr(codes.device)))
    return out


# The compiled host layer has the same functions (csrc/apis/quant.hpp): 5 to 6 us of host time a call instead of 15.
if _C is not None:
    cast_to_fp8, cast_from_fp8, swiglu_apply_weight_to_fp8 = _C.cast_to_fp8, _C.cast_from_fp8, _C.swiglu_apply_weight_to_fp8
    swiglu_apply_weight_to_fp8_with_checkpoint, swiglu_apply_weight_grad = _C.swiglu_apply_weight_to_fp8_with_checkpoint, _C.swiglu_apply_weight_grad
    rms_norm_to_fp8, rms_norm_grad = _C.rms_norm_to_fp8, _C.rms_norm_grad
    cast_to_fp4, cast_from_fp4 = _C.cast_to_fp4, _C.cast_from_fp4
