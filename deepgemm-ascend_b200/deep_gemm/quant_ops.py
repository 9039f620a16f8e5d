"""Producers of block-scaled FP8 and FP4 operands whose scale factors come out in the layout the GEMM reads.

`swiglu_apply_weight_to_fp8` mirrors the reference's third-party/tilelang_ops/swiglu_apply_weight_to_fp8.py:411-449
(same arguments, same return pair); `cast_to_fp8` is the same kernel without the SwiGLU step and has no counterpart in
the reference. Both return `(out, out_sf)` with `out` E4M3 [tokens, hidden] and `out_sf` int16 [tokens, hidden / 64]
whose stride(0) == 1: pass them to `fp8_gemm_*` / `m_grouped_fp8_gemm_*` as `(out, out_sf)` with `recipe_a=(1, 32)`
and no scale-factor transform runs. `cast_to_fp4` does the same for packed E2M1, in both majors, and `cast_from_fp4` is the way back.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L
from ._api import MK_ALIGNMENT, _C, _ceil_div, _host_assert, _stream_ptr


def _launch(x, hidden, swiglu, topk_weights, psum, clamp_value, expert_alignment):
    tokens = x.size(0)
    out = torch.empty((tokens, hidden), dtype=torch.float8_e4m3fn, device=x.device)
    cols = (hidden // 32 + 1) // 2
    storage = torch.empty((cols, tokens), dtype=torch.int16, device=x.device)
    if tokens:
        if topk_weights is not None:
            _host_assert(topk_weights.dtype == torch.float32 and topk_weights.is_contiguous() and topk_weights.numel() == tokens,
                         'topk_weights must be a contiguous float32 tensor with one weight per token')
        if psum is not None:
            _host_assert(psum.dtype == torch.int32 and psum.dim() == 1 and psum.is_contiguous() and psum.device == x.device,
                         'psum_num_tokens_per_expert must be a contiguous int32 vector on the device of x')
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
    _host_assert(x.dim() == 2 and x.is_contiguous() and x.dtype == torch.bfloat16, 'x must be a contiguous 2-D BF16 tensor')
    _host_assert(x.size(1) % 256 == 0, 'the row length of x must be a multiple of 256')
    return _launch(x, x.size(1) // 2, True, topk_weights, psum_num_tokens_per_expert, clamp_value, expert_alignment)


def cast_to_fp8(x: torch.Tensor, psum_num_tokens_per_expert: Optional[torch.Tensor] = None, expert_alignment: int = 128):
    """x [tokens, hidden] BF16 -> (E4M3 [tokens, hidden], packed UE8M0 scales per 1x32)."""
    _host_assert(x.dim() == 2 and x.stride(1) == 1 and x.dtype == torch.bfloat16, 'x must be a row-major 2-D BF16 tensor')
    _host_assert(x.size(1) % 32 == 0, 'the row length of x must be a multiple of 32')
    return _launch(x, x.size(1), False, None, psum_num_tokens_per_expert, None, expert_alignment)


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
    cast_to_fp8, swiglu_apply_weight_to_fp8 = _C.cast_to_fp8, _C.swiglu_apply_weight_to_fp8
    cast_to_fp4, cast_from_fp4 = _C.cast_to_fp4, _C.cast_from_fp4
