"""From the router's choices to the rows of a grouped layout and back: the steps in front of and behind the m-grouped GEMMs.

`moe_sort` orders the choices of a batch (the result of a top-k over the router's scores) by expert and answers a plan,
`(layout, token_rows, row_choices)`:

    layout        int32 [experts]      what the m-grouped GEMMs take as `grouped_layout` (psum layout) or `masked_m` (with `max_m`)
    token_rows    int32 [tokens, k]    the row of every choice; -1 where it has none (an expert outside [0, experts), such as the -1
                                       of another rank's, or one that has `max_m` choices in front of it already)
    row_choices   int32 [rows], or [experts, max_m]   the choice t * k + j that a row holds, -1 where it holds none

The other functions take the plan as it is. `rows` is the most that any choices can need (the number that they do need is known on the
device only); rows that hold no choice are neither read nor written, except for the zeros that `zero_padding` asks for. The order
inside an expert is that of the choices: nothing depends on timing. All tensors are on one device, whose current stream is used.

Experts are counted from 0: a rank that holds those from `first` on sorts `topk_idx - first`. With `max_m` nothing but the -1 in `token_rows` of a
choice for one of the experts here says that it was dropped; `layout` ends at `max_m`. The plan's tensors may share one allocation (they do in the
compiled host layer), so keeping one may keep all three. Groups start on multiples of 256 rows, which is the default of everything here and of `cast_to_fp4`;
`cast_to_fp8` and `swiglu_apply_weight_to_fp8` have the reference's 128 and want expert_alignment=256 for such a layout (with 128 every row with a choice
is right, but rows of the padding are read and written too).

    plan = moe_sort(topk_idx, experts)
    a = moe_dispatch_to_fp8(x, plan)
    m_grouped_fp8_gemm_nt_contiguous(a, w, y, plan[0], recipe=(1, 1, 32))
    out = moe_combine(y, plan, topk_weights)

Gradients: of `moe_combine` with weights, `moe_combine_grad`; without weights, `moe_dispatch`; of `moe_dispatch`, `moe_combine` without
weights. None of these has a counterpart in the reference, whose fused MoE does both steps inside its kernel.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L
from ._api import MK_ALIGNMENT, _C, _ceil_div, _host_assert, _stream_ptr
from .quant_ops import _empty_scales

_INT_MAX = 2 ** 31 - 1
_OUT_ROWS = "out must hold a row for each of the layout's, at one distance"
_IN_ROWS = "rows must hold a row for each of the layout's, at one distance"


class _Rows:
    """What moe_sort has made, checked against the device of the rows and the number of tokens."""

    def __init__(self, plan, x, num_tokens):
        self.layout, self.token_rows, self.row_choices = plan
        for t in plan:
            _host_assert(t.dtype == torch.int32 and t.is_contiguous() and t.device == x.device,
                         'plan must hold the three contiguous int32 tensors of moe_sort, on the device of the rows')
        masked = self.row_choices.dim() == 2
        _host_assert(self.layout.dim() == 1 and self.token_rows.dim() == 2 and
                     (self.row_choices.dim() == 1 or (masked and self.row_choices.size(0) == self.layout.size(0))),
                     'plan must hold the three tensors of moe_sort: layout, token_rows, row_choices')
        (self.tokens, self.topk), self.experts = self.token_rows.shape, self.layout.size(0)
        self.max_m = self.row_choices.size(1) if masked else 0
        self.rows = self.row_choices.numel()
        self.masked = masked
        _host_assert(max(self.tokens, self.topk, self.token_rows.numel(), self.rows) <= _INT_MAX, 'plan is too large')
        _host_assert(num_tokens is None or self.tokens == num_tokens, 'plan was made for another number of tokens')

    def shape(self, last):
        return (*self.row_choices.shape, last)

    def check_rows(self, t, what):
        _host_assert(t.dim() > 0 and tuple(t.shape) == self.shape(t.size(-1)) and t.stride(-1) == 1, what)
        per_group = self.max_m if self.masked else self.rows
        stride = t.stride(-2) if per_group > 1 else t.stride(0) if self.masked and self.experts > 1 else t.size(-1)
        _host_assert(stride >= t.size(-1) and (t.dim() == 2 or self.experts <= 1 or t.stride(0) == stride * self.max_m), what)
        return stride


def _is_float(t):
    return t.dtype in (torch.bfloat16, torch.float32)


def _row_stride(x):
    return x.stride(0) if x.size(0) > 1 else x.size(1)


def _check_tokens(x, what):
    _host_assert(x.is_cuda and x.dim() == 2 and x.stride(1) == 1 and _is_float(x), what)


def _check_alignment(expert_alignment):
    _host_assert(0 < expert_alignment <= _INT_MAX, 'expert_alignment must be positive')


def _check_weights(w, plan):
    _host_assert(w.dtype == torch.float32 and w.is_contiguous() and w.device == plan.token_rows.device and w.shape == plan.token_rows.shape,
                 'topk_weights must be a contiguous float32 tensor with one weight per choice, on the device of the rows')


def moe_sort(topk_idx: torch.Tensor, num_experts: int, expert_alignment: int = MK_ALIGNMENT, max_m: Optional[int] = None):
    """topk_idx int32 or int64 [tokens, k] -> (layout, token_rows, row_choices): the psum layout whose groups start on multiples of
    `expert_alignment` rows, or with `max_m` the masked layout of that many rows for each expert (choices behind those are
    dropped). At most 1024 experts."""
    _host_assert(topk_idx.is_cuda and topk_idx.dim() == 2 and topk_idx.is_contiguous() and topk_idx.dtype in (torch.int64, torch.int32),
                 'topk_idx must be a contiguous 2-D int32 or int64 tensor on a CUDA device')
    _host_assert(0 < num_experts <= 1024, 'num_experts must be between 1 and 1024')
    _host_assert(max_m is None or 0 < max_m <= _INT_MAX, 'max_m must be positive')
    _check_alignment(expert_alignment)
    _host_assert(topk_idx.numel() <= _INT_MAX, 'topk_idx is too large')
    rows = num_experts * max_m if max_m else L.lib().dg_moe_num_rows(topk_idx.numel(), num_experts, expert_alignment)
    _host_assert(rows <= _INT_MAX, 'the layout has too many rows')
    with torch.cuda.device(topk_idx.device):
        empty = lambda *shape: torch.empty(shape, dtype=torch.int32, device=topk_idx.device)  # noqa: E731
        layout, token_rows, row_choices = empty(num_experts), empty(*topk_idx.shape), empty(num_experts, max_m) if max_m else empty(rows)
        L.check(L.lib().dg_moe_sort_launch(
            topk_idx.data_ptr(), int(topk_idx.dtype == torch.int64), topk_idx.size(0), topk_idx.size(1), num_experts, expert_alignment, max_m or 0,
            layout.data_ptr(), token_rows.data_ptr(), row_choices.data_ptr(), rows, _stream_ptr(topk_idx.device)))
    return layout, token_rows, row_choices


def moe_dispatch(x: torch.Tensor, plan, out: Optional[torch.Tensor] = None, zero_padding: bool = False, expert_alignment: int = MK_ALIGNMENT):
    """x [tokens, hidden] BF16 or FP32 -> the rows of the layout, [rows, hidden] or [experts, max_m, hidden]: every token's row copied to
    those of its choices. `zero_padding` writes zeros to the rows without a choice between each group's end and the next multiple of
    `expert_alignment` (the k-grouped GEMM of a weight gradient reads them), or to the rest of an expert's `max_m`. `out` must not
    overlap x. Rows of x and out start on 16-byte boundaries."""
    _check_tokens(x, 'x must be a row-major 2-D BF16 or FP32 tensor on a CUDA device')
    p = _Rows(plan, x, x.size(0))
    _check_alignment(expert_alignment)
    with torch.cuda.device(x.device):
        if out is not None:
            _host_assert(out.dtype == x.dtype and out.device == x.device and out.size(-1) == x.size(1),
                         'out must have the type, the device and the row length of x')
        else:
            out = torch.empty(p.shape(x.size(1)), dtype=x.dtype, device=x.device)
        stride, es = p.check_rows(out, _OUT_ROWS), x.element_size()
        L.check(L.lib().dg_moe_dispatch_launch(
            x.data_ptr(), _row_stride(x) * es, p.tokens, p.topk, x.size(1) * es, p.token_rows.data_ptr(), p.row_choices.data_ptr(), p.rows, out.data_ptr(), stride * es,
            p.layout.data_ptr(), p.experts, expert_alignment, p.max_m, int(zero_padding), _stream_ptr(x.device)))
    return out


def moe_dispatch_to_fp8(x: torch.Tensor, plan, out=None):
    """x [tokens, hidden] BF16 -> (E4M3 rows of the layout, packed UE8M0 scales): what `cast_to_fp8` makes of the rows of
    `moe_dispatch`, each token quantised once. The scales, int16 [rows, hidden / 64] or [experts, max_m, hidden / 64] with consecutive
    rows contiguous, are in the layout that the GEMMs read. `out`: such a pair to write to."""
    _host_assert(x.is_cuda and x.dim() == 2 and x.stride(1) == 1 and x.dtype == torch.bfloat16, 'x must be a row-major 2-D BF16 tensor on a CUDA device')
    _host_assert(x.size(1) % 32 == 0, 'the row length of x must be a multiple of 32')
    _host_assert(x.size(1) <= _INT_MAX, 'x is too large')
    p = _Rows(plan, x, x.size(0))
    hidden = x.size(1)
    cols, per_group = _ceil_div(hidden, 64), p.max_m if p.max_m else p.rows
    with torch.cuda.device(x.device):
        if out is not None:
            out, sf = out
            _host_assert(out.dtype == torch.float8_e4m3fn and out.device == x.device and out.size(-1) == hidden,
                         'out must be an E4M3 tensor of the row length and the device of x, with its scales')
            _host_assert(sf.dtype == torch.int16 and sf.device == x.device and tuple(sf.shape) == p.shape(cols) and
                         (sf.stride(-2) == 1 or per_group <= 1) and (cols <= 1 or sf.stride(-1) >= per_group) and
                         (sf.dim() == 2 or p.experts <= 1 or sf.stride(0) >= ((cols - 1) * sf.stride(-1) if cols > 1 else 0) + per_group),
                         'the scales of out must be int16, one element for 64 channels of each row, contiguous along the rows')
        else:
            out = torch.empty(p.shape(hidden), dtype=torch.float8_e4m3fn, device=x.device)
            sf = _empty_scales(p.shape(cols), x.device)
        stride = p.check_rows(out, _OUT_ROWS)
        nbytes = L.lib().dg_moe_dispatch_fp8_scratch_bytes(p.tokens, hidden)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
        L.check(L.lib().dg_moe_dispatch_fp8_launch(
            x.data_ptr(), _row_stride(x), p.tokens, p.topk, hidden, p.token_rows.data_ptr(), p.row_choices.data_ptr(), p.rows, out.data_ptr(), stride,
            sf.data_ptr(), sf.stride(-1) if cols > 1 else per_group, sf.stride(0) if sf.dim() == 3 and p.experts > 1 else 0, per_group,
            scratch.data_ptr() if nbytes else None, nbytes, _stream_ptr(x.device)))
    return out, sf


def moe_combine(rows: torch.Tensor, plan, topk_weights: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None):
    """rows [rows, hidden] or [experts, max_m, hidden] BF16 or FP32 -> [tokens, hidden]: the rows of a token's choices times their weights
    (float32 [tokens, k]; 1 without them), summed in FP32 in the order of the choices and rounded once. A choice without a row adds
    nothing, whatever its weight. `out` must not overlap rows."""
    _host_assert(rows.is_cuda and rows.dim() in (2, 3) and _is_float(rows), 'rows must be a 2-D or 3-D BF16 or FP32 tensor on a CUDA device')
    p = _Rows(plan, rows, None)
    stride, hidden = p.check_rows(rows, _IN_ROWS), rows.size(-1)
    _host_assert(hidden <= _INT_MAX, 'rows are too long')
    if topk_weights is not None:
        _check_weights(topk_weights, p)
    with torch.cuda.device(rows.device):
        if out is not None:
            _host_assert(out.dtype == rows.dtype and out.device == rows.device and tuple(out.shape) == (p.tokens, hidden) and
                         out.stride(1) == 1 and _row_stride(out) >= hidden,
                         'out must be a row-major [tokens, hidden] tensor of the type and the device of rows')
        else:
            out = torch.empty((p.tokens, hidden), dtype=rows.dtype, device=rows.device)
        L.check(L.lib().dg_moe_combine_launch(
            rows.data_ptr(), int(rows.dtype == torch.float32), stride, p.rows, hidden, p.token_rows.data_ptr(), p.tokens, p.topk,
            topk_weights.data_ptr() if topk_weights is not None else None, out.data_ptr(), _row_stride(out), _stream_ptr(rows.device)))
    return out


def moe_combine_grad(grad_out: torch.Tensor, rows: torch.Tensor, plan, topk_weights: torch.Tensor, out: Optional[torch.Tensor] = None,
                     zero_padding: bool = False, expert_alignment: int = MK_ALIGNMENT):
    """Gradients of `moe_combine(rows, plan, topk_weights)` for grad_out [tokens, hidden]: (grad_rows like rows, grad_weights float32
    [tokens, k]). A choice without a row has the gradient 0. `zero_padding` as in `moe_dispatch`. `out`: where grad_rows goes; it may be
    `rows` itself and must not overlap it otherwise, nor grad_out."""
    _check_tokens(grad_out, 'grad_out must be a row-major 2-D BF16 or FP32 tensor on a CUDA device')
    p = _Rows(plan, grad_out, grad_out.size(0))
    hidden = grad_out.size(1)
    _host_assert(rows.dtype == grad_out.dtype and rows.device == grad_out.device and rows.size(-1) == hidden,
                 'rows must have the type, the device and the row length of grad_out')
    stride = p.check_rows(rows, _IN_ROWS)
    _host_assert(hidden <= _INT_MAX, 'rows are too long')
    _check_weights(topk_weights, p)
    _check_alignment(expert_alignment)
    with torch.cuda.device(grad_out.device):
        if out is not None:
            _host_assert(out.dtype == rows.dtype and out.device == rows.device and out.size(-1) == hidden,
                         'out must have the type, the device and the row length of rows')
        else:
            out = torch.empty(p.shape(hidden), dtype=rows.dtype, device=rows.device)
        out_stride = p.check_rows(out, _OUT_ROWS)
        grad_weights = torch.empty_like(topk_weights)
        L.check(L.lib().dg_moe_combine_grad_launch(
            grad_out.data_ptr(), int(rows.dtype == torch.float32), _row_stride(grad_out), rows.data_ptr(), stride, p.rows, hidden,
            p.token_rows.data_ptr(), p.row_choices.data_ptr(), p.tokens, p.topk, topk_weights.data_ptr(), out.data_ptr(), out_stride, grad_weights.data_ptr(),
            p.layout.data_ptr(), p.experts, expert_alignment, p.max_m, int(zero_padding), _stream_ptr(grad_out.device)))
    return out, grad_weights


# The compiled host layer has the same functions (csrc/apis/moe.hpp).
if _C is not None:
    moe_sort, moe_dispatch, moe_dispatch_to_fp8 = _C.moe_sort, _C.moe_dispatch, _C.moe_dispatch_to_fp8
    moe_combine, moe_combine_grad = _C.moe_combine, _C.moe_combine_grad
