"""CPU restatement of the SwiGLU / cast -> FP8 producer (test infrastructure, never shipped).

Follows third-party/tilelang_ops/swiglu_apply_weight_to_fp8.py of the reference: clamp (:156-161), SiLU by division
(:162-165), weight (:166), per-32-channel scale from the bit pattern of max(amax, 1e-4) * (1 / 448) rounded up to a
power of two (:80-90), value times the inverse scale rounded to E4M3 (:250-252), scale bytes packed two per int16
with consecutive tokens contiguous (:104-125, 446-449), tokens in psum padding skipped (:263-268).

Parity unpinned by the reference for this function: the reference's own test of the operator (tests/test_mega_moe.py)
needs the NPU kernel itself as ground truth and holds no fixture, so this restatement is checked against the formulas
above only. The GPU test compares with a tolerance because exp() differs in the last bit between implementations.
"""

from __future__ import annotations

import torch


def swiglu_quant_ref(x: torch.Tensor, topk_weights=None, psum=None, clamp_value=None, alignment: int = 128,
                     swiglu: bool = True):
    """Returns (codes uint8 [T, H], sf int16 [T, ceil(H/64)], valid bool [T], dequantised fp32 [T, H])."""
    t = x.size(0)
    xf = x.float()
    if swiglu:
        h = x.size(1) // 2
        xl, xr = xf[:, :h], xf[:, h:]
        if clamp_value is not None:
            xl = torch.clamp(xl, max=clamp_value)
            xr = torch.clamp(xr, min=-clamp_value, max=clamp_value)
        y = xl / (1.0 + torch.exp(-xl)) * xr
        if topk_weights is not None:
            y = y * topk_weights.float().reshape(-1, 1)
    else:
        h = x.size(1)
        y = xf
    groups = h // 32
    amax = y.reshape(t, groups, 32).abs().amax(dim=-1)
    scaled = (torch.clamp(amax, min=1e-4) * torch.tensor(1.0 / 448.0, dtype=torch.float32)).contiguous()
    bits = scaled.view(torch.int32)
    exponent = ((bits - 1) >> 23) + 1                                   # UE8M0 byte
    inverse = ((254 - exponent) << 23).view(torch.float32)
    q = (y.reshape(t, groups, 32) * inverse.unsqueeze(-1)).reshape(t, h).to(torch.float8_e4m3fn)
    scale = (exponent << 23).view(torch.float32)
    deq = (q.float().reshape(t, groups, 32) * scale.unsqueeze(-1)).reshape(t, h)
    e8 = exponent.to(torch.uint8)
    if groups % 2:
        e8 = torch.nn.functional.pad(e8, (0, 1))
    sf = e8.contiguous().view(torch.int16)                                # low byte = even 32-block
    valid = torch.ones(t, dtype=torch.bool)
    if psum is not None:
        valid[:] = False
        start = 0
        for p in psum:
            valid[start:min(int(p), t)] = True
            start = (int(p) + alignment - 1) // alignment * alignment
    return q.view(torch.uint8), sf, valid, deq


def cast_fp4_ref(x: torch.Tensor, axis: int, valid=None):
    """Microscaled E2M1 of x (any float type) in 64 bits, blocks of 32 along `axis` (-1 or -2), the last one perhaps short: (codes uint8 like
    x, scale bytes uint8 with `axis` divided by 32, values float64). The scale is the smallest power of two (2^-126 or more) with which the
    largest magnitude is at most 6; the nearest code, halves to the even one; scale byte 255 where a block holds an infinity or a
    NaN. `valid` (bool along axis -2): rows that do not count and are zero."""
    x = x.double()
    if valid is not None:
        x = torch.where(valid[:, None], x, 0.0)
    x = x.movedim(axis, -1)
    n = x.size(-1)
    blocks = torch.nn.functional.pad(x, (0, -n % 32)).unflatten(-1, (-1, 32))
    finite = torch.isfinite(blocks).all(-1)
    blocks = torch.where(finite[..., None], blocks, 0.0)
    mantissa, exponent = torch.frexp(blocks.abs().amax(-1) / 6)
    exponent = (exponent - (mantissa == 0.5).int()).clamp(min=-126)
    exponent = torch.where(blocks.abs().amax(-1) == 0, torch.full_like(exponent, -126), exponent)
    scaled = torch.ldexp(blocks, -exponent[..., None])
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    distance = (scaled.abs()[..., None] - grid).abs()
    best = distance.amin(-1, keepdim=True)
    tied = distance == best                                              # one code, or two neighbours: the even one of them
    code = torch.where(tied & (torch.arange(8) % 2 == 0), 2, torch.where(tied, 1, 0)).argmax(-1)
    values = torch.ldexp(grid[code], exponent[..., None]) * torch.where(torch.signbit(blocks), -1.0, 1.0)
    values = torch.where(finite[..., None], values, float('nan'))
    code = (code + 8 * torch.signbit(blocks)).to(torch.uint8)
    byte = torch.where(finite, exponent + 127, 255).to(torch.uint8)
    back = lambda t: t.flatten(-2)[..., :n].movedim(-1, axis)            # noqa: E731
    return back(code), byte.movedim(-1, axis), back(values)
