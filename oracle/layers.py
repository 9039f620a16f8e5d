"""The router's choice, the norm, the gradient of SwiGLU and 8-bit operands along the rows, restated in loops and 64 bits (test infrastructure, never
shipped). Written from the definitions: the reference has no counterpart to pin them to."""

from __future__ import annotations

import math

import torch


def moe_route_ref(logits, topk, scoring='softmax', bias=None, num_groups=1, topk_groups=1, group_best=2, renormalize=False, scale=1.0):
    """(topk_idx int32, topk_weights float64) on the CPU."""
    l = logits.double()
    tokens, experts = l.shape
    b = torch.zeros(experts, dtype=torch.float64) if bias is None else bias.double()
    if scoring == 'sigmoid':
        s = torch.sigmoid(l)
    else:
        s = torch.softmax(torch.where((l == -math.inf).all(1, keepdim=True), 0.0, l), dim=1)
    idx = torch.full((tokens, topk), -1, dtype=torch.int32)
    weights = torch.zeros(tokens, topk, dtype=torch.float64)
    size = experts // num_groups
    rank = lambda v: math.inf if v != v else v                         # NaN is the largest  # noqa: E731
    for t in range(tokens):
        can = [e for e in range(experts) if l[t, e] != -math.inf and b[e] != -math.inf]
        c = {e: float(s[t, e] + b[e]) for e in can}
        # (without a bias the order is that of the logits)
        order = {e: rank(float(l[t, e]) if bias is None else c[e]) for e in can}
        if num_groups > 1:
            def score(g):
                of = [c[e] if bias is not None or group_best == 2 else float(l[t, e]) for e in can if e // size == g]
                if any(v != v for v in of):
                    return math.inf
                best = sorted(of, reverse=True)[:group_best]
                return sum(best) if best else -math.inf
            scores = [score(g) for g in range(num_groups)]
            taken = sorted(range(num_groups), key=lambda g: (-scores[g], g))[:topk_groups]
            can = [e for e in can if e // size in taken]
        chosen = sorted(can, key=lambda e: (-order[e], e))[:topk]
        w = [float(s[t, e]) for e in chosen]
        if renormalize:
            total = sum(w)
            w = [v / (total if total != total else max(total, 1e-20)) for v in w]
        idx[t, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
        weights[t, :len(chosen)] = scale * torch.tensor(w, dtype=torch.float64)
    return idx, weights


def moe_route_grad_ref(grad_weights, logits, topk_idx, scoring='softmax', renormalize=False, scale=1.0):
    """float64 (grad_logits, sum of its terms' magnitudes)."""
    l, idx = logits.double(), topk_idx.long()
    tokens, experts = l.shape
    out, size = torch.zeros_like(l), torch.zeros_like(l)
    for t in range(tokens):
        js = [j for j in range(idx.size(1)) if 0 <= int(idx[t, j]) < experts]
        masked = bool((l[t] == -math.inf).all())
        p = torch.sigmoid(l[t]) if scoring == 'sigmoid' else torch.zeros(experts, dtype=torch.float64) if masked else torch.softmax(l[t], 0)
        slope = torch.sigmoid(-l[t]) if scoring == 'sigmoid' else torch.ones(experts, dtype=torch.float64)
        total = sum(p[int(idx[t, j])] for j in js)
        for j in js:
            g, e = scale * grad_weights[t, j].double(), int(idx[t, j])
            if renormalize:
                # q_j = s_j / total: d q_j / d log s_i = q_j ([i = j] - q_i); what a softmax's sum adds to log s is the same for all i and cancels
                for i in js:
                    other, q, same = int(idx[t, i]), p[int(idx[t, i])] / total, float(i == j)
                    out[t, other] += g * p[e] / total * (same - q) * slope[other]
                    size[t, other] += g.abs() * p[e] / total * (same + q) * slope[other]
            else:
                out[t, e] += g * p[e] * slope[e]
                size[t, e] += g.abs() * p[e] * slope[e]
                if scoring == 'softmax':
                    out[t] -= g * p[e] * p
                    size[t] += g.abs() * p[e] * p
    return out, size


def rms_norm_ref(h, weight, eps):
    """float64 (rstd, y) of the h that the residual stream holds."""
    h = h.double()
    rstd = 1 / torch.sqrt((h * h).mean(1) + eps)
    return rstd, h * rstd[:, None] * weight.double()


def rms_norm_grad_ref(grad_out, h, weight, rstd, grad_h=None):
    """float64 {'dx', 'dw', and the magnitudes that bound their errors: 'u', 'n', 'mean', 'mean_size', 'dw_size'}."""
    g, n, w = grad_out.double(), h.double() * rstd.double()[:, None], weight.double()
    u = g * w
    mean = (u * n).mean(1, keepdim=True)
    dx = rstd.double()[:, None] * (u - n * mean)
    if grad_h is not None:
        dx = dx + grad_h.double()
    return {'dx': dx, 'dw': (g * n).sum(0), 'u': u.abs(), 'n': n.abs(), 'mean': mean.abs(), 'mean_size': (u * n).abs().mean(1, keepdim=True),
            'dw_size': (g * n).abs().sum(0)}


def swiglu_grad_ref(grad_out, x, topk_weights=None, clamp_value=None):
    """float64 (dx_l, dx_r, dw, and l, r, p with g: what bounds their errors) of all rows."""
    g, x = grad_out.double(), x.double()
    h = x.size(1) // 2
    xl, xr = x[:, :h], x[:, h:]
    l = xl if clamp_value is None else torch.clamp(xl, max=clamp_value)
    r = xr if clamp_value is None else torch.clamp(xr, -clamp_value, clamp_value)
    w = torch.ones(x.size(0), 1, dtype=torch.float64) if topk_weights is None else topk_weights.double().reshape(-1, 1)
    p = torch.sigmoid(l)
    dl, dr = g * w * r * (p + l * p * (1 - p)), g * w * l * p
    if clamp_value is not None:
        dl, dr = torch.where(xl > clamp_value, 0.0, dl), torch.where(xr.abs() > clamp_value, 0.0, dr)
    return dl, dr, (g * l * p * r).sum(1), (g, l, r, p, w)


def cast_fp8_ref(x, axis, min_amax=1e-4, valid=None):
    """E4M3 of x (exact in FP32) with blocks of 32 along `axis` (0 or 1), the last one perhaps short: (codes uint8 like x, scale bytes with `axis`
    divided by 32, values float32). The scale's rule is in FP32: max(amax, min_amax) times 1 / 448 rounded up to a power of two, 2^-126 or more.
    Blocks with an infinity or a NaN have the byte 255. `valid` (bool along axis 0): rows that do not count and are zero."""
    x = x.float()
    if valid is not None:
        x = torch.where(valid[:, None], x, 0.0)
    x = x.movedim(axis, -1)
    n = x.size(-1)
    blocks = torch.nn.functional.pad(x, (0, -n % 32)).unflatten(-1, (-1, 32))
    finite = torch.isfinite(blocks).all(-1)
    amax = torch.where(finite, blocks.abs().amax(-1), 0.0).clamp(min=min_amax) * torch.tensor(1 / 448, dtype=torch.float32)
    byte = ((amax.contiguous().view(torch.int32) + 0x7FFFFF) >> 23).clamp(min=1)
    scaled = blocks.double() * torch.ldexp(torch.ones_like(byte, dtype=torch.float64), 127 - byte)[..., None]
    codes = torch.where(finite[..., None], scaled, 0.0).float().to(torch.float8_e4m3fn)
    values = torch.where(finite[..., None], codes.float() * torch.ldexp(torch.ones_like(byte, dtype=torch.float32), byte - 127)[..., None], float('nan'))
    byte = torch.where(finite, byte, 255).to(torch.uint8)
    back = lambda t: t.flatten(-2)[..., :n].movedim(-1, axis)            # noqa: E731
    return back(codes.view(torch.uint8)), byte.movedim(-1, axis), back(values)


def pack_scales(byte, axis):
    """Scale bytes -> int16 pairs along `axis`, zero where the last pair has no second byte."""
    byte = byte.movedim(axis, -1).int()
    byte = torch.nn.functional.pad(byte, (0, byte.size(-1) % 2))
    pairs = byte[..., 0::2] | (byte[..., 1::2] << 8)
    return torch.where(pairs >= 32768, pairs - 65536, pairs).to(torch.int16).movedim(-1, axis)
