"""Timed cases of the operators around the expert GEMMs and of the 4-bit quantiser.

A case is a dict of plain values. Its `kind` names the operator:

  sort        moe_sort: the router's choices -> the rows of the grouped layout (psum, or a fixed number of slots per expert)
  dispatch    moe_dispatch / moe_dispatch_to_fp8: every token's row copied (or quantised) to the rows of its choices
  combine     moe_combine: the rows of a token's choices, weighted and summed; without weights the gradient of a dispatch
  grad        moe_combine_grad: gradients of a combine with respect to its rows and to its weights
  fp4_linear  cast_to_fp4 on the activations and the FP4 x FP4 product with weights that are quantised already
  fp4_weights cast_to_fp4 on weights and cast_from_fp4 back: the values that a product with them sees. `mn_major`: blocks of
              32 run down the rows, as the gradient of the activations needs the weights

A layout is described by `tokens`, `topk`, `total` (the router's experts) and `experts` (those of this rank: choices of others are
-1), and `max_m` (0: psum layout; else the row slots of an expert). Everything comes from the seed.

Where a result is held in 8 bits, the E4M3 tensor is returned as it is (torch reads its values) beside the scale bytes, which
are whole numbers; what is held in 4 bits is returned as values.
"""

import math
import os
import sys

import torch

own = False

sys.path.insert(0, os.path.join(os.getcwd(), 'deepgemm-ascend_b200'))

ALIGN = 256         # rows on which a group of the psum layout starts


def listed():
    return [
        # The choices of a decoding step that reach one of eight ranks: 128 tokens, 32 of 256 experts, slots of the masked layout.
        {'name': 'sort_decode', 'kind': 'sort', 'tokens': 128, 'topk': 8, 'total': 256, 'experts': 32, 'max_m': 256},
        # A long prefill chunk with all experts on one GPU.
        {'name': 'sort_prefill', 'kind': 'sort', 'tokens': 16384, 'topk': 8, 'total': 256, 'experts': 256, 'max_m': 0},
        # The same decoding step's rows, quantised for the masked FP8 GEMM.
        {'name': 'dispatch_decode', 'kind': 'dispatch', 'tokens': 128, 'topk': 8, 'total': 256, 'experts': 32, 'max_m': 256,
         'hidden': 7168, 'to': 'fp8', 'zero_padding': False},
        # Prefill of 8192 tokens over 32 experts, quantised for the contiguous FP8 GEMM.
        {'name': 'dispatch_prefill', 'kind': 'dispatch', 'tokens': 8192, 'topk': 8, 'total': 32, 'experts': 32, 'max_m': 0,
         'hidden': 7168, 'to': 'fp8', 'zero_padding': False},
        # A training step of an odd number of tokens in BF16, with the zero rows between the groups that the weight gradient needs.
        {'name': 'dispatch_train', 'kind': 'dispatch', 'tokens': 4095, 'topk': 6, 'total': 64, 'experts': 64, 'max_m': 0,
         'hidden': 2048, 'to': 'bf16', 'zero_padding': True},
        # One token's eight rows: the smallest call. Latency.
        {'name': 'combine_token', 'kind': 'combine', 'tokens': 1, 'topk': 8, 'total': 256, 'experts': 256, 'max_m': 0,
         'hidden': 7168, 'dtype': 'bf16', 'weights': True},
        # The way back of the prefill above.
        {'name': 'combine_prefill', 'kind': 'combine', 'tokens': 8192, 'topk': 8, 'total': 32, 'experts': 32, 'max_m': 0,
         'hidden': 7168, 'dtype': 'bf16', 'weights': True},
        # Backward pass of the weighted sum, 4096 tokens.
        {'name': 'grad_step', 'kind': 'grad', 'tokens': 4096, 'topk': 8, 'total': 32, 'experts': 32, 'max_m': 0,
         'hidden': 7168, 'dtype': 'bf16'},
        # The same of a short odd chunk with FP32 rows (the grouped GEMM can write them).
        {'name': 'grad_ragged', 'kind': 'grad', 'tokens': 1531, 'topk': 6, 'total': 64, 'experts': 64, 'max_m': 0,
         'hidden': 2048, 'dtype': 'fp32'},
        # A projection of 64 tokens with FP4 activations and weights.
        {'name': 'fp4_linear_decode', 'kind': 'fp4_linear', 'm': 64, 'n': 4096, 'k': 7168, 'dtype': 'bf16'},
        # FP32 master weights of one projection.
        {'name': 'fp4_weights', 'kind': 'fp4_weights', 'groups': 1, 'rows': 2112, 'cols': 7168, 'dtype': 'fp32', 'mn_major': False},
        # BF16 weights of eight experts, quantised along the other axis for the gradient of the activations. The largest of these.
        {'name': 'fp4_experts_mn', 'kind': 'fp4_weights', 'groups': 8, 'rows': 4096, 'cols': 7168, 'dtype': 'bf16', 'mn_major': True},
    ]


def _log(rng, lo, hi, multiple=1):
    """A whole number in [lo, hi], spread over its logarithm, a multiple of `multiple`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(multiple, min(hi // multiple * multiple, int(round(v / multiple)) * multiple))


def draw(rng):
    most = work(next(c for c in listed() if c['name'] == 'combine_prefill'))['bytes']
    while True:
        case = _draw(rng)
        if work(case)['bytes'] <= most and work(case)['flops'] <= 4e11:
            return case


def _draw(rng):
    kind = rng.choice(['sort', 'dispatch', 'dispatch', 'combine', 'combine', 'grad', 'grad', 'fp4_linear', 'fp4_weights', 'fp4_weights'])
    if kind == 'fp4_linear':
        return {'kind': kind, 'm': _log(rng, 1, 4096), 'n': _log(rng, 512, 16384, 64), 'k': _log(rng, 512, 16384, 128),
                'dtype': rng.choice(['bf16', 'fp32'])}
    if kind == 'fp4_weights':
        return {'kind': kind, 'groups': rng.choice([1, 1, 4, 8]), 'rows': _log(rng, 1, 8192), 'cols': _log(rng, 256, 8192, 32),
                'dtype': rng.choice(['bf16', 'fp32']), 'mn_major': rng.random() < 0.5}
    total = rng.choice([8, 16, 32, 64, 128, 160, 256])
    experts = total if rng.random() < 0.5 else max(1, total // 8)
    masked = rng.random() < 0.25
    case = {'kind': kind, 'tokens': _log(rng, 1, 512 if masked else 16384), 'topk': rng.choice([1, 2, 4, 6, 8]), 'total': total,
            'experts': experts, 'max_m': rng.choice([64, 128, 256]) if masked else 0}
    if kind == 'sort':
        return case
    case['hidden'] = _log(rng, 512, 8192, 32)
    if kind == 'dispatch':
        case['to'] = rng.choice(['fp8', 'fp8', 'bf16', 'fp32'])
        case['zero_padding'] = not masked and case['to'] != 'fp8' and rng.random() < 0.5
        return case
    case['dtype'] = rng.choice(['bf16', 'bf16', 'fp32'])
    if kind == 'combine':
        case['weights'] = rng.random() < 0.7
    return case


# ------------------------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------------------------
_TYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}


def _rows_of(case):
    """Rows of the grouped layout: the most that any choice of experts can need, in whole alignments; or all slots."""
    if case['max_m']:
        return case['experts'] * case['max_m']
    n = case['tokens'] * case['topk']
    used = min(case['experts'], n)
    return ALIGN * (used + (n - used) // ALIGN)


def _choices(case, gen):
    """int64 [tokens, topk]: distinct experts of a router whose experts are not equally liked; -1 for those of other ranks."""
    liked = torch.randn(case['total'], device='cuda', generator=gen) * 0.5
    idx = (torch.randn(case['tokens'], case['total'], device='cuda', generator=gen) + liked).topk(case['topk'], dim=1).indices
    return torch.where(idx < case['experts'], idx, -1)


def _sorted(idx, experts, max_m):
    """(layout, token_rows, row_choices) of the choices `idx`, with elementary operations."""
    tokens, topk = idx.shape
    flat = idx.reshape(-1)
    n = flat.numel()
    valid = (flat >= 0) & (flat < experts)
    key = torch.where(valid, flat, experts)
    order = torch.argsort(key, stable=True)
    counts = (key[:, None] == torch.arange(experts + 1, device=idx.device)).sum(0)
    rank = torch.empty(n, dtype=torch.int64, device=idx.device)
    rank[order] = torch.arange(n, device=idx.device) - (counts.cumsum(0) - counts)[key[order]]
    counts = counts[:experts]
    if max_m:
        starts, layout = torch.arange(experts, device=idx.device) * max_m, counts.clamp(max=max_m)
        valid = valid & (rank < max_m)
        rows = experts * max_m
    else:
        whole = (counts + ALIGN - 1) // ALIGN * ALIGN
        starts = whole.cumsum(0) - whole
        layout = starts + counts
        used = min(experts, n)
        rows = ALIGN * (used + (n - used) // ALIGN)
    row = torch.where(valid, starts[key.clamp(max=experts - 1)] + rank, -1)
    # (one place more, which takes what has no row)
    choices = torch.full((rows + 1,), -1, dtype=torch.int32, device=idx.device)
    choices[torch.where(valid, row, rows)] = torch.arange(n, device=idx.device, dtype=torch.int32)
    choices = choices[:rows].clone()
    return layout.int(), row.int().view(tokens, topk), choices.view(experts, max_m) if max_m else choices


def _shape(case, last):
    return (case['experts'], case['max_m'], last) if case['max_m'] else (_rows_of(case), last)


def _scale_storage(case):
    """int16 scales of the dispatched rows, consecutive rows contiguous."""
    cols = (case['hidden'] // 32 + 1) // 2
    if case['max_m']:
        return torch.zeros((case['experts'], cols, case['max_m']), dtype=torch.int16, device='cuda').transpose(1, 2)
    return torch.zeros((cols, _rows_of(case)), dtype=torch.int16, device='cuda').t()


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    kind = case['kind']
    s = {'case': case}
    randn = lambda *shape, dt=torch.float32: torch.randn(shape, dtype=dt, device='cuda', generator=gen)  # noqa: E731
    if kind == 'fp4_linear':
        m, n, k = case['m'], case['n'], case['k']
        s['x'] = randn(m, k, dt=_TYPES[case['dtype']])
        s['w'] = _pack(*_quantised(randn(n, k) * k ** -0.5, 1))
        s['d'] = torch.zeros((m, n), dtype=torch.bfloat16, device='cuda')
        return s
    if kind == 'fp4_weights':
        shape = (case['groups'], case['rows'], case['cols']) if case['groups'] > 1 else (case['rows'], case['cols'])
        s['x'] = randn(*shape, dt=_TYPES[case['dtype']]) * case['cols'] ** -0.5
        return s
    s['idx'] = _choices(case, gen)
    if kind == 'sort':
        return s
    s['plan'] = _sorted(s['idx'], case['experts'], case['max_m'])
    t, h = case['tokens'], case['hidden']
    if kind == 'dispatch':
        s['x'] = randn(t, h, dt=_TYPES[case['to']] if case['to'] != 'fp8' else torch.bfloat16)
        if case['to'] == 'fp8':
            s['out'] = (torch.zeros(_shape(case, h), dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn), _scale_storage(case))
        else:
            s['out'] = torch.zeros(_shape(case, h), dtype=s['x'].dtype, device='cuda')
        return s
    dtype = _TYPES[case['dtype']]
    s['rows'] = randn(*_shape(case, h), dt=dtype)
    s['w'] = None
    if kind == 'grad' or case['weights']:
        w = torch.rand((t, case['topk']), device='cuda', generator=gen) + 0.05
        s['w'] = w / w.sum(1, keepdim=True)
    if kind == 'grad':
        s['g'] = randn(t, h, dt=dtype)
        s['out'] = torch.zeros(_shape(case, h), dtype=dtype, device='cuda')
    return s


# ------------------------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------------------------
def run(s):
    case = s['case']
    kind = case['kind']
    if own:
        import deep_gemm
        if kind == 'sort':
            return deep_gemm.moe_sort(s['idx'], case['experts'], max_m=case['max_m'] or None)
        if kind == 'dispatch':
            if case['to'] == 'fp8':
                return deep_gemm.moe_dispatch_to_fp8(s['x'], s['plan'], out=s['out'])
            return deep_gemm.moe_dispatch(s['x'], s['plan'], out=s['out'], zero_padding=case['zero_padding'])
        if kind == 'combine':
            return deep_gemm.moe_combine(s['rows'], s['plan'], s['w'])
        if kind == 'grad':
            return deep_gemm.moe_combine_grad(s['g'], s['rows'], s['plan'], s['w'], out=s['out'])
        if kind == 'fp4_linear':
            deep_gemm.fp8_fp4_gemm_nt(deep_gemm.cast_to_fp4(s['x']), s['w'], s['d'])
            return s['d']
        q = deep_gemm.cast_to_fp4(s['x'], mn_major=case['mn_major'])
        return deep_gemm.cast_from_fp4(q, out_dtype=s['x'].dtype, mn_major=case['mn_major'])
    if kind == 'sort':
        return _sorted(s['idx'], case['experts'], case['max_m'])
    if kind == 'dispatch':
        return _dispatch(s, case)
    if kind == 'combine':
        return _combine(s, case)
    if kind == 'grad':
        return _grad(s, case)
    if kind == 'fp4_linear':
        a = _values(*_quantised(s['x'].float(), 1), 1)
        w = _values(*_unpack(s['w']), 1)
        s['d'].copy_(a @ w.t())
        return s['d']
    axis = -2 if case['mn_major'] else -1
    return _values(*_quantised(s['x'].float(), axis), axis).to(s['x'].dtype)


def _live(plan):
    """(indices of the choices that have a row, their rows), flat."""
    rows = plan[1].reshape(-1).long()
    which = (rows >= 0).nonzero().reshape(-1)
    return which, rows[which]


def _zero_padding(out, layout):
    """The rows from each group's end to the next multiple of the alignment become zero."""
    row = torch.arange(out.size(0), device=out.device)
    ends = layout.long()
    whole = (ends + ALIGN - 1) // ALIGN * ALIGN
    out[((row[:, None] >= ends) & (row[:, None] < whole)).any(1)] = 0


def _dispatch(s, case):
    which, rows = _live(s['plan'])
    x = s['x'][which // case['topk']]
    if case['to'] != 'fp8':
        s['out'].view(-1, case['hidden'])[rows] = x
        if case['zero_padding']:
            _zero_padding(s['out'], s['plan'][0])
        return s['out']
    x = x.float().view(x.size(0), -1, 32)
    bits = (x.abs().amax(2).clamp(min=1e-4) * (1.0 / 448.0)).view(torch.int32)
    e = ((bits - 1) >> 23) + 1                                    # the smallest power of two that is not below
    x = x * ((254 - e) << 23).view(torch.float32)[:, :, None]
    out, sf = s['out']
    out.view(torch.uint8).view(-1, case['hidden'])[rows] = x.view(x.size(0), -1).to(torch.float8_e4m3fn).view(torch.uint8)
    e = torch.nn.functional.pad(e, (0, e.size(1) % 2))
    pairs = (e[:, 0::2] | (e[:, 1::2] << 8)).to(torch.int16)
    if case['max_m']:
        sf[rows // case['max_m'], rows % case['max_m']] = pairs
    else:
        sf[rows] = pairs
    return out, sf


def _weighted(s, case, dtype):
    """The rows of all choices [tokens, topk, hidden] (zeros where a choice has none), and its weights."""
    rows = s['plan'][1].long()
    y = s['rows'].view(-1, case['hidden'])[rows.clamp(min=0)].to(dtype)
    return y.masked_fill_((rows < 0)[:, :, None], 0.0), rows


def _combine(s, case):
    y, rows = _weighted(s, case, torch.float32)
    if s['w'] is not None:
        y *= torch.where(rows >= 0, s['w'], 0.0)[:, :, None]
    return y.sum(1).to(s['rows'].dtype)


def _grad(s, case):
    y, rows = _weighted(s, case, torch.float32)
    g = s['g'].float()
    dw = (y * g[:, None]).sum(2)
    which, live = _live(s['plan'])
    s['out'].view(-1, case['hidden'])[live] = (g[which // case['topk']] * s['w'].view(-1)[which][:, None]).to(s['out'].dtype)
    return s['out'], dw


def _quantised(x, axis):
    """FP32 x -> (signed E2M1 values, exponent bytes) with blocks of 32 along `axis`; the last block may be short. The scale is
    the smallest power of two with which the block's largest magnitude is at most 6; halves go to the even code."""
    x = x.movedim(axis, -1)
    n = x.size(-1)
    x = torch.nn.functional.pad(x, (0, -n % 32)).unflatten(-1, (-1, 32))
    e = (((x.abs().amax(-1).view(torch.int32) + 0x3FFFFF) >> 23) - 2).clamp(min=1)
    x = x * ((254 - e) << 23).view(torch.float32)[..., None]
    a = x.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = torch.copysign(torch.round(a / step) * step, x).flatten(-2)[..., :n]
    return q.movedim(-1, axis), e.movedim(-1, axis)


def _values(q, e, axis):
    scale = (e << 23).view(torch.float32).repeat_interleave(32, axis).narrow(axis, 0, q.size(axis))
    return q * scale


def _pack(q, e):
    """Values and exponent bytes of a K-major matrix -> (packed int8 [rows, k / 2], int16 scales, rows contiguous)."""
    a = q.abs()
    code = (torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).int() | (torch.signbit(q).int() << 3)).to(torch.uint8)
    e = torch.nn.functional.pad(e, (0, e.size(1) % 2))
    return ((code[:, 0::2] | (code[:, 1::2] << 4)).view(torch.int8), (e[:, 0::2] | (e[:, 1::2] << 8)).to(torch.int16).t().contiguous().t())


def _unpack(w):
    """The way back of _pack."""
    u, sf = w[0].view(torch.uint8), w[1].int()
    code = torch.stack((u & 15, u >> 4), dim=-1).flatten(1)
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=u.device)
    q = torch.where(code >= 8, -1.0, 1.0) * table[(code & 7).long()]
    e = torch.stack((sf & 255, (sf >> 8) & 255), dim=-1).flatten(1)[:, :q.size(1) // 32]
    return q, e


# ------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    kind = case['kind']
    if kind == 'sort':
        return None                                               # whole numbers only
    s = prepare(case, seed)
    if kind == 'fp4_linear':
        return _micro64(s['x'].double(), 1) @ _decode64(s['w']).t()
    if kind == 'fp4_weights':
        return _micro64(s['x'].double(), s['x'].dim() - (2 if case['mn_major'] else 1))
    h, k = case['hidden'], case['topk']
    choice = s['plan'][2].reshape(-1).long()                      # by rows: the choice that each holds
    live = choice >= 0
    token = choice.clamp(min=0) // k
    if kind == 'dispatch':
        rows = torch.where(live[:, None], s['x'].double()[token], 0.0)
        if case['to'] != 'fp8':
            return rows.view(_shape(case, h))
        blocks = rows.view(rows.size(0), h // 32, 32)
        scale = _power_at_least(blocks.abs().amax(2).clamp(min=1e-4) / 448)
        scaled = blocks / scale[:, :, None]
        grid = torch.exp2(torch.log2(scaled.abs().clamp(min=2.0 ** -6)).floor() - 3)      # three bits behind the leading one
        return ((scaled / grid).round() * grid).view(_shape(case, h)), None
    # by tokens, one choice after the other
    rows = s['rows'].view(-1, h)
    of = s['plan'][1].long()
    if kind == 'combine':
        out = torch.zeros((case['tokens'], h), dtype=torch.float64, device='cuda')
        for j in range(k):
            has = of[:, j] >= 0
            out[has] += rows[of[has, j]].double() * (1.0 if s['w'] is None else s['w'][has, j, None].double())
        return out
    dw = torch.zeros((case['tokens'], k), dtype=torch.float64, device='cuda')
    for j in range(k):
        has = of[:, j] >= 0
        dw[has, j] = torch.einsum('th,th->t', rows[of[has, j]].double(), s['g'][has].double())
    dy = s['g'].double()[token] * s['w'].double().reshape(-1)[choice.clamp(min=0)][:, None]
    return torch.where(live[:, None], dy, 0.0).view(_shape(case, h)), dw


def _power_at_least(v):
    """The smallest power of two that is not below v > 0."""
    mantissa, exponent = torch.frexp(v)
    return torch.ldexp(torch.ones_like(v), exponent - (mantissa == 0.5).int())


def _micro64(x, axis):
    """What a product with the quantised x sees: blocks of 32 along `axis`, the last one perhaps short."""
    parts = []
    for block in x.split(32, dim=axis):
        amax = block.abs().amax(axis, keepdim=True)
        scale = _power_at_least(torch.where(amax == 0, 1.0, amax) / 6).clamp(min=2.0 ** -126)
        y = block / scale
        grid = torch.exp2(torch.log2(y.abs().clamp(min=1.0)).floor() - 1)                 # one bit behind the leading one
        parts.append((y / grid).round() * grid * scale)
    return torch.cat(parts, dim=axis)


def _decode64(w):
    """Packed K-major weights and scales -> float64."""
    byte, sf = w[0].to(torch.int64) & 255, w[1].to(torch.int64) & 0xFFFF
    out = torch.empty((byte.size(0), 2 * byte.size(1)), dtype=torch.float64, device=byte.device)
    for half in (0, 1):
        code = (byte >> (4 * half)) & 15
        exponent, mantissa = (code >> 1) & 3, (code & 1).double()
        magnitude = torch.where(exponent == 0, mantissa / 2, torch.ldexp(1 + mantissa / 2, exponent - 1))
        out[:, half::2] = torch.where(code >= 8, -magnitude, magnitude)
    block = torch.arange(out.size(1), device=byte.device) // 32
    e = (sf[:, block // 2] >> (8 * (block % 2))) & 255
    return torch.ldexp(out, e - 127)


# ------------------------------------------------------------------------------------------------------------------
def work(case):
    """Bytes with each input read once and each output written once; of choices spread over more experts than this rank's, the
    expected share. Padding and rows behind the last group cost nothing, except where zeros are asked for (half an alignment for
    each expert)."""
    kind = case['kind']
    if kind == 'fp4_linear':
        m, n, k = case['m'], case['n'], case['k']
        return {'bytes': m * k * (2 if case['dtype'] == 'bf16' else 4) + n * k // 2 + n * k // 32 + m * n * 2, 'flops': 2 * m * n * k}
    if kind == 'fp4_weights':
        # (to packed codes and scales, and from them back)
        n = case['groups'] * case['rows'] * case['cols']
        return {'bytes': 2 * n * (2 if case['dtype'] == 'bf16' else 4) + 2 * (n // 2 + n // 32), 'flops': 4 * n}
    t, k = case['tokens'], case['topk']
    share = case['experts'] / case['total']
    live = t * k * share
    if case['max_m']:
        live = min(live, case['experts'] * case['max_m'])
    if kind == 'sort':
        return {'bytes': 12 * t * k + 4 * _rows_of(case) + 4 * case['experts'], 'flops': t * k}
    h = case['hidden']
    some = t * (1 - (1 - share) ** k)                             # tokens with a choice here
    if kind == 'dispatch':
        size = 4 if case['to'] == 'fp32' else 2
        out = h + h // 32 if case['to'] == 'fp8' else h * size
        pads = min(case['experts'], t * k) * ALIGN / 2 * out if case['zero_padding'] else 0
        return {'bytes': some * h * size + live * out + pads + 4 * t * k, 'flops': live * h}
    size = 4 if case['dtype'] == 'fp32' else 2
    if kind == 'combine':
        return {'bytes': live * h * size + t * h * size + t * k * (8 if case['weights'] else 4), 'flops': 2 * live * h}
    return {'bytes': some * h * size + 2 * live * h * size + t * k * 12, 'flops': 3 * live * h}
