"""Timed cases of the operators around an expert layer's products in training and serving with 8-bit operands.

A case is a dict of plain values. Its `kind` names the operator:

  route       moe_route: a router's scores -> the chosen experts and their weights (bias for balance, groups, renormalisation)
  route_grad  moe_route_grad: the gradient of the weights with respect to the router's logits
  norm        rms_norm_to_fp8: the residual's addition, the norm, E4M3 with scales; `rows`: the normed rows in BF16 too
  norm_grad   rms_norm_grad: gradients of the norm's input and of its weight, the residual stream's gradient added
  act         swiglu_apply_weight_to_fp8_with_checkpoint: the second product's operand, and the input kept in 8 bits
  act_grad    swiglu_apply_weight_grad: gradients of the input and of the rows' weights, from the BF16 input or from the checkpoint
  operand     cast_to_fp8(mn_major=True): a weight gradient's operand, blocks of 32 down the rows, from BF16 or from a checkpoint
  weights     cast_to_fp8(mn_major=True) and cast_from_fp8: weights for the gradient of the activations, and the values a product sees

`experts` > 0: the rows lie in a psum layout of that many groups, whose starts are multiples of 256. Everything comes from the seed.

What is held in 8 bits is returned as E4M3 values beside the scales, which are powers of two in 8 bits (torch reads the values of both).
"""

import math
import os
import sys

import torch

own = False

sys.path.insert(0, os.path.join(os.getcwd(), 'deepgemm-ascend_b200'))

ALIGN = 256         # rows on which a group of the psum layout starts
EPS = 1e-6


def listed():
    return [
        # A decoding step of 128 tokens: sigmoid scores, the bias for balance, four of eight groups. Latency.
        {'name': 'route_decode', 'kind': 'route', 'tokens': 128, 'experts': 256, 'topk': 8, 'scoring': 'sigmoid', 'bias': True,
         'groups': 8, 'topk_groups': 4, 'renormalize': True, 'dtype': 'fp32'},
        # The same router on a long prefill chunk.
        {'name': 'route_prefill', 'kind': 'route', 'tokens': 16384, 'experts': 256, 'topk': 8, 'scoring': 'sigmoid', 'bias': True,
         'groups': 8, 'topk_groups': 4, 'renormalize': True, 'dtype': 'fp32'},
        # Backward pass of a softmax router, 16384 tokens of a training step.
        {'name': 'route_grad', 'kind': 'route_grad', 'tokens': 16384, 'experts': 256, 'topk': 8, 'scoring': 'softmax',
         'renormalize': False, 'dtype': 'fp32'},
        # One token's norm in front of a projection: the smallest call. Latency.
        {'name': 'norm_token', 'kind': 'norm', 'tokens': 1, 'hidden': 7168, 'dtype': 'bf16', 'weight': 'bf16', 'residual': True, 'rows': False},
        # Prefill of 8192 tokens in front of an expert layer: 8-bit rows for the shared projection, BF16 rows for the router.
        {'name': 'norm_prefill', 'kind': 'norm', 'tokens': 8192, 'hidden': 7168, 'dtype': 'bf16', 'weight': 'bf16', 'residual': True, 'rows': True},
        # Backward pass of that norm.
        {'name': 'norm_grad', 'kind': 'norm_grad', 'tokens': 8192, 'hidden': 7168, 'dtype': 'bf16', 'weight': 'bf16', 'residual': True},
        # The same of a short odd chunk with an FP32 residual stream and FP32 master weights.
        {'name': 'norm_grad_ragged', 'kind': 'norm_grad', 'tokens': 1531, 'hidden': 2048, 'dtype': 'fp32', 'weight': 'fp32', 'residual': True},
        # Between the two expert products of a training step: 65536 rows of 32 experts.
        {'name': 'act_train', 'kind': 'act', 'tokens': 65536, 'hidden': 2048, 'experts': 32, 'weights': True, 'clamp': 0.0},
        # Its backward pass from the input in 8 bits. The largest of these.
        {'name': 'act_grad_train', 'kind': 'act_grad', 'tokens': 65536, 'hidden': 2048, 'experts': 32, 'weights': True, 'clamp': 0.0, 'from': 'fp8'},
        # The same of a shared expert on a few tokens, from the BF16 input, clamped.
        {'name': 'act_grad_few', 'kind': 'act_grad', 'tokens': 77, 'hidden': 2048, 'experts': 0, 'weights': False, 'clamp': 7.0, 'from': 'bf16'},
        # The dispatched rows of 32 experts, held in 8 bits since the forward pass, for the gradient of the experts' weights.
        {'name': 'operand_checkpoint', 'kind': 'operand', 'tokens': 32768, 'hidden': 7168, 'experts': 32, 'from': 'fp8'},
        # BF16 weights of one projection for the gradient of the activations, and the values that the product sees.
        {'name': 'weights_mn', 'kind': 'weights', 'tokens': 2112, 'hidden': 7168, 'out': 'bf16'},
    ]


def _log(rng, lo, hi, multiple=1):
    """A whole number in [lo, hi], spread over its logarithm, a multiple of `multiple`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(multiple, min(hi // multiple * multiple, int(round(v / multiple)) * multiple))


def draw(rng):
    most = work(next(c for c in listed() if c['name'] == 'act_grad_train'))['bytes']
    while True:
        case = _draw(rng)
        if work(case)['bytes'] <= most:
            return case


def _draw(rng):
    kind = rng.choice(['route', 'route', 'route_grad', 'norm', 'norm', 'norm_grad', 'norm_grad', 'act', 'act_grad', 'act_grad', 'operand', 'operand', 'weights'])
    if kind in ('route', 'route_grad'):
        groups = rng.choice([1, 1, 2, 4, 8]) if kind == 'route' else 1
        experts = groups * _log(rng, 8, 1024 // groups)
        case = {'kind': kind, 'tokens': _log(rng, 1, 32768), 'experts': experts, 'topk': rng.choice([1, 2, 4, 6, 8]), 'scoring': rng.choice(['softmax', 'sigmoid']),
                'renormalize': rng.random() < 0.5, 'dtype': rng.choice(['fp32', 'fp32', 'bf16'])}
        if kind == 'route':
            case |= {'bias': rng.random() < 0.5, 'groups': groups, 'topk_groups': rng.randint((groups + 1) // 2, groups)}
        return case
    if kind in ('norm', 'norm_grad'):
        case = {'kind': kind, 'tokens': _log(rng, 1, 16384), 'hidden': _log(rng, 256, 16384, 32), 'dtype': rng.choice(['bf16', 'bf16', 'fp32']),
                'weight': rng.choice(['bf16', 'fp32']), 'residual': rng.random() < 0.7}
        if kind == 'norm':
            case['rows'] = rng.random() < 0.5
        return case
    if kind == 'weights':
        return {'kind': kind, 'tokens': _log(rng, 1, 16384), 'hidden': _log(rng, 256, 8192, 32), 'out': rng.choice(['bf16', 'fp32'])}
    case = {'kind': kind, 'tokens': _log(rng, 1, 65536), 'hidden': _log(rng, 256, 8192, 32 if kind == 'operand' else 128), 'experts': rng.choice([0, 8, 32, 64])}
    if kind != 'operand':
        case |= {'weights': rng.random() < 0.6, 'clamp': rng.choice([0.0, 7.0])}
    if kind != 'act':
        case['from'] = rng.choice(['bf16', 'fp8', 'fp8'])
    return case


# ------------------------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------------------------
_TYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}


def _sizes(case):
    """Rows of each group: groups that are not equally liked, one of them empty."""
    n, g = case['tokens'], case['experts']
    share = [0.4 + (i * 7919 % 97) / 97.0 for i in range(g)]
    share[g // 2] = 0.0
    sizes = [int(n * s / sum(share)) for s in share]
    sizes[0] += n - sum(sizes)
    return sizes


def _layout(case):
    """(ends of the groups, rows in all): the groups start on multiples of the alignment."""
    ends, start = [], 0
    for size in _sizes(case):
        ends.append(start + size)
        start = (ends[-1] + ALIGN - 1) // ALIGN * ALIGN
    return ends, start


def _scale_storage(rows, hidden):
    """int16 scales of `rows` rows, consecutive rows contiguous."""
    return torch.empty_strided((rows, (hidden // 32 + 1) // 2), (1, rows), dtype=torch.int16, device='cuda').zero_()


def _fp8(rows, hidden):
    return torch.zeros((rows, hidden), dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn), _scale_storage(rows, hidden)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    kind, t = case['kind'], case['tokens']
    s = {'case': case}
    randn = lambda *shape, dt=torch.float32: torch.randn(shape, dtype=dt, device='cuda', generator=gen)  # noqa: E731
    if kind in ('route', 'route_grad'):
        s['logits'] = (randn(t, case['experts']) * 1.5).to(_TYPES[case['dtype']])
        s['bias'] = randn(case['experts']) * 0.1 if case.get('bias') else None
        if kind == 'route_grad':
            s['idx'] = (s['logits'].float() + randn(t, case['experts']) * 0.01).topk(case['topk'], dim=1).indices.int()
            s['g'] = randn(t, case['topk'])
        return s
    h = case['hidden']
    if kind in ('norm', 'norm_grad'):
        dt = _TYPES[case['dtype']]
        s['w'] = (1 + 0.1 * randn(h)).to(_TYPES[case['weight']])
        s['x'] = randn(t, h, dt=dt)
        s['residual'] = randn(t, h, dt=dt) * 2 if case['residual'] else None
        if kind == 'norm_grad':
            # (x stands for the sum; `residual` for the gradient that comes down the residual stream)
            s['rstd'] = _rstd(s['x'])
            s['g'] = randn(t, h, dt=torch.bfloat16)
        return s
    rows, s['psum'] = t, None
    if case.get('experts'):
        ends, rows = _layout(case)
        s['psum'] = torch.tensor(ends, dtype=torch.int32, device='cuda')
    s['live'] = _live(s['psum'], rows)
    if kind == 'weights':
        s['x'] = randn(rows, h, dt=torch.bfloat16) * h ** -0.5
        return s
    width = h if kind == 'operand' else 2 * h
    x = randn(rows, width, dt=torch.bfloat16)
    s['w'] = torch.rand(rows, device='cuda', generator=gen) * 0.5 + 0.01 if case.get('weights') else None
    if kind == 'act':
        s['x'] = x
        s['out'] = _fp8(rows, h), _fp8(rows, width)
        return s
    if case['from'] == 'fp8':
        q, e = _quantised(x.float())
        s['x'] = q.to(torch.float8_e4m3fn), _pairs(e)
    else:
        s['x'] = x
    if kind == 'act_grad':
        s['g'] = randn(rows, h, dt=torch.bfloat16)
        s['out'] = torch.zeros((rows, 2 * h), dtype=torch.bfloat16, device='cuda')
    return s


# ------------------------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------------------------
def _eight(pair, down=False):
    """(E4M3 values, the scales' powers of two) of a pair as the framework holds it; `down`: blocks run down the rows."""
    q, sf = pair
    return q, (sf if down else sf.t()).view(torch.float8_e8m0fnu)


def run(s):
    case = s['case']
    kind = case['kind']
    if own:
        import deep_gemm
        if kind == 'route':
            return deep_gemm.moe_route(s['logits'], case['topk'], case['scoring'], bias=s['bias'], num_groups=case['groups'], topk_groups=case['topk_groups'],
                                       renormalize=case['renormalize'], scale=2.5)
        if kind == 'route_grad':
            return deep_gemm.moe_route_grad(s['g'], s['logits'], s['idx'], case['scoring'], renormalize=case['renormalize'], scale=2.5)
        if kind == 'norm':
            pair, rows, h, rstd = deep_gemm.rms_norm_to_fp8(s['x'], s['w'], residual=s['residual'], eps=EPS, with_rows=case['rows'])
            return (*_eight(pair), rows, h, rstd)
        if kind == 'norm_grad':
            return deep_gemm.rms_norm_grad(s['g'], s['x'], s['w'], s['rstd'], grad_h=s['residual'])
        if kind == 'act':
            out, kept = deep_gemm.swiglu_apply_weight_to_fp8_with_checkpoint(s['x'], s['w'], s['psum'], case['clamp'] or None, ALIGN, out=s['out'])
            return (*_eight(out), *_eight(kept))
        if kind == 'act_grad':
            return deep_gemm.swiglu_apply_weight_grad(s['g'], s['x'], s['w'], s['psum'], case['clamp'] or None, ALIGN, out=s['out'])
        if kind == 'operand':
            return _eight(deep_gemm.cast_to_fp8(s['x'], s['psum'], ALIGN, mn_major=True), True)
        pair = deep_gemm.cast_to_fp8(s['x'], mn_major=True)
        return (*_eight(pair, True), deep_gemm.cast_from_fp8(pair, _TYPES[case['out']], mn_major=True))
    return _PLAIN[kind](s, case)


def _scores(logits, scoring):
    if scoring == 'sigmoid':
        return 1 / (1 + torch.exp(-logits))
    z = torch.exp(logits - logits.amax(1, keepdim=True))
    return z / z.sum(1, keepdim=True)


def _first(values, k):
    """The places of the k largest of each row, ties to the lowest."""
    return torch.sort(values, dim=1, descending=True, stable=True).indices[:, :k]


def _route(s, case):
    """(in 64 bits: scores next to one another decide who is chosen)"""
    t, e = s['logits'].shape
    scores = _scores(s['logits'].double(), case['scoring'])
    choice = scores if s['bias'] is None else scores + s['bias'].double()
    if s['bias'] is None:
        order = s['logits'].double()                              # the scores' own order, without their roundings
    else:
        order = choice
    if case['groups'] > 1:
        by_group = choice.view(t, case['groups'], -1)
        best = torch.sort(by_group, dim=2, descending=True).values[:, :, :2].sum(2)
        chosen = torch.zeros((t, case['groups']), dtype=torch.bool, device=choice.device)
        chosen.scatter_(1, _first(best, case['topk_groups']), True)
        order = torch.where(chosen.repeat_interleave(e // case['groups'], 1), order, -math.inf)
    idx = _first(order, case['topk'])
    w = scores.gather(1, idx)
    if case['renormalize']:
        w = w / w.sum(1, keepdim=True)
    return idx.int(), (w * 2.5).float()


def _route_grad(s, case):
    p, idx, g = _scores(s['logits'].float(), case['scoring']), s['idx'].long(), s['g'] * 2.5
    if case['renormalize']:
        # weights p_j / sum of the chosen p
        w = p.gather(1, idx)
        total = w.sum(1, keepdim=True)
        g = (g - (g * w).sum(1, keepdim=True) / total) / total
    dp = torch.zeros_like(p).scatter_(1, idx, g)
    if case['scoring'] == 'sigmoid':
        return (dp * p * (1 - p)).to(s['logits'].dtype)
    return (p * (dp - (dp * p).sum(1, keepdim=True))).to(s['logits'].dtype)


def _rstd(h):
    return (1 / torch.sqrt(h.double().square().mean(1) + EPS)).float()


def _norm(s, case):
    h = s['x'] if s['residual'] is None else (s['x'].float() + s['residual'].float()).to(s['x'].dtype)
    rstd = _rstd(h)
    y = h.float() * rstd[:, None] * s['w'].float()
    q, e = _quantised(y)
    return (*_eight((q.to(torch.float8_e4m3fn), _pairs(e))), y.bfloat16() if case['rows'] else None, h, rstd)


def _norm_grad(s, case):
    x, g = s['x'].float() * s['rstd'][:, None], s['g'].float()
    gw = g * s['w'].float()
    dx = s['rstd'][:, None] * (gw - x * (gw * x).mean(1, keepdim=True))
    if s['residual'] is not None:
        dx = dx + s['residual'].float()
    return dx.to(s['x'].dtype), (g * x).sum(0)


def _quantised(x):
    """FP32 [rows, cols] -> (values that E4M3 rounds, exponent bytes): blocks of 32 along the rows."""
    x = x.view(x.size(0), -1, 32)
    bits = (x.abs().amax(2).clamp(min=1e-4) * (1.0 / 448.0)).view(torch.int32)
    e = ((bits - 1) >> 23) + 1                                    # the smallest power of two that is not below
    return (x * ((254 - e) << 23).view(torch.float32)[:, :, None]).view(x.size(0), -1), e


def _pairs(e):
    """Exponent bytes [rows, blocks] -> int16 [rows, ceil(blocks / 2)], consecutive rows contiguous."""
    e = torch.nn.functional.pad(e, (0, e.size(1) % 2))
    pairs = torch.empty_strided((e.size(0), e.size(1) // 2), (1, e.size(0)), dtype=torch.int16, device=e.device)
    return pairs.copy_(e[:, 0::2] | (e[:, 1::2] << 8))


def _values(pair):
    """FP32 values of E4M3 with scales along the rows."""
    q, sf = pair
    e = torch.stack((sf.int() & 255, (sf.int() >> 8) & 255), dim=2).flatten(1)[:, :q.size(1) // 32]
    return (q.float().view(q.size(0), -1, 32) * (e << 23).view(torch.float32)[:, :, None]).view(q.shape)


def _live(psum, rows):
    """The rows that hold a value."""
    if psum is None:
        return torch.arange(rows, device='cuda')
    row, ends = torch.arange(rows, device='cuda'), psum.long()
    starts = torch.cat((ends.new_zeros(1), (ends[:-1] + ALIGN - 1) // ALIGN * ALIGN))
    return ((row[:, None] >= starts) & (row[:, None] < ends)).any(1).nonzero().view(-1)


def _halves(x, clamp):
    l, r = x.chunk(2, dim=1)
    return (l.clamp(max=clamp), r.clamp(-clamp, clamp)) if clamp else (l, r)


def _act(s, case):
    live = s['live']
    x = s['x'][live].float()
    l, r = _halves(x, case['clamp'])
    y = l / (1 + torch.exp(-l)) * r
    if s['w'] is not None:
        y = y * s['w'][live, None]
    got = []
    for (q, sf), v in zip(s['out'], (y, x)):
        v, e = _quantised(v)
        q.view(torch.uint8)[live] = v.to(torch.float8_e4m3fn).view(torch.uint8)
        sf[live] = _pairs(e)
        got += _eight((q, sf))
    return tuple(got)


def _act_grad(s, case):
    live = s['live']
    x = (_values(s['x']) if case['from'] == 'fp8' else s['x'].float())[live]
    g = s['g'][live].float()
    l, r = _halves(x, case['clamp'])
    sigma = 1 / (1 + torch.exp(-l))
    silu = l * sigma
    gw = g if s['w'] is None else g * s['w'][live, None]
    dl, dr = gw * r * (sigma + silu * (1 - sigma)), gw * silu
    if case['clamp']:
        xl, xr = x.chunk(2, dim=1)
        dl, dr = torch.where(xl <= case['clamp'], dl, 0.0), torch.where(xr.abs() <= case['clamp'], dr, 0.0)
    s['out'][live] = torch.cat((dl, dr), dim=1).bfloat16()
    if s['w'] is None:
        return s['out'], None
    dw = torch.zeros_like(s['w'])
    dw[live] = (g * silu * r).sum(1)
    return s['out'], dw


def _down(x):
    """FP32 [rows, cols] -> (E4M3, int16 scales [ceil(rows / 64), cols]): blocks of 32 down the rows, the last one perhaps short."""
    n = x.size(0)
    q, e = _quantised(torch.nn.functional.pad(x, (0, 0, 0, -n % 32)).t().contiguous())
    e = torch.where(torch.arange(e.size(1), device=e.device) * 32 < n, e, 0)
    return q.t()[:n].contiguous().to(torch.float8_e4m3fn), _pairs(e).t()


def _operand(s, case):
    x = _values(s['x']) if case['from'] == 'fp8' else s['x'].float()
    if s['psum'] is not None:
        keep = torch.zeros(x.size(0), dtype=torch.bool, device=x.device)
        keep[s['live']] = True
        x = torch.where(keep[:, None], x, 0.0)
    return _eight(_down(x), True)


def _weights(s, case):
    q, sf = _down(s['x'].float())
    e = torch.stack((sf.int() & 255, (sf.int() >> 8) & 255), dim=1).flatten(0, 1).repeat_interleave(32, 0)[:q.size(0)]
    return (*_eight((q, sf), True), (q.float() * (e << 23).view(torch.float32)).to(_TYPES[case['out']]))


_PLAIN = {'route': _route, 'route_grad': _route_grad, 'norm': _norm, 'norm_grad': _norm_grad, 'act': _act, 'act_grad': _act_grad,
          'operand': _operand, 'weights': _weights}


# ------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    kind = case['kind']
    s = prepare(case, seed)
    if kind in ('route', 'route_grad'):
        l = s['logits'].double()
        p = torch.sigmoid(l) if case['scoring'] == 'sigmoid' else torch.softmax(l, dim=1)
        if kind == 'route':
            c = p + (0 if s['bias'] is None else s['bias'].double())
            size = case['experts'] // case['groups']
            if case['groups'] > 1:
                best = torch.stack([c[:, i * size:(i + 1) * size].topk(min(2, size), dim=1).values.sum(1) for i in range(case['groups'])], dim=1)
                last = best.topk(case['topk_groups'], dim=1).values[:, -1:]
                c = c.masked_fill((best < last).repeat_interleave(size, dim=1), -math.inf)
            w = p.gather(1, c.topk(case['topk'], dim=1).indices)
            return None, 2.5 * (w / w.sum(1, keepdim=True) if case['renormalize'] else w)
        idx, g = s['idx'].long(), 2.5 * s['g'].double()
        l = l.requires_grad_()
        w = (torch.sigmoid(l) if case['scoring'] == 'sigmoid' else torch.softmax(l, dim=1)).gather(1, idx)
        if case['renormalize']:
            w = w / w.sum(1, keepdim=True)
        return torch.autograd.grad(w, l, g)[0]
    if kind in ('norm', 'norm_grad'):
        x, w = s['x'].double(), s['w'].double()
        if kind == 'norm':
            h = x if s['residual'] is None else x + s['residual'].double()
            held = h.to(s['x'].dtype).double()                    # what the residual stream holds, and the norm sees
            rstd = (held.pow(2).sum(1) / held.size(1) + EPS).rsqrt()
            y = held * rstd[:, None] * w
            return (*_micro64(y, 1), y if case['rows'] else None, h, rstd)
        r, g = s['rstd'].double()[:, None], s['g'].double()
        dot = torch.einsum('th,th,h->t', g, x, w)[:, None] / x.size(1)
        dx = r * w * g - r ** 3 * dot * x
        return dx if s['residual'] is None else dx + s['residual'].double(), torch.einsum('th,th->h', g, x * r)
    if kind == 'weights':
        q, e = _micro64(s['x'].double(), 0)
        return q, e, q * _power_of(s['x'].double(), 0)
    x = _decode64(s['x']) if case.get('from') == 'fp8' else s['x'].double()
    live = torch.zeros((x.size(0), 1), dtype=torch.bool, device=x.device)
    live[s['live']] = True
    x = torch.where(live, x, 0.0)
    if kind == 'operand':
        return _micro64(x, 0)
    h = case['hidden']
    xl, xr = x[:, :h], x[:, h:]
    l, r = (torch.minimum(xl, torch.full_like(xl, case['clamp'])), xr.clamp(-case['clamp'], case['clamp'])) if case['clamp'] else (xl, xr)
    w = torch.ones((x.size(0), 1), dtype=torch.float64, device=x.device) if s['w'] is None else s['w'].double()[:, None]
    silu = l * torch.sigmoid(l)
    if kind == 'act':
        got = []
        for v in (silu * r * w, x):
            q, e = _micro64(v, 1)
            # (rows without a value were never written)
            got += [torch.where(live, q, 0.0), torch.where(live.expand(-1, 2).reshape(-1), e, 2.0 ** -127)]
        return tuple(got)
    g = torch.where(live, s['g'].double(), 0.0)
    slope = torch.sigmoid(l)
    dl = g * w * r * slope * (1 + l * (1 - slope)) * ((xl <= case['clamp']) if case['clamp'] else 1.0)
    dr = g * w * silu * ((xr.abs() <= case['clamp']) if case['clamp'] else 1.0)
    return torch.cat((dl, dr), dim=1), None if s['w'] is None else torch.einsum('th,th->t', g, silu * r)


def _power_at_least(v):
    """The smallest power of two that is not below v > 0."""
    mantissa, exponent = torch.frexp(v)
    return torch.ldexp(torch.ones_like(v), exponent - (mantissa == 0.5).int())


def _blocks(x, axis):
    """[.., blocks, 32] of the blocks along `axis`, which comes last; zeros behind the end."""
    x = x.movedim(axis, -1)
    return torch.nn.functional.pad(x, (0, -x.size(-1) % 32)).unflatten(-1, (-1, 32))


def _power_of(x, axis):
    """The scale of every value of x."""
    scale = _power_at_least(_blocks(x, axis).abs().amax(-1).clamp(min=1e-4) / 448)
    return scale.repeat_interleave(32, dim=-1)[..., :x.size(axis)].movedim(-1, axis)


def _micro64(x, axis):
    """x in blocks of 32 along `axis` -> (E4M3 values, scales laid out as the pairs of int16 are: two bytes for each value along the other axis)."""
    n = x.size(axis)
    blocks = _blocks(x, axis)
    scale = _power_at_least(blocks.abs().amax(-1).clamp(min=1e-4) / 448)
    scaled = blocks / scale[..., None]
    grid = torch.exp2(torch.log2(scaled.abs().clamp(min=2.0 ** -6)).floor() - 3)          # three bits behind the leading one
    q = ((scaled / grid).round() * grid).flatten(-2)[..., :n].movedim(-1, axis)
    scale = torch.nn.functional.pad(scale, (0, scale.size(1) % 2), value=2.0 ** -127)      # [other axis, blocks]
    return q.contiguous(), scale.view(scale.size(0), -1, 2).transpose(0, 1).reshape(scale.size(1) // 2, -1)


def _decode64(pair):
    """E4M3 and scales along the rows -> float64."""
    q, sf = pair
    bits, e = q.view(torch.uint8).to(torch.int64), sf.to(torch.int64) & 0xFFFF
    exponent, mantissa = (bits >> 3) & 15, (bits & 7).double() / 8
    value = torch.where(exponent == 0, torch.ldexp(mantissa, torch.full_like(exponent, -6)), torch.ldexp(1 + mantissa, exponent - 7))
    value = torch.where(bits >= 128, -value, value)
    block = torch.arange(q.size(1), device=q.device) // 32
    return torch.ldexp(value, ((e[:, block // 2] >> (8 * (block % 2))) & 255) - 127)


# ------------------------------------------------------------------------------------------------------------------
def work(case):
    """Bytes with each input read once and each output written once. Padding costs nothing but where zeros are written."""
    kind, t = case['kind'], case['tokens']
    if kind in ('route', 'route_grad'):
        e, k, size = case['experts'], case['topk'], 4 if case['dtype'] == 'fp32' else 2
        if kind == 'route':
            return {'bytes': t * e * size + 8 * t * k + (4 * e if case['bias'] else 0), 'flops': 5 * t * e}
        return {'bytes': 2 * t * e * size + 8 * t * k, 'flops': 8 * t * e}
    h = case['hidden']
    size = 4 if case.get('dtype') == 'fp32' else 2
    if kind == 'norm':
        moved = 2 * h + (0 if case['dtype'] == 'bf16' else 2 * h)                            # x
        moved += 2 * h * size if case['residual'] else 0                                    # the residual, and the sum
        moved += h + h // 32 + (2 * h if case['rows'] else 0) + 4
        return {'bytes': t * moved + h * (4 if case['weight'] == 'fp32' else 2), 'flops': 6 * t * h}
    if kind == 'norm_grad':
        return {'bytes': t * (2 * h + h * size * (3 if case['residual'] else 2) + 4) + h * (8 if case['weight'] == 'fp32' else 6), 'flops': 10 * t * h}
    held = h + h // 32                                                                      # a row in 8 bits
    if kind == 'weights':
        return {'bytes': t * (2 * h + 2 * held + h * (2 if case['out'] == 'bf16' else 4)), 'flops': 4 * t * h}
    if kind == 'operand':
        rows = _layout(case)[1] if case['experts'] else t
        return {'bytes': t * (held if case['from'] == 'fp8' else 2 * h) + rows * held, 'flops': 4 * t * h}
    per_row = 4 if case['weights'] else 0
    if kind == 'act':
        return {'bytes': t * (4 * h + 3 * held + per_row), 'flops': 12 * t * h}
    return {'bytes': t * ((2 * held if case['from'] == 'fp8' else 4 * h) + 6 * h + 2 * per_row), 'flops': 20 * t * h}
