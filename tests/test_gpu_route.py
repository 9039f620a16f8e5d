"""The router's choice and its gradient against loops in 64 bits on the CPU (oracle/layers.py).

Tolerances, e = 2^-24. Sigmoid: the exponential within 2 ulp (4 e), one addition, one division: a score within 8 e of its value; a weight
that is divided by a sum of at most 32 of them within 8 e + 8 e + 7 e. Softmax: rounding l - max moves a score by e |l - max| of its value, the
exponential by 4 e, the sum of at most 64 + 5 additions (and its terms) by 69 e + what moves them, the division by e: within
(2 |l - max| + 90) e in all, |l - max| the largest of the row's. A gradient is a sum of at most 32 + 5 terms made of a few such factors: within three
times that bound, and 40 e, of the sum of its terms' magnitudes; its rounding to BF16 adds 2^-8 of the value. A score under 2^-126 is held
in steps of 2^-149, which the least sum, 1e-20, turns into 2^-82 of a weight."""

import math

import pytest
import torch

import deep_gemm
import oracle
from both_hosts import moe_hosts, python_layer
from helpers import seed_all

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
INF, NAN = math.inf, math.nan


def _relative(logits, scoring):
    """[tokens, 1]: how far a score may be from its value, relative."""
    if scoring == 'sigmoid':
        return torch.full((logits.size(0), 1), 24 * E, dtype=torch.float64)
    l = torch.where(logits == -INF, NAN, logits.double())
    spread = torch.stack([(r[~r.isnan()].max() - r[~r.isnan()].min()) if (~r.isnan()).any() else torch.tensor(0.0).double() for r in l])
    return ((2 * spread + 90) * E)[:, None]


def _check(logits, topk, scoring='softmax', host=deep_gemm, **kw):
    cuda = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    idx, w = host.moe_route(logits.cuda(), topk, scoring, **cuda)
    ref_idx, ref_w = oracle.moe_route_ref(logits, topk, scoring, **kw)
    assert idx.dtype == torch.int32 and w.dtype == torch.float32 and idx.shape == w.shape == ref_idx.shape
    assert torch.equal(idx.cpu(), ref_idx)
    assert ((w.cpu().double() - ref_w).abs() <= (2 * _relative(logits, scoring) + 8 * E) * ref_w.abs() + 2.0 ** -82).all()
    return idx, w


ROUTERS = [(1, 1, 1, 1, 1), (1, 256, 8, 8, 4), (7, 64, 6, 1, 1), (33, 160, 6, 8, 3), (50, 60, 4, 3, 2), (9, 1000, 10, 5, 2), (5, 1024, 32, 32, 16), (3, 1020, 8, 17, 4),
           (40, 8, 8, 4, 4), (20, 33, 32, 1, 1), (12, 31, 2, 31, 7), (128, 256, 8, 8, 4)]


@pytest.mark.parametrize('host', moe_hosts)
@pytest.mark.parametrize('tokens,experts,topk,groups,taken', ROUTERS)
@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_choices(host, tokens, experts, topk, groups, taken, scoring, dtype):
    seed_all(tokens + experts)
    logits = (torch.randn(tokens, experts) * 2).to(dtype)
    bias = torch.randn(experts) * 0.1
    for best in (1, 2):
        for b in (None, bias, torch.zeros(experts)):
            _check(logits, topk, scoring, host, bias=b, num_groups=groups, topk_groups=taken, group_best=best, renormalize=best == 2, scale=2.5)


def test_choices_that_32_bits_leave_open():
    """Scores that differ by less than FP32 holds, and ties."""
    seed_all(1)
    for scoring in ('softmax', 'sigmoid'):
        base = torch.randn(64, 32)
        logits = torch.cat([base, torch.nextafter(base, torch.tensor(INF)), base, base + 1e-6], dim=1)[:, torch.randperm(128)]
        for groups, taken in ((1, 1), (8, 3), (16, 16)):
            for bias in (None, torch.zeros(128), torch.full((128,), 0.25), torch.randn(4).repeat(32) * 1e-7, 8 + torch.randn(128) * 1e-6):
                for best in (1, 2):
                    _check(logits, 8, scoring, bias=bias, num_groups=groups, topk_groups=taken, group_best=best)
        # all that there are, and all but one; as many as lanes
        for bias in (None, torch.zeros(128), torch.randn(4).repeat(32) * 1e-7):
            for n in (8, 9, 32, 33):
                _check(logits[:, :n].contiguous(), min(n, 8 if n < 10 else 32), scoring, bias=None if bias is None else bias[:n].contiguous())
        # a bias that makes up for the scores' differences
        logits = torch.randn(1, 64).expand(40, 64) + torch.randn(40, 1)
        scores = torch.sigmoid(logits) if scoring == 'sigmoid' else torch.softmax(logits, 1)
        bias = (2 - scores[0]).float()
        _check(logits.contiguous(), 6, scoring, bias=bias)
        _check(logits.contiguous(), 6, scoring, bias=bias, num_groups=8, topk_groups=4)


def test_large_and_equal_logits():
    seed_all(2)
    _check(torch.zeros(5, 100), 7)
    _check(torch.zeros(5, 96), 7, 'sigmoid', bias=torch.zeros(96), num_groups=4, topk_groups=2)
    _check(torch.tensor([[0.0, -0.0, 0.0, -0.0, -1.0]]), 4)
    _check(torch.tensor([[0.0, -0.0, 0.0, -0.0, -1.0]]), 4, 'sigmoid', bias=torch.zeros(5))
    _check(torch.randn(9, 64) * 1e4, 4)                                   # scores of exactly 0
    _check(torch.randn(9, 64) * 30, 4, 'sigmoid', renormalize=True)
    _check(-90 + torch.randn(9, 64), 4, 'sigmoid', renormalize=True)      # a sum below the least one
    _check(torch.full((3, 8), 3e38), 2)


def test_masked_experts():
    seed_all(3)
    logits = torch.randn(30, 48)
    logits[torch.rand(30, 48) < 0.9] = -INF
    logits[4] = -INF
    logits[5, 1:] = -INF
    logits[6, :-1] = -INF
    bias = torch.randn(48)
    bias[::5] = -INF
    for scoring in ('softmax', 'sigmoid'):
        for b in (None, bias):
            for groups, taken in ((1, 1), (6, 2), (12, 5)):
                idx, w = _check(logits, 6, scoring, bias=b, num_groups=groups, topk_groups=taken, renormalize=True)
                assert (idx[4] == -1).all() and (w[4] == 0).all()
    layout, token_rows, _ = deep_gemm.moe_sort(idx, 48)
    assert (token_rows[4] == -1).all() and ((token_rows >= 0) == (idx >= 0)).all()


def test_what_is_not_finite_shows():
    logits = torch.randn(4, 40)
    logits[1, 7], logits[2, 9], logits[2, 3] = NAN, NAN, NAN
    idx, w = deep_gemm.moe_route(logits.cuda(), 3, 'sigmoid')
    assert idx[1, 0] == 7 and w[1, 0].isnan() and not w[1, 1:].isnan().any() and idx[2, :2].tolist() == [3, 9] and w[2, :2].isnan().all()
    assert not w[0].isnan().any() and not w[3].isnan().any()
    idx, w = deep_gemm.moe_route(logits.cuda(), 3, bias=torch.zeros(40, device='cuda'), num_groups=4, topk_groups=1)
    assert w[1].isnan().all() and w[2].isnan().all() and not w[3].isnan().any() and (idx >= 0).all() and (idx < 40).all()
    logits = torch.full((2, 40), -INF)
    logits[0, 4] = NAN
    assert deep_gemm.moe_route(logits.cuda(), 2)[0].tolist() == [[4, -1], [-1, -1]] and deep_gemm.moe_route(logits.cuda(), 2)[1][0, 0].isnan()
    logits = torch.randn(1, 40)
    logits[0, 9] = INF
    assert deep_gemm.moe_route(logits.cuda(), 2)[0][0, 0] == 9


def test_many_tokens():
    """Against torch on the GPU in 64 bits: an odd number of tokens over many CTAs."""
    seed_all(4)
    logits, bias = torch.randn(30001, 256, device='cuda') * 1.5, torch.randn(256, device='cuda') * 0.1
    idx, w = deep_gemm.moe_route(logits, 8, 'sigmoid', bias=bias, num_groups=8, topk_groups=4, renormalize=True)
    s = torch.sigmoid(logits.double())
    c = s + bias.double()
    best = c.view(-1, 8, 32).topk(2, dim=2).values.sum(2)
    taken = torch.zeros(30001, 8, dtype=torch.bool, device='cuda').scatter_(1, best.topk(4, dim=1).indices, True)
    want = torch.where(taken.repeat_interleave(32, 1), c, -INF).topk(8, dim=1).indices
    assert torch.equal(idx.long(), want)
    p = s.gather(1, want)
    assert ((w - p / p.sum(1, keepdim=True)).abs() <= 56 * E * w).all()
    logits = logits.bfloat16()
    idx, w = deep_gemm.moe_route(logits, 8)
    order = torch.sort(logits.float(), dim=1, descending=True, stable=True)
    assert torch.equal(idx.long(), order.indices[:, :8])


# --------------------------------------------------------------------------------------------------------------- gradient
@pytest.mark.parametrize('host', moe_hosts)
@pytest.mark.parametrize('tokens,experts,topk', [(1, 1, 1), (5, 8, 2), (17, 64, 6), (6, 33, 32), (9, 160, 8), (3, 1024, 8), (2, 1000, 31)])
@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_gradient(host, tokens, experts, topk, scoring, dtype):
    seed_all(tokens)
    logits, g = (torch.randn(tokens, experts) * 2).to(dtype), torch.randn(tokens, topk)
    for renormalize in (False, True):
        idx, _ = host.moe_route(logits.cuda(), topk, scoring)
        if topk > 1 and tokens > 1:
            idx[1, 0], g[1, 0] = -1, NAN                                  # a choice that is none, whatever its gradient
        if topk > 2 and tokens > 2:
            idx[2, 1] = idx[2, 0]                                         # the same twice
        for index in (idx, idx.long()):
            got = host.moe_route_grad(g.cuda(), logits.cuda(), index, scoring, renormalize, 2.5)
            assert got.dtype == dtype and got.shape == logits.shape
            want, size = oracle.moe_route_grad_ref(g, logits, idx.cpu(), scoring, renormalize, 2.5)
            err = (3 * _relative(logits, scoring) + 40 * E) * size
            err += HALF[dtype] * (want.abs() + err) + 2.0 ** -140
            assert ((got.cpu().double() - want).abs() <= err).all()


def test_gradient_of_masked_rows_and_far_logits():
    seed_all(6)
    logits, g = torch.randn(6, 40), torch.randn(6, 4)
    logits[1] = -INF
    logits[2, 3:] = -INF
    logits[3] *= 40
    for scoring in ('softmax', 'sigmoid'):
        for renormalize in (False, True):
            idx, _ = deep_gemm.moe_route(logits.cuda(), 4, scoring, renormalize=renormalize)
            got = deep_gemm.moe_route_grad(g.cuda(), logits.cuda(), idx, scoring, renormalize).cpu().double()
            want, size = oracle.moe_route_grad_ref(g, logits, idx.cpu(), scoring, renormalize)
            assert torch.isfinite(got).all() and (got[1] == 0).all()
            if renormalize:
                got, want, size = (torch.cat((t[:3], t[4:])) for t in (got, want, size))      # (40 apart: sums near the least one)
            far = torch.where(logits == -INF, 0.0, logits).abs().max()
            assert ((got - want).abs() <= (3 * (4 * far + 90) * E + 40 * E) * size + 2.0 ** -100).all()


def test_gradient_against_differences():
    seed_all(7)
    logits, g = torch.randn(4, 24, dtype=torch.float64), torch.randn(4, 3)
    for scoring in ('softmax', 'sigmoid'):
        for renormalize in (False, True):
            idx = oracle.moe_route_ref(logits, 3, scoring)[0]
            got = deep_gemm.moe_route_grad(g.cuda(), logits.float().cuda(), idx.cuda(), scoring, renormalize, 1.5).cpu().double()

            def loss(l):
                s = (torch.sigmoid(l) if scoring == 'sigmoid' else torch.softmax(l, 1)).gather(1, idx.long())
                return float((g.double() * 1.5 * (s / s.sum(1, keepdim=True) if renormalize else s)).sum())
            for t, e in ((0, int(idx[0, 0])), (1, int(idx[1, 2])), (2, 5), (3, 23)):
                step = torch.zeros_like(logits)
                step[t, e] = 1e-5
                # (a central difference in 64 bits: 1e-10 of the third derivative, 1e-11 from rounding; FP32: 1e-6 of values around 1)
                assert abs((loss(logits + step) - loss(logits - step)) / 2e-5 - float(got[t, e])) < 2e-5


def test_refusals():
    x = torch.zeros(4, 64, device='cuda')
    for host in moe_hosts:
        for kw, match in ((dict(topk=0), 'topk must be'), (dict(topk=33), 'topk must be'), (dict(topk=2, scoring='relu'), 'scoring must be'),
                          (dict(topk=2, bias=torch.zeros(63, device='cuda')), 'bias must be'), (dict(topk=2, bias=torch.zeros(64)), 'bias must be'),
                          (dict(topk=2, bias=torch.zeros(64, device='cuda').bfloat16()), 'bias must be'), (dict(topk=2, num_groups=3), 'num_groups must be'),
                          (dict(topk=2, num_groups=64), 'num_groups must be'), (dict(topk=2, num_groups=4, topk_groups=5), 'topk_groups must be'),
                          (dict(topk=2, num_groups=4, group_best=3), 'group_best must be'), (dict(topk=20, num_groups=4, topk_groups=1), 'fewer experts than topk')):
            with pytest.raises(RuntimeError, match=match):
                host.moe_route(x, **kw)
        with pytest.raises(RuntimeError, match='logits must be'):
            host.moe_route(x.t(), 2)
        with pytest.raises(RuntimeError, match='logits must be'):
            host.moe_route(x.half(), 2)
        with pytest.raises(RuntimeError, match='number of experts'):
            host.moe_route(torch.zeros(2, 1025, device='cuda'), 2)
        idx, g = torch.zeros(4, 2, dtype=torch.int32, device='cuda'), torch.zeros(4, 2, device='cuda')
        for args, match in (((g[:, :1], x, idx), 'grad_weights must be'), ((g.bfloat16(), x, idx), 'grad_weights must be'), ((g, x, idx.short()), 'topk_idx must be'),
                            ((g, x, idx.t()), 'topk_idx must be'), ((g, x[:3], idx), 'topk_idx must be')):
            with pytest.raises(RuntimeError, match=match):
                host.moe_route_grad(*args)
        for out in (x.bfloat16(), x[:3], x.expand(4, 64)[:, :32], torch.zeros(1, 64, device='cuda').expand(4, 64)):
            with pytest.raises(RuntimeError, match='out must be'):
                host.moe_route_grad(g, x, idx, out=out)


def test_no_tokens_strides_and_in_place():
    seed_all(8)
    for host in moe_hosts:
        idx, w = host.moe_route(torch.zeros(0, 64, device='cuda'), 4)
        assert idx.shape == w.shape == (0, 4)
        assert host.moe_route_grad(w, torch.zeros(0, 64, device='cuda'), idx).shape == (0, 64)
        wide = torch.randn(21, 200, device='cuda')
        x = wide[:, 3:163]
        idx, w = host.moe_route(x, 5)
        again = host.moe_route(x.contiguous(), 5)
        assert torch.equal(idx, again[0]) and torch.equal(w, again[1])
        g = torch.randn(21, 5, device='cuda')
        want = host.moe_route_grad(g, x.contiguous(), idx)
        before = wide.clone()
        assert host.moe_route_grad(g, x, idx, out=x).data_ptr() == x.data_ptr()
        assert torch.equal(x, want) and torch.equal(wide[:, :3], before[:, :3]) and torch.equal(wide[:, 163:], before[:, 163:])
        same = torch.randn(1, 160, device='cuda').expand(5, 160)          # a broadcast input
        idx, w = host.moe_route(same, 5)
        assert (idx == idx[0]).all() and (w == w[0]).all()


def test_rows_behind_32_bits():
    """Rows whose offsets pass 2^32 bytes."""
    tokens, experts = 70000, 16
    base = torch.zeros(tokens * 16640, dtype=torch.float32, device='cuda')
    x = base.as_strided((tokens, experts), (16640, 1))
    x.copy_(torch.randn(tokens, experts))
    idx, w = deep_gemm.moe_route(x, 3)
    again = deep_gemm.moe_route(x.contiguous(), 3)
    assert torch.equal(idx, again[0]) and torch.equal(w, again[1])
    g = torch.randn(tokens, 3, device='cuda')
    want = deep_gemm.moe_route_grad(g, x.contiguous(), idx)
    assert torch.equal(deep_gemm.moe_route_grad(g, x, idx, out=x), want)


def test_another_stream_a_captured_run_and_both_hosts():
    seed_all(9)
    layer = python_layer('moe_ops')
    x, bias, g = torch.randn(300, 64, device='cuda'), torch.randn(64, device='cuda') * 0.1, torch.randn(300, 6, device='cuda')

    def way(host=deep_gemm):
        idx, w = host.moe_route(x, 6, 'sigmoid', bias=bias, num_groups=4, topk_groups=2, renormalize=True)
        return idx, w, host.moe_route_grad(g, x, idx, 'sigmoid', True)
    want = way()
    assert all(torch.equal(a, b) for a, b in zip(want, way(layer)))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = way()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = way()
    x.copy_(torch.randn(300, 64, device='cuda'))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, way()))
