"""The first call of a process inside a stream capture (the sort then sets its kernels' limits there), and plans made in inference mode."""

import os
import subprocess
import sys
import textwrap

import pytest
import torch

import deep_gemm

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = textwrap.dedent('''
    import sys
    sys.path.insert(0, %r)
    import torch
    import deep_gemm

    tokens, topk, experts, h = 2500, 4, 64, 2048                 # a sort over a cluster, an FP8 dispatch in two launches
    idx = torch.randint(-1, experts, (tokens, topk), device='cuda')
    x, w = torch.randn(tokens, h, device='cuda').bfloat16(), torch.rand(tokens, topk, device='cuda')


    def way():
        plan = deep_gemm.moe_sort(idx, experts)
        y = deep_gemm.moe_dispatch(x, plan, zero_padding=True)
        q, sf = deep_gemm.moe_dispatch_to_fp8(x, plan)
        c, s = deep_gemm.cast_to_fp4(y, plan[0])
        live = plan[2] >= 0
        return (*plan, deep_gemm.moe_combine(y, plan, w), deep_gemm.moe_combine_grad(x, y, plan, w)[1], deep_gemm.cast_from_fp4((c, s))), (q, sf, live)


    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, (q, sf, live) = way()
    graph.replay()
    torch.cuda.synchronize()
    fresh, (q2, sf2, live2) = way()
    rows = live2.nonzero().view(-1)
    assert torch.equal(live, live2) and all(torch.equal(a, b) for a, b in zip(held[:5], fresh[:5])) and torch.equal(held[5][rows], fresh[5][rows])
    assert torch.equal(q.view(torch.uint8)[rows], q2.view(torch.uint8)[rows]) and torch.equal(sf[rows], sf2[rows])
    print('PASS')
''') % os.path.join(ROOT, 'deepgemm-ascend_b200')


@pytest.mark.parametrize('python_host', ['0', '1'])
def test_a_capture_that_holds_the_first_call(python_host):
    proc = subprocess.run([sys.executable, '-c', SCRIPT], capture_output=True, text=True, timeout=600, env={**os.environ, 'DG_PYTHON_HOST': python_host})
    assert proc.returncode == 0 and 'PASS' in proc.stdout, proc.stderr[-3000:]


def test_a_plan_made_in_inference_mode():
    idx, x = torch.randint(0, 16, (70, 2), device='cuda'), torch.randn(70, 64, device='cuda', requires_grad=True)
    with torch.inference_mode():
        plan = deep_gemm.moe_sort(idx, 16)
        inside = deep_gemm.moe_combine(deep_gemm.moe_dispatch(x, plan), plan)
    outside = deep_gemm.moe_combine(deep_gemm.moe_dispatch(x.detach(), plan), plan)
    assert torch.equal(inside, outside) and torch.equal(outside, 2 * x.detach())
    assert all(torch.equal(a, b) for a, b in zip(plan, deep_gemm.moe_sort(idx, 16)))
