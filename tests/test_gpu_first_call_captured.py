"""The first call of the fused block operators in a process may be a captured one: the modules load and the memory pool
is set up without ending the capture.  Each order begins with another operator, in a process of its own; the replays
give the bits of the calls alone."""
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

PROGRAM = textwrap.dedent("""
    import sys
    import torch
    from bee_b200 import tensor_cuda as tc

    g = torch.Generator().manual_seed(0)
    t = lambda *shape, scale=1.0: (torch.randn(*shape, generator=g) * scale).bfloat16().cuda()
    x, w, wg, wu, few = t(300, 1000), t(1000), t(520, 1000, scale=0.03), t(520, 1000, scale=0.03), t(3, 1000)
    gg, u, dout, targets = t(300, 520), t(300, 520), t(300, 520), torch.arange(300).cuda()
    m, ls, ent, gl = x.float().amax(-1), torch.full((300,), 2.0).cuda(), torch.ones(300).cuda(), torch.ones(300).cuda()

    def norm(o):
        tc.norm_gate_residual(x, x, o[0], o[1], w_post=w, w_pre=w)
    def norm_backward(o):
        tc.norm_gate_residual_backward(x, x, x, x, o[0], o[1], w_post=w, gate=w, w_pre=w, dw_post=o[2], dgate=o[3], dw_pre=o[4])
    def linear(o):
        tc.gated_linear(x, wg, wu, o[0], trans=True, g=o[1], u=o[2])
    def linear_few(o):
        tc.gated_linear(few, wg, wu, o[0], trans=True)
    def linear_backward(o):
        tc.gated_linear_backward(x, wg, wu, gg, u, dout, o[0], o[1], o[2], trans=True)
    def logprobs(o):
        tc.token_logprobs(x, targets, *o[:4], top_ids=o[4], top_logprobs=o[5])
    def logprobs_backward(o):
        tc.token_logprobs_backward(x, targets, m, ls, ent, gl, gl, o[0])

    e, f = torch.empty_like, lambda *s, **k: torch.empty(*s, device="cuda", **k)
    outputs = {"norm": lambda: [e(x), e(x)], "norm_backward": lambda: [e(x), e(x), e(w), e(w), e(w)], "linear": lambda: [e(gg), e(gg), e(gg)],
               "linear_few": lambda: [few.new_empty(3, 520)], "linear_backward": lambda: [e(x), e(wg), e(wu)],
               "logprobs": lambda: [f(300), f(300), f(300), f(300), f(300, 5, dtype=torch.int32), f(300, 5)], "logprobs_backward": lambda: [e(x)]}
    for name in sys.argv[1].split(","):
        o, graph = outputs[name](), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            globals()[name](o)
        graph.replay()
        want = outputs[name]()
        globals()[name](want)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(o, want)), name
    print("captured ok")
""")


@pytest.mark.parametrize("order", ["norm_backward,norm,linear,linear_few,logprobs,logprobs_backward", "linear_backward,linear"])
def test_first_calls(cuda, order):
    r = subprocess.run([sys.executable, "-c", PROGRAM, order], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and "captured ok" in r.stdout, r.stdout + r.stderr
