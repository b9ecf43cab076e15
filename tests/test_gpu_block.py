"""The fused operators run together, as a decoder layer's second half and the
head use them: training with every gradient, and single tokens in a CUDA graph.

Tolerance: a chain of at most 12 tensors, each rounded to bf16 once (half a step,
2^-9 of its own scale at most on average over a tensor, 2^-8 at worst): the norm
of the error is below 12 * 2^-8 of the norm of the result, whatever the
correlations; the operators' own fp32 errors are far below that."""
import math
import subprocess
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

BIN = Path(__file__).resolve().parent.parent / "bee_b200" / "_lib" / "test_host_bridge_block"


def test_cpp_bridge(cuda):
    assert BIN.exists(), "build the library first (python -m bee_b200.build)"
    r = subprocess.run([str(BIN)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "host bridge block ok" in r.stdout


def product(torch, a, b, b_trans=False):
    """a . b (or a . b^T) through the framework's own product."""
    from bee_b200 import _capi as C
    out = torch.empty(a.shape[0], b.shape[0] if b_trans else b.shape[1], dtype=a.dtype, device="cuda")
    C.call("bee_b200_bmm", C.BF16, C.BF16, a.data_ptr(), b.data_ptr(), out.data_ptr(), 1, a.shape[0], a.shape[1], out.shape[1],
           int(b_trans), 1.0, torch.cuda.current_stream().cuda_stream)
    return out


def transposed(torch, a):
    from bee_b200 import _capi as C
    out = torch.empty(a.shape[1], a.shape[0], dtype=a.dtype, device="cuda")
    C.call("bee_b200_transpose_2d", C.BF16, a.data_ptr(), out.data_ptr(), a.shape[0], a.shape[1], torch.cuda.current_stream().cuda_stream)
    return out


class Block:
    """h0 (attention's output) and x0 to logits, and back."""

    def __init__(self, torch, tokens, sequences, d, f, vocab, seed):
        g = torch.Generator().manual_seed(seed)

        def t(*shape, scale=1.0, shift=0.0):
            return (torch.randn(*shape, generator=g) * scale + shift).bfloat16().cuda()

        self.torch, self.tokens = torch, tokens
        self.p = {"h0": t(tokens, d), "x0": t(tokens, d), "gate0": t(sequences, d, scale=0.3, shift=0.8), "post0": t(d, scale=0.1, shift=1.0),
                  "pre0": t(d, scale=0.1, shift=1.0), "wg": t(f, d, scale=d ** -0.5), "wu": t(f, d, scale=d ** -0.5),
                  "wd": t(f, d, scale=2 * f ** -0.5), "post1": t(d, scale=0.1, shift=1.0), "pre1": t(d, scale=0.1, shift=1.0),
                  "head": t(d, vocab, scale=1.5 * d ** -0.5)}
        self.targets = torch.randint(0, vocab, (tokens,), generator=g).cuda()
        self.targets[-1] = -1
        self.weight = torch.rand(tokens, generator=g).cuda()
        self.f, self.vocab = f, vocab

    def forward(self, save=True, top=0):
        from bee_b200 import tensor_cuda as tc
        torch, p, n = self.torch, self.p, self.tokens
        s = {"x1": torch.empty_like(p["x0"]), "y1": torch.empty_like(p["x0"]), "x2": torch.empty_like(p["x0"]), "y2": torch.empty_like(p["x0"])}
        s |= {k: torch.empty(n, self.f, dtype=torch.bfloat16, device="cuda") for k in ("a", "g", "u")}
        s |= {k: torch.empty(n, device="cuda") for k in ("logprob", "entropy", "row_max", "log_sum")}
        tc.norm_gate_residual(p["h0"], p["x0"], s["x1"], s["y1"], w_post=p["post0"], gate=p["gate0"], w_pre=p["pre0"])
        tc.gated_linear(s["y1"], p["wg"], p["wu"], s["a"], trans=True, g=s["g"] if save else None, u=s["u"] if save else None)
        s["h1"] = product(torch, s["a"], p["wd"])
        tc.norm_gate_residual(s["h1"], s["x1"], s["x2"], s["y2"], w_post=p["post1"], w_pre=p["pre1"], beta=0.5)
        s["logits"] = product(torch, s["y2"], p["head"])
        if top:
            s["ids"], s["top"] = torch.empty(n, top, dtype=torch.int32, device="cuda"), torch.empty(n, top, device="cuda")
        tc.token_logprobs(s["logits"], self.targets, s["logprob"], s["entropy"], s["row_max"], s["log_sum"], temperature=0.9,
                          top_ids=s.get("ids"), top_logprobs=s.get("top"))
        return s

    def backward(self, s):
        """Gradients of -sum(weight logprob) - 0.1 sum(entropy)."""
        from bee_b200 import tensor_cuda as tc
        torch, p = self.torch, self.p
        d = {"d" + k: torch.empty_like(v) for k, v in p.items()}
        dlogits = torch.empty_like(s["logits"])
        tc.token_logprobs_backward(s["logits"], self.targets, s["row_max"], s["log_sum"], s["entropy"], -self.weight,
                                   torch.full_like(self.weight, -0.1), dlogits, temperature=0.9)
        dy2 = product(torch, dlogits, p["head"], b_trans=True)
        d["dhead"] = product(torch, transposed(torch, s["y2"]), dlogits)
        dh1, dx1 = torch.empty_like(dy2), torch.empty_like(dy2)
        tc.norm_gate_residual_backward(s["h1"], s["x1"], None, dy2, dh1, dx1, w_post=p["post1"], w_pre=p["pre1"], dw_post=d["dpost1"],
                                       dw_pre=d["dpre1"], beta=0.5)
        da = product(torch, dh1, p["wd"], b_trans=True)
        d["dwd"] = product(torch, transposed(torch, s["a"]), dh1)
        dy1 = torch.empty_like(dy2)
        tc.gated_linear_backward(s["y1"], p["wg"], p["wu"], s["g"], s["u"], da, dy1, d["dwg"], d["dwu"], trans=True)
        tc.norm_gate_residual_backward(p["h0"], p["x0"], dx1, dy1, d["dh0"], d["dx0"], w_post=p["post0"], gate=p["gate0"], w_pre=p["pre0"],
                                       dw_post=d["dpost0"], dgate=d["dgate0"], dw_pre=d["dpre0"])
        return d

    def exact(self):
        """Loss terms and gradients in 64 bits, by differentiation."""
        torch, n = self.torch, self.tokens
        p = {k: v.double().requires_grad_() for k, v in self.p.items()}

        def rms(v, w):
            return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w

        gate = p["gate0"].repeat_interleave(n // p["gate0"].shape[0], 0)
        x1 = p["x0"] + gate * rms(p["h0"], p["post0"])
        y1 = rms(x1, p["pre0"])
        g = y1 @ p["wg"].t()
        h1 = (g * torch.sigmoid(g) * (y1 @ p["wu"].t())) @ p["wd"]
        y2 = rms(x1 + 0.5 * rms(h1, p["post1"]), p["pre1"])
        lp = torch.log_softmax(y2 @ p["head"] / 0.9, -1)
        inside = self.targets >= 0
        logprob = lp.gather(1, self.targets.clamp(min=0)[:, None])[:, 0] * inside
        entropy = -(lp.exp() * lp).sum(-1)
        loss = -(self.weight.double() * logprob).sum() - 0.1 * entropy.sum()
        return logprob, entropy, dict(zip(("d" + k for k in p), torch.autograd.grad(loss, list(p.values()))))


def test_training_step(cuda):
    torch = cuda
    b = Block(torch, tokens=600, sequences=5, d=512, f=1096, vocab=1000, seed=0)
    s = b.forward()
    d = b.backward(s)
    logprob, entropy, want = b.exact()
    bound = 12 * 2.0 ** -8

    def off(got, ref):
        return float((got.double() - ref.detach()).norm() / ref.detach().norm())

    assert off(s["logprob"], logprob) < bound and off(s["entropy"], entropy) < bound
    for k in want:
        assert off(d[k], want[k]) < bound, (k, off(d[k], want[k]))
    again = b.backward(b.forward())
    assert all(torch.equal(again[k], d[k]) for k in d)


def test_single_tokens_in_a_graph(cuda):
    """Two sequences a token at a time: a captured step gives the bits of the eager one, and tops agree with the logits."""
    torch = cuda
    b = Block(torch, tokens=2, sequences=2, d=1024, f=2048, vocab=20000, seed=1)
    want = b.forward(save=False, top=5)
    torch.cuda.synchronize()
    assert torch.equal(want["ids"].long(), want["logits"].float().sort(dim=-1, descending=True, stable=True).indices[:, :5])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = b.forward(save=False, top=5)
    keep = b.p["h0"].clone()
    b.p["h0"].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(s["logits"], want["logits"])
    b.p["h0"].copy_(keep)
    graph.replay()
    torch.cuda.synchronize()
    for k in ("x2", "y2", "logits", "logprob", "entropy", "ids", "top"):
        assert torch.equal(s[k], want[k]), k
    assert all(math.isfinite(v) for v in s["entropy"].tolist())
