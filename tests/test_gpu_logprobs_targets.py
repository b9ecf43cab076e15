"""Targets outside the vocabulary: the gradient says so where the log probability does."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [7, 4001, 50000])
@pytest.mark.parametrize("dtype", ["int32", "int64"])
def test_gradient_of_a_target_past_the_vocabulary(cuda, vocab, dtype):
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    logits = torch.randn(6, vocab, generator=torch.Generator().manual_seed(vocab)).cuda()
    logits[4] = -math.inf
    targets = torch.tensor([2, vocab, vocab + 3, 2 ** 31 - 1, vocab, vocab], dtype=getattr(torch, dtype), device="cuda")
    gl = torch.tensor([1.0, 1.0, -0.5, 2.0, 1.0, 0.0], device="cuda")  # the last asks for nothing, the fifth row is masked
    logprob, entropy, m, ls = (torch.empty(6, device="cuda") for _ in range(4))
    tc.token_logprobs(logits, targets, logprob, entropy, m, ls)
    for gh in (None, torch.zeros(6, device="cuda")):
        d = torch.full_like(logits, 7.0)
        tc.token_logprobs_backward(logits, targets, m, ls, entropy, gl, gh, d)
        assert torch.isnan(logprob[1:]).all()
        assert torch.isfinite(d[0]).all() and torch.isnan(d[1:4]).all() and (d[4:] == 0).all()
