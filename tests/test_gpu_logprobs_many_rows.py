"""token_logprobs and its gradient where every CTA takes several rows, one after the other: rows of all kinds in turn (a
masked one, ties, NaN, infinities, too few unmasked entries), so that what one leaves behind would meet the next.
References and tolerances are those of test_gpu_logprobs.py."""
import math

import pytest

from test_gpu_logprobs import check_forward, check_gradients, make

pytestmark = pytest.mark.gpu


def spoil(torch, logits, targets):
    """Every 13th row is of a kind of its own, the others stay."""
    rows, vocab = logits.shape
    low = torch.finfo(logits.dtype).min
    for i in range(0, rows, 13):
        row, kind = logits[i], i // 13 % 8
        if kind == 0:
            row.fill_(-math.inf)
        elif kind == 1:
            row.fill_(0.5)
        elif kind == 2:
            row[vocab // 3] = math.nan
        elif kind == 3:
            row[vocab - 1] = math.inf
        elif kind == 4:
            row.fill_(-math.inf)
            row[vocab // 2], row[vocab - 1] = 1.0, -2.0
        elif kind == 5:
            row.fill_(low)
        elif kind == 6:
            targets[i] = -1
        else:
            row[::3] = 4.0


# more rows than CTAs: 8 per SM of 128 threads (vocabularies up to 512 vectors), 4 of 256
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,extra,lead,k", [(3001, 700, 0, 0, 20), (2500, 97, 3, 1, 32), (4000, 33, 0, 0, 5), (1300, 5003, 0, 3, 7),
                                                     (1900, 2048, 8, 0, 0), (1250, 9000, 5, 0, 0)])
def test_forward(cuda, rows, vocab, extra, lead, k, dtype):
    torch = cuda
    logits, _, g = make(torch, rows, vocab, dtype, rows, ld=vocab + extra, lead=lead, mask=0.1)
    targets = torch.randint(0, vocab, (rows,), generator=g)
    spoil(torch, logits, targets)
    check_forward(torch, logits, targets.cuda(), 0.9, k)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,extra,lead", [(3001, 700, 0, 0), (2500, 97, 3, 1), (700, 9001, 7, 0)])
def test_backward(cuda, rows, vocab, extra, lead, dtype):
    torch = cuda
    logits, _, g = make(torch, rows, vocab, dtype, rows, ld=vocab + extra, lead=lead, mask=0.1)
    targets = torch.randint(-1, vocab, (rows,), generator=g).cuda()
    logits[::11] = -math.inf
    gl, gh = torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda()
    check_gradients(torch, logits, targets, gl, gh, 1.1)


@pytest.mark.parametrize("rows,vocab,dtype,k", [(150, 131071, "f32", 20), (151, 262152, "bf16", 0)])
def test_clusters_of_ctas_with_several_rows(cuda, rows, vocab, dtype, k):
    """So long that 74 clusters of 8 CTAs take two or three rows each."""
    torch = cuda
    logits, _, g = make(torch, rows, vocab, dtype, rows, mask=0.1)
    targets = torch.randint(0, vocab, (rows,), generator=g)
    spoil(torch, logits, targets)
    check_forward(torch, logits, targets.cuda(), 1.0, k)
