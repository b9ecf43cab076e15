"""token_logprobs and its gradient against the definition in 64 bits.

Tolerances, from the arithmetic.  A partial sum of exponentials passes through
at most 16 (a batch of chunks, two lanes wide) + vocab / (16 * 128) (batches of
the smallest block's thread) + 29 (lanes, warps, cluster) fp32 additions; for
every size here that is below 2^8, so the relative error of S is below
2^8 * 2^-24 = 2^-16, plus 2^-21 for the exponential and its argument's rounding
on the terms that matter.  log S, and with it logp, is then off by at most
2^-15 absolute, plus 2^-22 of |z| for the scaled difference z (three roundings,
the reciprocal temperature included).  The entropy adds the same relative error
of sum e z / S, whose value is log S - H.  A gradient in fp32 is p (A + B logp):
a relative error 2^-14 of p's scale times (|gl| + |gH| (|logp| + H)); 16-bit
gradients add half a step of their type, and 2^-25 where fp16 is subnormal."""
import math

import pytest

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


def make(torch, rows, vocab, dtype, seed, ld=None, lead=0, mask=0.0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * scale
    if mask:
        x[torch.rand(rows, vocab, generator=g) < mask] = -math.inf
    ld = ld or vocab
    buf = torch.full((lead + rows * ld + 16,), 7.0, dtype=getattr(torch, DT[dtype]), device="cuda")
    view = torch.as_strided(buf, (rows, vocab), (ld, 1), lead)
    view.copy_(x.to(view.dtype))
    return view, buf, g


def reference(torch, logits, targets, temperature, k):
    x = logits.double().cpu()
    m = x.amax(-1)
    empty = m == -math.inf
    z = (x - torch.where(empty, 0.0, m)[:, None]) / temperature
    e = z.exp()
    s = e.sum(-1)
    log_s = s.log()
    lp = z - log_s[:, None]
    lp[empty] = -math.inf
    ent = torch.where(empty, 0.0, log_s - torch.where(e > 0, e * z, 0.0).sum(-1) / s)
    t = targets.cpu().long()
    got = lp.gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    got = torch.where(t < 0, 0.0, torch.where(t >= x.shape[1], math.nan, got))
    bad = ~torch.isfinite(s)
    got[bad & (t >= 0)] = math.nan
    ids = x.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    top = lp.gather(1, ids)
    ids[bad], top[bad] = -1, math.nan
    ent[bad] = math.nan
    return {"logprob": got, "entropy": ent, "row_max": m, "log_sum": log_s, "ids": ids, "top": top, "lp": lp, "p": lp.exp()}


def close(torch, got, want, tol, what):
    # the outputs' type is fp32 at most: what is beyond its range rounds to infinity
    # (a lowest logit under a temperature below 1: 3.39e38 / 0.9 > 3.403e38)
    got, want = got.double().cpu(), want.double()
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, want.float().double(), want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    ok = torch.isfinite(want)
    assert torch.isfinite(got[ok]).all(), what
    bad = (got - want).abs()[ok] > (tol.expand_as(want)[ok] if isinstance(tol, torch.Tensor) else tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} outside, worst {(got - want).abs()[ok].max():.3e}"


def forward(torch, logits, targets, temperature, k):
    from bee_b200 import tensor_cuda as tc
    rows = logits.shape[0]
    out = {n: torch.full((rows,), 9.0, device="cuda") for n in ("logprob", "entropy", "row_max", "log_sum")}
    if k:
        out["ids"] = torch.full((rows, k), -7, device="cuda", dtype=torch.int32)
        out["top"] = torch.full((rows, k), 9.0, device="cuda")
    tc.token_logprobs(logits, targets, out["logprob"], out["entropy"], out["row_max"], out["log_sum"],
                      temperature=temperature, top_ids=out.get("ids"), top_logprobs=out.get("top"))
    torch.cuda.synchronize()
    return out


def check_forward(torch, logits, targets, temperature, k):
    got, want = forward(torch, logits, targets, temperature, k), reference(torch, logits, targets, temperature, k)
    z = want["log_sum"].nan_to_num(0.0, 0.0, 0.0).abs()
    close(torch, got["row_max"], want["row_max"], 0.0, "row_max") if not torch.isnan(want["row_max"]).any() else None
    bad = torch.isnan(want["entropy"])
    keep = ~bad
    close(torch, got["log_sum"][keep.cuda()], want["log_sum"][keep], 2.0 ** -15, "log_sum")
    lp = want["logprob"].nan_to_num(0.0, 0.0, 0.0).abs()
    close(torch, got["logprob"], want["logprob"], 2.0 ** -15 + 2.0 ** -21 * (lp + z), "logprob")
    close(torch, got["entropy"], want["entropy"], 2.0 ** -14 * (1 + z), "entropy")
    if k:
        assert torch.equal(got["ids"].cpu().long(), want["ids"]), "top_ids"
        close(torch, got["top"], want["top"], 2.0 ** -15 + 2.0 ** -21 * (want["top"].nan_to_num(0.0, 0.0, 0.0).abs() + z[:, None]), "top")
    return got, want


# vocabularies around the vector width, the block sizes and the cluster split; rows for one, several and many per SM
SHAPES = [(1, 1), (1, 2), (3, 7), (2, 8), (5, 9), (1, 31), (4, 33), (7, 100), (300, 513), (33, 1000), (9, 4096), (3, 4099),
          (2, 8200), (160, 5001), (17, 20011), (70, 20011), (1, 50257), (40, 50257), (2, 131072), (1, 262144)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_forward(cuda, rows, vocab, dtype):
    torch = cuda
    k = min(vocab, [0, 1, 5, 20, 32][(rows + vocab) % 5])
    logits, _, g = make(torch, rows, vocab, dtype, rows * 7 + vocab)
    targets = torch.randint(0, vocab, (rows,), generator=g).cuda()
    check_forward(torch, logits, targets, [1.0, 0.7, 1.9][rows % 3], k)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lead", [0, 1, 3, 7])
@pytest.mark.parametrize("ld_extra", [0, 1, 5, 8])
def test_forward_strided(cuda, dtype, lead, ld_extra):
    torch = cuda
    for vocab in (5, 300, 9001):
        logits, buf, g = make(torch, 6, vocab, dtype, lead * 31 + ld_extra, ld=vocab + ld_extra, lead=lead)
        targets = torch.randint(0, vocab, (6,), generator=g).cuda().int()
        check_forward(torch, logits, targets, 1.0, 5)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(1, 6000), (2, 40000), (50, 900), (200, 6001)])
def test_masked_and_special_rows(cuda, dtype, rows, vocab):
    torch = cuda
    logits, _, g = make(torch, rows, vocab, dtype, 5, mask=0.9)
    targets = torch.randint(0, vocab, (rows,), generator=g)
    low = torch.finfo(logits.dtype).min
    special = ["empty", "lowest", "one", "lowest_but_one", "constant", "zeros", "few", "huge", "nan", "inf", "nan_masked", "none", "outside"]
    for i in range(rows):
        name = special[i % len(special)] if rows > 2 else special[(i + rows) % 4]
        row = logits[i]
        if name == "empty":
            row.fill_(-math.inf)
        elif name == "lowest":
            row.fill_(low)
        elif name == "one":
            row.fill_(-math.inf)
            row[vocab // 2] = 3.0
        elif name == "lowest_but_one":
            row.fill_(low)
            row[vocab - 1] = -2.0
        elif name == "constant":
            row.fill_(1.25)
        elif name == "zeros":  # equal values of both signs: ties go to the lowest index
            row.fill_(0.0)
            row[::2] = -0.0
        elif name == "few":  # fewer unmasked entries than alternatives
            row.fill_(-math.inf)
            row[[1, vocab - 2, vocab // 3]] = torch.tensor([1.0, 2.0, 1.0], dtype=row.dtype, device="cuda")
        elif name == "huge":
            row.copy_(torch.randn(vocab, generator=g).to(row.dtype) * 1e4)
        elif name == "nan":
            row[vocab // 5] = math.nan
        elif name == "inf":
            row[vocab // 7] = math.inf
        elif name == "nan_masked":
            row.fill_(-math.inf)
            row[vocab - 1] = math.nan
        elif name == "none":
            targets[i] = -1 - i
        else:
            targets[i] = vocab + i
    check_forward(torch, logits, targets.cuda(), 0.9, 20)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [600, 5000, 70000])
@pytest.mark.parametrize("order", ["up", "down", "coarse", "block"])
def test_alternatives_of_ordered_rows(cuda, vocab, order, dtype):
    """Rows where the largest elements sit together, arrive last, or tie in great numbers."""
    torch = cuda
    i = torch.arange(vocab)
    x = {"up": i / 64.0, "down": -i / 64.0, "coarse": (i * 7919 % 13).float(), "block": torch.where(i // 8 == vocab // 16, 5.0 + i % 8, 0.0)}[order]
    for rows in (1, 5, 200):
        logits = x.to(getattr(torch, DT[dtype])).cuda().repeat(rows, 1)
        check_forward(torch, logits, torch.zeros(rows, dtype=torch.int64, device="cuda"), 1.0, 32)


def test_outputs_are_optional(cuda):
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    logits, _, _ = make(torch, 5, 3001, "bf16", 1)
    want = reference(torch, logits, torch.zeros(5, dtype=torch.int64), 1.0, 3)
    ent = torch.empty(5, device="cuda")
    tc.token_logprobs(logits, None, entropy=ent)
    close(torch, ent, want["entropy"], 2.0 ** -12, "entropy")
    ids, top = torch.empty(5, 3, dtype=torch.int32, device="cuda"), torch.empty(5, 3, device="cuda")
    tc.token_logprobs(logits, None, top_ids=ids, top_logprobs=top)
    assert torch.equal(ids.cpu().long(), want["ids"])
    tc.token_logprobs(logits[:0], None, entropy=ent[:0])


def gradients(torch, logits, targets, dlogprob, dentropy, temperature, inplace=False, dst=None):
    from bee_b200 import tensor_cuda as tc
    st = forward(torch, logits, targets, temperature, 0)
    d = logits if inplace else (torch.full_like(logits, 7.0) if dst is None else dst)
    tc.token_logprobs_backward(logits, targets, st["row_max"], st["log_sum"], st["entropy"], dlogprob, dentropy, d,
                               temperature=temperature)
    torch.cuda.synchronize()
    return d


def check_gradients(torch, logits, targets, gl, gh, temperature, **how):
    want = reference(torch, logits, targets, temperature, 1)
    p, lp = want["p"], want["lp"].clamp(min=-1e30)
    t = targets.cpu().long()
    empty = want["row_max"] == -math.inf
    p[empty] = 0.0
    l = torch.zeros(len(t)) if gl is None else torch.where(t < 0, 0.0, gl.cpu())
    h = torch.zeros(len(t)) if gh is None else gh.cpu()
    d = -p * (l[:, None] + h[:, None] * (lp + want["entropy"][:, None]))
    size = p * (l.abs()[:, None] + h.abs()[:, None] * (lp.abs() + want["entropy"][:, None])) / temperature
    d.scatter_add_(1, t.clamp(min=0)[:, None], torch.where(empty, 0.0, l.double())[:, None])
    d /= temperature
    got = gradients(torch, logits, targets, gl, gh, temperature, **how)
    half = torch.finfo(logits.dtype).eps / 2
    tol = 2.0 ** -13 * size + half * d.abs() + (2.0 ** -25 if logits.dtype == torch.float16 else 1e-38) + 2.0 ** -22 * l.abs()[:, None] / temperature
    close(torch, got, d, tol, "dlogits")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (9, 33), (300, 513), (5, 8192), (40, 20011), (2, 131072)])
def test_backward(cuda, rows, vocab, dtype):
    torch = cuda
    logits, _, g = make(torch, rows, vocab, dtype, rows + vocab, mask=0.2 if vocab > 30 else 0.0)
    targets = torch.randint(-1, vocab, (rows,), generator=g).cuda()
    if rows > 2:
        logits[1] = -math.inf
    gl, gh = torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda()
    for a, b in ((gl, gh), (gl, None), (None, gh)):
        check_gradients(torch, logits, targets, a, b, 0.8)
    check_gradients(torch, logits.clone(), targets, gl, gh, 1.0)
    inplace = logits.clone()
    sep = gradients(torch, logits, targets, gl, gh, 0.8)
    gradients(torch, inplace, targets, gl, gh, 0.8, inplace=True)
    assert torch.equal(inplace, sep)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lead,extra,dlead,dextra", [(0, 0, 1, 0), (3, 5, 3, 5), (3, 5, 3, 13), (1, 0, 0, 3), (0, 8, 0, 0)])
def test_backward_strided(cuda, dtype, lead, extra, dlead, dextra):
    torch = cuda
    for vocab in (9, 1000, 5003):
        logits, _, g = make(torch, 6, vocab, dtype, 3, ld=vocab + extra, lead=lead)
        dst, buf, _ = make(torch, 6, vocab, dtype, 4, ld=vocab + dextra, lead=dlead)
        before = buf.clone()
        targets = torch.randint(0, vocab, (6,), generator=g).cuda()
        gl, gh = torch.randn(6, generator=g).cuda(), torch.randn(6, generator=g).cuda()
        check_gradients(torch, logits, targets, gl, gh, 1.0, dst=dst)
        inside = torch.zeros_like(buf, dtype=torch.bool)
        torch.as_strided(inside, (6, vocab), (vocab + dextra, 1), dlead).fill_(True)
        assert torch.equal(buf[~inside], before[~inside])  # nothing outside the rows is written


def test_gradient_against_differences(cuda):
    """Central differences of the kernel's own fp32 forward, step 2^-6: truncation below 2^-12 * |third
    derivative| / 6 < 2^-13, rounding 2 * 2^-15 / 2^-5 = 2^-9 of the outputs' scale."""
    torch = cuda
    logits, _, g = make(torch, 1, 40, "f32", 11, scale=1.0)
    targets, gl, gh = torch.tensor([13]).cuda(), torch.tensor([0.7]).cuda(), torch.tensor([-0.4]).cuda()
    d = gradients(torch, logits, targets, gl, gh, 0.9)

    def value(x):
        o = forward(torch, x, targets, 0.9, 0)
        return float(gl * o["logprob"] + gh * o["entropy"])

    for i in range(0, 40, 3):
        up, down = logits.clone(), logits.clone()
        up[0, i] += 2.0 ** -6
        down[0, i] -= 2.0 ** -6
        assert abs((value(up) - value(down)) * 2.0 ** 5 - float(d[0, i])) < 2.0 ** -8


def test_rows_without_gradient_are_zero_whatever_they_hold(cuda):
    torch = cuda
    logits, _, _ = make(torch, 4, 3000, "bf16", 2)
    logits[1] = math.nan
    logits[2, 5] = math.inf
    targets = torch.tensor([3, -1, 7, 9]).cuda()
    gl = torch.tensor([1.0, 5.0, 0.0, 1.0]).cuda()
    d = gradients(torch, logits, targets, gl, None, 1.0)
    assert (d[1] == 0).all() and (d[2] == 0).all() and torch.isfinite(d).all() and (d[0] != 0).any()


def test_streams_graphs_and_repeats(cuda):
    """The same call on a side stream, captured and replayed on new inputs, and twice: the same bits."""
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    for rows, vocab in ((2, 60000), (300, 4000)):
        logits, _, g = make(torch, rows, vocab, "bf16", 8)
        other, _, _ = make(torch, rows, vocab, "bf16", 9)
        targets = torch.randint(0, vocab, (rows,), generator=g).cuda()
        want = {s: forward(torch, x, targets, 1.0, 8) for s, x in (("a", logits), ("b", other))}
        x = logits.clone()
        out = {n: torch.empty_like(v) for n, v in want["a"].items()}

        def call():
            tc.token_logprobs(x, targets, out["logprob"], out["entropy"], out["row_max"], out["log_sum"], top_ids=out["ids"],
                              top_logprobs=out["top"])

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(out[n], want["a"][n]) for n in out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        for s, src in (("b", other), ("a", logits), ("b", other)):
            x.copy_(src)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(out[n], want[s][n]) for n in out)
