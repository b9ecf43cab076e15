"""The fused block operators at the ends of what they take: offsets past 32 bits,
two calls at once on two streams, and inputs made on another stream."""
import math

import pytest

pytestmark = pytest.mark.gpu


def test_logit_rows_past_32_bits(cuda):
    """Rows 2^30 + 24 elements apart: the third begins past 2^31 elements.  Against the rows side by side, aligned alike
    (a row's sums run over its 16-byte blocks, so another alignment adds in another order)."""
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    ld, vocab = 2 ** 30 + 24, 3008
    buf = torch.empty(2 * ld + vocab, dtype=torch.bfloat16, device="cuda")
    far = torch.as_strided(buf, (3, vocab), (ld, 1))
    g = torch.Generator().manual_seed(0)
    far.copy_(torch.randn(3, vocab, generator=g).bfloat16())
    near = far.contiguous()
    targets = torch.tensor([1, 2, 3], device="cuda")
    gl = torch.ones(3, device="cuda")
    got = []
    for x in (far, near):
        out = [torch.empty(3, device="cuda") for _ in range(4)]
        ids, top = torch.empty(3, 5, dtype=torch.int32, device="cuda"), torch.empty(3, 5, device="cuda")
        tc.token_logprobs(x, targets, *out, top_ids=ids, top_logprobs=top)
        tc.token_logprobs_backward(x, targets, out[2], out[3], out[1], gl, gl, x)
        got.append((*out, ids, top, x.clone()))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_norm_of_more_than_2_31_elements(cuda):
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    cols = 8192
    rows = 2 ** 31 // cols + 40
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_()
    h = torch.empty_like(x).normal_()
    w = torch.rand(cols, device="cuda").bfloat16() + 0.5
    xo, y = torch.empty_like(x), torch.empty_like(x)
    tc.norm_gate_residual(h, x, xo, y, w_post=w, gate=w, w_pre=w)
    dh, dx, dw, dg, dp = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w), torch.empty_like(w), torch.empty_like(w)
    tc.norm_gate_residual_backward(h, x, x, h, dh, dx, w_post=w, gate=w, w_pre=w, dw_post=dw, dgate=dg, dw_pre=dp)
    last = slice(rows - 50, rows)
    s = {k: v[last].contiguous() for k, v in (("h", h), ("x", x))}
    sxo, sy, sdh, sdx = (torch.empty_like(s["x"]) for _ in range(4))
    tc.norm_gate_residual(s["h"], s["x"], sxo, sy, w_post=w, gate=w, w_pre=w)
    tc.norm_gate_residual_backward(s["h"], s["x"], s["x"], s["h"], sdh, sdx, w_post=w, gate=w, w_pre=w, dw_post=dw.clone(),
                                   dgate=dg.clone(), dw_pre=dp.clone())
    for a, b in ((xo, sxo), (y, sy), (dh, sdh), (dx, sdx)):
        assert torch.equal(a[last], b)


def test_gated_rows_past_32_bits(cuda):
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    ld, d, f = 2 ** 30 + 8, 136, 72
    buf = torch.empty(2 * ld + d, dtype=torch.bfloat16, device="cuda")
    far = torch.as_strided(buf, (3, d), (ld, 1))
    far.copy_(torch.randn(3, d).bfloat16())
    near = far.contiguous()
    w = [(torch.randn(f, d) * 0.1).bfloat16().cuda() for _ in range(2)]
    out = [torch.empty(3, f, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for x, o in zip((far, near), out):
        tc.gated_linear(x, *w, o, trans=True)
    assert torch.equal(*out)


def test_two_streams_at_once(cuda):
    """Every operator on two streams side by side, several times: the bits of the calls alone (no workspace is shared)."""
    torch = cuda
    from bee_b200 import tensor_cuda as tc

    def make(seed):
        g = torch.Generator().manual_seed(seed)

        def t(*shape, scale=1.0):
            return (torch.randn(*shape, generator=g) * scale).bfloat16().cuda()

        return {"h": t(900, 1024), "x": t(900, 1024), "w": t(1024), "gate": t(9, 1024), "wg": t(2048, 1024, scale=0.03),
                "wu": t(2048, 1024, scale=0.03), "few": t(5, 1024), "logits": t(30, 50000, scale=3.0),
                "targets": torch.randint(0, 50000, (30,), generator=g).cuda()}

    def call(s):
        e = torch.empty_like
        o = {"xo": e(s["x"]), "y": e(s["x"]), "dh": e(s["x"]), "dx": e(s["x"]), "dw": e(s["w"]), "dg": e(s["gate"]), "dp": e(s["w"])}
        more = {"w_post": s["w"], "gate": s["gate"], "w_pre": s["w"]}
        tc.norm_gate_residual(s["h"], s["x"], o["xo"], o["y"], **more)
        tc.norm_gate_residual_backward(s["h"], s["x"], s["x"], s["h"], o["dh"], o["dx"], dw_post=o["dw"], dgate=o["dg"], dw_pre=o["dp"], **more)
        n = s["x"].shape[0]
        o |= {k: s["x"].new_empty(n, 2048) for k in "agu"}
        tc.gated_linear(s["x"], s["wg"], s["wu"], o["a"], trans=True, g=o["g"], u=o["u"])
        o |= {"gx": e(s["x"]), "dwg": e(s["wg"]), "dwu": e(s["wu"]), "few": s["x"].new_empty(5, 2048)}
        tc.gated_linear_backward(s["x"], s["wg"], s["wu"], o["g"], o["u"], o["a"], o["gx"], o["dwg"], o["dwu"], trans=True)
        tc.gated_linear(s["few"], s["wg"], s["wu"], o["few"], trans=True)
        o |= {k: torch.empty(30, device="cuda") for k in ("lp", "ent", "m", "ls")}
        o |= {"ids": torch.empty(30, 7, dtype=torch.int32, device="cuda"), "top": torch.empty(30, 7, device="cuda"), "dl": e(s["logits"])}
        tc.token_logprobs(s["logits"], s["targets"], o["lp"], o["ent"], o["m"], o["ls"], top_ids=o["ids"], top_logprobs=o["top"])
        tc.token_logprobs_backward(s["logits"], s["targets"], o["m"], o["ls"], o["ent"], o["lp"], o["ent"], o["dl"])
        return o

    sets = [make(1), make(2)]
    want = [call(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(call(s))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for k in b:
                assert torch.equal(a[k], b[k]), k


def test_a_stream_argument(cuda):
    """stream=: the call runs there, after the work that is already on it."""
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    st = torch.cuda.Stream()
    x = torch.zeros(64, 4096, device="cuda")
    xo = torch.empty_like(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        for _ in range(50):
            x.add_(1.0)
    tc.norm_gate_residual(x, x, xo, stream=st, sync=True)
    assert (xo == 100).all()


def test_wrapper_refusals(cuda):
    """What only the Python layer can see: devices, dtypes, shapes and strides."""
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    x, w = torch.zeros(8, 64, device="cuda"), torch.ones(64, device="cuda")
    logits, t, f = torch.zeros(4, 32, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(4, device="cuda")
    b, wb, ob = torch.zeros(4, 64).bfloat16().cuda(), torch.zeros(32, 64).bfloat16().cuda(), torch.zeros(4, 32).bfloat16().cuda()
    calls = [
        lambda: tc.norm_gate_residual(x.cpu(), x, x),
        lambda: tc.norm_gate_residual(x.half(), x, x),
        lambda: tc.norm_gate_residual(x[:, ::2], x[:, ::2], x[:, ::2]),
        lambda: tc.norm_gate_residual(x, x, x, w_pre=w),
        lambda: tc.norm_gate_residual(x, x, x, w_post=w[:32]),
        lambda: tc.norm_gate_residual(x, x, x, gate=torch.ones(3, 64, device="cuda")),
        lambda: tc.norm_gate_residual_backward(x, x, x, None, x, x, w_post=w),
        lambda: tc.token_logprobs(logits, t.float(), f),
        lambda: tc.token_logprobs(logits, t[:3], f),
        lambda: tc.token_logprobs(logits, None, f),
        lambda: tc.token_logprobs(logits, t, f.double()),
        lambda: tc.token_logprobs(logits.t(), t, f),
        lambda: tc.token_logprobs(logits[:1].expand(4, 32), t, f),
        lambda: tc.token_logprobs(logits, t, f, top_ids=torch.zeros(4, 2, dtype=torch.int32, device="cuda")),
        lambda: tc.token_logprobs(logits, t, f, temperature=math.nan),
        lambda: tc.token_logprobs_backward(logits, t, f, f, f, f, f, logits.half()),
        lambda: tc.gated_linear(b, wb, wb, ob, trans=False),
        lambda: tc.gated_linear(b, wb, wb.float(), ob, trans=True),
        lambda: tc.gated_linear(b, wb, wb, ob, trans=True, act="relu"),
        lambda: tc.gated_linear(b, wb, wb, ob, trans=True, g=ob),
        lambda: tc.gated_linear(b.float(), wb.float(), wb.float(), ob.float(), trans=True),
        lambda: tc.gated_linear_backward(b, wb, wb, ob, ob, ob, trans=True),
        lambda: tc.gated_linear_backward(b, wb, wb, ob, ob, ob, None, wb, wb[:, :32], trans=True),
    ]
    for i, c in enumerate(calls):
        with pytest.raises(tc.BeeError):
            c()
            pytest.fail(f"call {i} was taken")
