"""gated_linear and its gradient against the definition in 64 bits.

Tolerances, from the arithmetic.  The tensor cores add K / 16 partial products
to an fp32 accumulator, each step off by at most 2^-22 of the running sum's size
(their sums may truncate): for K <= 4096 a product is off by at most 2^-14 of
|x| |W| ("size").  The activation's derivative is at most 1.13 and the functions
themselves are good to 2^-20, so out = act(g) u is off by at most
2^-14 (1.13 size_g |u| + |act(g)| size_u) + 2^-20 |out| and half a step.  In the backward dg and du are
rounded to the type (half a step each of their own size) before the products,
which adds half a step of |dg| |W| to the 2^-14 of it."""
import math

import pytest

pytestmark = pytest.mark.gpu

DT = {"bf16": "bfloat16", "f16": "float16"}
ACTS = ["silu", "gelu", "gelu_tanh"]


def strided(torch, rows, cols, dt, gen, scale, extra=0, lead=0):
    buf = torch.full((lead + rows * (cols + extra) + 8,), 3.0, dtype=dt, device="cuda")
    view = torch.as_strided(buf, (rows, cols), (cols + extra, 1), lead)
    view.copy_((torch.randn(rows, cols, generator=gen) * scale).to(dt))
    return view


def make(torch, m, d, f, dtype, trans, seed, extra=0, lead=0):
    gen = torch.Generator().manual_seed(seed)
    dt = getattr(torch, DT[dtype])
    x = strided(torch, m, d, dt, gen, 1.0, extra, lead)
    shape = (f, d) if trans else (d, f)
    wg, wu = (strided(torch, *shape, dt, gen, 1.5 * d ** -0.5, extra, lead) for _ in range(2))
    return x, wg, wu, (torch.randn(m, f, generator=gen) * 0.3).to(dt).cuda()


def act_and_grad(g, kind):
    import torch
    if kind == "silu":
        p = torch.sigmoid(g)
        return g * p, p * (1 + g * (1 - p))
    if kind == "gelu":
        p = 0.5 * torch.erfc(-g / math.sqrt(2))  # 1 + erf cancels below g = -8, also in 64 bits
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    c, a = math.sqrt(2 / math.pi), 0.044715
    p = torch.sigmoid(2 * c * (g + a * g ** 3))  # (1 + tanh z) / 2, which cancels below z = -18, also in 64 bits
    return g * p, p + g * p * (1 - p) * 2 * c * (1 + 3 * a * g * g)


def within(torch, got, ref, tol, what):
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 1e-37
    tol = tol + torch.finfo(got.dtype).eps / 2 * ref.abs() + tiny
    g = got.double()
    bad = ~((g - ref).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {((g - ref).abs() / tol).max():.2f} times the bound"


def forward(torch, x, wg, wu, act, trans, save=True):
    from bee_b200 import tensor_cuda as tc
    m, f = x.shape[0], wg.shape[0] if trans else wg.shape[1]
    out, g, u = (torch.full((m, f), 7.0, dtype=x.dtype, device="cuda") for _ in range(3))
    tc.gated_linear(x, wg, wu, out, act=act, trans=trans, g=g if save else None, u=u if save else None)
    return out, g, u


def check_forward(torch, x, wg, wu, act, trans):
    got, g, u = forward(torch, x, wg, wu, act, trans)
    X, G, U = x.double(), wg.double(), wu.double()
    if trans:
        G, U = G.t(), U.t()
    rg, ru = X @ G, X @ U
    sg, su = 2.0 ** -14 * (X.abs() @ G.abs()), 2.0 ** -14 * (X.abs() @ U.abs())
    a, _ = act_and_grad(rg, act)
    within(torch, g, rg, sg, "g")
    within(torch, u, ru, su, "u")
    within(torch, got, a * ru, 1.13 * sg * ru.abs() + (a.abs() + 1.13 * sg) * su + 2.0 ** -20 * (a * ru).abs(), "out")
    only, _, _ = forward(torch, x, wg, wu, act, trans, save=False)
    assert torch.equal(only, got)


def check_backward(torch, x, wg, wu, g, u, dout, act, trans, extra=0):
    from bee_b200 import tensor_cuda as tc
    dx = torch.full((x.shape[0], x.shape[1]), 7.0, dtype=x.dtype, device="cuda")
    r, c = wg.shape
    bufs = [torch.full((r * (c + extra) + 8,), 5.0, dtype=x.dtype, device="cuda") for _ in range(2)]
    dwg, dwu = (torch.as_strided(b, (r, c), (c + extra, 1), 0) for b in bufs)
    tc.gated_linear_backward(x, wg, wu, g, u, dout, dx, dwg, dwu, act=act, trans=trans)
    X, G, U = x.double(), wg.double(), wu.double()
    if trans:
        G, U = G.t(), U.t()
    a, da = act_and_grad(g.double(), act)
    dg, du = dout.double() * u.double() * da, dout.double() * a
    e = 2.0 ** -14 + torch.finfo(x.dtype).eps / 2
    sg, su = e * dg.abs(), e * du.abs()
    if x.dtype == torch.float16:
        sg, su = sg + 2.0 ** -25, su + 2.0 ** -25
    within(torch, dx, dg @ G.t() + du @ U.t(), sg @ G.t().abs() + su @ U.t().abs(), "dx")
    for got, d, s, n in ((dwg, dg, sg, "dwg"), (dwu, du, su, "dwu")):
        ref, tol = X.t() @ d, X.t().abs() @ s
        within(torch, got, ref.t() if trans else ref, tol.t() if trans else tol, n)
    if extra:
        for b in bufs:
            outside = torch.ones_like(b, dtype=torch.bool)
            torch.as_strided(outside, (r, c), (c + extra, 1), 0).fill_(False)
            assert (b[outside] == 5.0).all()
    only = torch.empty_like(dx)
    tc.gated_linear_backward(x, wg, wu, g, u, dout, only, act=act, trans=trans)
    assert torch.equal(only, dx)
    og, ou = torch.empty(r, c, dtype=x.dtype, device="cuda"), torch.empty(r, c, dtype=x.dtype, device="cuda")
    tc.gated_linear_backward(x, wg, wu, g, u, dout, None, og, ou, act=act, trans=trans)
    assert torch.equal(og, dwg) and torch.equal(ou, dwu)


# rows around each padding of the few-rows kernel, its border, and the 256-row tiles; columns below, at and past the
# 128-column tile; contractions of less than one block, odd counts of blocks, and cut by clusters
# or over the last round of pairs (after whole rounds and without any)
SHAPES = [(1, 8, 8), (1, 64, 128), (2, 200, 136), (16, 512, 264), (17, 1000, 128), (32, 4096, 256), (33, 72, 520), (64, 2048, 1032),
          (65, 640, 384), (128, 1096, 392), (129, 512, 256), (255, 128, 136), (256, 384, 128), (257, 1000, 776), (520, 2056, 640),
          (1000, 264, 2048), (300, 4096, 520), (66, 2056, 1000), (2600, 2048, 1032), (2100, 520, 264)]


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,d,f", SHAPES)
def test_shapes(cuda, m, d, f, dtype, trans):
    torch = cuda
    act = ACTS[(m + d + f) % 3]
    x, wg, wu, dout = make(torch, m, d, f, dtype, trans, m + d + f)
    check_forward(torch, x, wg, wu, act, trans)
    _, g, u = forward(torch, x, wg, wu, act, trans)
    check_backward(torch, x, wg, wu, g, u, dout, act, trans)


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("act", ACTS)
def test_activations(cuda, act, trans):
    torch = cuda
    for m in (5, 300):
        x, wg, wu, dout = make(torch, m, 256, 200, "bf16", trans, 3)
        check_forward(torch, x, wg, wu, act, trans)
        _, g, u = forward(torch, x, wg, wu, act, trans)
        g = (g.float() * 20).to(g.dtype)  # far into both tails
        check_backward(torch, x, wg, wu, g, u, dout, act, trans)


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,d,f", [(1, 1, 1), (3, 7, 5), (9, 333, 129), (40, 65, 1001), (130, 131, 67), (300, 515, 261)])
def test_odd_sizes(cuda, m, d, f, dtype, trans):
    torch = cuda
    x, wg, wu, dout = make(torch, m, d, f, dtype, trans, 1)
    check_forward(torch, x, wg, wu, "silu", trans)
    _, g, u = forward(torch, x, wg, wu, "silu", trans)
    check_backward(torch, x, wg, wu, g, u, dout, "silu", trans)


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("extra,lead", [(8, 0), (64, 8), (3, 0), (0, 1), (5, 3)])
def test_strided(cuda, extra, lead, trans):
    torch = cuda
    for m in (4, 200):
        x, wg, wu, dout = make(torch, m, 192, 264, "bf16", trans, 2, extra, lead)
        check_forward(torch, x, wg, wu, "gelu", trans)
        _, g, u = forward(torch, x, wg, wu, "gelu", trans)
        check_backward(torch, x, wg, wu, g, u, dout, "gelu", trans, extra)


@pytest.mark.parametrize("trans", [False, True])
def test_slices_of_one_fused_matrix(cuda, trans):
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    m, d, f = 70, 128, 96
    gen = torch.Generator().manual_seed(0)
    w = (torch.randn(*((2 * f, d) if trans else (d, 2 * f)), generator=gen) * 0.1).bfloat16().cuda()
    x = torch.randn(m, d, generator=gen).bfloat16().cuda()
    halves = (w[:f], w[f:]) if trans else (w[:, :f], w[:, f:])
    check_forward(torch, x, *halves, "silu", trans)
    _, g, u = forward(torch, x, *halves, "silu", trans)
    dout = torch.randn(m, f, generator=gen).bfloat16().cuda()
    want = [torch.empty(halves[0].shape, dtype=x.dtype, device="cuda") for _ in range(2)]
    tc.gated_linear_backward(x, *halves, g, u, dout, None, *want, act="silu", trans=trans)
    dw = torch.empty_like(w)
    tc.gated_linear_backward(x, *halves, g, u, dout, None, *((dw[:f], dw[f:]) if trans else (dw[:, :f], dw[:, f:])), act="silu", trans=trans)
    assert torch.equal(dw, torch.cat(want, 0 if trans else 1))


def test_no_rows(cuda):
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    x, w = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(64, 32, dtype=torch.bfloat16, device="cuda")
    e = torch.empty(0, 32, dtype=torch.bfloat16, device="cuda")
    tc.gated_linear(x, w, w, e)
    dwg, dwu = torch.ones_like(w), torch.ones_like(w)
    tc.gated_linear_backward(x, w, w, e, e, e, x.clone(), dwg, dwu)
    assert (dwg == 0).all() and (dwu == 0).all()


def test_extreme_gates(cuda):
    """Gates at the ends of the type's range: no overflow of an inner power reaches the result."""
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    big = torch.tensor([[1e30, -1e30, 3e38, -3e38, 40.0, -40.0, 0.0, -0.0]]).bfloat16().cuda()
    one = torch.ones_like(big)
    w = torch.eye(8).bfloat16().cuda()
    for act in ACTS:
        dwg, dwu = torch.empty_like(w), torch.empty_like(w)
        tc.gated_linear_backward(one, w, w, big, one, one, None, dwg, dwu, act=act)
        a, da = act_and_grad(big.double().clamp(-60, 60), act)
        assert torch.equal(dwg.float().round(), da.float().expand(8, 8).round()), act
        out = torch.empty(1, 8, dtype=torch.bfloat16, device="cuda")
        tc.gated_linear(one, torch.diag(big[0]), w, out, act=act)
        want = torch.where(big > 1, big, torch.zeros_like(big))
        assert ((out.double() - want.double()).abs() <= 1e-12).all(), (act, out)  # act(-40) is below 1e-15


def test_gradient_against_differences(cuda):
    """Central differences of the 64-bit definition at the kernel's inputs: step 2^-10, truncation below 2^-20."""
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    x, wg, wu, dout = make(torch, 3, 16, 8, "bf16", False, 4)
    for act in ACTS:
        _, g, u = forward(torch, x, wg, wu, act, False)
        dx, dwg, dwu = torch.empty_like(x), torch.empty(16, 8, dtype=x.dtype, device="cuda"), torch.empty(16, 8, dtype=x.dtype, device="cuda")
        tc.gated_linear_backward(x, wg, wu, g, u, dout, dx, dwg, dwu, act=act)
        args = [t.double().clone() for t in (x, wg, wu)]

        def value():
            a, _ = act_and_grad(args[0] @ args[1], act)
            return float((a * (args[0] @ args[2]) * dout.double()).sum())

        for t, d in zip(args, (dx, dwg, dwu)):
            for i in range(0, t.numel(), 7):
                flat = t.view(-1)
                keep = float(flat[i])
                flat[i] = keep + 2.0 ** -10
                up = value()
                flat[i] = keep - 2.0 ** -10
                down = value()
                flat[i] = keep
                # g, u, dg, du and the result each rounded to 8 bits: a few 2^-8 of sums of up to 8 terms of size 1
                assert abs((up - down) * 2.0 ** 9 - float(d.reshape(-1)[i])) < 8 * 4 * 2.0 ** -9, act


@pytest.mark.parametrize("m", [8, 300])
def test_streams_graphs_and_repeats(cuda, m):
    """On a side stream, and captured twice with the two graphs replayed in turn: the same bits every time."""
    torch = cuda
    from bee_b200 import _capi, tensor_cuda as tc
    sets = [make(torch, m, 1000, 777, "bf16", True, s) for s in (1, 2)]
    want, graphs = [], []

    def call(s, o):
        x, wg, wu, dout = s
        tc.gated_linear(x, wg, wu, o[0], trans=True, g=o[1], u=o[2])
        tc.gated_linear_backward(x, wg, wu, o[1], o[2], dout, o[3], o[4], o[5], trans=True)

    def outputs(s):
        x, wg, wu, dout = s
        return [torch.zeros_like(dout) for _ in range(3)] + [torch.zeros_like(x), torch.zeros_like(wg), torch.zeros_like(wu)]

    for s in sets:
        want.append(outputs(s))
        call(s, want[-1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = outputs(sets[0])
        call(sets[0], o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(o, want[0]))
    for s in sets:
        o, g = outputs(s), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(s, o)
        graphs.append((g, o))
    for _ in range(3):
        for g, o in graphs:
            for t in o:
                t.zero_()
            g.replay()
    torch.cuda.synchronize()
    for (g, o), w in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))
    import ctypes
    code = ctypes.c_int(-1)
    _capi.call("bee_b200_device_status", ctypes.byref(code))
    assert code.value == 0
