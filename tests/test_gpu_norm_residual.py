"""norm_gate_residual and its gradient against the definition in 64 bits.

Tolerances, from the arithmetic.  Every row statistic is an fp32 sum of at most
8 (a thread's pairs) + 1 + 5 + 32 (lanes and warps) terms per chain: an error
below 2^6 * 2^-24 = 2^-18 of the sum of the terms' sizes; the reciprocal root
adds 2^-22.  An output is a sum of at most three such products of at most six
factors, each rounded: below 2^-16 of the sum of its terms' sizes ("size"
below), plus half a step of the type when it is rounded.  Column sums add the
rows of a CTA and then the CTAs' partial sums, fewer than 2^8 terms per chain in
these sizes: another 2^-16 of the sum of the terms' sizes."""
import pytest

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


def make(torch, rows, cols, dtype, seed, gate="row", post=True, pre=True, lead=0):
    g = torch.Generator().manual_seed(seed)
    dt = getattr(torch, DT[dtype])

    def t(*shape, scale=1.0, shift=0.0):
        v = torch.randn(*shape, generator=g) * scale + shift
        buf = torch.zeros(v.numel() + lead + 8, dtype=dt, device="cuda")
        out = buf[lead:lead + v.numel()].view(*shape)
        out.copy_(v.to(dt))
        return out

    s = {"h": t(rows, cols, scale=0.8), "x": t(rows, cols, scale=1.5), "dx_out": t(rows, cols, scale=0.2),
         "w_post": t(cols, scale=0.2, shift=1.0) if post else None, "w_pre": t(cols, scale=0.2, shift=1.0) if pre else None,
         "dy": t(rows, cols, scale=0.3) if pre else None, "gate": None}
    if gate == "row":
        s["gate"] = t(cols, scale=0.4, shift=0.6)
    elif gate:
        s["gate"] = t(gate, cols, scale=0.4, shift=0.6)
    return s


def reference(s, alpha, beta, eps):
    """Outputs, gradients and the sizes of their terms, in float64."""
    import torch
    d = {k: v.double().cpu() if v is not None else None for k, v in s.items()}
    h, x = d["h"], d["x"]
    rows, cols = x.shape
    gate = d["gate"]
    groups = 1 if gate is None or gate.dim() == 1 else gate.shape[0]
    G = torch.ones(1, cols, dtype=torch.float64) if gate is None else gate.view(groups, cols).repeat_interleave(rows // groups, 0)
    one = torch.ones(cols, dtype=torch.float64)
    wp = one if d["w_post"] is None else d["w_post"]
    rh = torch.ones(rows, 1, dtype=torch.float64) if d["w_post"] is None else 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    hh = h * rh
    n = hh * wp
    xo = alpha * x + beta * G * n
    size_xo = (alpha * x).abs() + (beta * G * n).abs()
    out = {"x_out": (xo, size_xo)}
    dx_out = d["dx_out"] if d["dx_out"] is not None else torch.zeros_like(x)
    D, size_D = dx_out.clone(), dx_out.abs()
    if d["w_pre"] is not None:
        rx = 1 / torch.sqrt((xo * xo).mean(-1, keepdim=True) + eps)
        xh = xo * rx
        # x' enters through its unrounded sum: an error of 2^-16 of its terms
        size_xh = size_xo * rx
        out["y"] = (xh * d["w_pre"], size_xh * d["w_pre"].abs())
        t = d["dy"] * d["w_pre"]
        D = D + rx * (t - xh * (t * xh).mean(-1, keepdim=True))
        size_D = size_D + rx * (t.abs() + size_xh * 2 * (t * size_xh).abs().mean(-1, keepdim=True))
        out["dw_pre"] = ((d["dy"] * xh).sum(0), (d["dy"].abs() * size_xh).sum(0))
    out["dx"] = (alpha * D, abs(alpha) * size_D)
    dn, size_dn = beta * D, abs(beta) * size_D
    if gate is not None:
        dg, sg = dn * n, size_dn * n.abs()
        out["dgate"] = tuple(v.view(groups, rows // groups, cols).sum(1).view(gate.shape) for v in (dg, sg))
        dn, size_dn = dn * G, size_dn * G.abs()
    if d["w_post"] is not None:
        out["dw_post"] = ((dn * hh).sum(0), (size_dn * hh.abs()).sum(0))
        t, st = dn * wp, size_dn * wp.abs()
        dn = rh * (t - hh * (t * hh).mean(-1, keepdim=True))
        size_dn = rh * (st + hh.abs() * 2 * (st * hh.abs()).mean(-1, keepdim=True))
    out["dh"] = (dn, size_dn)
    return out


def check(torch, got, want, what):
    ref, size = want
    half = torch.finfo(got.dtype).eps / 2
    g = got.double().cpu()
    tol = 2.0 ** -15 * size + half * ref.abs() + (2.0 ** -25 if got.dtype == torch.float16 else 1e-37)
    bad = ~((g - ref).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {((g - ref).abs() / tol).max():.2f} times the bound"


def run(torch, s, alpha, beta, eps=1e-5):
    from bee_b200 import tensor_cuda as tc
    names = [k for k in ("w_post", "gate", "w_pre") if s[k] is not None]
    more = {"w_post": s["w_post"], "gate": s["gate"], "w_pre": s["w_pre"], "alpha": alpha, "beta": beta, "eps": eps}
    out = {"x_out": torch.full_like(s["x"], 7), "dh": torch.full_like(s["x"], 7), "dx": torch.full_like(s["x"], 7)}
    y = torch.full_like(s["x"], 7) if s["w_pre"] is not None else None
    tc.norm_gate_residual(s["h"], s["x"], out["x_out"], y, **more)
    for k in names:
        out["d" + k] = torch.full_like(s[k], 7)
    tc.norm_gate_residual_backward(s["h"], s["x"], s["dx_out"], s["dy"], out["dh"], out["dx"], **more,
                                   **{"d" + k: out["d" + k] for k in names})
    torch.cuda.synchronize()
    if y is not None:
        out["y"] = y
    return out


def check_all(torch, s, alpha=0.75, beta=1.25):
    got, want = run(torch, s, alpha, beta), reference(s, alpha, beta, 1e-5)
    assert sorted(got) == sorted(want)
    for k in got:
        check(torch, got[k], want[k], k)


# widths around the vector, the warp and each block size; rows below, at and above one per CTA
SHAPES = [(1, 1), (2, 3), (3, 8), (1, 64), (40, 100), (7, 512), (500, 513), (3, 1000), (9, 1024), (600, 1100), (20, 1536), (1, 2048), (310, 2056), (11, 2049),
          (150, 4096), (5, 4100), (450, 4104), (2, 2560), (9, 5120), (160, 6000), (2, 8192), (151, 8200), (3, 8193), (5, 12288)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_shapes(cuda, rows, cols, dtype):
    check_all(cuda, make(cuda, rows, cols, dtype, rows * 13 + cols))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(3, 16384), (160, 16384), (2, 16383), (149, 12289)])
def test_widest(cuda, rows, cols, dtype):
    check_all(cuda, make(cuda, rows, cols, dtype, cols, gate="row"))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("pre", [True, False])
@pytest.mark.parametrize("gate", [None, "row", 4])
def test_parts(cuda, dtype, post, pre, gate):
    for rows, cols in ((12, 520), (8, 333)):
        check_all(cuda, make(cuda, rows, cols, dtype, 3, gate=gate, post=post, pre=pre), alpha=1.0, beta=-0.5)


# groups inside one CTA's range, equal to it, cut by it, and longer than several
@pytest.mark.parametrize("rows,cols,groups", [(600, 4096, 600), (600, 4096, 300), (600, 4096, 200), (600, 4096, 8), (600, 4096, 1),
                                              (1176, 2048, 84), (900, 520, 3), (5000, 96, 10), (5000, 96, 1250), (5000, 97, 2500),
                                              (888, 8192, 4), (888, 8192, 148), (444, 16384, 3), (444, 16384, 148), (444, 16384, 222)])
def test_gate_groups(cuda, rows, cols, groups):
    check_all(cuda, make(cuda, rows, cols, "bf16", groups, gate=groups))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lead", [1, 3])
@pytest.mark.parametrize("cols", [64, 333, 4096])
def test_unaligned(cuda, dtype, lead, cols):
    check_all(cuda, make(cuda, 9, cols, dtype, 4, lead=lead))


def test_outputs_in_place(cuda):
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    for cols in (4096, 1001):
        s = make(torch, 700, cols, "bf16", 6)
        want = run(torch, s, 1.0, 1.0)
        more = {"w_post": s["w_post"], "gate": s["gate"], "w_pre": s["w_pre"], "eps": 1e-5}
        h, x = s["h"].clone(), s["x"].clone()
        tc.norm_gate_residual(h, x, x, h, **more)
        assert torch.equal(x, want["x_out"]) and torch.equal(h, want["y"])
        dxo, dy = s["dx_out"].clone(), s["dy"].clone()
        grads = {k: torch.empty_like(s[k[1:]]) for k in ("dw_post", "dgate", "dw_pre")}
        tc.norm_gate_residual_backward(s["h"], s["x"], dxo, dy, dy, dxo, **more, **grads)
        assert torch.equal(dxo, want["dx"]) and torch.equal(dy, want["dh"])
        assert all(torch.equal(v, want[k]) for k, v in grads.items())


def test_no_residual_gradient(cuda):
    torch = cuda
    s = make(torch, 33, 1024, "f32", 2)
    s["dx_out"] = None
    check_all(torch, s)


def test_no_rows(cuda):
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    x = torch.empty(0, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    g = {k: torch.full((64,), 5.0, device="cuda") for k in ("dw_post", "dgate", "dw_pre")}
    tc.norm_gate_residual(x, x, x.clone(), x.clone(), w_post=w, gate=w, w_pre=w)
    tc.norm_gate_residual_backward(x, x, x, x, x.clone(), x.clone(), w_post=w, gate=w, w_pre=w, **g)
    assert all((v == 0).all() for v in g.values())


def test_rows_do_not_meet(cuda):
    """A row with a NaN or an infinity spoils itself and the column sums, not the other rows."""
    torch = cuda
    s = make(torch, 40, 2048, "bf16", 9)
    clean = run(torch, s, 1.0, 1.0)
    s["h"][7, 3], s["x"][20, 5] = float("nan"), float("inf")
    got = run(torch, s, 1.0, 1.0)
    keep = [r for r in range(40) if r not in (7, 20)]
    for k in ("x_out", "y", "dh", "dx"):
        assert torch.equal(got[k][keep], clean[k][keep]), k
        assert torch.isnan(got[k][7]).any()


def test_gradient_against_differences(cuda):
    """Central differences of the kernel's fp32 forward with step 2^-7: truncation below 2^-14 / 6 of the third
    derivative (of order 2^2), rounding of a sum of 2 * 24 outputs of size 2 below 2^-15, divided by 2^-6."""
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    s = make(torch, 2, 12, "f32", 5)
    got = run(torch, s, 0.75, 1.25)

    def value():
        xo, y = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        tc.norm_gate_residual(s["h"], s["x"], xo, y, w_post=s["w_post"], gate=s["gate"], w_pre=s["w_pre"], alpha=0.75, beta=1.25, eps=1e-5)
        return float((xo.double() * s["dx_out"].double()).sum() + (y.double() * s["dy"].double()).sum())

    for name in ("h", "x", "w_post", "gate", "w_pre"):
        flat, grad = s[name].view(-1), got["d" + name].view(-1)
        for i in range(0, flat.numel(), 5):
            keep = float(flat[i])
            flat[i] = keep + 2.0 ** -7
            up = value()
            flat[i] = keep - 2.0 ** -7
            down = value()
            flat[i] = keep
            assert abs((up - down) * 2.0 ** 6 - float(grad[i])) < 2.0 ** -8, (name, i)


def test_streams_graphs_and_repeats(cuda):
    """On a side stream, and captured twice (the two graphs replayed in turn): the same bits every time."""
    torch = cuda
    s, o = make(torch, 700, 4096, "bf16", 1, gate=7), make(torch, 700, 4096, "bf16", 2, gate=7)
    want = {"s": run(torch, s, 1.0, 1.0), "o": run(torch, o, 1.0, 1.0)}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(torch, s, 1.0, 1.0)
    assert all(torch.equal(got[k], want["s"][k]) for k in got)
    from bee_b200 import tensor_cuda as tc
    graphs = []
    for v in (s, o):
        out = {k: torch.empty_like(v[k[1:]]) for k in ("dh", "dx", "dw_post", "dgate", "dw_pre")}
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            tc.norm_gate_residual_backward(v["h"], v["x"], v["dx_out"], v["dy"], out["dh"], out["dx"], w_post=v["w_post"], gate=v["gate"],
                                           w_pre=v["w_pre"], eps=1e-5, **{k: out[k] for k in ("dw_post", "dgate", "dw_pre")})
        graphs.append((g, out))
    for _ in range(3):
        for g, out in graphs:
            for v in out.values():
                v.zero_()
            g.replay()
    torch.cuda.synchronize()
    for (g, out), k in zip(graphs, "so"):
        assert all(torch.equal(out[n], want[k][n]) for n in out)
