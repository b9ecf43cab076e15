"""The fused transformer operators of ``bee_b200.tensor_cuda``, as cases that can be timed and compared.

Three operators, each in both directions:

* ``norm_gate_residual``: x' = alpha x + beta gate * rmsnorm(h) w_post, y = rmsnorm(x') w_pre, the step
  from one block's output to the next block's input;
* ``gated_linear``: h = act(x Wg) * (x Wu), the first half of a gated feed-forward block;
* ``token_logprobs``: log probabilities of given tokens under logits / T, with entropy and the top alternatives.

``run`` computes a case with elementary torch operations in 32 bits where ``own`` is false, and with the
framework's kernels where it is true; ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


# ---------------------------------------------------------------- cases


def _norm(name, rows, cols, dtype, backward, gate, post=True, pre=True, alpha=1.0, beta=1.0):
    """gate: "none", "row" (one gate for all rows) or "group" (one per sequence)."""
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "dtype": dtype, "backward": backward, "gate": gate,
            "post": post, "pre": pre, "alpha": alpha, "beta": beta}


def _linear(name, rows, d, f, dtype, backward, act, trans, save=False):
    """trans: weights stored [f, d] (as a torch Linear keeps them), else [d, f]; save: g and u are kept for training."""
    return {"name": name, "op": "linear", "rows": rows, "d": d, "f": f, "dtype": dtype, "backward": backward, "act": act,
            "trans": trans, "save": save}


def _logprobs(name, rows, vocab, dtype, backward, top, temperature, masked, padded):
    """masked: a grammar or a nucleus has set entries to -inf; padded: the last rows hold no token (target -1)."""
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "backward": backward, "top": top,
            "temperature": temperature, "masked": masked, "padded": padded}


def listed():
    return [
        # eight sequences decoding one token each, between attention and the feed-forward block: latency
        _norm("norm_fwd_decode", 8, 4096, "bf16", False, "none"),
        # a training batch of 16 sequences of 2048 tokens, gated residual with a scale
        _norm("norm_fwd_train", 32768, 4096, "bf16", False, "row", alpha=1.0, beta=0.5),
        # its gradient at a wider model, one gate per sequence (conditioning on the sequence's embedding)
        _norm("norm_bwd_train", 8192, 8192, "bf16", True, "group"),
        # a ragged batch in full precision with a width that is no multiple of a vector
        _norm("norm_bwd_ragged", 4099, 1111, "f32", True, "row", alpha=0.75, beta=1.25),
        # one token through a feed-forward block: the weights are read once
        _linear("linear_fwd_token", 1, 4096, 14336, "bf16", False, "silu", True),
        # a serving batch of 48 tokens
        _linear("linear_fwd_serve", 48, 4096, 11008, "f16", False, "gelu_tanh", False),
        # a training step's forward, keeping g and u
        _linear("linear_fwd_train", 8192, 4096, 14336, "bf16", False, "silu", True, save=True),
        # a training step's backward on a ragged number of tokens
        _linear("linear_bwd_train", 4001, 4096, 11008, "bf16", True, "silu", True),
        # four sequences sampling under a grammar, with 20 alternatives each: latency
        _logprobs("logprobs_fwd_decode", 4, 131072, "bf16", False, 20, 0.8, True, False),
        # scoring a prompt, odd vocabulary, logits kept in 32 bits
        _logprobs("logprobs_fwd_score", 256, 100003, "f32", False, 5, 1.0, False, False),
        # a training or policy-gradient step over 4096 tokens, the last of them padding
        _logprobs("logprobs_fwd_train", 4096, 131072, "bf16", False, 0, 1.0, False, True),
        # its gradient, with an entropy bonus
        _logprobs("logprobs_bwd_train", 4096, 131072, "bf16", True, 0, 1.0, False, True),
    ]


def _spread(rng, lo, hi, multiple=1):
    """A whole number between lo and hi, spread over its logarithm; a multiple of `multiple`."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(multiple, n // multiple * multiple)


def draw(rng):
    kind = rng.choice(["norm", "linear", "logprobs"])
    backward = rng.random() < 0.5
    if kind == "norm":
        cols = _spread(rng, 64, 12288, rng.choice([1, 8, 64, 128]))
        rows = _spread(rng, 1, max(2, min(32768, 2 ** 26 // cols)))
        gate = rng.choice(["none", "row", "group"])
        return {k: v for k, v in _norm("", rows, cols, rng.choice(["bf16", "bf16", "f16", "f32"]), backward, gate,
                                       post=rng.random() < 0.8, pre=rng.random() < 0.9,
                                       alpha=rng.choice([1.0, 0.75]), beta=rng.choice([1.0, 0.5])).items() if k != "name"}
    if kind == "linear":
        multiple = rng.choice([8, 8, 64, 128, 1])
        d, f = _spread(rng, 128, 8192, multiple), _spread(rng, 128, 16384, multiple)
        most = 2 ** 38 if not backward else 2 ** 37
        rows = _spread(rng, 1, max(2, min(8192, most // (d * f))))
        return {k: v for k, v in _linear("", rows, d, f, rng.choice(["bf16", "f16"]), backward,
                                         rng.choice(["silu", "gelu", "gelu_tanh"]), rng.random() < 0.5,
                                         save=rng.random() < 0.5 and not backward).items() if k != "name"}
    vocab = _spread(rng, 500, 262144, rng.choice([1, 8, 64, 128]))
    top = 0 if backward else rng.choice([0, 1, 5, 20, 32])
    rows = _spread(rng, 1, max(2, min(8192, (2 ** 29 if top == 0 else 2 ** 26) // vocab)))
    return {k: v for k, v in _logprobs("", rows, vocab, rng.choice(["bf16", "bf16", "f16", "f32"]), backward, top,
                                       rng.choice([1.0, 0.8, 1.5]), rng.random() < 0.3, rng.random() < 0.3).items()
            if k != "name"}


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        n, back = case["rows"] * case["cols"], case["backward"]
        tensors = (2 + 1 + int(case["pre"])) if not back else (2 + 1 + int(case["pre"]) + 2)
        vectors = (int(case["post"]) + int(case["pre"])) * case["cols"]
        if case["gate"] != "none":
            vectors += case["cols"] * (_groups(case) if case["gate"] == "group" else 1)
        return {"bytes": es * (tensors * n + vectors * (2 if back else 1)), "flops": n * (40 if back else 15)}
    if case["op"] == "linear":
        m, d, f = case["rows"], case["d"], case["f"]
        if case["backward"]:
            return {"bytes": es * (2 * m * d + 4 * d * f + 3 * m * f), "flops": 8 * m * d * f}
        return {"bytes": es * (m * d + 2 * d * f + m * f * (3 if case["save"] else 1)), "flops": 4 * m * d * f}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * es * (2 if case["backward"] else 1) + case["rows"] * (24 + 8 * case["top"]), "flops": 8 * n}


def _groups(case):
    """Number of sequences in the batch: the largest of 16, 8, ... that divides its rows."""
    return next(g for g in (16, 8, 4, 2, 1) if case["rows"] % g == 0)


# ---------------------------------------------------------------- inputs


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + shift).to(dt)

    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        s = {"case": case, "h": rand(rows, cols, scale=0.7), "x": rand(rows, cols, scale=2.0), "w_post": None, "gate": None, "w_pre": None}
        if case["post"]:
            s["w_post"] = rand(cols, scale=0.1, shift=1.0)
        if case["gate"] != "none":
            shape = (cols,) if case["gate"] == "row" else (_groups(case), cols)
            s["gate"] = rand(*shape, scale=0.3, shift=0.5)
        if case["pre"]:
            s["w_pre"] = rand(cols, scale=0.1, shift=1.0)
        if case["backward"]:
            s["dx_out"], s["dy"] = rand(rows, cols, scale=0.1), rand(rows, cols, scale=0.1) if case["pre"] else None
        return s
    if case["op"] == "linear":
        m, d, f = case["rows"], case["d"], case["f"]
        shape = (f, d) if case["trans"] else (d, f)
        s = {"case": case, "x": rand(m, d), "wg": rand(*shape, scale=d ** -0.5), "wu": rand(*shape, scale=d ** -0.5)}
        if case["backward"]:  # what the forward pass kept, and the gradient that arrives
            s["g"], s["u"] = (s["x"] @ (s[w].t() if case["trans"] else s[w]) for w in ("wg", "wu"))
            s["dout"] = rand(m, f, scale=0.1)
        return s
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.empty(rows, vocab, device="cuda", dtype=dt)
    for r in range(0, rows, 1024):
        logits[r:r + 1024] = rand(min(1024, rows - r), vocab, scale=2.5)
    targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    if case["masked"]:
        for r in range(0, rows, 1024):
            logits[r:r + 1024].masked_fill_(torch.rand(min(1024, rows - r), vocab, generator=gen, device="cuda") < 0.3, -math.inf)
        if rows > 2:
            logits[rows // 2] = -math.inf  # nothing is allowed here
    # half of the tokens were likely ones
    likely = torch.rand(rows, generator=gen, device="cuda") < 0.5
    likely[rows // 2] = False
    at = likely.nonzero().squeeze(1)
    logits[at, targets[at]] = rand(at.numel(), scale=1.0, shift=14.0)
    if case["padded"]:
        targets[rows - rows // 16:] = -1
    s = {"case": case, "logits": logits, "targets": targets}
    if case["backward"]:
        # statistics that the forward pass kept
        x = logits.float() / case["temperature"]
        log_z = torch.logsumexp(x, -1)
        m = logits.amax(-1).float()
        empty = torch.isinf(m)
        p = torch.exp(x - torch.where(empty, 0.0, log_z)[:, None])
        x.clamp_(min=-3e38)
        s["row_max"] = m
        s["log_sum"] = torch.where(empty, -math.inf, log_z - m / case["temperature"])
        s["entropy"] = torch.where(empty, 0.0, log_z - (p * x).sum(-1))
        s["dlogprob"] = torch.randn(rows, generator=gen, device="cuda")
        s["dentropy"] = torch.randn(rows, generator=gen, device="cuda") * 0.1
    return s


# ---------------------------------------------------------------- plain forms


def _rstd(v):
    return torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)


def _gate_rows(gate, rows):
    """The gate of every row, as float32: [rows, cols] or [1, cols]."""
    if gate.dim() == 1:
        return gate.float()[None]
    return gate.float().repeat_interleave(rows // gate.shape[0], 0)


def _norm_forward(s):
    c, f = s["case"], lambda t: t.float()
    dt = s["x"].dtype
    n = f(s["h"])
    if s["w_post"] is not None:
        n = n * _rstd(n) * f(s["w_post"])
    n = n * c["beta"]
    if s["gate"] is not None:
        n = n * _gate_rows(s["gate"], c["rows"])
    xo = c["alpha"] * f(s["x"]) + n
    y = xo * _rstd(xo) * f(s["w_pre"]) if s["w_pre"] is not None else None
    return {"x_out": xo.to(dt), "y": y.to(dt) if y is not None else None}


def _norm_backward(s):
    c, f = s["case"], lambda t: t.float()
    dt = s["x"].dtype
    h, wp = f(s["h"]), f(s["w_post"]) if s["w_post"] is not None else None
    rh = _rstd(h) if wp is not None else None
    n = h * rh * wp if wp is not None else h
    gate = _gate_rows(s["gate"], c["rows"]) if s["gate"] is not None else None
    xo = c["alpha"] * f(s["x"]) + c["beta"] * (n * gate if gate is not None else n)
    d, out = f(s["dx_out"]), {}
    if s["w_pre"] is not None:
        rx = _rstd(xo)
        xh, dy = xo * rx, f(s["dy"])
        dxh = dy * f(s["w_pre"])
        d = d + rx * (dxh - xh * (dxh * xh).mean(-1, keepdim=True))
        out["dw_pre"] = (dy * xh).sum(0).to(dt)
    out["dx"] = (c["alpha"] * d).to(dt)
    dn = c["beta"] * d
    if gate is not None:
        dg = dn * n
        out["dgate"] = (dg.sum(0) if s["gate"].dim() == 1 else dg.view(s["gate"].shape[0], -1, c["cols"]).sum(1)).to(dt)
        dn = dn * gate
    if wp is not None:
        hh = h * rh
        dhh = dn * wp
        out["dw_post"] = (dn * hh).sum(0).to(dt)
        dn = rh * (dhh - hh * (dhh * hh).mean(-1, keepdim=True))
    out["dh"] = dn.to(dt)
    return out


def _act(g, kind):
    """The activation and its derivative."""
    if kind == "silu":
        p = 1 / (1 + torch.exp(-g))
        return g * p, p * (1 + g * (1 - p))
    if kind == "gelu":
        p = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * p, p + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def _linear_forward(s):
    c, dt = s["case"], s["x"].dtype
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    g, u = x @ (wg.t() if c["trans"] else wg), x @ (wu.t() if c["trans"] else wu)
    out = {"out": (_act(g, c["act"])[0] * u).to(dt)}
    if c["save"]:
        out["g"], out["u"] = g.to(dt), u.to(dt)
    return out


def _linear_backward(s):
    c, dt = s["case"], s["x"].dtype
    x, wg, wu, g, u, dout = (s[k].float() for k in ("x", "wg", "wu", "g", "u", "dout"))
    a, da = _act(g, c["act"])
    dg, du = dout * u * da, dout * a
    if c["trans"]:
        return {"dx": (dg @ wg + du @ wu).to(dt), "dwg": (dg.t() @ x).to(dt), "dwu": (du.t() @ x).to(dt)}
    return {"dx": (dg @ wg.t() + du @ wu.t()).to(dt), "dwg": (x.t() @ dg).to(dt), "dwu": (x.t() @ du).to(dt)}


def _logprobs_forward(s):
    c, t = s["case"], s["targets"]
    x = s["logits"].float()
    m = x.amax(-1)
    empty = m == -math.inf
    z = (x - torch.where(empty, 0.0, m)[:, None]) / c["temperature"]
    e = torch.exp(z)
    total = e.sum(-1)
    log_sum = torch.log(total)
    none = torch.full_like(m, -math.inf)
    zt = z.gather(1, t.clamp(min=0)[:, None])[:, 0]
    logprob = torch.where(t < 0, 0.0, torch.where(empty, none, zt - log_sum))
    entropy = torch.where(empty, 0.0, log_sum - (e * z.clamp(min=-3e38)).sum(-1) / total)
    out = {"logprob": logprob, "entropy": entropy, "row_max": m, "log_sum": log_sum}
    if c["top"]:
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
        lp = z.gather(1, ids) - log_sum[:, None]
        out["top_ids"], out["top_logprobs"] = ids.to(torch.int32), torch.where(empty[:, None], none[:, None], lp)
    return out


def _logprobs_backward(s):
    c, t = s["case"], s["targets"]
    m, log_sum = s["row_max"], s["log_sum"]
    empty = (m == -math.inf)[:, None]
    lp = (s["logits"].float() - torch.where(empty, 0.0, m[:, None])) / c["temperature"] - torch.where(empty, 0.0, log_sum[:, None])
    p = torch.where(empty, 0.0, torch.exp(lp))
    gl = torch.where(t < 0, 0.0, s["dlogprob"])[:, None]
    d = -p * (gl + s["dentropy"][:, None] * (lp.clamp(min=-3e38) + s["entropy"][:, None]))
    d.scatter_add_(1, t.clamp(min=0)[:, None], torch.where(empty, 0.0, gl))
    return {"dlogits": (d / c["temperature"]).to(s["logits"].dtype)}


# ---------------------------------------------------------------- the framework's operators


def _own(s):
    from bee_b200 import tensor_cuda as tc
    c = s["case"]
    if c["op"] == "norm":
        h, x = s["h"], s["x"]
        more = {"w_post": s["w_post"], "gate": s["gate"], "w_pre": s["w_pre"], "alpha": c["alpha"], "beta": c["beta"], "eps": EPS}
        if not c["backward"]:
            xo, y = torch.empty_like(x), torch.empty_like(x) if c["pre"] else None
            tc.norm_gate_residual(h, x, xo, y, **more)
            return {"x_out": xo, "y": y}
        out = {"dh": torch.empty_like(h), "dx": torch.empty_like(x)}
        for k in ("w_post", "gate", "w_pre"):
            if s[k] is not None:
                out["d" + k] = torch.empty_like(s[k])
        tc.norm_gate_residual_backward(h, x, s["dx_out"], s["dy"], out["dh"], out["dx"], dw_post=out.get("dw_post"),
                                       dgate=out.get("dgate"), dw_pre=out.get("dw_pre"), **more)
        return out
    if c["op"] == "linear":
        x, wg, wu = s["x"], s["wg"], s["wu"]
        if not c["backward"]:
            out = {k: x.new_empty(c["rows"], c["f"]) for k in (("out", "g", "u") if c["save"] else ("out",))}
            tc.gated_linear(x, wg, wu, out["out"], act=c["act"], trans=c["trans"], g=out.get("g"), u=out.get("u"))
            return out
        out = {"dx": torch.empty_like(x), "dwg": torch.empty_like(wg), "dwu": torch.empty_like(wu)}
        tc.gated_linear_backward(x, wg, wu, s["g"], s["u"], s["dout"], out["dx"], out["dwg"], out["dwu"], act=c["act"],
                                 trans=c["trans"])
        return out
    logits, rows = s["logits"], c["rows"]
    if not c["backward"]:
        out = {k: torch.empty(rows, device="cuda") for k in ("logprob", "entropy", "row_max", "log_sum")}
        if c["top"]:
            out["top_ids"] = torch.empty(rows, c["top"], device="cuda", dtype=torch.int32)
            out["top_logprobs"] = torch.empty(rows, c["top"], device="cuda")
        tc.token_logprobs(logits, s["targets"], out["logprob"], out["entropy"], out["row_max"], out["log_sum"],
                          temperature=c["temperature"], top_ids=out.get("top_ids"), top_logprobs=out.get("top_logprobs"))
        return out
    out = {"dlogits": torch.empty_like(logits)}
    tc.token_logprobs_backward(logits, s["targets"], s["row_max"], s["log_sum"], s["entropy"], s["dlogprob"], s["dentropy"],
                               out["dlogits"], temperature=c["temperature"])
    return out


def run(state):
    if own:
        return _own(state)
    c = state["case"]
    forward, backward = {"norm": (_norm_forward, _norm_backward), "linear": (_linear_forward, _linear_backward),
                         "logprobs": (_logprobs_forward, _logprobs_backward)}[c["op"]]
    return (backward if c["backward"] else forward)(state)


# ---------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    """Gradients come from differentiating the forward definitions, not from the formulas of the plain forms."""
    s = prepare(case, seed)
    d = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    if case["op"] == "norm":
        names = [k for k in ("h", "x", "w_post", "gate", "w_pre") if d[k] is not None]
        for k in names:
            d[k].requires_grad_(case["backward"])

        def rms(v, w):
            return v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + EPS) * w

        def branch(h, gate):
            v = h if d["w_post"] is None else rms(h, d["w_post"])
            return v if gate is None else v * gate

        gate = d["gate"]
        if gate is not None and gate.dim() == 2:
            v = branch(d["h"].view(gate.shape[0], -1, case["cols"]), gate[:, None]).reshape(case["rows"], case["cols"])
        else:
            v = branch(d["h"], gate)
        xo = case["alpha"] * d["x"] + case["beta"] * v
        y = rms(xo, d["w_pre"]) if d["w_pre"] is not None else None
        if not case["backward"]:
            return {"x_out": xo, "y": y}
        loss = (xo * d["dx_out"]).sum() + ((y * d["dy"]).sum() if y is not None else 0)
        return {"d" + k: g for k, g in zip(names, torch.autograd.grad(loss, [d[k] for k in names]))}
    if case["op"] == "linear":
        def act(g):
            if case["act"] == "silu":
                return torch.nn.functional.silu(g)
            return torch.nn.functional.gelu(g, approximate="tanh" if case["act"] == "gelu_tanh" else "none")

        wg, wu = (d["wg"].t(), d["wu"].t()) if case["trans"] else (d["wg"], d["wu"])
        if not case["backward"]:
            g, u = d["x"] @ wg, d["x"] @ wu
            return {"out": act(g) * u, **({"g": g, "u": u} if case["save"] else {})}
        g, u = d["g"].requires_grad_(), d["u"].requires_grad_()
        dg, du = torch.autograd.grad((act(g) * u * d["dout"]).sum(), [g, u])
        dwg, dwu = d["x"].t() @ dg, d["x"].t() @ du
        return {"dx": dg @ wg.t() + du @ wu.t(), "dwg": dwg.t() if case["trans"] else dwg, "dwu": dwu.t() if case["trans"] else dwu}
    t, inside = d["targets"], d["targets"] >= 0
    rows = torch.arange(case["rows"], device=t.device)
    x = d["logits"] / case["temperature"]
    empty = torch.isinf(x.amax(-1))
    if case["backward"]:
        x = torch.where(empty[:, None], 0.0, x).requires_grad_()
        lp = torch.log_softmax(x, -1)
        entropy = -(lp.exp() * lp.masked_fill(torch.isinf(lp), 0.0)).sum(-1)
        loss = (lp[rows, t.clamp(min=0)] * inside * ~empty * d["dlogprob"]).sum() + (entropy * ~empty * d["dentropy"]).sum()
        return {"dlogits": torch.autograd.grad(loss, x)[0] / case["temperature"]}
    lp = torch.log_softmax(torch.where(empty[:, None], 0.0, x), -1)
    none = torch.full_like(lp[:, 0], -math.inf)
    top = lp.topk(case["top"]).values if case["top"] else None
    m = d["logits"].amax(-1)
    return {"logprob": torch.where(inside, torch.where(empty, none, lp[rows, t.clamp(min=0)]), 0.0),
            "entropy": torch.where(empty, 0.0, torch.special.entr(lp.exp()).sum(-1)), "row_max": m,
            "log_sum": torch.where(empty, none, torch.logsumexp(x, -1) - m / case["temperature"]),
            **({"top_ids": None, "top_logprobs": torch.where(empty[:, None], none[:, None], top)} if top is not None else {})}
