"""Calls that the fused operators refuse, on the host: no kernel is launched."""
import math

import pytest

from bee_b200 import _capi

P = 4096  # a 16-byte aligned address that is never read: every call here is refused first
F32, BF16, F16, I32, I64 = _capi.F32, _capi.BF16, _capi.F16, _capi.I32, _capi.I64


def refused(name, *args):
    rc = getattr(_capi.lib(), name)(*args)
    msg = _capi.last_error()
    assert rc == 1 and msg, (name, rc, msg)
    return msg


def accepted(name, *args):
    assert getattr(_capi.lib(), name)(*args) == 0, _capi.last_error()


def logprobs(dt=BF16, logits=P, ld=64, tdt=I64, targets=P, rows=4, vocab=64, temperature=1.0, logprob=P, entropy=P,
             row_max=P, log_sum=P, top=0, ids=None, lps=None):
    return ("bee_b200_token_logprobs", dt, logits, ld, tdt, targets, rows, vocab, temperature, logprob, entropy, row_max,
            log_sum, top, ids, lps, None)


@pytest.mark.parametrize("change,word", [
    ({"dt": I32}, "dtype"), ({"logits": None}, "null"), ({"ld": 63}, "stride"), ({"tdt": F32}, "targets"),
    ({"targets": None}, "null"), ({"vocab": 0, "ld": 0}, "vocab"), ({"vocab": 2 ** 31, "ld": 2 ** 31}, "vocab"),
    ({"temperature": 0.0}, "temperature"), ({"temperature": -1.0}, "temperature"), ({"temperature": math.nan}, "temperature"),
    ({"temperature": math.inf}, "temperature"), ({"temperature": 1e-45}, "temperature"), ({"top": 33, "ids": P, "lps": P}, "alternatives"),
    ({"top": 9, "vocab": 8, "ids": P, "lps": P}, "alternatives"), ({"top": 2, "lps": P}, "null"), ({"top": 2, "ids": P}, "null"),
    ({"logits": P + 1}, "aligned"), ({"dt": F32, "logits": P + 2}, "aligned"),
])
def test_logprobs_refusals(change, word):
    assert word in refused(*logprobs(**change))


def test_logprobs_of_no_rows():
    accepted(*logprobs(rows=0, logits=None, targets=None, logprob=None, entropy=None, row_max=None, log_sum=None))


def logprobs_backward(dt=BF16, logits=P, ld=64, tdt=I64, targets=P, rows=4, vocab=64, temperature=1.0, row_max=P, log_sum=P,
                      entropy=P, dlogprob=P, dentropy=P, dlogits=2 * P, ldd=64):
    return ("bee_b200_token_logprobs_backward", dt, logits, ld, tdt, targets, rows, vocab, temperature, row_max, log_sum,
            entropy, dlogprob, dentropy, dlogits, ldd, None)


@pytest.mark.parametrize("change,word", [
    ({"dt": I64}, "dtype"), ({"logits": None}, "null"), ({"dlogits": None}, "null"), ({"ld": 63}, "stride"), ({"ldd": 10}, "stride"),
    ({"row_max": None}, "null"), ({"log_sum": None}, "null"), ({"entropy": None}, "null"), ({"targets": None}, "null"),
    ({"tdt": BF16}, "targets"), ({"temperature": 0.0}, "temperature"), ({"dlogits": P, "ldd": 72}, "in place"),
    ({"dlogits": 2 * P + 1}, "aligned"), ({"vocab": 0}, "vocab"),
])
def test_logprobs_backward_refusals(change, word):
    assert word in refused(*logprobs_backward(**change))


def norm(dt=BF16, h=P, x=P, w_post=P, gate=P, w_pre=P, x_out=P, y=P, rows=8, cols=64, group=0, alpha=1.0, beta=1.0, eps=1e-6):
    return ("bee_b200_norm_gate_residual", dt, h, x, w_post, gate, w_pre, x_out, y, rows, cols, group, alpha, beta, eps, None)


def norm_backward(dt=BF16, h=P, x=P, w_post=P, gate=P, w_pre=P, dx_out=P, dy=P, dh=P, dx=P, dw_post=P, dgate=P, dw_pre=P,
                  rows=8, cols=64, group=0, alpha=1.0, beta=1.0, eps=1e-6):
    return ("bee_b200_norm_gate_residual_backward", dt, h, x, w_post, gate, w_pre, dx_out, dy, dh, dx, dw_post, dgate,
            dw_pre, rows, cols, group, alpha, beta, eps, None)


@pytest.mark.parametrize("call", [norm, norm_backward])
@pytest.mark.parametrize("change,word", [
    ({"dt": I32}, "dtype"), ({"h": None}, "null"), ({"x": None}, "null"), ({"cols": 0}, "columns"), ({"cols": 16385}, "columns"),
    ({"dt": F32, "cols": 12289}, "columns"), ({"group": 3}, "group"), ({"eps": -1.0}, "eps"), ({"eps": math.nan}, "eps"),
    ({"eps": math.inf}, "eps"), ({"alpha": math.nan}, "alpha"), ({"beta": math.inf}, "alpha"), ({"x": P + 1}, "aligned"),
    ({"gate": P + 1}, "aligned"),
])
def test_norm_refusals(call, change, word):
    assert word in refused(*call(**change))


def test_norm_forward_refusals():
    assert "null" in refused(*norm(x_out=None))
    assert "null" in refused(*norm(y=None))
    accepted(*norm(rows=0, h=None, x=None, x_out=None, y=None))


@pytest.mark.parametrize("missing", ["dh", "dx", "dy", "dw_post", "dgate", "dw_pre"])
def test_norm_backward_refusals(missing):
    assert "null" in refused(*norm_backward(**{missing: None}))


def test_norm_backward_needs_a_gradient():
    assert "null" in refused(*norm_backward(w_pre=None, dw_pre=None, dy=None, dx_out=None))


def gated(dt=BF16, act=0, x=P, ldx=64, wg=P, wu=P, ldw=96, trans=0, out=P, g=None, u=None, M=8, D=64, F=96):
    return ("bee_b200_gated_linear", dt, act, x, ldx, wg, wu, ldw, trans, out, g, u, M, D, F, None)


def gated_backward(dt=BF16, act=0, x=P, ldx=64, wg=P, wu=P, ldw=96, trans=0, g=P, u=P, dout=P, dx=P, dwg=P, dwu=P, lddw=96,
                   M=8, D=64, F=96):
    return ("bee_b200_gated_linear_backward", dt, act, x, ldx, wg, wu, ldw, trans, g, u, dout, dx, dwg, dwu, lddw, M, D, F, None)


@pytest.mark.parametrize("call", [gated, gated_backward])
@pytest.mark.parametrize("change,word", [
    ({"dt": F32}, "dtype"), ({"act": 3}, "activation"), ({"act": -1}, "activation"), ({"D": 0}, "extents"), ({"F": 0}, "extents"),
    ({"M": 2 ** 31}, "extents"), ({"F": 2 ** 31, "ldw": 2 ** 31}, "extents"), ({"ldx": 63}, "stride"), ({"ldw": 95}, "stride"),
    ({"ldw": 63, "trans": 1}, "stride"), ({"x": None}, "null"), ({"wg": None}, "null"), ({"wu": None}, "null"), ({"x": P + 1}, "aligned"),
    ({"wu": P + 1}, "aligned"),
])
def test_gated_refusals(call, change, word):
    assert word in refused(*call(**change))


def test_gated_forward_refusals():
    assert "null" in refused(*gated(out=None))
    assert "null" in refused(*gated(g=P))
    accepted(*gated(M=0, x=None, wg=None, wu=None, out=None))


@pytest.mark.parametrize("change", [{"g": None}, {"u": None}, {"dout": None}, {"dwg": None}, {"dwu": None},
                                    {"dx": None, "dwg": None, "dwu": None}])
def test_gated_backward_refusals(change):
    assert "null" in refused(*gated_backward(**change))


def test_gated_backward_stride():
    assert "stride" in refused(*gated_backward(lddw=95))
    accepted(*gated_backward(M=0, dwg=None, dwu=None, x=None, wg=None, wu=None, g=None, u=None, dout=None))


def test_gated_wrappers_refuse_what_is_no_matrix(monkeypatch):
    torch = pytest.importorskip("torch")
    from bee_b200 import tensor_cuda as tc
    monkeypatch.setattr(tc, "_current", lambda *a: None)  # the shapes are looked at on the host
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    for bad in (x[0, 0], x[0], x[None]):
        with pytest.raises(tc.BeeError):
            tc.gated_linear(x, x, x, bad)
        with pytest.raises(tc.BeeError):
            tc.gated_linear_backward(x, x, x, bad, x, x, dx=x)
    with pytest.raises(tc.BeeError):
        tc.gated_linear_backward(x, x, x, None, None, x, dx=x)


@pytest.mark.parametrize("change", [{"out": P}, {"out": 2 * P}, {"out": 3 * P}, {"g": P, "u": 7 * P}, {"g": 6 * P, "u": 3 * P},
                                    {"g": 6 * P, "u": 6 * P}, {"g": 4 * P, "u": 6 * P}])
def test_gated_outputs_apart(change):
    assert "overlap" in refused(*gated(**{"x": P, "wg": 2 * P, "wu": 3 * P, "out": 4 * P, **change}))


@pytest.mark.parametrize("change", [{"dx": P}, {"dx": 2 * P}, {"dwg": 3 * P}, {"dwu": P}, {"dwg": 9 * P, "dwu": 9 * P},
                                    {"dx": 9 * P, "dwg": 9 * P}])
def test_gated_gradients_apart(change):
    apart = {"x": P, "wg": 2 * P, "wu": 3 * P, "g": 4 * P, "u": 5 * P, "dout": 6 * P, "dx": 7 * P, "dwg": 8 * P, "dwu": 10 * P}
    assert "overlap" in refused(*gated_backward(**{**apart, **change}))
