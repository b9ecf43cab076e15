"""Python mirror of ``bee::tensor::cuda`` (Bee/Tensor/Cuda/Backend.hpp:20-84).

Same operation names and argument meaning as the reference's host bridge, over
torch CUDA tensors (torch supplies device memory and the stream; every kernel is
ours, reached through the C ABI).  Like the reference bridge each call is
synchronous from the caller's point of view only if ``sync=True``; by default
work is enqueued on torch's current stream and ordered with other torch work.
Errors raise ``BeeError`` carrying the status and message; there is no CPU path.
"""
from __future__ import annotations

import torch

from . import _capi as C
from ._capi import BeeError  # noqa: F401  (re-export)

DTYPE_CODE = {
    torch.bool: C.BOOL, torch.uint8: C.U8, torch.int32: C.I32, torch.int64: C.I64,
    torch.float32: C.F32, torch.float64: C.F64, torch.int8: C.I8, torch.float16: C.F16,
    torch.bfloat16: C.BF16,
}


def _code(t: torch.Tensor) -> int:
    try:
        return DTYPE_CODE[t.dtype]
    except KeyError:
        raise BeeError("dtype", 1, f"unsupported torch dtype {t.dtype}") from None


def _dev(*ts: torch.Tensor) -> None:
    for t in ts:
        if not t.is_cuda:
            raise BeeError("device", 1, "tensor is not on a CUDA device")
        if not t.is_contiguous():
            raise BeeError("layout", 1, "tensor is not contiguous")


# the current stream's handle without building a Stream object (0.1 us against 3 us a call), where torch offers it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(stream=None) -> int:
    if stream is None and _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device())
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _done(sync: bool, stream=None) -> None:
    if sync:
        C.call("bee_b200_stream_synchronize", _stream(stream))


def ew_binary(op: int, a: torch.Tensor, b: torch.Tensor, out: torch.Tensor, *, stream=None, sync=False):
    """out = a (op) b elementwise (tensor::cuda::ew_binary, Backend.hpp:51)."""
    _dev(a, b, out)
    if not (a.dtype == b.dtype == out.dtype) or not (a.numel() == b.numel() == out.numel()):
        raise BeeError("ew_binary", 1, "a, b, out must share dtype and element count")
    C.call("bee_b200_ew_binary", op, _code(a), a.data_ptr(), b.data_ptr(), out.data_ptr(), a.numel(), _stream(stream))
    _done(sync, stream)
    return out


def ew_unary(op: int, src: torch.Tensor, dst: torch.Tensor, *, stream=None, sync=False):
    """dst = op(src) (tensor::cuda::ew_unary, Backend.hpp:54)."""
    _dev(src, dst)
    C.call("bee_b200_ew_unary", op, _code(src), src.data_ptr(), dst.data_ptr(), src.numel(), _stream(stream))
    _done(sync, stream)
    return dst


def ew_cast(src: torch.Tensor, dst: torch.Tensor, *, stream=None, sync=False):
    """dst = cast(src) (tensor::cuda::ew_cast, Backend.hpp:57), incl. fp32 -> bf16."""
    _dev(src, dst)
    if src.numel() != dst.numel():
        raise BeeError("ew_cast", 1, "element counts differ")
    C.call("bee_b200_ew_cast", _code(src), src.data_ptr(), _code(dst), dst.data_ptr(), src.numel(), _stream(stream))
    _done(sync, stream)
    return dst


def scale_fp(buf: torch.Tensor, factor: float, *, stream=None, sync=False):
    """buf *= factor (tensor::cuda::scale_fp, Backend.hpp:66)."""
    _dev(buf)
    C.call("bee_b200_scale_fp", _code(buf), buf.data_ptr(), float(factor), buf.numel(), _stream(stream))
    _done(sync, stream)
    return buf


def reduce_global(op: int, src: torch.Tensor, dst: torch.Tensor, *, stream=None, sync=False):
    """dst[0] = reduce(src) (tensor::cuda::reduce_global, Backend.hpp:60)."""
    _dev(src, dst)
    C.call("bee_b200_reduce_global", op, _code(src), src.data_ptr(), dst.data_ptr(), src.numel(), _stream(stream))
    _done(sync, stream)
    return dst


def reduce_axis(op: int, src: torch.Tensor, dst: torch.Tensor, outer: int, axis: int, inner: int, *, stream=None,
                sync=False):
    """[outer, axis, inner] -> [outer, inner] (tensor::cuda::reduce_axis, Backend.hpp:63)."""
    _dev(src, dst)
    C.call("bee_b200_reduce_axis", op, _code(src), src.data_ptr(), dst.data_ptr(), outer, axis, inner,
           _stream(stream))
    _done(sync, stream)
    return dst


def softmax_rows(src: torch.Tensor, dst: torch.Tensor, *, stream=None, sync=False):
    """Row softmax of a [rows, cols] tensor (last dim)."""
    _dev(src, dst)
    cols = src.shape[-1]
    rows = src.numel() // cols if cols else 0
    C.call("bee_b200_softmax_rows", _code(src), src.data_ptr(), dst.data_ptr(), rows, cols, _stream(stream))
    _done(sync, stream)
    return dst


def rms_norm_rows(x: torch.Tensor, w: torch.Tensor, y: torch.Tensor, eps: float = 1e-6, *, stream=None, sync=False):
    """y = x / sqrt(mean(x^2) + eps) * w over the last dim."""
    _dev(x, w, y)
    cols = x.shape[-1]
    C.call("bee_b200_rms_norm_rows", _code(x), x.data_ptr(), w.data_ptr(), y.data_ptr(), x.numel() // cols, cols,
           float(eps), _stream(stream))
    _done(sync, stream)
    return y


def rope(x: torch.Tensor, y: torch.Tensor, seq: int, heads: int, head_dim: int, theta: float = 10000.0,
         pos_offset: int = 0, *, stream=None, sync=False):
    """Rotate-half RoPE on x viewed [rows, heads, head_dim], position = row % seq + pos_offset."""
    _dev(x, y)
    rows = x.numel() // (heads * head_dim)
    C.call("bee_b200_rope", _code(x), x.data_ptr(), y.data_ptr(), rows, seq, heads, head_dim, float(theta),
           pos_offset, _stream(stream))
    _done(sync, stream)
    return y


def rms_norm_rope(x: torch.Tensor, w: torch.Tensor, y: torch.Tensor, seq: int, heads: int, head_dim: int,
                  eps: float = 1e-6, theta: float = 10000.0, pos_offset: int = 0, *, stream=None, sync=False):
    """RMSNorm then RoPE in one pass over [rows, heads*head_dim]."""
    _dev(x, w, y)
    rows = x.numel() // (heads * head_dim)
    C.call("bee_b200_rms_norm_rope", _code(x), x.data_ptr(), w.data_ptr(), y.data_ptr(), rows, seq, heads, head_dim,
           float(eps), float(theta), pos_offset, _stream(stream))
    _done(sync, stream)
    return y


def _current(op: str, *ts) -> None:
    """Checks that every given tensor lives on the calling thread's current device, where the kernels run."""
    dev = None
    for t in ts:
        if t is None:
            continue
        at = t.get_device()  # -1 on the CPU
        if at != dev:
            if not t.is_cuda:
                raise BeeError(op, 1, "tensor is not on a CUDA device")
            if dev is None:
                dev = torch.cuda.current_device()
            if at != dev:
                raise BeeError(op, 1, f"tensor is on cuda:{at}, the current device is cuda:{dev}")


def _rows(op: str, name: str, t: torch.Tensor) -> int:
    """Row stride (in elements) of a 2-D tensor whose rows are contiguous and do not overlap."""
    if t.dim() != 2:
        raise BeeError(op, 1, f"{name} must be 2-D")
    r, c = t.shape
    s0, s1 = t.stride()
    if (s1 != 1 and c > 1) or (s0 < c and r > 1):
        raise BeeError(op, 1, f"{name}: rows must be contiguous and must not overlap")
    return s0 if r > 1 else max(c, 1)


def _vector(op: str, name: str, t, n: int, dtype) -> int:
    """Pointer of an optional contiguous vector of n elements."""
    if t is None:
        return None
    if t.dtype != dtype or t.numel() != n or not t.is_contiguous():
        raise BeeError(op, 1, f"{name} must be contiguous, {dtype}, with {n} elements")
    return t.data_ptr()


def _like(op: str, name: str, t, x: torch.Tensor) -> int:
    """Pointer of an optional contiguous tensor of x's dtype and shape."""
    if t is None:
        return None
    if t.dtype != x.dtype or t.shape != x.shape or not t.is_contiguous():
        raise BeeError(op, 1, f"{name} must be contiguous, {x.dtype}, {tuple(x.shape)}")
    return t.data_ptr()


def _gate(op: str, name: str, gate, rows: int, cols: int, dtype):
    """Pointer and group of an optional gate: [cols], or [groups, cols] with groups dividing the rows."""
    if gate is None:
        return None, 0
    if gate.dim() == 1:
        return _vector(op, name, gate, cols, dtype), 0
    if gate.dim() != 2 or gate.shape[1] != cols or gate.dtype != dtype or not gate.is_contiguous():
        raise BeeError(op, 1, f"{name} must be contiguous, {dtype}, [cols] or [groups, cols]")
    groups = gate.shape[0]
    if groups == 0 and rows == 0:
        return gate.data_ptr(), 1
    if groups == 0 or rows % groups or rows == 0:
        raise BeeError(op, 1, f"{rows} rows are not a multiple of {groups} gate rows")
    return gate.data_ptr(), rows // groups


def norm_gate_residual(h: torch.Tensor, x: torch.Tensor, x_out: torch.Tensor, y=None, *, w_post=None, gate=None,
                       w_pre=None, alpha: float = 1.0, beta: float = 1.0, eps: float = 1e-6, stream=None, sync=False):
    """x_out = alpha x + beta gate rmsnorm(h) w_post and y = rmsnorm(x_out) w_pre, over the last dim of [rows, cols].

    w_post and w_pre [cols] and gate ([cols], or [groups, cols]: one for each rows / groups consecutive rows) are optional;
    without w_post h is not normalised, without w_pre there is no y."""
    op = "norm_gate_residual"
    _current(op, h, x, x_out, y, w_post, gate, w_pre)
    if x.dim() != 2 or not x.is_contiguous():
        raise BeeError(op, 1, "x must be a contiguous [rows, cols] tensor")
    rows, cols = x.shape
    if (y is None) != (w_pre is None):
        raise BeeError(op, 1, "y and w_pre go together")
    gptr, group = _gate(op, "gate", gate, rows, cols, x.dtype)
    C.call("bee_b200_norm_gate_residual", _code(x), _like(op, "h", h, x), x.data_ptr(),
           _vector(op, "w_post", w_post, cols, x.dtype), gptr, _vector(op, "w_pre", w_pre, cols, x.dtype),
           _like(op, "x_out", x_out, x), _like(op, "y", y, x), rows, cols, group, float(alpha), float(beta), float(eps),
           _stream(stream))
    _done(sync, stream)
    return x_out


def norm_gate_residual_backward(h: torch.Tensor, x: torch.Tensor, dx_out, dy, dh: torch.Tensor, dx: torch.Tensor, *,
                                w_post=None, gate=None, w_pre=None, dw_post=None, dgate=None, dw_pre=None,
                                alpha: float = 1.0, beta: float = 1.0, eps: float = 1e-6, stream=None, sync=False):
    """Gradients dh, dx (and dw_post, dgate, dw_pre of whichever is given) from the forward's inputs and the gradients
    dx_out (None: zero) and dy of its outputs."""
    op = "norm_gate_residual_backward"
    _current(op, h, x, dx_out, dy, dh, dx, w_post, gate, w_pre, dw_post, dgate, dw_pre)
    if x.dim() != 2 or not x.is_contiguous():
        raise BeeError(op, 1, "x must be a contiguous [rows, cols] tensor")
    rows, cols = x.shape
    for name, v, d in (("w_post", w_post, dw_post), ("gate", gate, dgate), ("w_pre", w_pre, dw_pre)):
        if (v is None) != (d is None):
            raise BeeError(op, 1, f"{name} and d{name} go together")
    if (dy is None) != (w_pre is None):
        raise BeeError(op, 1, "dy and w_pre go together")
    gptr, group = _gate(op, "gate", gate, rows, cols, x.dtype)
    if gate is not None and dgate.shape != gate.shape:
        raise BeeError(op, 1, "dgate must have the gate's shape")
    dgptr, _ = _gate(op, "dgate", dgate, rows, cols, x.dtype)
    C.call("bee_b200_norm_gate_residual_backward", _code(x), _like(op, "h", h, x), x.data_ptr(),
           _vector(op, "w_post", w_post, cols, x.dtype), gptr, _vector(op, "w_pre", w_pre, cols, x.dtype),
           _like(op, "dx_out", dx_out, x), _like(op, "dy", dy, x), _like(op, "dh", dh, x), _like(op, "dx", dx, x),
           _vector(op, "dw_post", dw_post, cols, x.dtype), dgptr, _vector(op, "dw_pre", dw_pre, cols, x.dtype), rows, cols,
           group, float(alpha), float(beta), float(eps), _stream(stream))
    _done(sync, stream)
    return dx


def _targets(op: str, targets, rows: int):
    if targets is None:
        return C.I64, None
    if targets.dtype not in (torch.int32, torch.int64):
        raise BeeError(op, 1, "targets must be int32 or int64")
    return DTYPE_CODE[targets.dtype], _vector(op, "targets", targets, rows, targets.dtype)


def token_logprobs(logits: torch.Tensor, targets, logprob=None, entropy=None, row_max=None, log_sum=None, *,
                   temperature: float = 1.0, top_ids=None, top_logprobs=None, stream=None, sync=False):
    """Log probabilities of `targets` [rows] under softmax(logits / temperature), logits [rows, vocab] (rows may be strided).

    Writes whichever of logprob, entropy, row_max, log_sum (float32 [rows]) and top_ids / top_logprobs (int32 /
    float32 [rows, k], k <= 32: the k largest logits, equal ones by lowest index) are given.  A negative target means
    that the row holds no token (logprob 0).  row_max and log_sum are what the backward needs."""
    op = "token_logprobs"
    _current(op, logits, targets, logprob, entropy, row_max, log_sum, top_ids, top_logprobs)
    ld = _rows(op, "logits", logits)
    rows, vocab = logits.shape
    f32 = torch.float32
    if logprob is not None and targets is None:
        raise BeeError(op, 1, "logprob needs targets")
    tdt, tptr = _targets(op, targets, rows)
    if (top_ids is None) != (top_logprobs is None):
        raise BeeError(op, 1, "top_ids and top_logprobs go together")
    k = 0
    if top_ids is not None:
        if top_ids.dim() != 2 or top_ids.shape[0] != rows:
            raise BeeError(op, 1, "top_ids must be [rows, k]")
        k = top_ids.shape[1]
    C.call("bee_b200_token_logprobs", _code(logits), logits.data_ptr(), ld, tdt, tptr, rows, vocab, float(temperature),
           _vector(op, "logprob", logprob, rows, f32), _vector(op, "entropy", entropy, rows, f32),
           _vector(op, "row_max", row_max, rows, f32), _vector(op, "log_sum", log_sum, rows, f32), k,
           _vector(op, "top_ids", top_ids, rows * k, torch.int32),
           _vector(op, "top_logprobs", top_logprobs, rows * k, f32), _stream(stream))
    _done(sync, stream)
    return logprob


def token_logprobs_backward(logits: torch.Tensor, targets, row_max: torch.Tensor, log_sum: torch.Tensor, entropy,
                            dlogprob, dentropy, dlogits: torch.Tensor, *, temperature: float = 1.0, stream=None,
                            sync=False):
    """dlogits = gradient of sum(dlogprob * logprob + dentropy * entropy); row_max, log_sum and entropy come from the
    forward, dlogprob and dentropy (float32 [rows]) may be None.  dlogits may be logits itself."""
    op = "token_logprobs_backward"
    _current(op, logits, targets, row_max, log_sum, entropy, dlogprob, dentropy, dlogits)
    ld, ldd = _rows(op, "logits", logits), _rows(op, "dlogits", dlogits)
    rows, vocab = logits.shape
    f32 = torch.float32
    if dlogits.dtype != logits.dtype or dlogits.shape != logits.shape:
        raise BeeError(op, 1, "dlogits must have the logits' dtype and shape")
    if dlogprob is not None and targets is None:
        raise BeeError(op, 1, "dlogprob needs targets")
    tdt, tptr = _targets(op, targets, rows)
    C.call("bee_b200_token_logprobs_backward", _code(logits), logits.data_ptr(), ld, tdt, tptr, rows, vocab,
           float(temperature), _vector(op, "row_max", row_max, rows, f32), _vector(op, "log_sum", log_sum, rows, f32),
           _vector(op, "entropy", entropy, rows, f32), _vector(op, "dlogprob", dlogprob, rows, f32),
           _vector(op, "dentropy", dentropy, rows, f32), dlogits.data_ptr(), ldd, _stream(stream))
    _done(sync, stream)
    return dlogits


ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


def _act(op: str, act: str) -> int:
    try:
        return ACTIVATIONS[act]
    except KeyError:
        raise BeeError(op, 1, f"act must be one of {', '.join(ACTIVATIONS)}") from None


def _pair(op: str, names: str, a: torch.Tensor, b: torch.Tensor, shape, dtype) -> int:
    """Common row stride of two matrices of one shape."""
    ld = _rows(op, names, a)
    if _rows(op, names, b) != ld or a.shape != shape or b.shape != shape or a.dtype != dtype or b.dtype != dtype:
        raise BeeError(op, 1, f"{names} must both be {dtype}, {tuple(shape)}, with the same row stride")
    return ld


def _width(op: str, name: str, t) -> int:
    """Columns of a matrix that has to be given."""
    if t is None or t.dim() != 2:
        raise BeeError(op, 1, f"{name} must be 2-D")
    return t.shape[1]


def _matrix(op: str, name: str, t, m: int, n: int, dtype) -> int:
    """Pointer of an optional contiguous [m, n] matrix."""
    if t is None:
        return None
    if t.dtype != dtype or t.shape != (m, n) or not t.is_contiguous():
        raise BeeError(op, 1, f"{name} must be contiguous, {dtype}, ({m}, {n})")
    return t.data_ptr()


def gated_linear(x: torch.Tensor, wg: torch.Tensor, wu: torch.Tensor, out: torch.Tensor, *, act: str = "silu",
                 trans: bool = False, g=None, u=None, stream=None, sync=False):
    """out = act(x @ wg) * (x @ wu): x [M, D], out [M, F]; wg and wu [D, F], or [F, D] with trans.

    x and the weights may have strided rows.  act is "silu", "gelu" or "gelu_tanh".  g and u [M, F], when given, receive
    the two products for the backward."""
    op = "gated_linear"
    _current(op, x, wg, wu, out, g, u)
    ldx = _rows(op, "x", x)
    m, d = x.shape
    f = _width(op, "out", out)
    ldw = _pair(op, "wg and wu", wg, wu, (f, d) if trans else (d, f), x.dtype)
    if (g is None) != (u is None):
        raise BeeError(op, 1, "g and u go together")
    C.call("bee_b200_gated_linear", _code(x), _act(op, act), x.data_ptr(), ldx, wg.data_ptr(), wu.data_ptr(), ldw, int(trans),
           _matrix(op, "out", out, m, f, x.dtype), _matrix(op, "g", g, m, f, x.dtype), _matrix(op, "u", u, m, f, x.dtype), m, d,
           f, _stream(stream))
    _done(sync, stream)
    return out


def gated_linear_backward(x: torch.Tensor, wg: torch.Tensor, wu: torch.Tensor, g: torch.Tensor, u: torch.Tensor,
                          dout: torch.Tensor, dx=None, dwg=None, dwu=None, *, act: str = "silu", trans: bool = False,
                          stream=None, sync=False):
    """Gradients dx [M, D] and dwg, dwu (in the weights' layout; rows may be strided) from the forward's inputs, its g and
    u, and dout [M, F].  dx, or dwg and dwu, may be None."""
    op = "gated_linear_backward"
    _current(op, x, wg, wu, g, u, dout, dx, dwg, dwu)
    ldx = _rows(op, "x", x)
    m, d = x.shape
    f = _width(op, "g", g)
    shape = (f, d) if trans else (d, f)
    ldw = _pair(op, "wg and wu", wg, wu, shape, x.dtype)
    if (dwg is None) != (dwu is None):
        raise BeeError(op, 1, "dwg and dwu go together")
    if dx is None and dwg is None:
        raise BeeError(op, 1, "no gradient is asked for")
    lddw = _pair(op, "dwg and dwu", dwg, dwu, shape, x.dtype) if dwg is not None else 0
    C.call("bee_b200_gated_linear_backward", _code(x), _act(op, act), x.data_ptr(), ldx, wg.data_ptr(), wu.data_ptr(), ldw,
           int(trans), _matrix(op, "g", g, m, f, x.dtype), _matrix(op, "u", u, m, f, x.dtype),
           _matrix(op, "dout", dout, m, f, x.dtype), _matrix(op, "dx", dx, m, d, x.dtype),
           dwg.data_ptr() if dwg is not None else None, dwu.data_ptr() if dwu is not None else None, lddw, m, d, f,
           _stream(stream))
    _done(sync, stream)
    return dx
