"""The dense operators around the routed layer, over the C ABI (include/zeromoe.h): the unquantized matrix product with
its epilogue, the layer norm, the weighted sum of the experts' rows, and their gradients with that of the routing.

Device tensors in, device tensors out, on the current stream or on `stream`; outputs and workspaces come from torch's
allocator for that stream, so a call may be captured into a graph.  Gradients are calls of their own: nothing here is
recorded by autograd."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from ._lib import ZmLinearDesc, check, lib
from .ops import _spec

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4, "sigmoid": 5}
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_F32, _I32 = torch.float32, torch.int32


def _on(fn):
    """Runs the call where its first tensor lies and on `stream`, whose allocations are then that stream's."""
    def call(*args, stream=None, **kw):
        t = args[0]
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"{fn.__name__}: device tensors are needed")
        d = t.get_device()
        if stream is not None:
            if stream.device.index != d:
                raise ValueError(f"{fn.__name__}: the stream belongs to another device than the tensors")
            with torch.cuda.stream(stream):
                return fn(stream.cuda_stream, *args, **kw)
        if d != torch.cuda.current_device():
            with torch.cuda.device(d):
                return fn(torch.cuda.current_stream(d).cuda_stream, *args, **kw)
        return fn(torch.cuda.current_stream(d).cuda_stream, *args, **kw)

    call.__name__, call.__qualname__, call.__doc__, call.__wrapped__ = fn.__name__, fn.__qualname__, fn.__doc__, fn
    return call


def _need(t: torch.Tensor, what: str, like: torch.Tensor, dtypes, shape) -> torch.Tensor:
    """`t` with the device, type and shape that the call needs."""
    if t.device != like.device:
        raise ValueError(f"{what} is on another device")
    if t.dtype not in dtypes:
        raise ValueError(f"{what} is {t.dtype}: {', '.join(str(d) for d in dtypes)} needed")
    if tuple(t.shape) != shape:
        raise ValueError(f"{what} has shape {tuple(t.shape)}: {shape} needed")
    return t


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` with contiguous columns; rows keep their stride."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _out(t: torch.Tensor, what: str, like: torch.Tensor, dtype, shape) -> torch.Tensor:
    _need(t, what, like, (dtype,), shape)
    if t.stride(-1) != 1 and shape[-1] != 1:
        raise ValueError(f"{what} needs contiguous columns")
    return t


def _vector(t: Optional[torch.Tensor], what: str, like: torch.Tensor, n: int):
    return None if t is None else _need(t, what, like, (_F32,), (n,)).contiguous()


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _space(n: int, like: torch.Tensor):
    return torch.empty(n, dtype=torch.uint8, device=like.device) if n else None


def _act(act) -> int:
    if act not in ACTIVATIONS:
        raise ValueError(f"unknown activation {act!r}: {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS[act]


def _linear_types(x, w):
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"x (S, I) and w (O, I) are needed, not {tuple(x.shape)} and {tuple(w.shape)}")
    if w.device != x.device:
        raise ValueError("w is on another device")
    if x.dtype not in _TYPES or w.dtype not in _TYPES or (x.dtype != _F32 and w.dtype != x.dtype):
        raise ValueError(f"x {x.dtype} with w {w.dtype}: float32 activations with float32, float16 or bfloat16 weights, "
                         "or both of one 16-bit type")
    if w.stride(1) != 1 and w.shape[1] != 1:
        raise ValueError("w needs contiguous columns")


@_on
def linear(st, x: torch.Tensor, w: torch.Tensor, bias=None, act: str = "none", residual=None, out=None, out_dtype=None,
           save_pre: bool = False):
    """act(x w^T + bias) + residual: x (S, I), w (O, I), bias (O) float32, residual (S, O) of the result's type.

    x float32 with w float32, float16 or bfloat16, or both float16 or both bfloat16; the result is of x's type or
    float32 (`out_dtype`, or `out`'s type).  act: none, relu, gelu, gelu_tanh, silu, sigmoid.  `out` may be `residual`
    itself.  save_pre: also returns x w^T + bias, in the result's type, for linear_backward.  (zm_linear)"""
    _linear_types(x, w)
    S, I = x.shape
    O = w.shape[0]
    x = _rows(x)
    dtype = out_dtype or (out.dtype if out is not None else x.dtype)
    if dtype != _F32 and dtype != x.dtype:
        raise ValueError(f"the result is float32 or {x.dtype}, not {dtype}")
    y = torch.empty((S, O), dtype=dtype, device=x.device) if out is None else _out(out, "out", x, dtype, (S, O))
    if residual is not None:
        residual = _rows(_need(residual, "residual", x, (dtype,), (S, O)))
    bias = _vector(bias, "bias", x, O)
    pre = torch.empty((S, O), dtype=dtype, device=x.device) if save_pre else None
    d = ZmLinearDesc(_TYPES[x.dtype], _TYPES[w.dtype], _TYPES[dtype], _act(act), S, I, O, x.stride(0), w.stride(0),
                     y.stride(0), residual.stride(0) if residual is not None else 0, O)
    L = lib()
    ws = _space(L.zm_linear_workspace_size(d), x)
    check(L.zm_linear(d, x.data_ptr(), w.data_ptr(), _ptr(bias), _ptr(residual), y.data_ptr(), _ptr(pre), _ptr(ws),
                      0 if ws is None else ws.numel(), st), "zm_linear")
    return (y, pre) if save_pre else y


@_on
def linear_backward(st, dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, act: str = "none", pre=None,
                    need_dx: bool = True, need_dw: bool = True, need_dbias: bool = True):
    """(dx, dw, dbias) of linear() for dy (S, O), its gradient by the result: dx (S, I) of x's type, dw (O, I) and
    dbias (O) float32; None in the place of one that is not needed.  The residual's gradient is dy itself.  pre: what
    linear(save_pre=True) returned, needed with an activation.  (zm_linear_backward)"""
    _linear_types(x, w)
    S, I = x.shape
    O = w.shape[0]
    x = _rows(x)
    dy = _rows(_need(dy, "dy", x, (_F32, x.dtype), (S, O)))
    a = _act(act)
    if a:
        if pre is None:
            raise ValueError("an activation's gradient needs pre")
        pre = _rows(_need(pre, "pre", x, (dy.dtype,), (S, O)))
    else:
        pre = None
    dev = x.device
    dx = torch.empty((S, I), dtype=x.dtype, device=dev) if need_dx else None
    dw = torch.empty((O, I), dtype=_F32, device=dev) if need_dw else None
    db = torch.empty(O, dtype=_F32, device=dev) if need_dbias else None
    d = ZmLinearDesc(_TYPES[x.dtype], _TYPES[w.dtype], _TYPES[dy.dtype], a, S, I, O, x.stride(0), w.stride(0),
                     dy.stride(0), 0, pre.stride(0) if pre is not None else 0)
    L = lib()
    ws = _space(L.zm_linear_backward_workspace_size(d), x)
    check(L.zm_linear_backward(d, dy.data_ptr(), x.data_ptr(), w.data_ptr(), _ptr(pre), _ptr(dx), _ptr(dw), _ptr(db),
                               _ptr(ws), 0 if ws is None else ws.numel(), st), "zm_linear_backward")
    return dx, dw, db


def _norm_rows(x, what="x"):
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"{what} (rows, n) is needed, not {tuple(x.shape)}")
    if x.dtype not in _TYPES:
        raise ValueError(f"{what} is {x.dtype}: float32, float16 or bfloat16 needed")


@_on
def layer_norm(st, x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5, out=None, stats: bool = False):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the rows of x (rows, n), in x's type; weight and bias (n)
    float32.  `out` may be x itself.  stats: also returns each row's mean and 1 / sqrt(variance + eps), for
    layer_norm_backward.  (zm_layer_norm)"""
    _norm_rows(x)
    rows, n = x.shape
    x = _rows(x)
    y = torch.empty((rows, n), dtype=x.dtype, device=x.device) if out is None else _out(out, "out", x, x.dtype, (rows, n))
    weight, bias = _vector(weight, "weight", x, n), _vector(bias, "bias", x, n)
    mean = rstd = None
    if stats:
        mean, rstd = torch.empty((2, rows), dtype=_F32, device=x.device).unbind(0)
    check(lib().zm_layer_norm(_TYPES[x.dtype], x.data_ptr(), x.stride(0), _ptr(weight), _ptr(bias), eps, rows, n,
                              y.data_ptr(), y.stride(0), _ptr(mean), _ptr(rstd), st), "zm_layer_norm")
    return (y, mean, rstd) if stats else y


@_on
def layer_norm_backward(st, dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, weight=None,
                        need_dx: bool = True, need_dweight: bool = True, need_dbias: bool = True):
    """(dx, dweight, dbias) of layer_norm() for dy (rows, n) of x's type, with the statistics that it returned: dx of
    x's type, dweight and dbias (n) float32; None in the place of one that is not needed.  (zm_layer_norm_backward)"""
    _norm_rows(x)
    rows, n = x.shape
    x = _rows(x)
    dy = _rows(_need(dy, "dy", x, (x.dtype,), (rows, n)))
    mean, rstd = _vector(mean, "mean", x, rows), _vector(rstd, "rstd", x, rows)
    weight = _vector(weight, "weight", x, n)
    dx = torch.empty((rows, n), dtype=x.dtype, device=x.device) if need_dx else None
    dw = torch.empty(n, dtype=_F32, device=x.device) if need_dweight else None
    db = torch.empty(n, dtype=_F32, device=x.device) if need_dbias else None
    L = lib()
    ws = _space(L.zm_layer_norm_backward_workspace_size(rows, n) if need_dweight or need_dbias else 0, x)
    check(L.zm_layer_norm_backward(_TYPES[x.dtype], dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), _ptr(weight),
                                   mean.data_ptr(), rstd.data_ptr(), rows, n, _ptr(dx), n, _ptr(dw), _ptr(db), _ptr(ws),
                                   0 if ws is None else ws.numel(), st), "zm_layer_norm_backward")
    return dx, dw, db


def _routes(y, what="y"):
    if y.dim() != 3 or y.dtype != _F32:
        raise ValueError(f"{what} (S, K, H) float32 is needed, not {tuple(y.shape)} {y.dtype}")
    return _rows(y)


@_on
def combine(st, y: torch.Tensor, weights: torch.Tensor, ids=None, residual=None, out=None):
    """residual + sum over k of weights[:, k] * y[:, k]: the experts' rows y (S, K, H) as mul_mat_id returns them,
    weights (S, K), residual (S, H) and the result, all float32.  A route with a negative id in ids (S, K) int32 takes
    no part.  `out` may be `residual` itself.  (zm_combine)"""
    y = _routes(y)
    S, K, H = y.shape
    weights = _need(weights, "weights", y, (_F32,), (S, K)).contiguous()
    if ids is not None:
        ids = _need(ids, "ids", y, (_I32,), (S, K)).contiguous()
    if residual is not None:
        residual = _need(residual, "residual", y, (_F32,), (S, H)).contiguous()
    if out is None:
        out = torch.empty((S, H), dtype=_F32, device=y.device)
    elif not _out(out, "out", y, _F32, (S, H)).is_contiguous():
        raise ValueError("out needs to be contiguous")
    check(lib().zm_combine(y.data_ptr(), y.stride(0), y.stride(1), weights.data_ptr(), _ptr(ids), _ptr(residual), S, K, H,
                           out.data_ptr(), st), "zm_combine")
    return out


@_on
def combine_backward(st, dout: torch.Tensor, y: torch.Tensor, weights=None, ids=None, need_dy: bool = False):
    """dweights (S, K) of combine() for dout (S, H): the dot products of dout with the experts' rows, 0 for a route with
    a negative id.  need_dy: (dweights, dy), dy (S, K, H) = weights * dout, which needs weights.  The residual's
    gradient is dout itself.  (zm_combine_backward)"""
    y = _routes(y)
    S, K, H = y.shape
    dout = _need(dout, "dout", y, (_F32,), (S, H)).contiguous()
    if ids is not None:
        ids = _need(ids, "ids", y, (_I32,), (S, K)).contiguous()
    if need_dy and weights is None:
        raise ValueError("dy needs weights")
    if weights is not None:
        weights = _need(weights, "weights", y, (_F32,), (S, K)).contiguous()
    dweights = torch.empty((S, K), dtype=_F32, device=y.device)
    dy = torch.empty((S, K, H), dtype=_F32, device=y.device) if need_dy else None
    check(lib().zm_combine_backward(dout.data_ptr(), y.data_ptr(), y.stride(0), y.stride(1), _ptr(weights), _ptr(ids), S,
                                    K, H, dweights.data_ptr(), _ptr(dy), st), "zm_combine_backward")
    return (dweights, dy) if need_dy else dweights


@_on
def router_backward(st, logits: torch.Tensor, ids: torch.Tensor, dweights: torch.Tensor, gating="softmax",
                    logit_bias=None, weights_norm: bool = False, weights_scale: float = 0.0, dprobs=None):
    """The gradient of router()'s weights by its logits (S, E) float32, the selection held fixed: ids (S, K) int32 are
    expert ids (router() without a slot table), dweights (S, K).  A negative id takes no part; a row of them alone has
    a zero gradient.  dprobs (E): added to the gradient of every routed token's gate probabilities, as a balance loss
    on their mean has it.  The gradient by logit_bias is the result's sum over the tokens.  (zm_router_backward)"""
    if logits.dim() != 2 or logits.dtype != _F32 or ids.dim() != 2:
        raise ValueError("logits (S, E) float32 and ids (S, K) are needed")
    logits = logits.contiguous()
    S, E = logits.shape
    K = ids.shape[1]
    ids = _need(ids, "ids", logits, (_I32,), (S, K)).contiguous()
    dweights = _need(dweights, "dweights", logits, (_F32,), (S, K)).contiguous()
    logit_bias, dprobs = _vector(logit_bias, "logit_bias", logits, E), _vector(dprobs, "dprobs", logits, E)
    out = torch.empty((S, E), dtype=_F32, device=logits.device)
    spec = _spec(E, K, gating, 0, 0, weights_norm, weights_scale)
    check(lib().zm_router_backward(spec, logits.data_ptr(), _ptr(logit_bias), ids.data_ptr(), dweights.data_ptr(),
                                   _ptr(dprobs), S, out.data_ptr(), st), "zm_router_backward")
    return out
