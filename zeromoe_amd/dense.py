"""The dense operators around the routed layer, over the C ABI (include/zeromoe.h): the unquantized matrix product with
its epilogue, the layer norm, the weighted sum of the experts' rows, and their gradients with that of the routing.

Device tensors in, device tensors out, on the current stream or on `stream`; outputs and workspaces come from torch's
allocator for that stream, so a call may be captured into a graph.  Gradients are calls of their own: nothing here is
recorded by autograd, so a tensor that requires a gradient is refused unless torch.no_grad() (or a Function of the
caller's around a pair of calls) says that none is expected."""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import ZmGluDesc, ZmLinearDesc, check, lib
from .ops import _spec

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4, "sigmoid": 5}
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_F32, _I32 = torch.float32, torch.int32
_F32S, _I32S = (_F32,), (_I32,)
_ROWS = torch.contiguous_format


# the current stream's handle without a Stream object around it, and the current device: 0.1 us each of a call's 7,
# against 1.1 and 0.3
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _index(t: torch.Tensor, who: str) -> int:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{who}: device tensors are needed")
    return t.get_device()


_grad_mode = torch.is_grad_enabled


def _not_recorded(who: str):
    raise ValueError(f"{who}: an argument requires a gradient, which is not recorded here: call it under torch.no_grad() "
                     "and take the gradient from its own call, or pass the tensor detached")


def _there(fn, d: int, stream, *args):
    """The call on the device of its tensors and on `stream`, whose allocations are then that stream's."""
    if stream is None:
        with torch.cuda.device(d):
            return fn(*args)
    if stream.device.index != d:
        raise ValueError(f"{fn.__name__}: the stream belongs to another device than the tensors")
    with torch.cuda.stream(stream):
        return fn(*args)


def _need(t: torch.Tensor, what: str, d: int, dtypes, shape) -> torch.Tensor:
    """`t` with the device, type and shape that the call needs."""
    if t.get_device() != d:
        raise ValueError(f"{what} is on another device")
    if t.dtype not in dtypes:
        raise ValueError(f"{what} is {t.dtype}: {', '.join(str(x) for x in dtypes)} needed")
    if t.shape != shape:
        raise ValueError(f"{what} has shape {tuple(t.shape)}: {shape} needed")
    return t


_COUNTS = 1 << 31  # sizes from here on do not fit the C calls' 32-bit counts, which would take them for others


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` with contiguous columns; rows keep their stride."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _flat(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def _out(t: torch.Tensor, what: str, d: int, dtype, shape) -> torch.Tensor:
    _need(t, what, d, (dtype,), shape)
    if t.stride(-1) != 1 and shape[-1] != 1:
        raise ValueError(f"{what} needs contiguous columns")
    return t


def _vector(t: Optional[torch.Tensor], what: str, d: int, n: int):
    return None if t is None else _flat(_need(t, what, d, _F32S, (n,)))


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _space(n: int, like: torch.Tensor):
    return like.new_empty(n, dtype=torch.uint8) if n else None


def _act(act) -> int:
    if act not in ACTIVATIONS:
        raise ValueError(f"unknown activation {act!r}: {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS[act]


def _linear_types(d, x, w):
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"x (S, I) and w (O, I) are needed, not {tuple(x.shape)} and {tuple(w.shape)}")
    if x.get_device() != d or w.get_device() != d:
        raise ValueError("x or w is on another device")
    if x.dtype not in _TYPES or w.dtype not in _TYPES or (x.dtype != _F32 and w.dtype != x.dtype):
        raise ValueError(f"x {x.dtype} with w {w.dtype}: float32 activations with float32, float16 or bfloat16 weights, "
                         "or both of one 16-bit type")
    if w.stride(1) != 1 and w.shape[1] != 1:
        raise ValueError("w needs contiguous columns")


def linear(x: torch.Tensor, w: torch.Tensor, bias=None, act: str = "none", residual=None, out=None, out_dtype=None,
           save_pre: bool = False, stream=None):
    """act(x w^T + bias) + residual: x (S, I), w (O, I), bias (O) float32, residual (S, O) of the result's type.

    x float32 with w float32, float16 or bfloat16, or both float16 or both bfloat16; the result is of x's type or
    float32 (`out_dtype`, or `out`'s type).  act: none, relu, gelu, gelu_tanh, silu, sigmoid.  `out` may be `residual`
    itself, and overlaps no other operand.  save_pre: also returns x w^T + bias, in the result's type, for
    linear_backward.  (zm_linear)"""
    d = _index(x, "linear")
    if stream is not None or d != _device():
        return _there(linear, d, stream, x, w, bias, act, residual, out, out_dtype, save_pre)
    if _grad_mode() and (x.requires_grad or w.requires_grad or bias is not None and bias.requires_grad
                         or residual is not None and residual.requires_grad or out is not None and out.requires_grad):
        _not_recorded("linear")
    st = _raw_stream(d)
    _linear_types(d, x, w)
    S, I = x.shape
    O = w.shape[0]
    x = _rows(x)
    dtype = out_dtype or (out.dtype if out is not None else x.dtype)
    if dtype != _F32 and dtype != x.dtype:
        raise ValueError(f"the result is float32 or {x.dtype}, not {dtype}")
    y = x.new_empty((S, O), dtype=dtype) if out is None else _out(out, "out", d, dtype, (S, O))
    if residual is not None:
        residual = _rows(_need(residual, "residual", d, (dtype,), (S, O)))
    bias = _vector(bias, "bias", d, O)
    pre = x.new_empty((S, O), dtype=dtype) if save_pre else None
    desc = ZmLinearDesc(_TYPES[x.dtype], _TYPES[w.dtype], _TYPES[dtype], _act(act), S, I, O, x.stride(0), w.stride(0),
                        y.stride(0), residual.stride(0) if residual is not None else 0, O)
    L = lib()
    ws = _space(L.zm_linear_workspace_size(desc), x)
    check(L.zm_linear(desc, x.data_ptr(), w.data_ptr(), _ptr(bias), _ptr(residual), y.data_ptr(), _ptr(pre), _ptr(ws),
                      0 if ws is None else ws.numel(), st), "zm_linear")
    return (y, pre) if save_pre else y


def linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, act: str = "none", pre=None,
                    need_dx: bool = True, need_dw: bool = True, need_dbias: bool = True, stream=None):
    """(dx, dw, dbias) of linear() for dy (S, O), its gradient by the result: dx (S, I) of x's type, dw (O, I) and
    dbias (O) float32; None in the place of one that is not needed.  The residual's gradient is dy itself.  pre: what
    linear(save_pre=True) returned, needed with an activation.  Behind an activation, or from a float32 dy, a 16-bit dx
    takes 16 bits of dy act'(pre).  (zm_linear_backward)"""
    d = _index(dy, "linear_backward")
    if stream is not None or d != _device():
        return _there(linear_backward, d, stream, dy, x, w, act, pre, need_dx, need_dw, need_dbias)
    if _grad_mode() and (dy.requires_grad or x.requires_grad or w.requires_grad
                         or pre is not None and pre.requires_grad):
        _not_recorded("linear_backward")
    st = _raw_stream(d)
    _linear_types(d, x, w)
    S, I = x.shape
    O = w.shape[0]
    x = _rows(x)
    dy = _rows(_need(dy, "dy", d, (_F32, x.dtype), (S, O)))
    a = _act(act)
    if a:
        if pre is None:
            raise ValueError("an activation's gradient needs pre")
        pre = _rows(_need(pre, "pre", d, (dy.dtype,), (S, O)))
    else:
        pre = None
    dx = x.new_empty((S, I)) if need_dx else None
    dw = x.new_empty((O, I), dtype=_F32) if need_dw else None
    db = x.new_empty(O, dtype=_F32) if need_dbias else None
    desc = ZmLinearDesc(_TYPES[x.dtype], _TYPES[w.dtype], _TYPES[dy.dtype], a, S, I, O, x.stride(0), w.stride(0),
                        dy.stride(0), 0, pre.stride(0) if pre is not None else 0)
    L = lib()
    ws = _space(L.zm_linear_backward_workspace_size(desc), x)
    check(L.zm_linear_backward(desc, dy.data_ptr(), x.data_ptr(), w.data_ptr(), _ptr(pre), _ptr(dx), _ptr(dw), _ptr(db),
                               _ptr(ws), 0 if ws is None else ws.numel(), st), "zm_linear_backward")
    return dx, dw, db


def _glu_weights(d, x, w_gate, w_up):
    _linear_types(d, x, w_gate)
    _need(w_up, "w_up", d, (w_gate.dtype,), w_gate.shape)
    F, I = w_gate.shape
    if w_up.stride(1) != 1 and I != 1:
        raise ValueError("w_up needs contiguous columns")
    if w_up.stride(0) != w_gate.stride(0) and F != 1:
        raise ValueError(f"w_gate and w_up need rows of one stride, not {w_gate.stride(0)} and {w_up.stride(0)}")


def glu(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate=None, b_up=None, act: str = "silu", out=None,
        out_dtype=None, save: bool = False, stream=None):
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up), the gated half of a feed-forward block in one product: x (S, I),
    w_gate and w_up (F, I) of one type and stride, b_gate and b_up (F) float32, each optional; types and activations as
    linear()'s.  save: also returns both factors before the activation, (S, F) each in the result's type, for
    glu_backward.  `out` overlaps no operand.  (zm_glu)"""
    d = _index(x, "glu")
    if stream is not None or d != _device():
        return _there(glu, d, stream, x, w_gate, w_up, b_gate, b_up, act, out, out_dtype, save)
    if _grad_mode() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad
                         or b_gate is not None and b_gate.requires_grad or b_up is not None and b_up.requires_grad
                         or out is not None and out.requires_grad):
        _not_recorded("glu")
    st = _raw_stream(d)
    _glu_weights(d, x, w_gate, w_up)
    S, I = x.shape
    F = w_gate.shape[0]
    x = _rows(x)
    dtype = out_dtype or (out.dtype if out is not None else x.dtype)
    if dtype != _F32 and dtype != x.dtype:
        raise ValueError(f"the result is float32 or {x.dtype}, not {dtype}")
    y = x.new_empty((S, F), dtype=dtype) if out is None else _out(out, "out", d, dtype, (S, F))
    b_gate, b_up = _vector(b_gate, "b_gate", d, F), _vector(b_up, "b_up", d, F)
    gate = up = None
    if save:
        gate, up = x.new_empty((S, F), dtype=dtype), x.new_empty((S, F), dtype=dtype)
    desc = ZmGluDesc(_TYPES[x.dtype], _TYPES[w_gate.dtype], _TYPES[dtype], _act(act), S, I, F, x.stride(0),
                     w_gate.stride(0), y.stride(0), F, F)
    L = lib()
    ws = _space(L.zm_glu_workspace_size(desc), x)
    check(L.zm_glu(desc, x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), _ptr(b_gate), _ptr(b_up), y.data_ptr(),
                   _ptr(gate), _ptr(up), _ptr(ws), 0 if ws is None else ws.numel(), st), "zm_glu")
    return (y, gate, up) if save else y


def glu_backward(dy: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, gate: torch.Tensor,
                 up: torch.Tensor, act: str = "silu", need_dx: bool = True, need_dw: bool = True, need_db: bool = True,
                 stream=None):
    """(dx, dw_gate, dw_up, db_gate, db_up) of glu() for dy (S, F), its gradient by the result, with the factors gate and
    up that glu(save=True) returned, all three of one type: dx (S, I) of x's type, the weights' (F, I) and the biases'
    (F) float32; None in the place of those that are not needed.  A 16-bit dx takes 16 bits of the factors' gradients.
    (zm_glu_backward)"""
    d = _index(dy, "glu_backward")
    if stream is not None or d != _device():
        return _there(glu_backward, d, stream, dy, x, w_gate, w_up, gate, up, act, need_dx, need_dw, need_db)
    if _grad_mode() and (dy.requires_grad or x.requires_grad or w_gate.requires_grad or w_up.requires_grad
                         or gate.requires_grad or up.requires_grad):
        _not_recorded("glu_backward")
    st = _raw_stream(d)
    _glu_weights(d, x, w_gate, w_up)
    S, I = x.shape
    F = w_gate.shape[0]
    x = _rows(x)
    dy = _rows(_need(dy, "dy", d, (_F32, x.dtype), (S, F)))
    gate = _rows(_need(gate, "gate", d, (dy.dtype,), (S, F)))
    up = _rows(_need(up, "up", d, (dy.dtype,), (S, F)))
    dx = x.new_empty((S, I)) if need_dx else None
    dw = x.new_empty((2, F, I), dtype=_F32) if need_dw else None
    db = x.new_empty((2, F), dtype=_F32) if need_db else None
    desc = ZmGluDesc(_TYPES[x.dtype], _TYPES[w_gate.dtype], _TYPES[dy.dtype], _act(act), S, I, F, x.stride(0),
                     w_gate.stride(0), dy.stride(0), gate.stride(0), up.stride(0))
    L = lib()
    ws = _space(L.zm_glu_backward_workspace_size(desc), x)
    check(L.zm_glu_backward(desc, dy.data_ptr(), x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), gate.data_ptr(),
                            up.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), 0 if ws is None else ws.numel(), st),
          "zm_glu_backward")
    dw_gate, dw_up = (None, None) if dw is None else dw.unbind(0)
    db_gate, db_up = (None, None) if db is None else db.unbind(0)
    return dx, dw_gate, dw_up, db_gate, db_up


def _norm_rows(d, x):
    if x.get_device() != d:
        raise ValueError("x is on another device")
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"x (rows, n) is needed, not {tuple(x.shape)}")
    if x.dtype not in _TYPES:
        raise ValueError(f"x is {x.dtype}: float32, float16 or bfloat16 needed")


def layer_norm(x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5, out=None, stats: bool = False, stream=None):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the rows of x (rows, n), in x's type; weight and bias (n)
    float32.  `out` may be x itself.  stats: also returns each row's mean and 1 / sqrt(variance + eps), for
    layer_norm_backward.  (zm_layer_norm)"""
    d = _index(x, "layer_norm")
    if stream is not None or d != _device():
        return _there(layer_norm, d, stream, x, weight, bias, eps, out, stats)
    if _grad_mode() and (x.requires_grad or weight is not None and weight.requires_grad
                         or bias is not None and bias.requires_grad or out is not None and out.requires_grad):
        _not_recorded("layer_norm")
    st = _raw_stream(d)
    _norm_rows(d, x)
    rows, n = x.shape
    x = _rows(x)
    y = torch.empty_like(x, memory_format=_ROWS) if out is None else _out(out, "out", d, x.dtype, (rows, n))
    weight, bias = _vector(weight, "weight", d, n), _vector(bias, "bias", d, n)
    mean = rstd = None
    if stats:
        mean, rstd = x.new_empty((2, rows), dtype=_F32).unbind(0)
    check(lib().zm_layer_norm(_TYPES[x.dtype], x.data_ptr(), x.stride(0), _ptr(weight), _ptr(bias), eps, rows, n,
                              y.data_ptr(), y.stride(0), _ptr(mean), _ptr(rstd), st), "zm_layer_norm")
    return (y, mean, rstd) if stats else y


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, weight=None,
                        need_dx: bool = True, need_dweight: bool = True, need_dbias: bool = True, stream=None):
    """(dx, dweight, dbias) of layer_norm() for dy (rows, n) of x's type, with the statistics that it returned: dx of
    x's type, dweight and dbias (n) float32; None in the place of one that is not needed.  (zm_layer_norm_backward)"""
    d = _index(dy, "layer_norm_backward")
    if stream is not None or d != _device():
        return _there(layer_norm_backward, d, stream, dy, x, mean, rstd, weight, need_dx, need_dweight, need_dbias)
    if _grad_mode() and (dy.requires_grad or x.requires_grad or mean.requires_grad or rstd.requires_grad
                         or weight is not None and weight.requires_grad):
        _not_recorded("layer_norm_backward")
    st = _raw_stream(d)
    _norm_rows(d, x)
    rows, n = x.shape
    x = _rows(x)
    dy = _rows(_need(dy, "dy", d, (x.dtype,), (rows, n)))
    mean, rstd = _vector(mean, "mean", d, rows), _vector(rstd, "rstd", d, rows)
    weight = _vector(weight, "weight", d, n)
    dx = torch.empty_like(x, memory_format=_ROWS) if need_dx else None
    dw = x.new_empty(n, dtype=_F32) if need_dweight else None
    db = x.new_empty(n, dtype=_F32) if need_dbias else None
    L = lib()
    ws = _space(L.zm_layer_norm_backward_workspace_size(rows, n) if need_dweight or need_dbias else 0, x)
    check(L.zm_layer_norm_backward(_TYPES[x.dtype], dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), _ptr(weight),
                                   mean.data_ptr(), rstd.data_ptr(), rows, n, _ptr(dx), n, _ptr(dw), _ptr(db), _ptr(ws),
                                   0 if ws is None else ws.numel(), st), "zm_layer_norm_backward")
    return dx, dw, db


def _routes(y):
    if y.dim() != 3 or y.dtype != _F32:
        raise ValueError(f"y (S, K, H) float32 is needed, not {tuple(y.shape)} {y.dtype}")
    if y.shape[1] >= _COUNTS or y.shape[2] >= _COUNTS:
        raise ValueError(f"y of {tuple(y.shape)} is too large")
    return _rows(y)


def combine(y: torch.Tensor, weights: torch.Tensor, ids=None, residual=None, out=None, stream=None):
    """residual + sum over k of weights[:, k] * y[:, k]: the experts' rows y (S, K, H) as mul_mat_id returns them,
    weights (S, K), residual (S, H) and the result, all float32.  A route with a negative id in ids (S, K) int32 takes
    no part.  `out` may be `residual` itself.  (zm_combine)"""
    d = _index(y, "combine")
    if stream is not None or d != _device():
        return _there(combine, d, stream, y, weights, ids, residual, out)
    if _grad_mode() and (y.requires_grad or weights.requires_grad or residual is not None and residual.requires_grad
                         or out is not None and out.requires_grad):
        _not_recorded("combine")
    st = _raw_stream(d)
    y = _routes(y)
    S, K, H = y.shape
    weights = _flat(_need(weights, "weights", d, _F32S, (S, K)))
    if ids is not None:
        ids = _flat(_need(ids, "ids", d, _I32S, (S, K)))
    if residual is not None:
        residual = _flat(_need(residual, "residual", d, _F32S, (S, H)))
    if out is None:
        out = y.new_empty((S, H))
    elif not _out(out, "out", d, _F32, (S, H)).is_contiguous():
        raise ValueError("out needs to be contiguous")
    check(lib().zm_combine(y.data_ptr(), y.stride(0), y.stride(1), weights.data_ptr(), _ptr(ids), _ptr(residual), S, K, H,
                           out.data_ptr(), st), "zm_combine")
    return out


def combine_backward(dout: torch.Tensor, y: torch.Tensor, weights=None, ids=None, need_dy: bool = False, stream=None):
    """dweights (S, K) of combine() for dout (S, H): the dot products of dout with the experts' rows, 0 for a route with
    a negative id.  need_dy: (dweights, dy), dy (S, K, H) = weights * dout, which needs weights.  The residual's
    gradient is dout itself.  (zm_combine_backward)"""
    d = _index(dout, "combine_backward")
    if stream is not None or d != _device():
        return _there(combine_backward, d, stream, dout, y, weights, ids, need_dy)
    if _grad_mode() and (dout.requires_grad or y.requires_grad or weights is not None and weights.requires_grad):
        _not_recorded("combine_backward")
    st = _raw_stream(d)
    y = _routes(y)
    S, K, H = y.shape
    if y.get_device() != d:
        raise ValueError("y is on another device")
    dout = _flat(_need(dout, "dout", d, _F32S, (S, H)))
    if ids is not None:
        ids = _flat(_need(ids, "ids", d, _I32S, (S, K)))
    if need_dy and weights is None:
        raise ValueError("dy needs weights")
    if weights is not None:
        weights = _flat(_need(weights, "weights", d, _F32S, (S, K)))
    dweights = y.new_empty((S, K))
    dy = y.new_empty((S, K, H)) if need_dy else None
    check(lib().zm_combine_backward(dout.data_ptr(), y.data_ptr(), y.stride(0), y.stride(1), _ptr(weights), _ptr(ids), S,
                                    K, H, dweights.data_ptr(), _ptr(dy), st), "zm_combine_backward")
    return (dweights, dy) if need_dy else dweights


def router_backward(logits: torch.Tensor, ids: torch.Tensor, dweights: torch.Tensor, gating="softmax",
                    logit_bias=None, weights_norm: bool = False, weights_scale: float = 0.0, dprobs=None, stream=None):
    """The gradient of router()'s weights by its logits (S, E) float32, the selection held fixed: ids (S, K) int32 are
    expert ids (router() without a slot table or a mask), dweights (S, K).  A negative id takes no part; a row of them
    alone has a zero gradient.  dprobs (E): added to the gradient of every routed token's gate probabilities, as a
    balance loss on their mean has it.  The gradient by logit_bias is the result's sum over the tokens.
    (zm_router_backward)"""
    d = _index(logits, "router_backward")
    if stream is not None or d != _device():
        return _there(router_backward, d, stream, logits, ids, dweights, gating, logit_bias, weights_norm, weights_scale,
                      dprobs)
    if _grad_mode() and (logits.requires_grad or dweights.requires_grad
                         or logit_bias is not None and logit_bias.requires_grad
                         or dprobs is not None and dprobs.requires_grad):
        _not_recorded("router_backward")
    st = _raw_stream(d)
    if logits.dim() != 2 or logits.dtype != _F32 or ids.dim() != 2:
        raise ValueError("logits (S, E) float32 and ids (S, K) are needed")
    S, E = logits.shape
    K = ids.shape[1]
    if S >= _COUNTS or E >= _COUNTS or K >= _COUNTS:
        raise ValueError(f"logits of {tuple(logits.shape)} or ids of {tuple(ids.shape)} are too large")
    logits = _flat(logits)
    ids = _flat(_need(ids, "ids", d, _I32S, (S, K)))
    dweights = _flat(_need(dweights, "dweights", d, _F32S, (S, K)))
    logit_bias, dprobs = _vector(logit_bias, "logit_bias", d, E), _vector(dprobs, "dprobs", d, E)
    out = torch.empty_like(logits)
    spec = _spec(E, K, gating, 0, 0, weights_norm, weights_scale)
    check(lib().zm_router_backward(spec, logits.data_ptr(), _ptr(logit_bias), ids.data_ptr(), dweights.data_ptr(),
                                   _ptr(dprobs), S, out.data_ptr(), st), "zm_router_backward")
    return out
