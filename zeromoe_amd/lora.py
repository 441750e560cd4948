"""Low-rank adapters beside a projection that all tokens share, over the C ABI (include/zeromoe.h).

Device tensors in, device tensors out, on the current stream or on `stream`, with workspaces from torch's allocator, so a
call may be captured into a graph.  Gradients are calls of their own, as those of the dense operators."""
from __future__ import annotations

import torch

from ._lib import ZmLoraDesc, check, lib
from .dense import (_F32, _F32S, _I32S, _TYPES, _device, _flat, _grad_mode, _index, _need, _not_recorded, _out, _ptr,
                    _raw_stream, _rows, _space, _there, _vector)


def _operands(d, x, a, b, ids, scale):
    """ids, scale, the sizes (S, I, O, R, n) and the strides of both adapters; each tensor's are asked for once (0.2 us)."""
    xs, sa, sb = x.shape, a.shape, b.shape
    if len(xs) != 2 or len(sa) != 3 or len(sb) != 3 or sa[2] != xs[1] or sb[2] != sa[1] or sb[0] != sa[0]:
        raise ValueError(f"x (S, I), a (n, R, I) and b (n, O, R) are needed, not {tuple(xs)}, {tuple(sa)} and {tuple(sb)}")
    if x.get_device() != d or a.get_device() != d or b.get_device() != d:
        raise ValueError("x, a or b is on another device")
    tx, ta = x.dtype, a.dtype
    if tx not in _TYPES or ta not in _TYPES or ta != b.dtype or (tx != _F32 and ta != tx):
        raise ValueError(f"x {tx} with a {ta} and b {b.dtype}: float32 activations with float32, float16 or bfloat16 "
                         "adapters, or all of one 16-bit type")
    n, R, I = sa
    la, lb = a.stride(), b.stride()
    if (la[2] != 1 and I != 1) or (lb[2] != 1 and R != 1):
        raise ValueError("a and b need contiguous columns")
    ids = _flat(_need(ids, "ids", d, _I32S, (xs[0],)))
    return ids, _vector(scale, "scale", d, n), (xs[0], I, sb[1], R, n), la, lb


def lora(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor, scale=None, residual=None, out=None,
         out_dtype=None, save: bool = False, stream=None):
    """residual + scale[e] * (x a[e]^T) b[e]^T with e = ids[s] for each token s: x (S, I), a (n, R, I) and b (n, O, R) of all
    adapters, ids (S) int32, scale (n) float32, residual (S, O) of the result's type.

    x float32 with adapters float32, float16 or bfloat16, or all float16 or all bfloat16; the result is of x's type or
    float32 (`out_dtype`, or `out`'s type).  A token with a negative id has no adapter: its row is the residual (or zeros).
    `out` may be `residual` itself, and overlaps no other operand.  save: also returns v = x a[e]^T (S, R) float32, for
    lora_backward.  At most 512 adapters, of a rank of at most 256.  (zm_lora)"""
    d = _index(x, "lora")
    if stream is not None or d != _device():
        return _there(lora, d, stream, x, a, b, ids, scale, residual, out, out_dtype, save)
    if _grad_mode() and (x.requires_grad or a.requires_grad or b.requires_grad or scale is not None and scale.requires_grad
                         or residual is not None and residual.requires_grad or out is not None and out.requires_grad):
        _not_recorded("lora")
    st = _raw_stream(d)
    ids, scale, (S, I, O, R, n), la, lb = _operands(d, x, a, b, ids, scale)
    x = _rows(x)
    dtype = out_dtype or (out.dtype if out is not None else x.dtype)
    if dtype != _F32 and dtype != x.dtype:
        raise ValueError(f"the result is float32 or {x.dtype}, not {dtype}")
    y = x.new_empty((S, O), dtype=dtype) if out is None else _out(out, "out", d, dtype, (S, O))
    if residual is not None:
        residual = _rows(_need(residual, "residual", d, (dtype,), (S, O)))
    v = x.new_empty((S, R), dtype=_F32) if save else None
    desc = ZmLoraDesc(_TYPES[x.dtype], _TYPES[a.dtype], _TYPES[dtype], n, R, S, I, O, x.stride(0), y.stride(0),
                      residual.stride(0) if residual is not None else 0, la[1], la[0], lb[1], lb[0])
    L = lib()
    ws = _space(L.zm_lora_workspace_size(desc), x)
    check(L.zm_lora(desc, x.data_ptr(), a.data_ptr(), b.data_ptr(), ids.data_ptr(), _ptr(scale), _ptr(residual), y.data_ptr(),
                    _ptr(v), _ptr(ws), 0 if ws is None else ws.numel(), st), "zm_lora")
    return (y, v) if save else y


def lora_backward(dy: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor, v=None, scale=None,
                  need_dx: bool = True, need_da: bool = True, need_db: bool = True, stream=None):
    """(dx, da, db) of lora() for dy (S, O), its gradient by the result: dx (S, I) of x's type, da (n, R, I) and db (n, O, R)
    float32, zero for adapters that no token names; None in the place of one that is not needed.  v: what lora(save=True)
    returned, needed for db.  The residual's gradient is dy itself.  (zm_lora_backward)"""
    d = _index(dy, "lora_backward")
    if stream is not None or d != _device():
        return _there(lora_backward, d, stream, dy, x, a, b, ids, v, scale, need_dx, need_da, need_db)
    if _grad_mode() and (dy.requires_grad or x.requires_grad or a.requires_grad or b.requires_grad
                         or v is not None and v.requires_grad or scale is not None and scale.requires_grad):
        _not_recorded("lora_backward")
    st = _raw_stream(d)
    ids, scale, (S, I, O, R, n), la, lb = _operands(d, x, a, b, ids, scale)
    x = _rows(x)
    dy = _rows(_need(dy, "dy", d, (_F32, x.dtype), (S, O)))
    if v is not None:
        v = _flat(_need(v, "v", d, _F32S, (S, R)))
    elif need_db:
        raise ValueError("db needs v")
    dx = x.new_empty((S, I)) if need_dx else None
    da = x.new_empty((n, R, I), dtype=_F32) if need_da else None
    db = x.new_empty((n, O, R), dtype=_F32) if need_db else None
    desc = ZmLoraDesc(_TYPES[x.dtype], _TYPES[a.dtype], _TYPES[dy.dtype], n, R, S, I, O, x.stride(0), dy.stride(0), 0, la[1],
                      la[0], lb[1], lb[0])
    L = lib()
    ws = _space(L.zm_lora_backward_workspace_size(desc), x)
    check(L.zm_lora_backward(desc, dy.data_ptr(), x.data_ptr(), a.data_ptr(), b.data_ptr(), ids.data_ptr(), _ptr(scale),
                             _ptr(v), _ptr(dx), _ptr(da), _ptr(db), _ptr(ws), 0 if ws is None else ws.numel(), st),
          "zm_lora_backward")
    return dx, da, db
