"""The gradients of a whole step, over the C ABI (include/zeromoe.h): their norm, and scaling them down to a largest one.

Device tensors in, device tensors out, on the current stream or on `stream`, with workspaces from torch's allocator: a call
may be captured into a graph and nothing synchronises."""
from __future__ import annotations

import struct

import torch

from ._lib import check, lib
from .dense import _TYPES, _F32, _device, _grad_mode, _index, _not_recorded, _raw_stream, _space, _there


def _dense(t: torch.Tensor) -> bool:
    """Whether t's values fill one piece of memory, each once, in any order of its dimensions."""
    if t.is_contiguous():
        return True
    need = 1
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != need:
            return False
        need *= n
    return True


def _list(grads, who: str):
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if not grads:
        raise ValueError(f"{who}: no gradients")
    return grads, _index(grads[0], who)


def _check(grads, d: int, what: str):
    mode, types = _grad_mode(), _TYPES
    for i, g in enumerate(grads):
        if not isinstance(g, torch.Tensor) or g.get_device() != d:
            raise ValueError(f"{what} {i} is not a tensor of the first one's device")
        if g.dtype not in types:
            raise ValueError(f"{what} {i} is {g.dtype}: float32, float16 or bfloat16 needed")
        if mode and g.requires_grad:
            _not_recorded(what)


def grad_norm(grads, stream=None) -> torch.Tensor:
    """sqrt of the sum of the squares of all values of a list of tensors (float32, float16, bfloat16), summed in float64:
    a float32 tensor of no dimensions.  (zm_grad_norm)"""
    grads, d = _list(grads, "grad_norm")
    if stream is not None or d != _device():
        return _there(grad_norm, d, stream, grads)
    _check(grads, d, "gradient")
    grads = [g if _dense(g) else g.contiguous() for g in grads]
    n = len(grads)
    flat = [v for g in grads for v in (g.data_ptr(), 0, g.numel(), _TYPES[g.dtype], 0)]
    norm = grads[0].new_empty((), dtype=_F32)
    L = lib()
    ws = _space(L.zm_grad_norm_workspace_size(n), norm)
    check(L.zm_grad_norm(struct.pack("=" + "QQqii" * n, *flat), n, norm.data_ptr(), ws.data_ptr(), ws.numel(),
                         _raw_stream(d)), "zm_grad_norm")
    return norm


def clip_grad_norm(grads, max_norm: float, eps: float = 1e-6, out=None, stream=None) -> torch.Tensor:
    """Scales all tensors of a list by min(1, max_norm / (norm + eps)), norm being grad_norm() of the list, and returns
    the norm (before the scaling, float32, on the device).  In place, or into `out`, tensors of the same shapes and
    strides (each of the gradient's type or float32); each gradient fills one piece of memory and overlaps no other.
    In place nothing is written where the norm is small enough.  (zm_grad_clip)"""
    grads, d = _list(grads, "clip_grad_norm")
    if out is not None:
        out = [out] if isinstance(out, torch.Tensor) else list(out)
    if stream is not None or d != _device():
        return _there(clip_grad_norm, d, stream, grads, max_norm, eps, out)
    _check(grads, d, "gradient")
    flat, types = [], _TYPES
    if out is None:
        for i, g in enumerate(grads):
            if not g.is_contiguous() and not _dense(g):
                raise ValueError(f"gradient {i} does not fill one piece of memory: strides {g.stride()} of {tuple(g.shape)}")
            p, k = g.data_ptr(), types[g.dtype]
            flat += (p, p, g.numel(), k, k)
    else:
        _check(out, d, "result")
        if len(out) != len(grads):
            raise ValueError(f"{len(grads)} gradients and {len(out)} results")
        for i, (g, o) in enumerate(zip(grads, out)):
            if g.shape != o.shape or not (g.is_contiguous() and o.is_contiguous()) and g.stride() != o.stride():
                raise ValueError(f"result {i} needs its gradient's shape and strides: {tuple(g.shape)}, {g.stride()}")
            if not g.is_contiguous() and not _dense(g):
                raise ValueError(f"gradient {i} does not fill one piece of memory: strides {g.stride()} of {tuple(g.shape)}")
            if o.dtype != g.dtype and o.dtype != _F32:
                raise ValueError(f"result {i} is {o.dtype}: {g.dtype} or float32 needed")
            flat += (g.data_ptr(), o.data_ptr(), g.numel(), types[g.dtype], types[o.dtype])
    n = len(grads)
    norm = grads[0].new_empty((), dtype=_F32)
    L = lib()
    ws = _space(L.zm_grad_norm_workspace_size(n), norm)
    check(L.zm_grad_clip(struct.pack("=" + "QQqii" * n, *flat), n, max_norm, eps, norm.data_ptr(), ws.data_ptr(), ws.numel(),
                         _raw_stream(d)), "zm_grad_clip")
    return norm
