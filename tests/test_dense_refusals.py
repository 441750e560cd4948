"""What the dense operators refuse, and the sizes of their workspaces: host code only, no GPU.  The C entry points are
given pointers that are never followed: every call here ends before a launch."""
import ctypes as C

import pytest
import torch

import zeromoe_amd as Z
from zeromoe_amd._lib import ZmLinearDesc, ZmRouterSpec, lib

P = 4096  # an address that nothing reads
F32, F16, BF16, I32 = 0, 1, 30, 26


def desc(**kw):
    d = dict(x_type=F32, w_type=F32, y_type=F32, act=0, S=16, I=64, O=32)
    d.update(kw)
    for name, n in (("x_stride", "I"), ("w_stride", "I"), ("y_stride", "O"), ("res_stride", "O"), ("pre_stride", "O")):
        d.setdefault(name, d[n])
    return ZmLinearDesc(**d)


def error():
    return lib().zm_last_error().decode()


@pytest.mark.parametrize("change,why", [
    (dict(x_type=I32), "types are"), (dict(w_type=12), "types are"), (dict(y_type=14), "types are"),
    (dict(x_type=BF16), "weights of their own type"), (dict(x_type=F16, w_type=BF16), "weights of their own type"),
    (dict(y_type=BF16), "activations' type"), (dict(x_type=F16, w_type=F16, y_type=BF16), "activations' type"),
    (dict(act=-1), "unknown activation"), (dict(act=6), "unknown activation"),
    (dict(S=-1), "S >= 0"), (dict(I=0), "I > 0"), (dict(O=-5), "O > 0"), (dict(S=1 << 31), "below 2\\^31"),
    (dict(I=1 << 40), "below 2\\^31"), (dict(x_stride=-1), "negative stride"), (dict(res_stride=-8), "negative stride"),
    (dict(S=1 << 30, O=1 << 20), "too large"),
])
def test_linear_descriptions(change, why):
    d = desc(**change)
    L = lib()
    import re

    assert L.zm_linear(d, P, P, None, None, P, None, P, 1 << 40, None) == -1 and re.search(why, error())
    assert L.zm_linear_backward(d, P, P, P, P, P, P, P, P, 1 << 40, None) == -1 and re.search(why, error())
    assert L.zm_linear_workspace_size(d) == 0 and L.zm_linear_backward_workspace_size(d) == 0


def test_linear_pointers_strides_and_workspace():
    L = lib()
    assert L.zm_linear(None, P, P, None, None, P, None, None, 0, None) == -1 and "null" in error()
    assert L.zm_linear_backward(None, P, P, P, None, P, P, P, None, 0, None) == -1 and "null" in error()
    for k in (1, 2, 5):
        a = [desc(), P, P, None, None, P, None, None, 0, None]
        a[k] = None
        assert L.zm_linear(*a) == -1 and "null pointer" in error()
    assert L.zm_linear(desc(y_stride=31), P, P, None, None, P, None, None, 0, None) == -1 and "rows of y overlap" in error()
    assert L.zm_linear(desc(pre_stride=0), P, P, None, None, P, P, None, 0, None) == -1 and "rows of pre overlap" in error()
    d = desc(S=512, I=8192, O=64)
    n = L.zm_linear_workspace_size(d)
    assert n > 0 and n % 256 == 0
    for ws, size in ((None, 0), (P, n - 256), (P + 16, n)):
        assert L.zm_linear(d, P, P, None, None, P, None, ws, size, None) == -1 and "workspace" in error()
    d = desc(act=4, S=40)
    n = L.zm_linear_backward_workspace_size(d)
    assert n >= 40 * 32 * 4
    assert L.zm_linear_backward(d, P, P, P, None, P, P, P, P, n, None) == -1 and "needs pre" in error()
    for ws, size in ((None, 0), (P, n - 1), (P + 128, n)):
        assert L.zm_linear_backward(d, P, P, P, P, P, P, P, ws, size, None) == -1 and "workspace" in error()
    assert L.zm_linear_backward(d, None, P, P, P, P, P, P, P, n, None) == -1 and "null pointer" in error()
    assert L.zm_linear_backward(d, P, None, P, P, P, P, P, P, n, None) == -1 and "null pointer" in error()
    assert L.zm_linear_backward(d, P, P, None, P, P, P, P, P, n, None) == -1 and "null pointer" in error()
    # nothing to do
    assert L.zm_linear(desc(S=0), None, None, None, None, None, None, None, 0, None) == 0
    assert L.zm_linear_backward(d, P, P, P, P, None, None, None, None, 0, None) == 0


def test_layer_norm_refusals():
    L = lib()

    def fwd(t=F32, x=P, xs=64, eps=1e-5, rows=4, n=64, y=P, ys=64):
        return L.zm_layer_norm(t, x, xs, None, None, eps, rows, n, y, ys, None, None, None)

    def bwd(t=F32, dy=P, x=P, mean=P, rows=4, n=64, xs=64, gs=64, dx=P, ds=64, ws=P, size=1 << 40):
        return L.zm_layer_norm_backward(t, dy, gs, x, xs, None, mean, P, rows, n, dx, ds, P, P, ws, size, None)

    for call, why in ((lambda: fwd(t=12), "types are"), (lambda: fwd(rows=-1), "rows"), (lambda: fwd(rows=1 << 24), "rows"),
                      (lambda: fwd(n=0), "n is"), (lambda: fwd(n=1 << 25), "n is"), (lambda: fwd(x=None), "null"),
                      (lambda: fwd(y=None), "null"), (lambda: fwd(xs=-1), "stride"), (lambda: fwd(ys=63), "stride"),
                      (lambda: fwd(eps=-1.0), "eps"), (lambda: fwd(eps=float("nan")), "eps"),
                      (lambda: bwd(t=I32), "types are"), (lambda: bwd(rows=-1), "rows"), (lambda: bwd(n=-1), "n is"),
                      (lambda: bwd(dy=None), "null"), (lambda: bwd(x=None), "null"), (lambda: bwd(mean=None), "null"),
                      (lambda: bwd(xs=-1), "stride"), (lambda: bwd(gs=-1), "stride"), (lambda: bwd(ds=10), "stride"),
                      (lambda: bwd(ws=None), "workspace"), (lambda: bwd(ws=P + 4), "workspace"),
                      (lambda: bwd(size=16), "workspace")):
        assert call() == -1 and why in error(), why
    assert fwd(rows=0, x=None) == 0
    assert L.zm_layer_norm_backward_workspace_size(0, 64) == 0
    assert L.zm_layer_norm_backward_workspace_size(5, 64) >= 2 * 64 * 4


def test_combine_refusals():
    L = lib()

    def fwd(y=P, t=256, r=64, w=P, S=4, K=4, H=64, out=P):
        return L.zm_combine(y, t, r, w, None, None, S, K, H, out, None)

    def bwd(d=P, y=P, t=256, r=64, w=P, S=4, K=4, H=64, dw=P, dy=P):
        return L.zm_combine_backward(d, y, t, r, w, None, S, K, H, dw, dy, None)

    for f in (fwd, bwd):
        for kw, why in ((dict(S=-1), "S >= 0"), (dict(K=0), "K"), (dict(K=65), "K"), (dict(H=0), "H > 0"), (dict(y=None), "null"),
                        (dict(S=1 << 24), "too large"), (dict(S=(1 << 24) - 1, K=8), "too large"), (dict(t=-1), "stride"),
                        (dict(r=-64), "stride"), (dict(w=None), "null")):
            assert f(**kw) == -1 and why in error(), kw
        assert f(S=0) == 0
    assert fwd(out=None) == -1 and bwd(d=None) == -1
    assert bwd(dw=None, dy=None) == 0


def test_router_backward_refusals():
    L = lib()

    def call(spec=(0, 64, 4), logits=P, ids=P, dw=P, S=8, out=P):
        s = None if spec is None else ZmRouterSpec(*spec, 0, 0, 0, 0.0)
        return L.zm_router_backward(s, logits, None, ids, dw, None, S, out, None)

    for kw, why in ((dict(spec=None), "null"), (dict(spec=(0, 0, 1)), "n_experts"), (dict(spec=(0, 1025, 1)), "n_experts"),
                    (dict(spec=(0, 64, 0)), "topk"), (dict(spec=(0, 64, 65)), "topk"), (dict(spec=(0, 256, 65)), "topk"),
                    (dict(spec=(3, 64, 4)), "gating"), (dict(spec=(-1, 64, 4)), "gating"), (dict(S=-1), "S out"),
                    (dict(S=1 << 26), "S out"), (dict(logits=None), "null"), (dict(ids=None), "null"), (dict(dw=None), "null"),
                    (dict(out=None), "null")):
        assert call(**kw) == -1 and why in error(), kw
    assert call(S=0, logits=None) == 0


def test_wrappers_refuse_host_tensors():
    x = torch.zeros(2, 4)
    for f, a in ((Z.linear, (x, x)), (Z.linear_backward, (x, x, x)), (Z.layer_norm, (x,)), (Z.layer_norm_backward, (x, x, x, x)),
                 (Z.combine, (x, x)), (Z.combine_backward, (x, x)), (Z.router_backward, (x, x, x))):
        with pytest.raises(ValueError, match="device tensors"):
            f(*a)
