"""What the gated product, the adapters and the gradient clipping refuse, and their workspaces: host code only, no GPU.  The C
entry points are given pointers that are never followed: every call here ends before a launch."""
import struct

import pytest
import torch

import zeromoe_amd as Z
from zeromoe_amd._lib import ZmGluDesc, ZmLoraDesc, lib

P = 4096  # an address that nothing reads
F32, F16, BF16, I32 = 0, 1, 30, 26


def error():
    return lib().zm_last_error().decode()


def glu_desc(**kw):
    d = dict(x_type=F32, w_type=F32, y_type=F32, act=4, S=16, I=64, F=32)
    d.update(kw)
    for name, n in (("x_stride", "I"), ("w_stride", "I"), ("y_stride", "F"), ("gate_stride", "F"), ("up_stride", "F")):
        d.setdefault(name, d[n])
    return ZmGluDesc(**d)


@pytest.mark.parametrize("change,why", [
    (dict(x_type=I32), "types are"), (dict(w_type=12), "types are"), (dict(y_type=14), "types are"),
    (dict(x_type=BF16), "weights of their own type"), (dict(x_type=F16, w_type=BF16), "weights of their own type"),
    (dict(y_type=BF16), "activations' type"), (dict(act=-1), "unknown activation"), (dict(act=6), "unknown activation"),
    (dict(S=-1), "S >= 0"), (dict(I=0), "I > 0"), (dict(F=0), "F from 1"), (dict(F=1 << 30), "F from 1"),
    (dict(S=1 << 31), "below 2^31"), (dict(I=1 << 40), "below 2^31"), (dict(x_stride=-1), "negative stride"),
    (dict(w_stride=-1), "negative stride"), (dict(up_stride=-8), "negative stride"), (dict(S=1 << 29, F=1 << 20), "too large"),
])
def test_glu_descriptions(change, why):
    d, L = glu_desc(**change), lib()
    assert L.zm_glu(d, P, P, P, None, None, P, None, None, P, 1 << 40, None) == -1 and why in error()
    assert L.zm_glu_backward(d, P, P, P, P, P, P, P, P, P, P, 1 << 40, None) == -1 and why in error()
    assert L.zm_glu_workspace_size(d) == 0 and L.zm_glu_backward_workspace_size(d) == 0


def test_glu_pointers_strides_and_workspace():
    L = lib()
    assert L.zm_glu(None, P, P, P, None, None, P, None, None, None, 0, None) == -1 and "null" in error()
    assert L.zm_glu_backward(None, P, P, P, P, P, P, P, P, P, None, 0, None) == -1 and "null" in error()
    for k in (1, 2, 3, 6):
        a = [glu_desc(), P, P, P, None, None, P, None, None, None, 0, None]
        a[k] = None
        assert L.zm_glu(*a) == -1 and "null pointer" in error()
    for k in (7, 8):
        a = [glu_desc(), P, P, P, None, None, P, P, P, None, 0, None]
        a[k] = None
        assert L.zm_glu(*a) == -1 and "together" in error()
    a = (P, P, P, None, None, P, P, P, P, 1 << 40, None)
    for kw, what in ((dict(y_stride=31), "y"), (dict(gate_stride=0), "gate"), (dict(up_stride=1), "up")):
        assert L.zm_glu(glu_desc(**kw), *a) == -1 and f"rows of {what} overlap" in error()
    d = glu_desc(S=512, I=8192, F=64)
    n = L.zm_glu_workspace_size(d)
    assert n > 0 and n % 256 == 0
    for ws, size in ((None, 0), (P, n - 256), (P + 16, n)):
        assert L.zm_glu(d, P, P, P, None, None, P, None, None, ws, size, None) == -1 and "workspace" in error()
    d = glu_desc(S=40)
    n = L.zm_glu_backward_workspace_size(d)
    assert n >= 40 * 64 * 4
    for ws, size in ((None, 0), (P, n - 1), (P + 128, n)):
        assert L.zm_glu_backward(d, P, P, P, P, P, P, P, P, P, ws, size, None) == -1 and "workspace" in error()
    for k in range(1, 7):
        a = [d, P, P, P, P, P, P, P, P, P, P, n, None]
        a[k] = None
        assert L.zm_glu_backward(*a) == -1 and "null pointer" in error()
    # nothing to do
    assert L.zm_glu(glu_desc(S=0), None, None, None, None, None, None, None, None, None, 0, None) == 0
    assert L.zm_glu_backward(d, P, P, P, P, P, P, None, None, None, None, 0, None) == 0
    assert L.zm_glu_workspace_size(glu_desc(S=0)) == 0 and L.zm_glu_backward_workspace_size(glu_desc(S=0)) == 0


def lora_desc(**kw):
    d = dict(x_type=F32, w_type=F32, y_type=F32, n=4, R=8, S=16, I=64, O=32)
    d.update(kw)
    for name, n in (("x_stride", d["I"]), ("y_stride", d["O"]), ("res_stride", d["O"]), ("a_stride", d["I"]),
                    ("a_adapter", d["I"] * d["R"]), ("b_stride", d["R"]), ("b_adapter", d["R"] * d["O"])):
        d.setdefault(name, n)
    return ZmLoraDesc(**d)


BIG = dict(S=20000)  # past what one launch does without a workspace


@pytest.mark.parametrize("change,why", [
    (dict(x_type=I32), "types are"), (dict(w_type=12), "types are"), (dict(y_type=14), "types are"),
    (dict(x_type=BF16), "adapters of their own type"), (dict(x_type=F16, w_type=BF16), "adapters of their own type"),
    (dict(y_type=BF16), "activations' type"), (dict(n=0), "1 to 512 adapters"), (dict(n=513), "1 to 512 adapters"),
    (dict(R=0), "rank of 1 to 256"), (dict(R=257), "rank of 1 to 256"), (dict(S=-1), "S from 0"), (dict(S=1 << 24), "S from 0"),
    (dict(I=0), "I and O"), (dict(O=-3), "I and O"), (dict(I=1 << 30), "I and O"), (dict(x_stride=-1), "negative stride"),
    (dict(a_adapter=-1), "negative stride"), (dict(b_stride=-1), "negative stride"), (dict(a_stride=1 << 27), "below 2^31 bytes"),
    (dict(b_stride=1 << 26), "below 2^31 bytes"), (dict(n=512, R=1, I=1 << 27), "too large"),
])
def test_lora_descriptions(change, why):
    d, L = lora_desc(**change), lib()
    assert L.zm_lora(d, P, P, P, P, None, None, P, None, P, 1 << 40, None) == -1 and why in error()
    assert L.zm_lora_backward(d, P, P, P, P, P, None, P, P, P, P, P, 1 << 40, None) == -1 and why in error()
    assert L.zm_lora_workspace_size(d) == 0 and L.zm_lora_backward_workspace_size(d) == 0


@pytest.mark.parametrize("change", [dict(R=5, a_stride=1 << 62), dict(O=33, b_stride=1 << 59), dict(R=3, a_stride=(1 << 63) - 1)])
def test_lora_strides_whose_extent_passes_64_bits(change):
    d, L = lora_desc(**change), lib()
    assert L.zm_lora_workspace_size(d) == 0 and "below 2^31 bytes" in error()
    assert L.zm_lora_backward_workspace_size(d) == 0 and "below 2^31 bytes" in error()
    assert L.zm_lora(d, P, P, P, P, None, None, P, None, P, 1 << 40, None) == -1 and "below 2^31 bytes" in error()
    assert L.zm_lora_backward(d, P, P, P, P, P, None, P, P, P, P, P, 1 << 40, None) == -1 and "below 2^31 bytes" in error()
    one = lora_desc(R=1, a_stride=1 << 62, a_adapter=64, S=20000)  # (a single row has no stride)
    assert L.zm_lora_workspace_size(one) > 0


def test_lora_pointers_strides_and_workspace():
    L = lib()
    assert L.zm_lora(None, P, P, P, P, None, None, P, None, P, 0, None) == -1 and "null" in error()
    assert L.zm_lora_backward(None, P, P, P, P, P, None, P, P, P, P, P, 0, None) == -1 and "null" in error()
    for size in ({}, BIG):
        for k in (1, 2, 3, 4, 7):
            a = [lora_desc(**size), P, P, P, P, None, None, P, None, P, 1 << 40, None]
            a[k] = None
            assert L.zm_lora(*a) == -1 and "null pointer" in error()
        assert L.zm_lora(lora_desc(y_stride=31, **size), P, P, P, P, None, None, P, None, P, 1 << 40, None) == -1
        assert "rows of y overlap" in error()
        assert L.zm_lora(lora_desc(res_stride=40, **size), P, P, P, P, None, P, P, None, P, 1 << 40, None) == -1
        assert "has y's stride" in error()
    assert L.zm_lora_workspace_size(lora_desc()) == 0  # few tokens: none
    d = lora_desc(**BIG)
    n = L.zm_lora_workspace_size(d)
    assert n >= 20000 * 4 and n % 256 == 0
    for ws, size in ((None, 0), (P, n - 1), (P + 16, n)):
        assert L.zm_lora(d, P, P, P, P, None, None, P, None, ws, size, None) == -1 and "workspace" in error()
    for d in (lora_desc(), lora_desc(**BIG)):
        n = L.zm_lora_backward_workspace_size(d)
        assert n >= d.S * d.R * 4
        for ws, size in ((None, 0), (P, n - 1), (P + 64, n)):
            assert L.zm_lora_backward(d, P, P, P, P, P, None, P, P, P, P, ws, size, None) == -1 and "workspace" in error()
        for k in (1, 2, 3, 4, 5, 7):
            a = [d, P, P, P, P, P, None, P, P, P, P, P, n, None]
            a[k] = None
            assert L.zm_lora_backward(*a) == -1 and "null pointer" in error()
        assert L.zm_lora_backward(d, P, P, P, P, P, None, P, None, None, None, None, 0, None) == 0
    assert L.zm_lora(lora_desc(S=0), None, None, None, None, None, None, None, None, None, 0, None) == 0


def grads(*rows):
    return struct.pack("=" + "QQqii" * len(rows), *[v for r in rows for v in r])


def test_clip_refusals():
    L = lib()
    n = L.zm_grad_norm_workspace_size(2)
    assert n > 0 and n % 256 == 0 and L.zm_grad_norm_workspace_size(-1) == 0 and L.zm_grad_norm_workspace_size(1 << 24) == 0

    def norm(g, k, out=P, ws=P, size=1 << 40):
        return L.zm_grad_norm(g, k, out, ws, size, None)

    def clip(g, k, m=1.0, e=1e-6, ws=P, size=1 << 40):
        return L.zm_grad_clip(g, k, m, e, P, ws, size, None)

    ok = grads((P, P, 100, F32, F32), (8192, 8192, 100, F16, F16))
    for g, k, why in ((None, 1, "a list"), (ok, -1, "a list"), (ok, 1 << 24, "a list"),
                      (grads((P, P, 10, I32, F32)), 1, "types are"), (grads((P, P, -1, F32, F32)), 1, "possible size"),
                      (grads((P, P, 1 << 43, F32, F32)), 1, "possible size"), (grads((0, P, 10, F32, F32)), 1, "null pointer"),
                      (grads(*[(P, P, (1 << 42) - 1, F32, F32)] * 3), 3, "too many values")):
        assert norm(g, k) == -1 and why in error(), why
        assert clip(g, k) == -1 and why in error(), why
    for g, k, why in ((grads((P, P, 10, F32, 12)), 1, "types are"), (grads((P, 0, 10, F32, F32)), 1, "null pointer"),
                      (grads((P, P, 10, F16, F32)), 1, "keeps its type"),
                      (grads((P, P, 10, F32, F32), (P, P, 10, F32, F32)), 2, "overlaps"),
                      (grads((P, P, 10, F32, F32), (P + 36, P + 36, 10, F32, F32)), 2, "overlaps"),
                      (grads((P, P + 8, 10, F32, F32)), 1, "overlaps"),
                      (grads((P, 8192, 10, F32, F32), (16384, 8192 + 20, 10, BF16, BF16)), 2, "overlaps"),
                      (grads((P, 8192, 10, F32, F32), (8192 + 20, 16384, 10, BF16, BF16)), 2, "overlaps")):
        assert clip(g, k) == -1 and why in error(), why
    for m, e in ((-1.0, 0.0), (float("nan"), 0.0), (1.0, -1e-9), (1.0, float("inf")), (1.0, float("nan"))):
        assert clip(ok, 2, m, e) == -1 and "max_norm" in error()
    assert norm(ok, 2, out=None) == -1 and "null" in error()
    for ws, size in ((None, 0), (P, n - 1), (P + 8, n)):
        assert norm(ok, 2, ws=ws, size=size) == -1 and "workspace" in error()
        assert clip(ok, 2, ws=ws, size=size) == -1 and "workspace" in error()


def test_norm_in_the_place_of_a_gradient():
    L = lib()
    size = L.zm_grad_norm_workspace_size(2)
    for g in ((P, P, 10, F32, F32), (P, 65536, 10, F32, F32), (65536, P, 10, F32, F32), (P, 65536, 20, BF16, BF16)):
        for norm in (P - 3, P, P + 36, P + 39):
            assert L.zm_grad_clip(grads((8192, 8192, 5, F32, F32), g), 2, 1.0, 1e-6, norm, 1 << 20, size, None) == -1
            assert "norm overlaps" in error()


def test_wrappers_refuse_host_tensors():
    x, a = torch.zeros(2, 4), torch.zeros(1, 2, 4)
    ids = torch.zeros(2, dtype=torch.int32)
    for f, args in ((Z.glu, (x, x, x)), (Z.glu_backward, (x, x, x, x, x, x)), (Z.lora, (x, a, a, ids)),
                    (Z.lora_backward, (x, x, a, a, ids)), (Z.grad_norm, ([x],)), (Z.grad_norm, (x,)),
                    (Z.clip_grad_norm, ([x], 1.0))):
        with pytest.raises(ValueError, match="device tensors"):
            f(*args)
    for f, args in ((Z.grad_norm, ([],)), (Z.clip_grad_norm, ([], 1.0))):
        with pytest.raises(ValueError, match="no gradients"):
            f(*args)
