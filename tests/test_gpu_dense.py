"""The dense operators around the routed layer against their definitions in 64 bits.

Tolerances.  A result's last rounding is eps / 2 of its type.  A sum of n products in f32 is off by at most 2^-24 of
a partial sum at each of its additions; partial sums are below sum |a b| and the roundings' signs are unrelated, so
(4 + 2 sqrt n) 2^-24 sum |a b| covers it (the terms left out of an f32 product are below 2^-26 |a b|).  Where dz
enters a product with fewer bits (see each case) its rounding is added to that."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid"]
U = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def act64(z, act):
    F = torch.nn.functional
    return {"none": lambda v: v, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda v: F.gelu(v, approximate="tanh"),
            "silu": F.silu, "sigmoid": torch.sigmoid}[act](z)


def slope64(z, act):
    z = z.detach().clone().requires_grad_()
    return torch.autograd.grad(act64(z, act).sum(), z)[0]


def rand(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def close(got, want, tol):
    err = (got.double() - want).abs()
    assert got.isfinite().all()
    worst = (err / tol.clamp(min=1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the tolerance"


def sum_tol(n, absdot):
    return U * (4 + 2 * math.sqrt(n)) * absdot + 1e-37  # (and what lies below the smallest normal number)


def linear_tol(x, w, bias, residual, y64, dtype):
    absdot = x.double().abs() @ w.double().abs().t()
    t = sum_tol(x.shape[1], absdot) * 1.2  # no activation here is steeper than 1.13
    if bias is not None:
        t = t + 2 * U * (bias.double().abs() + absdot)
    t = t + 8 * U * (y64.abs() + 1e-3)  # the activation's own functions, a few steps of f32; sums with the residual
    if residual is not None:
        t = t + 2 * U * residual.double().abs()
    return t + half_step(dtype) * y64.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)


def check_linear(S, I, O, xt, wt, act="none", bias=True, residual=True, ydt=None, seed=1, x=None, w=None, out=None):
    import zeromoe_amd as Z

    x = rand(S, I, seed=seed, dtype=TYPES[xt]) if x is None else x
    w = rand(O, I, seed=seed + 1, scale=1 / math.sqrt(I), dtype=TYPES[wt]) if w is None else w
    dtype = TYPES[ydt or xt]
    b = rand(O, seed=seed + 2) if bias else None
    r = rand(S, O, seed=seed + 3, dtype=dtype) if residual else None
    y = Z.linear(x, w, bias=b, act=act, residual=r, out_dtype=dtype, out=out)
    assert y.dtype == dtype and y.shape == (S, O)
    z = x.double() @ w.double().t()
    if bias:
        z = z + b.double()
    y64 = act64(z, act)
    if residual:
        y64 = y64 + r.double()
    close(y, y64, linear_tol(x, w, b, r, y64, dtype))


SHAPES = [(1, 1, 1), (1, 256, 32), (1, 4096, 96), (3, 7, 5), (2, 64, 257), (5, 1000, 31), (8, 512, 128), (9, 264, 100),
          (24, 2048, 160), (33, 96, 129), (64, 1024, 64), (65, 136, 260), (127, 257, 33), (130, 640, 130),
          (300, 72, 1000), (513, 1288, 384)]


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S,I,O", SHAPES)
def test_linear(S, I, O, xt, wt):
    check_linear(S, I, O, xt, wt)
    check_linear(S, I, O, xt, wt, bias=False, residual=False, ydt="f32", seed=11)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("S", [1, 20, 200])
def test_linear_activations(act, S):
    check_linear(S, 320, 200, "f32", "bf16", act)
    check_linear(S, 320, 200, "bf16", "bf16", act, residual=False)


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S", [1, 7, 40, 150])
def test_linear_strides_and_alignment(xt, wt, S):
    """Rows that lie apart, on odd addresses, and a result whose neighbours stay as they are."""
    import zeromoe_amd as Z

    I, O = 264, 72
    for off, pad in ((0, 8), (1, 3), (4, 4)):
        xb = rand(S * (I + pad) + 16, seed=3, dtype=TYPES[xt])
        wb = rand(O * (I + pad) + 16, seed=4, scale=0.06, dtype=TYPES[wt])
        x, w = (b[off:off + n * (I + pad)].view(n, I + pad)[:, :I] for b, n in ((xb, S), (wb, O)))
        yb = torch.full((S + 2, O + pad + off), 7.0, device="cuda", dtype=TYPES[xt])
        check_linear(S, I, O, xt, wt, x=x, w=w, out=yb[1:S + 1, off:off + O])
        keep = torch.ones_like(yb, dtype=torch.bool)
        keep[1:S + 1, off:off + O] = False
        assert (yb[keep] == 7.0).all()
    x = rand(I, S, seed=5, dtype=TYPES[xt]).t()  # columns apart: copied
    check_linear(S, I, O, xt, wt, x=x)
    x = rand(1, I, seed=6, dtype=TYPES[xt]).expand(S, I)  # one row, repeated
    check_linear(S, I, O, xt, wt, x=x)
    with pytest.raises(ValueError, match="contiguous columns"):
        Z.linear(x, rand(I, O, seed=7, dtype=TYPES[wt]).t())


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S", [1, 4, 5, 40, 150])
def test_linear_on_odd_addresses(S, xt, wt):
    """Shapes that allow 16-byte loads on addresses that do not: of x, of w, of the result alone; long rows too."""
    for I, O in ((264, 72), (4104, 40)):
        xb, wb = rand(S * (I + 8) + 16, seed=3, dtype=TYPES[xt]), rand(O * (I + 8) + 16, seed=4, scale=0.06, dtype=TYPES[wt])
        for ox, ow, oy in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (8, 8, 8)):
            x, w = (b[off:off + n * (I + 8)].view(n, I + 8)[:, :I] for b, off, n in ((xb, ox, S), (wb, ow, O)))
            yb = torch.full((S, O + 8), 7.0, device="cuda", dtype=TYPES[xt])
            check_linear(S, I, O, xt, wt, x=x, w=w, out=yb[:, oy:oy + O])
            assert (yb[:, :oy] == 7.0).all() and (yb[:, oy + O:] == 7.0).all()


def test_linear_no_rows_pre_and_in_place():
    import zeromoe_amd as Z

    w = rand(48, 64, seed=1)
    y = Z.linear(torch.empty(0, 64, device="cuda"), w)
    assert y.shape == (0, 48)
    dx, dw, db = Z.linear_backward(y, torch.empty(0, 64, device="cuda"), w)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()
    for S in (1, 30, 140):
        x, b, r = rand(S, 64, seed=2), rand(48, seed=3), rand(S, 48, seed=4)
        want = Z.linear(x, w, bias=b, act="silu", residual=r)
        y, pre = Z.linear(x, w, bias=b, act="silu", residual=r, save_pre=True)
        assert torch.equal(y, want)
        close(pre, x.double() @ w.double().t() + b.double(), sum_tol(64, x.double().abs() @ w.double().abs().t() + b.abs()))
        z = r.clone()
        assert Z.linear(x, w, bias=b, act="silu", residual=z, out=z) is z and torch.equal(z, want)


def test_linear_f32_keeps_its_digits():
    """Values that need all 24 bits, over the whole range of exponents, and values past bf16's largest."""
    import zeromoe_amd as Z

    for S in (2, 40, 140):
        e = torch.randint(-60, 60, (S, 128), device="cuda", generator=torch.Generator("cuda").manual_seed(5))
        x = torch.ldexp(rand(S, 128, seed=6).clamp(-4, 4), e.float())
        for wt in ("f32", "f16", "bf16"):
            w = rand(40, 128, seed=7, dtype=TYPES[wt])
            y = Z.linear(x, w)
            close(y, x.double() @ w.double().t(), sum_tol(128, x.double().abs() @ w.double().abs().t()))
        x = torch.zeros(S, 128, device="cuda")
        x[:, 3] = torch.finfo(torch.float32).max
        x[:, 5] = -torch.finfo(torch.float32).max
        w = torch.zeros(40, 128, device="cuda")
        w[:, 3], w[0, 5] = 0.25, 0.5
        y = Z.linear(x, w)
        close(y, x.double() @ w.double().t(), sum_tol(128, x.double().abs() @ w.double().abs().t()))
        # an infinity or a NaN reaches the results of its row and no other
        x = rand(S, 128, seed=8)
        x[0, 9] = float("inf")
        x[1, 10] = float("nan")
        y = Z.linear(x, rand(40, 128, seed=9))
        assert not y[:2].isfinite().any() and y[2:].isfinite().all()


@pytest.mark.parametrize("S", [2, 40, 200])
def test_linear_smallest_values(S):
    """Subnormal f16 and bf16 values, and f32 values whose last bf16 term is one (steps of 2^-133)."""
    import zeromoe_amd as Z

    for dtype, e in ((torch.float16, -20.0), (torch.bfloat16, -128.0)):
        x = torch.ldexp(rand(S, 128, seed=1), torch.tensor(e, device="cuda")).to(dtype)
        w = (rand(64, 128, seed=2) * (64.0 if dtype == torch.float16 else 2.0 ** 60)).to(dtype)
        y = Z.linear(x, w, out_dtype=torch.float32)
        # (what an instruction adds in one go may be rounded at its largest product's place: up to 32 products)
        close(y, x.double() @ w.double().t(), 8 * sum_tol(128, x.double().abs() @ w.double().abs().t()))
    for e in (-100.0, -115.0, -126.0):
        x, w = torch.ldexp(rand(S, 128, seed=3), torch.tensor(e, device="cuda")), rand(64, 128, seed=4) * 2.0 ** 60
        a = x.double().abs() @ w.double().abs().t()
        lost = 2.0 ** -133 * w.double().abs().sum(1)[None]
        close(Z.linear(x, w), x.double() @ w.double().t(), sum_tol(128, a) + lost)


def test_offsets_past_32_bits():
    """Operands and results of more than 2^31 values: the last rows against the same rows by themselves."""
    import zeromoe_amd as Z

    S, I, O = (1 << 20) + 7, 2056, 40
    x, w = torch.empty(S, I, device="cuda", dtype=torch.bfloat16), rand(O, I, seed=1, scale=0.02, dtype=torch.bfloat16)
    x.copy_(rand(1, I, seed=2).to(torch.bfloat16).expand(S, I))
    x[-300:] = rand(300, I, seed=3, dtype=torch.bfloat16)
    y = Z.linear(x, w, out_dtype=torch.float32)
    z = x[-300:].double() @ w.double().t()
    close(y[-300:], z, sum_tol(I, x[-300:].double().abs() @ w.double().abs().t()))
    h, mean, rstd = Z.layer_norm(x, stats=True)
    assert torch.equal(h[-300:], Z.layer_norm(x[-300:]))
    dy = torch.zeros_like(x)
    dy[-300:] = rand(300, I, seed=4, dtype=torch.bfloat16)
    dx, dw, db = Z.layer_norm_backward(dy, x, mean, rstd)
    ex, ew, eb = Z.layer_norm_backward(dy[-300:], x[-300:], mean[-300:], rstd[-300:])
    assert torch.equal(dx[-300:], ex) and (dx[:-300] == 0).all()
    assert (dw - ew).abs().max() <= 1e-5 * ew.abs().max() and (db - eb).abs().max() <= 1e-5 * eb.abs().max()  # 300 f32 additions
    del h, dy, dx
    dx = Z.linear_backward(y, x, w, need_dw=False, need_dbias=False)[0]
    assert torch.equal(dx[-128:], Z.linear_backward(y[-128 * 3:], x[-128 * 3:], w, need_dw=False, need_dbias=False)[0][-128:])
    del x, y, dx
    S, K, H = 70000, 8, 4100
    r, wt, d = torch.zeros(S, K, H, device="cuda"), rand(S, K, seed=5), rand(S, H, seed=6)
    r[-50:] = rand(50, K, H, seed=7)
    assert torch.equal(Z.combine(r, wt, residual=d)[-50:], Z.combine(r[-50:], wt[-50:], residual=d[-50:]))
    dw, dy = Z.combine_backward(d, r, weights=wt, need_dy=True)
    assert torch.equal(dw[-50:], Z.combine_backward(d[-50:], r[-50:])) and torch.equal(dy[-1, -1], wt[-1, -1] * d[-1])


@pytest.mark.parametrize("S", [3, 40, 200])
def test_linear_rows_far_apart(S):
    """Rows up to 8 MB apart, where 32-bit offsets of a tile end, and further."""
    import zeromoe_amd as Z

    w = rand(24, 72, seed=1)
    for ld in ((1 << 21) - 4, 1 << 21, (1 << 21) + 4):
        x = torch.empty((S - 1) * ld + 72, device="cuda").as_strided((S, 72), (ld, 1))
        x.copy_(rand(S, 72, seed=2))
        assert torch.equal(Z.linear(x[:3], w), Z.linear(x[:3].contiguous(), w))
        close(Z.linear(x, w), x.double() @ w.double().t(), sum_tol(72, x.double().abs() @ w.double().abs().t()))
        dy = rand(S, 24, seed=3)
        dw = Z.linear_backward(dy, x, w, need_dx=False)[1]
        close(dw, dy.double().t() @ x.double(), sum_tol(S, dy.double().abs().t() @ x.double().abs()) + U)
        h = Z.layer_norm(x)
        assert torch.equal(h, Z.layer_norm(x.contiguous()))


def check_linear_backward(S, I, O, xt, wt, act="none", ydt=None, seed=1, need=(True, True, True)):
    import zeromoe_amd as Z

    dtype, yt = TYPES[xt], TYPES[ydt or xt]
    x, w = rand(S, I, seed=seed, dtype=dtype), rand(O, I, seed=seed + 1, scale=1 / math.sqrt(I), dtype=TYPES[wt])
    dy = rand(S, O, seed=seed + 2, scale=0.1, dtype=yt)
    pre = rand(S, O, seed=seed + 3, scale=1.5, dtype=yt) if act != "none" else None
    dx, dw, db = Z.linear_backward(dy, x, w, act=act, pre=pre, need_dx=need[0], need_dw=need[1], need_dbias=need[2])
    assert [t is None for t in (dx, dw, db)] == [not n for n in need]
    dz = dy.double() if act == "none" else dy.double() * slope64(pre.double(), act)
    adz = dz.abs() + (dy.double().abs() * 16 * U if act != "none" else 0)  # the slope in f32
    f32_dz = act != "none" or yt == torch.float32
    # dz's rounding where it enters with fewer bits than it has: one bf16 term for dx next to bf16, two for f16
    cut_x = 0.0 if not f32_dz else {"bf16": 2.0 ** -8, "f16": 2.0 ** -16, "f32": 0.0}[xt]
    slope = 16 * U if act != "none" else 0.0
    if dx is not None:
        want, absdot = dz @ w.double(), adz @ w.double().abs()
        assert dx.dtype == dtype
        close(dx, want, sum_tol(O, absdot) + (cut_x + slope) * absdot + half_step(dtype) * want.abs() + (2.0 ** -25 if xt == "f16" else 0))
    if dw is not None:
        want, absdot = dz.t() @ x.double(), adz.t() @ x.double().abs()
        assert dw.dtype == torch.float32
        close(dw, want, sum_tol(S, absdot) + slope * absdot + half_step(torch.float32) * want.abs())
    if db is not None:
        close(db, dz.sum(0), sum_tol(S, adz.sum(0)) + slope * adz.sum(0))


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S,I,O", [(1, 1, 1), (1, 256, 32), (3, 7, 5), (20, 264, 100), (64, 512, 160), (65, 136, 260),
                                   (127, 257, 33), (300, 72, 1000), (1030, 640, 96)])
def test_linear_backward(S, I, O, xt, wt):
    check_linear_backward(S, I, O, xt, wt)
    check_linear_backward(S, I, O, xt, wt, "silu", seed=21)
    check_linear_backward(S, I, O, xt, wt, ydt="f32", seed=31)


@pytest.mark.parametrize("S,I,O", [(700, 264, 160), (700, 1000, 288), (1100, 2048, 152), (390, 136, 320), (2000, 128, 130)])
def test_linear_narrow_w(S, I, O):
    """f32 products whose w fills tiles of 160 rows better than tiles of 128."""
    check_linear(S, I, O, "f32", "f32", "silu")
    check_linear_backward(S, I, O, "f32", "f32")
    check_linear_backward(S, I, O, "f32", "f32", "gelu")


@pytest.mark.parametrize("S,I,O", [(2100, 40, 2600), (2093, 520, 2603), (2500, 8, 2500), (16493, 264, 157)])
def test_linear_f32_more_tiles_than_cus(S, I, O):
    """More tiles of 128 x 128 than CUs: tiles of one buffer, two on a CU, and tiles of 160 rows of w (the last)."""
    check_linear(S, I, O, "f32", "f32")
    check_linear(S, I, O, "f32", "f32", "gelu", bias=False, residual=False, seed=41)


@pytest.mark.parametrize("S,I,O", [(2100, 2600, 40), (2093, 2604, 520), (2500, 2500, 8), (259, 16516, 156)])
def test_linear_backward_f32_more_tiles_than_cus(S, I, O):
    """The same for the gradients: one buffer by x, tiles of 160 rows by w (the last)."""
    check_linear_backward(S, I, O, "f32", "f32")
    check_linear_backward(S, I, O, "f32", "f32", "silu", seed=21)


@pytest.mark.parametrize("act", ACTS)
def test_linear_backward_activations(act):
    check_linear_backward(70, 96, 56, "f32", "bf16", act)
    check_linear_backward(70, 96, 56, "bf16", "bf16", act, ydt="f32")


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (False, True, True)])
def test_linear_backward_parts(need):
    check_linear_backward(70, 96, 56, "bf16", "bf16", "gelu", need=need)
    check_linear_backward(70, 96, 56, "f32", "f32", need=need)


def test_linear_backward_by_differences():
    """The gradients against differences of the forward pass, where those are exact enough: sums of 64-bit values of
    the formula; and the formula's own slopes far out."""
    import zeromoe_amd as Z

    S, I, O = 3, 12, 5
    x, w, b = rand(S, I, seed=1).double(), rand(O, I, seed=2).double(), rand(O, seed=3).double()
    dy = rand(S, O, seed=4).double()
    for act in ACTS[2:]:
        f = lambda a, c, d: (act64(a @ c.t() + d, act) * dy).sum().item()  # noqa: E731
        pre = (x @ w.t() + b).float()
        dx, dw, db = Z.linear_backward(dy.float(), x.float(), w.float(), act=act, pre=pre)
        h = 1e-5
        for t, g, at in ((x, dx, (1, 3)), (w, dw, (2, 7)), (b, db, (4,))):
            up, down = t.clone(), t.clone()
            up[at] += h
            down[at] -= h
            args = [(up, down)[k] if v is t else v for k in (0, 1) for v in (x, w, b)]
            diff = (f(*args[:3]) - f(*args[3:])) / (2 * h)
            assert abs(g[at].item() - diff) <= 1e-5 * (1 + abs(diff))  # f32 inputs and results; h^2 of the difference
        far = torch.tensor([[-1e30, -300.0, -40.0, 40.0, 300.0, 1e30, -3e38, 3e38]], device="cuda")
        db = Z.linear_backward(torch.ones_like(far), torch.zeros(1, 4, device="cuda"), torch.zeros(8, 4, device="cuda"),
                               act=act, pre=far)[2]
        want = (far > 0).float()[0] if act != "sigmoid" else torch.zeros(8, device="cuda")
        assert (db - want).abs().max() < 1e-6


def test_wrappers_check_their_tensors():
    import zeromoe_amd as Z

    x, w, h = rand(4, 64), rand(8, 64), rand(4, 64).half()
    d = rand(4, 8)
    bad = [lambda: Z.linear(x, rand(8, 63)), lambda: Z.linear(x[0], w), lambda: Z.linear(x.double(), w), lambda: Z.linear(h, w),
           lambda: Z.linear(x, w, bias=rand(7)), lambda: Z.linear(x, w, bias=rand(8).half()), lambda: Z.linear(x, w, act="tanh"),
           lambda: Z.linear(x, w, residual=d.half()), lambda: Z.linear(x, w, residual=rand(8, 4)),
           lambda: Z.linear(x, w, out_dtype=torch.float16), lambda: Z.linear(x, w, out=rand(4, 9)), lambda: Z.linear(x, w.cpu()),
           lambda: Z.linear(x, w, out=rand(8, 4).t()), lambda: Z.linear_backward(d, x, w, act="silu"),
           lambda: Z.linear_backward(d.half(), x, w), lambda: Z.linear_backward(d, x, w, act="relu", pre=d[:3]),
           lambda: Z.linear_backward(rand(5, 8), x, w), lambda: Z.layer_norm(x[0]), lambda: Z.layer_norm(x.int()),
           lambda: Z.layer_norm(x, weight=rand(63)), lambda: Z.layer_norm(x, out=h), lambda: Z.layer_norm(x[:, :0]),
           lambda: Z.layer_norm_backward(h, x, d[:, 0], d[:, 0]), lambda: Z.layer_norm_backward(x, x, rand(3), rand(4)),
           lambda: Z.combine(x, w), lambda: Z.combine(rand(4, 2, 8), rand(4, 3)), lambda: Z.combine(rand(4, 2, 8).half(), rand(4, 2)),
           lambda: Z.combine(rand(4, 2, 8), rand(4, 2), ids=torch.zeros(4, 2, device="cuda", dtype=torch.int64)),
           lambda: Z.combine_backward(rand(4, 8), rand(4, 2, 8), need_dy=True), lambda: Z.combine_backward(rand(4, 9), rand(4, 2, 8)),
           lambda: Z.router_backward(x, torch.zeros(4, 2, device="cuda"), rand(4, 2)),
           lambda: Z.router_backward(x, torch.zeros(3, 2, device="cuda", dtype=torch.int32), rand(4, 2)),
           lambda: Z.router_backward(x, torch.zeros(4, 2, device="cuda", dtype=torch.int32), rand(4, 2), dprobs=rand(63))]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("accepted:", i)
    with pytest.raises(RuntimeError, match="1 <= K"):
        Z.combine(rand(1, 65, 8), rand(1, 65))


# ---------------------------------------------------------------- layer norm


def check_norm(x, weight, bias, eps=1e-5, train=True, out=None):
    import zeromoe_amd as Z

    rows, n = x.shape
    y, mean, rstd = Z.layer_norm(x, weight, bias, eps=eps, stats=True, out=out)
    x64 = x.double().detach().requires_grad_()
    w64 = torch.ones(n, device="cuda", dtype=torch.float64) if weight is None else weight.double()
    b64 = torch.zeros(n, device="cuda", dtype=torch.float64) if bias is None else bias.double()
    w64.requires_grad_()
    b64.requires_grad_()
    y64 = torch.nn.functional.layer_norm(x64, (n,), w64, b64, eps)
    m64 = x64.mean(-1, keepdim=True).detach()
    r64 = 1 / torch.sqrt(x64.detach().var(-1, unbiased=False, keepdim=True) + eps)
    h64 = (x64.detach() - m64) * r64
    # the mean is off by (4 + sqrt n) roundings of mean |x|, and so is every difference from it; rstd by as many of itself
    k = U * (8 + math.sqrt(n))
    shift = x64.detach().abs().mean(-1, keepdim=True) * r64
    htol = k * (shift + h64.abs() * (2 + shift) + 1)
    assert (mean.double() - m64[:, 0]).abs().le(k * x64.detach().abs().mean(-1) + 1e-37).all()
    assert (rstd.double() / r64[:, 0] - 1).abs().le(2 * k * (1 + shift[:, 0])).all()
    y64d = y64.detach()
    small = 2.0 ** -25 if x.dtype == torch.float16 else 0
    close(y, y64d, htol * w64.detach().abs() + 4 * U * (y64d.abs() + b64.detach().abs()) + half_step(x.dtype) * y64d.abs() + small)
    if not train:
        return
    dy = rand(rows, n, seed=77, scale=0.3, dtype=x.dtype)
    dx, dw, db = Z.layer_norm_backward(dy, x, mean, rstd, weight)
    ex, ew, eb = torch.autograd.grad(y64, (x64, w64, b64), dy.double())
    g = (dy.double() * w64.detach()).abs()
    gm, ghm = g.mean(-1, keepdim=True), (g * h64.abs()).mean(-1, keepdim=True)
    tol = r64 * (k * (1 + shift) * 4 * (g + gm + h64.abs() * ghm) + htol * (ghm + g.mean(-1, keepdim=True)))
    close(dx, ex, tol + half_step(x.dtype) * ex.abs() + small)
    a = dy.double().abs()
    close(dw, ew, sum_tol(rows, (a * h64.abs()).sum(0)) + (a * htol).sum(0))
    close(db, eb, sum_tol(rows, a.sum(0)))


@pytest.mark.parametrize("xt", list(TYPES))
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 64), (2, 5), (3, 256), (5, 257), (4, 512), (7, 1000), (9, 1024), (3, 2047),
                                    (6, 2048), (5, 4096), (3, 5120), (2, 7168), (2, 8192), (700, 72), (2, 8200), (2, 20000),
                                    (1500, 264)])
def test_layer_norm(rows, n, xt):
    x = rand(rows, n, seed=1, dtype=TYPES[xt])
    check_norm(x, 1 + 0.3 * rand(n, seed=2), rand(n, seed=3))


@pytest.mark.parametrize("xt", list(TYPES))
def test_layer_norm_strides_far_means_and_constant_rows(xt):
    import zeromoe_amd as Z

    dtype = TYPES[xt]
    for off, pad in ((0, 8), (1, 3)):
        x = rand(6 * (520 + pad) + 16, seed=4, dtype=dtype)[off:off + 6 * (520 + pad)].view(6, 520 + pad)[:, :520]
        check_norm(x, None, None)
        check_norm(x, rand(520, seed=5), None)
        check_norm(x, None, rand(520, seed=5))
    check_norm(rand(520, 6, seed=6, dtype=dtype).t(), rand(520, seed=5), None)
    check_norm((rand(4, 1024, seed=7) + 100.0).to(dtype), None, None)  # a mean far from zero
    x = torch.full((3, 640), 2.5, device="cuda", dtype=dtype)  # no variance: h = 0, dx = rstd (g - mean g)
    check_norm(x, rand(640, seed=8), rand(640, seed=9))
    y = Z.layer_norm(torch.zeros(2, 8, device="cuda", dtype=dtype), eps=0.0)
    assert y.isnan().all()  # 0 / 0, as the formula has it
    x = rand(5, 300, seed=10, dtype=dtype)
    want = Z.layer_norm(x)
    assert Z.layer_norm(x, out=x) is x and torch.equal(x, want)
    e = torch.empty(0, 16, device="cuda", dtype=dtype)
    y, mean, rstd = Z.layer_norm(e, stats=True)
    dx, dw, db = Z.layer_norm_backward(y, e, mean, rstd)
    assert dx.shape == (0, 16) and (dw == 0).all() and (db == 0).all()
    buf = torch.full((5, 40), 7.0, device="cuda", dtype=dtype)
    Z.layer_norm(rand(3, 32, seed=11, dtype=dtype), out=buf[1:4, :32])
    assert (buf[0] == 7).all() and (buf[4] == 7).all() and (buf[:, 32:] == 7).all()


def test_layer_norm_backward_parts():
    import zeromoe_amd as Z

    x, dy = rand(9, 96, seed=1), rand(9, 96, seed=2)
    _, mean, rstd = Z.layer_norm(x, stats=True)
    dx, dw, db = Z.layer_norm_backward(dy, x, mean, rstd)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        got = Z.layer_norm_backward(dy, x, mean, rstd, need_dx=need[0], need_dweight=need[1], need_dbias=need[2])
        for g, n, w in zip(got, need, (dx, dw, db)):
            assert (g is None) if not n else torch.equal(g, w)


# ---------------------------------------------------------------- weighted sum


@pytest.mark.parametrize("S,K,H", [(1, 1, 1), (1, 8, 4096), (3, 2, 5), (24, 8, 7168), (7, 10, 1027), (65, 6, 2048), (2, 64, 260),
                                   (1000, 4, 36)])
def test_combine(S, K, H):
    import zeromoe_amd as Z

    y, w, r, d = rand(S, K, H, seed=1), rand(S, K, seed=2), rand(S, H, seed=3), rand(S, H, seed=4)
    ids = torch.randint(-1, 3, (S, K), device="cuda", dtype=torch.int32, generator=torch.Generator("cuda").manual_seed(5))
    if S > 2:
        ids[1] = -1  # a row without a route
    for use in (ids, None):
        on = torch.ones(S, K, device="cuda", dtype=torch.bool) if use is None else use >= 0
        yy = torch.where(on[:, :, None], y, torch.full_like(y, float("nan")))  # what is not read
        w64, y64 = torch.where(on, w, torch.zeros_like(w)).double(), torch.where(on[:, :, None], y, torch.zeros_like(y)).double()
        absum = (w64[:, :, None] * y64).abs().sum(1)
        for res in (r, None):
            want = (w64[:, :, None] * y64).sum(1) + (0 if res is None else res.double())
            close(Z.combine(yy, w, ids=use, residual=res), want, sum_tol(2 * K, absum + (0 if res is None else res.abs())))
        out = r.clone()
        assert Z.combine(yy, w, ids=use, residual=out, out=out) is out
        assert torch.equal(out, Z.combine(yy, w, ids=use, residual=r))
        dw, dy = Z.combine_backward(d, yy, weights=w, ids=use, need_dy=True)
        close(dw, (y64 * d.double()[:, None]).sum(-1), sum_tol(H, (y64 * d.double()[:, None]).abs().sum(-1)))
        assert torch.equal(dy, torch.where(on[:, :, None], w[:, :, None] * d[:, None], torch.zeros_like(y)))
        assert torch.equal(Z.combine_backward(d, yy, ids=use), dw)


def test_combine_strides():
    import zeromoe_amd as Z

    for off, H in ((0, 64), (1, 63)):
        base = rand(6, 5, 72, seed=1)
        y, w, d = base[::2, 1:4, off:off + H], rand(3, 3, seed=2), rand(3, H, seed=3)
        assert torch.equal(Z.combine(y, w), Z.combine(y.contiguous(), w))
        assert torch.equal(Z.combine_backward(d, y), Z.combine_backward(d, y.contiguous()))
    y = rand(1, 1, 64, seed=4).expand(5, 3, 64)
    assert torch.equal(Z.combine(y, rand(5, 3, seed=5)), Z.combine(y.contiguous(), rand(5, 3, seed=5)))
    assert Z.combine(rand(0, 3, 8), rand(0, 3)).shape == (0, 8)
    assert Z.combine_backward(rand(0, 8), rand(0, 3, 8)).shape == (0, 3)


# ---------------------------------------------------------------- gradient of the routing


def gate64(z, gating):
    if gating == "softmax":
        return torch.softmax(z, -1)
    if gating == "sigmoid":
        return torch.sigmoid(z)
    return torch.nn.functional.softplus(z, threshold=1e9).sqrt()


def route_grad64(logits, ids, dw, gating, bias, norm, scale, dprobs):
    z = logits.double().requires_grad_()
    p = gate64(z if bias is None else z + bias.double(), gating)
    on = (ids >= 0).double()
    w = p.gather(1, ids.clamp(min=0).long()) * on
    if norm:
        w = w / w.sum(-1, keepdim=True).clamp(min=2.0 ** -14)
    loss = (w * torch.where(ids >= 0, dw, torch.zeros_like(dw)).double()).sum() * (scale or 1.0)
    if dprobs is not None:
        loss = loss + ((p * dprobs.double()).sum(-1) * on.amax(-1)).sum()
    return torch.autograd.grad(loss, z)[0]


@pytest.mark.parametrize("gating", ["softmax", "sigmoid", "sqrt_softplus"])
@pytest.mark.parametrize("S,E,K", [(1, 1, 1), (1, 128, 8), (3, 5, 2), (65, 60, 4), (17, 160, 8), (50, 256, 8), (9, 384, 10),
                                   (6, 1000, 64), (5, 1024, 1)])
def test_router_backward(S, E, K, gating):
    import zeromoe_amd as Z

    logits, bias, sel = rand(S, E, seed=1, scale=2.0), rand(E, seed=2, scale=0.3), rand(E, seed=3, scale=0.05)
    for norm, scale, lb, dp in ((False, 0.0, None, None), (True, 2.5, bias, None), (True, 0.0, None, rand(E, seed=4)),
                                (False, 1.5, bias, rand(E, seed=5))):
        ids, w = Z.router(logits, K, gating=gating, logit_bias=lb, sel_bias=sel, weights_norm=norm, weights_scale=scale)
        if S > 2:
            ids[1] = -1          # a padding row
            ids[2, 0] = -1       # one route left out
        dw = rand(S, K, seed=6)
        got = Z.router_backward(logits, ids, dw, gating=gating, logit_bias=lb, weights_norm=norm, weights_scale=scale, dprobs=dp)
        want = route_grad64(logits, ids, dw, gating, lb, norm, scale, dp)
        # p g and sum p g are off by a few roundings of sums over E and K values and of exp's argument (|z| below 16)
        p = gate64(logits.double() + (0 if lb is None else lb.double()), gating)
        big = dw.abs().double().sum(-1, keepdim=True) * (scale or 1.0)
        if norm:
            total = (p.gather(1, ids.clamp(min=0).long()) * (ids >= 0)).sum(-1, keepdim=True).clamp(min=2.0 ** -14)
            big = 2 * big / total
        if dp is not None:
            big = big + dp.abs().double() + (p * dp.abs().double()).sum(-1, keepdim=True)
        close(got, want, U * (40 + 2 * math.sqrt(E) + 2 * math.sqrt(K)) * big * p.clamp(min=1e-6) * 2 + 1e-37)
        if S > 2:
            assert (got[1] == 0).all()


@pytest.mark.parametrize("gating", ["softmax", "sigmoid", "sqrt_softplus"])
def test_router_backward_masked_logits_and_odd_ids(gating):
    import zeromoe_amd as Z

    E, K = 100, 4
    logits = rand(7, E, seed=1)
    logits[0, 10:] = -float("inf")
    logits[1, 10:] = torch.finfo(torch.float32).min
    logits[2] = -float("inf")
    logits[3] = -200.0
    logits[5, :50] = 80.0
    ids = torch.stack([torch.randperm(10, generator=torch.Generator().manual_seed(s))[:K] for s in range(7)]).int().cuda()
    dw = rand(7, K, seed=2)
    dw[6, 1] = float("nan")
    ids[6, 1] = -1  # a left-out route's NaN goes nowhere
    ids[4] = ids[4, 0]  # one expert four times
    for norm in (False, True):
        got = Z.router_backward(logits, ids, dw, gating=gating, weights_norm=norm)
        assert got.isfinite().all()
        assert (got[0, 10:] == 0).all() and (got[1, 10:] == 0).all() and (got[2] == 0).all()
        keep = [0, 1, 4, 5, 6]
        safe = logits.clone()
        safe[0, 10:] = safe[1, 10:] = -600.0  # far enough for 64 bits, and the oracle's square root still has a slope
        want = route_grad64(safe, ids, dw, gating, None, norm, 0.0, None)
        tol = 1e-5 * (1 + want.abs().amax(-1, keepdim=True))  # 150 roundings of the largest value
        assert ((got.double() - want).abs() <= tol)[keep].all()
    ids[0, 0], ids[1, 2] = E, 2 ** 31 - 1
    got = Z.router_backward(logits, ids, dw, gating=gating)
    assert got[:2].isnan().all() and got[2:].isfinite().all()


@pytest.mark.parametrize("gating", ["sigmoid", "sqrt_softplus"])
def test_router_backward_small_sums(gating):
    """Weights whose sum is below the least that they are divided by: the divisor is a constant there."""
    import zeromoe_amd as Z

    logits = rand(6, 40, seed=1) - (13.0 if gating == "sigmoid" else 25.0)
    ids = torch.topk(logits, 4)[1].int()
    dw = rand(6, 4, seed=2)
    got = Z.router_backward(logits, ids, dw, gating=gating, weights_norm=True, weights_scale=2.0)
    want = route_grad64(logits, ids, dw, gating, None, True, 2.0, None)
    p = gate64(logits.double(), gating)
    total = p.gather(1, ids.long()).sum(-1, keepdim=True)
    assert (total < 2.0 ** -14).any()
    # exp's argument is up to 28 (its rounding is 28 of the result's), then a few roundings of d and sum d p / N
    close(got, want, 60 * U * p * 4 * dw.abs().double().sum(-1, keepdim=True) / total.clamp(min=2.0 ** -14) + 1e-37)


def test_router_backward_by_differences():
    """Against differences of router()'s own weights for one selection, in 64 bits of the formula."""
    import zeromoe_amd as Z

    logits = rand(2, 12, seed=1)
    dw = rand(2, 3, seed=2)
    for gating in ("softmax", "sigmoid", "sqrt_softplus"):
        ids, w = Z.router(logits, 3, gating=gating, weights_norm=True, weights_scale=2.0)
        got = Z.router_backward(logits, ids, dw, gating=gating, weights_norm=True, weights_scale=2.0)

        def f(z):
            p = gate64(z, gating).gather(1, ids.long())
            return (2.0 * p / p.sum(-1, keepdim=True) * dw.double()).sum().item()

        z = logits.double()
        p = gate64(z, gating).gather(1, ids.long())
        assert (w.double() - 2.0 * p / p.sum(-1, keepdim=True)).abs().max() < 1e-6  # the forward pass is this formula
        for at in ((0, int(ids[0, 0])), (1, int(ids[1, 2])), (1, 11)):
            up, down = z.clone(), z.clone()
            up[at] += 1e-5
            down[at] -= 1e-5
            diff = (f(up) - f(down)) / 2e-5
            assert abs(got[at].item() - diff) < 1e-6 * (1 + dw.abs().sum().item())  # f32 results; 1e-10 of the difference


# ---------------------------------------------------------------- streams, graphs, repeats


def all_calls(seed, S=70):
    """One call of each operator on inputs of its own; the outputs as a list."""
    import zeromoe_amd as Z

    x, w, dy = rand(S, 520, seed=seed, dtype=torch.bfloat16), rand(96, 520, seed=seed + 1, dtype=torch.bfloat16), rand(S, 96, seed=seed + 2, dtype=torch.bfloat16)
    pre, xf, wf = rand(S, 96, seed=seed + 3, dtype=torch.bfloat16), rand(S, 2056, seed=seed + 4), rand(40, 2056, seed=seed + 5)
    logits, dwt = rand(S, 40, seed=seed + 6), rand(S, 4, seed=seed + 7)
    y, wt, d = rand(S, 4, 256, seed=seed + 8), rand(S, 4, seed=seed + 9), rand(S, 256, seed=seed + 10)
    ids = Z.router(logits, 4)[0]

    def call(stream=None):
        k = dict(stream=stream)
        out = [Z.linear(x, w, act="gelu", **k), Z.linear(xf, wf, **k), Z.linear(xf[:1], wf, **k), Z.linear(xf[:20], wf, **k),
               *Z.linear_backward(dy, x, w, act="silu", pre=pre, **k), *Z.layer_norm(x, stats=True, **k)]
        out += Z.layer_norm_backward(x, x, out[-2], out[-1], **k)
        out += [Z.combine(y, wt, **k), *Z.combine_backward(d, y, weights=wt, need_dy=True, **k),
                Z.router_backward(logits, ids, dwt, **k)]
        return out
    return call


def test_calls_repeat_their_bits_on_any_stream():
    call = all_calls(1)
    want = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [call(stream=s) for s in streams for _ in range(2)]
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_two_graphs_replayed_together():
    """Two captured graphs, each with its own workspaces, replayed on two streams at once and again behind other work."""
    calls = [all_calls(1), all_calls(100)]
    want = [c() for c in calls]
    graphs, outs = [], []
    for c in calls:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            c()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c())
        graphs.append(g)
    for _ in range(4):
        for o in outs:
            for t in o:
                t.fill_(float("nan"))
        all_calls(200)()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w))


# ---------------------------------------------------------------- together


def test_router_step_over_frozen_experts():
    """norm -> router product -> routing -> quantized experts -> weighted sum, and the gradients of norm and router, the
    experts' rows held fixed: as a step does that fits a router to quantized experts."""
    import zeromoe_amd as Z
    import zm_oracle as O

    Z.init()
    S, H, F, E, K = 37, 512, 256, 24, 4
    t = O.TYPE_Q4_K
    wg, wu, wd = (torch.from_numpy(O.random_blocks(t, E * r, n, seed=s).reshape(E, r, -1)).cuda()
                  for r, n, s in ((F, H, 1), (F, H, 2), (H, F, 3)))
    x, gain, shift = rand(S, H, seed=4), 1 + 0.1 * rand(H, seed=5), 0.1 * rand(H, seed=6)
    wr, br = rand(E, H, seed=7, scale=0.05).to(torch.bfloat16), rand(E, seed=8, scale=0.1)
    sel = rand(E, seed=9, scale=0.02)
    dout = rand(S, H, seed=10, scale=0.1)

    h, mean, rstd = Z.layer_norm(x, gain, shift, stats=True)
    logits = Z.linear(h, wr, bias=br)
    ids, w = Z.router(logits, K, gating="sigmoid", sel_bias=sel, weights_norm=True, weights_scale=2.5)
    g = Z.mul_mat_id(wg, t, H, h.view(S, 1, H), ids)
    u = Z.mul_mat_id(wu, t, H, h.view(S, 1, H), ids)
    y = Z.mul_mat_id(wd, t, F, Z.swiglu(g, u), ids)
    out = Z.combine(y, w, ids=ids, residual=x)

    dweights = Z.combine_backward(dout, y, ids=ids)
    dlogits = Z.router_backward(logits, ids, dweights, gating="sigmoid", weights_norm=True, weights_scale=2.5)
    dh, dwr, dbr = Z.linear_backward(dlogits, h, wr)
    dx, dgain, dshift = Z.layer_norm_backward(dh, x, mean, rstd, gain)
    dx = dx + dout  # the residual's

    p = [v.double().requires_grad_() for v in (x, gain, shift, wr.float(), br)]
    h64 = torch.nn.functional.layer_norm(p[0], (H,), p[1], p[2], 1e-5)
    probs = torch.sigmoid(h64 @ p[3].t() + p[4]).gather(1, ids.long())
    w64 = probs / probs.sum(-1, keepdim=True) * 2.5
    out64 = p[0] + (w64[:, :, None] * y.double()).sum(1)
    want = torch.autograd.grad(out64, p, dout.double())
    # each step's own bound is tested above; through the chain f32 roundings stay below 2^-24 times some thousand
    # additions of the largest values: 1e-4 of a tensor's own size
    assert ((out.double() - out64).norm() / out64.norm()).item() < 1e-5
    for got, ref in zip((dx, dgain, dshift, dwr, dbr), want):
        assert ((got.double() - ref).norm() / ref.norm()).item() < 1e-4


def test_decode_block_in_one_graph():
    """One token: norm, router product and the routed layer, with a shared expert in 16-bit weights added behind it,
    captured and replayed against the plain calls."""
    import zeromoe_amd as Z
    import zm_oracle as O

    Z.init()
    H, F, E, K = 512, 256, 16, 4
    t = O.TYPE_Q4_K
    wg, wu, wd = (torch.from_numpy(O.random_blocks(t, E * r, n, seed=s).reshape(E, r, -1)).cuda()
                  for r, n, s in ((F, H, 1), (F, H, 2), (H, F, 3)))
    L = Z.MoELayer(H=H, F=F, n_experts=E, topk=K, type_gate=t, type_up=t, type_down=t, w_gate=wg, w_up=wu, w_down=wd)
    x, wr = rand(1, H, seed=4), rand(E, H, seed=5, scale=0.05)
    sg, su, sd = (rand(r, n, seed=s, scale=0.05, dtype=torch.bfloat16) for r, n, s in ((F, H, 6), (F, H, 7), (H, F, 8)))

    def block():
        h = Z.layer_norm(x)
        out = L.forward(h, Z.linear(h, wr))[0]
        a = Z.swiglu(Z.linear(h, sg), Z.linear(h, su))
        return Z.linear(a, sd, residual=Z.combine(out.view(1, 1, H), torch.ones(1, 1, device="cuda"), residual=x))

    want = block()
    torch.cuda.synchronize()
    h = torch.nn.functional.layer_norm(x.double(), (H,))
    shared = (torch.nn.functional.silu(h @ sg.double().t()) * (h @ su.double().t())) @ sd.double().t()
    routed = L.forward(Z.layer_norm(x), Z.linear(Z.layer_norm(x), wr))[0].double()
    assert ((want.double() - (x.double() + routed + shared)).abs().max() < 1e-4 * want.abs().max().item())  # sums of f32
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = block()
    for _ in range(3):
        got.fill_(float("nan"))
        block()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert L.status(1) == 0
