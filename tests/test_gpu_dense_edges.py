"""The dense operators where a formula taken as it stands loses its digits or its infinities: rows that one expert
dominates, values next to a border, infinities and NaN.  Against the definitions in 64 bits."""
import math

import pytest
import torch

from test_gpu_dense import ACTS, PAIRS, TYPES, U, act64, close, gate64, half_step, rand, route_grad64, slope64, sum_tol

pytestmark = pytest.mark.gpu

GATINGS = ["softmax", "sigmoid", "sqrt_softplus"]


# ---------------------------------------------------------------- gradient of the routing


@pytest.mark.parametrize("gating", GATINGS)
@pytest.mark.parametrize("S,E", [(1, 1), (4, 60), (565, 200), (33, 384), (7, 1024)])
def test_one_renormalised_route_has_no_gradient(S, E, gating):
    """Its weight is a constant, so the gradient is 0 and not the rounding of a difference."""
    import zeromoe_amd as Z

    logits, dw = rand(S, E, seed=1, scale=1.5), rand(S, 1, seed=2)
    ids, w = Z.router(logits, 1, gating=gating, weights_norm=True, weights_scale=2.5)
    k = dict(gating=gating, weights_norm=True, weights_scale=2.5)
    assert (Z.router_backward(logits, ids, dw, **k) == 0).all()
    # the same route among others that take no part, and one expert named by every route
    wide = torch.full((S, min(E, 4)), -1, device="cuda", dtype=torch.int32)
    wide[:, -1:] = ids
    assert (Z.router_backward(logits, wide, rand(*wide.shape, seed=3), **k) == 0).all()
    twice, d2 = ids.expand(S, min(E, 2)).contiguous(), rand(S, min(E, 2), seed=4)
    # the two routes' results are each other's negative but for a few roundings of dw / N
    p = gate64(logits.double(), gating).gather(1, ids.long())
    assert (Z.router_backward(logits, twice, d2, **k).abs() <= 16 * U * 2.5 * d2.abs().sum(-1, keepdim=True) / p).all()
    # what a balance loss adds stays
    dp = rand(E, seed=5)
    got = Z.router_backward(logits, ids, dw, dprobs=dp, **k)
    want = route_grad64(logits, ids, torch.zeros_like(dw), gating, None, True, 2.5, dp)
    p = gate64(logits.double(), gating)
    close(got, want, U * (40 + 2 * math.sqrt(E)) * (dp.abs().double() + (p * dp.abs().double()).sum(-1, keepdim=True)) * p * 2 + 1e-37)


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("gating", GATINGS)
def test_a_dominated_row_keeps_its_digits(gating, norm):
    """One expert has nearly all of the weight: every result, its own among them, to within roundings of itself.

    A result is a product and quotient of sums without cancellation (the dw below have none), each of up to E terms of
    one sign and one size: 2 log2 E roundings of pairwise sums, exp's argument up to 20 (20 roundings), exp, log1p and
    the divisions a few each: 100 roundings cover them."""
    import zeromoe_amd as Z

    for E, seed in ((12, 1), (200, 2), (1000, 3)):
        chosen = torch.randperm(E, generator=torch.Generator().manual_seed(seed))[:4].int().cuda()
        logits = torch.full((1, E), -19.0, device="cuda") - rand(1, E, seed=seed).abs().clamp(max=1)
        logits[0, chosen.long()] = torch.tensor([1.25, -12.0, -13.0, -12.5], device="cuda")
        ids, dw = chosen[None].contiguous(), torch.tensor([[0.3, -0.5, 0.7, 0.2]], device="cuda")
        got = Z.router_backward(logits, ids, dw, gating=gating, weights_norm=norm)
        want = route_grad64(logits, ids, dw, gating, None, norm, 0.0, None)
        if norm or gating != "softmax":  # the others' are 0
            want = torch.zeros_like(want).scatter_(1, ids.long(), want.gather(1, ids.long()))
        close(got, want, 100 * U * want.abs())


# ---------------------------------------------------------------- infinities and NaN in the gradients of a product


@pytest.mark.parametrize("S,I,O", [(9, 264, 40), (200, 96, 133), (300, 512, 256)])
@pytest.mark.parametrize("act,ydt", [("none", None), ("none", "f32"), ("silu", None), ("gelu", "f32")])
@pytest.mark.parametrize("xt,wt", PAIRS)
def test_a_gradient_that_overflowed_shows(xt, wt, act, ydt, S, I, O):
    """An infinity and a NaN in dy reach the rows of dx, the rows of dw and the entries of dbias that are theirs, and no
    others: a check for overflow sees them wherever it looks."""
    import zeromoe_amd as Z

    x, w = rand(S, I, seed=1, dtype=TYPES[xt]), rand(O, I, seed=2, scale=0.02, dtype=TYPES[wt])
    yt = TYPES[ydt or xt]
    dy, pre = rand(S, O, seed=3, scale=0.01, dtype=yt), None if act == "none" else rand(S, O, seed=4, dtype=yt)
    dy[2, 5], dy[7, 30] = float("inf"), float("nan")
    dx, dw, db = Z.linear_backward(dy, x, w, act=act, pre=pre)
    rows, cols = torch.zeros(S, device="cuda", dtype=torch.bool), torch.zeros(O, device="cuda", dtype=torch.bool)
    rows[[2, 7]] = cols[[5, 30]] = True
    assert not dx[rows].isfinite().any() and dx[~rows].isfinite().all()
    assert not dw[cols].isfinite().any() and dw[~cols].isfinite().all()
    assert not db[cols].isfinite().any() and db[~cols].isfinite().all()


@pytest.mark.parametrize("act", ACTS[1:])
@pytest.mark.parametrize("xt,wt", PAIRS)
def test_a_nan_before_the_activation_shows(xt, wt, act):
    """Its result is NaN, and so are the gradients that it takes part in."""
    import zeromoe_amd as Z

    S, I, O = 40, 72, 24
    x, w = rand(S, I, seed=1, dtype=TYPES[xt]), rand(O, I, seed=2, dtype=TYPES[wt])
    dy, pre = rand(S, O, seed=3, dtype=TYPES[xt]), rand(S, O, seed=4, dtype=TYPES[xt])
    pre[11, 6] = float("nan")
    dx, dw, db = Z.linear_backward(dy, x, w, act=act, pre=pre)
    rows, cols = torch.arange(S, device="cuda") == 11, torch.arange(O, device="cuda") == 6
    assert dx[rows].isnan().all() and dx[~rows].isfinite().all()
    assert dw[cols].isnan().all() and dw[~cols].isfinite().all()
    assert db[cols].isnan().all() and db[~cols].isfinite().all()
    for n in (1, 7, 40):  # the forward pass, by its kernels for few rows and many
        y = x[:n].clone()
        y[0, 3] = float("nan")
        y = Z.linear(y, w, act=act)
        assert y[0].isnan().all() and y[1:].isfinite().all()


# ---------------------------------------------------------------- layer norm


@pytest.mark.parametrize("xt", list(TYPES))
@pytest.mark.parametrize("n", [72, 264, 1000, 2047, 4096, 5120, 7168, 8192, 20000])
def test_layer_norm_of_small_spreads_far_from_zero(n, xt):
    """Constant rows whose sums are not whole numbers of f32, and spreads of a millionth of the mean.

    A first mean is off by D standard deviations, D = (4 + 2 sqrt n) 2^-24 mean|x| rstd, and every difference from it is
    exact to 2^-24 of itself; their own mean is off by (4 + 2 sqrt n) 2^-24 of their size, 1 + D.  So h is off by as much,
    and 1 / rstd^2 by as much of 1 + D^2.  The saved mean is rounded once, 2^-24 of it, and the gradients' h with it."""
    import zeromoe_amd as Z

    noise = rand(6, n, seed=1)
    x = torch.stack([torch.full((n,), 12345.6), torch.full((n,), 3000.7), torch.full((n,), -0.1)]).cuda()
    x = torch.cat([x, 1e4 + 0.01 * noise[:1], -3e3 + 0.1 * noise[1:2], 50 + 1e-3 * noise[2:3], noise[3:]]).to(TYPES[xt])
    gain, shift, eps = 1 + 0.2 * rand(n, seed=2), rand(n, seed=3), 1e-5
    y, mean, rstd = Z.layer_norm(x, gain, shift, eps=eps, stats=True)
    x64 = x.double()
    m64 = x64.mean(-1, keepdim=True)
    r64 = 1 / torch.sqrt(x64.var(-1, unbiased=False, keepdim=True) + eps)
    h64 = (x64 - m64) * r64
    k = U * (4 + 2 * math.sqrt(n))
    D = k * x64.abs().mean(-1, keepdim=True) * r64
    htol = 4 * k * (1 + h64.abs()) * (1 + D) ** 2
    y64 = h64 * gain.double() + shift.double()
    last = half_step(x.dtype) * y64.abs() + (2.0 ** -25 if xt == "f16" else 0)
    close(y, y64, htol * gain.double().abs() + 2 * U * (y64.abs() + shift.double().abs()) + last)
    close(mean, m64[:, 0], (U * m64.abs() + 2 * k * (1 + D) / r64)[:, 0])
    close(rstd, r64[:, 0], (4 * k * (1 + D) ** 2 * r64)[:, 0])
    dy = rand(x.shape[0], n, seed=4, dtype=x.dtype)
    dx, dw, db = Z.layer_norm_backward(dy, x, mean, rstd, gain)
    hb = htol + U * m64.abs() * r64
    g = dy.double() * gain.double()
    s1, s2 = g.mean(-1, keepdim=True), (g * h64).mean(-1, keepdim=True)
    want = r64 * (g - s1 - h64 * s2)
    a = g.abs().mean(-1, keepdim=True)
    ah = (g.abs() * h64.abs()).mean(-1, keepdim=True)
    tol = r64 * (8 * k * (1 + D) ** 2 * (g.abs() + a + h64.abs() * ah) + hb * (s2.abs() + a) + (h64.abs() + hb) * (g.abs() * hb).mean(-1, keepdim=True))
    close(dx, want, tol + half_step(x.dtype) * want.abs() + (2.0 ** -25 if xt == "f16" else 0))
    close(dw, (dy.double() * h64).sum(0), (dy.double().abs() * (hb + 8 * U * h64.abs())).sum(0) + 1e-37)


@pytest.mark.parametrize("n", [1, 7, 72, 100, 264, 2000, 4100])
def test_layer_norm_backward_of_huge_constant_rows(n):
    """Rows that are finite, and so are their gradients by the formula: h is 0, dx = rstd (g - mean g)."""
    import zeromoe_amd as Z

    dy = rand(4, n, seed=1, scale=1e-3)
    x = torch.tensor([1e38 / n, -3e38 / n, 1e37 / n, 2.0], device="cuda")[:, None].expand(4, n).contiguous()
    rstd = torch.full((4,), 1e3 * n, device="cuda")
    dx, dw, db = Z.layer_norm_backward(dy, x, x[:, 0], rstd)
    g = dy.double()
    mean = g.mean(-1, keepdim=True)
    close(dx, rstd.double()[:, None] * (g - mean), rstd.double()[:, None] * (sum_tol(n, g.abs().mean(-1, keepdim=True)) + 4 * U * (g.abs() + mean.abs())))
    assert (dw == 0).all()
    close(db, g.sum(0), sum_tol(4, g.abs().sum(0)))


@pytest.mark.parametrize("S,I,O", [(3, 64, 40), (40, 264, 100), (130, 512, 257), (600, 1000, 160), (2048, 256, 96)])
@pytest.mark.parametrize("act,ydt", [("none", "f32"), ("gelu", None), ("silu", "f32")])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_a_16_bit_dx_keeps_sixteen_bits_of_dz(t, act, ydt, S, I, O):
    """A gradient whose rows sum to about zero times a w whose rows are alike: the sum cancels, and what dz has lost
    before it shows.  Two bf16 terms of dz leave out 2^-16 of |dz w| at most."""
    import zeromoe_amd as Z

    dtype, yt = TYPES[t], TYPES[ydt or t]
    x = rand(S, I, seed=1, dtype=dtype)
    w = (1.0 + 0.05 * rand(O, I, seed=2)).to(dtype)
    pre = None if act == "none" else rand(S, O, seed=4, scale=1.5, dtype=yt)
    slope = 1.0 if act == "none" else slope64(pre.double(), act)
    dz = rand(S, O, seed=3).double()
    # dz with a sum of zero: dy is that over the slope, where there is one to divide by
    dz = dz - dz.mean(-1, keepdim=True)
    dy = dz if act == "none" else dz / torch.where(slope.abs() < 0.05, torch.full_like(slope, 0.05), slope)
    dy = dy.to(yt)
    dx = Z.linear_backward(dy, x, w, act=act, pre=pre, need_dw=False, need_dbias=False)[0]
    dz = dy.double() * slope
    want = dz @ w.double()
    absdot = (dz.abs() + (16 * U * dy.double().abs() if act != "none" else 0)) @ w.double().abs()
    small = 2.0 ** -25 if t == "f16" else 0
    close(dx, want, sum_tol(O, absdot) + (2.0 ** -16 + (16 * U if act != "none" else 0)) * absdot + half_step(dtype) * want.abs() + small)


# ---------------------------------------------------------------- slopes


def test_slope_of_a_saturated_sigmoid():
    """sigmoid'(z) = sigmoid(z) sigmoid(-z) to within roundings of itself, also where sigmoid(z) is 1 in f32: exp of an
    exact argument to two steps, a sum, a division and three products: 16 roundings cover them."""
    import zeromoe_amd as Z

    z = torch.cat([torch.linspace(-60, 60, 481), torch.tensor([16.6, 17.0, 25.0, 80.0])]).cuda()
    slope = torch.sigmoid(z.double()) * torch.sigmoid(-z.double())
    dy = rand(1, z.numel(), seed=1)
    x, w = torch.zeros(1, 4, device="cuda"), torch.zeros(z.numel(), 4, device="cuda")
    db = Z.linear_backward(dy, x, w, act="sigmoid", pre=z[None])[2]
    want = dy[0].double() * slope
    close(db, want, 16 * U * want.abs())
    # as a gating: 97 rows of five experts, all of them routed
    logits = z.view(97, 5)
    ids, dw = torch.arange(5, device="cuda", dtype=torch.int32).expand(97, 5).contiguous(), rand(97, 5, seed=2)
    want = dw.double() * slope.view(97, 5)
    close(Z.router_backward(logits, ids, dw, gating="sigmoid"), want, 16 * U * want.abs())


# ---------------------------------------------------------------- infinities in a product


def products64(a, b):
    """a b^T value by value (a library product may pad with zeros, and 0 inf is NaN)."""
    return torch.stack([(a.double() * row.double()).sum(-1) for row in b], -1)


def same(got, want, tol):
    """Infinities and NaN where the formula has them; elsewhere within the tolerance."""
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got.isinf(), inf) and (got[inf].double() == want[inf]).all()
    ok = want.isfinite()
    close(got[ok], want[ok], tol[ok])


@pytest.mark.parametrize("I,O", [(72, 24), (520, 133), (2056, 40), (4100, 600)])
@pytest.mark.parametrize("S", [2, 5, 24, 100, 300])
@pytest.mark.parametrize("xt,wt", PAIRS)
def test_infinities_go_by_the_formula(xt, wt, S, I, O):
    """Whatever kernel the number of rows brings: an infinity times a weight is one of its sign, times zero NaN, and two
    of both signs are NaN."""
    import zeromoe_amd as Z

    inf = float("inf")
    x, w = rand(S, I, seed=1, dtype=TYPES[xt]), rand(O, I, seed=2, scale=0.05, dtype=TYPES[wt])
    b = rand(O, seed=3)
    x[0, 9] = inf
    x[1, 3], x[1, I - 1] = -inf, inf
    x[S - 1, 5] = -inf
    w[4, 5] = w[7, 9] = 0.0  # times an infinity
    w[11, 20], w[12, 21] = inf, float("nan")
    xf, wf = torch.where(x.isfinite(), x, torch.zeros_like(x)), torch.where(w.isfinite(), w, torch.zeros_like(w))
    tol = sum_tol(I, xf.double().abs() @ wf.double().abs().t() + b.double().abs())
    want = products64(x, w) + b.double()
    y, pre = Z.linear(x, w, bias=b, act="relu", out_dtype=torch.float32, save_pre=True)
    same(pre, want, tol)
    same(y, torch.where(want.isnan(), want, want.clamp(min=0)), tol)
    p = torch.sigmoid(want)  # of an infinity 0 or 1
    same(Z.linear(x, w, bias=b, act="sigmoid", out_dtype=torch.float32), p, tol + 8 * U)


@pytest.mark.parametrize("S,I,O", [(3, 72, 40), (40, 264, 133), (300, 520, 72), (130, 1000, 640)])
@pytest.mark.parametrize("act,ydt", [("none", None), ("none", "f32"), ("silu", None)])
@pytest.mark.parametrize("xt,wt", PAIRS)
def test_infinities_in_gradients_go_by_the_formula(xt, wt, act, ydt, S, I, O):
    import zeromoe_amd as Z

    inf, yt = float("inf"), TYPES[ydt or xt]
    x, w = rand(S, I, seed=1, dtype=TYPES[xt]), rand(O, I, seed=2, scale=0.05, dtype=TYPES[wt])
    dy, pre = rand(S, O, seed=3, dtype=yt), None if act == "none" else rand(S, O, seed=4, dtype=yt)
    dy[0, 9], dy[1, 3], dy[1, O - 1] = inf, -inf, inf
    w[9, 5] = x[0, 6] = 0.0
    w[11, 20], x[S - 1, 30] = inf, -inf
    slope = 1.0 if act == "none" else slope64(pre.double(), act)
    dz = dy.double() * slope
    z, xf, wf = (torch.where(t.isfinite(), t, torch.zeros_like(t)).double() for t in (dz, x, w))
    # silu' = g (1 + z (1 - g)), |z| up to 4.5 here: g is off by up to 3 roundings (exp's of e^-z, the sum's, the
    # quotient's), so z (1 - g) by 3 |z| and its own, and the slope by up to 16 2^-24 of 1, not of itself: it passes
    # through 0 at z = -1.28.  dz is off by as much of |dy|, whatever is left of the sum
    off = (16 * U if act != "none" else 0.0) * torch.where(dy.isfinite(), dy, torch.zeros_like(dy)).double().abs()
    dx, dw, db = Z.linear_backward(dy, x, w, act=act, pre=pre)
    t = z.abs() @ wf.abs()
    want = products64(dz, w.t())
    small = 2.0 ** -25 if xt == "f16" else 0
    same(dx, want, sum_tol(O, t) + 2.0 ** -16 * t + off @ wf.abs() + half_step(dx.dtype) * (z @ wf).abs() + small)
    t = z.abs().t() @ xf.abs()
    same(dw, products64(dz.t(), x.t()), sum_tol(S, t) + off.t() @ xf.abs() + half_step(torch.float32) * t)
    same(db, dz.sum(0), sum_tol(S, z.abs().sum(0)) + off.sum(0))


def test_sums_whose_terms_overflow():
    """Products of terms may pass f32's largest where the products of values and their sum do not."""
    import zeromoe_amd as Z

    for S in (2, 40, 200):
        x = torch.zeros(S, 64, device="cuda")
        x[:, 3], x[:, 8] = 2.0 ** 127 * 1.99, 1.0
        w = torch.zeros(24, 64, device="cuda")
        w[:, 3] = torch.linspace(0.9, 1.0048, 24)  # up to a hair below 2^128
        y = Z.linear(x, w)
        want = products64(x, w)
        assert (want < 2.0 ** 128).all()
        close(y, want, 2 * U * want.abs())


# ---------------------------------------------------------------- arguments


def test_a_gradient_does_not_end_silently():
    """In grad mode a tensor that requires a gradient is refused by every call that takes it; under no_grad it is taken."""
    import zeromoe_amd as Z

    x, w, b, y3, wt = rand(4, 16), rand(8, 16), rand(8), rand(4, 2, 16), rand(4, 2)
    dy, r = rand(4, 8), rand(4, 8)
    ids = torch.zeros(4, 2, device="cuda", dtype=torch.int32)
    _, mean, rstd = Z.layer_norm(x, stats=True)
    calls = [(Z.linear, dict(x=x, w=w, bias=b, residual=r)), (Z.linear_backward, dict(dy=dy, x=x, w=w, act="silu", pre=r)),
             (Z.layer_norm, dict(x=x, weight=x[0].clone(), bias=x[1].clone())),
             (Z.layer_norm_backward, dict(dy=x.clone(), x=x, mean=mean, rstd=rstd, weight=x[0].clone())),
             (Z.combine, dict(y=y3, weights=wt, residual=x)), (Z.combine_backward, dict(dout=x, y=y3, weights=wt, need_dy=True)),
             (Z.router_backward, dict(logits=r, ids=ids, dweights=wt, logit_bias=b, dprobs=b.clone()))]
    for f, args in calls:
        want = f(**args)
        want = want if isinstance(want, tuple) else (want,)
        for name, t in args.items():
            if not isinstance(t, torch.Tensor) or t is ids:
                continue
            p = dict(args, **{name: t.clone().requires_grad_()})
            with pytest.raises(ValueError, match="requires a gradient"):
                f(**p)
            with pytest.raises(ValueError, match="requires a gradient"):
                f(**p, stream=torch.cuda.Stream())
            with torch.no_grad():
                got = f(**p)
            assert all(torch.equal(u, v) and not u.requires_grad for u, v in zip(got if isinstance(got, tuple) else (got,), want))


def test_sizes_past_32_bits_are_refused():
    """Not taken for what their lower 32 bits say."""
    import zeromoe_amd as Z

    n = (1 << 32) + 1
    one, i32 = torch.zeros(1, 1, device="cuda"), torch.zeros(1, 1, device="cuda", dtype=torch.int32)
    for f in (lambda: Z.router_backward(one.expand(n, 1), i32.expand(n, 1), one.expand(n, 1)),
              lambda: Z.combine(one.view(1, 1, 1).expand(1, 1, n), one),
              lambda: Z.combine(one.view(1, 1, 1).expand(1, n, 1), one.expand(1, n)),
              lambda: Z.router_backward(one.expand(1, n), i32, one),
              lambda: Z.combine_backward(one.expand(1, n), one.view(1, 1, 1).expand(1, 1, n))):
        with pytest.raises(ValueError, match="too large"):
            f()


# ---------------------------------------------------------------- allowed calls that are not the usual ones


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S,I,O", [(1, 264, 72), (5, 72, 40), (50, 264, 72), (300, 72, 264), (257, 1000, 40)])
def test_linear_backward_of_strided_rows_on_any_address(xt, wt, S, I, O):
    """dy, x, w and pre as columns of wider buffers, on even and odd addresses: the results of contiguous copies, but for
    the order of sums that another kernel has; and the neighbours of nothing are read as values."""
    import zeromoe_amd as Z

    def view(n, width, off, pad, seed, dtype, scale=1.0):
        b = torch.full((n * (width + pad) + 16,), float("nan"), device="cuda", dtype=dtype)
        v = b[off:off + n * (width + pad)].view(n, width + pad)[:, :width]
        return v.copy_(rand(n, width, seed=seed, dtype=dtype, scale=scale))

    for off, pad in ((0, 8), (1, 3), (4, 4), (1, 8)):
        for act, ydt in (("none", None), ("silu", None), ("gelu_tanh", "f32")):
            yt = TYPES[ydt or xt]
            x, w = view(S, I, off, pad, 1, TYPES[xt]), view(O, I, off, pad, 2, TYPES[wt], 0.05)
            dy, pre = view(S, O, off, pad, 3, yt, 0.1), view(S, O, off, pad + 8, 4, yt)
            dx, dw, db = Z.linear_backward(dy, x, w, act=act, pre=pre)
            slope = 1.0 if act == "none" else slope64(pre.double(), act)
            dz = dy.double() * slope
            offs = (16 * U if act != "none" else 0.0) * dy.double().abs()  # the slope's own roundings, of 1
            t = dz.abs() @ w.double().abs()
            want = dz @ w.double()
            close(dx, want, sum_tol(O, t) + (2.0 ** -16 if xt != "f32" else 0) * t + offs @ w.double().abs()
                  + half_step(dx.dtype) * want.abs() + (2.0 ** -25 if xt == "f16" else 0))
            t = dz.abs().t() @ x.double().abs()
            close(dw, dz.t() @ x.double(), sum_tol(S, t) + offs.t() @ x.double().abs() + U * t)
            close(db, dz.sum(0), sum_tol(S, dz.abs().sum(0)) + offs.sum(0))


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S", [1, 3, 20, 130, 700])
def test_linear_strided_residual_pre_and_repeated_weight_rows(S, xt, wt):
    import zeromoe_amd as Z

    I, O = 2056, 72
    x, w = rand(S, I, seed=1, dtype=TYPES[xt]), rand(1, I, seed=2, scale=0.02, dtype=TYPES[wt]).expand(O, I)
    for dtype in {TYPES[xt], torch.float32}:
        for off, pad in ((0, 8), (3, 5)):
            r = rand(S, O + off + pad, seed=3, dtype=dtype)[:, off:off + O]
            y, pre = Z.linear(x, w, residual=r, act="relu", out_dtype=dtype, save_pre=True)
            y2, pre2 = Z.linear(x, w.contiguous(), residual=r.contiguous(), act="relu", out_dtype=dtype, save_pre=True)
            z = x.double() @ w.double().t()
            tol = sum_tol(I, x.double().abs() @ w.double().abs().t())
            for p, q in ((pre, y), (pre2, y2)):
                small = 2.0 ** -25 if dtype == torch.float16 else 0
                close(p, z, tol + half_step(dtype) * z.abs() + small)
                want = z.clamp(min=0) + r.double()
                close(q, want, tol + 2 * U * r.double().abs() + half_step(dtype) * want.abs() + small)


@pytest.mark.parametrize("xt", list(TYPES))
@pytest.mark.parametrize("n", [5, 64, 257, 1024, 4100, 8192, 20000])
def test_layer_norm_gradient_over_its_operands(n, xt):
    """dx in the place of dy, and of x, as the C call allows."""
    import zeromoe_amd as Z
    from zeromoe_amd._lib import check, lib

    rows, code = 700, {"f32": 0, "f16": 1, "bf16": 30}[xt]
    x, dy, gain = rand(rows, n, seed=1, dtype=TYPES[xt]), rand(rows, n, seed=2, dtype=TYPES[xt]), rand(n, seed=3)
    _, mean, rstd = Z.layer_norm(x, gain, stats=True)
    want = Z.layer_norm_backward(dy, x, mean, rstd, gain)
    ws = torch.empty(lib().zm_layer_norm_backward_workspace_size(rows, n), device="cuda", dtype=torch.uint8)
    st = torch.cuda.current_stream().cuda_stream
    for over in ("dy", "x"):
        a, b = dy.clone(), x.clone()
        d, dw, db = a if over == "dy" else b, torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        check(lib().zm_layer_norm_backward(code, a.data_ptr(), n, b.data_ptr(), n, gain.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                           rows, n, d.data_ptr(), n, dw.data_ptr(), db.data_ptr(), ws.data_ptr(), ws.numel(), st), "ln")
        for got, w in zip((d, dw, db), want):
            assert torch.equal(got, w)
    x2 = x.clone()
    y, m2, r2 = Z.layer_norm(x2, gain, stats=True, out=x2)
    assert y is x2 and torch.equal(m2, mean) and torch.equal(r2, rstd) and torch.equal(y, Z.layer_norm(x, gain))


def test_combine_gradient_without_its_rows():
    """dy alone reads no y, and dweights alone no weights."""
    from zeromoe_amd._lib import check, lib

    S, K, H = 9, 3, 68
    d, w, st = rand(S, H, seed=1), rand(S, K, seed=2), torch.cuda.current_stream().cuda_stream
    ids = torch.randint(-1, 2, (S, K), device="cuda", dtype=torch.int32, generator=torch.Generator("cuda").manual_seed(3))
    dy = torch.empty(S, K, H, device="cuda")
    check(lib().zm_combine_backward(d.data_ptr(), None, 0, 0, w.data_ptr(), ids.data_ptr(), S, K, H, None, dy.data_ptr(), st), "dy")
    assert torch.equal(dy, torch.where((ids >= 0)[:, :, None], w[:, :, None] * d[:, None], torch.zeros_like(dy)))


def test_combine_of_most_routes_and_single_columns():
    import zeromoe_amd as Z

    for S, K, H in ((3, 64, 1), (1, 64, 260), (5, 33, 3)):
        y, w, d = rand(S, K, H, seed=1), rand(S, K, seed=2), rand(S, H, seed=3)
        off = torch.full((S, K), -1, device="cuda", dtype=torch.int32)
        close(Z.combine(y, w), (w.double()[:, :, None] * y.double()).sum(1), sum_tol(2 * K, (w[:, :, None] * y).abs().double().sum(1)))
        assert torch.equal(Z.combine(y, w, ids=off, residual=d), d) and (Z.combine(y, w, ids=off) == 0).all()
        assert (Z.combine_backward(d, y, ids=off) == 0).all()
        t = y.transpose(0, 1).contiguous().transpose(0, 1)  # routes outermost, as one expert after the other leaves them
        assert torch.equal(Z.combine(t, w), Z.combine(y, w)) and torch.equal(Z.combine_backward(d, t), Z.combine_backward(d, y))


@pytest.mark.parametrize("gating", GATINGS)
@pytest.mark.parametrize("K", [2, 5, 8, 17, 40, 64])
def test_a_dominated_row_wherever_its_routes_stand(gating, K):
    """The dominating route at every place of a row, others left out before and behind it: within roundings as above."""
    import zeromoe_amd as Z

    E = 128
    g = torch.Generator().manual_seed(K)
    ids = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(K)]).int()
    logits = torch.full((K, E), -19.0)
    logits.scatter_(1, ids.long(), -12.0 - torch.rand(K, K, generator=g))
    at = torch.arange(K)
    logits[at, ids[at, at].long()] = 1.25
    left = torch.rand(K, K, generator=g) < 0.3
    left[at, at] = False
    ids[left] = -1
    dw = 0.1 + torch.rand(K, K, generator=g)
    dw[at, at] = -0.4  # sum of (d - d0) p: no cancellation
    ids, logits, dw = ids.cuda(), logits.cuda(), dw.cuda()
    got = Z.router_backward(logits, ids, dw, gating=gating, weights_norm=True)
    want = route_grad64(logits, ids, dw, gating, None, True, 0.0, None)
    on = torch.zeros(K, E + 1, device="cuda", dtype=torch.bool).scatter_(1, torch.where(ids < 0, torch.full_like(ids, E), ids).long(), True)[:, :E]
    alone = (ids >= 0).sum(-1, keepdim=True) == 1
    want = torch.where(on & ~alone, want, torch.zeros_like(want))
    # d' - sum d' p / N: for sqrt-softplus the others' p add to a tenth of N and more; the difference keeps at least a
    # quarter of its larger part
    close(got, want, 4 * 100 * U * want.abs())
