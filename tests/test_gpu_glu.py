"""The gated product and its gradients against their definition in 64 bits.

Tolerances.  Each factor is a sum of n products in f32: (4 + 2 sqrt n) 2^-24 sum |a b|, as for linear (test_gpu_dense).  The
result act(z) u moves by |u| |act'| of the first's error (no activation here is steeper than 1.2), by |act(z)| of the
second's, and by the activation's own error, 8 steps of f32; its last rounding is eps / 2 of its type."""
import math

import pytest
import torch

from test_gpu_dense import ACTS, PAIRS, TYPES, U, act64, close, half_step, rand, slope64, sum_tol

pytestmark = pytest.mark.gpu


def factors64(x, w_gate, w_up, b_gate, b_up):
    out = []
    for w, b in ((w_gate, b_gate), (w_up, b_up)):
        z, a = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
        t = sum_tol(x.shape[1], a)
        if b is not None:
            z, t = z + b.double(), t + 2 * U * (b.double().abs() + a)
        out += [z, t]
    return out


def smallest(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 1e-37


def check_glu(S, I, F, xt, wt, act="silu", bias=True, save=True, ydt=None, seed=1, x=None, w_gate=None, w_up=None, out=None):
    import zeromoe_amd as Z

    x = rand(S, I, seed=seed, dtype=TYPES[xt]) if x is None else x
    w_gate = rand(F, I, seed=seed + 1, scale=1 / math.sqrt(I), dtype=TYPES[wt]) if w_gate is None else w_gate
    w_up = rand(F, I, seed=seed + 2, scale=1 / math.sqrt(I), dtype=TYPES[wt]) if w_up is None else w_up
    b_gate, b_up = (rand(F, seed=seed + 3), rand(F, seed=seed + 4)) if bias else (None, None)
    dtype = TYPES[ydt or xt]
    y = Z.glu(x, w_gate, w_up, b_gate, b_up, act=act, out_dtype=dtype, save=save, out=out)
    z, tz, u, tu = factors64(x, w_gate, w_up, b_gate, b_up)
    if save:
        y, gate, up = y
        for got, want, t in ((gate, z, tz), (up, u, tu)):
            assert got.dtype == dtype and got.shape == (S, F)
            close(got, want, t + half_step(dtype) * want.abs() + smallest(dtype))
    assert y.dtype == dtype and y.shape == (S, F)
    a = act64(z, act)
    tol = 1.2 * tz * (u.abs() + tu) + tu * a.abs() + 8 * U * (a.abs() + 1e-3) * u.abs()
    close(y, a * u, tol + half_step(dtype) * (a * u).abs() + smallest(dtype))
    return y


SHAPES = [(1, 1, 1), (1, 256, 32), (1, 4096, 96), (2, 264, 2050), (3, 7, 5), (4, 64, 257), (5, 1000, 31), (8, 512, 128),
          (9, 264, 100), (24, 2048, 160), (31, 640, 2100), (33, 96, 129), (64, 1024, 64), (65, 136, 260), (127, 257, 33),
          (130, 640, 130), (300, 72, 1000), (513, 1288, 384)]


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S,I,F", SHAPES)
def test_glu(S, I, F, xt, wt):
    check_glu(S, I, F, xt, wt)
    check_glu(S, I, F, xt, wt, bias=False, save=False, ydt="f32", seed=11)


@pytest.mark.parametrize("xt,wt", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("S,I,F", [(700, 264, 1000), (1030, 512, 160), (2048, 1024, 1536), (257, 4096, 20)])
def test_glu_tiles(S, I, F, xt, wt):
    """All tiles, and slices of k."""
    check_glu(S, I, F, xt, wt)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("S", [1, 20, 200])
def test_glu_activations(act, S):
    check_glu(S, 320, 200, "f32", "bf16", act)
    check_glu(S, 320, 200, "bf16", "bf16", act)


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S", [1, 7, 40, 150, 300])
def test_glu_strides_and_alignment(xt, wt, S):
    """Rows that lie apart, on odd addresses, and a result whose neighbours stay as they are."""
    I, F = 264, 72
    for ox, og, ou, pad in ((0, 0, 0, 8), (1, 0, 0, 8), (0, 1, 0, 8), (0, 0, 1, 8), (1, 3, 5, 3), (8, 8, 0, 0)):
        xb = rand(S * (I + pad) + 16, seed=3, dtype=TYPES[xt])
        wb = [rand(F * (I + pad) + 16, seed=4 + i, scale=0.06, dtype=TYPES[wt]) for i in range(2)]
        x, g, u = (b[o:o + n * (I + pad)].view(n, I + pad)[:, :I] for b, o, n in ((xb, ox, S), (wb[0], og, F), (wb[1], ou, F)))
        yb = torch.full((S + 2, F + pad + ox), 7.0, device="cuda", dtype=TYPES[xt])
        check_glu(S, I, F, xt, wt, x=x, w_gate=g, w_up=u, out=yb[1:S + 1, ox:ox + F])
        keep = torch.ones_like(yb, dtype=torch.bool)
        keep[1:S + 1, ox:ox + F] = False
        assert (yb[keep] == 7.0).all()
    both = rand(2 * F, I, seed=9, scale=0.06, dtype=TYPES[wt])  # one tensor of both weights, in either order, and interleaved
    check_glu(S, I, F, xt, wt, w_gate=both[:F], w_up=both[F:])
    check_glu(S, I, F, xt, wt, w_gate=both[F:], w_up=both[:F])
    check_glu(S, I, F, xt, wt, w_gate=both[0::2], w_up=both[1::2])
    check_glu(S, I, F, xt, wt, w_gate=both[:F], w_up=both[:F])
    check_glu(S, I, F, xt, wt, x=rand(1, I, seed=6, dtype=TYPES[xt]).expand(S, I))
    check_glu(S, I, F, xt, wt, x=rand(I, S, seed=5, dtype=TYPES[xt]).t())


def test_glu_no_rows():
    import zeromoe_amd as Z

    w = rand(24, 72, seed=1)
    y, gate, up = Z.glu(rand(0, 72), w, w, save=True)
    assert y.shape == gate.shape == up.shape == (0, 24)
    dx, dg, du, bg, bu = Z.glu_backward(y, rand(0, 72), w, w, gate, up)
    assert dx.shape == (0, 72)
    for t in (dg, du, bg, bu):
        assert (t == 0).all() and t.shape in ((24, 72), (24,))


def check_glu_backward(S, I, F, xt, wt, act="silu", ydt=None, seed=1, need=(True, True, True), x=None, w_gate=None,
                       w_up=None, dy=None, gate=None, up=None):
    import zeromoe_amd as Z

    dtype, yt = TYPES[xt], TYPES[ydt or xt]
    x = rand(S, I, seed=seed, dtype=dtype) if x is None else x
    w_gate = rand(F, I, seed=seed + 1, scale=1 / math.sqrt(I), dtype=TYPES[wt]) if w_gate is None else w_gate
    w_up = rand(F, I, seed=seed + 2, scale=1 / math.sqrt(I), dtype=TYPES[wt]) if w_up is None else w_up
    dy = rand(S, F, seed=seed + 3, scale=0.1, dtype=yt) if dy is None else dy
    gate = rand(S, F, seed=seed + 4, scale=1.5, dtype=yt) if gate is None else gate
    up = rand(S, F, seed=seed + 5, scale=1.5, dtype=yt) if up is None else up
    r = Z.glu_backward(dy, x, w_gate, w_up, gate, up, act=act, need_dx=need[0], need_dw=need[1], need_db=need[2])
    assert [t is None for t in r] == [not need[i] for i in (0, 1, 1, 2, 2)]
    dx, dwg, dwu, dbg, dbu = r
    d, g, u = dy.double(), gate.double(), up.double()
    dg, du = d * u * slope64(g, act), d * act64(g, act)
    # the slope in f32: 16 steps of values below 1.2.  The activation: 8 steps of itself, and the rounding of what its
    # function is taken of, 2 steps of z / sqrt 2 for gelu (erfc(a) moves by 2 a^2 of itself) and 4 of the argument
    # w = 0.8 (z + 0.045 z^3) for gelu_tanh (exp(2 w) by 2 |w|): both below 8 z^2 steps from |z| = 1 on, and 8 before
    eg, eu = 18 * U * (d * u).abs(), (10 + 8 * g * g) * U * du.abs() + 1e-37
    cut = {"bf16": 2.0 ** -16, "f16": 2.0 ** -16, "f32": 0.0}[xt]  # 16 bits of dg and du for a 16-bit dx
    if dx is not None:
        wg, wu = w_gate.double(), w_up.double()
        want = dg @ wg + du @ wu
        absdot = dg.abs() @ wg.abs() + du.abs() @ wu.abs()
        assert dx.dtype == dtype and dx.shape == (S, I)
        close(dx, want, sum_tol(2 * F, absdot) + cut * absdot + eg @ wg.abs() + eu @ wu.abs() + half_step(dtype) * want.abs()
              + smallest(dtype))
    for dw, dz, e in ((dwg, dg, eg), (dwu, du, eu)):
        if dw is not None:
            want, absdot = dz.t() @ x.double(), dz.abs().t() @ x.double().abs()
            assert dw.dtype == torch.float32 and dw.shape == (F, I) and dw.is_contiguous()
            close(dw, want, sum_tol(S, absdot) + e.t() @ x.double().abs() + half_step(torch.float32) * want.abs())
    for db, dz, e in ((dbg, dg, eg), (dbu, du, eu)):
        if db is not None:
            close(db, dz.sum(0), sum_tol(S, dz.abs().sum(0)) + e.sum(0))


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S,I,F", [(1, 1, 1), (1, 256, 32), (3, 7, 5), (20, 264, 100), (64, 512, 160), (65, 136, 260),
                                   (127, 257, 33), (300, 72, 1000), (1030, 640, 96), (260, 1000, 36)])
def test_glu_backward(S, I, F, xt, wt):
    check_glu_backward(S, I, F, xt, wt)
    check_glu_backward(S, I, F, xt, wt, "gelu", seed=21)
    check_glu_backward(S, I, F, xt, wt, "none", ydt="f32", seed=31)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("xt,wt", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32")])
def test_glu_backward_activations(act, xt, wt):
    check_glu_backward(70, 320, 200, xt, wt, act)
    for need in ((True, False, False), (False, True, False), (False, False, True)):
        check_glu_backward(70, 320, 200, xt, wt, act, need=need)


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S", [1, 40, 300])
def test_glu_backward_strides_and_alignment(xt, wt, S):
    I, F = 264, 72

    def view(n, width, off, pad, seed, t, scale=1.0):
        return rand(n * (width + pad) + 16, seed=seed, dtype=TYPES[t], scale=scale)[off:off + n * (width + pad)].view(
            n, width + pad)[:, :width]

    for o, pad in ((0, 8), (1, 8), (3, 5)):
        check_glu_backward(S, I, F, xt, wt, x=view(S, I, o, pad, 1, xt), w_gate=view(F, I, 0, pad, 2, wt, 0.06),
                           w_up=view(F, I, o, pad, 3, wt, 0.06), dy=view(S, F, o, pad, 4, xt, 0.1),
                           gate=view(S, F, 2, pad, 5, xt), up=view(S, F, o, pad + 1, 6, xt))
    both = rand(2 * F, I, seed=9, scale=0.06, dtype=TYPES[wt])
    check_glu_backward(S, I, F, xt, wt, w_gate=both[F:], w_up=both[:F])
    check_glu_backward(S, I, F, xt, wt, w_gate=both[:F], w_up=both[:F], dy=rand(1, F, dtype=TYPES[xt]).expand(S, F))


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S", [2, 40, 300])
def test_glu_infinities_go_by_the_formula(xt, wt, S):
    """An infinity in a row of x, in a row of one weight and in dy: what the formula gives, in the rows and columns that
    it reaches and no others."""
    import zeromoe_amd as Z

    I, F = 136, 72
    x, g, u = rand(S, I, seed=1, dtype=TYPES[xt]), rand(F, I, seed=2, scale=0.1, dtype=TYPES[wt]), rand(F, I, seed=3, scale=0.1, dtype=TYPES[wt])
    x[1, 5] = math.inf
    u[7, 9] = -math.inf
    x[:, 9] = x[:, 9].abs() + 1
    y, gate, up = Z.glu(x, g, u, act="none", save=True)
    zg, zu = ((x.double()[:, None, :] * w.double()[None]).sum(-1) for w in (g, u))
    for got, want in ((gate, zg), (up, zu), (y, zg * zu)):
        assert torch.equal(got.double().isnan(), want.isnan())
        inf = want.isinf()
        assert torch.equal(got.double()[inf], want[inf])
        assert got[~inf & ~want.isnan()].isfinite().all()
    dy, gt, ut = (rand(S, F, seed=4 + i, dtype=TYPES[xt]) for i in range(3))
    dy[1, 3] = math.inf
    x = rand(S, I, seed=1, dtype=TYPES[xt])
    u = rand(F, I, seed=3, scale=0.1, dtype=TYPES[wt])
    dx, dwg, dwu, dbg, dbu = Z.glu_backward(dy, x, g, u, gt, ut, act="none")
    dg, du = dy.double() * ut.double(), dy.double() * gt.double()
    at = torch.zeros(S, I, dtype=torch.bool, device="cuda")
    at[1] = True
    assert not dx[at].isfinite().any() and dx[~at].isfinite().all()
    for dw, db, dz in ((dwg, dbg, dg), (dwu, dbu, du)):
        want = dz.t()[:, :, None] * x.double()[None]
        want = want.sum(1)
        inf = want.isinf()
        assert inf.any() and torch.equal(dw.double()[inf], want[inf]) and torch.equal(db.double()[3], dz[:, 3].sum())
        assert dw[~inf].isfinite().all()


def test_glu_graph_and_streams():
    """A captured forward and backward pass, replayed with new inputs and with eager work between; a call on a stream."""
    import zeromoe_amd as Z

    S, I, F = 40, 264, 100
    x, g, u, dy = rand(S, I, seed=1), rand(F, I, seed=2, scale=0.1), rand(F, I, seed=3, scale=0.1), rand(S, F, seed=4)

    def step():
        y, gate, up = Z.glu(x, g, u, save=True)
        return (y, *Z.glu_backward(dy, x, g, u, gate, up))

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (5, 6, 7):
        x.copy_(rand(S, I, seed=seed))
        dy.copy_(rand(S, F, seed=seed + 10))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y = Z.glu(x, g, u, stream=side)
    side.synchronize()
    assert torch.equal(y, outs[0])


def test_glu_repeats_its_bits():
    import zeromoe_amd as Z

    for S, I, F, t in ((24, 4096, 512, torch.bfloat16), (300, 2048, 160, torch.float32)):
        x, g, u = rand(S, I, seed=1, dtype=t), rand(F, I, seed=2, dtype=t), rand(F, I, seed=3, dtype=t)
        y, gate, up = Z.glu(x, g, u, save=True)
        first = (y, *Z.glu_backward(y, x, g, u, gate, up))
        for _ in range(3):
            y, gate, up = Z.glu(x, g, u, save=True)
            assert all(torch.equal(a, b) for a, b in zip(first, (y, *Z.glu_backward(y, x, g, u, gate, up))))


def test_glu_gradient_by_differences():
    """The gradients against central differences of the 64-bit formula at the same point."""
    import zeromoe_amd as Z

    S, I, F = 5, 24, 20
    x, g, u, dy = rand(S, I, seed=1), rand(F, I, seed=2, scale=0.3), rand(F, I, seed=3, scale=0.3), rand(S, F, seed=4)
    _, gate, up = Z.glu(x, g, u, save=True)
    dx, dwg, dwu, _, _ = Z.glu_backward(dy, x, g, u, gate, up)

    def loss(x, g, u):
        return ((act64(x @ g.t(), "silu") * (x @ u.t())) * dy.double()).sum()

    args, h = [x.double(), g.double(), u.double()], 1e-5
    for k, d in ((0, dx), (1, dwg), (2, dwu)):
        e = rand(*args[k].shape, seed=20 + k).double()
        up_, dn = [list(args), list(args)]
        up_[k], dn[k] = args[k] + h * e, args[k] - h * e
        want = ((loss(*up_) - loss(*dn)) / (2 * h)).item()
        # third differences: h^2; sums of 2^-24 of some hundred products
        assert abs((d.double() * e).sum().item() - want) <= 1e-4 * max(1.0, (d.double() * e).abs().sum().item())
