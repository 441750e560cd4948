"""Slopes of both gelus, which keep their digits where they are small.

One row: the bias gradients are the values themselves.  Tolerances, in steps of f32 (2^-24) of the parts that are added:
gelu's slope is Phi + z phi with Phi = erfc(-z / sqrt 2) / 2, phi = exp(-z^2 / 2) / sqrt(2 pi).  The argument of erfc is off by
two steps, which moves it by 2 z^2 steps, that of exp by z^2; four for each function, and eight roundings around them.  The
tanh form's is s + z s (1 - s) 2 w', s = 1 / (1 + exp(-2 w)), w = 0.798 (z + 0.0447 z^3): 2 w is off by six steps, so exp by
12 |w|, s and 1 - s with it, their product by 24 |w|; and 24 for the functions and roundings."""
import math

import pytest
import torch

from test_gpu_dense import U, rand

pytestmark = pytest.mark.gpu

N = 8192


def parts(z, act):
    """(the slope, its parts' sum, steps)"""
    if act == "gelu":
        phi = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        cdf = torch.special.erfc(-z / math.sqrt(2)) / 2
        return cdf + z * phi, cdf + (z * phi).abs(), 16 + 3 * z * z
    k = math.sqrt(2 / math.pi)
    w = k * (z + 0.044715 * z ** 3)
    s, n = torch.sigmoid(2 * w), torch.sigmoid(-2 * w)
    more = z * s * n * 2 * k * (1 + 3 * 0.044715 * z * z)
    return s + more, s + more.abs(), 24 + 24 * w.abs()


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh"])
def test_slopes_keep_their_digits(act):
    import zeromoe_amd as Z

    z = torch.linspace(-12, 12, N, device="cuda")[None].contiguous()
    d, up = rand(1, N, seed=1), rand(1, N, seed=2)
    want, size, steps = (t[0] for t in parts(z.double(), act))
    x, w = rand(1, 8), rand(N, 8)
    got = Z.linear_backward(d, x, w, act=act, pre=z, need_dx=False, need_dw=False)[2]
    gate = Z.glu_backward(d, x, w, w, z, up, act=act, need_dx=False, need_dw=False)[3]
    for g, f in ((got, d[0].double()), (gate, (d * up)[0].double())):
        err = (g.double() - want * f).abs()
        tol = (steps + 2) * U * size * f.abs() + 1e-37
        assert (err <= tol).all(), ((err / tol).max().item(), z[0, (err / tol).argmax()].item())


@pytest.mark.parametrize("act,low", [("relu", 0.0), ("gelu", 0.0), ("gelu_tanh", 0.0), ("silu", 0.0), ("sigmoid", 0.0), ("none", 1.0)])
def test_slopes_far_out(act, low):
    """Where the activation is 0 or z, and a NaN."""
    import zeromoe_amd as Z

    z = torch.tensor([[-math.inf, -3e38, -1e4, -300.0, 300.0, 1e4, 3e38, math.inf, math.nan]], device="cuda")
    n = z.shape[1]
    x, w, d = rand(1, 8), rand(n, 8), torch.ones(1, n, device="cuda")
    high = 0.0 if act == "sigmoid" else 1.0
    want = torch.tensor([low] * 4 + [high] * 4, device="cuda")
    got = Z.linear_backward(d, x, w, act="none" if act == "none" else act, pre=z, need_dx=False, need_dw=False)[2]
    gate = Z.glu_backward(d, x, w, w, z, d, act=act, need_dx=False, need_dw=False)[3]
    for g in (gate,) if act == "none" else (got, gate):
        assert torch.equal(g[:8], want) and (act == "none" or g[8].isnan())


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_no_activation_has_a_slope_of_one(t):
    """A NaN of the gate reaches up's gradient, which it multiplies, and not its own."""
    import zeromoe_amd as Z

    S, I, F = 20, 264, 100
    x, w, dy, gate, up = (rand(*s, seed=i, dtype=t) for i, s in enumerate(((S, I), (F, I), (S, F), (S, F), (S, F))))
    gate[3, 7] = math.nan
    dx, dwg, dwu, dbg, dbu = Z.glu_backward(dy, x, w, w, gate, up, act="none")
    assert dwg.isfinite().all() and dbg.isfinite().all()
    for m in (dwu, dbu):
        assert m[7].isnan().all() and m[:7].isfinite().all() and m[8:].isfinite().all()
    assert dx[3].isnan().all() and dx[:3].isfinite().all() and dx[4:].isfinite().all()
