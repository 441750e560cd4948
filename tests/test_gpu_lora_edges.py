"""Adapters where the formula leaves the ordinary: infinities, scales of adapters that no token names, and the backward pass
of few tokens whose long axis is shared by several workgroups.  Tolerances as in test_gpu_lora."""
import math

import pytest
import torch

from test_gpu_dense import PAIRS, TYPES, U, rand
from test_gpu_lora import adapters, check_backward, some_ids

pytestmark = pytest.mark.gpu


# ids of one slice of tokens for each adapter, and of several (few columns and more than 512 tokens)
@pytest.mark.parametrize("xt,wt", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("S,I,O,R", [(3, 72, 40, 5), (700, 264, 520, 16), (6000, 128, 96, 24), (40, 300, 8192, 65)])
def test_scale_of_an_adapter_without_tokens(S, I, O, R, xt, wt):
    """Nothing reads it: zeros for its gradients, and all other results as with a scale of 1 in its place."""
    import zeromoe_amd as Z

    n = 5
    a, b = adapters(n, R, I, O, wt)
    x, dy, v = rand(S, I, seed=3, dtype=TYPES[xt]), rand(S, O, seed=4, dtype=TYPES[xt]), rand(S, R, seed=5)
    ids = torch.tensor([1, 3], device="cuda", dtype=torch.int32)[some_ids(S, 2, "runs").long()]
    scale = rand(n, seed=6)
    scale[0], scale[2], scale[4] = math.inf, math.nan, -math.inf
    good = scale.nan_to_num(1.0, 1.0, 1.0)
    got = (Z.lora(x, a, b, ids, scale=scale), *Z.lora_backward(dy, x, a, b, ids, v, scale=scale))
    want = (Z.lora(x, a, b, ids, scale=good), *Z.lora_backward(dy, x, a, b, ids, v, scale=good))
    for g, w in zip(got, want):
        assert torch.equal(g, w)
    for g in got[2:]:
        assert (g[[0, 2, 4]] == 0).all()


# O of several slices in the backward pass, ranks of each kind of kernel, odd sizes
SPLIT = [(1, 520, 8200, 128, 3), (63, 300, 8192, 65, 1), (40, 260, 4099, 200, 3), (5, 1030, 4608, 30, 2), (2, 2100, 8191, 16, 1),
         (100, 131, 5121, 100, 4)]


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S,I,O,R,n", SPLIT)
def test_backward_of_few_tokens_and_a_long_axis(S, I, O, R, n, xt, wt):
    for need in ((True, True, True), (True, False, False), (False, True, False)):
        check_backward(S, I, O, R, n, xt, wt, need=need)
    check_backward(S, I, O, R, n, xt, wt, "one", ydt="f32", seed=21)


def same_as(got, want, ok, what):
    """An infinity for an infinity, a NaN for a NaN, a finite value for a finite one, wherever the signs are sure."""
    inf = want.isinf() & ok
    assert torch.equal(got.isnan() & ok, want.isnan() & ok) and torch.equal(got.isinf() & ok, inf), what
    assert torch.equal(got.double()[inf], want[inf]), what


def by_definition(p, p_ok, q):
    """p (S, K) times q (J, K)^T in 64 bits, each product formed (an infinity times zero is a NaN), and where its sign is
    sure: not where the sum is within 1e-4 of its terms from zero (f32 sums are off by far less), nor where such a p meets
    an infinity of q.  Signs matter only where an infinity follows."""
    few = max(1, (1 << 26) // p.numel())
    y, size = (torch.cat([f(p[:, None] * c[None]).sum(-1) for c in q.split(few)], 1) for f in (lambda t: t, torch.abs))
    unsure = ((~p_ok).double() @ q.isinf().double().t().contiguous()) > 0
    return y, ~unsure & (~y.isfinite() | (y.abs() > 1e-4 * size)), ~unsure


# tokens, widths and ranks of the kernel of few tokens, of the items, and of items whose axes are launches of their own
KINDS = [(12, 264, 72, 1), (12, 264, 300, 9), (12, 8200, 72, 72), (12, 8193, 40, 130), (5000, 260, 72, 1), (5000, 136, 100, 24),
         (4500, 96, 130, 50), (4300, 72, 65, 100), (40, 9000, 260, 128), (300, 4100, 257, 33)]


def unusual(S, I, O, R, xt, wt):
    """Four adapters; infinities in x, a, b and the scale, each reaching tokens of its own among the first twelve."""
    a, b = adapters(4, R, I, O, wt)
    x = rand(S, I, seed=3, dtype=TYPES[xt])
    ids = torch.arange(S, device="cuda").remainder(4).to(torch.int32)
    scale = torch.tensor([1.5, -0.5, 2.0, 1.0], device="cuda")
    b[:] = b.abs() + 0.01
    a[0, :, 5] = a[0, :, 5].abs() + 0.01  # x: infinities of one sign in v
    x[0, 5], x[4, 5] = math.inf, -math.inf
    x[8, 7] = math.inf                    # of both
    a[1, R // 2, 9] = math.inf            # one adapter's v by the sign of x
    x[5, 9] = 0.0                         # (and zero times it)
    b[2, 3, R - 1] = -math.inf            # one adapter's column
    scale[3] = math.inf                   # one adapter's rows
    return x, a, b, ids, scale


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S,I,O,R", KINDS)
def test_infinities_go_by_the_formula(S, I, O, R, xt, wt):
    import zeromoe_amd as Z

    x, a, b, ids, scale = unusual(S, I, O, R, xt, wt)
    res = rand(S, O, seed=8, dtype=TYPES[xt])
    res[7, 1] = -math.inf
    y, v = Z.lora(x, a, b, ids, scale=scale, residual=res, save=True)
    for e in range(4):
        at = (ids == e).nonzero()[:, 0]
        v64, v_ok, ok = by_definition(x[at].double(), torch.ones(len(at), I, device="cuda", dtype=torch.bool), a[e].double())
        same_as(v[at], v64, ok, ("v", e))
        y64, y_ok, ok = by_definition(v64, v_ok, b[e].double())
        same_as(y[at], y64 * scale[e].double() + res[at].double(), ok if scale[e].isfinite() else y_ok, ("y", e))


@pytest.mark.parametrize("S,I,O,R", KINDS)
def test_one_token_and_many_agree_on_infinities(S, I, O, R):
    """The same rows alone: infinities and NaN in the same places."""
    import zeromoe_amd as Z

    x, a, b, ids, scale = unusual(S, I, O, R, "bf16", "bf16")
    y = Z.lora(x, a, b, ids, scale=scale)
    for s in range(12):
        one = Z.lora(x[s:s + 1], a, b, ids[s:s + 1], scale=scale)[0]
        same_as(one, y[s].double(), torch.ones_like(one, dtype=torch.bool), s)


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S,I,O,R", [(12, 264, 72, 1), (12, 264, 300, 9), (12, 72, 8200, 72), (5000, 130, 96, 1),
                                     (5000, 100, 136, 24), (4500, 130, 72, 50), (40, 260, 4100, 128), (1030, 64, 33, 100)])
def test_gradients_of_infinities_go_by_the_formula(S, I, O, R, xt, wt):
    import zeromoe_amd as Z

    a, b = adapters(4, R, I, O, wt)
    x, dy, v = rand(S, I, seed=3, dtype=TYPES[xt]), rand(S, O, seed=4, dtype=TYPES[xt]), rand(S, R, seed=5)
    ids = torch.arange(S, device="cuda").remainder(4).to(torch.int32)
    scale = torch.tensor([1.5, -0.5, 2.0, math.inf], device="cuda")
    a[0] = a[0].abs() + 0.01
    b[0, 5] = b[0, 5].abs() + 0.01
    dy[4, 5] = math.inf            # u of one token, all of its dx, da of the adapter
    x[1, 3] = -math.inf            # one column of da
    v[5, R // 2] = math.inf        # one column of db
    b[2, 7, R - 1] = math.inf      # one r of u
    dx, da, db = Z.lora_backward(dy, x, a, b, ids, v, scale=scale)
    for e in range(4):
        at, c = (ids == e).nonzero()[:, 0], scale[e].double()
        d, xe, ve = dy[at].double(), x[at].double(), v[at].double()
        sure = torch.ones(len(at), O, device="cuda", dtype=torch.bool)
        u, u_ok, _ = by_definition(d, sure, b[e].double().t().contiguous())
        t = lambda m: m.t().contiguous()  # noqa: E731
        for name, got, (want, last, ok) in (("dx", dx[at], by_definition(u, u_ok, t(a[e].double()))),
                                            ("da", da[e], by_definition(t(u), t(u_ok), t(xe))),
                                            ("db", db[e], by_definition(t(d), t(sure), t(ve)))):
            same_as(got, want * c, ok if c.isfinite() else last, (name, e))


def test_gradients_of_the_widest_rows():
    """An adapter of 2^29 columns: its gradient takes more workgroups than one launch has."""
    import zeromoe_amd as Z

    I, O = (1 << 29) + 70, 40
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    a = torch.randn((1, 1, I), device="cuda", generator=g, dtype=torch.bfloat16)
    x = torch.randn((2, I), device="cuda", generator=g, dtype=torch.bfloat16)
    b, dy, v = rand(1, O, 1, seed=2, dtype=torch.bfloat16), rand(2, O, seed=3, dtype=torch.bfloat16), rand(2, 1, seed=4)
    ids, scale = torch.tensor([-1, 0], device="cuda", dtype=torch.int32), torch.tensor([0.5], device="cuda")
    dx, da, db = Z.lora_backward(dy, x, a, b, ids, v, scale=scale)
    u = (dy[1].double() @ b[0, :, 0].double()).item()
    # u in f32: O products, as in test_gpu_lora; one product with it, the scale, and the rounding of the result
    tu = U * (4 + 2 * math.sqrt(O)) * (dy[1].double().abs() @ b[0, :, 0].double().abs()).item()
    assert not dx[0].any()
    for at in range(0, I, 1 << 26):
        k = slice(at, min(at + (1 << 26), I))
        for got, m, step in ((da[0, 0, k], x[1, k], U), (dx[1, k], a[0, 0, k], 2.0 ** -8)):
            want = 0.5 * u * m.double()
            tol = 0.5 * tu * m.double().abs() + (step + 4 * U) * want.abs() + 1e-37
            assert ((got.double() - want).abs() <= tol).all()
    want = 0.5 * dy[1].double() * v[1].double()
    assert ((db[0, :, 0].double() - want).abs() <= 4 * U * want.abs() + 1e-37).all()
