"""The norm of many gradients and their clipping against 64 bits.

Tolerances.  The norm is summed in f64 (n 2^-53 of itself, nothing beside f32) and rounded to f32 once: 2^-24.  A clipped
value is a product in f64, rounded to f32 and from there to its type: 2^-24 + eps / 2."""
import math

import pytest
import torch

from test_gpu_dense import TYPES, U, rand

pytestmark = pytest.mark.gpu


def norm64(grads):
    return math.sqrt(math.fsum((g.double() ** 2).sum().item() for g in grads))


def check_norm(got, grads):
    want = norm64(grads)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(got.item() - want) <= 1.01 * U * want + 1e-45, (got.item(), want)
    return want


def check_clip(grads, max_norm, eps=1e-6, out=None):
    import zeromoe_amd as Z

    before = [g.clone() for g in grads]
    got = Z.clip_grad_norm(grads, max_norm, eps=eps, out=out)
    want = check_norm(got, before)
    c = min(1.0, max_norm / (want + eps)) if want + eps > 0 else 1.0  # (max_norm / 0: an infinity)
    for i, (b, r) in enumerate(zip(before, grads if out is None else out)):
        exact = b.double() * c
        half = torch.finfo(r.dtype).eps / 2 if r.dtype != torch.float32 else 0.0
        least = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[r.dtype]
        err = (r.double() - exact).abs()
        assert (err <= (1.01 * U + half) * exact.abs() + least).all(), (i, b.shape)
        if out is not None:
            assert torch.equal(grads[i], b)
        elif c == 1.0:
            assert torch.equal(r, b)


SIZES = [[1], [4096], [5], [4095, 1, 4097], [1000, 3, 70000, 0, 17], [1 << 20, 12345], [7] * 119, [33] * 120, [129] * 121,
         [2049] * 400, [3] * 1000, [0, 0], [5_000_011]]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16", "mixed"])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_clip(sizes, t):
    import zeromoe_amd as Z

    types = list(TYPES) if t == "mixed" else [t]
    grads = [rand(n, seed=i, dtype=TYPES[types[i % len(types)]]) for i, n in enumerate(sizes)]
    check_norm(Z.grad_norm(grads), grads)
    norm = norm64(grads)
    check_clip([g.clone() for g in grads], 0.3 * norm + 1e-3)
    check_clip([g.clone() for g in grads], 2.0 * norm + 1.0)
    check_clip(grads, 0.3 * norm + 1e-3, out=[torch.full_like(g, 9.0) for g in grads])
    check_clip(grads, 2.0 * norm + 1.0, out=[torch.full_like(g, 9.0) for g in grads])
    check_clip(grads, 0.1 * norm + 1e-3, eps=0.0, out=[torch.full_like(g, 9.0, dtype=torch.float32) for g in grads])


@pytest.mark.parametrize("t", list(TYPES))
def test_clip_at_any_address(t):
    """Gradients and results as pieces of flat buffers, one after the other or with gaps, whose neighbours stay."""
    sizes = [3, 4096, 1, 8191, 64, 5000, 2]
    for gap in (0, 1, 5):
        total = sum(sizes) + gap * (len(sizes) + 1)
        flat, res = rand(total, seed=1, dtype=TYPES[t]), torch.full((total + 3,), 7.0, device="cuda", dtype=TYPES[t])
        at, grads, out, keep = gap, [], [], torch.ones(total + 3, dtype=torch.bool, device="cuda")
        for n in sizes:
            grads.append(flat[at:at + n])
            out.append(res[at + 3:at + 3 + n])
            keep[at + 3:at + 3 + n] = False
            at += n + gap
        check_clip(grads, 0.5, out=out)
        assert (res[keep] == 7.0).all()
        hold = flat.clone()
        check_clip(grads, 0.5)
        assert torch.equal(flat[:gap], hold[:gap])


def test_clip_orders_of_dimensions():
    import zeromoe_amd as Z

    a, b = rand(40, 70, seed=1).t(), rand(3, 5, 7, seed=2).permute(2, 0, 1)
    c = rand(64, 128, seed=3)[:, :100]
    check_clip([a, b, rand(1, 9, seed=4)[:, None]], 0.25)
    check_norm(Z.grad_norm([a, c]), [a, c])
    check_norm(Z.grad_norm(c), [c])
    with pytest.raises(ValueError, match="one piece of memory"):
        Z.clip_grad_norm([a, c], 1.0)
    with pytest.raises(ValueError, match="strides"):
        Z.clip_grad_norm([a], 1.0, out=[torch.empty(70, 40, device="cuda")])


def test_clip_of_extreme_values():
    """Squares past f32's range, below it, and both together; a coefficient below f32's smallest number."""
    import zeromoe_amd as Z

    big, small = torch.full((5000,), 3e38, device="cuda"), torch.full((5000,), 1e-38, device="cuda")
    check_norm(Z.grad_norm([small]), [small])
    assert Z.grad_norm([big]).isinf()  # sqrt(5000) 3e38 is past f32
    n64 = math.sqrt(5000) * big.double()[0].item()
    out = [torch.empty_like(big)]
    Z.clip_grad_norm([big], 1.0, out=out)
    want = big.double() / n64
    assert ((out[0].double() - want).abs() <= 1.01 * U * want).all()
    check_clip([torch.full((3,), 1e38, device="cuda"), small], 1e-3)
    check_clip([small.clone()], 1e-40, eps=0.0)
    check_clip([rand(100, seed=1).to(torch.float16) * 1e-6], 1e-7)
    check_clip([rand(100, seed=1), torch.zeros(50, device="cuda")], 0.0)
    check_clip([torch.zeros(50, device="cuda")], 1.0)
    check_clip([rand(1000, seed=2)], math.inf)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_clip_of_what_is_not_finite(bad):
    """By the formula: an infinite norm makes finite values 0 and infinities NaN, a NaN makes all NaN."""
    import zeromoe_amd as Z

    a, b = rand(5000, seed=1), rand(300, seed=2, dtype=torch.bfloat16)
    a[4321] = bad
    norm = Z.clip_grad_norm([a, b], 1.0)
    if math.isnan(bad):
        assert norm.isnan() and a.isnan().all() and b.isnan().all()
    else:
        assert norm.item() == math.inf and a[4321].isnan() and (b == 0).all()
        assert (a[:4321] == 0).all() and (a[4322:] == 0).all()


def test_clip_refusals_on_device():
    import zeromoe_amd as Z

    a = rand(100, seed=1)
    for grads, out in (([a, a], None), ([a[:60], a[50:]], None), ([a[:50], a[50:]], [a[50:], a[:50]]),
                       ([a[:50]], [a[1:51]]), ([rand(50), rand(50)], [a[:50], a[:50]])):
        with pytest.raises(RuntimeError, match="overlaps"):
            Z.clip_grad_norm(grads, 1.0, out=out)
    check_clip([a, rand(3)], 1.0, out=[torch.empty_like(a), torch.empty(3, device="cuda")])
    check_norm(Z.grad_norm([a, a]), [a, a])
    for m, e in ((-1.0, 0.0), (math.nan, 0.0), (1.0, -1.0), (1.0, math.inf), (1.0, math.nan)):
        with pytest.raises(RuntimeError, match="max_norm"):
            Z.clip_grad_norm([a], m, eps=e)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        Z.grad_norm([a.double()])
    with pytest.raises(ValueError, match="device"):
        Z.grad_norm([a, torch.zeros(3)])
    with pytest.raises(ValueError, match="results"):
        Z.clip_grad_norm([a], 1.0, out=[a, a])
    with pytest.raises(ValueError, match="float32 needed"):
        Z.clip_grad_norm([a], 1.0, out=[a.half()])
    with pytest.raises(ValueError, match="requires a gradient"):
        Z.clip_grad_norm([a.clone().requires_grad_()], 1.0)
    with torch.no_grad():
        Z.grad_norm([a.clone().requires_grad_()])


def test_clip_graph_streams_and_bits():
    import zeromoe_amd as Z

    grads = [rand(n, seed=n) for n in (100000, 7, 4097, 33)] * 1
    out = [torch.empty_like(g) for g in grads]
    first = Z.clip_grad_norm(grads, 0.5, out=out)
    hold = [o.clone() for o in out]
    for _ in range(3):
        assert torch.equal(Z.clip_grad_norm(grads, 0.5, out=out), first)
        assert all(torch.equal(a, b) for a, b in zip(out, hold))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = Z.clip_grad_norm(grads, 0.5, out=out)
    for seed in (1, 2, 3):
        for g in grads:
            g.copy_(rand(*g.shape, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        got, res = norm.clone(), [o.clone() for o in out]
        assert torch.equal(Z.clip_grad_norm(grads, 0.5, out=out), got) and all(torch.equal(a, b) for a, b in zip(out, res))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    n = Z.grad_norm(grads, stream=side)
    side.synchronize()
    assert torch.equal(n, got)


def test_norm_of_more_than_32_bits():
    """2^31 values and more in one tensor."""
    import zeromoe_amd as Z

    n = (1 << 31) + 12345
    g = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g[-1], g[0], g[1 << 30] = 3.0, 4.0, 12.0
    assert Z.grad_norm([g]).item() == 13.0
    assert Z.clip_grad_norm([g], 6.5, eps=0.0).item() == 13.0
    assert g[-1].item() == 1.5 and g[0].item() == 2.0 and g[1 << 30].item() == 6.0
