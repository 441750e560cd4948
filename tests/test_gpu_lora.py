"""Adapters that each token names, and their gradients, against their definition in 64 bits.

Tolerances.  v is a sum of I products in f32, y one of R products with it: (4 + 2 sqrt n) 2^-24 of the sum of their absolute
values, as for linear (test_gpu_dense), the first carried through |b|; scale and residual add a few roundings; the last
rounding is eps / 2 of the result's type.  The gradients likewise, each over its own axis."""
import math

import pytest
import torch

from test_gpu_dense import PAIRS, TYPES, U, close, half_step, rand, sum_tol

pytestmark = pytest.mark.gpu


def least(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 1e-37


def some_ids(S, n, kind, seed=5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if kind == "runs":
        ids = torch.sort(torch.randint(0, n, (S,), device="cuda", generator=g))[0]
    elif kind == "one":
        ids = torch.full((S,), n - 1, device="cuda")
    elif kind == "none":
        ids = torch.full((S,), -1, device="cuda")
    else:
        ids = torch.randint(0, n, (S,), device="cuda", generator=g)
        ids[torch.rand(S, device="cuda", generator=g) < 0.2] = -1
    return ids.to(torch.int32)


def adapters(n, R, I, O, wt, seed=1):
    return (rand(n, R, I, seed=seed, scale=1 / math.sqrt(I), dtype=TYPES[wt]),
            rand(n, O, R, seed=seed + 1, scale=0.7 / math.sqrt(R), dtype=TYPES[wt]))


def lora64(x, a, b, ids, scale):
    """(v, its tolerance, delta, its tolerance)"""
    S, R, O = x.shape[0], a.shape[1], b.shape[1]
    v, tv = (torch.zeros(S, R, device="cuda", dtype=torch.float64) for _ in range(2))
    y, ty = (torch.zeros(S, O, device="cuda", dtype=torch.float64) for _ in range(2))
    for e in range(a.shape[0]):
        at = (ids == e).nonzero()[:, 0]
        if not len(at):
            continue
        xe, ae, be, c = x[at].double(), a[e].double(), b[e].double(), 1.0 if scale is None else scale[e].double()
        v[at] = xe @ ae.t()
        tv[at] = sum_tol(x.shape[1], xe.abs() @ ae.abs().t())
        y[at] = c * (v[at] @ be.t())
        ab = v[at].abs() @ be.abs().t()
        ty[at] = abs(c) * (sum_tol(R, ab) + 4 * U * ab + (1 + 32 * U) * (tv[at] @ be.abs().t()))
    return v, tv, y, ty


def check_lora(S, I, O, R, n, xt, wt, kind="mixed", residual=True, scaled=True, ydt=None, seed=1, x=None, a=None, b=None,
               ids=None, out=None, save=True, res=None):
    import zeromoe_amd as Z

    dtype = TYPES[ydt or xt]
    x = rand(S, I, seed=seed, dtype=TYPES[xt]) if x is None else x
    if a is None:
        a, b = adapters(n, R, I, O, wt, seed + 1)
    ids = some_ids(S, n, kind) if ids is None else ids
    scale = rand(n, seed=seed + 3) if scaled else None
    if res is None and residual:
        res = rand(S, O, seed=seed + 4, dtype=dtype)
    hold = None if res is None else res.double()
    y = Z.lora(x, a, b, ids, scale=scale, residual=res, out=out, out_dtype=dtype, save=save)
    v64, tv, y64, ty = lora64(x, a, b, ids, scale)
    if save:
        y, v = y
        assert v.dtype == torch.float32 and v.shape == (S, R)
        close(v, v64, tv + U * v64.abs() + 1e-37)
        assert (v[ids < 0] == 0).all()
    if hold is not None:
        y64 = y64 + hold
        ty = ty + 2 * U * hold.abs()
    assert y.dtype == dtype and y.shape == (S, O)
    close(y, y64, ty + (U + half_step(dtype)) * y64.abs() + least(dtype))
    if hold is not None:
        assert torch.equal(y[ids < 0].double(), hold[ids < 0])
    return y


# few tokens, and with ranks above 64 or many tokens the bucketed kernels
SHAPES = [(1, 1, 1, 1, 1), (1, 4096, 513, 16, 9), (3, 72, 40, 5, 2), (17, 264, 700, 8, 64), (40, 1000, 31, 20, 3),
          (64, 2048, 1100, 64, 7), (130, 257, 129, 33, 5), (700, 520, 264, 16, 4), (1500, 96, 260, 100, 300),
          (2100, 1288, 72, 32, 11), (900, 512, 512, 128, 2), (3000, 136, 136, 4, 512)]


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S,I,O,R,n", SHAPES)
def test_lora(S, I, O, R, n, xt, wt):
    for kind in ("mixed", "runs"):
        check_lora(S, I, O, R, n, xt, wt, kind)
    check_lora(S, I, O, R, n, xt, wt, residual=False, scaled=False, save=False, ydt="f32", seed=11)


# sizes that few_tokens leaves to the bucketed kernels, from one token on
BIG = [(1, 8200, 600, 128, 3), (5, 8192, 130, 256, 2), (40, 9000, 260, 64, 40), (63, 8192, 300, 65, 1), (64, 8195, 72, 129, 2),
       (65, 8192, 40, 200, 3), (5000, 520, 520, 16, 3), (4999, 511, 333, 24, 60), (8200, 260, 100, 7, 5)]


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S,I,O,R,n", BIG)
def test_lora_bucketed(S, I, O, R, n, xt, wt):
    for kind in ("mixed", "runs", "one", "none"):
        check_lora(S, I, O, R, n, xt, wt, kind)


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S,I,R", [(6, 264, 12), (100, 8200, 72), (5000, 260, 12)])
def test_lora_strides_and_alignment(xt, wt, S, I, R):
    """Rows, adapters and results that lie apart, on odd addresses; neighbours of the result stay as they are."""
    n, O = 3, 72
    for off, pad in ((0, 8), (1, 8), (3, 5)):
        x = rand(S * (I + pad) + 16, seed=3, dtype=TYPES[xt])[off:off + S * (I + pad)].view(S, I + pad)[:, :I]
        a = rand(n * (R + 1) * (I + pad) + 16, seed=4, scale=0.05, dtype=TYPES[wt])[off:off + n * (R + 1) * (I + pad)].view(
            n, R + 1, I + pad)[:, :R, :I]
        b = rand(n * (O + 2) * (R + pad) + 16, seed=6, scale=0.2, dtype=TYPES[wt])[off:off + n * (O + 2) * (R + pad)].view(
            n, O + 2, R + pad)[:, 1:O + 1, :R]
        buf = torch.full((S + 2, O + pad + off), 7.0, device="cuda", dtype=TYPES[xt])
        res = rand(S, O + pad, seed=8, dtype=TYPES[xt])[:, :O]
        check_lora(S, I, O, R, n, xt, wt, x=x, a=a, b=b, out=buf[1:S + 1, off:off + O], res=res)
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep[1:S + 1, off:off + O] = False
        assert (buf[keep] == 7.0).all()
    y = rand(S, O, seed=9, dtype=TYPES[xt])
    check_lora(S, I, O, R, n, xt, wt, res=y, out=y)  # in place
    one = rand(1, R, I, seed=10, scale=0.05, dtype=TYPES[wt]).expand(n, R, I)  # all adapters share their a
    check_lora(S, I, O, R, n, xt, wt, x=rand(1, I, seed=2, dtype=TYPES[xt]).expand(S, I), a=one,
               b=adapters(n, R, I, O, wt)[1])


def check_backward(S, I, O, R, n, xt, wt, kind="mixed", scaled=True, ydt=None, seed=1, need=(True, True, True), x=None, a=None,
                   b=None, dy=None, v=None, ids=None):
    import zeromoe_amd as Z

    dtype, yt = TYPES[xt], TYPES[ydt or xt]
    x = rand(S, I, seed=seed, dtype=dtype) if x is None else x
    if a is None:
        a, b = adapters(n, R, I, O, wt, seed + 1)
    ids = some_ids(S, n, kind) if ids is None else ids
    scale = rand(n, seed=seed + 3) if scaled else None
    dy = rand(S, O, seed=seed + 4, scale=0.1, dtype=yt) if dy is None else dy
    v = rand(S, R, seed=seed + 5) if v is None else v
    r = Z.lora_backward(dy, x, a, b, ids, v, scale=scale, need_dx=need[0], need_da=need[1], need_db=need[2])
    assert [t is None for t in r] == [not k for k in need]
    dx, da, db = r
    if dx is not None:
        assert dx.dtype == dtype and dx.shape == (S, I) and (dx[ids < 0] == 0).all()
    for e in range(n):
        at = (ids == e).nonzero()[:, 0]
        c = 1.0 if scale is None else scale[e].double()
        d, xe, ae, be, ve = (t.double() for t in (dy[at], x[at], a[e], b[e], v[at]))
        u = d @ be
        tu = sum_tol(O, d.abs() @ be.abs())
        if dx is not None and len(at):
            want, absdot = c * (u @ ae), abs(c) * (u.abs() @ ae.abs())
            close(dx[at], want, sum_tol(R, absdot) + 4 * U * absdot + abs(c) * 1.01 * (tu @ ae.abs())
                  + (U + half_step(dtype)) * want.abs() + least(dtype))
        if da is not None:
            want, absdot = c * (u.t() @ xe), abs(c) * (u.abs().t() @ xe.abs())
            close(da[e], want, sum_tol(len(at), absdot) + 4 * U * absdot + abs(c) * 1.01 * (tu.t() @ xe.abs()))
        if db is not None:
            want, absdot = c * (d.t() @ ve), abs(c) * (d.abs().t() @ ve.abs())
            close(db[e], want, sum_tol(len(at), absdot) + 4 * U * absdot)
        if not len(at):
            assert (da is None or (da[e] == 0).all()) and (db is None or (db[e] == 0).all())


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S,I,O,R,n", [(1, 1, 1, 1, 1), (1, 4096, 513, 16, 9), (3, 72, 40, 5, 2), (17, 264, 700, 8, 40),
                                       (130, 257, 129, 33, 5), (700, 520, 264, 16, 4), (1500, 96, 260, 100, 30),
                                       (900, 512, 512, 128, 2), (65, 1024, 40, 200, 3), (5000, 136, 264, 4, 1)])
def test_lora_backward(S, I, O, R, n, xt, wt):
    for kind in ("mixed", "runs"):
        check_backward(S, I, O, R, n, xt, wt, kind)
    check_backward(S, I, O, R, n, xt, wt, scaled=False, ydt="f32", seed=11)


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (False, True, True)])
@pytest.mark.parametrize("S,R", [(3, 8), (70, 40), (3000, 16)])
def test_lora_backward_parts(need, S, R):
    check_backward(S, 520, 1030, R, 5, "bf16", "bf16", need=need)
    check_backward(S, 520, 1030, R, 5, "f32", "f16", "none", need=need)


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S,R", [(6, 12), (500, 12), (90, 70)])
def test_lora_backward_strides_and_alignment(xt, wt, S, R):
    n, I, O = 3, 264, 72
    for off, pad in ((0, 8), (1, 8), (3, 5)):
        x = rand(S * (I + pad) + 16, seed=3, dtype=TYPES[xt])[off:off + S * (I + pad)].view(S, I + pad)[:, :I]
        dy = rand(S * (O + pad) + 16, seed=5, dtype=TYPES[xt])[off:off + S * (O + pad)].view(S, O + pad)[:, :O]
        a = rand(n * (R + 1) * (I + pad) + 16, seed=4, scale=0.05, dtype=TYPES[wt])[off:off + n * (R + 1) * (I + pad)].view(
            n, R + 1, I + pad)[:, :R, :I]
        b = rand(n * (O + 2) * (R + pad) + 16, seed=6, scale=0.2, dtype=TYPES[wt])[off:off + n * (O + 2) * (R + pad)].view(
            n, O + 2, R + pad)[:, 1:O + 1, :R]
        check_backward(S, I, O, R, n, xt, wt, x=x, a=a, b=b, dy=dy)
    check_backward(S, I, O, R, n, xt, wt, dy=rand(1, O, seed=2, dtype=TYPES[xt]).expand(S, O))


@pytest.mark.parametrize("S,I,R", [(40, 264, 12), (5000, 264, 12), (30, 8200, 72)])
def test_lora_rows_without_a_valid_adapter(S, I, R):
    """NaN rows for ids past the last adapter and zeros for negative ones, whatever lies in x, dy and v there; all other
    rows and the adapters' gradients as without them."""
    import zeromoe_amd as Z

    n, O = 4, 300
    a, b = adapters(n, R, I, O, "f32")
    x, dy, v, ids = rand(S, I, seed=3), rand(S, O, seed=4), rand(S, R, seed=6), some_ids(S, n, "mixed")
    ids[3], ids[7], ids[8], ids[-1] = n, 1 << 30, -(1 << 31), n + 5
    bad = (ids < 0) | (ids >= n)
    x[bad], dy[bad], v[bad] = math.nan, math.inf, math.nan
    y, vs = Z.lora(x, a, b, ids, save=True)
    dx, da, db = Z.lora_backward(dy, x, a, b, ids, v)
    for t in (y, vs, dx):
        assert t[ids >= n].isnan().all() and (t[ids < 0] == 0).all() and t[~bad].isfinite().all()
    res = rand(S, O, seed=8)
    z = Z.lora(x, a, b, ids, residual=res)
    assert z[ids >= n].isnan().all() and torch.equal(z[ids < 0], res[ids < 0])
    keep = ~bad
    for got, want in zip((da, db), Z.lora_backward(dy[keep], x[keep], a, b, ids[keep], v[keep])[1:]):
        assert got.isfinite().all() and (got - want).abs().max() <= 1e-5 * want.abs().max()
    _, _, y64, ty = lora64(x[keep], a, b, ids[keep], None)
    y64 = y64 + res[keep].double()
    close(z[keep], y64, ty + 2 * U * res[keep].double().abs() + 2 * U * y64.abs() + 1e-37)


@pytest.mark.parametrize("counts", [(4096,), (4097,), (4095, 0, 1), (2049, 2032), (2050, 2033, 0, 0, 7), (16 * 250 + 1, 1, 1, 1, 1),
                                    (16 * 250 + 1, 1, 1, 1, 1, 1), tuple([17] * 128), tuple([17] * 129), (4096, 1500), (5500, 0)])
def test_lora_tokens_of_an_item(counts):
    """Up to 256 groups of 16 tokens of an adapter, and more (which are taken 32 at a time), with tokens of none between."""
    n, I, O, R = len(counts), 1032, 264, 16
    ids = torch.cat([torch.full((c,), e) for e, c in enumerate(counts)] + [torch.full((300,), -1)])
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(1))].to(torch.int32).cuda()
    check_lora(len(ids), I, O, R, n, "bf16", "bf16", ids=ids)
    check_backward(len(ids), I, O, R, n, "bf16", "bf16", ids=ids)


def test_lora_no_tokens():
    import zeromoe_amd as Z

    a, b = adapters(2, 4, 72, 24, "f32")
    ids = torch.zeros(0, device="cuda", dtype=torch.int32)
    y, v = Z.lora(rand(0, 72), a, b, ids, save=True)
    assert y.shape == (0, 24) and v.shape == (0, 4)
    dx, da, db = Z.lora_backward(y, rand(0, 72), a, b, ids, v)
    assert dx.shape == (0, 72) and da.shape == a.shape and db.shape == b.shape and (da == 0).all() and (db == 0).all()


def test_lora_graph_streams_and_bits():
    import zeromoe_amd as Z

    for S, I, O, R, n in ((24, 512, 300, 16, 8), (6000, 264, 300, 16, 8)):
        a, b = adapters(n, R, I, O, "bf16")
        x, dy, ids = rand(S, I, seed=3, dtype=torch.bfloat16), rand(S, O, seed=4, dtype=torch.bfloat16), some_ids(S, n, "mixed")
        scale, res = rand(n, seed=5), rand(S, O, seed=6, dtype=torch.bfloat16)

        def step():
            y, v = Z.lora(x, a, b, ids, scale=scale, residual=res, save=True)
            return (y, v, *Z.lora_backward(dy, x, a, b, ids, v, scale=scale))

        first = step()
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(first, step()))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for seed in (5, 6, 7):
            x.copy_(rand(S, I, seed=seed))
            ids.copy_(some_ids(S, n, "runs" if seed == 6 else "mixed", seed))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs, step()))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        y = Z.lora(x, a, b, ids, scale=scale, residual=res, stream=side)
        side.synchronize()
        assert torch.equal(y, outs[0])


def test_lora_offsets_past_32_bits():
    """Activations, adapters and results of more than 2^31 values: the last ones against the same by themselves."""
    import zeromoe_amd as Z

    S, I, O, R = (1 << 20) + 70, 2056, 72, 8
    a, b = adapters(2, R, I, O, "bf16")
    x = torch.zeros(S, I, device="cuda", dtype=torch.bfloat16)
    x[-70:] = rand(70, I, seed=3, dtype=torch.bfloat16)
    ids = torch.full((S,), -1, device="cuda", dtype=torch.int32)
    ids[-70:] = some_ids(70, 2, "runs")
    y, v = Z.lora(x, a, b, ids, save=True)
    v64, tv, y64, ty = lora64(x[-70:], a, b, ids[-70:], None)
    close(v[-70:], v64, tv + U * v64.abs())
    close(y[-70:], y64, ty + (U + 2.0 ** -8) * y64.abs())
    assert (y[:-70] == 0).all()
    dy = torch.zeros(S, O, device="cuda", dtype=torch.bfloat16)
    dy[-70:] = rand(70, O, seed=4, dtype=torch.bfloat16)
    dx, da, db = Z.lora_backward(dy, x, a, b, ids, v)
    assert (dx[:-70] == 0).all()
    for e in range(2):
        at = (ids[-70:] == e).nonzero()[:, 0]
        u = dy[-70:][at].double() @ b[e].double()
        want = u.t() @ x[-70:][at].double()
        assert (da[e].double() - want).abs().max() <= 1e-5 * want.abs().max()
        want = dy[-70:][at].double().t() @ v[-70:][at].double()
        assert (db[e].double() - want).abs().max() <= 1e-5 * want.abs().max()
    del x, y, dx, dy
    n, R, I, O = 300, 200, 40000, 64  # a: 2.4e9 values
    a = torch.zeros(n, R, I, device="cuda", dtype=torch.bfloat16)
    a[-1] = rand(R, I, seed=5, scale=0.01, dtype=torch.bfloat16)
    b = rand(n, O, R, seed=6, dtype=torch.bfloat16)
    for S in (2, 70):
        x = rand(S, I, seed=7, dtype=torch.bfloat16)
        ids = torch.full((S,), n - 1, device="cuda", dtype=torch.int32)
        y = Z.lora(x, a, b, ids)
        _, _, y64, ty = lora64(x, a[-1:], b[-1:], torch.zeros_like(ids), None)
        close(y, y64, ty + (U + 2.0 ** -8) * y64.abs() + 1e-37)
        dx, _, _ = Z.lora_backward(y, x, a, b, ids, need_da=False, need_db=False)
        u, w = y.double() @ b[-1].double(), a[-1].double()
        tu = sum_tol(O, y.double().abs() @ b[-1].double().abs())
        want, absdot = u @ w, u.abs() @ w.abs()
        close(dx, want, sum_tol(R, absdot) + 4 * U * absdot + 1.01 * (tu @ w.abs()) + (U + 2.0 ** -8) * want.abs() + 1e-37)


def test_lora_gradient_by_differences():
    import zeromoe_amd as Z

    S, I, O, R, n = 9, 24, 20, 3, 2
    a, b = adapters(n, R, I, O, "f32")
    x, dy, ids, scale = rand(S, I, seed=3), rand(S, O, seed=4), some_ids(S, n, "mixed"), rand(n, seed=5)
    _, v = Z.lora(x, a, b, ids, scale=scale, save=True)
    grads = Z.lora_backward(dy, x, a, b, ids, v, scale=scale)

    def loss(x, a, b):
        at = ids.clamp(min=0).long()
        y = torch.matmul(b[at], torch.matmul(a[at], x[:, :, None]))[:, :, 0] * scale.double()[at][:, None]
        return (y * (ids >= 0)[:, None] * dy.double()).sum()

    args, h = [x.double(), a.double(), b.double()], 1e-5
    for k, d in enumerate(grads):
        e = rand(*args[k].shape, seed=20 + k).double()
        up, dn = list(args), list(args)
        up[k], dn[k] = args[k] + h * e, args[k] - h * e
        want = ((loss(*up) - loss(*dn)) / (2 * h)).item()
        assert abs((d.double() * e).sum().item() - want) <= 1e-4 * max(1.0, (d.double() * e).abs().sum().item())
