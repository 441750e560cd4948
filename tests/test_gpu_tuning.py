"""The operators of fine-tuning together, as a step and as a server use them."""
import math

import pytest
import torch

from test_gpu_dense import rand

pytestmark = pytest.mark.gpu


def test_step_over_frozen_experts():
    """norm -> router -> quantized experts, beside them a shared expert (gated product, down projection with adapters of two
    tasks) -> weighted sum; back to the gradients of norm, router, shared expert and adapters; all of them clipped.  The
    quantized experts' rows are held fixed."""
    import zeromoe_amd as Z
    import zm_oracle as O

    Z.init()
    S, H, F, E, K, Fs, R, n = 37, 512, 256, 24, 4, 192, 8, 2
    t = O.TYPE_Q4_K
    wg, wu, wd = (torch.from_numpy(O.random_blocks(t, E * r, m, seed=s).reshape(E, r, -1)).cuda()
                  for r, m, s in ((F, H, 1), (F, H, 2), (H, F, 3)))
    x, gain, shift = rand(S, H, seed=4), 1 + 0.1 * rand(H, seed=5), 0.1 * rand(H, seed=6)
    wr = rand(E, H, seed=7, scale=0.05)
    sg, su, sd = (rand(r, m, seed=s, scale=1 / math.sqrt(m)) for r, m, s in ((Fs, H, 8), (Fs, H, 9), (H, Fs, 10)))
    a, b, scale = rand(n, R, Fs, seed=11, scale=0.1), rand(n, H, R, seed=12, scale=0.2), torch.tensor([2.0, 0.5], device="cuda")
    task = torch.where(torch.arange(S, device="cuda") % 5 == 4, -1, torch.arange(S, device="cuda") // 20).to(torch.int32)
    dout = rand(S, H, seed=13, scale=0.1)

    h, mean, rstd = Z.layer_norm(x, gain, shift, stats=True)
    logits = Z.linear(h, wr)
    ids, w = Z.router(logits, K, gating="sigmoid", weights_norm=True, weights_scale=2.5)
    up, gate = (Z.mul_mat_id(m, t, H, h.view(S, 1, H), ids) for m in (wu, wg))
    y = Z.mul_mat_id(wd, t, F, Z.swiglu(gate, up), ids)
    f, fg, fu = Z.glu(h, sg, su, save=True)
    shared, v = Z.lora(f, a, b, task, scale=scale, residual=Z.linear(f, sd, residual=x), save=True)
    out = Z.combine(y, w, ids=ids, residual=shared)

    dlogits = Z.router_backward(logits, ids, Z.combine_backward(dout, y, ids=ids), gating="sigmoid", weights_norm=True,
                                weights_scale=2.5)
    dh, dwr, _ = Z.linear_backward(dlogits, h, wr, need_dbias=False)
    df, da, db = Z.lora_backward(dout, f, a, b, task, v, scale=scale)
    df2, dsd, _ = Z.linear_backward(dout, f, sd, need_dbias=False)
    dh2, dsg, dsu, _, _ = Z.glu_backward(df + df2, h, sg, su, fg, fu, need_db=False)
    dx, dgain, dshift = Z.layer_norm_backward(dh + dh2, x, mean, rstd, gain)
    got = [dgain, dshift, dwr, dsg, dsu, dsd, da, db]
    raw = [g.clone() for g in got]
    norm = Z.clip_grad_norm(got, 0.01)

    p = [u.double().requires_grad_() for u in (gain, shift, wr, sg, su, sd, a, b)]
    h64 = torch.nn.functional.layer_norm(x.double(), (H,), p[0], p[1], 1e-5)
    probs = torch.sigmoid(h64 @ p[2].t()).gather(1, ids.long())
    w64 = probs / probs.sum(-1, keepdim=True) * 2.5
    f64 = torch.nn.functional.silu(h64 @ p[3].t()) * (h64 @ p[4].t())
    at = task.clamp(min=0).long()
    low = torch.matmul(p[7][at], torch.matmul(p[6][at], f64[:, :, None]))[:, :, 0] * scale.double()[at][:, None]
    out64 = x.double() + f64 @ p[5].t() + low * (task >= 0)[:, None] + (w64[:, :, None] * y.double()).sum(1)
    want = torch.autograd.grad(out64, p, dout.double())
    # each step's own bound is tested by itself; through the chain f32 roundings stay below 2^-24 times some thousand
    # additions of the largest values: 1e-4 of a tensor's own size
    assert ((out.double() - out64).norm() / out64.norm()).item() < 1e-5
    for g, ref in zip(raw, want):
        assert ((g.double() - ref).norm() / ref.norm()).item() < 1e-4
    n64 = math.sqrt(sum((g ** 2).sum().item() for g in want))
    assert abs(norm.item() - n64) <= 1e-4 * n64 and n64 > 0.01
    for g, r in zip(got, raw):
        c = 0.01 / (norm.item() + 1e-6)
        assert ((g.double() - r.double() * c).norm() <= 1e-6 * (r.double() * c).norm()).item()


@pytest.mark.parametrize("S", [1, 24, 700])
def test_serving_in_one_graph(S):
    """Requests with their adapters through a gated block, captured and replayed with other requests, on two streams at
    once in the end."""
    import zeromoe_amd as Z

    H, F, R, n, t = 512, 384, 16, 5, torch.bfloat16
    sg, su, sd = (rand(r, m, seed=s, scale=1 / math.sqrt(m), dtype=t) for r, m, s in ((F, H, 1), (F, H, 2), (H, F, 3)))
    a, b = rand(n, R, F, seed=4, scale=0.1, dtype=t), rand(n, H, R, seed=5, scale=0.2, dtype=t)

    def block(x, ids):
        f = Z.glu(x, sg, su)
        return Z.lora(f, a, b, ids, residual=Z.linear(f, sd, residual=x))

    def request(seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        return rand(S, H, seed=seed, dtype=t), torch.randint(-1, n, (S,), device="cuda", generator=g).to(torch.int32)

    x, ids = request(10)
    block(x, ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block(x, ids)
    for seed in (11, 12, 13):
        for held, new in zip((x, ids), request(seed)):
            held.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, block(x, ids))
        x64 = x.double()
        f = torch.nn.functional.silu(x64 @ sg.double().t()) * (x64 @ su.double().t())
        at = ids.clamp(min=0).long()
        want = x64 + f @ sd.double().t() + torch.matmul(b[at].double(), torch.matmul(a[at].double(), f[:, :, None]))[:, :, 0] * (
            ids >= 0)[:, None]
        # three results rounded to bf16 on the way (2^-9 each as a rule, f, the projection and the sum), the last 2^-9
        assert ((y.double() - want).norm() / want.norm()).item() < 4 * 2.0 ** -9
    streams = [torch.cuda.Stream() for _ in range(2)]
    asked = [request(20 + i) for i in range(2)]
    want = [block(*r) for r in asked]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = block(*asked[i])
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_wrapper_refusals():
    import zeromoe_amd as Z

    x, w, a, b = rand(4, 64), rand(32, 64), rand(3, 8, 64), rand(3, 32, 8)
    ids = torch.zeros(4, device="cuda", dtype=torch.int32)
    g = rand(4, 32)
    for f, why in ((lambda: Z.glu(x, w, rand(32, 72)[:, :64]), "one stride"), (lambda: Z.glu(x, w, rand(31, 64)), "shape"),
                   (lambda: Z.glu(x, w, w.half()), "float32"), (lambda: Z.glu(x, w, rand(64, 32).t()), "contiguous columns"),
                   (lambda: Z.glu(x.half(), w, w), "16-bit|float16"), (lambda: Z.glu(x, w, w, b_up=rand(31)), "shape"),
                   (lambda: Z.glu(x, w, w, act="swish"), "unknown activation"), (lambda: Z.glu(x, w, w, out_dtype=torch.float16), "float32"),
                   (lambda: Z.glu_backward(g, x, w, w, g, g.half()), "float32"), (lambda: Z.glu_backward(g, x, w, w, g[:3], g), "shape"),
                   (lambda: Z.lora(x, a, b[:2], ids), "needed"), (lambda: Z.lora(x, a, rand(3, 32, 9), ids), "needed"),
                   (lambda: Z.lora(x, a, b, ids.long()), "int32"), (lambda: Z.lora(x, a, b, ids[:3]), "shape"),
                   (lambda: Z.lora(x, a, b.half(), ids), "adapters"), (lambda: Z.lora(x, a, b, ids, scale=rand(2)), "shape"),
                   (lambda: Z.lora(x, a.transpose(1, 2).contiguous().transpose(1, 2), b, ids), "contiguous columns"),
                   (lambda: Z.lora(x, a, b, ids, residual=g.half()), "float32"),
                   (lambda: Z.lora_backward(g, x, a, b, ids), "db needs v"),
                   (lambda: Z.lora_backward(g, x, a, b, ids, rand(4, 7)), "shape"),
                   (lambda: Z.lora(x, a.requires_grad_(), b, ids), "requires a gradient"),
                   (lambda: Z.glu(x.clone().requires_grad_(), w, w), "requires a gradient")):
        with pytest.raises(ValueError, match=why):
            f()
    with pytest.raises(RuntimeError, match="rank of 1 to 256"):
        Z.lora(x, rand(2, 257, 64), rand(2, 32, 257), ids)
    with pytest.raises(RuntimeError, match="1 to 512 adapters"):
        Z.lora(x, rand(513, 2, 64), rand(513, 32, 2), ids)
