"""The dense operators around the routed experts, and what their speed is judged by.

Beside the routed experts themselves a MoE block has a norm, the router's product, the routing's gradient and the
weighted sum of the experts' rows; its unquantized projections (router, shared expert, attention output) are matrix
products with a bias, an activation and a residual.  A case is one call of one of them, in serving or in a step that
trains the router and the norm over frozen quantized experts:

  linear            y = act(x w^T + bias) + residual
  linear_backward   dx, dw, dbias of act(x w^T + bias)
  layer_norm        the forward pass, or the forward and backward pass of a training step
  router_backward   gradient of the routed experts' weights by the logits
  combine           sum of the experts' rows times their weights, plus the residual; or the gradient of the weights

`listed()` names the standing cases, `draw()` gives further ones of the same ranges, `prepare()` makes the inputs,
`run()` is one pass, and `exact()` gives its results in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False  # True: run() calls the framework's operators; False: their plain forms

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
MOST_FLOPS = 2.0 * 8192 * 7168 * 2048  # of a drawn matrix product
MOST_BYTES = 4.0 * 2048 * 9 * 4096 * 1.1  # of a drawn pass that is bound by memory


# ---------------------------------------------------------------- cases


def _linear(S, I, O, x, w, act="none", bias=True, residual=False, y=None):
    return dict(op="linear", S=S, I=I, O=O, x=x, w=w, y=y or x, act=act, bias=bias, residual=residual)


def _linear_backward(S, I, O, x, w, act="none"):
    return dict(op="linear_backward", S=S, I=I, O=O, x=x, w=w, act=act)


def _layer_norm(S, n, x, train):
    return dict(op="layer_norm", S=S, n=n, x=x, train=train)


def _router_backward(S, E, K, gating, norm, scale=0.0, balance=False):
    return dict(op="router_backward", S=S, E=E, K=K, gating=gating, norm=norm, scale=scale, balance=balance)


def _combine(S, K, H, train):
    return dict(op="combine", S=S, K=K, H=H, train=train)


def listed():
    return [
        # one token through the gate projection of an unquantized shared expert: 16-bit weights read once
        dict(_linear(1, 4096, 1536, "f32", "bf16", "silu"), name="linear_decode"),
        # two dozen sequences decoded together: a down projection added to the residual stream
        dict(_linear(24, 2048, 7168, "f32", "f16", residual=True), name="linear_batch24"),
        # the fp32 router's logits over a prefill chunk
        dict(_linear(512, 7168, 256, "f32", "f32"), name="linear_router512"),
        # a long prompt through an attention output projection with its residual, all in bf16
        dict(_linear(8192, 7168, 2048, "bf16", "bf16", residual=True), name="linear_prompt8192"),
        # training: gradients of the fp32 router over a ragged batch
        dict(_linear_backward(4095, 5120, 160, "f32", "f32"), name="linear_backward_router"),
        # training: gradients of a bf16 projection with its activation (the pre-activations were kept)
        dict(_linear_backward(2048, 4096, 1536, "bf16", "bf16", "silu"), name="linear_backward_bf16"),
        # the norm of one token in front of the router
        dict(_layer_norm(1, 4096, "f32", False), name="layer_norm_decode"),
        # the norm over a long batch in bf16, forward and backward
        dict(_layer_norm(4096, 7168, "bf16", True), name="layer_norm_train4096"),
        # gradient of the routing of a small batch: sigmoid scores, renormalised and scaled
        dict(_router_backward(64, 160, 8, "sigmoid", True, 2.5), name="router_backward64"),
        # gradient of the routing of a long batch: softmax over 256 experts, with a balance loss on the probabilities
        dict(_router_backward(8192, 256, 8, "softmax", True, 0.0, True), name="router_backward8192"),
        # the weighted sum of two dozen tokens' expert rows, added to the residual
        dict(_combine(24, 8, 7168, False), name="combine24"),
        # the gradient of the weights from the experts' rows of a long batch
        dict(_combine(2048, 8, 4096, True), name="combine_train2048"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def _width(rng, lo, hi):
    """A feature count: most are multiples of 32, some of 4, some anything."""
    n = _log_int(rng, lo, hi)
    step = rng.choice([32, 32, 32, 4, 1])
    return max(lo, n // step * step)


def draw(rng):
    """A case of the listed ones' ranges: other sizes (odd ones too), types, activations and gatings, none of it costing
    more than the largest listed case."""
    op = rng.choice(["linear", "linear", "linear_backward", "layer_norm", "router_backward", "combine"])
    if op in ("linear", "linear_backward"):
        train = op == "linear_backward"
        x, w = rng.choice([("f32", "bf16"), ("f32", "f32"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
        I, O = _width(rng, 256, 8192), _width(rng, 32, 8192)
        most = MOST_FLOPS / (4.0 if train else 2.0) / (4.0 if "f32" in x else 1.0) / (I * O)
        S = _log_int(rng, 1, max(1, min(8192, int(most))))
        act = rng.choice(["none", "none", "silu", "gelu", "gelu_tanh", "relu", "sigmoid"])
        if train:
            return _linear_backward(S, I, O, x, w, act)
        return _linear(S, I, O, x, w, act, rng.random() < 0.7, rng.random() < 0.4, rng.choice([x, "f32"]))
    if op == "layer_norm":
        n, x, train = _width(rng, 64, 8192), rng.choice(["f32", "f16", "bf16"]), rng.random() < 0.6
        most = 4096 * 7168 * 2 / (n * SIZE[x])
        return _layer_norm(_log_int(rng, 1, max(1, min(16384, int(most)))), n, x, train)
    if op == "router_backward":
        E = rng.choice([8, 32, 60, 64, 96, 128, 160, 200, 256, 384])
        K = rng.choice([k for k in (1, 2, 4, 6, 8, 10) if k <= E])
        return _router_backward(_log_int(rng, 1, 8192), E, K, rng.choice(["softmax", "sigmoid", "sqrt_softplus"]),
                                rng.random() < 0.6, rng.choice([0.0, 2.5]), rng.random() < 0.3)
    H, K = _width(rng, 256, 8192), rng.choice([1, 2, 4, 6, 8, 10])
    S = _log_int(rng, 1, max(1, min(8192, int(MOST_BYTES / (4.0 * (K + 2) * H)))))
    return _combine(S, K, H, rng.random() < 0.5)


# ---------------------------------------------------------------- inputs


def _gate(z, gating):
    if gating == "softmax":
        return torch.softmax(z, -1)
    if gating == "sigmoid":
        return torch.sigmoid(z)
    return torch.sqrt(torch.log1p(torch.exp(-z.abs())) + z.clamp(min=0))


def prepare(c, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, device="cuda", generator=gen)  # noqa: E731
    s = dict(c=c)
    op, S = c["op"], c["S"]
    if op in ("linear", "linear_backward"):
        I, O = c["I"], c["O"]
        # activations behind a norm: unit size, a few channels far larger
        loud = 1.0 + 7.0 * (torch.rand(I, device="cuda", generator=gen) < 0.005)
        s["x"] = (rand(S, I) * loud).to(DTYPE[c["x"]])
        s["w"] = (rand(O, I) * (1.0 / math.sqrt(I))).to(DTYPE[c["w"]])
        if op == "linear":
            s["bias"] = rand(O) * 0.2 if c["bias"] else None
            s["residual"] = (rand(S, O) * 2.0).to(DTYPE[c["y"]]) if c["residual"] else None
        else:
            s["dy"] = (rand(S, O) * 0.01).to(DTYPE[c["x"]])
            s["pre"] = None if c["act"] == "none" else (rand(S, O) * 1.2).to(DTYPE[c["x"]])
    elif op == "layer_norm":
        n = c["n"]
        # a residual stream: rows of different sizes, a few loud channels, a mean that is not zero
        loud = 1.0 + 20.0 * (torch.rand(n, device="cuda", generator=gen) < 0.003)
        s["x"] = (rand(S, n) * loud * (0.3 + 3.0 * torch.rand(S, 1, device="cuda", generator=gen)) + 0.5).to(DTYPE[c["x"]])
        s["weight"] = 1.0 + 0.2 * rand(n)
        s["bias"] = 0.1 * rand(n)
        s["dy"] = (rand(S, n) * 0.05).to(DTYPE[c["x"]]) if c["train"] else None
    elif op == "router_backward":
        E, K = c["E"], c["K"]
        s["logits"] = rand(S, E) * 1.5
        # selection by score plus a balance bias; a tenth of the rows of a long batch are padding
        ids = torch.topk(_gate(s["logits"], c["gating"]) + 0.02 * rand(E), K, dim=-1)[1].to(torch.int32)
        if S >= 16:
            ids[torch.rand(S, device="cuda", generator=gen) < 0.1] = -1
        s["ids"] = ids.contiguous()
        s["dweights"] = rand(S, K) * 0.1
        s["dprobs"] = rand(E) * 0.01 if c["balance"] else None
    else:
        K, H = c["K"], c["H"]
        s["y"] = rand(S, K, H)
        w = torch.rand((S, K), device="cuda", generator=gen) + 0.05
        s["weights"] = w / w.sum(-1, keepdim=True)
        # a quarter of the routes belong to experts that are computed elsewhere
        ids = torch.randint(0, 128, (S, K), device="cuda", generator=gen, dtype=torch.int32)
        s["ids"] = torch.where(torch.rand((S, K), device="cuda", generator=gen) < 0.25, torch.full_like(ids, -1), ids)
        s["residual" if not c["train"] else "dout"] = rand(S, H)
    return s


# ---------------------------------------------------------------- one pass


def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * k * (1.0 + 3 * 0.044715 * z * z)
    g = 1.0 / (1.0 + torch.exp(-z))
    return g * (1.0 + z * (1.0 - g)) if act == "silu" else g * (1.0 - g)


def _plain(s):
    c = s["c"]
    op = c["op"]
    if op == "linear":
        z = s["x"].float() @ s["w"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"]
        y = _act(z, c["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return {"y": y.to(DTYPE[c["y"]])}
    if op == "linear_backward":
        dz = s["dy"].float()
        if c["act"] != "none":
            dz = dz * _act_slope(s["pre"].float(), c["act"])
        return {"dx": (dz @ s["w"].float()).to(DTYPE[c["x"]]), "dw": dz.t() @ s["x"].float(), "dbias": dz.sum(0)}
    if op == "layer_norm":
        x = s["x"].float()
        mean = x.mean(-1, keepdim=True)
        d = x - mean
        rstd = torch.rsqrt((d * d).mean(-1, keepdim=True) + 1e-5)
        h = d * rstd
        y = (h * s["weight"] + s["bias"]).to(s["x"].dtype)
        if not c["train"]:
            return {"y": y}
        dy = s["dy"].float()
        g = dy * s["weight"]
        dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
        return {"y": y, "dx": dx.to(s["x"].dtype), "dweight": (dy * h).sum(0), "dbias": dy.sum(0)}
    if op == "router_backward":
        p = _gate(s["logits"], c["gating"])
        valid = s["ids"] >= 0
        at = s["ids"].clamp(min=0).long()
        chosen = torch.where(valid, torch.gather(p, 1, at), torch.zeros((), device=p.device))
        d = torch.where(valid, s["dweights"], torch.zeros((), device=p.device)) * (c["scale"] or 1.0)
        if c["norm"]:
            total = chosen.sum(-1, keepdim=True)
            low = total < 2.0 ** -14
            total = total.clamp(min=2.0 ** -14)
            d = (d - torch.where(low, torch.zeros_like(total), (d * chosen).sum(-1, keepdim=True) / total)) / total
            d = torch.where(valid, d, torch.zeros((), device=p.device))
        g = torch.zeros_like(p).scatter_add_(1, at, d)
        if s["dprobs"] is not None:
            g = g + s["dprobs"] * valid.any(-1, keepdim=True)
        if c["gating"] == "softmax":
            return {"dlogits": p * (g - (p * g).sum(-1, keepdim=True))}
        if c["gating"] == "sigmoid":
            return {"dlogits": g * p * (1.0 - p)}
        return {"dlogits": g * torch.sigmoid(s["logits"]) / (2.0 * p)}
    valid = s["ids"] >= 0
    zero = torch.zeros((), device=s["y"].device)
    if c["train"]:
        return {"dweights": torch.where(valid, (s["y"] * s["dout"][:, None, :]).sum(-1), zero)}
    return {"out": s["residual"] + (s["y"] * torch.where(valid, s["weights"], zero)[:, :, None]).sum(1)}


def _own(s):
    import zeromoe_amd as Z

    c = s["c"]
    op = c["op"]
    if op == "linear":
        return {"y": Z.linear(s["x"], s["w"], bias=s["bias"], act=c["act"], residual=s["residual"],
                              out_dtype=DTYPE[c["y"]])}
    if op == "linear_backward":
        dx, dw, dbias = Z.linear_backward(s["dy"], s["x"], s["w"], act=c["act"], pre=s["pre"])
        return {"dx": dx, "dw": dw, "dbias": dbias}
    if op == "layer_norm":
        if not c["train"]:
            return {"y": Z.layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5)}
        y, mean, rstd = Z.layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5, stats=True)
        dx, dweight, dbias = Z.layer_norm_backward(s["dy"], s["x"], mean, rstd, s["weight"])
        return {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias}
    if op == "router_backward":
        return {"dlogits": Z.router_backward(s["logits"], s["ids"], s["dweights"], gating=c["gating"],
                                             weights_norm=c["norm"], weights_scale=c["scale"], dprobs=s["dprobs"])}
    if c["train"]:
        return {"dweights": Z.combine_backward(s["dout"], s["y"], ids=s["ids"])}
    return {"out": Z.combine(s["y"], s["weights"], ids=s["ids"], residual=s["residual"])}


def run(s):
    return _own(s) if own else _plain(s)


# ---------------------------------------------------------------- costs and 64-bit results


def work(c):
    op, S = c["op"], c["S"]
    if op == "linear":
        I, O = c["I"], c["O"]
        out = S * O * SIZE[c["y"]]
        return {"bytes": float(S * I * SIZE[c["x"]] + O * I * SIZE[c["w"]] + out * (2 if c["residual"] else 1) + 4 * O * c["bias"]),
                "flops": 2.0 * S * I * O}
    if op == "linear_backward":
        I, O = c["I"], c["O"]
        e = SIZE[c["x"]]
        return {"bytes": float(S * O * e * (1 if c["act"] == "none" else 2) + 2 * S * I * e + O * I * (SIZE[c["w"]] + 4) + 4 * O),
                "flops": 4.0 * S * I * O}
    if op == "layer_norm":
        n, e = c["n"], SIZE[c["x"]]
        # forward: x in, y out; a training step reads x again behind the whole forward pass, and dy, and writes dx
        return {"bytes": float(S * n * e * (4 if c["train"] else 2) + n * (16 if c["train"] else 8)),
                "flops": float(S * n * (20 if c["train"] else 8))}
    if op == "router_backward":
        return {"bytes": float(S * (8 * c["E"] + 8 * c["K"])), "flops": float(S * c["E"] * 12)}
    n = (c["K"] + (1 if c["train"] else 2)) * S * c["H"]
    return {"bytes": float(4 * n + S * c["K"] * 8), "flops": float(2 * S * c["K"] * c["H"])}


def _grad(outputs, inputs, grads):
    return torch.autograd.grad(outputs, inputs, grads)


def exact(c, seed):
    s = prepare(c, seed)
    D = lambda t: None if t is None else t.double()  # noqa: E731
    F = torch.nn.functional
    act = {"none": lambda z: z, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"),
           "silu": F.silu, "sigmoid": torch.sigmoid}
    op = c["op"]
    if op == "linear":
        y = act[c["act"]](F.linear(D(s["x"]), D(s["w"]), D(s["bias"])))
        return {"y": y if s["residual"] is None else y + D(s["residual"])}
    if op == "linear_backward":
        dz = D(s["dy"])
        if s["pre"] is not None:
            z = D(s["pre"]).requires_grad_()
            dz, = _grad(act[c["act"]](z), z, dz)
        return {"dx": torch.mm(dz, D(s["w"])), "dw": torch.mm(dz.t().contiguous(), D(s["x"])), "dbias": dz.sum(0)}
    if op == "layer_norm":
        x, w, b = (D(s[k]).requires_grad_() for k in ("x", "weight", "bias"))
        y = F.layer_norm(x, (c["n"],), w, b, 1e-5)
        if not c["train"]:
            return {"y": y.detach()}
        dx, dw, db = _grad(y, (x, w, b), D(s["dy"]))
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if op == "router_backward":
        z = D(s["logits"]).requires_grad_()
        p = {"softmax": lambda t: t.softmax(-1), "sigmoid": torch.sigmoid,
             "sqrt_softplus": lambda t: F.softplus(t, threshold=1e6).sqrt()}[c["gating"]](z)
        valid = (s["ids"] >= 0).double()
        w = p.gather(1, s["ids"].clamp(min=0).long()) * valid
        if c["norm"]:
            w = w / w.sum(-1, keepdim=True).clamp(min=2.0 ** -14)
        loss = (w * D(s["dweights"])).sum() * (c["scale"] or 1.0)
        if s["dprobs"] is not None:
            loss = loss + ((p * D(s["dprobs"])).sum(-1) * valid.amax(-1)).sum()
        return {"dlogits": _grad(loss, z, None)[0]}
    y = D(s["y"]) * (s["ids"] >= 0)[:, :, None]
    if c["train"]:
        return {"dweights": torch.matmul(y, D(s["dout"])[:, :, None]).squeeze(-1)}
    return {"out": D(s["residual"]) + torch.matmul(D(s["weights"])[:, None, :], y).squeeze(1)}
