"""Operators of fine-tuning and of serving fine-tuned models beside the routed experts, and what their speed is judged by.

The quantized experts stay as they are; what is unquantized, trained or different for every request lies beside them: a
shared expert's gated projections, low-rank adapters, and the gradients of all that.  A case is one call of one operator:

  glu            h = act(x w_gate^T + b_gate) * (x w_up^T + b_up), with both factors kept for a training step
  glu_backward   gradients of it by x, both weights and both biases
  lora           y = residual + scale * (x a^T) b^T with the adapter that each token's id names
  lora_backward  gradients of it by x and by the adapters
  clip           the norm of all gradients together, and the gradients scaled down to a largest norm

`listed()` names the standing cases, `draw()` gives further ones of the same ranges, `prepare()` makes the inputs,
`run()` is one pass, and `exact()` gives its results in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False  # True: run() calls the framework's operators; False: their plain forms

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
PAIRS = [("f32", "bf16"), ("f32", "f32"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")]
MOST_FLOPS = 4.0 * 8192 * 7168 * 2048  # of a drawn pair of products
MOST_ROWS = 8192 * (7168 + 2 * 2048)   # values that a drawn lora call reads and writes
MOST_ADAPTERS = 1 << 24                # values of all adapters of a drawn lora call
MOST_GRADIENTS = 1 << 27               # values of a drawn clip call
MAX_NORM, EPS = 1.0, 1e-6


# ---------------------------------------------------------------- cases


def _glu(S, I, F, x, w, act="silu", bias=False, save=False):
    return dict(op="glu", S=S, I=I, F=F, x=x, w=w, act=act, bias=bias, save=save)


def _glu_backward(S, I, F, x, w, act="silu"):
    return dict(op="glu_backward", S=S, I=I, F=F, x=x, w=w, act=act)


def _lora(S, I, O, R, n, x, w, runs):
    return dict(op="lora", S=S, I=I, O=O, R=R, n=n, x=x, w=w, runs=runs)


def _lora_backward(S, I, O, R, n, x, w, runs):
    return dict(op="lora_backward", S=S, I=I, O=O, R=R, n=n, x=x, w=w, runs=runs)


def _clip(layers, E, H, F, R, w, over):
    return dict(op="clip", layers=layers, E=E, H=H, F=F, R=R, w=w, over=over)


def listed():
    return [
        # one token through the gated projections of an unquantized shared expert: both weights read once
        dict(_glu(1, 4096, 1536, "f32", "bf16"), name="glu_decode"),
        # two dozen sequences decoded together through a wide shared expert in bf16
        dict(_glu(24, 7168, 2048, "bf16", "bf16"), name="glu_batch24"),
        # a training step's forward pass in f32 on an odd number of tokens, both factors kept
        dict(_glu(511, 2048, 768, "f32", "f32", "gelu_tanh", True, True), name="glu_train511"),
        # a long prompt through a wide shared expert in bf16
        dict(_glu(8192, 7168, 2048, "bf16", "bf16"), name="glu_prompt8192"),
        # training: gradients of a bf16 shared expert's gated projections
        dict(_glu_backward(2048, 4096, 1536, "bf16", "bf16"), name="glu_backward_bf16"),
        # training: the same in f32 on a ragged batch, with gelu
        dict(_glu_backward(1023, 2048, 768, "f32", "f32", "gelu"), name="glu_backward_f32"),
        # one token of one request with its adapter beside an attention output projection
        dict(_lora(1, 4096, 4096, 16, 64, "bf16", "bf16", False), name="lora_decode"),
        # four dozen requests decoded together, each with one of 64 adapters, beside an f32 residual stream
        dict(_lora(48, 4096, 1536, 32, 64, "f32", "bf16", False), name="lora_batch48"),
        # prompts of a few requests, one after the other, in bf16
        dict(_lora(8192, 7168, 2048, 64, 8, "bf16", "bf16", True), name="lora_prompt8192"),
        # training: four adapters at once on a ragged batch
        dict(_lora_backward(4095, 4096, 1536, 16, 4, "bf16", "bf16", True), name="lora_backward4095"),
        # the gradients of one layer's router, norm and adapters
        dict(_clip(1, 128, 2048, 0, 16, "f32", True), name="clip_router"),
        # the gradients of a dozen layers: router, norm, shared expert and adapters of each
        dict(_clip(12, 128, 4096, 1536, 16, "f32", True), name="clip_layers12"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def _width(rng, lo, hi):
    """A feature count: most are multiples of 32, some of 4, some anything."""
    n = _log_int(rng, lo, hi)
    step = rng.choice([32, 32, 32, 4, 1])
    return max(lo, n // step * step)


def draw(rng):
    """A case of the listed ones' ranges: other sizes (odd ones too), types, activations and adapters, none of it costing
    more than the largest listed case."""
    op = rng.choice(["glu", "glu", "glu_backward", "lora", "lora", "lora_backward", "clip"])
    if op in ("glu", "glu_backward"):
        train = op == "glu_backward"
        x, w = rng.choice(PAIRS)
        I, F = _width(rng, 256, 8192), _width(rng, 32, 4096)
        most = MOST_FLOPS / (8.0 if train else 4.0) / (6.0 if x == "f32" else 3.0 if train else 1.0) / (I * F)
        S = _log_int(rng, 1, max(1, min(8192, int(most))))
        act = rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu", "sigmoid", "none"])
        if train:
            return _glu_backward(S, I, F, x, w, act)
        return _glu(S, I, F, x, w, act, rng.random() < 0.4, rng.random() < 0.4)
    if op in ("lora", "lora_backward"):
        train = op == "lora_backward"
        x, w = rng.choice(PAIRS)
        I, O, R = _width(rng, 256, 8192), _width(rng, 256, 8192), rng.choice([4, 8, 8, 16, 16, 32, 64, 100, 128])
        n = max(1, min(_log_int(rng, 1, 8 if train else 128), MOST_ADAPTERS // (R * (I + O))))
        S = _log_int(rng, 1, max(1, min(8192, MOST_ROWS // ((I + 2 * O) * (3 if train else 1) * SIZE[x] // 2))))
        return (_lora_backward if train else _lora)(S, I, O, R, n, x, w, rng.random() < 0.5)
    E, H, F, R = rng.choice([8, 64, 128, 160, 256]), _width(rng, 256, 8192), rng.choice([0, 768, 1536]), rng.choice([4, 8, 16, 64])
    each = H * (E + 2 + 3 * F + 2 * R) + 4 * R
    return _clip(_log_int(rng, 1, max(1, min(48, MOST_GRADIENTS // each))), E, H, F, R, rng.choice(["f32", "f32", "bf16", "f16"]),
                 rng.random() < 0.8)


# ---------------------------------------------------------------- inputs


def _ids(c, gen):
    """An adapter for each token: one after the other in runs, as prompts lie in a batch, or any for any token, as in
    decoding; a few tokens have none."""
    S, n = c["S"], c["n"]
    if c["runs"]:
        cuts = torch.sort(torch.randint(0, S + 1, (n - 1,), device="cuda", generator=gen))[0]
        names = torch.randperm(n, device="cuda", generator=gen)
        ids = names[torch.searchsorted(cuts, torch.arange(S, device="cuda"), right=True)]
    else:
        ids = torch.randint(0, n, (S,), device="cuda", generator=gen)
    if S > 1:
        ids = torch.where(torch.rand(S, device="cuda", generator=gen) < 0.05, torch.full_like(ids, -1), ids)
    return ids.to(torch.int32)


def prepare(c, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, device="cuda", generator=gen)  # noqa: E731
    s = dict(c=c)
    op = c["op"]
    if op == "clip":
        # for each layer: router, norm, shared expert, adapters; sizes of the entries differ from tensor to tensor
        E, H, F, R, t = c["E"], c["H"], c["F"], c["R"], DTYPE[c["w"]]
        shapes = [(E, H), (H,), (H,)] + ([(F, H), (F, H), (H, F)] if F else []) + [(R, H), (H, R), (R, 4)]
        shapes = shapes * c["layers"]
        total = sum(math.prod(sh) for sh in shapes)
        size = (4.0 if c["over"] else 0.25) * MAX_NORM / math.sqrt(total)
        s["grads"] = [(rand(*sh) * size * (0.5 + (i * 7 % 10) / 10.0)).to(torch.float32 if len(sh) == 1 else t)
                      for i, sh in enumerate(shapes)]
        # the clipped ones go to flat buffers, one for each type, as data-parallel training keeps them
        s["flat"] = {k: torch.empty(sum(g.numel() for g in s["grads"] if g.dtype == k), device="cuda", dtype=k)
                     for k in sorted({g.dtype for g in s["grads"]}, key=str)}
        s["out"], used = [], dict.fromkeys(s["flat"], 0)
        for g in s["grads"]:
            at = used[g.dtype]
            s["out"].append(s["flat"][g.dtype][at:at + g.numel()].view(g.shape))
            used[g.dtype] = at + g.numel()
        return s
    S, I, x = c["S"], c["I"], DTYPE[c["x"]]
    # activations behind a norm: unit size, a few channels far larger
    loud = 1.0 + 7.0 * (torch.rand(I, device="cuda", generator=gen) < 0.005)
    s["x"] = (rand(S, I) * loud).to(x)
    if op in ("glu", "glu_backward"):
        F = c["F"]
        s["w_gate"], s["w_up"] = ((rand(F, I) * (1.0 / math.sqrt(I))).to(DTYPE[c["w"]]) for _ in range(2))
        if op == "glu":
            s["b_gate"], s["b_up"] = (rand(F) * 0.2, rand(F) * 0.2) if c["bias"] else (None, None)
        else:
            s["gate"], s["up"] = ((rand(S, F) * 1.2).to(x) for _ in range(2))
            s["dh"] = (rand(S, F) * 0.01).to(x)
        return s
    O, R, n = c["O"], c["R"], c["n"]
    s["a"] = (rand(n, R, I) * (1.0 / math.sqrt(I))).to(DTYPE[c["w"]])
    s["b"] = (rand(n, O, R) * (0.3 / math.sqrt(R))).to(DTYPE[c["w"]])
    s["scale"] = 0.5 + 1.5 * torch.rand(n, device="cuda", generator=gen)
    s["ids"] = _ids(c, gen)
    if op == "lora":
        s["residual"] = (rand(S, O) * 2.0).to(x)
    else:
        s["v"] = rand(S, R) * 1.2  # x a^T, as the forward pass left it
        s["dy"] = (rand(S, O) * 0.01).to(x)
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
    if act == "none":
        return torch.ones_like(z)
    g = 1.0 / (1.0 + torch.exp(-z))
    return g * (1.0 + z * (1.0 - g)) if act == "silu" else g * (1.0 - g)


def _rows_by(m, at, t):
    """m[t] (S, K) times the matrix that each row's id names: (S, J) of matrices `at` (n, K, J); ids below 0 give zeros."""
    ids, n = t, at.shape[0]
    S, K, J = m.shape[0], at.shape[1], at.shape[2]
    if S * K * J <= 1 << 27 and S <= 8 * n:  # the matrices gathered for every row
        y = torch.matmul(m[:, None, :], at[ids.clamp(min=0).long()])[:, 0]
        return torch.where((ids >= 0)[:, None], y, torch.zeros((), device=y.device))
    y = torch.zeros((S, J), device=m.device)
    for i in range(n):
        y = y + (m * (ids == i)[:, None]) @ at[i]
    return y


def _plain(s):
    c = s["c"]
    op = c["op"]
    if op == "clip":
        total = torch.zeros((), dtype=torch.float64, device="cuda")
        for g in s["grads"]:
            d = g.double()
            total = total + (d * d).sum()
        norm = torch.sqrt(total)
        scale = torch.clamp(MAX_NORM / (norm + EPS), max=1.0).float()
        for g, o in zip(s["grads"], s["out"]):
            o.copy_(g.float() * scale)
        return {"norm": norm.float(), "grads": list(s["flat"].values())}
    t = DTYPE[c["x"]]
    x = s["x"].float()
    if op == "glu":
        g, u = x @ s["w_gate"].float().t(), x @ s["w_up"].float().t()
        if s["b_gate"] is not None:
            g, u = g + s["b_gate"], u + s["b_up"]
        h = (_act(g, c["act"]) * u).to(t)
        return {"h": h, "gate": g.to(t), "up": u.to(t)} if c["save"] else {"h": h}
    if op == "glu_backward":
        g, u, dh = s["gate"].float(), s["up"].float(), s["dh"].float()
        dg, du = dh * u * _act_slope(g, c["act"]), dh * _act(g, c["act"])
        return {"dx": (dg @ s["w_gate"].float() + du @ s["w_up"].float()).to(t), "dw_gate": dg.t() @ x, "dw_up": du.t() @ x,
                "db_gate": dg.sum(0), "db_up": du.sum(0)}
    a, b, ids = s["a"].float(), s["b"].float(), s["ids"]
    scale = s["scale"][ids.clamp(min=0).long()][:, None]
    if op == "lora":
        v = _rows_by(x, a.transpose(1, 2).contiguous(), ids) * scale
        return {"y": (s["residual"].float() + _rows_by(v, b.transpose(1, 2).contiguous(), ids)).to(t)}
    dy = s["dy"].float() * scale
    u = _rows_by(dy, b, ids)
    mine = [(ids == i)[:, None] for i in range(c["n"])]
    return {"dx": _rows_by(u, a, ids).to(t), "da": torch.stack([(u * m).t() @ x for m in mine]),
            "db": torch.stack([(dy * m).t() @ s["v"] for m in mine])}


def _own(s):
    import zeromoe_amd as Z

    c = s["c"]
    op = c["op"]
    if op == "clip":
        norm = Z.clip_grad_norm(s["grads"], MAX_NORM, eps=EPS, out=s["out"])
        return {"norm": norm, "grads": list(s["flat"].values())}
    if op == "glu":
        r = Z.glu(s["x"], s["w_gate"], s["w_up"], s["b_gate"], s["b_up"], act=c["act"], save=c["save"])
        return {"h": r[0], "gate": r[1], "up": r[2]} if c["save"] else {"h": r}
    if op == "glu_backward":
        dx, dw_gate, dw_up, db_gate, db_up = Z.glu_backward(s["dh"], s["x"], s["w_gate"], s["w_up"], s["gate"], s["up"],
                                                            act=c["act"])
        return {"dx": dx, "dw_gate": dw_gate, "dw_up": dw_up, "db_gate": db_gate, "db_up": db_up}
    if op == "lora":
        return {"y": Z.lora(s["x"], s["a"], s["b"], s["ids"], scale=s["scale"], residual=s["residual"])}
    dx, da, db = Z.lora_backward(s["dy"], s["x"], s["a"], s["b"], s["ids"], s["v"], scale=s["scale"])
    return {"dx": dx, "da": da, "db": db}


def run(s):
    return _own(s) if own else _plain(s)


# ---------------------------------------------------------------- costs and 64-bit results


def work(c):
    op = c["op"]
    if op == "clip":
        e, H, R = SIZE[c["w"]], c["H"], c["R"]
        mats, vecs = c["layers"] * (H * (c["E"] + 3 * c["F"] + 2 * R) + 4 * R), c["layers"] * 2 * H
        return {"bytes": float(2 * (mats * e + vecs * 4) + 4), "flops": float(3 * (mats + vecs))}
    S, I, e, we = c["S"], c["I"], SIZE[c["x"]], SIZE[c["w"]]
    if op == "glu":
        F = c["F"]
        return {"bytes": float(S * I * e + 2 * F * I * we + S * F * e * (3 if c["save"] else 1) + 8 * F * c["bias"]),
                "flops": 4.0 * S * I * F}
    if op == "glu_backward":
        F = c["F"]
        return {"bytes": float(3 * S * F * e + 2 * S * I * e + 2 * F * I * (we + 4) + 8 * F), "flops": 8.0 * S * I * F}
    O, R, n = c["O"], c["R"], c["n"]
    if op == "lora":  # the adapters of as many requests as there are, at most all
        return {"bytes": float(S * (I + 2 * O) * e + min(S, n) * R * (I + O) * we + 4 * S), "flops": 2.0 * S * R * (I + O)}
    return {"bytes": float(S * (2 * I + O) * e + 4 * S * R + min(S, n) * R * (I + O) * we + 4 * n * R * (I + O) + 4 * S),
            "flops": 4.0 * S * R * (I + O)}


def exact(c, seed):
    s = prepare(c, seed)
    D = lambda t: None if t is None else t.double()  # noqa: E731
    F = torch.nn.functional
    op = c["op"]
    if op == "clip":
        norm = math.sqrt(math.fsum(torch.linalg.vector_norm(g.double()).item() ** 2 for g in s["grads"]))
        scale = min(1.0, MAX_NORM / (norm + EPS))
        return {"norm": torch.tensor(norm, dtype=torch.float64, device="cuda"),
                "grads": [torch.cat([g.double().flatten() * scale for g in s["grads"] if g.dtype == k]) for k in s["flat"]]}
    if op in ("glu", "glu_backward"):
        act = {"none": lambda z: z, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"),
               "silu": F.silu, "sigmoid": torch.sigmoid}[c["act"]]
        if op == "glu":
            g, u = (F.linear(D(s["x"]), D(s["w_" + k]), D(s["b_" + k])) for k in ("gate", "up"))
            return {"h": act(g) * u, "gate": g, "up": u} if c["save"] else {"h": act(g) * u}
        g, u = D(s["gate"]).requires_grad_(), D(s["up"]).requires_grad_()
        dg, du = torch.autograd.grad(act(g) * u, (g, u), D(s["dh"]))
        return {"dx": torch.mm(torch.cat([dg, du], 1), torch.cat([D(s["w_gate"]), D(s["w_up"])], 0)),
                "dw_gate": torch.mm(dg.t().contiguous(), D(s["x"])), "dw_up": torch.mm(du.t().contiguous(), D(s["x"])),
                "db_gate": dg.sum(0), "db_up": du.sum(0)}
    x, a, b = D(s["x"]), D(s["a"]), D(s["b"])
    if op == "lora":
        y = D(s["residual"])
        for i in range(c["n"]):
            at = (s["ids"] == i).nonzero()[:, 0]
            if len(at):
                y[at] += torch.mm(torch.mm(x[at], a[i].t()), b[i].t()) * D(s["scale"])[i]
        return {"y": y}
    dx, da, db, dy = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b), D(s["dy"])
    for i in range(c["n"]):
        at = (s["ids"] == i).nonzero()[:, 0]
        if len(at):
            u = torch.mm(dy[at], b[i]) * D(s["scale"])[i]
            dx[at] = torch.mm(u, a[i])
            da[i] = torch.mm(u.t().contiguous(), x[at])
            db[i] = torch.mm(dy[at].t().contiguous(), D(s["v"])[at]) * D(s["scale"])[i]
    return {"dx": dx, "da": da, "db": db}
