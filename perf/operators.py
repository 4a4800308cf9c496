"""What the MoE block's four-bit and router operators are measured on.

Four operators: the NVFP4 quantisation of activations and weights, the linear on NVFP4 activations and weights
(quantisation and product), the routing of many tokens with its per-expert counts and its gradient, and the balance
loss with its gradient. `run` computes each in plain torch operations, or, with `own`, by the framework's calls."""
import os
import random  # noqa: F401  (draw() takes a random.Random)
import sys

import torch

own = False

PACKAGE = "nemotron-super-8gb_b200"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _framework():
    at = os.path.join(os.getcwd(), PACKAGE)
    if at not in sys.path:
        sys.path.insert(0, at)
    import dense_q
    import router
    return dense_q, router


def listed():
    return [
        # one token's hidden state on its way into a four-bit projection
        {"name": "quantize_token", "op": "quantize", "m": 1, "k": 4096, "type": "bf16", "per_row": True},
        # a ragged batch of shared-expert activations in half precision
        {"name": "quantize_ragged", "op": "quantize", "m": 777, "k": 2688, "type": "f16", "per_row": True},
        # the hidden states of a long prompt
        {"name": "quantize_prompt", "op": "quantize", "m": 16384, "k": 4096, "type": "bf16", "per_row": True},
        # a checkpoint's projection weight, brought into the weight format with one scale for the tensor
        {"name": "quantize_weight", "op": "quantize", "m": 12288, "k": 4096, "type": "f32", "per_row": False},
        # the shared expert's up projection of one decoded token
        {"name": "linear_token", "op": "linear", "m": 1, "n": 2688, "k": 4096, "type": "bf16", "act": "none"},
        # its down projection, added to the routed output, over a small decode batch
        {"name": "linear_batch", "op": "linear", "m": 37, "n": 4096, "k": 2688, "type": "bf16", "act": "add"},
        # its up projection with the squared ReLU over a prompt
        {"name": "linear_prompt", "op": "linear", "m": 2048, "n": 2688, "k": 4096, "type": "bf16", "act": "relu2"},
        # a large projection over a long prompt
        {"name": "linear_long", "op": "linear", "m": 8192, "n": 12288, "k": 4096, "type": "bf16", "act": "none"},
        # the router of a decode batch, serving
        {"name": "route_batch", "op": "route", "t": 64, "e": 512, "k": 22, "type": "f32", "score": "sigmoid", "groups": 1,
         "kept": 1, "norm": False, "train": False},
        # the router of a training batch, with the gradient of the weights
        {"name": "route_train", "op": "route", "t": 16384, "e": 512, "k": 22, "type": "f32", "score": "sigmoid",
         "groups": 1, "kept": 1, "norm": True, "train": True},
        # the balance loss of a small batch of logits kept in bf16, with its gradient
        {"name": "balance_small", "op": "balance", "t": 200, "e": 128, "k": 6, "type": "bf16", "score": "softmax",
         "masked": False},
        # the same over a long padded batch of the 512-expert router
        {"name": "balance_long", "op": "balance", "t": 32768, "e": 512, "k": 22, "type": "f32", "score": "sigmoid",
         "masked": True},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over their logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("quantize", "linear", "route", "balance"))
    kind = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op == "quantize":
        k = 16 * _spread(rng, 4, 512)
        return {"op": op, "m": _spread(rng, 1, min(16384, 12288 * 4096 // k)), "k": k, "type": kind,
                "per_row": rng.random() < 0.75}
    if op == "linear":
        k, n = 32 * _spread(rng, 8, 256), _spread(rng, 100, 12288)
        return {"op": op, "m": min(_spread(rng, 1, 8192), 8192 * 12288 * 4096 // (n * k)), "n": n, "k": k, "type": kind,
                "act": rng.choice(("none", "relu2", "add"))}
    if op == "route":
        score = rng.choice(("sigmoid", "sigmoid", "softmax"))
        groups, kept = rng.choice(((1, 1), (1, 1), (8, 4), (4, 2)))
        e = groups * _spread(rng, 8, 1024 // groups)
        return {"op": op, "t": _spread(rng, 1, 16384), "e": e, "k": rng.randint(1, min(32, e // 2)), "type": kind,
                "score": score, "groups": groups, "kept": kept, "norm": rng.random() < 0.5, "train": rng.random() < 0.5}
    e = _spread(rng, 8, 1024)
    return {"op": op, "t": min(_spread(rng, 16, 32768), 32768 * 512 // e), "e": e, "k": rng.randint(1, min(32, e // 2)),
            "type": kind, "score": rng.choice(("sigmoid", "softmax")), "masked": rng.random() < 0.5}


def _seeded(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _hidden(g, m, k, kind):
    """Hidden states: a few channels much larger than the rest, rows of different size."""
    channel = 1.0 + 20.0 * (torch.rand(k, generator=g, device="cuda") < 0.004)
    size = torch.exp(0.5 * torch.randn(m, 1, generator=g, device="cuda"))
    return (torch.randn(m, k, generator=g, device="cuda") * channel * size).to(TYPES[kind])


def _weight(g, n, k):
    """An NVFP4 weight as a checkpoint holds it: normal values over a tensor scale, which is no power of two."""
    w = torch.randn(n, k // 16, 16, generator=g, device="cuda") * 0.02
    s = w.abs().max() / 2688.0
    sc = (w.abs().amax(-1) / 6.0 / s).to(torch.float8_e4m3fn)
    q = (w.abs() / (sc.float() * s).clamp_min(1e-30)[..., None]).clamp_max(6.0)
    bounds = torch.tensor((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), device="cuda")
    code = torch.bucketize(q, bounds).to(torch.uint8) | ((w < 0).to(torch.uint8) << 3)
    code = code.reshape(n, k)
    return {"fmt": "nvfp4", "w": (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(),
            "sc": sc.view(torch.uint8).contiguous(), "s": s.reshape(1), "N": n, "K": k}


def prepare(case, seed):
    g, c = _seeded(seed), case
    st = {"case": c}
    if c["op"] == "quantize":
        st["x"] = _hidden(g, c["m"], c["k"], c["type"])
    elif c["op"] == "linear":
        st["x"] = _hidden(g, c["m"], c["k"], c["type"])
        st["q"] = _weight(g, c["n"], c["k"])
        st["residual"] = _hidden(g, c["m"], c["n"], c["type"]) if c["act"] == "add" else None
        if own:   # a weight's scales are laid out for the tensor cores once, when it is loaded
            st["q"] = _framework()[0].prepare(st["q"])
    else:
        t, e = c["t"], c["e"]
        # router logits of trained models: a token's few likely experts over a broad rest, some experts popular
        x = torch.randn(t, e, generator=g, device="cuda") * 1.3 + torch.randn(e, generator=g, device="cuda") * 0.4 - 1.0
        st["logits"] = x.to(TYPES[c["type"]])
        if c["op"] == "route":
            st["bias"] = torch.randn(e, generator=g, device="cuda") * 0.01 if c["score"] == "sigmoid" else None
            st["dw"] = torch.randn(t, c["k"], generator=g, device="cuda")
            st["leaf"] = st["logits"].clone().requires_grad_()
        else:
            st["ids"] = torch.topk(st["logits"].float(), c["k"], dim=-1)[1]
            st["mask"] = torch.arange(t, device="cuda") < max(1, int(t * 0.8)) if c["masked"] else None
            st["leaf"] = st["logits"].clone().requires_grad_()
    return st


# ---------------------------------------------------------------------------------------------- the framework's calls
def _own(st):
    D, R = _framework()
    c = st["case"]
    if c["op"] == "quantize":
        q = D.quantize(st["x"], per_row=c["per_row"])
        return {"values": D.dequant(q), "scales": q["sc"].view(torch.float8_e4m3fn), "s": q["s"]}
    if c["op"] == "linear":
        return D.qlinear_a4(st["q"], st["x"], act=c["act"] if c["act"] == "relu2" else None, residual=st["residual"])
    if c["op"] == "route":
        args = dict(top_k=c["k"], scaling=5.0, n_group=c["groups"], topk_group=c["kept"], norm_topk_prob=c["norm"],
                    score=c["score"])
        if not c["train"]:
            ids, w, n = R.route(st["logits"], st["bias"], **args)
            return {"ids": ids, "weights": w, "counts": n}
        ids, w, n = R.route(st["leaf"], st["bias"], **args)
        return {"ids": ids, "weights": w.detach(), "counts": n, "dlogits": torch.autograd.grad(w, st["leaf"], st["dw"])[0]}
    loss, n = R.balance_loss(st["leaf"], st["ids"], mask=st["mask"], score=c["score"], coef=0.01)
    return {"loss": loss.detach(), "counts": n, "dlogits": torch.autograd.grad(loss, st["leaf"])[0]}


# ---------------------------------------------------------------------------------------------- plain forms
def _e4m3_table(device, dtype):
    i = torch.arange(127, device=device, dtype=dtype)
    e, m = torch.floor(i / 8), torch.remainder(i, 8)
    return torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e - 10))


def _quantize(x, per_row):
    """(codes' values, block scales, s): s the smallest power of two with the largest value <= 6 * 448 * s, block scale
    the nearest e4m3 of amax / 6, values the nearest e2m1, ties to even. Midpoints times a scale have few bits: each
    comparison is exact in 32 bits."""
    m, k = x.shape
    x = x.float()
    finite = torch.isfinite(x)
    a = torch.where(finite, x.abs(), 0.0)
    amax = a.amax(1) if per_row else a.max().reshape(1)
    mant, ex = torch.frexp(amax)          # amax = mant * 2^ex, mant in [0.5, 1)
    s = torch.ldexp(torch.ones_like(amax), torch.where(mant * 2 <= 1.3125, ex - 12, ex - 11).clamp(min=-126))
    s = torch.where(amax > 0, s, 2.0 ** -126)
    u = (x / s[:, None]).reshape(m, k // 16, 16)
    au = u.abs()
    table = _e4m3_table(x.device, torch.float32)
    bounds = 6 * 0.5 * (table[1:] + table[:-1])
    bmax = torch.where(torch.isfinite(u), au, 0.0).amax(-1)
    low, up = torch.bucketize(bmax, bounds), torch.bucketize(bmax, bounds, right=True)
    sc = table[torch.where(low % 2 == 0, low, up)]
    d = sc[..., None]
    v = 0.5 * (au > 0.25 * d) + 0.5 * (au >= 0.75 * d) + 0.5 * (au > 1.25 * d) + 0.5 * (au >= 1.75 * d)
    v = v + 1.0 * (au > 2.5 * d) + 1.0 * (au >= 3.5 * d) + 2.0 * (au > 5.0 * d)
    v = torch.where(d > 0, torch.copysign(v, u), 0.0)
    sc = torch.where(finite.reshape(m, k // 16, 16).all(-1), sc, float("nan"))
    return v, sc, s


def _values(q):
    """A stored weight's values, without its tensor scale."""
    lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), device="cuda")
    code = torch.stack((q["w"] & 15, q["w"] >> 4), -1).reshape(q["N"], q["K"] // 16, 16)
    return (lut[code.long()] * q["sc"].view(torch.float8_e4m3fn).float()[..., None]).reshape(q["N"], q["K"])


def _act(y, kind, residual, to):
    y = y.to(to)
    if kind == "relu2":
        return torch.relu(y.float()).square().to(to)
    if kind == "add":
        return (y.float() + residual.float()).to(to)
    return y


def _scores(x, score):
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    z = torch.exp(x - x.amax(-1, keepdim=True))
    return z / z.sum(-1, keepdim=True)


def _choose(choice, groups, kept, k, fill):
    t, e = choice.shape
    if groups > 1:
        g = choice.reshape(t, groups, e // groups)
        best = torch.sort(g, dim=-1, descending=True)[0][..., :2].sum(-1)
        order = torch.sort(best, dim=-1, descending=True, stable=True)[1][:, :kept]
        keep = torch.zeros_like(best).scatter_(1, order, 1.0) > 0
        choice = torch.where(keep[..., None], g, fill).reshape(t, e)
    return torch.sort(choice, dim=-1, descending=True, stable=True)[1][:, :k]


def _plain(st):
    c = st["case"]
    if c["op"] == "quantize":
        v, sc, s = _quantize(st["x"], c["per_row"])
        values = (v * (sc * s[:, None])[..., None]).reshape(st["x"].shape).to(torch.bfloat16)
        return {"values": values, "scales": sc.to(torch.float8_e4m3fn), "s": s}
    if c["op"] == "linear":
        x, q = st["x"], st["q"]
        v, sc, s = _quantize(x, True)
        y = (v * sc[..., None]).reshape(x.shape) @ _values(q).t()
        return _act(y * s[:, None] * q["s"], c["act"], st["residual"], x.dtype)
    x = st["logits"].float()
    t, e = x.shape
    s = _scores(x, c["score"])
    if c["op"] == "route":
        # a softmax is chosen by its logits, which have its order; a left-out group counts as 0, or as -inf for logits
        choice = s + st["bias"] if c["score"] == "sigmoid" else x
        ids = _choose(choice, c["groups"], c["kept"], c["k"], 0.0 if c["score"] == "sigmoid" else -float("inf"))
        n = torch.zeros(e, dtype=torch.int32, device=x.device)
        n = n.scatter_add_(0, ids.reshape(-1), torch.ones_like(ids.reshape(-1), dtype=torch.int32))
        picked = s.gather(1, ids)
        total = picked.sum(-1, keepdim=True) + 1e-20
        w = (picked / total if c["norm"] else picked) * 5.0
        out = {"ids": ids, "weights": w, "counts": n}
        if c["train"]:
            d = st["dw"] * 5.0
            if c["norm"]:
                d = (d - (d * picked).sum(-1, keepdim=True) / total) / total
            ds = torch.zeros_like(s).scatter_(1, ids, d)
            if c["score"] == "sigmoid":
                dl = ds * s * (1.0 - s)
            else:
                dl = s * (ds - (ds * s).sum(-1, keepdim=True))
            out["dlogits"] = dl.to(st["logits"].dtype)
        return out
    keep = st["mask"] if st["mask"] is not None else torch.ones(t, dtype=torch.bool, device=x.device)
    rows = keep.sum()
    ids = torch.where(keep[:, None], st["ids"], e).reshape(-1)
    n = torch.zeros(e + 1, dtype=torch.int32, device=x.device)
    n = n.scatter_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))[:e]
    f = n.float() * (e / (c["k"] * rows.float()))
    total = s.sum(-1, keepdim=True)
    p = torch.where(keep[:, None], s / total, 0.0)
    loss = 0.01 * (f * (p.sum(0) / rows)).sum()
    a = 0.01 * f / rows
    d = a - (a * p).sum(-1, keepdim=True)
    dl = p * d * (1.0 - s) if c["score"] == "sigmoid" else p * d
    return {"loss": loss, "counts": n, "dlogits": torch.where(keep[:, None], dl, 0.0).to(st["logits"].dtype)}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------- what a pass has to do
def work(case):
    c = case
    size = {"bf16": 2, "f16": 2, "f32": 4}[c["type"]]
    if c["op"] == "quantize":   # the values come back too, in two bytes each
        n = c["m"] * c["k"]
        return {"bytes": n * (size + 0.5625 + 2) + 4 * c["m"], "flops": 4 * n}
    if c["op"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * k * size + 0.5625 * n * k + m * n * size * (2 if c["act"] == "add" else 1), "flops": 2 * m * n * k}
    t, e, k = c["t"], c["e"], c["k"]
    if c["op"] == "route":
        grad = t * e * size + t * k * 4 if c["train"] else 0
        return {"bytes": t * e * size + 12 * t * k + 8 * e + grad, "flops": 8 * t * e}
    return {"bytes": 2 * t * e * size + 8 * t * k + 4 * e, "flops": 12 * t * e}


# ---------------------------------------------------------------------------------------------- in 64 bits
def _exact_quantize(x, per_row):
    x = x.double()
    m, k = x.shape
    top = x.abs().amax(1) if per_row else x.abs().max().reshape(1)
    s = torch.exp2(torch.ceil(torch.log2((top / 2688).clamp_min(2.0 ** -126))))
    s = torch.where(top > 2688 * s, 2 * s, torch.where(2 * top <= 2688 * s, s / 2, s)).clamp_min(2.0 ** -126)
    b = x.reshape(m, k // 16, 16) / s[:, None, None]
    r = b.abs().amax(-1) / 6
    step = torch.exp2(torch.floor(torch.log2(r.clamp_min(2.0 ** -6))) - 3)
    sc = torch.round(r / step) * step                       # torch.round: halves to even
    r = torch.where(sc[..., None] > 0, b / sc[..., None], 0.0)
    step = torch.where(r.abs() < 2, 0.5, torch.where(r.abs() < 4, 1.0, 2.0)).to(r.dtype)
    return torch.clamp(torch.round(r / step) * step, -6, 6), sc, s


def exact(case, seed):
    st = prepare(case, seed)
    c = case
    if c["op"] == "quantize":
        v, sc, s = _exact_quantize(st["x"], c["per_row"])
        return {"values": (v * sc[..., None]).reshape(c["m"], c["k"]) * s[:, None], "scales": sc, "s": s}
    if c["op"] == "linear":
        q = st["q"]
        v, sc, s = _exact_quantize(st["x"], True)
        lut = torch.tensor(E2M1 + tuple(-x for x in E2M1), device="cuda", dtype=torch.float64)
        w = torch.empty(c["n"], c["k"], device="cuda", dtype=torch.float64)
        w[:, 0::2], w[:, 1::2] = lut[(q["w"] & 15).int()], lut[(q["w"] >> 4).int()]
        w *= q["sc"].view(torch.float8_e4m3fn).double().repeat_interleave(16, 1) * q["s"].double()
        y = ((v * sc[..., None]).reshape(c["m"], c["k"]) * s[:, None]) @ w.T
        if c["act"] == "relu2":
            y = y.clamp_min(0) ** 2
        return y + st["residual"].double() if c["act"] == "add" else y
    x = st["logits"].double()
    p = torch.sigmoid(x) if c["score"] == "sigmoid" else torch.softmax(x, -1)
    if c["op"] == "route":
        # the choice is made on 32-bit scores: their order is the definition
        pick = (torch.sigmoid(st["logits"].float()) + st["bias"]) if c["score"] == "sigmoid" else st["logits"].float()
        if c["groups"] > 1:
            g = pick.unflatten(1, (c["groups"], -1))
            best = g.topk(2, -1)[0].sum(-1)
            rank = ((best[:, None, :] > best[:, :, None]) | ((best[:, None, :] == best[:, :, None]) &
                    torch.ones(c["groups"], c["groups"], device="cuda").tril(-1).bool())).sum(-1)
            pick = torch.where((rank < c["kept"])[..., None], g, 0.0 if c["score"] == "sigmoid" else -torch.inf).flatten(1)
        ids = torch.argsort(pick, dim=1, descending=True, stable=True)[:, :c["k"]]
        leaf = x.clone().requires_grad_()
        q = torch.sigmoid(leaf) if c["score"] == "sigmoid" else torch.softmax(leaf, -1)
        w = q.gather(1, ids)
        w = 5.0 * (w / (w.sum(1, True) + 1e-20) if c["norm"] else w)
        out = {"ids": ids, "weights": w.detach(), "counts": torch.bincount(ids.flatten(), minlength=c["e"])}
        if c["train"]:
            out["dlogits"] = torch.autograd.grad(w, leaf, st["dw"].double())[0]
        return out
    keep = st["mask"] if st["mask"] is not None else torch.ones(c["t"], dtype=torch.bool, device="cuda")
    n = torch.bincount(st["ids"][keep].flatten(), minlength=c["e"])
    leaf = x[keep].requires_grad_()
    p = torch.sigmoid(leaf) if c["score"] == "sigmoid" else torch.softmax(leaf, -1)
    loss = 0.01 * (n * (c["e"] / (c["k"] * int(keep.sum()))) * (p / p.sum(-1, True)).mean(0)).sum()
    grad = torch.zeros_like(x)
    grad[keep] = torch.autograd.grad(loss, leaf)[0]
    return {"loss": loss.detach(), "counts": n, "dlogits": grad}
