"""The operators of a training step around the library's products, as cases that can be timed and compared.

``norm``       y = layer norm of x, its rows' mean and 1 / deviation kept for the backward pass
``norm_grad``  its gradients: dx, and the weight's and bias's over all rows
``glu``        h = act(x Wg^T) * (x Wu^T), the gated feed-forward block up to its down projection; W holds
               the gate's rows, then the up projection's; a training pass keeps both projections
``glu_grad``   its gradients dx and dW from dh and the kept projections
``xent``       softmax cross entropy of the logits x W^T without keeping them: each row's loss and log-sum-exp
``xent_grad``  its gradients dx and dW, from the rows' loss gradients

``run`` computes them in plain fp32 torch operations, or, where ``own`` is true, by the library's entry points.
Sizes are those of the repository's benchmark and tests where it has them, and generic layer sizes elsewhere.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
IGNORE = -100
EPS = 1e-5


def listed():
    return [
        # one token through a norm in front of a projection: launch latency
        {"name": "norm_f16_token", "op": "norm", "dtype": "f16", "w_dtype": "f16", "m": 1, "n": 4096},
        # a training batch of 8192 tokens, the weight in fp32: memory traffic
        {"name": "norm_bf16_train", "op": "norm", "dtype": "bf16", "w_dtype": "f32", "m": 8192, "n": 4096},
        # the gradients of that batch
        {"name": "norm_grad_bf16_train", "op": "norm_grad", "dtype": "bf16", "w_dtype": "f32", "m": 8192, "n": 4096},
        # gradients of a small fp32 model's norm, rows that are multiples of no vector
        {"name": "norm_grad_f32_ragged", "op": "norm_grad", "dtype": "f32", "w_dtype": "f32", "m": 1003, "n": 997},
        # one token through a large gated block: its weights are read once
        {"name": "glu_f16_token", "op": "glu", "dtype": "f16", "act": "silu", "m": 1, "n": 14336, "k": 4096,
         "keep": False},
        # a small fp32 gated block whose sizes are multiples of no tile
        {"name": "glu_f32_ragged", "op": "glu", "dtype": "f32", "act": "gelu", "m": 200, "n": 500, "k": 784,
         "keep": True},
        # the training pass of a large block on 8192 tokens
        {"name": "glu_bf16_train", "op": "glu", "dtype": "bf16", "act": "silu", "m": 8192, "n": 11008, "k": 4096,
         "keep": True},
        # its gradients
        {"name": "glu_grad_bf16_train", "op": "glu_grad", "dtype": "bf16", "act": "silu", "m": 8192, "n": 11008,
         "k": 4096},
        # the loss of a small model over an odd number of classes
        {"name": "xent_f16_classes", "op": "xent", "dtype": "f16", "m": 1000, "n": 32003, "k": 1024},
        # its gradients
        {"name": "xent_grad_f16_classes", "op": "xent_grad", "dtype": "f16", "m": 1000, "n": 32003, "k": 1024},
        # the loss of a large model over a large vocabulary on 4096 tokens
        {"name": "xent_bf16_train", "op": "xent", "dtype": "bf16", "m": 4096, "n": 128000, "k": 4096},
        # its gradients: the largest case
        {"name": "xent_grad_bf16_train", "op": "xent_grad", "dtype": "bf16", "m": 4096, "n": 128000, "k": 4096},
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _size(rng, lo, hi):
    """A size between lo and hi: a multiple of 64, a multiple of 8, or any number."""
    v = _log(rng, lo, hi)
    step = rng.choice((64, 64, 8, 1))
    return int(min(hi, max(lo, step * max(1, round(v / step)))))


def draw(rng):
    while True:
        op = rng.choice(("norm", "norm_grad", "glu", "glu_grad", "xent", "xent_grad"))
        dtype = rng.choice(("f16", "bf16", "bf16", "f32"))
        c = {"op": op, "dtype": dtype}
        if op in ("norm", "norm_grad"):
            c["w_dtype"] = rng.choice((dtype, "f32"))
            c.update(m=int(_log(rng, 1, 16385)), n=_size(rng, 64, 16384))
        elif op in ("glu", "glu_grad"):
            c.update(act=rng.choice(("silu", "gelu", "gelu_tanh", "relu")), m=int(_log(rng, 1, 8193)),
                     n=_size(rng, 64, 14336), k=_size(rng, 64, 8192))
            if op == "glu":
                c["keep"] = rng.choice((True, False))
        else:
            c.update(m=int(_log(rng, 1, 8193)), n=_size(rng, 256, 131072), k=_size(rng, 64, 8192))
        w = work(c)
        flops = 1.3e12 if dtype == "f32" else 1.28e13   # at most about the time of the largest listed case
        if 3072 not in (c["m"], c["n"], c.get("k")) and w["flops"] <= flops and 2e4 <= w["bytes"] <= 3e9:
            return c


def work(case):
    op, es, m, n = case["op"], SIZE[case["dtype"]], case["m"], case["n"]
    if op == "norm":
        return {"bytes": 2 * es * m * n + 2 * SIZE[case["w_dtype"]] * n + 8 * m, "flops": 8 * m * n}
    if op == "norm_grad":
        return {"bytes": 3 * es * m * n + 3 * SIZE[case["w_dtype"]] * n + 8 * m, "flops": 14 * m * n}
    k = case["k"]
    if op == "glu":
        return {"bytes": es * (m * k + 2 * n * k + m * n * (3 if case["keep"] else 1)), "flops": 4 * m * n * k}
    if op == "glu_grad":
        # dh, the projections, x and W read, dx and dW written
        return {"bytes": es * (3 * m * n + 2 * m * k + 4 * n * k), "flops": 8 * m * n * k}
    if op == "xent":
        return {"bytes": es * (m * k + n * k) + 16 * m, "flops": 2 * m * n * k}
    # the logits again, then both gradients
    return {"bytes": 2 * es * (m * k + n * k) + 16 * m, "flops": 6 * m * n * k}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dt, m, n = case["op"], TORCH[case["dtype"]], case["m"], case["n"]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    def empty(*shape, dtype=dt):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    s = {"case": case}
    if op in ("norm", "norm_grad"):
        wt = TORCH[case["w_dtype"]]
        # a residual stream: channels of their own offset and spread, a few of them large
        spread = torch.exp(0.5 * torch.randn(n, device="cuda", generator=g))
        offset = 0.3 * torch.randn(n, device="cuda", generator=g)
        s["x"] = (torch.randn(m, n, device="cuda", generator=g) * spread + offset).to(dt)
        s["w"] = (1 + 0.1 * torch.randn(n, device="cuda", generator=g)).to(wt)
        s["b"] = normal(n, scale=0.1, dtype=wt)
        if op == "norm":
            s["y"] = empty(m, n)
            s["mean"], s["rstd"] = empty(m, dtype=torch.float32), empty(m, dtype=torch.float32)
            return s
        x = s["x"].float()
        s["mean"] = x.mean(1)
        s["rstd"] = torch.rsqrt((x - s["mean"][:, None]).square().mean(1) + EPS)
        s["dy"] = normal(m, n, scale=0.1)
        s["dx"], s["dw"], s["db"] = empty(m, n), empty(n, dtype=wt), empty(n, dtype=wt)
        return s

    k = case["k"]
    s["x"] = normal(m, k)
    if op in ("glu", "glu_grad"):
        s["w"] = normal(2 * n, k, scale=k ** -0.5)
        if op == "glu":
            s["h"] = empty(m, n)
            s["gu"] = empty(m, 2 * n) if case["keep"] else None
            return s
        s["gu"] = (s["x"].float() @ s["w"].float().t()).to(dt)
        s["dh"] = normal(m, n, scale=0.1)
        s["dx"], s["dw"] = empty(m, k), empty(2 * n, k)
        return s

    # logits of a spread of 2; targets that favour the low classes, as token frequencies do, some rows ignored
    s["w"] = normal(n, k, scale=2.0 * k ** -0.5)
    u = torch.rand(m, device="cuda", generator=g)
    t = (n ** u - 1).long().clamp(0, n - 1)
    skip = torch.rand(m, device="cuda", generator=g) < 0.05
    s["target"] = torch.where(skip, torch.full_like(t, IGNORE), t)
    if op == "xent":
        s["loss"], s["lse"] = empty(m, dtype=torch.float32), empty(m, dtype=torch.float32)
        return s
    s["lse"] = torch.logsumexp(s["x"].float() @ s["w"].float().t(), 1)
    # the mean over the rows that count; fp16 programs scale their loss so that gradients keep their bits
    scale = (1024.0 if case["dtype"] == "f16" else 1.0) / max(1, m - int(skip.sum()))
    s["dloss"] = torch.full((m,), scale, device="cuda")
    s["dx"], s["dw"] = empty(m, k), empty(n, k)
    return s


# ---------------------------------------------------------------- plain form

def _act(name, g):
    if name == "silu":
        return g / (1 + torch.exp(-g))
    if name == "gelu":
        return 0.5 * g * (1 + torch.erf(g * 0.5 ** 0.5))
    if name == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh((2 / math.pi) ** 0.5 * (g + 0.044715 * g * g * g)))
    return torch.where(g > 0, g, torch.zeros_like(g))


def _act_slope(name, g):
    if name == "silu":
        p = 1 / (1 + torch.exp(-g))
        return p * (1 + g * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(g * 0.5 ** 0.5)) + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        t = torch.tanh(c * (g + 0.044715 * g * g * g))
        return 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)
    return (g > 0).to(g.dtype)


def _plain(s):
    case = s["case"]
    op, dt, n = case["op"], TORCH[case["dtype"]], case["n"]
    x, w = s["x"].float(), s["w"].float()
    if op == "norm":
        mean = x.mean(1)
        c = x - mean[:, None]
        rstd = torch.rsqrt((c * c).mean(1) + EPS)
        y = c * rstd[:, None] * w + s["b"].float()
        return {"y": y.to(dt), "mean": mean, "rstd": rstd}
    if op == "norm_grad":
        wt, dy, rstd = TORCH[case["w_dtype"]], s["dy"].float(), s["rstd"][:, None]
        xh = (x - s["mean"][:, None]) * rstd
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        return {"dx": dx.to(dt), "dw": (dy * xh).sum(0).to(wt), "db": dy.sum(0).to(wt)}
    if op == "glu":
        gu = x @ w.t()
        h = (_act(case["act"], gu[:, :n]) * gu[:, n:]).to(dt)
        return {"h": h, "gu": gu.to(dt)} if case["keep"] else h
    if op == "glu_grad":
        gu, dh = s["gu"].float(), s["dh"].float()
        g, u = gu[:, :n], gu[:, n:]
        d = torch.cat((dh * u * _act_slope(case["act"], g), dh * _act(case["act"], g)), 1)
        return {"dx": (d @ w).to(dt), "dw": (d.t() @ x).to(dt)}
    z = x @ w.t()
    t, some = s["target"].clamp(min=0), s["target"] != IGNORE
    if op == "xent":
        top = z.max(1).values
        lse = top + torch.log(torch.exp(z - top[:, None]).sum(1))
        loss = torch.where(some, lse - z.gather(1, t[:, None])[:, 0], torch.zeros_like(lse))
        return {"loss": loss, "lse": lse}
    d = torch.exp(z - s["lse"][:, None])
    d[torch.arange(case["m"], device=d.device), t] -= 1
    d *= (s["dloss"] * some)[:, None]
    return {"dx": (d @ w).to(dt), "dw": (d.t() @ x).to(dt)}


# ------------------------------------------------------- the library's calls

def _own(s):
    import vkblas_amd as vk
    case = s["case"]
    op, m, n = case["op"], case["m"], case["n"]
    code = {"f32": vk.DT_F32, "f16": vk.DT_F16, "bf16": vk.DT_BF16}
    et = code[case["dtype"]]
    stream = torch.cuda.current_stream().cuda_stream
    x, w = s["x"].data_ptr(), s["w"].data_ptr()
    if op == "norm":
        vk.layer_norm_async(et, code[case["w_dtype"]], m, n, x, n, w, s["b"].data_ptr(), EPS, s["y"].data_ptr(), n,
                            s["mean"].data_ptr(), s["rstd"].data_ptr(), stream=stream)
        return {"y": s["y"], "mean": s["mean"], "rstd": s["rstd"]}
    if op == "norm_grad":
        wt = code[case["w_dtype"]]
        vk.layer_norm_backward_async(et, wt, m, n, s["dy"].data_ptr(), n, x, n, w, s["mean"].data_ptr(),
                                     s["rstd"].data_ptr(), s["dx"].data_ptr(), n, s["dw"].data_ptr(),
                                     s["db"].data_ptr(), wt, 0.0, stream=stream)
        return {"dx": s["dx"], "dw": s["dw"], "db": s["db"]}
    k = case["k"]
    if op in ("glu", "glu_grad"):
        act = {"silu": vk.ACT_SILU, "gelu": vk.ACT_GELU, "gelu_tanh": vk.ACT_GELU_TANH,
               "relu": vk.ACT_RELU}[case["act"]]
    if op == "glu":
        gu = s["gu"].data_ptr() if case["keep"] else None
        vk.glu_async(et, act, m, n, k, x, k, w, k, s["h"].data_ptr(), n, gu, 2 * n, stream=stream)
        return {"h": s["h"], "gu": s["gu"]} if case["keep"] else s["h"]
    if op == "glu_grad":
        vk.glu_backward_async(et, act, m, n, k, s["dh"].data_ptr(), n, s["gu"].data_ptr(), 2 * n, x, k, w, k,
                              None, 0, s["dx"].data_ptr(), k, s["dw"].data_ptr(), k, et, 0.0, stream=stream)
        return {"dx": s["dx"], "dw": s["dw"]}
    if op == "xent":
        vk.linear_xent_async(et, m, n, k, x, k, w, k, s["target"].data_ptr(), IGNORE, s["loss"].data_ptr(),
                             s["lse"].data_ptr(), stream=stream)
        return {"loss": s["loss"], "lse": s["lse"]}
    vk.linear_xent_backward_async(et, m, n, k, x, k, w, k, s["target"].data_ptr(), IGNORE, s["lse"].data_ptr(),
                                  s["dloss"].data_ptr(), s["dx"].data_ptr(), k, s["dw"].data_ptr(), k, et, 0.0,
                                  stream=stream)
    return {"dx": s["dx"], "dw": s["dw"]}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------ the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op, m, n = case["op"], case["m"], case["n"]
    x, w = s["x"].double(), s["w"].double()
    if op == "norm":
        var, mean = torch.var_mean(x, 1, unbiased=False)
        y = (x - mean[:, None]) / torch.sqrt(var + EPS)[:, None] * w + s["b"].double()
        return {"y": y, "mean": mean, "rstd": 1 / torch.sqrt(var + EPS)}
    if op == "norm_grad":
        # dx is the gradient of sum(dy y) with the row's statistics as functions of x: the projection of
        # dy w off the constant vector and off x - mean, times rstd
        dy, r = s["dy"].double(), s["rstd"].double()[:, None]
        xh = (x - s["mean"].double()[:, None]) * r
        g = dy * w
        along = torch.stack([g.sum(1), (g * xh).sum(1)]) / n
        return {"dx": (g - along[0][:, None] - along[1][:, None] * xh) * r,
                "dw": torch.einsum("mn,mn->n", dy, xh), "db": dy.sum(0)}
    if op in ("glu", "glu_grad"):
        f = torch.nn.functional
        act = {"silu": f.silu, "gelu": f.gelu, "gelu_tanh": lambda a: f.gelu(a, approximate="tanh"),
               "relu": f.relu}[case["act"]]
    if op == "glu":
        g, u = x @ w[:n].t(), x @ w[n:].t()
        h = act(g) * u
        return {"h": h, "gu": torch.cat((g, u), 1)} if case["keep"] else h
    if op == "glu_grad":
        gu = s["gu"].double().requires_grad_()
        with torch.enable_grad():
            h = act(gu[:, :n]) * gu[:, n:]
        d, = torch.autograd.grad(h, gu, s["dh"].double())
        return {"dx": d @ w, "dw": d.t() @ x}
    some = s["target"] != IGNORE
    if op == "xent":
        z = x @ w.t()
        loss = torch.nn.functional.cross_entropy(z, s["target"], ignore_index=IGNORE, reduction="none")
        return {"loss": loss, "lse": torch.logsumexp(z, 1)}
    scale = s["dloss"].double() * some
    dx, dw = torch.empty_like(x), torch.zeros_like(w)
    for a in range(0, m, 1024):
        rows = slice(a, min(m, a + 1024))
        p = torch.exp(x[rows] @ w.t() - s["lse"].double()[rows, None])
        hot = torch.nn.functional.one_hot(s["target"][rows].clamp(min=0), n)
        d = (p - hot) * scale[rows, None]
        dx[rows] = d @ w
        dw += d.t() @ x[rows]
    return {"dx": dx, "dw": dw}
