"""The two ends of a training step beside those of perf/operators.py, as cases that can be timed and compared.

``embed``         y = scale * w[ids], a token's row of the embedding; zeros for padding
``embed_grad``    its gradient over the whole vocabulary, scale times the sum of each token's rows of dy
``distill``       the distillation loss of the logits x W^T, which are not kept, from a teacher's top logits of each
                  row: loss, log-sum-exp of the tempered logits and the logits at the teacher's entries
``distill_grad``  its gradients dx and dW, from the rows' loss gradients
``policy``        clipped policy loss with a KL term over a padded batch of token log probabilities: its mean, that of
                  the KL term, of the clipped tokens and of the ratio, and each sequence's weight for the backward pass
``policy_grad``   its gradient for every token's log probability

``run`` computes them in plain torch operations in fp32 (the policy loss in fp64, for ratios next to a bound and the
sums over a batch), or, where ``own`` is true, by the library's entry points.  Sizes are those of the repository's
benchmark, examples and tests where it has them, and generic ones elsewhere.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
PAD = -1
CLIP = (0.2, 0.28)
KL = 0.05


def listed():
    return [
        # one decoded token: launch latency
        {"name": "embed_f16_token", "op": "embed", "dtype": "f16", "w_dtype": "f16", "m": 1, "v": 32000, "n": 4096},
        # a training batch out of an fp32 master weight: memory traffic
        {"name": "embed_bf16_train", "op": "embed", "dtype": "bf16", "w_dtype": "f32", "m": 16384, "v": 128000,
         "n": 4096},
        # the gradient of a small fp32 model whose sizes are multiples of no vector
        {"name": "embed_grad_f32_ragged", "op": "embed_grad", "dtype": "f32", "w_dtype": "f32", "m": 1003, "v": 997,
         "n": 515},
        # the gradient of that training batch: most of the vocabulary gets zeros, a few tokens hundreds of rows
        {"name": "embed_grad_bf16_train", "op": "embed_grad", "dtype": "bf16", "w_dtype": "bf16", "m": 16384,
         "v": 128000, "n": 4096},
        # a small student over an odd number of classes
        {"name": "distill_f16_classes", "op": "distill", "dtype": "f16", "t_dtype": "f32", "m": 300, "v": 32003,
         "k": 1024, "top": 20, "temp": 2.0},
        # its gradients
        {"name": "distill_grad_f16_classes", "op": "distill_grad", "dtype": "f16", "t_dtype": "f32", "m": 300,
         "v": 32003, "k": 1024, "top": 20, "temp": 2.0},
        # a large student over a large vocabulary on 4096 tokens
        {"name": "distill_bf16_train", "op": "distill", "dtype": "bf16", "t_dtype": "bf16", "m": 4096, "v": 128000,
         "k": 4096, "top": 64, "temp": 1.0},
        # its gradients: the largest case
        {"name": "distill_grad_bf16_train", "op": "distill_grad", "dtype": "bf16", "t_dtype": "bf16", "m": 4096,
         "v": 128000, "k": 4096, "top": 64, "temp": 1.0},
        # a few short answers, the mean of the sequences' means: launch latency
        {"name": "policy_few", "op": "policy", "mean": "sequences", "b": 8, "t": 100, "ref": True, "per_token": False},
        # its gradient
        {"name": "policy_grad_few", "op": "policy_grad", "mean": "sequences", "b": 8, "t": 100, "ref": True,
         "per_token": False},
        # a batch of long answers with an advantage for each token: memory traffic
        {"name": "policy_train", "op": "policy", "mean": "tokens", "b": 1024, "t": 8192, "ref": True,
         "per_token": True},
        # its gradient
        {"name": "policy_grad_train", "op": "policy_grad", "mean": "tokens", "b": 1024, "t": 8192, "ref": True,
         "per_token": True},
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
        op = rng.choice(("embed", "embed_grad", "embed_grad", "distill", "distill_grad", "distill_grad", "policy",
                         "policy_grad"))
        dtype = rng.choice(("f16", "bf16", "bf16", "f32"))
        c = {"op": op}
        if op in ("embed", "embed_grad"):
            c.update(dtype=dtype, w_dtype=rng.choice((dtype, "f32")), m=int(_log(rng, 1, 65537)),
                     v=_size(rng, 64, 262144), n=_size(rng, 64, 8192))
            big = c["v"] * c["n"] > 6e8 or c["m"] * c["n"] > 3e8
        elif op in ("distill", "distill_grad"):
            c.update(dtype=dtype, t_dtype=rng.choice((dtype, "f32")), m=int(_log(rng, 1, 8193)),
                     v=_size(rng, 512, 131072), k=_size(rng, 64, 8192), top=int(_log(rng, 1, 257)),
                     temp=rng.choice((1.0, 1.0, 0.7, 2.0, 4.0)))
            # at most about the time of the largest listed case
            big = work(c)["flops"] > (1.3e12 if dtype == "f32" else 1.28e13)
        else:
            c.update(mean=rng.choice(("tokens", "sequences", "sum")), b=int(_log(rng, 1, 2049)),
                     t=_size(rng, 1, 32768), ref=rng.choice((True, True, False)), per_token=rng.choice((True, False)))
            big = c["b"] * c["t"] > 1024 * 8192
        if not big:
            return c


def work(case):
    op = case["op"]
    if op in ("embed", "embed_grad"):
        m, v, n, es, ws = case["m"], case["v"], case["n"], SIZE[case["dtype"]], SIZE[case["w_dtype"]]
        if op == "embed":
            return {"bytes": m * n * (es + ws) + 8 * m, "flops": m * n}
        return {"bytes": m * n * es + v * n * ws + 8 * m, "flops": m * n}
    if op in ("distill", "distill_grad"):
        m, v, k, es = case["m"], case["v"], case["k"], SIZE[case["dtype"]]
        entries = m * case["top"] * (12 + SIZE[case["t_dtype"]])
        if op == "distill":
            return {"bytes": es * (m * k + v * k) + entries + 8 * m, "flops": 2 * m * v * k}
        # the logits again, then both gradients
        return {"bytes": 2 * es * (m * k + v * k) + entries + 8 * m, "flops": 6 * m * v * k}
    tokens = case["b"] * case["t"]
    arrays = 2 + case["ref"] + case["per_token"] + (op == "policy_grad")
    return {"bytes": tokens * (4 * arrays + 1) + 8 * case["b"], "flops": 20 * tokens}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    def empty(*shape, dtype=torch.float32):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    s = {"case": case}
    if op in ("embed", "embed_grad"):
        m, v, n, dt, wt = case["m"], case["v"], case["n"], TORCH[case["dtype"]], TORCH[case["w_dtype"]]
        # tokens that favour the low ids, as token frequencies do, and the padding behind sequences of a batch
        ids = (v ** rand(m) - 1).long().clamp(0, v - 1)
        s["ids"] = torch.where(torch.arange(m, device="cuda") % 512 >= 512 - int(64 * rand(1)), PAD, ids)
        s["scale"] = float(torch.tensor(n ** 0.5))    # as an fp32 argument holds it
        if op == "embed":
            s["w"], s["y"] = normal(v, n, scale=n ** -0.5, dtype=wt), empty(m, n, dtype=dt)
        else:
            s["dy"], s["dw"] = normal(m, n, scale=0.1, dtype=dt), empty(v, n, dtype=wt)
        return s

    if op in ("distill", "distill_grad"):
        m, v, k, top = case["m"], case["v"], case["k"], min(case["top"], case["v"])
        dt, tt = TORCH[case["dtype"]], TORCH[case["t_dtype"]]
        s["x"], s["w"] = normal(m, k, dtype=dt), normal(v, k, scale=2.0 * k ** -0.5, dtype=dt)
        # distinct classes that favour the low ones, in the order of the teacher's logits
        j = torch.arange(top, device="cuda")
        ids = ((v - top + 1) ** ((j + rand(m, top)) / top) - 1).long().clamp(0, v - top) + j
        t, order = torch.sort(normal(m, top, scale=2.0), 1, descending=True)
        ids = ids.gather(1, torch.argsort(rand(m, top), 1)).gather(1, order)
        # a row in three keeps only its first entries, and one in twenty (a prompt's) has no teacher
        kept = torch.where(rand(m) < 0.33, (1 + top * rand(m)).long(), top)
        kept = torch.where(rand(m) < 0.05, 0, kept)
        absent = j >= kept[:, None]
        s["top"] = torch.where(absent, -1, ids).contiguous()
        s["t"] = torch.where(absent, float("-inf"), t).to(tt)
        s["loss"], s["lse"], s["z_top"] = empty(m), empty(m), empty(m, top)
        if op == "distill":
            return s
        z = s["x"].float() @ s["w"].float().t()
        s["z_top"] = torch.where(absent, 0.0, z.gather(1, s["top"].clamp(min=0)))
        s["lse"] = torch.logsumexp(z.div_(case["temp"]), 1)
        # the mean over the rows that count; fp16 programs scale their loss so that gradients keep their bits
        count = int((kept > 0).sum())
        s["dloss"] = torch.full((m,), (1024.0 if case["dtype"] == "f16" else 1.0) / max(1, count), device="cuda")
        s["dx"], s["dw"] = empty(m, k, dtype=dt), empty(v, k, dtype=dt)
        return s

    b, t = case["b"], case["t"]
    # log probabilities of a policy a few updates away from the one that wrote the answers, and from the reference
    s["old"] = torch.log(rand(b, t) + 1e-6)
    s["logp"] = s["old"] + normal(b, t, scale=0.15)
    s["ref"] = s["old"] + normal(b, t, scale=0.3) if case["ref"] else None
    s["adv"] = normal(b, t) if case["per_token"] else normal(b, 1)
    lengths = (1 + t * rand(b)).long()
    s["mask"] = (torch.arange(t, device="cuda") < lengths[:, None]).to(torch.uint8)
    if op == "policy":
        s["stats"], s["norm"] = empty(4), empty(b)
        return s
    s["norm"] = _norm(case["mean"], s["mask"]).float()
    s["dloss"], s["dlogp"] = torch.ones((), device="cuda"), empty(b, t)
    return s


def _norm(mean, mask):
    """The weight of a token of each sequence, in 64 bits; 0 for sequences without tokens."""
    n = mask.double().sum(1)
    some = (n > 0).double()
    if mean == "tokens":
        return some / n.sum().clamp(min=1)
    if mean == "sequences":
        return some / (n.clamp(min=1) * some.sum().clamp(min=1))
    return some


def _bounds():
    """Those of the ratio, from the fp32 numbers that a call is given."""
    low, high = torch.tensor(CLIP).double().tolist()
    return 1 - low, 1 + high


# ---------------------------------------------------------------- plain form

def _teacher(t, top, temp):
    """The teacher's probabilities q over a row's entries and their logarithms; q is 0 for absent entries and in rows
    without any."""
    t = torch.where(top >= 0, t.float() / temp, float("-inf"))
    high = t.max(1, keepdim=True).values
    t = t - torch.where(high > float("-inf"), high, 0.0)
    total = torch.exp(t).sum(1, keepdim=True)
    log_q = t - torch.log(torch.where(total > 0, total, 1.0))
    return torch.exp(log_q), log_q


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "embed":
        y = s["w"][s["ids"].clamp(min=0)].float() * s["scale"]
        return torch.where((s["ids"] == PAD)[:, None], 0.0, y).to(s["y"].dtype)
    if op == "embed_grad":
        rows = s["dy"].float() * (s["scale"] * (s["ids"] != PAD))[:, None]
        dw = torch.zeros(case["v"], case["n"], device="cuda")
        return dw.index_add_(0, s["ids"].clamp(min=0), rows).to(s["dw"].dtype)
    if op in ("distill", "distill_grad"):
        temp, top = case["temp"], s["top"]
        x, w = s["x"].float(), s["w"].float()
        z = x @ w.t()
        q, log_q = _teacher(s["t"], top, temp)
        if op == "distill":
            z_top = torch.where(top >= 0, z.gather(1, top.clamp(min=0)), 0.0)
            z = z / temp
            high = z.max(1).values
            lse = high + torch.log(torch.exp(z - high[:, None]).sum(1))
            terms = torch.where(q > 0, q * (log_q - (z_top / temp - lse[:, None])), 0.0)
            return {"loss": temp * temp * terms.sum(1), "lse": lse, "z_top": z_top}
        d = torch.exp(z / temp - s["lse"][:, None])
        d.scatter_add_(1, top.clamp(min=0), -q)
        d *= (temp * s["dloss"] * (top >= 0).any(1))[:, None]
        return {"dx": (d @ w).to(s["x"].dtype), "dw": (d.t() @ x).to(s["w"].dtype)}
    # in fp64: which side of a bound a ratio lies on, the KL term's difference, the sums over the batch
    keep, adv, (low, high) = s["mask"] != 0, s["adv"].double(), _bounds()
    ratio = torch.exp(s["logp"].double() - s["old"].double())
    clipped = torch.where(ratio > high, high, torch.where(ratio < low, low, ratio))
    taken = ratio * adv <= clipped * adv
    d = s["ref"].double() - s["logp"].double() if case["ref"] else torch.zeros_like(ratio)
    if op == "policy_grad":
        grad = KL * (1 - torch.exp(d)) - torch.where(taken, ratio * adv, 0.0)
        return torch.where(keep, s["dloss"] * s["norm"][:, None] * grad, 0.0).float()
    norm = _norm(case["mean"], s["mask"])
    kl = torch.exp(d) - d - 1
    loss = KL * kl - torch.where(taken, ratio, clipped) * adv

    def mean(a):
        return (torch.where(keep, a.double(), 0.0).sum(1) * norm).sum()
    return {"stats": torch.stack([mean(loss), mean(kl), mean(~taken), mean(ratio)]).float(), "norm": norm.float()}


# ------------------------------------------------------- the library's calls

def _own(s):
    import vkblas_amd as vk
    case = s["case"]
    op = case["op"]
    code = {"f32": vk.DT_F32, "f16": vk.DT_F16, "bf16": vk.DT_BF16}
    stream = torch.cuda.current_stream().cuda_stream
    if op in ("embed", "embed_grad"):
        m, v, n, et, wt = case["m"], case["v"], case["n"], code[case["dtype"]], code[case["w_dtype"]]
        if op == "embed":
            vk.embedding_async(et, wt, m, v, n, s["ids"].data_ptr(), PAD, s["w"].data_ptr(), n, s["scale"],
                               s["y"].data_ptr(), n, stream=stream)
            return s["y"]
        vk.embedding_backward_async(et, m, v, n, s["ids"].data_ptr(), PAD, s["dy"].data_ptr(), n, s["scale"],
                                    s["dw"].data_ptr(), n, wt, 0.0, stream=stream)
        return s["dw"]
    if op in ("distill", "distill_grad"):
        m, v, k, et, tt = case["m"], case["v"], case["k"], code[case["dtype"]], code[case["t_dtype"]]
        top = s["top"].shape[1]
        x, w, ids, t = s["x"].data_ptr(), s["w"].data_ptr(), s["top"].data_ptr(), s["t"].data_ptr()
        if op == "distill":
            vk.linear_distill_async(et, m, v, k, x, k, w, k, top, ids, top, tt, t, top, case["temp"],
                                    s["loss"].data_ptr(), s["lse"].data_ptr(), s["z_top"].data_ptr(), stream=stream)
            return {"loss": s["loss"], "lse": s["lse"], "z_top": s["z_top"]}
        vk.linear_distill_backward_async(et, m, v, k, x, k, w, k, top, ids, top, tt, t, top, case["temp"],
                                         s["lse"].data_ptr(), s["z_top"].data_ptr(), s["dloss"].data_ptr(),
                                         s["dx"].data_ptr(), k, s["dw"].data_ptr(), k, et, 0.0, stream=stream)
        return {"dx": s["dx"], "dw": s["dw"]}
    b, t = case["b"], case["t"]
    mean = {"tokens": vk.REDUCE_TOKENS, "sequences": vk.REDUCE_SEQUENCES, "sum": vk.REDUCE_SUM}[case["mean"]]
    ref = s["ref"].data_ptr() if case["ref"] else None
    args = (mean, b, t, s["logp"].data_ptr(), t, s["old"].data_ptr(), t, ref, t, s["adv"].data_ptr(),
            t if case["per_token"] else 1, int(case["per_token"]), s["mask"].data_ptr(), t, *CLIP, KL)
    if op == "policy":
        vk.policy_loss_async(*args, s["stats"].data_ptr(), s["norm"].data_ptr(), stream=stream)
        return {"stats": s["stats"], "norm": s["norm"]}
    vk.policy_loss_backward_async(*args[1:], s["norm"].data_ptr(), s["dloss"].data_ptr(), s["dlogp"].data_ptr(), t,
                                  stream=stream)
    return s["dlogp"]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------ the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embed":
        one = torch.zeros(1, case["n"], device="cuda", dtype=torch.float64)
        return torch.cat((s["w"].double() * s["scale"], one))[s["ids"]]    # PAD is the last row
    if op == "embed_grad":
        if case["v"] * case["n"] > 2e9:
            return None
        dw = torch.zeros(case["v"] + 1, case["n"], device="cuda", dtype=torch.float64)
        dw.index_add_(0, torch.where(s["ids"] == PAD, case["v"], s["ids"]), s["dy"].double())
        return dw[:-1] * s["scale"]
    if op in ("distill", "distill_grad"):
        # the row's loss as T^2 times a cross entropy minus the teacher's entropy, over the classes themselves
        temp, m, v = case["temp"], case["m"], case["v"]
        x, w = s["x"].double(), s["w"].double()
        there = s["top"] >= 0
        counted = there.any(1)
        out = {"loss": [], "lse": [], "z_top": []}
        dx, dw = torch.empty_like(x), torch.zeros_like(w)
        for a in range(0, m, 512):
            r = slice(a, min(m, a + 512))
            t = torch.where(there[r], s["t"][r].double() / temp, float("-inf"))
            q = torch.where(counted[r, None], torch.softmax(t, 1), 0.0)
            z = x[r] @ w.t()
            if op == "distill":
                lse = torch.logsumexp(z / temp, 1)
                at = z.gather(1, s["top"][r].clamp(min=0))
                cross = (q * (lse[:, None] - at / temp)).sum(1)
                out["loss"].append(temp ** 2 * (cross + torch.special.xlogy(q, q).sum(1)))
                out["lse"].append(lse)
                out["z_top"].append(torch.where(there[r], at, 0.0))
                continue
            d = torch.exp(z / temp - s["lse"][r].double()[:, None])
            d.scatter_add_(1, s["top"][r].clamp(min=0), -q)
            d *= (temp * s["dloss"][r].double() * counted[r])[:, None]
            dx[r] = d @ w
            dw += d.t() @ x[r]
        return {k: torch.cat(a) for k, a in out.items()} if op == "distill" else {"dx": dx, "dw": dw}
    logp = s["logp"].double().requires_grad_()
    keep = s["mask"] != 0
    norm = _norm(case["mean"], s["mask"])
    with torch.enable_grad():
        adv = s["adv"].double()
        ratio = torch.exp(logp - s["old"].double())
        plain, bounded = ratio * adv, ratio.clamp(*_bounds()) * adv
        kl = torch.zeros_like(ratio)
        if case["ref"]:
            d = s["ref"].double() - logp
            kl = torch.expm1(d) - d
        loss = KL * kl - torch.minimum(plain, bounded)
    if op == "policy":
        means = [(torch.where(keep, a.double(), 0.0).sum(1) * norm).sum()
                 for a in (loss.detach(), kl.detach(), plain > bounded, ratio.detach())]
        return {"stats": torch.stack(means), "norm": norm}
    weight = torch.where(keep, s["norm"].double()[:, None], 0.0)
    return torch.autograd.grad((loss * weight).sum(), logp)[0] * s["dloss"].double()
