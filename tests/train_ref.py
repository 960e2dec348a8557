"""Definitions in float64 (torch) of the operators in vkblas_train.h, with bounds on how far a correct fp32 evaluation
may be from them; conventions and constants are nn_ref's.

Distillation.  A logit's error is a dot product's (nn_ref.dot_bound, ez).  log-sum-exp moves with the largest of them
over T, and a sum of V positive terms joined in trees and runs of at most 600 is within 600 e relative.  The teacher's
log q has a few roundings of t / T and of the log of a sum of n_top terms (32 e relative for it), so q moves by that
relative to itself.
"""
import math

import torch

from nn_ref import E, STEP, TINY, U, close, dot_bound, rounded  # noqa: F401

PAD = -1


def embedding(w, ids, scale, pad=PAD):
    """y, NaN for ids outside the vocabulary."""
    V = w.shape[0]
    y = scale * w[ids.clamp(0, V - 1)]
    y[(ids < 0) | (ids >= V)] = float("nan")
    y[ids == pad] = 0.0
    return y


def embedding_grad(dy, ids, V, scale, pad=PAD, beta=0.0, dw0=None):
    """dw and its fp32 evaluation's error before the rounding: sums of n rows in any order, scaled and added."""
    there = (ids != pad) & (ids >= 0) & (ids < V)
    zero = torch.zeros(V, dy.shape[1], dtype=torch.float64, device=dy.device)
    at = ids[there]
    total, size = zero.index_add(0, at, dy[there]), zero.index_add(0, at, dy[there].abs())
    n = torch.zeros(V, dtype=torch.float64, device=dy.device).index_add(0, at, torch.ones(len(at), dtype=torch.float64,
                                                                                           device=dy.device))
    old = zero if dw0 is None or beta == 0.0 else beta * dw0
    return scale * total + old, (n[:, None] + 4) * E * (abs(scale) * size + old.abs())


def teacher(top, t, temp, V):
    """q and log q over a row's entries (0 and -inf where absent), which rows count, and which are bad."""
    there = top >= 0
    t = torch.where(there, t / temp, torch.full_like(t, -math.inf))
    high = t.amax(1, keepdim=True)
    counted = high[:, 0] != -math.inf
    t = t - torch.where(counted[:, None], high, torch.zeros_like(high))
    log_q = t - torch.log(torch.where(counted[:, None], t.exp().sum(1, keepdim=True), torch.ones_like(high)))
    return log_q.exp(), log_q, counted, (top >= V).any(1)


def distill(x, w, top, t, temp):
    """loss, lse and z_top with their bounds; NaN losses for bad rows, 0 for rows that are not counted."""
    V = w.shape[0]
    z = x @ w.t()
    ez = dot_bound(x, w.t())
    lse = torch.logsumexp(z / temp, 1)
    e_lse = ez.amax(1) / temp + 600 * E + STEP * (lse.abs() + 1)
    q, log_q, counted, bad = teacher(top, t, temp, V)
    at = top.clamp(0, V - 1)
    zt, ezt = z.gather(1, at), ez.gather(1, at)
    mass = q > 0
    term = torch.where(mass, log_q - zt / temp + lse[:, None], torch.zeros_like(q))
    lq = torch.where(mass, log_q.abs(), torch.zeros_like(q))
    eq = STEP * (4 + lq + (t / temp).nan_to_num(0, 0, 0).abs()) + 32 * E
    e = q * (eq * (1 + term.abs()) + ezt / temp + e_lse[:, None] + STEP * (zt.abs() / temp + lse.abs()[:, None]))
    loss = temp ** 2 * (q * term).sum(1)
    e_loss = temp ** 2 * (e.sum(1) + (top.shape[1] + 8) * E * (q * term.abs()).sum(1)) + 4 * E * loss.abs()
    loss = torch.where(counted, loss, torch.zeros_like(loss))
    loss = torch.where(bad, torch.full_like(loss, math.nan), loss)
    zt = torch.where(top < 0, torch.zeros_like(zt), torch.where(top >= V, torch.full_like(zt, math.nan), zt))
    return (loss, e_loss), (lse, e_lse), (zt, ezt)


def distill_grad(x, w, top, t, temp, lse, dloss, dt, beta=0.0, dw0=None):
    """dx and dw with their errors before the results' rounding.  D is rounded to dt, over the largest |dloss| (fp16:
    times 2^13)."""
    V = w.shape[0]
    z = x @ w.t()
    q, log_q, counted, _ = teacher(top, t, temp, V)
    q = torch.where(counted[:, None] & (top >= 0), q, torch.zeros_like(q))
    lq = torch.where(q > 0, log_q.abs(), torch.zeros_like(q))
    eq = q * (STEP * (4 + lq + (t / temp).nan_to_num(0, 0, 0).abs()) + (32 + top.shape[1]) * E)
    at = top.clamp(0, V - 1)
    p = torch.exp(z / temp - lse[:, None])
    d = p.scatter_add(1, at, -q)
    ed = p * (dot_bound(x, w.t()) / temp + STEP * (1 + (z / temp).abs() + lse.abs()[:, None])) + 4 * E * p
    ed = ed.scatter_add(1, at, eq)
    k = torch.where(counted, temp * dloss, torch.zeros_like(dloss))[:, None]
    d, ed = k * d, k.abs() * (ed + 4 * E * d.abs())
    ed = ed + U[dt] * (d.abs() + ed) + (2.0 ** -25 * 2.0 ** -13 * float(k.abs().max()) if dt == "f16" else 0.0)
    old = torch.zeros_like(w) if dw0 is None else dw0
    return ((d @ w, ed @ w.abs() + dot_bound(d.abs() + ed, w)),
            (d.t() @ x + beta * old,
             ed.t() @ x.abs() + dot_bound((d.abs() + ed).t(), x) + 4 * E * (beta * old).abs()))


def policy(logp, old, ref, adv, mask, low, high, kl, reduce):
    """stats and norm; adv of one column is a sequence's.  low, high, kl: as fp32 holds them."""
    loss, kl_term, taken, ratio = policy_terms(logp, old, ref, adv, low, high, kl)
    n = mask.double().sum(1)
    some = n > 0
    one = torch.ones_like(n)
    each = {"tokens": one / max(1.0, float(n.sum())),
            "sequences": 1 / torch.where(some, n, one) / max(1, int(some.sum())), "sum": one}[reduce]
    norm = torch.where(some, each, torch.zeros_like(n))

    def total(a):
        a = torch.where(mask, a, torch.zeros_like(a))
        return (a.sum(1) * norm).sum(), (a.abs().sum(1) * norm).sum()
    sums = [total(a) for a in (loss, kl_term, taken.double(), ratio)]
    return torch.stack([s for s, _ in sums]), torch.stack([s for _, s in sums]), norm


def policy_terms(logp, old, ref, adv, low, high, kl):
    ratio = torch.exp(logp - old)
    bounded = ratio.clamp(1 - low, 1 + high)
    d = torch.zeros_like(logp) if ref is None else ref - logp
    # exp(d) - d - 1 has no cancellation left in float64 where d is an fp32 difference of at least 2^-20
    term = torch.where(d.abs() < 1e-3, d * d * (0.5 + d / 6 + d * d / 24 + d ** 3 / 120), torch.exp(d) - d - 1)
    return kl * term - torch.minimum(ratio * adv, bounded * adv), term, ratio * adv > bounded * adv, ratio


def policy_grad(logp, old, ref, adv, mask, low, high, kl, norm, dloss):
    """dlogp and the sum of its terms' magnitudes."""
    ratio = torch.exp(logp - old)
    bounded = ratio.clamp(1 - low, 1 + high)
    a = torch.where(ratio * adv > bounded * adv, torch.zeros_like(ratio), -adv * ratio)
    b = torch.zeros_like(logp) if ref is None else -kl * torch.expm1(ref - logp)
    w = torch.where(mask, (dloss * norm)[:, None], torch.zeros_like(logp))
    zero = torch.zeros_like(logp)
    return torch.where(mask, w * (a + b), zero), torch.where(mask, (w * (a.abs() + b.abs())).abs(), zero)


def f32(v):
    """v as an fp32 argument holds it."""
    return float(torch.tensor(v, dtype=torch.float32))
