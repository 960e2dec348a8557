"""PyTorch functions of the operators in include/vkblas_nn.h and include/vkblas_train.h, with their gradients.

    embedding(ids, weight, scale=1.0, padding_idx=None, dtype=None)
    layer_norm(x, weight=None, bias=None, eps=1e-5)
    gated_linear(x, weight, activation="silu")                 act(x Wg^T) * (x Wu^T)
    linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean")
    linear_distillation(x, weight, classes, teacher_logits, temperature=1.0, reduction="mean")
    policy_loss(logp, old_logp, advantages, ref_logp=None, mask=None, clip=(0.2, 0.2), kl_coef=0.0,
                reduction="tokens")                            loss and its statistics

Each checks its arguments (ValueError), runs the library's kernels on the current stream of the tensors' device
and takes part in autograd (once: a gradient of a gradient raises).  There is no fallback: a call the library refuses
raises VkblasError.

Tensors are fp32, fp16 or bf16 on one GPU; leading dimensions of x are its rows.  Rows may be strided (a slice of
a wider matrix) as long as their elements are adjacent; others are copied.  A weight's gradient has the weight's
type.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

import vkblas_amd as vk

_TYPES = {torch.float32: vk.DT_F32, torch.float16: vk.DT_F16, torch.bfloat16: vk.DT_BF16}
ACTIVATIONS = {"silu": vk.ACT_SILU, "gelu": vk.ACT_GELU, "gelu_tanh": vk.ACT_GELU_TANH, "relu": vk.ACT_RELU}


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as a matrix of its last dimension whose rows' elements are adjacent, and whose rows are no farther apart than
    a leading dimension holds."""
    m = t.reshape(-1, t.shape[-1])
    return m if m.stride(1) == 1 and m.shape[1] <= m.stride(0) < 2 ** 31 else m.contiguous()


def _ld(m: torch.Tensor) -> int:
    return max(m.stride(0), m.shape[1]) if m.shape[0] > 1 else m.shape[1]


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _check(name, x, weight, dims, same_type):
    if x.dim() < 1 or x.dtype not in _TYPES or not x.is_cuda:
        raise ValueError(f"{name}: x must be an fp32, fp16 or bf16 tensor on a GPU")
    if not x.shape[-1]:
        raise ValueError(f"{name}: x's rows are empty: {tuple(x.shape)}")
    if weight is not None:
        if weight.dim() != dims or weight.shape[-1] != x.shape[-1] or weight.device != x.device:
            raise ValueError(f"{name}: a weight of {dims} dimension(s), the last {x.shape[-1]}, on x's device; "
                             f"not {tuple(weight.shape)} on {weight.device}")
        if weight.dtype != x.dtype and (same_type or weight.dtype != torch.float32):
            raise ValueError(f"{name}: weight of {weight.dtype} with x of {x.dtype}")


# Results are allocated in the shape they are returned in: a view that a Function returns cannot be changed in place.


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        m = _rows(x)
        y = torch.empty(x.shape, dtype=m.dtype, device=m.device)
        mean, rstd = torch.empty(2, m.shape[0], dtype=torch.float32, device=m.device)
        ref = weight if weight is not None else bias
        ctx.w_type = _TYPES[ref.dtype] if ref is not None else _TYPES[m.dtype]
        with torch.cuda.device(m.device):
            vk.layer_norm_async(_TYPES[m.dtype], ctx.w_type, *m.shape, _ptr(m), _ld(m), _ptr(weight), _ptr(bias), eps,
                                _ptr(y), m.shape[1], _ptr(mean), _ptr(rstd), stream=_stream(m))
        ctx.save_for_backward(m, weight, bias, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        m, weight, bias, mean, rstd = ctx.saved_tensors
        d = _rows(dy)
        dx = torch.empty(m.shape, dtype=m.dtype, device=m.device) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        db = torch.empty_like(bias) if ctx.needs_input_grad[2] else None
        with torch.cuda.device(m.device):
            vk.layer_norm_backward_async(_TYPES[m.dtype], ctx.w_type, *m.shape, _ptr(d), _ld(d), _ptr(m), _ld(m),
                                         _ptr(weight), _ptr(mean), _ptr(rstd), _ptr(dx), m.shape[1], _ptr(dw), _ptr(db),
                                         ctx.w_type, 0.0, stream=_stream(m))
        return dx.view(dy.shape) if dx is not None else None, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of x's last dimension; weight and bias of x's type or fp32 (both of one type)."""
    _check("layer_norm", x, weight, 1, False)
    _check("layer_norm", x, bias, 1, False)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"layer_norm: weight of {weight.dtype} with bias of {bias.dtype}")
    w, b = (None if t is None else t.contiguous() for t in (weight, bias))
    return _LayerNorm.apply(x, w, b, float(eps))


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, act, keep):
        m, w = _rows(x), _rows(weight)
        N = w.shape[0] // 2
        h = torch.empty(*x.shape[:-1], N, dtype=m.dtype, device=m.device)
        gu = torch.empty(m.shape[0], 2 * N, dtype=m.dtype, device=m.device) if keep else None
        with torch.cuda.device(m.device):
            vk.glu_async(_TYPES[m.dtype], act, m.shape[0], N, m.shape[1], _ptr(m), _ld(m), _ptr(w), _ld(w), _ptr(h), N,
                         _ptr(gu), 2 * N, stream=_stream(m))
        ctx.act = act
        ctx.save_for_backward(m, w, gu)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        m, w, gu = ctx.saved_tensors
        d, N = _rows(dh), w.shape[0] // 2
        dx = torch.empty(m.shape, dtype=m.dtype, device=m.device) if ctx.needs_input_grad[0] else None
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if ctx.needs_input_grad[1] else None
        with torch.cuda.device(m.device):
            vk.glu_backward_async(_TYPES[m.dtype], ctx.act, m.shape[0], N, m.shape[1], _ptr(d), _ld(d), _ptr(gu), 2 * N,
                                  _ptr(m), _ld(m), _ptr(w), _ld(w), None, 0, _ptr(dx), m.shape[1], _ptr(dw), m.shape[1],
                                  _TYPES[w.dtype], 0.0, stream=_stream(m))
        return dx.view(*dh.shape[:-1], m.shape[1]) if dx is not None else None, dw, None, None


def gated_linear(x, weight, activation="silu"):
    """act(x Wg^T) * (x Wu^T); weight holds Wg's rows, then Wu's, and has x's type."""
    _check("gated_linear", x, weight, 2, True)
    if weight.shape[0] % 2 or not weight.shape[0]:
        raise ValueError("gated_linear: the weight's rows are the gate's and as many of the up projection")
    if activation not in ACTIVATIONS:
        raise ValueError(f"gated_linear: activation {activation!r}, not one of {sorted(ACTIVATIONS)}")
    # both projections are kept only for a backward pass; inside a Function grad mode is off and a parameter
    # asks for its gradient under no_grad too
    keep = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)
    return _GatedLinear.apply(x, weight, ACTIVATIONS[activation], keep)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index):
        m, w = _rows(x), _rows(weight)
        t = target.reshape(-1).contiguous()
        # two tensors: loss is the program's to change, lse the backward pass's
        loss = torch.empty(target.shape, dtype=torch.float32, device=m.device)
        lse = torch.empty(m.shape[0], dtype=torch.float32, device=m.device)
        with torch.cuda.device(m.device):
            vk.linear_xent_async(_TYPES[m.dtype], m.shape[0], w.shape[0], m.shape[1], _ptr(m), _ld(m), _ptr(w), _ld(w),
                                 _ptr(t), ignore_index, _ptr(loss), _ptr(lse), stream=_stream(m))
        ctx.ignore_index, ctx.x_shape = ignore_index, x.shape
        ctx.save_for_backward(m, w, t, lse)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        m, w, t, lse = ctx.saved_tensors
        d = dloss.contiguous()
        dx = torch.empty(m.shape, dtype=m.dtype, device=m.device) if ctx.needs_input_grad[0] else None
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if ctx.needs_input_grad[1] else None
        with torch.cuda.device(m.device):
            vk.linear_xent_backward_async(_TYPES[m.dtype], m.shape[0], w.shape[0], m.shape[1], _ptr(m), _ld(m), _ptr(w),
                                          _ld(w), _ptr(t), ctx.ignore_index, _ptr(lse), _ptr(d), _ptr(dx), m.shape[1],
                                          _ptr(dw), m.shape[1], _TYPES[w.dtype], 0.0, stream=_stream(m))
        return dx.view(ctx.x_shape) if dx is not None else None, dw, None, None


def linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean"):
    """Cross entropy of the logits x W^T, which are not kept; target: int64, x's leading dimensions.  reduction:
    "mean" over the targets that are not ignore_index, "sum" or "none" (fp32 in all)."""
    _check("linear_cross_entropy", x, weight, 2, True)
    if target.dtype != torch.int64 or target.shape != x.shape[:-1] or target.device != x.device:
        raise ValueError(f"linear_cross_entropy: an int64 target of shape {tuple(x.shape[:-1])} on x's device")
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"linear_cross_entropy: reduction {reduction!r}")
    loss = _LinearCrossEntropy.apply(x, weight, target, int(ignore_index))
    if reduction == "none":
        return loss
    total = loss.sum()
    return total if reduction == "sum" else total / (target != ignore_index).sum()


NO_ID = -2 ** 63    # a padding_idx that no token has


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, pad, dtype):
        w, i = _rows(weight), ids.reshape(-1).contiguous()
        y = torch.empty(*ids.shape, w.shape[1], dtype=dtype, device=w.device)
        with torch.cuda.device(w.device):
            vk.embedding_async(_TYPES[dtype], _TYPES[w.dtype], i.shape[0], *w.shape, _ptr(i), pad, _ptr(w), _ld(w),
                               scale, _ptr(y), w.shape[1], stream=_stream(w))
        ctx.scale, ctx.pad, ctx.w_shape, ctx.w_type = scale, pad, w.shape, w.dtype
        ctx.save_for_backward(i)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        i, = ctx.saved_tensors
        d = _rows(dy)
        dw = torch.empty(ctx.w_shape, dtype=ctx.w_type, device=dy.device)
        with torch.cuda.device(dy.device):
            vk.embedding_backward_async(_TYPES[d.dtype], i.shape[0], *ctx.w_shape, _ptr(i), ctx.pad, _ptr(d), _ld(d),
                                        ctx.scale, _ptr(dw), ctx.w_shape[1], _TYPES[ctx.w_type], 0.0, stream=_stream(d))
        return dw, None, None, None, None


def embedding(ids, weight, scale=1.0, padding_idx=None, dtype=None):
    """scale * weight[ids]: int64 ids of any shape; rows of zeros without a gradient where ids are padding_idx, of NaN
    where they are outside the vocabulary.  dtype: the result's, the weight's own or, of an fp32 weight, another."""
    _check("embedding", weight, None, 2, True)
    if weight.dim() != 2 or not weight.shape[0]:
        raise ValueError(f"embedding: a weight of vocabulary x width, not {tuple(weight.shape)}")
    if ids.dtype != torch.int64 or ids.device != weight.device:
        raise ValueError(f"embedding: int64 ids on the weight's device, not {ids.dtype} on {ids.device}")
    dtype = weight.dtype if dtype is None else dtype
    if dtype not in _TYPES or (weight.dtype != dtype and weight.dtype != torch.float32):
        raise ValueError(f"embedding: weight of {weight.dtype} with a result of {dtype}")
    return _Embedding.apply(weight, ids, float(scale), NO_ID if padding_idx is None else int(padding_idx), dtype)


class _LinearDistillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, classes, teacher, temperature):
        m, w, c, t = _rows(x), _rows(weight), _rows(classes), _rows(teacher)
        n = c.shape[1]
        loss = torch.empty(x.shape[:-1], dtype=torch.float32, device=m.device)
        lse = torch.empty(m.shape[0], dtype=torch.float32, device=m.device)
        z_top = torch.empty(m.shape[0], n, dtype=torch.float32, device=m.device)
        with torch.cuda.device(m.device):
            vk.linear_distill_async(_TYPES[m.dtype], m.shape[0], w.shape[0], m.shape[1], _ptr(m), _ld(m), _ptr(w),
                                    _ld(w), n, _ptr(c), _ld(c), _TYPES[t.dtype], _ptr(t), _ld(t), temperature,
                                    _ptr(loss), _ptr(lse), _ptr(z_top), stream=_stream(m))
        ctx.temperature, ctx.x_shape = temperature, x.shape
        ctx.save_for_backward(m, w, c, t, lse, z_top)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        m, w, c, t, lse, z_top = ctx.saved_tensors
        d = dloss.contiguous()
        dx = torch.empty(m.shape, dtype=m.dtype, device=m.device) if ctx.needs_input_grad[0] else None
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if ctx.needs_input_grad[1] else None
        with torch.cuda.device(m.device):
            vk.linear_distill_backward_async(_TYPES[m.dtype], m.shape[0], w.shape[0], m.shape[1], _ptr(m), _ld(m),
                                             _ptr(w), _ld(w), c.shape[1], _ptr(c), _ld(c), _TYPES[t.dtype], _ptr(t),
                                             _ld(t), ctx.temperature, _ptr(lse), _ptr(z_top), _ptr(d), _ptr(dx),
                                             m.shape[1], _ptr(dw), m.shape[1], _TYPES[w.dtype], 0.0, stream=_stream(m))
        return dx.view(ctx.x_shape) if dx is not None else None, dw, None, None, None


def linear_distillation(x, weight, classes, teacher_logits, temperature=1.0, reduction="mean"):
    """temperature^2 times the divergence of softmax(x W^T / temperature) from the teacher's, which is the softmax of
    its logits at some classes of each row (x's leading dimensions, then the entries; int64, negative: no entry).
    reduction: "mean" over the rows with a teacher, "sum" or "none" (fp32 in all)."""
    _check("linear_distillation", x, weight, 2, True)
    if classes.dtype != torch.int64 or classes.device != x.device or classes.shape[:-1] != x.shape[:-1]:
        raise ValueError(f"linear_distillation: int64 classes of shape {tuple(x.shape[:-1])} x entries on x's device")
    if not 0 < classes.shape[-1] <= vk.DISTILL_TOP:
        raise ValueError(f"linear_distillation: 1 to {vk.DISTILL_TOP} entries, not {classes.shape[-1]}")
    if (teacher_logits.shape != classes.shape or teacher_logits.device != x.device
            or teacher_logits.dtype not in (x.dtype, torch.float32)):
        raise ValueError("linear_distillation: the teacher's logits at the classes, in x's type or fp32")
    if teacher_logits.requires_grad:
        raise ValueError("linear_distillation: the teacher's logits get no gradient; detach them")
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"linear_distillation: reduction {reduction!r}")
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"linear_distillation: temperature {temperature}")
    loss = _LinearDistillation.apply(x, weight, classes, teacher_logits, float(temperature))
    if reduction == "none":
        return loss
    total = loss.sum()
    if reduction == "sum":
        return total
    return total / ((classes >= 0) & (teacher_logits != -float("inf"))).any(-1).sum()


REDUCTIONS = {"tokens": vk.REDUCE_TOKENS, "sequences": vk.REDUCE_SEQUENCES, "sum": vk.REDUCE_SUM}


def _policy_args(logp, old, ref, adv, mask, clip, kl_coef):
    """The arguments that the policy loss and its gradient share, from matrices of a row for each sequence."""
    B, T = logp.shape
    return (B, T, _ptr(logp), _ld(logp), _ptr(old), _ld(old), _ptr(ref), _ld(ref) if ref is not None else 0, _ptr(adv),
            _ld(adv), int(adv.shape[1] == T), _ptr(mask), _ld(mask) if mask is not None else 0, *clip, kl_coef)


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logp, old, ref, adv, mask, clip, kl_coef, reduce):
        rows = [None if t is None else _rows(t) for t in (logp, old, ref, adv, mask)]
        p = rows[0]
        stats, norm = (torch.empty(n, dtype=torch.float32, device=p.device) for n in (4, p.shape[0]))
        if not p.shape[0]:
            stats.zero_()
        with torch.cuda.device(p.device):
            vk.policy_loss_async(reduce, *_policy_args(*rows, clip, kl_coef), _ptr(stats), _ptr(norm),
                                 stream=_stream(p))
        ctx.clip, ctx.kl_coef, ctx.shape = clip, kl_coef, logp.shape
        ctx.save_for_backward(*rows, norm)
        loss = torch.empty((), dtype=torch.float32, device=p.device)
        loss.copy_(stats[0])
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        *rows, norm = ctx.saved_tensors
        dlogp = torch.empty(ctx.shape, dtype=torch.float32, device=norm.device)
        with torch.cuda.device(norm.device):
            vk.policy_loss_backward_async(*_policy_args(*rows, ctx.clip, ctx.kl_coef), _ptr(norm), _ptr(dloss),
                                          _ptr(dlogp), ctx.shape[-1], stream=_stream(norm))
        return dlogp, None, None, None, None, None, None, None


def policy_loss(logp, old_logp, advantages, ref_logp=None, mask=None, clip=(0.2, 0.2), kl_coef=0.0, reduction="tokens"):
    """Clipped policy loss of token log probabilities (fp32, sequences x tokens; linear_cross_entropy's losses with
    reduction "none" are their negatives), plus kl_coef times the KL term against ref_logp: the loss, and a tensor of
    it, the KL term, the share of the tokens held by a bound and the ratio, without gradients.

    advantages: one for each token or for each sequence.  mask (bool or uint8): the tokens that count, all without one.
    clip: the ratio is held within [1 - clip[0], 1 + clip[1]].  reduction: the mean over the "tokens", over the
    "sequences" of their tokens' means, or the "sum"."""
    if logp.dim() < 1 or logp.dtype != torch.float32 or not logp.is_cuda or not logp.shape[-1]:
        raise ValueError("policy_loss: logp must be an fp32 tensor of sequences x tokens on a GPU")
    if advantages.shape == logp.shape[:-1]:
        advantages = advantages.unsqueeze(-1)
    for name, t, shapes in (("old_logp", old_logp, (logp.shape,)), ("ref_logp", ref_logp, (logp.shape,)),
                            ("advantages", advantages, (logp.shape, (*logp.shape[:-1], 1)))):
        if t is None and name == "ref_logp":
            continue
        if t.dtype != torch.float32 or t.device != logp.device or t.shape not in shapes:
            raise ValueError(f"policy_loss: {name} in fp32 on logp's device and of its shape, not {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
        if t.requires_grad:
            raise ValueError(f"policy_loss: {name} gets no gradient; detach it")
    if mask is not None:
        if mask.shape != logp.shape or mask.dtype not in (torch.bool, torch.uint8) or mask.device != logp.device:
            raise ValueError(f"policy_loss: a bool or uint8 mask of shape {tuple(logp.shape)} on logp's device")
        mask = mask.view(torch.uint8)
    if reduction not in REDUCTIONS:
        raise ValueError(f"policy_loss: reduction {reduction!r}, not one of {sorted(REDUCTIONS)}")
    low, high = float(clip[0]), float(clip[1])
    if not (low >= 0.0 and high >= 0.0):
        raise ValueError(f"policy_loss: clip {clip!r}")
    return _PolicyLoss.apply(logp, old_logp, ref_logp, advantages, mask, (low, high), float(kl_coef),
                             REDUCTIONS[reduction])
