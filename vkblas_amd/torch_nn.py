"""PyTorch functions of the operators in include/vkblas_nn.h, with their gradients.

    layer_norm(x, weight=None, bias=None, eps=1e-5)
    gated_linear(x, weight, activation="silu")                 act(x Wg^T) * (x Wu^T)
    linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean")

Each checks its arguments (ValueError), runs the library's kernels on the current stream of the tensors' device
and takes part in autograd (once: a gradient of a gradient raises).  There is no fallback: a call the library refuses raises VkblasError.

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
