"""Definitions in float64 (torch, on the CPU) of the operators in vkblas_nn.h, with bounds on
how far a correct fp32 evaluation may be from them, and device buffers for their tests.

Bounds.  u = unit roundoff of the result's type, e = 2^-24 that of fp32.  A dot product of K
terms summed in fp32 in any order is within K e sum |a_k b_k| of exact; DOT allows 8 more roundings.
Elementwise steps of a few fp32 operations and hardware exponentials (1 unit, argument rounding
|x| e) are within STEP = 16 e relative, plus their argument's error times the function's slope.
An operand rounded to the type before a product adds u |operand| to its error.  A rounding to
fp16 adds at most 2^-25 below the normal range.
"""
import torch

import vkblas_amd as vk

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ENGINE = {"f32": vk.DT_F32, "f16": vk.DT_F16, "bf16": vk.DT_BF16}
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}
E = 2.0 ** -24
STEP = 16 * E
ACTS = {"silu": vk.ACT_SILU, "gelu": vk.ACT_GELU, "gelu_tanh": vk.ACT_GELU_TANH, "relu": vk.ACT_RELU}


def dot_bound(a, b):
    """Error bound of fp32 a @ b."""
    return (a.shape[1] + 8) * E * (a.abs() @ b.abs())


def rounded(x, dt, err=0.0):
    """Bound on a result x rounded to dt, whose value before the rounding has error err."""
    return err + U[dt] * (x.abs() + err) + TINY[dt]


class Buf:
    """rows x cols of dt on the GPU with a leading dimension of cols + pad, `off` elements past a 256-byte
    boundary, NaN around it."""

    def __init__(self, rows, cols, dt, pad=0, off=0, values=None):
        self.rows, self.cols, self.ld, self.off = rows, cols, cols + pad, off
        self.all = torch.full((rows * self.ld + off + 64,), float("nan"), dtype=TORCH[dt], device="cuda")
        self.t = self.all[off:off + rows * self.ld].view(rows, self.ld)[:, :cols]
        if values is not None:
            self.t.copy_(values.to(TORCH[dt]))

    @property
    def ptr(self):
        return self.all.data_ptr() + self.off * self.all.element_size()

    def get(self, device="cpu"):
        torch.cuda.synchronize()
        return self.t.double().to(device)

    def check_around(self):
        """Nothing was written outside the matrix."""
        torch.cuda.synchronize()
        inside = torch.zeros(self.all.numel(), dtype=torch.bool, device="cuda")
        inside[self.off:self.off + self.rows * self.ld].view(self.rows, self.ld)[:, :self.cols] = True
        assert bool(torch.isnan(self.all[~inside]).all()), "written outside the matrix"


def values(rows, cols, dt, seed, scale=1.0):
    """Random values of dt, as float64."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, cols, generator=g, dtype=torch.float64) * scale).to(TORCH[dt]).double()


def close(got, ref, bound, what):
    got = got.to(ref.device)
    bad = ~((got - ref).abs() <= bound)
    if bool(bad.any()):
        i = int(torch.argmax(((got - ref).abs() / (bound + 1e-300)).nan_to_num(nan=float("inf")).flatten()))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, worst at {i}: "
                             f"{got.flatten()[i]} for {ref.flatten()[i]}, bound {bound.expand_as(ref).flatten()[i]}")


def act(name, g):
    f = torch.nn.functional
    return {"silu": f.silu, "gelu": f.gelu, "gelu_tanh": lambda t: f.gelu(t, approximate="tanh"),
            "relu": f.relu}[name](g)


def act_slope(name, g):
    g = g.clone().requires_grad_()
    return torch.autograd.grad(act(name, g).sum(), g)[0]


def norm(x, w, b, eps):
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    return (x - mean) * rstd * w + b, mean[:, 0], rstd[:, 0]


def norm_grad(dy, x, w, mean, rstd):
    xh = (x - mean[:, None]) * rstd[:, None]
    g = dy * w
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def xent(x, w, target, ignore):
    z = x @ w.t()
    lse = torch.logsumexp(z, 1)
    loss = lse - z.gather(1, target.clamp(0, w.shape[0] - 1)[:, None])[:, 0]
    loss = torch.where((target < 0) | (target >= w.shape[0]), torch.full_like(loss, float("nan")), loss)
    return z, torch.where(target == ignore, torch.zeros_like(loss), loss), lse
