"""What vkblas_amd.torch_nn returns is an ordinary tensor: a program may change it in place before the backward pass,
as it may the results of torch.nn.functional's own functions.  On the CPU with the library's calls stubbed (autograd's
checks do not depend on values), and on the GPU with values."""
import contextlib

import pytest
import torch

import nn_ref as R
import vkblas_amd as vk

NN_CALLS = [f"{name}_async" for name in vk._NN_ARGS]


@pytest.fixture
def vnn(monkeypatch):
    """torch_nn on the CPU, its launches stubbed."""
    from vkblas_amd import torch_nn
    for name in NN_CALLS:
        monkeypatch.setattr(vk, name, lambda *a, **k: vk.OK)
    monkeypatch.setattr(torch_nn, "_check", lambda *a: None)
    monkeypatch.setattr(torch_nn, "_stream", lambda t: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    return torch_nn


CALLS = {
    "layer_norm": lambda m, x, w, t: m.layer_norm(x, w[0]),
    "gated_linear": lambda m, x, w, t: m.gated_linear(x, w),
    "none": lambda m, x, w, t: m.linear_cross_entropy(x, w, t, reduction="none"),
    "sum": lambda m, x, w, t: m.linear_cross_entropy(x, w, t, reduction="sum"),
    "mean": lambda m, x, w, t: m.linear_cross_entropy(x, w, t),
}
IN_PLACE = {"mul": lambda y: y.mul_(2.0), "add": lambda y: y.add_(torch.ones_like(y)),
            "dropout": lambda y: torch.nn.functional.dropout(y, 0.5, inplace=True)}


@pytest.mark.parametrize("shape", [(8,), (5, 8), (2, 3, 8), (0, 8)], ids=str)
@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("change", IN_PLACE)
def test_results_may_be_changed_in_place(vnn, shape, call, change):
    x, w = torch.zeros(shape, requires_grad=True), torch.zeros(6, 8, requires_grad=True)
    t = torch.zeros(shape[:-1], dtype=torch.int64)
    y = CALLS[call](vnn, x, w, t)
    assert y.shape == {"layer_norm": shape, "gated_linear": shape[:-1] + (3,), "none": shape[:-1]}.get(call, ())
    IN_PLACE[change](y).sum().backward()
    assert x.grad.shape == x.shape and w.grad.shape == w.shape


@pytest.mark.parametrize("call", ["layer_norm", "gated_linear", "none"])
def test_results_own_their_memory(vnn, call):
    """No result is a part of a larger tensor, whose rest it would keep alive and share a version with."""
    x, w = torch.zeros(2, 3, 8, requires_grad=True), torch.zeros(6, 8, requires_grad=True)
    y = CALLS[call](vnn, x, w, torch.zeros(2, 3, dtype=torch.int64))
    assert y._base is None and y.untyped_storage().nbytes() == y.numel() * y.element_size()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_values_of_results_changed_in_place(dt):
    """A residual added, rows masked and losses weighted in place, against PyTorch's own functions in float64."""
    from vkblas_amd import torch_nn as real
    f = torch.nn.functional
    g = torch.Generator().manual_seed(1)
    x0 = torch.randn(2, 20, 64, generator=g).to(R.TORCH[dt])
    w0 = (torch.randn(64, 64, generator=g) * 0.1).to(R.TORCH[dt])
    r0 = torch.randn(2, 20, 64, generator=g).to(R.TORCH[dt])
    mask, t = torch.rand(2, 20, generator=g) < 0.5, torch.randint(0, 64, (2, 20), generator=g)

    def own(x, w, r, mask, t):
        y = real.layer_norm(x)
        y += r
        h = real.gated_linear(y, w)
        h.mul_(mask[..., None])
        loss = real.linear_cross_entropy(torch.cat((h, h), -1), w, t, reduction="none")
        loss *= mask
        return loss.sum()

    def ref(x, w, r, mask, t):
        y = f.layer_norm(x, (64,)) + r
        a, b = f.linear(y, w).chunk(2, -1)
        h = f.silu(a) * b * mask[..., None]
        z = f.linear(torch.cat((h, h), -1), w)
        return (f.cross_entropy(z.flatten(0, 1), t.flatten(), reduction="none").view(t.shape) * mask).sum()

    out = []
    for fn, move in ((own, lambda v: v.cuda()), (ref, lambda v: v.double())):
        x, w = move(x0).requires_grad_(), move(w0).requires_grad_()
        loss = fn(x, w, move(r0), mask.cuda() if fn is own else mask, t.cuda() if fn is own else t)
        loss.backward()
        out.append([v.detach().double().cpu() for v in (loss, x.grad, w.grad)])
    # a chain of a few roundings to dt of values of the results' own size
    for a, b in zip(*out):
        assert float((a - b).abs().max()) <= max(16 * R.U[dt], 1e-5) * float(b.abs().max())
