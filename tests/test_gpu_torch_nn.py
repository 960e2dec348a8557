"""vkblas_amd.torch_nn: the operators as PyTorch functions against PyTorch's own on the CPU in float64, through
autograd, on strided and many-dimensional inputs; their refusals; and the training example, which runs them together."""
import os
import sys

import pytest
import torch

import nn_ref as R

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def both(fn, ref, dt, *args):
    """fn on the GPU in dt and ref on the CPU in float64 of the same values: results and gradients."""
    out = []
    for f, move in ((fn, lambda t: t.cuda()), (ref, lambda t: t.double())):
        a = [move(t).requires_grad_() if t.is_floating_point() else t.cuda() if f is fn else t for t in args]
        y = f(*a)
        g = torch.randn(y.shape, generator=torch.Generator().manual_seed(5), dtype=torch.float64).to(R.TORCH[dt])
        y.backward(g.to(y.device, y.dtype))
        out.append([y.detach().double().cpu()] + [t.grad.double().cpu() for t in a if t.requires_grad])
    return out


def near(got, ref, dt, times=8):
    # chains of a few roundings to dt of values of the result's own size: 8 units of the largest
    for a, b in zip(got, ref):
        assert a.shape == b.shape
        tol = max(times * R.U[dt], 1e-5) * float(b.abs().max())
        assert float((a - b).abs().max()) <= tol


def values(*shape, dt, seed, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(R.TORCH[dt])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_layer_norm(dt):
    from vkblas_amd import torch_nn as vnn
    x, w, b = values(2, 3, 7, 200, dt=dt, seed=1), values(200, dt=dt, seed=2), values(200, dt=dt, seed=3)
    near(*both(vnn.layer_norm, lambda x, w, b: torch.nn.functional.layer_norm(x, (200,), w, b), dt, x, w, b), dt)
    near(*both(vnn.layer_norm, lambda x: torch.nn.functional.layer_norm(x, (200,)), dt, x), dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 64), (2, 70, 128)])
def test_gated_linear(dt, shape):
    from vkblas_amd import torch_nn as vnn
    x, w = values(*shape, dt=dt, seed=1), values(2 * 96, shape[-1], dt=dt, seed=2, scale=0.1)

    def ref(x, w):
        g, u = torch.nn.functional.linear(x, w).chunk(2, -1)
        return torch.nn.functional.gelu(g) * u
    near(*both(lambda x, w: vnn.gated_linear(x, w, "gelu"), ref, dt, x, w), dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_linear_cross_entropy(dt, reduction):
    from vkblas_amd import torch_nn as vnn
    x, w = values(3, 40, 128, dt=dt, seed=1), values(333, 128, dt=dt, seed=2, scale=0.2)
    t = torch.randint(0, 333, (3, 40), generator=torch.Generator().manual_seed(3))
    t[0, :7] = -100

    def ref(x, w, t):
        z = torch.nn.functional.linear(x, w)
        return torch.nn.functional.cross_entropy(z.view(-1, 333), t.view(-1), reduction=reduction).view(
            (3, 40) if reduction == "none" else ())
    near(*both(lambda x, w, t: vnn.linear_cross_entropy(x, w, t, reduction=reduction), ref, dt, x, w, t), dt)


@pytest.mark.gpu
def test_strided_inputs_and_no_gradients():
    from vkblas_amd import torch_nn as vnn
    wide = values(50, 300, dt="f32", seed=1).cuda()
    for x in (wide[:, 20:148], wide[::2, :128], wide.t()[:128].t(), wide[:1, :128].expand(50, 128)):
        w = values(64, 128, dt="f32", seed=2).cuda()
        g, u = (x @ w.t()).chunk(2, 1)
        with torch.no_grad():
            y = vnn.gated_linear(x, w)
        assert torch.allclose(y, torch.nn.functional.silu(g) * u, rtol=1e-4, atol=1e-4)
        assert torch.allclose(vnn.layer_norm(x), torch.nn.functional.layer_norm(x, (128,)), rtol=1e-4, atol=1e-4)
    assert vnn.layer_norm(wide[:0]).shape == (0, 300)


@pytest.mark.gpu
def test_projections_are_kept_for_a_backward_pass_only(monkeypatch):
    import vkblas_amd as vk
    from vkblas_amd import torch_nn as vnn
    x, w = values(50, 128, dt="bf16", seed=1).cuda(), values(64, 128, dt="bf16", seed=2).cuda()
    kept, call = [], vk.glu_async
    monkeypatch.setattr(vk, "glu_async", lambda *a, **k: (kept.append(a[11]), call(*a, **k))[1])
    vnn.gated_linear(x, w)
    w.requires_grad_()
    with torch.no_grad():
        vnn.gated_linear(x, w)
    with torch.inference_mode():
        vnn.gated_linear(x, w)
    assert kept == [None] * 3
    assert vnn.gated_linear(x, w).requires_grad and kept[-1]


@pytest.mark.gpu
def test_empty_rows_are_refused():
    from vkblas_amd import torch_nn as vnn
    x, w = torch.zeros(4, 0, device="cuda"), torch.zeros(6, 0, device="cuda")
    for call in (lambda: vnn.layer_norm(x), lambda: vnn.gated_linear(x, w),
                 lambda: vnn.linear_cross_entropy(x, w, torch.zeros(4, dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError, match="empty"):
            call()


@pytest.mark.gpu
def test_example_learns():
    sys.path.insert(0, os.path.join(REPO, "examples"))
    import train_step
    losses = train_step.train(steps=25, tokens=1024, width=256, hidden=300, layers=2, classes=1003, lr=3e-3,
                              log=lambda *a, **k: None)
    # from about log(1003) = 6.9 plus the initial logits' spread
    assert losses[0] > 5.0 and losses[-1] < 0.6 * losses[0]


def test_refusals():
    from vkblas_amd import torch_nn as vnn
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="on a GPU"):
        vnn.layer_norm(x)
    with pytest.raises(ValueError, match="on a GPU"):
        vnn.gated_linear(x, torch.zeros(4, 8))


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    from vkblas_amd import torch_nn as vnn
    x = torch.zeros(4, 8, device="cuda")
    bad = [lambda: vnn.layer_norm(x, torch.ones(7, device="cuda")), lambda: vnn.layer_norm(x, torch.ones(8)),
           lambda: vnn.layer_norm(x.double()), lambda: vnn.layer_norm(x, torch.ones(8, device="cuda").half()),
           lambda: vnn.gated_linear(x, torch.zeros(3, 8, device="cuda")),
           lambda: vnn.gated_linear(x, torch.zeros(4, 8, device="cuda"), "tanh"),
           lambda: vnn.gated_linear(x, torch.zeros(4, 8, device="cuda").half()),
           lambda: vnn.linear_cross_entropy(x, torch.zeros(5, 8, device="cuda"), torch.zeros(4, device="cuda")),
           lambda: vnn.linear_cross_entropy(x, torch.zeros(5, 8, device="cuda"),
                                            torch.zeros(3, dtype=torch.int64, device="cuda")),
           lambda: vnn.linear_cross_entropy(x, torch.zeros(5, 8, device="cuda"),
                                            torch.zeros(4, dtype=torch.int64, device="cuda"), reduction="max")]
    for call in bad:
        with pytest.raises(ValueError):
            call()
