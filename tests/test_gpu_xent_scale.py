"""The factor that the cross entropy's 16-bit D is divided by comes from the rows that count: what an ignored row's
loss gradient holds, or one row's that is not finite, costs the other rows nothing."""
import pytest
import torch

import test_gpu_linear_xent as X
import vkblas_amd as vk

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")

# rows on the joined path, on the pipelined kernel (its own search for the factor), and past its 1024 rows
SIZES = [(60, 400, 64), (300, 513, 128), (1500, 700, 128)]


def counted(args):
    """args with the loss gradients of ignored rows zero, as the definition takes them."""
    x, w, t, lse, dloss = args
    return x, w, t, lse, torch.where(t == X.IGNORE, torch.zeros_like(dloss), dloss)


@pytest.mark.parametrize("M,V,K", SIZES)
@pytest.mark.parametrize("value", [1e4, 1e20, 1e35, INF, -INF, NAN])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_ignored_rows_loss_gradients(M, V, K, value, dt):
    x, w, t, lse, dloss = X.grad_inputs(M, V, K, dt, 1e-3)
    dloss[t == X.IGNORE] = value
    args = (x, w, t, lse, dloss)
    X.check_backward(X.backward(*args, dt, wt="f32"), *counted(args), dt, wt="f32")


@pytest.mark.parametrize("M,V,K", SIZES)
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_rows_of_an_invalid_target(M, V, K, dt):
    """Their own gradient is NaN; the other rows' as without them."""
    x, w, t, lse, dloss = X.grad_inputs(M, V, K, dt, 1e-3)
    t[3], dloss[3] = V, 1e20
    dx, _ = X.backward(x, w, t, lse, dloss, dt)
    assert bool(torch.isnan(dx[3]).all())
    rows = torch.arange(M) != 3
    args = (x[rows], w, t[rows], lse[rows], dloss[rows])
    X.check_backward((dx[rows], None), *counted(args), dt, want="x")


@pytest.mark.parametrize("M,V,K", SIZES)
@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_a_row_whose_loss_gradient_is_not_finite(M, V, K, value, dt):
    x, w, t, lse, dloss = X.grad_inputs(M, V, K, dt, 1e-3)
    dloss[3] = value
    dx, _ = X.backward(x, w, t, lse, dloss, dt)
    assert not bool(torch.isfinite(dx[3]).any())
    rows = torch.arange(M) != 3
    args = (x[rows], w, t[rows], lse[rows], dloss[rows])
    X.check_backward((dx[rows], None), *counted(args), dt, want="x")


@pytest.mark.parametrize("M,V,K", SIZES)
@pytest.mark.parametrize("loss_scale", [1e-30, 1e-28, 1e28, 1e33, 1e37])
def test_loss_gradients_of_any_size(M, V, K, loss_scale):
    """fp32 weight gradients of fp16 operands, far outside the type's own range."""
    args = X.grad_inputs(M, V, K, "f16", loss_scale)
    X.check_backward(X.backward(*args, "f16", wt="f32", want="w"), *args, "f16", wt="f32", want="w")
