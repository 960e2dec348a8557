"""A layer norm gradient whose weight gradients are not wanted takes any g_type, for few rows as for many."""
import pytest
import torch

import nn_ref as R
import vkblas_amd as vk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N", [(3, 64), (1024, 200), (1025, 200), (512, 8000), (513, 8000), (4, 5), (4, 20000)])
@pytest.mark.parametrize("dt,g", [("f16", vk.DT_BF16), ("bf16", vk.DT_F16), ("f32", vk.DT_BF16), ("bf16", 77)])
def test_any_type_of_gradients_that_are_not_wanted(M, N, dt, g):
    x, dy = R.values(M, N, dt, 1), R.values(M, N, dt, 2)
    _, mean, rstd = R.norm(x, 1.0, 0.0, 1e-5)
    bx, bd, dx = R.Buf(M, N, dt, values=x), R.Buf(M, N, dt, values=dy), R.Buf(M, N, dt)
    bm, br = R.Buf(1, M, "f32", values=mean[None]), R.Buf(1, M, "f32", values=rstd[None])
    vk.layer_norm_backward_async(R.ENGINE[dt], R.ENGINE[dt], M, N, bd.ptr, N, bx.ptr, N, None, bm.ptr, br.ptr, dx.ptr, N,
                                 None, None, g, stream=torch.cuda.current_stream().cuda_stream)
    dx.check_around()
    ref, _, _ = R.norm_grad(dy, x, 1.0, bm.get()[0], br.get()[0])
    # dx is a few products and sums of N values of the size of dy rstd: their mean's error is below 64 e of it
    err = (rstd[:, None] * (dy.abs() + 4 * dy.abs().max())) * 64 * R.E * (1 + x.abs())
    R.close(dx.get(), ref, R.rounded(ref, dt, err), "dx")
