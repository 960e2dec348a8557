"""Under stream capture, a call of vkblas_nn.h whose workspace would only hold the partial sums of a K split runs
without the split, as a GEMM does; one that needs its workspace is refused before anything is enqueued."""
import pytest
import torch

import nn_ref as R
import vkblas_amd as vk

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


def captured(call):
    """The call's status under capture, and its graph."""
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        st = call()
    return st, g


# sizes whose two products the planner splits along K, on the side-by-side path, and without a split
@pytest.mark.parametrize("M,N,K", [(256, 4096, 256), (300, 3000, 264), (512, 256, 128), (1024, 1024, 1024)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_gated_gradient_with_a_place_for_its_projections_gradient(M, N, K, dt):
    dh, gu, x, w = (R.values(a, b, dt, 1 + i, 0.1).to(R.TORCH[dt]).cuda()
                    for i, (a, b) in enumerate(((M, N), (M, 2 * N), (M, K), (2 * N, K))))
    d, dx, dw = torch.empty_like(gu), torch.empty_like(x), torch.empty_like(w)

    def call():
        return vk.glu_backward_async(R.ENGINE[dt], vk.ACT_SILU, M, N, K, dh.data_ptr(), N, gu.data_ptr(), 2 * N,
                                     x.data_ptr(), K, w.data_ptr(), K, d.data_ptr(), 2 * N, dx.data_ptr(), K,
                                     dw.data_ptr(), K, R.ENGINE[dt], 0.0, stream=stream(), check=False)
    assert call() == vk.OK
    torch.cuda.synchronize()
    st, g = captured(call)
    assert st == vk.OK
    for seed in range(3):
        dh.copy_(R.values(M, N, dt, 10 + seed, 0.1).to(R.TORCH[dt]))
        assert call() == vk.OK
        torch.cuda.synchronize()
        eager = [v.double().clone() for v in (d, dx, dw)]
        for v in (d, dx, dw):
            v.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(d.double(), eager[0])
        D = eager[0]
        for got, ref, mag, n in ((dx, D @ w.double(), D.abs() @ w.double().abs(), 2 * N),
                                 (dw, D.t() @ x.double(), D.abs().t() @ x.double().abs(), M)):
            R.close(got.double(), ref, R.rounded(ref, dt, (n + 8) * R.E * mag), "product")


def test_gated_projection_into_its_kept_projections():
    """fp32 with gu: the product goes there, so a K split's sums are all that the workspace is for."""
    M, N, K, dt = 96, 128, 8192, "f32"
    x, w = (R.values(a, K, dt, 1 + i, 0.1).float().cuda() for i, a in enumerate((M, 2 * N)))
    h, gu = torch.empty(M, N, device="cuda"), torch.empty(M, 2 * N, device="cuda")

    def call():
        return vk.glu_async(vk.DT_F32, vk.ACT_RELU, M, N, K, x.data_ptr(), K, w.data_ptr(), K, h.data_ptr(), N,
                            gu.data_ptr(), 2 * N, stream=stream(), check=False)
    assert call() == vk.OK and vk.last_kernel() == vk.KERNEL_JOINED
    st, g = captured(call)
    assert st == vk.OK
    for seed in range(3):
        x.copy_(R.values(M, K, dt, 10 + seed, 0.1))
        assert call() == vk.OK
        torch.cuda.synchronize()
        h.fill_(float("nan"))
        gu.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        z = x.double() @ w.double().t()
        err = R.dot_bound(x.double(), w.double().t())
        R.close(gu.double(), z, R.rounded(z, dt, err), "gu")
        u = z[:, N:]
        R.close(h.double(), z[:, :N].relu() * u,
                R.rounded(z[:, :N].relu() * u, dt, err[:, :N] * (u.abs() + err[:, N:]) + z[:, :N].abs() * err[:, N:]), "h")


def test_refused_before_anything_is_enqueued():
    """A decode-shaped product splits K and has no form without: refused, and dgu is not written."""
    M, N, K = 20, 8192, 512
    dt = "bf16"
    dh, gu, x, w = (R.values(a, b, dt, 1 + i, 0.1).to(R.TORCH[dt]).cuda()
                    for i, (a, b) in enumerate(((M, N), (M, 2 * N), (M, K), (2 * N, K))))
    d, dx = torch.zeros_like(gu), torch.zeros_like(x)

    def call():
        return vk.glu_backward_async(R.ENGINE[dt], vk.ACT_SILU, M, N, K, dh.data_ptr(), N, gu.data_ptr(), 2 * N,
                                     x.data_ptr(), K, w.data_ptr(), K, d.data_ptr(), 2 * N, dx.data_ptr(), K, None, K,
                                     R.ENGINE[dt], 0.0, stream=stream(), check=False)
    y = torch.zeros(4, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y += 1
        st = call()
    g.replay()
    torch.cuda.synchronize()
    assert st in (vk.OK, vk.ERR_INIT)
    if st == vk.ERR_INIT:
        assert not d.any() and not dx.any()
