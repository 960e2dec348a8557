"""The operators of vkblas_train.h under stream capture: those without a workspace replay with new values as eager calls
compute them, those that need one are refused before anything is enqueued."""
import pytest
import torch

import nn_ref as R
import vkblas_amd as vk

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


def captured(call):
    """The call's status under capture, its graph, and what the graph counts in, so that one of refused calls alone is
    not empty."""
    count, g = torch.zeros(4, device="cuda"), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        count += 1
        st = call()
    return st, g, count


def replays(call, change, outputs):
    assert call() == vk.OK
    torch.cuda.synchronize()
    st, g, count = captured(call)
    assert st == vk.OK
    for turn in range(3):
        change(turn)
        assert call() == vk.OK
        torch.cuda.synchronize()
        want = [t.clone() for t in outputs]
        for t in outputs:
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outputs, want))
        assert not any(bool(torch.isnan(t).any()) for t in want) and bool((count == turn + 1).all())


def refused(call, outputs):
    for t in outputs:
        t.fill_(7.0)
    torch.cuda.synchronize()
    st, g, count = captured(call)
    assert st == vk.ERR_INIT
    g.replay()
    torch.cuda.synchronize()
    assert all(bool((t == 7.0).all()) for t in outputs) and bool((count == 1).all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("M", [5, 4096])
def test_embedding(dt, M):
    V, N, t = 300, 72, R.TORCH[dt]
    w, dy = torch.randn(V, N, device="cuda").to(t), torch.randn(M, N, device="cuda").to(t)
    ids = torch.zeros(M, dtype=torch.int64, device="cuda")
    y, dw = torch.empty(M, N, device="cuda", dtype=t), torch.empty(V, N, device="cuda", dtype=t)

    def change(turn):
        ids.copy_(torch.randint(-1, V, (M,)))
        dy.copy_(torch.randn(M, N))
    replays(lambda: vk.embedding_async(R.ENGINE[dt], R.ENGINE[dt], M, V, N, ids.data_ptr(), -1, w.data_ptr(), N, 2.0,
                                       y.data_ptr(), N, stream=stream(), check=False), change, [y])
    replays(lambda: vk.embedding_backward_async(R.ENGINE[dt], M, V, N, ids.data_ptr(), -1, dy.data_ptr(), N, 2.0,
                                                dw.data_ptr(), N, R.ENGINE[dt], 0.0, stream=stream(), check=False),
            change, [dw])


def policy(B, T):
    old, logp, ref, adv, stats, norm, dlogp = (torch.randn(*s, device="cuda") * 0.1 for s in (
        (B, T), (B, T), (B, T), (B, 1), (4,), (B,), (B, T)))
    mask, dloss = torch.ones(B, T, dtype=torch.uint8, device="cuda"), torch.ones(1, device="cuda")
    args = (B, T, logp.data_ptr(), T, old.data_ptr(), T, ref.data_ptr(), T, adv.data_ptr(), 1, 0, mask.data_ptr(), T,
            0.2, 0.2, 0.1)

    def loss():
        return vk.policy_loss_async(vk.REDUCE_SEQUENCES, *args, stats.data_ptr(), norm.data_ptr(), stream=stream(),
                                    check=False)

    def grad():
        return vk.policy_loss_backward_async(*args, norm.data_ptr(), dloss.data_ptr(), dlogp.data_ptr(), T,
                                             stream=stream(), check=False)

    def change(turn):
        logp.copy_(torch.randn(B, T) * 0.1)
        mask.copy_(torch.rand(B, T) < 0.7)
    loss.alive = grad.alive = old, logp, ref, adv, mask     # the arguments hold their addresses alone
    return loss, grad, change, [stats, norm], [dlogp]


def test_policy_loss():
    loss, grad, change, out, dlogp = policy(8, 500)
    replays(loss, change, out)
    replays(grad, change, dlogp)
    _, grad, change, _, dlogp = policy(300, 700)
    replays(grad, change, dlogp)


def test_refused_before_anything_is_enqueued():
    loss, _, _, out, _ = policy(300, 700)
    refused(loss, out)
    M, V, N = 5000, 300, 64
    ids, dy = torch.zeros(M, dtype=torch.int64, device="cuda"), torch.randn(M, N, device="cuda")
    dw = torch.empty(V, N, device="cuda")
    refused(lambda: vk.embedding_backward_async(vk.DT_F32, M, V, N, ids.data_ptr(), -1, dy.data_ptr(), N, 1.0,
                                                dw.data_ptr(), N, vk.DT_F32, 0.0, stream=stream(), check=False), [dw])
    M, V, K, n = 100, 500, 64, 8
    x, w, t = (torch.randn(a, b, device="cuda") for a, b in ((M, K), (V, K), (M, n)))
    top = torch.randint(0, V, (M, n), device="cuda")
    loss, lse, zt, dx, dw = (torch.zeros(*s, device="cuda") for s in ((M,), (M,), (M, n), (M, K), (V, K)))
    args = (vk.DT_F32, M, V, K, x.data_ptr(), K, w.data_ptr(), K, n, top.data_ptr(), n, vk.DT_F32, t.data_ptr(), n, 1.0)
    refused(lambda: vk.linear_distill_async(*args, loss.data_ptr(), lse.data_ptr(), zt.data_ptr(), stream=stream(),
                                            check=False), [loss, lse, zt])
    refused(lambda: vk.linear_distill_backward_async(*args, lse.data_ptr(), zt.data_ptr(), loss.data_ptr(),
                                                     dx.data_ptr(), K, dw.data_ptr(), K, vk.DT_F32, 0.0, stream=stream(),
                                                     check=False), [dx, dw])
