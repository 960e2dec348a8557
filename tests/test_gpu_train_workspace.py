"""The workspaces of vkblas_train.h's operators: streams at once, threads at once, calls of other sizes and of other
operators between them, and a release."""
import threading

import pytest
import torch

import nn_ref as R
import vkblas_amd as vk

pytestmark = pytest.mark.gpu


class Step:
    """One call of an operator that takes a workspace, on inputs of its own, and its results."""

    def __init__(self, op, M, V, K, dt, seed):
        t = R.TORCH[dt]
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda") * 0.1
        self.op, self.M, self.V, self.K, self.dt = op, M, V, K, R.ENGINE[dt]
        if op == "embedding":
            self.ids = (V ** torch.rand(M, generator=g, device="cuda") - 1).long()
            self.x, self.out = rand(M, K).to(t), [torch.empty(V, K, device="cuda", dtype=t)]
        elif op == "policy":
            self.logp, self.old, self.adv = rand(M, V), rand(M, V), rand(M, V)
            self.out = [torch.empty(4, device="cuda"), torch.empty(M, device="cuda")]
        else:
            self.x, self.w, self.t = rand(M, K).to(t), rand(V, K).to(t), rand(M, 12)
            self.top = torch.randint(-1, V, (M, 12), generator=g, device="cuda")
            self.lse, self.zt = torch.full((M,), 5.0, device="cuda"), rand(M, 12)
            self.dloss = torch.ones(M, device="cuda")
            if op == "distill":
                self.out = [torch.empty(s, device="cuda") for s in (M, M, (M, 12))]
            else:
                self.out = [torch.empty_like(self.x), torch.empty_like(self.w)]

    def run(self, stream):
        p, M, V, K, dt = [v.data_ptr() for v in self.out], self.M, self.V, self.K, self.dt
        if self.op == "embedding":
            vk.embedding_backward_async(dt, M, V, K, self.ids.data_ptr(), -1, self.x.data_ptr(), K, 1.0, p[0], K, dt,
                                        0.0, stream=stream)
            return
        if self.op == "policy":
            vk.policy_loss_async(vk.REDUCE_TOKENS, M, V, self.logp.data_ptr(), V, self.old.data_ptr(), V, None, 0,
                                 self.adv.data_ptr(), V, 1, None, 0, 0.2, 0.2, 0.0, *p, stream=stream)
            return
        args = (dt, M, V, K, self.x.data_ptr(), K, self.w.data_ptr(), K, 12, self.top.data_ptr(), 12, vk.DT_F32,
                self.t.data_ptr(), 12, 2.0)
        if self.op == "distill":
            vk.linear_distill_async(*args, *p, stream=stream)
        else:
            vk.linear_distill_backward_async(*args, self.lse.data_ptr(), self.zt.data_ptr(), self.dloss.data_ptr(), p[0],
                                             K, p[1], K, dt, 0.0, stream=stream)

    def bits(self):
        torch.cuda.synchronize()
        return [v.clone() for v in self.out]


STEPS = [("embedding", 5000, 300, 264, "bf16"), ("distill", 300, 5003, 256, "bf16"), ("policy", 300, 700, 1, "f32"),
         ("distill_grad", 300, 5003, 256, "f16"), ("embedding", 40000, 2000, 65, "f32"),
         ("distill_grad", 40, 900, 72, "f32"), ("distill", 9, 20000, 64, "f32"), ("policy", 20, 9000, 1, "f32"),
         ("distill_grad", 1200, 2003, 200, "bf16"), ("distill", 11000, 300, 4096, "bf16"), ("policy", 9000, 300, 1, "f32"),
         ("policy", 300, 90, 1, "f32")]


def alone():
    """The steps and their results, one after the other on one stream."""
    steps, want = [Step(*s, seed=10 + i) for i, s in enumerate(STEPS)], []
    for s in steps:
        s.run(torch.cuda.current_stream().cuda_stream)
        want.append(s.bits())
        for v in s.out:
            v.fill_(float("nan"))
    torch.cuda.synchronize()
    return steps, want


def same(steps, want):
    for s, w in zip(steps, want):
        assert all(torch.equal(a, b) for a, b in zip(s.bits(), w)), s.op


def test_streams_at_once():
    steps, want = alone()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(6):
        for i, s in enumerate(steps):
            s.run(streams[(i + turn) % 3].cuda_stream)
        same(steps, want)


@pytest.mark.parametrize("shared", [False, True])
def test_threads_at_once(shared):
    """Each thread on its own stream, or all on one."""
    steps, want = alone()
    streams = [torch.cuda.Stream() for _ in steps]
    errors = []

    def work(i):
        try:
            for _ in range(8):
                steps[i].run(streams[0 if shared else i].cuda_stream)
        except Exception as e:       # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(steps))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors
    same(steps, want)


def test_after_smaller_larger_and_released_workspaces():
    """Calls without a wait between them whose workspaces differ in size, on a fresh stream and after a release."""
    steps, want = alone()
    order = sorted(range(len(steps)), key=lambda i: steps[i].M * steps[i].V)
    st = torch.cuda.Stream()
    for turn in range(3):
        for i in order + order[::-1]:
            steps[i].run(st.cuda_stream)
        same(steps, want)
        vk.workspace_release()
