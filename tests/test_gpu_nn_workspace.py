"""The operators' workspaces: streams at once, threads at once, and a workspace that grew or shrank between calls."""
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
        rand = lambda *s: (torch.randn(*s, generator=g, device="cuda") * 0.1).to(t)
        self.op, self.M, self.V, self.K, self.dt = op, M, V, K, R.ENGINE[dt]
        self.x, self.w = rand(M, K), rand(2 * V if op == "glu_backward" else V, K)
        if op == "norm":
            self.dy, self.mean = rand(M, K), torch.zeros(M, device="cuda")
            self.rstd, self.out = torch.ones(M, device="cuda"), [torch.empty_like(self.x), *torch.empty(2, K, device="cuda")]
        elif op == "glu_backward":
            self.dh, self.gu = rand(M, V), rand(M, 2 * V)
            self.out = [torch.empty_like(self.x), torch.empty_like(self.w)]
        else:
            self.t = torch.randint(0, V, (M,), generator=g, device="cuda")
            self.lse, self.dloss = torch.full((M,), 5.0, device="cuda"), torch.ones(M, device="cuda")
            self.out = (list(torch.empty(2, M, device="cuda")) if op == "xent"
                        else [torch.empty_like(self.x), torch.empty_like(self.w)])

    def run(self, stream):
        p, M, V, K, dt = [v.data_ptr() for v in self.out], self.M, self.V, self.K, self.dt
        x, w = self.x.data_ptr(), self.w.data_ptr()
        if self.op == "norm":
            vk.layer_norm_backward_async(dt, vk.DT_F32, M, K, self.dy.data_ptr(), K, x, K, None, self.mean.data_ptr(),
                                         self.rstd.data_ptr(), p[0], K, p[1], p[2], vk.DT_F32, stream=stream)
        elif self.op == "glu_backward":
            vk.glu_backward_async(dt, vk.ACT_GELU, M, V, K, self.dh.data_ptr(), V, self.gu.data_ptr(), 2 * V, x, K, w, K,
                                  None, 0, p[0], K, p[1], K, dt, stream=stream)
        elif self.op == "xent":
            vk.linear_xent_async(dt, M, V, K, x, K, w, K, self.t.data_ptr(), -100, p[0], p[1], stream=stream)
        else:
            vk.linear_xent_backward_async(dt, M, V, K, x, K, w, K, self.t.data_ptr(), -100, self.lse.data_ptr(),
                                          self.dloss.data_ptr(), p[0], K, p[1], K, dt, stream=stream)

    def bits(self):
        torch.cuda.synchronize()
        return [v.clone() for v in self.out]


STEPS = [("xent", 300, 5003, 256, "bf16"), ("xent_backward", 300, 5003, 256, "f16"), ("norm", 2000, 1, 520, "bf16"),
         ("glu_backward", 260, 700, 320, "bf16"), ("xent_backward", 40, 900, 72, "f32"), ("glu_backward", 5, 333, 77, "f32"),
         ("xent", 9, 20000, 64, "f32"), ("xent_backward", 1200, 2003, 200, "bf16")]


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
