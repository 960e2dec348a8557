"""vkblas_amd.torch_nn's embedding, distillation and policy loss against PyTorch's own in float64 through autograd, on
strided and many-dimensional inputs, with their refusals, and run together as a training step runs them; on the CPU
with the library's calls stubbed where values do not matter."""
import contextlib

import pytest
import torch

import nn_ref as R
import vkblas_amd as vk
from test_gpu_torch_nn import near, values

f = torch.nn.functional


@pytest.fixture
def vnn(monkeypatch):
    """torch_nn on the CPU, its launches stubbed."""
    from vkblas_amd import torch_nn
    for name in vk._NN_ARGS:
        monkeypatch.setattr(vk, f"{name}_async", lambda *a, **k: vk.OK)
    monkeypatch.setattr(torch_nn, "_check", lambda *a: None)
    monkeypatch.setattr(torch_nn, "_stream", lambda t: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    return torch_nn


def classes_of(shape, V, n, seed=7):
    """Distinct classes and the teacher's logits there; some rows shorter, one without a teacher."""
    g = torch.Generator().manual_seed(seed)
    c = torch.rand(*shape, V, generator=g).argsort(-1)[..., :n].clone()
    c[..., 1::3, n // 2:] = -1
    c[..., 0, :] = -1
    return c, torch.randn(*shape, n, generator=g) * 2


def distillation(x, w, c, t, temperature):
    """Each row's loss in plain operations."""
    log_p = f.log_softmax(f.linear(x, w) / temperature, -1)
    t = torch.where(c >= 0, t / temperature, torch.full_like(t, -1e30))
    some = (c >= 0).any(-1)
    q, log_q = f.softmax(t, -1), f.log_softmax(t, -1)
    terms = torch.where(c >= 0, q * (log_q - log_p.gather(-1, c.clamp(min=0))), torch.zeros_like(q))
    return torch.where(some, temperature ** 2 * terms.sum(-1), torch.zeros_like(terms[..., 0])), some


def policy(logp, old, adv, ref, mask, clip, kl, reduction):
    ratio = torch.exp(logp - old)
    adv = adv if adv.dim() == logp.dim() else adv.unsqueeze(-1)
    loss = -torch.minimum(ratio * adv, ratio.clamp(1 - clip[0], 1 + clip[1]) * adv)
    if ref is not None:
        loss = loss + kl * (torch.expm1(ref - logp) - (ref - logp))
    loss = torch.where(mask, loss, torch.zeros_like(loss))
    n = mask.sum(-1)
    if reduction == "tokens":
        return loss.sum() / n.sum()
    if reduction == "sequences":
        return (loss.sum(-1) / n.clamp(min=1))[n > 0].sum() / (n > 0).sum()
    return loss.sum()


# ---- without a GPU

@pytest.mark.parametrize("change", [lambda y: y.mul_(2.0), lambda y: y.add_(1.0)])
def test_results_may_be_changed_in_place(vnn, change, monkeypatch):
    w = torch.zeros(6, 8, requires_grad=True)
    change(vnn.embedding(torch.zeros(2, 3, dtype=torch.int64), w)).sum().backward()
    assert w.grad.shape == w.shape
    x, c = torch.zeros(2, 3, 8, requires_grad=True), torch.zeros(2, 3, 4, dtype=torch.int64)
    for reduction in ("none", "sum", "mean"):
        y = vnn.linear_distillation(x, w, c, torch.zeros(2, 3, 4), reduction=reduction)
        assert y.shape == ((2, 3) if reduction == "none" else ())
        change(y).sum().backward()
    assert x.grad.shape == x.shape
    y = vnn.embedding(torch.zeros(2, 3, dtype=torch.int64), w)
    assert y.shape == (2, 3, 8) and y._base is None
    y = vnn.linear_distillation(x, w, c, torch.zeros(2, 3, 4), reduction="none")
    assert y._base is None and y.untyped_storage().nbytes() == 24


def test_refusals_without_a_gpu():
    from vkblas_amd import torch_nn
    x = torch.zeros(4, 8)
    for call in (lambda: torch_nn.embedding(torch.zeros(3, dtype=torch.int64), x),
                 lambda: torch_nn.linear_distillation(x, x, torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2)),
                 lambda: torch_nn.policy_loss(x, x, x)):
        with pytest.raises(ValueError, match="on a GPU"):
            call()


# ---- on the GPU

@pytest.mark.gpu
@pytest.mark.parametrize("dt,out", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("f32", "f16")])
def test_embedding(dt, out):
    from vkblas_amd import torch_nn as vnn
    w = values(50, 72, dt=dt, seed=1)
    ids = torch.randint(0, 50, (3, 40), generator=torch.Generator().manual_seed(2))
    ids[:, 30:] = 7
    got, ref = w.cuda().requires_grad_(), w.double().requires_grad_()
    y = vnn.embedding(ids.cuda(), got, scale=1.5, padding_idx=7, dtype=R.TORCH[out])
    assert y.dtype == R.TORCH[out] and y.shape == (3, 40, 72)
    z = 1.5 * ref[ids] * (ids != 7)[..., None]
    g = values(3, 40, 72, dt=out, seed=3)
    y.backward(g.cuda())
    z.backward(g.double())
    assert got.grad.dtype == w.dtype
    near([y.detach().double().cpu(), got.grad.double().cpu()], [z.detach(), ref.grad], out)
    with torch.no_grad():
        assert torch.equal(vnn.embedding(ids.cuda()[:, ::2], w.cuda()).cpu(), w[ids[:, ::2]])
        wide = values(50, 100, dt=dt, seed=5)
        assert torch.equal(vnn.embedding(ids.cuda(), wide.cuda()[:, 20:80]).cpu(), wide[:, 20:80][ids])
        assert vnn.embedding(ids.cuda()[:0], w.cuda()).shape == (0, 40, 72)
        assert bool(torch.isnan(vnn.embedding(torch.tensor([-1, 50], device="cuda"), w.cuda())).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_linear_distillation(dt, reduction, temperature):
    from vkblas_amd import torch_nn as vnn
    x, w = values(3, 40, 128, dt=dt, seed=1), values(333, 128, dt=dt, seed=2, scale=0.2)
    c, t = classes_of((3, 40), 333, 20)
    out = []
    for own in (True, False):
        a, b = (v.cuda() if own else v.double() for v in (x, w))
        a.requires_grad_(), b.requires_grad_()
        if own:
            y = vnn.linear_distillation(a, b, c.cuda(), t.cuda(), temperature, reduction)
        else:
            y, some = distillation(a, b, c, t.double(), temperature)
            y = y if reduction == "none" else y.sum() / (some.sum() if reduction == "mean" else 1)
        g = torch.randn(y.shape, generator=torch.Generator().manual_seed(5), dtype=torch.float64).float()
        y.backward(g.to(y.device, y.dtype))
        out.append([v.detach().double().cpu() for v in (y, a.grad, b.grad)])
    near(*out, dt)


@pytest.mark.gpu
def test_linear_distillation_of_strided_entries():
    from vkblas_amd import torch_nn as vnn
    x, w = values(40, 128, dt="bf16", seed=1).cuda(), values(333, 128, dt="bf16", seed=2, scale=0.2).cuda()
    c, t = classes_of((40,), 333, 20)
    c, t = c.cuda(), t.bfloat16().cuda()
    want = vnn.linear_distillation(x, w, c[:, :7].contiguous(), t[:, :7].contiguous(), 2.0, "none")
    assert torch.equal(vnn.linear_distillation(x, w, c[:, :7], t[:, :7], 2.0, "none"), want)
    assert torch.equal(vnn.linear_distillation(x, w, c.t().contiguous().t()[:, :7], t.t().contiguous().t()[:, :7], 2.0,
                                               "none"), want)
    one = vnn.linear_distillation(x, w, c[5:6].expand(40, 20), t[5:6].expand(40, 20), 1.0, "none")
    assert torch.equal(one, vnn.linear_distillation(x, w, c[5:6].repeat(40, 1), t[5:6].repeat(40, 1), 1.0, "none"))


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["tokens", "sequences", "sum"])
@pytest.mark.parametrize("shape", [(6, 50), (2, 3, 50), (50,), (90, 400)])
@pytest.mark.parametrize("per_token", [True, False])
def test_policy_loss(reduction, shape, per_token):
    from vkblas_amd import torch_nn as vnn
    g = torch.Generator().manual_seed(1)
    old = torch.log(torch.rand(shape, generator=g) + 1e-3)
    logp, ref = (old + s * torch.randn(shape, generator=g) for s in (0.2, 0.3))
    adv = torch.randn(shape if per_token else shape[:-1], generator=g)
    mask = torch.rand(shape, generator=g) < 0.7
    clip = tuple(float(torch.tensor(c)) for c in (0.2, 0.3))
    a, b = logp.cuda().requires_grad_(), logp.double().requires_grad_()
    loss, stats = vnn.policy_loss(a, old.cuda(), adv.cuda(), ref.cuda(), mask.cuda(), clip, 0.25, reduction)
    want = policy(b, old.double(), adv.double(), ref.double(), mask, clip, 0.25, reduction)
    (3 * loss).backward()
    (3 * want).backward()
    assert stats.shape == (4,) and not stats.requires_grad and torch.equal(stats[0], loss.detach())
    near([a.grad.double().cpu()], [b.grad], "f32")
    size = policy(b, old.double(), -adv.double().abs(), ref.double(), mask, clip, 0.25, reduction)
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * float(size.detach())
    loss.mul_(2.0)      # an ordinary tensor


@pytest.mark.gpu
def test_policy_loss_of_strided_rows_and_an_empty_batch():
    from vkblas_amd import torch_nn as vnn
    wide = torch.log(torch.rand(4, 10, 60, device="cuda") + 1e-3)
    old, logp = wide[0][:, :50], wide[1][:, 5:55]
    adv = torch.randn(10, 60, device="cuda")[:, 3:53]
    mask = torch.rand(10, 60, device="cuda")[:, 2:52] < 0.5
    got = vnn.policy_loss(logp, old, adv, mask=mask)[0]
    assert torch.equal(got, vnn.policy_loss(*(t.contiguous() for t in (logp, old, adv)), mask=mask.contiguous())[0])
    empty = torch.zeros(0, 5, device="cuda", requires_grad=True)
    loss, stats = vnn.policy_loss(empty, empty.detach(), empty.detach())
    loss.backward()
    assert float(loss) == 0.0 and bool((stats == 0).all()) and empty.grad.shape == (0, 5)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    from vkblas_amd import torch_nn as vnn
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(6, 8, device="cuda")
    i, c, t = (torch.zeros(*s, dtype=d, device="cuda") for s, d in (((3,), torch.int64), ((4, 2), torch.int64),
                                                                    ((4, 2), torch.float32)))
    p = torch.zeros(4, 5, device="cuda")
    many = vk.DISTILL_TOP + 1
    bad = [lambda: vnn.embedding(i.int(), w), lambda: vnn.embedding(i.cpu(), w), lambda: vnn.embedding(i, w[0]),
           lambda: vnn.embedding(i, w[:0]), lambda: vnn.embedding(i, w.half(), dtype=torch.float32),
           lambda: vnn.embedding(i, w, dtype=torch.float64), lambda: vnn.embedding(i, w[:, :0]),
           lambda: vnn.linear_distillation(x, w[:, :7], c, t), lambda: vnn.linear_distillation(x, w, c.int(), t),
           lambda: vnn.linear_distillation(x, w, c[:3], t[:3]), lambda: vnn.linear_distillation(x, w, c, t[:, :1]),
           lambda: vnn.linear_distillation(x, w, c, t.half()), 
           lambda: vnn.linear_distillation(x, w, c[:, :0], t[:, :0]),
           lambda: vnn.linear_distillation(x, w, c.repeat(1, many), t.repeat(1, many)),
           lambda: vnn.linear_distillation(x, w, c, t.clone().requires_grad_()),
           lambda: vnn.linear_distillation(x, w, c, t, 0.0), lambda: vnn.linear_distillation(x, w, c, t, float("nan")),
           lambda: vnn.linear_distillation(x, w, c, t, reduction="max"),
           lambda: vnn.policy_loss(p.half(), p, p), lambda: vnn.policy_loss(p, p[:3], p),
           lambda: vnn.policy_loss(p, p, p[0]), lambda: vnn.policy_loss(p, p.half(), p),
           lambda: vnn.policy_loss(p, p, p, p.cpu()), lambda: vnn.policy_loss(p, p, p, mask=p), lambda: vnn.policy_loss(p, p, p, mask=(p == 0)[:2]),
           lambda: vnn.policy_loss(p, p.clone().requires_grad_(), p),
           lambda: vnn.policy_loss(p, p, p, clip=(-0.1, 0.1)),
           lambda: vnn.policy_loss(p, p, p, clip=(0.1, float("nan"))),
           lambda: vnn.policy_loss(p, p, p, reduction="mean"),
           lambda: vnn.policy_loss(p[:, :0], p[:, :0], p[:, :0])]
    for call in bad:
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_a_step_of_them_together(dt):
    """Tied embedding, norm, gated block, then the three losses of one hidden state: cross entropy, distillation and,
    on its log probabilities, the policy loss.  Against PyTorch's own operations in float64."""
    from vkblas_amd import torch_nn as real
    V, N, shape = 200, 64, (4, 30)
    g = torch.Generator().manual_seed(1)
    e0, g0 = values(V, N, dt=dt, seed=2, scale=0.5), values(2 * N, N, dt=dt, seed=3, scale=0.1)
    ids, target = (torch.randint(1, V, shape, generator=g) for _ in range(2))
    ids[:, 25:] = 0
    mask = ids != 0
    c, t = classes_of(shape, V, 10)
    adv = torch.randn(4, generator=g)
    noise, clip = 0.1 * torch.randn(shape, generator=g), (0.25, 0.25)

    def own(e, gu):
        x = real.embedding(ids.cuda(), e, scale=2.0, padding_idx=0)
        h = real.layer_norm(x + real.gated_linear(real.layer_norm(x), gu))
        nll = real.linear_cross_entropy(h, e, target.cuda(), reduction="none")
        distilled = real.linear_distillation(h, e, c.cuda(), t.cuda(), 2.0)
        loss, _ = real.policy_loss(-nll, (noise.cuda() - nll).detach(), adv.cuda(), (-nll - noise.cuda()).detach(),
                                   mask.cuda(), clip, 0.125)
        return nll.mean() + distilled + loss

    def ref(e, gu):
        x = 2.0 * e[ids] * mask[..., None]
        a, b = f.linear(f.layer_norm(x, (N,)), gu).chunk(2, -1)
        h = f.layer_norm(x + f.silu(a) * b, (N,))
        nll = f.cross_entropy(f.linear(h, e).flatten(0, 1), target.flatten(), reduction="none").view(shape)
        rows, some = distillation(h, e, c, t.double(), 2.0)
        loss = policy(-nll, (noise - nll).detach(), adv.double(), (-nll - noise).detach(), mask, clip, 0.125, "tokens")
        return nll.mean() + rows.sum() / some.sum() + loss

    out = []
    for fn, move in ((own, lambda v: v.cuda()), (ref, lambda v: v.double())):
        e, gu = move(e0).requires_grad_(), move(g0).requires_grad_()
        loss = fn(e, gu)
        loss.backward()
        out.append([v.detach().double().cpu() for v in (loss, e.grad, gu.grad)])
    # a chain of about twenty roundings to dt, each of values of the results' own size
    for a, b in zip(*out):
        assert float((a - b).abs().max()) <= max(20 * R.U[dt], 1e-5) * float(b.abs().max())
