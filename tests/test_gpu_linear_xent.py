"""vkblas_linear_xent_async and its backward pass against the definition in float64: types, one row to several
tiles, vocabularies of one class to several pieces, ignored and invalid targets, infinite logits, gradients far
below fp16's range."""
import pytest
import torch

import nn_ref as R
import vkblas_amd as vk

pytestmark = pytest.mark.gpu
IGNORE = -100


def stream():
    return torch.cuda.current_stream().cuda_stream


def inputs(M, V, K, dt, seed=1, scale=2.0, device="cpu"):
    x, w = R.values(M, K, dt, seed), R.values(V, K, dt, seed + 1, scale * K ** -0.5)
    g = torch.Generator().manual_seed(seed + 2)
    t = torch.randint(0, V, (M,), generator=g)
    t[::5] = IGNORE
    t[0], t[-1] = 0, V - 1
    return x.to(device), w.to(device), t.to(device)


def forward(x, w, t, dt, pad=0, off=0, ignore=IGNORE, want_loss=True):
    M, K = x.shape
    bx, bw = R.Buf(M, K, dt, pad, off, x), R.Buf(w.shape[0], K, dt, pad, off, w)
    loss, lse, tt = R.Buf(1, M, "f32"), R.Buf(1, M, "f32"), t.cuda()
    vk.linear_xent_async(R.ENGINE[dt], M, w.shape[0], K, bx.ptr, bx.ld, bw.ptr, bw.ld,
                         tt.data_ptr() if want_loss else None, ignore, loss.ptr if want_loss else None, lse.ptr,
                         stream=stream())
    loss.check_around()
    lse.check_around()
    return loss.get()[0], lse.get()[0]


def check_forward(got, x, w, t, ignore=IGNORE):
    z, loss, lse = R.xent(x, w, t, ignore)
    # a logit's error moves the log-sum-exp by at most the largest; a sum of V positive terms joined in trees
    # and runs of at most 600: 600 e relative
    ez = R.dot_bound(x, w.t()).max(1).values
    e = ez + 600 * R.E + R.STEP * (lse.abs() + 1)
    R.close(got[1], lse, e, "lse")
    fine = ~torch.isnan(loss)
    got = [v.to(loss.device) for v in got]
    assert torch.equal(torch.isnan(got[0]), ~fine)
    R.close(got[0][fine], loss[fine], (e + ez + 4 * R.E * z.abs().max(1).values)[fine], "loss")
    assert bool((got[0][t == ignore] == 0).all())


SIZES = [(1, 1, 1), (1, 5, 8), (2, 77, 9), (4, 3000, 515), (5, 1031, 2056), (8, 20000, 520), (9, 513, 1031), (16, 999, 700),
         (15, 1024, 1024), (1, 1000, 256), (3, 333, 72), (17, 4097, 64), (64, 515, 128), (65, 1000, 100),
         (128, 256, 128), (200, 300, 64), (256, 256, 192), (257, 1001, 128), (300, 700, 320), (511, 130, 128),
         (100, 10007, 77), (40, 20001, 64), (9, 5001, 9), (16, 17003, 515), (17, 4097, 1031), (32, 16500, 131), (3, 16384, 72), (3, 16385, 72)]


@pytest.mark.parametrize("M,V,K", SIZES)
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_forward(M, V, K, dt):
    x, w, t = inputs(M, V, K, dt)
    check_forward(forward(x, w, t, dt), x, w, t)


@pytest.mark.parametrize("M,V,K", [(5, 300, 128), (300, 513, 128)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,off", [(8, 0), (4, 4), (1, 0), (3, 1)])
def test_strides_and_alignment(M, V, K, dt, pad, off):
    x, w, t = inputs(M, V, K, dt)
    check_forward(forward(x, w, t, dt, pad, off), x, w, t)


# K that ends inside a step, in its first one, on it, and NaN behind each row; few tiles and many, of both sizes
@pytest.mark.parametrize("M,V", [(300, 513), (1100, 6500), (2100, 9000)])
@pytest.mark.parametrize("K", [8, 32, 64, 72, 136, 200, 232, 328])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_ends_of_k(M, V, K, dt):
    args = grad_inputs(M, V, K, dt, 64.0, device="cuda")
    x, w, t = args[:3]
    check_forward(forward(x, w, t, dt, pad=8), x, w, t)
    check_backward(backward(*args, dt, pad=8), *args, dt)


@pytest.mark.parametrize("M", [4, 300])
def test_targets(M):
    """An ignore_index inside the vocabulary, all rows ignored, invalid targets (NaN), lse alone."""
    x, w, t = inputs(M, 400, 128, "f32")
    t[1] = 7
    check_forward(forward(x, w, t, "f32", ignore=7), x, w, torch.where(t == IGNORE, torch.full_like(t, 400), t), 7)
    t[2], t[3] = 400, -1
    check_forward(forward(x, w, t, "f32"), x, w, t)
    none = torch.full_like(t, IGNORE)
    check_forward(forward(x, w, none, "f32"), x, w, none)
    _, lse = forward(x, w, t, "f32", want_loss=False)
    assert torch.equal(lse, forward(x, w, t, "f32")[1])


@pytest.mark.parametrize("M,V", [(3, 300), (300, 600)])
def test_large_and_infinite_logits(M, V):
    """Logits of +-1000 do not overflow; -inf classes count nothing, a +inf class makes lse +inf, NaN stays in
    its row, a row of only -inf has lse -inf."""
    K = 128
    x, w = torch.zeros(M, K, dtype=torch.float64), torch.zeros(V, K, dtype=torch.float64)
    x[:, 0] = 1.0
    w[:, 0] = torch.linspace(-1000, 1000, V, dtype=torch.float64).float().double()
    t = torch.arange(M) % V
    check_forward(forward(x, w, t, "f32"), x, w, t)
    w[: V - 5, 0] = float("-inf")
    w[0, 0] = 3.0
    loss, lse = forward(x, w, t, "f32")
    ref = torch.logsumexp(torch.cat((w[:1, 0], w[V - 5:, 0])), 0)
    R.close(lse, ref.expand(M), torch.full((M,), 1e-3, dtype=torch.float64), "lse")
    assert bool(torch.isinf(loss[1]))
    w[:, 0] = float("-inf")
    assert bool((forward(x, w, t, "f32")[1] == float("-inf")).all())
    w[:, 0] = 0.0
    w[3, 0] = float("inf")
    assert bool((forward(x, w, t, "f32")[1] == float("inf")).all())
    w[3, 0] = 0.0
    x[1, 0] = float("nan")
    _, lse = forward(x, w, t, "f32")
    assert bool(torch.isnan(lse[1])) and int(torch.isnan(lse).sum()) == 1


def backward(x, w, t, lse, dloss, dt, wt=None, pad=0, off=0, beta=0.0, dw0=None, want="xw", ignore=IGNORE):
    M, K = x.shape
    V, wt = w.shape[0], wt or dt
    bx, bw, tt = R.Buf(M, K, dt, pad, off, x), R.Buf(V, K, dt, pad, off, w), t.cuda()
    bl, bd = R.Buf(1, M, "f32", values=lse[None]), R.Buf(1, M, "f32", values=dloss[None])
    dx, dw = R.Buf(M, K, dt, pad, off), R.Buf(V, K, wt, pad, off, dw0)
    vk.linear_xent_backward_async(R.ENGINE[dt], M, V, K, bx.ptr, bx.ld, bw.ptr, bw.ld, tt.data_ptr(), ignore, bl.ptr,
                                  bd.ptr, dx.ptr if "x" in want else None, dx.ld, dw.ptr if "w" in want else None,
                                  dw.ld, R.ENGINE[wt], beta, stream=stream())
    dx.check_around()
    dw.check_around()
    return dx.get(), dw.get()


def check_backward(got, x, w, t, lse, dloss, dt, wt=None, beta=0.0, dw0=None, want="xw", ignore=IGNORE):
    wt = wt or dt
    z = x @ w.t()
    p = torch.exp(z - lse[:, None])
    hot = torch.nn.functional.one_hot(t.clamp(0, w.shape[0] - 1), w.shape[0])
    k = torch.where(t == ignore, torch.zeros_like(dloss), dloss)[:, None]
    d = (p - hot) * k
    # p moves with its logit's error and with the rounding of z - lse
    ed = k.abs() * (p * (R.dot_bound(x, w.t()) + R.STEP * (1 + (z - lse[:, None]).abs())) + 4 * R.E)
    # rounded to the type; over max |dloss|, fp16 times 2^13
    ed = ed + R.U[dt] * (d.abs() + ed) + (2.0 ** -25 * 2.0 ** -13 * float(dloss.abs().max()) if dt == "f16" else 0.0)
    if "x" in want:
        dx = d @ w
        R.close(got[0], dx, R.rounded(dx, dt, ed @ w.abs() + R.dot_bound(d.abs() + ed, w)), "dx")
    if "w" in want:
        old = torch.zeros_like(w) if dw0 is None else dw0
        dw = d.t() @ x + beta * old
        err = ed.t() @ x.abs() + R.dot_bound((d.abs() + ed).t(), x) + 4 * R.E * (beta * old).abs()
        R.close(got[1], dw, R.rounded(dw, wt, err), "dw")


def grad_inputs(M, V, K, dt, loss_scale=1.0, device="cpu"):
    x, w, t = inputs(M, V, K, dt, device=device)
    lse = torch.logsumexp(x @ w.t(), 1).float().double()
    dloss = (R.values(1, M, "f32", 9)[0].abs() + 0.5) * loss_scale / M
    return x, w, t, lse, dloss.float().double().to(device)


@pytest.mark.parametrize("M,V,K", SIZES)
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_backward(M, V, K, dt):
    args = grad_inputs(M, V, K, dt, 1024.0 if dt == "f16" else 1.0)
    check_backward(backward(*args, dt), *args, dt)


@pytest.mark.parametrize("M,V,K", [(5, 300, 128), (70, 600, 64), (300, 513, 128)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_backward_forms(M, V, K, dt):
    """Single outputs, fp32 accumulation, strides and alignment."""
    args = grad_inputs(M, V, K, dt, 64.0)
    dw0 = R.values(V, K, "f32", 30, 2.0)
    for kw in (dict(want="x"), dict(want="w"), dict(wt="f32", beta=0.5, dw0=dw0), dict(wt="f32"), dict(pad=8),
               dict(pad=3, off=1)):
        check_backward(backward(*args, dt, **kw), *args, dt,
                       **{k: v for k, v in kw.items() if k in ("wt", "beta", "dw0", "want")})


@pytest.mark.parametrize("loss_scale", [1e-12, 1.0, 1e20])
def test_fp16_gradients_of_any_size(loss_scale):
    """fp32 weight gradients of fp16 operands are as exact for loss gradients outside fp16's range; zero ones
    give zeros."""
    args = grad_inputs(60, 400, 64, "f16", loss_scale)
    got = backward(*args, "f16", wt="f32", want="w")
    check_backward(got, *args, "f16", wt="f32", want="w")
    zero = (*args[:4], torch.zeros_like(args[4]))
    assert all(bool((v == 0).all()) for v in backward(*zero, "f16"))


def test_gradient_of_ignored_and_invalid_rows():
    """An ignored row adds nothing, whatever its logits hold; an invalid target makes the row's gradient NaN."""
    x, w, t, lse, dloss = grad_inputs(300, 400, 128, "bf16")
    t[7] = IGNORE
    lse[7] = float("nan")
    dx, dw = backward(x, w, t, lse, dloss, "bf16")
    assert bool((dx[7] == 0).all()) and bool(torch.isfinite(dw).all())
    t[9] = 400
    dx, _ = backward(x, w, t, lse, dloss, "bf16")
    assert bool(torch.isnan(dx[9]).all()) and int(torch.isnan(dx).any(1).sum()) == 1
    t[:] = IGNORE
    dx, dw = backward(x, w, t, lse, dloss, "bf16")
    assert bool((dx == 0).all()) and bool((dw == 0).all())


def test_gradients_against_differences():
    """<gradient, v> against central differences of the definition, h = 1e-4."""
    M, V, K, h = 6, 50, 40, 1e-4
    x, w, t = inputs(M, V, K, "f32")
    c = R.values(1, M, "f32", 60)[0]
    f = lambda x, w: float((R.xent(x, w, t, IGNORE)[1] * c).sum())
    dx, dw = backward(x, w, t, R.xent(x, w, t, IGNORE)[2], c, "f32")
    for i, (grad, at) in enumerate(((dx, x), (dw, w))):
        v = R.values(*at.shape, "f32", 61 + i)
        lo, hi = [x, w], [x, w]
        hi[i], lo[i] = at + h * v, at - h * v
        diff = (f(*hi) - f(*lo)) / (2 * h)
        assert abs(float((grad * v).sum()) - diff) <= 2e-5 * float((grad * v).abs().sum()) + 1e-6


def test_empty_batch():
    dw = R.Buf(20, 30, "f32", 2, values=torch.full((20, 30), 3.0))
    assert vk.linear_xent_async(0, 0, 20, 30, None, 30, None, 30, None, IGNORE, None, None) == vk.OK
    for beta, want in ((0.5, 1.5), (0.0, 0.0)):
        vk.linear_xent_backward_async(0, 0, 20, 30, None, 30, None, 30, None, IGNORE, None, None, None, 30, dw.ptr,
                                      dw.ld, 0, beta, stream=stream())
        assert bool((dw.get() == want).all())
    dw.check_around()


@pytest.mark.parametrize("K", [16, 128])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_pieces(dt, K):
    """More rows than one piece of the vocabulary's logits (K = 16) or of their gradient holds: several pieces, a
    ragged last one.  References in float64 on the GPU."""
    M, V = 70000, 1000 if K == 16 else 4101
    x, w, t = inputs(M, V, K, dt, device="cuda")
    check_forward(forward(x, w, t, dt), x, w, t)
    lse = torch.logsumexp(x @ w.t(), 1).float().double()
    args = (x, w, t, lse, torch.full((M,), 1.0 / 64, dtype=torch.float64, device="cuda"))
    check_backward(backward(*args, dt), *args, dt)


# work that is worth copies: K in no 16-byte units, classes and rows in no whole steps, together and alone
LARGE = [(300, 2003, 1001), (1000, 10003, 512), (1025, 40000, 520), (640, 8205, 1024)]


@pytest.mark.parametrize("M,V,K", LARGE)
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_padded_operands(M, V, K, dt):
    args = grad_inputs(M, V, K, dt, 64.0, device="cuda")
    x, w, t = args[:3]
    check_forward(forward(x, w, t, dt), x, w, t)
    assert (vk.last_kernel() == vk.KERNEL_FUSED) == (M > 300 or dt != "f32")   # few tiles: joined
    dw0 = R.values(V, K, "f32", 30, 2.0).cuda()
    for kw in (dict(), dict(want="x"), dict(want="w"), dict(wt="f32", beta=0.5, dw0=dw0), dict(pad=3, off=1)):
        check_backward(backward(*args, dt, **kw), *args, dt,
                       **{k: v for k, v in kw.items() if k in ("wt", "beta", "dw0", "want")})


def test_offsets_past_32_bits():
    """A weight of 2.5e9 elements: statistics and gradients reach its last classes."""
    M, V, K = 65, 600000, 4096
    x = torch.randn(M, K, device="cuda").bfloat16()
    w = torch.randn(V, K, device="cuda", dtype=torch.bfloat16) * 0.03
    t = V - 1 - torch.arange(M, device="cuda")
    loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    vk.linear_xent_async(vk.DT_BF16, M, V, K, x.data_ptr(), K, w.data_ptr(), K, t.data_ptr(), IGNORE, loss.data_ptr(),
                         lse.data_ptr(), stream=stream())
    z = x.float() @ w.float().t()
    want = torch.logsumexp(z.double(), 1)
    R.close(lse.double(), want, 1e-4 * want.abs(), "lse")
    R.close(loss.double(), want - z.gather(1, t[:, None])[:, 0], 1e-3 * want.abs(), "loss")
    dloss = torch.ones(M, device="cuda")
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    vk.linear_xent_backward_async(vk.DT_BF16, M, V, K, x.data_ptr(), K, w.data_ptr(), K, t.data_ptr(), IGNORE,
                                  lse.data_ptr(), dloss.data_ptr(), dx.data_ptr(), K, dw.data_ptr(), K, vk.DT_BF16, 0.0,
                                  stream=stream())
    d = torch.exp(z - lse[:, None])
    d[torch.arange(M, device="cuda"), t] -= 1
    tail = (d[:, V - 200:].double().t() @ x.double())
    R.close(dw[V - 200:].double(), tail, 2.0 ** -7 * (d[:, V - 200:].abs().double().t() @ x.abs().double()), "dw")
    ref = (d @ w.float()).double()
    R.close(dx.double(), ref, 2.0 ** -7 * ref.abs() + 1e-3 * ref.abs().max(), "dx")


def test_workspace_under_capture():
    """Needs a workspace: refused while the stream captures, nothing written."""
    x, w = (torch.randn(r, 128, device="cuda").half() for r in (300, 400))
    t, loss, lse = torch.zeros(300, dtype=torch.int64, device="cuda"), *torch.zeros(2, 300, device="cuda")
    y = torch.zeros(4, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y += 1
        st = vk.linear_xent_async(vk.DT_F16, 300, 400, 128, x.data_ptr(), 128, w.data_ptr(), 128, t.data_ptr(), IGNORE,
                                  loss.data_ptr(), lse.data_ptr(), stream=stream(), check=False)
    assert st == vk.ERR_INIT
    g.replay()
    torch.cuda.synchronize()
    assert not lse.any()
