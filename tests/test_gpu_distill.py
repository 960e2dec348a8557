"""vkblas_linear_distill_async and its backward pass against the definition in float64: types, one row to several
tiles and pieces, temperatures, ragged and empty rows, classes that occur twice or do not exist, entries without
probability, infinities and NaN where nothing counts, strides, gradients against differences."""
import pytest
import torch

import nn_ref as R
import train_ref as D
import vkblas_amd as vk

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


class Top:
    """The teacher's entries on the GPU, rows of ld elements, with what may not be read around them."""

    def __init__(self, top, t, tt, pad=0):
        M, n = top.shape
        self.top, self.t = torch.full((M, n + pad), 2 ** 40, device="cuda"), R.Buf(M, n, tt, pad, 0, t)
        self.top[:, :n] = top
        self.ld = n + pad


def inputs(M, V, K, n, dt, tt="f32", seed=1, scale=2.0, device="cpu"):
    x, w = R.values(M, K, dt, seed), R.values(V, K, dt, seed + 1, scale * K ** -0.5)
    g = torch.Generator().manual_seed(seed + 2)
    top = torch.randint(0, V, (M, n), generator=g)      # classes occur twice where n is near V
    top[0, 0], top[-1, -1] = V - 1, 0
    top[1::5, n // 2:] = -1
    top[3::11] = -7
    t = R.values(M, n, tt, seed + 3, 3.0)
    t[top < 0] = float("nan")
    t[2::9, : n // 3] = float("-inf")
    return [v.to(device) for v in (x, w, top, t)]


def forward(x, w, top, t, temp, dt, tt="f32", pad=0, off=0):
    M, K = x.shape
    V, n = w.shape[0], top.shape[1]
    bx, bw, e = R.Buf(M, K, dt, pad, off, x), R.Buf(V, K, dt, pad, off, w), Top(top, t, tt, pad)
    loss, lse, zt = R.Buf(1, M, "f32"), R.Buf(1, M, "f32"), R.Buf(M, n, "f32")
    vk.linear_distill_async(R.ENGINE[dt], M, V, K, bx.ptr, bx.ld, bw.ptr, bw.ld, n, e.top.data_ptr(), e.ld,
                            R.ENGINE[tt], e.t.ptr, e.t.ld, temp, loss.ptr, lse.ptr, zt.ptr, stream=stream())
    for b in (loss, lse, zt):
        b.check_around()
    return loss.get()[0], lse.get()[0], zt.get()


def check_forward(got, x, w, top, t, temp):
    names = ("loss", "lse", "z_top")
    for g, (ref, bound), name in zip(got, D.distill(x, w, top, t, temp), names):
        g = g.to(ref.device)
        assert torch.equal(torch.isnan(g), torch.isnan(ref)), name
        there = ~torch.isnan(ref)
        R.close(g[there], ref[there], bound[there], name)


# rows, classes, K, entries: decode-sized, joined and fused products, 16-byte units and not
SIZES = [(1, 1, 1, 1), (1, 5, 8, 3), (2, 77, 9, 10), (4, 3000, 515, 64), (8, 20000, 520, 5), (9, 513, 1031, 70),
         (16, 999, 700, 1), (64, 515, 128, 33), (65, 1000, 100, 300), (128, 256, 128, 1024), (200, 300, 64, 7),
         (257, 1001, 128, 65), (300, 700, 320, 20), (511, 130, 128, 13), (17, 17003, 264, 40)]
FORMS = [("f32", "f32", 1.0), ("f16", "f32", 2.0), ("bf16", "bf16", 0.75), ("f16", "f16", 8.0)]


@pytest.mark.parametrize("M,V,K,n", SIZES)
@pytest.mark.parametrize("dt,tt,temp", FORMS)
def test_forward(M, V, K, n, dt, tt, temp):
    args = inputs(M, V, K, n, dt, tt)
    check_forward(forward(*args, temp, dt, tt), *args, temp)


@pytest.mark.parametrize("M,V,K,n", [(5, 300, 128, 9), (300, 513, 128, 17)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,off", [(8, 0), (4, 4), (1, 0), (3, 1)])
def test_strides_and_alignment(M, V, K, n, dt, pad, off):
    args = inputs(M, V, K, n, dt, dt)
    check_forward(forward(*args, 1.5, dt, dt, pad, off), *args, 1.5)


def grad_inputs(M, V, K, n, dt, temp, tt="f32", loss_scale=1.0, device="cpu"):
    x, w, top, t = inputs(M, V, K, n, dt, tt, device=device)
    lse = torch.logsumexp(x @ w.t() / temp, 1).float().double()
    dloss = ((R.values(1, M, "f32", 9)[0].abs() + 0.5) * loss_scale / M).float().double().to(device)
    return x, w, top, t, lse, dloss


def z_top(x, w, top):
    """As the forward pass leaves it, rounded from float64."""
    V = w.shape[0]
    z = (x @ w.t()).gather(1, top.clamp(0, V - 1))
    z[top >= V] = float("nan")
    return torch.where(top < 0, torch.zeros_like(z), z).float().double()


def backward(x, w, top, t, lse, dloss, temp, dt, tt="f32", wt=None, pad=0, off=0, beta=0.0, dw0=None, want="xw"):
    M, K = x.shape
    V, n, wt = w.shape[0], top.shape[1], wt or dt
    bx, bw, e = R.Buf(M, K, dt, pad, off, x), R.Buf(V, K, dt, pad, off, w), Top(top, t, tt, pad)
    bl, bd = R.Buf(1, M, "f32", values=lse[None]), R.Buf(1, M, "f32", values=dloss[None])
    zt = R.Buf(M, n, "f32", values=z_top(x, w, top))
    dx, dw = R.Buf(M, K, dt, pad, off), R.Buf(V, K, wt, pad, off, dw0)
    vk.linear_distill_backward_async(R.ENGINE[dt], M, V, K, bx.ptr, bx.ld, bw.ptr, bw.ld, n, e.top.data_ptr(), e.ld,
                                     R.ENGINE[tt], e.t.ptr, e.t.ld, temp, bl.ptr, zt.ptr, bd.ptr,
                                     dx.ptr if "x" in want else None, dx.ld, dw.ptr if "w" in want else None, dw.ld,
                                     R.ENGINE[wt], beta, stream=stream())
    dx.check_around()
    dw.check_around()
    return dx.get(), dw.get()


def check_backward(got, x, w, top, t, lse, dloss, temp, dt, wt=None, beta=0.0, dw0=None, want="xw"):
    wt = wt or dt
    want_grads = D.distill_grad(x, w, top, t, temp, lse, dloss, dt, beta, dw0)
    for g, (ref, err), name, ty in zip(got, want_grads, "xw", (dt, wt)):
        if name in want:
            R.close(g, ref, R.rounded(ref, ty, err), "d" + name)


@pytest.mark.parametrize("M,V,K,n", SIZES)
@pytest.mark.parametrize("dt,tt,temp", FORMS)
def test_backward(M, V, K, n, dt, tt, temp):
    args = grad_inputs(M, V, K, n, dt, temp, tt, 1024.0 if dt == "f16" else 1.0)
    check_backward(backward(*args, temp, dt, tt), *args, temp, dt)


@pytest.mark.parametrize("M,V,K,n", [(5, 300, 128, 9), (70, 600, 64, 30), (300, 513, 128, 17)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_backward_forms(M, V, K, n, dt):
    """Single outputs, fp32 accumulation, strides and alignment."""
    args = grad_inputs(M, V, K, n, dt, 1.25, loss_scale=64.0)
    dw0 = R.values(V, K, "f32", 30, 2.0)
    for kw in (dict(want="x"), dict(want="w"), dict(wt="f32", beta=0.5, dw0=dw0), dict(wt="f32"), dict(pad=8),
               dict(pad=3, off=1)):
        check_backward(backward(*args, 1.25, dt, **kw), *args, 1.25, dt,
                       **{k: v for k, v in kw.items() if k in ("wt", "beta", "dw0", "want")})


@pytest.mark.parametrize("M,V,K,n", [(300, 2003, 1001, 40), (1025, 40000, 520, 64), (1000, 10003, 512, 9)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_large(M, V, K, n, dt):
    """Work that is worth copies, a tail of classes, the scale found by its own kernel (1025 rows)."""
    args = grad_inputs(M, V, K, n, dt, 2.0, loss_scale=64.0, device="cuda")
    check_forward(forward(*args[:4], 2.0, dt), *args[:4], 2.0)
    check_backward(backward(*args, 2.0, dt), *args, 2.0, dt)


# enough entries that the tiles of the logits leave those at the entries: tiles of 128 (in four LDS stages and two) and
# of 256, an odd K, more slices than 1023, more rows than workgroups
@pytest.mark.parametrize("M,V,K,n,dt", [(1100, 1000, 1024, 480, "bf16"), (1100, 1000, 1027, 480, "f16"),
                                        (1100, 6001, 1024, 480, "bf16"), (600, 20000, 2048, 448, "f16"),
                                        (515, 140001, 1024, 1024, "bf16"), (70001, 600, 520, 16, "bf16"),
                                        (1050, 129, 1024, 500, "f16")])
@pytest.mark.parametrize("pad", [0, 5])
def test_many_entries(M, V, K, n, dt, pad):
    x, w, top, t = inputs(M, V, K, n, dt, device="cuda")
    top[7, 3], top[8, n - 1], top[9] = V, 2 ** 40, 5        # two bad rows, and one of one class
    t[9] = t[9].nan_to_num(0.5, 0.5, 0.5)
    check_forward(forward(x, w, top, t, 1.5, dt, pad=pad), x, w, top, t, 1.5)


@pytest.mark.parametrize("K", [16, 128])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_pieces(dt, K):
    """More rows than one piece of the vocabulary's logits or of their gradient holds: entries in each piece."""
    M, V, n = 70000, 1000 if K == 16 else 4101, 6
    args = grad_inputs(M, V, K, n, dt, 1.5, loss_scale=64.0, device="cuda")
    check_forward(forward(*args[:4], 1.5, dt), *args[:4], 1.5)
    check_backward(backward(*args, 1.5, dt), *args, 1.5, dt)


@pytest.mark.parametrize("M,V", [(12, 60), (300, 700)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_rows_that_do_not_count_and_bad_classes(M, V, dt):
    """No entry, or none with a probability: loss 0 and no gradient whatever dloss and lse hold.  A class past V: NaN
    in its row alone."""
    K, n = 128, 12
    x, w, top, t, lse, dloss = grad_inputs(M, V, K, n, dt, 1.0)
    top[4], top[5] = -1, torch.arange(n)
    t[5] = float("-inf")
    got = forward(x, w, top, t, 1.0, dt)
    assert float(got[0][4]) == 0.0 and float(got[0][5]) == 0.0
    check_forward(got, x, w, top, t, 1.0)
    dloss[4], dloss[5], lse[4] = float("nan"), float("inf"), float("nan")
    dx, dw = backward(x, w, top, t, lse, dloss, 1.0, dt)
    assert bool((dx[4:6] == 0).all()) and bool(torch.isfinite(dw).all())
    clean = dloss.clone(), lse.clone()
    clean[0][4:6], clean[1][4] = 0.0, 0.0
    check_backward((dx, dw), x, w, top, t, clean[1], clean[0], 1.0, dt)
    for bad, logit in ((V, 0.0), (2 ** 40, float("-inf")), (2 ** 31, 1.0)):
        top[6], t[6] = torch.arange(n), 1.0
        top[6, 3], t[6, 3] = bad, logit
        got = forward(x, w, top, t, 1.0, dt)
        assert bool(torch.isnan(got[0][6])) and int(torch.isnan(got[0]).sum()) == 1
        assert bool(torch.isnan(got[2][6, 3])) and int(torch.isnan(got[2]).sum()) == 1
        dx, _ = backward(x, w, top, t, lse, dloss, 1.0, dt)
        assert bool(torch.isnan(dx[6]).all()) and int(torch.isnan(dx).any(1).sum()) == 1
    top[6] = torch.arange(n)
    t[6, 3] = float("nan")
    got = forward(x, w, top, t, 1.0, dt)
    assert bool(torch.isnan(got[0][6])) and int(torch.isnan(got[0]).sum()) == 1
    t[6] = float("nan")
    assert bool(torch.isnan(forward(x, w, top, t, 1.0, dt)[0][6]))


def test_extreme_logits():
    """Teacher's logits of the type's lowest value and of +-1000, the student's too: nothing overflows; a student
    without a class that the teacher names has an infinite loss."""
    M, V, K, n = 6, 300, 64, 5
    x, w = torch.zeros(M, K, dtype=torch.float64), torch.zeros(V, K, dtype=torch.float64)
    x[:, 0] = 1.0
    w[:, 0] = torch.linspace(-1000, 1000, V, dtype=torch.float64).float().double()
    top = torch.tensor([[299, 0, 10, 298, 5]]).repeat(M, 1)
    t = torch.tensor([[1000.0, -1000.0, 999.0, torch.finfo(torch.float32).min, -torch.inf]]).double().repeat(M, 1)
    check_forward(forward(x, w, top, t, 1.0, "f32"), x, w, top, t, 1.0)
    check_forward(forward(x, w, top, t, 4.0, "f32"), x, w, top, t, 4.0)
    w[0, 0] = float("-inf")
    t[:] = 1.0
    loss, lse, zt = forward(x, w, top, t, 1.0, "f32")
    assert bool((loss == float("inf")).all()) and bool(torch.isfinite(lse).all())
    assert bool((zt[:, 1] == -float("inf")).all())


@pytest.mark.parametrize("tt,dt", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("temp", [0.25, 1.0])
def test_teachers_lowest_values_over_a_small_temperature(tt, dt, temp):
    """Logits that leave the type's range once they are over the temperature count by their differences, as others of
    the same differences do, in both passes."""
    M, V, K, n = 9, 300, 64, 6
    x, w, top, t, lse, dloss = grad_inputs(M, V, K, n, dt, temp, tt)
    top, top[5, 2] = torch.arange(7, 7 + n).repeat(M, 1), -1
    high = torch.finfo(R.TORCH[tt]).max
    results = []
    for level in (0.0, -high, high):
        t = torch.full((M, n), level, dtype=torch.float64)
        t[1::2, 3] = -torch.inf if level <= 0.0 else -high
        results.append((*forward(x, w, top, t, temp, dt, tt),
                        *backward(x, w, top, t, lse, dloss, temp, dt, tt)))
        assert all(bool(torch.isfinite(r).all()) for r in results[-1])
        assert all(torch.equal(a, b) for a, b in zip(results[-1], results[0]))


@pytest.mark.parametrize("loss_scale", [1e-12, 1.0, 1e20])
def test_fp16_gradients_of_any_size(loss_scale):
    args = grad_inputs(60, 400, 64, 20, "f16", 4.0, loss_scale=loss_scale)
    check_backward(backward(*args, 4.0, "f16", wt="f32", want="w"), *args, 4.0, "f16", wt="f32", want="w")


@pytest.mark.parametrize("temp", [0.5, 1.0, 3.0])
def test_gradients_against_differences(temp):
    """<gradient, v> against central differences of the definition, h = 1e-4."""
    M, V, K, n, h = 7, 50, 40, 9, 1e-4
    x, w, top, t = inputs(M, V, K, n, "f32")
    c = R.values(1, M, "f32", 60)[0]
    f = lambda x, w: float((D.distill(x, w, top, t, temp)[0][0] * c).sum())
    lse = D.distill(x, w, top, t, temp)[1][0]
    dx, dw = backward(x, w, top, t, lse, c, temp, "f32")
    for i, (grad, at) in enumerate(((dx, x), (dw, w))):
        v = R.values(*at.shape, "f32", 61 + i)
        lo, hi = [x, w], [x, w]
        hi[i], lo[i] = at + h * v, at - h * v
        diff = (f(*hi) - f(*lo)) / (2 * h)
        # differences: third derivatives of the loss, bounded by those of log-sum-exp at 1 / temp, times h^2 / 6 |v|^3
        assert abs(float((grad * v).sum()) - diff) <= 2e-5 * float((grad * v).abs().sum()) + 1e-5


def test_equal_calls_give_equal_bits():
    args = grad_inputs(300, 1003, 128, 30, "bf16", 2.0)
    first = forward(*args[:4], 2.0, "bf16"), backward(*args, 2.0, "bf16")
    for _ in range(3):
        again = forward(*args[:4], 2.0, "bf16"), backward(*args, 2.0, "bf16")
        assert all(torch.equal(a, b) for p, q in zip(first, again) for a, b in zip(p, q))


def test_empty_batch():
    dw = R.Buf(20, 30, "f32", 2, values=torch.full((20, 30), 3.0))
    args = 0, 0, 20, 30, None, 30, None, 30, 4, None, 4, 0, None, 4, 1.0
    assert vk.linear_distill_async(*args, None, None, None) == vk.OK
    for beta, want in ((0.5, 1.5), (0.0, 0.0)):
        vk.linear_distill_backward_async(*args, None, None, None, None, 30, dw.ptr, dw.ld, 0, beta, stream=stream())
        assert bool((dw.get() == want).all())
    dw.check_around()


@pytest.mark.parametrize("M,V,K", [(5, 300, 64), (300, 2000, 128)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("temp", [4.3e-39, 1.84e19])
def test_temperatures_at_the_ends_of_fp32(M, V, K, dt, temp):
    """Equal logits: log V whatever divides them, and a loss that is T^2 log(V / n) with n of the entries at the
    teacher's highest logit, or all: 0 or infinite in fp32.  No NaN in the gradients."""
    x, w = torch.zeros(M, K, dtype=torch.float64), R.values(V, K, dt, 2)
    top, t = torch.arange(6).repeat(M, 1), torch.zeros(M, 6, dtype=torch.float64)
    t[1::2, 2] = -1.0
    loss, lse, zt = forward(x, w, top, t, temp, dt)
    want = torch.full((M,), float(torch.tensor(float(V), dtype=torch.float64).log()), dtype=torch.float64)
    R.close(lse, want, 600 * R.E + R.STEP * (want + 1), "lse")
    assert torch.equal(loss.float(), D.distill(x, w, top, t, temp)[0][0].float()) and bool((zt == 0).all())
    assert float(loss[0]) == (0.0 if temp < 1 else float("inf"))
    dx, dw = backward(x, w, top, t, want, torch.ones(M, dtype=torch.float64), temp, dt, wt="f32")
    assert bool(torch.isfinite(dx).all()) and bool((dw == 0).all())


@pytest.mark.parametrize("n", [3, 256, 257, 1024])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_rows_of_one_class_and_of_two(n, dt):
    """Every entry of a row the same class, and two classes in turn: one of their entries has all of the probability."""
    M, V, K = 40, 700, 64
    x, w, top, t, lse, dloss = grad_inputs(M, V, K, n, dt, 1.5)
    t = t.nan_to_num(0.25, 0.25, 0.25)
    top[::2], top[1::2] = 5, 699
    top[1::2, ::2] = 0
    check_forward(forward(x, w, top, t, 1.5, dt), x, w, top, t, 1.5)
    check_backward(backward(x, w, top, t, lse, dloss, 1.5, dt), x, w, top, t, lse, dloss, 1.5, dt)
