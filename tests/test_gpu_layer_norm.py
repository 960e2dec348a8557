"""vkblas_layer_norm_async and its backward pass against the definition in float64: every row map (one, four
and sixteen waves a row, rows read again), types, strides, alignments, constant rows, NaN and infinities."""
import pytest
import torch

import nn_ref as R
import vkblas_amd as vk

pytestmark = pytest.mark.gpu
EPS = 1e-5


def stream():
    return torch.cuda.current_stream().cuda_stream


def forward(x, w, b, dt, wt, pad=0, off=0, inplace=False, eps=EPS):
    M, N = x.shape
    bx = R.Buf(M, N, dt, pad, off, x)
    by = bx if inplace else R.Buf(M, N, dt, pad, off)
    bw, bb = (R.Buf(1, N, wt, 0, off, v[None]) if v is not None else None for v in (w, b))
    mean, rstd = R.Buf(1, M, "f32"), R.Buf(1, M, "f32")
    vk.layer_norm_async(R.ENGINE[dt], R.ENGINE[wt], M, N, bx.ptr, bx.ld, bw and bw.ptr, bb and bb.ptr, eps, by.ptr,
                        by.ld, mean.ptr, rstd.ptr, stream=stream())
    for o in (by, mean, rstd):
        o.check_around()
    return by.get(), mean.get()[0], rstd.get()[0]


def check_forward(got, x, w, b, dt, eps=EPS):
    M, N = x.shape
    one, zero = torch.ones(N, dtype=torch.float64), torch.zeros(N, dtype=torch.float64)
    w, b = one if w is None else w, zero if b is None else b
    y, mean, rstd = R.norm(x, w, b, eps)
    # a sum of N fp32 terms in a tree of depth <= 32: 32 e of the terms' sum of magnitudes
    emean = 32 * R.E * x.abs().mean(1) + R.E * mean.abs()
    R.close(got[1], mean, emean, "mean")
    # the squares' sum: 40 e relative, and twice the mean's error times the mean deviation, which sums to 0 but
    # for the rounding of the deviations; the mean's error enters squared
    erstd = rstd * (40 * R.E + (emean * rstd) ** 2 + 4 * R.E * x.abs().mean(1) * rstd)
    R.close(got[2], rstd, erstd, "rstd")
    err = (w.abs() * rstd[:, None] * (emean[:, None] + 4 * R.E * (x.abs() + mean.abs()[:, None])) +
           ((x - mean[:, None]) * w).abs() * erstd[:, None] + 4 * R.E * (y.abs() + b.abs()))
    R.close(got[0], y, R.rounded(y, dt, err), "y")


SIZES = [(1, 1), (3, 7), (3, 8), (5, 9), (2, 15), (5, 64), (2, 511), (9, 512), (4, 513), (6, 1000), (3, 1024), (2, 1025), (5, 2047), (2, 2048),
         (3, 4096), (2, 4097), (3, 5003), (2, 8192), (2, 9001), (1, 16384), (2, 16385), (2, 40000), (1500, 96),
         (1024, 200), (1025, 200), (512, 4500), (513, 4500), (4500, 40), (1100, 1100), (300, 5000)]


@pytest.mark.parametrize("M,N", SIZES)
@pytest.mark.parametrize("dt,wt", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
def test_forward(M, N, dt, wt):
    x = R.values(M, N, dt, 1, 2.0) + 0.5
    x = x.to(R.TORCH[dt]).double()
    w, b = 1 + 0.2 * R.values(1, N, wt, 2)[0], R.values(1, N, wt, 3)[0]
    w = w.to(R.TORCH[wt]).double()
    check_forward(forward(x, w, b, dt, wt), x, w, b, dt)
    assert vk.last_kernel() == (vk.KERNEL_NORM_LONG if N > 16384 or N < 8 else vk.KERNEL_NORM)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,N", [(3, 100), (5, 777), (4, 3000), (3, 6000), (2, 20000)])
def test_strides_alignment_inplace_and_no_params(dt, M, N):
    x = R.values(M, N, dt, 4)
    w, b = R.values(1, N, dt, 5)[0], R.values(1, N, dt, 6)[0]
    for pad, off, inplace in ((1, 1, False), (8, 0, False), (5, 3, True)):
        check_forward(forward(x, w, b, dt, dt, pad, off, inplace), x, w, b, dt)
    check_forward(forward(x, None, None, dt, dt), x, None, None, dt)
    check_forward(forward(x, w, None, dt, dt), x, w, None, dt)


@pytest.mark.parametrize("N", [40, 700, 3000, 9000, 17000])
def test_large_mean_and_constant_rows(N):
    """A mean 1000 times the deviation loses nothing to cancellation; a constant row has rstd = eps^-1/2."""
    x = (R.values(4, N, "f32", 7) + 1000.0).float().double()
    check_forward(forward(x, None, None, "f32", "f32"), x, None, None, "f32")
    c = torch.full((2, N), 0.5, dtype=torch.float64)
    y, mean, rstd = forward(c, None, None, "f32", "f32")
    assert bool((y == 0).all()) and bool((mean == 0.5).all())
    assert torch.allclose(rstd, torch.full_like(rstd, EPS ** -0.5), rtol=1e-6)


@pytest.mark.parametrize("N", [40, 700, 3000, 9000, 17000])
def test_nan_and_inf_stay_in_their_rows(N):
    x = R.values(5, N, "f32", 8)
    x[1, N // 2], x[3, 0] = float("nan"), float("inf")
    y, _, _ = forward(x, None, None, "f32", "f32")
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[3]).all())
    assert bool(torch.isfinite(y[[0, 2, 4]]).all())


def backward(dy, x, w, mean, rstd, dt, wt, gt, pad=0, off=0, beta=0.0, dw0=None, want="xwb", alias=None):
    M, N = x.shape
    bd, bx = R.Buf(M, N, dt, pad, off, dy), R.Buf(M, N, dt, pad, off, x)
    bw = R.Buf(1, N, wt, 0, off, w[None]) if w is not None else None
    bm, br = R.Buf(1, M, "f32", values=mean[None]), R.Buf(1, M, "f32", values=rstd[None])
    dx = {"dy": bd, "x": bx, None: None}[alias] or R.Buf(M, N, dt, pad, off)
    dw, db = (R.Buf(1, N, gt, 0, off, dw0) for _ in range(2))
    vk.layer_norm_backward_async(R.ENGINE[dt], R.ENGINE[wt], M, N, bd.ptr, bd.ld, bx.ptr, bx.ld, bw and bw.ptr, bm.ptr,
                                 br.ptr, dx.ptr if "x" in want else None, dx.ld, dw.ptr if "w" in want else None,
                                 db.ptr if "b" in want else None, R.ENGINE[gt], beta, stream=stream())
    for o in (dx, dw, db):
        o.check_around()
    return dx.get(), dw.get()[0], db.get()[0]


def check_backward(got, dy, x, w, mean, rstd, dt, gt, beta=0.0, dw0=None, want="xwb"):
    M, N = x.shape
    w1 = torch.ones(N, dtype=torch.float64) if w is None else w
    dx, dw, db = R.norm_grad(dy, x, w1, mean, rstd)
    r = rstd[:, None]
    xh = (x - mean[:, None]) * r
    exh = 4 * R.E * (xh.abs() + (x.abs() + mean.abs()[:, None]) * r)
    g = (dy * w1).abs()
    # row sums in trees of depth <= 48
    e1 = 48 * R.E * g.mean(1, keepdim=True)
    e2 = 48 * R.E * (g * xh.abs()).mean(1, keepdim=True) + (g * exh).mean(1, keepdim=True)
    s2 = (dy * w1 * xh).mean(1, keepdim=True).abs()
    ex = r * (8 * R.E * (g + g.mean(1, keepdim=True) + xh.abs() * s2) + e1 + xh.abs() * e2 + exh * s2)
    if "x" in want:
        R.close(got[0], dx, R.rounded(dx, dt, ex), "dx")
    # column sums of M terms: at most M + 8 roundings deep
    old = torch.zeros(N, dtype=torch.float64) if dw0 is None else dw0[0]
    for k, ref, terms, more in ((1, dw, dy * xh, (dy.abs() * exh).sum(0)), (2, db, dy, 0.0)):
        if "xwb"[k] in want:
            ref = ref + beta * old
            R.close(got[k], ref, R.rounded(ref, gt, (M + 8) * R.E * (terms.abs().sum(0) + (beta * old).abs()) + more),
                    "dw" if k == 1 else "db")


@pytest.mark.parametrize("M,N", SIZES)
@pytest.mark.parametrize("dt,wt,gt", [("f32", "f32", "f32"), ("f16", "f16", "f16"), ("bf16", "f32", "f32"),
                                      ("bf16", "bf16", "f32")])
def test_backward(M, N, dt, wt, gt):
    x, dy = R.values(M, N, dt, 11, 2.0), R.values(M, N, dt, 12, 0.1)
    w = R.values(1, N, wt, 13)[0]
    _, mean, rstd = R.norm(x, w, w, EPS)
    mean, rstd = mean.float().double(), rstd.float().double()
    got = backward(dy, x, w, mean, rstd, dt, wt, gt)
    check_backward(got, dy, x, w, mean, rstd, dt, gt)
    again = backward(dy, x, w, mean, rstd, dt, wt, gt)
    assert all(torch.equal(a, b) for a, b in zip(got, again)), "equal calls differ"


# rows and columns on both sides of where a workgroup takes 16 columns and where 32, last columns ragged
@pytest.mark.parametrize("M,N", [(256, 33), (257, 9), (300, 17), (511, 2047), (512, 2049), (700, 1000), (1003, 997),
                                 (1024, 1024), (1024, 1040)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_backward_of_columns(dt, M, N):
    x, dy, w = R.values(M, N, dt, 24), R.values(M, N, dt, 25), R.values(1, N, dt, 26)[0]
    _, mean, rstd = R.norm(x, w, w, EPS)
    mean, rstd = mean.float().double(), rstd.float().double()
    dw0 = R.values(1, N, "f32", 27, 3.0)
    for kw in (dict(), dict(pad=1, off=1, want="wb"), dict(beta=0.5, dw0=dw0)):
        got = backward(dy, x, w, mean, rstd, dt, dt, "f32", **kw)
        check_backward(got, dy, x, w, mean, rstd, dt, "f32",
                       **{k: v for k, v in kw.items() if k in ("beta", "dw0", "want")})


@pytest.mark.parametrize("N", [1100, 2100, 3000, 5000, 8000, 9000])
def test_equal_calls_of_rows_of_several_waves(N):
    """Each element of dx is one thread's: no two write it, so equal calls give equal bits, time after time."""
    M = 300
    x, dy, w = (torch.randn(r, N, device="cuda").half() for r in (M, M, 1))
    mean, rstd = x.float().mean(1), 1 / x.float().std(1)
    outs = []
    for _ in range(20):
        dx, dw, db = torch.empty_like(x), *torch.empty(2, N, device="cuda", dtype=torch.half)
        vk.layer_norm_backward_async(vk.DT_F16, vk.DT_F16, M, N, dy.data_ptr(), N, x.data_ptr(), N, w.data_ptr(),
                                     mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), N, dw.data_ptr(), db.data_ptr(),
                                     vk.DT_F16, 0.0, stream=stream())
        outs.append((dx, dw, db))
    assert all(torch.equal(a, b) for o in outs[1:] for a, b in zip(o, outs[0]))


@pytest.mark.parametrize("M,N", [(3, 100), (70, 777), (4, 3000), (3, 6000), (2, 20000)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_backward_forms(dt, M, N):
    """Strides, alignment, dx in the place of dy or x, accumulation, single outputs, no weight."""
    x, dy, w = R.values(M, N, dt, 14), R.values(M, N, dt, 15), R.values(1, N, dt, 16)[0]
    _, mean, rstd = R.norm(x, w, w, EPS)
    mean, rstd = mean.float().double(), rstd.float().double()
    dw0 = R.values(1, N, "f32", 17, 3.0)
    for kw in (dict(pad=1, off=1), dict(pad=8, alias="dy"), dict(alias="x"), dict(beta=0.5, dw0=dw0), dict(want="x"),
               dict(want="wb"), dict(want="w"), dict(want="b")):
        got = backward(dy, x, w, mean, rstd, dt, dt, "f32", **kw)
        check_backward(got, dy, x, w, mean, rstd, dt, "f32",
                       **{k: v for k, v in kw.items() if k in ("beta", "dw0", "want")})
    check_backward(backward(dy, x, None, mean, rstd, dt, dt, dt), dy, x, None, mean, rstd, dt, dt)


def test_gradients_against_differences():
    """<gradient, v> against central differences of the definition, h = 1e-4: their error is about h^2 plus
    2^-52 / h, far below the kernel's own bound of 1e-5 of the terms."""
    M, N, h = 6, 130, 1e-4
    x, w, b, c = (R.values(r, N, "f32", s) for r, s in ((M, 21), (1, 22), (1, 23), (M, 24)))
    f = lambda x, w, b: float((R.norm(x, w[0], b[0], EPS)[0] * c).sum())
    _, mean, rstd = R.norm(x, w[0], b[0], EPS)
    dx, dw, db = backward(c, x, w[0], mean, rstd, "f32", "f32", "f32")
    for i, (grad, at) in enumerate(((dx, x), (dw[None], w), (db[None], b))):
        v = R.values(at.shape[0], N, "f32", 30 + i)
        args = [[x, w, b], [x, w, b]]
        args[0][i], args[1][i] = at + h * v, at - h * v
        diff = (f(*args[0]) - f(*args[1])) / (2 * h)
        assert abs(float((grad * v).sum()) - diff) <= 1e-5 * float((grad * v).abs().sum()) + 1e-6


def test_empty_batch():
    dw, db = (R.Buf(1, 50, "f32", values=torch.full((1, 50), 3.0)) for _ in range(2))
    assert vk.layer_norm_async(0, 0, 0, 50, None, 50, None, None, EPS, None, 50) == vk.OK
    for beta, want in ((0.5, 1.5), (0.0, 0.0)):
        vk.layer_norm_backward_async(0, 0, 0, 50, None, 50, None, 50, None, None, None, None, 50, dw.ptr, db.ptr, 0,
                                     beta, stream=stream())
        assert bool((dw.get() == want).all()) and bool((db.get() == want).all())
    dw.check_around()


def test_side_stream():
    """On a stream of the caller's, ordered after its own work there."""
    s = torch.cuda.Stream()
    x = R.values(64, 3000, "f32", 40)
    with torch.cuda.stream(s):
        a = torch.zeros(64, 3000, device="cuda")
        a += x.float().cuda()
        y, mean, rstd = torch.empty_like(a), torch.empty(64, device="cuda"), torch.empty(64, device="cuda")
        vk.layer_norm_async(0, 0, 64, 3000, a.data_ptr(), 3000, None, None, EPS, y.data_ptr(), 3000, mean.data_ptr(),
                            rstd.data_ptr(), stream=s.cuda_stream)
        z = y * 2
    s.synchronize()
    check_forward((z.cpu().double() / 2, mean.cpu().double(), rstd.cpu().double()), x, None, None, "f32")


def test_offsets_past_32_bits():
    """2.2e9 elements: the last rows and the sums over all of them."""
    M, N = 140000, 16000
    x = torch.randn(M, N, device="cuda", dtype=torch.bfloat16)
    y = torch.empty_like(x)
    mean, rstd = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    vk.layer_norm_async(vk.DT_BF16, 0, M, N, x.data_ptr(), N, None, None, EPS, y.data_ptr(), N, mean.data_ptr(),
                        rstd.data_ptr(), stream=stream())
    end = slice(M - 3, M)
    check_forward([v[end].double().cpu() for v in (y, mean, rstd)], x[end].double().cpu(), None, None, "bf16")
    dw, db = torch.empty(N, device="cuda"), torch.empty(N, device="cuda")
    dx = torch.empty_like(x)
    vk.layer_norm_backward_async(vk.DT_BF16, 0, M, N, y.data_ptr(), N, x.data_ptr(), N, None, mean.data_ptr(),
                                 rstd.data_ptr(), dx.data_ptr(), N, dw.data_ptr(), db.data_ptr(), 0, 0.0,
                                 stream=stream())
    args = [v[end].double().cpu() for v in (y, x)] + [None] + [v[end].double().cpu() for v in (mean, rstd)]
    check_backward((dx[end].double().cpu(), None, None), *args, "bf16", "f32", want="x")
    cols = slice(N - 64, N)
    d = y[:, cols].double()
    ref = (d * (x[:, cols].double() - mean[:, None]) * rstd[:, None]).sum(0)
    assert torch.allclose(dw[cols].double(), ref, rtol=1e-4) and torch.allclose(db[cols].double(), d.sum(0), atol=0.5)


def test_graph_capture():
    """The forward pass needs no workspace: captured, replayed with eager work between, equal each time; the
    backward pass's sums need one: refused, nothing launched."""
    x = torch.randn(1100, 3000, device="cuda")
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    mean, rstd, dw = torch.zeros(1100, device="cuda"), torch.zeros(1100, device="cuda"), torch.zeros(3000, device="cuda")

    def call():
        vk.layer_norm_async(0, 0, 1100, 3000, x.data_ptr(), 3000, None, None, EPS, y.data_ptr(), 3000, mean.data_ptr(),
                            rstd.data_ptr(), stream=stream())
    call()
    torch.cuda.synchronize()
    eager = y.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
        st = vk.layer_norm_backward_async(0, 0, 1100, 3000, x.data_ptr(), 3000, x.data_ptr(), 3000, None,
                                          mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), 3000, dw.data_ptr(), None, 0,
                                          stream=stream(), check=False)
    assert st == vk.ERR_INIT
    for _ in range(3):
        y.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
        call()
    assert not dx.any() and not dw.any()
