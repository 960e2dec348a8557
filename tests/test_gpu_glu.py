"""vkblas_glu_async and its backward pass against the definition in float64: activations, types, one row to
several tiles, ragged sizes, strides, alignments, accumulation, and values at the ends of the activations."""
import pytest
import torch

import nn_ref as R
import vkblas_amd as vk

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


def forward(x, w, dt, act, keep=True, pad=0, off=0):
    M, K = x.shape
    N = w.shape[0] // 2
    bx, bw = R.Buf(M, K, dt, pad, off, x), R.Buf(2 * N, K, dt, pad, off, w)
    h, gu = R.Buf(M, N, dt, pad, off), R.Buf(M, 2 * N, dt, pad, off)
    vk.glu_async(R.ENGINE[dt], R.ACTS[act], M, N, K, bx.ptr, bx.ld, bw.ptr, bw.ld, h.ptr, h.ld,
                 gu.ptr if keep else None, gu.ld, stream=stream())
    h.check_around()
    gu.check_around()
    return h.get(), gu.get() if keep else None


def check_forward(got, x, w, dt, act):
    N = w.shape[0] // 2
    gu, e = x @ w.t(), R.dot_bound(x, w.t())
    g, u = gu[:, :N], gu[:, N:]
    a = R.act(act, g)
    # the activations' slopes are below 1.13; their own error is STEP of the argument and of the value
    ea = 1.13 * e[:, :N] + R.STEP * (g.abs() + a.abs())
    h = a * u
    R.close(got[0], h, R.rounded(h, dt, ea * (u.abs() + e[:, N:]) + a.abs() * e[:, N:] + R.STEP * h.abs()), "h")
    if got[1] is not None:
        R.close(got[1], gu, R.rounded(gu, dt, e), "gu")


# one row, decode batches, rows of one and of several tiles, whole and ragged
SIZES = [(1, 1, 1), (1, 64, 64), (1, 3, 8), (2, 40, 9), (3, 17, 515), (4, 70, 4100), (5, 33, 2056), (8, 100, 520),
         (9, 51, 1031), (16, 250, 700), (15, 64, 1024), (17, 65, 96), (1, 500, 784), (2, 129, 72), (7, 256, 512), (16, 320, 128), (33, 100, 100),
         (64, 128, 256), (65, 192, 192), (100, 33, 57), (128, 128, 128), (200, 500, 784), (255, 320, 64),
         (256, 128, 128), (257, 129, 128), (300, 200, 320), (511, 264, 192), (130, 72, 1000),
         (9, 2100, 77), (16, 2048, 1031), (17, 2050, 515), (31, 2500, 9), (32, 9001, 130), (1500, 700, 200),
         (1000, 500, 1000), (70, 15, 40), (70, 16, 32)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_forward(M, N, K, dt):
    x, w = R.values(M, K, dt, 1), R.values(2 * N, K, dt, 2, K ** -0.5)
    check_forward(forward(x, w, dt, "silu"), x, w, dt, "silu")
    check_forward(forward(x, w, dt, "silu", keep=False), x, w, dt, "silu")


@pytest.mark.parametrize("M,N,K", [(1, 300, 256), (40, 96, 128), (300, 160, 128), (90, 41, 77)])
@pytest.mark.parametrize("act", list(R.ACTS))
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_activations(M, N, K, act, dt):
    x, w = R.values(M, K, dt, 3), R.values(2 * N, K, dt, 4, 2 * K ** -0.5)
    check_forward(forward(x, w, dt, act), x, w, dt, act)


@pytest.mark.parametrize("M,N,K", [(1, 128, 128), (30, 128, 128), (300, 136, 192)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,off", [(8, 0), (4, 4), (1, 0), (3, 1)])
def test_strides_and_alignment(M, N, K, dt, pad, off):
    x, w = R.values(M, K, dt, 5), R.values(2 * N, K, dt, 6, K ** -0.5)
    check_forward(forward(x, w, dt, "gelu", pad=pad, off=off), x, w, dt, "gelu")


# small calls on tiles with both projections: of 32 rows and of 64, ragged in M and N, K shorter than a step, on
# one, past some, and past every step that is loaded ahead; rows at any alignment, NaN behind them
@pytest.mark.parametrize("M,N", [(6, 500), (33, 17), (64, 250), (97, 31), (400, 123), (1000, 300)])
@pytest.mark.parametrize("K", [3, 16, 40, 129, 500])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_small_tiles(M, N, K, dt):
    x, w = R.values(M, K, dt, 70), R.values(2 * N, K, dt, 71, K ** -0.5)
    for kw in (dict(), dict(keep=False), dict(pad=8), dict(pad=3, off=1)):
        check_forward(forward(x, w, dt, "gelu_tanh", **kw), x, w, dt, "gelu_tanh")
        if M > 32:
            assert vk.last_kernel() == vk.KERNEL_FUSED


def test_small_call_under_capture():
    """A small fp32 call needs no workspace: captured, and each replay equal to the eager result."""
    M, N, K = 200, 77, 130
    x, w = torch.randn(M, K, device="cuda"), torch.randn(2 * N, K, device="cuda")
    h = torch.zeros(M, N, device="cuda")

    def call():
        vk.glu_async(vk.DT_F32, vk.ACT_SILU, M, N, K, x.data_ptr(), K, w.data_ptr(), K, h.data_ptr(), N,
                     stream=stream())
    call()
    torch.cuda.synchronize()
    eager = h.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for _ in range(3):
        h.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, eager)
        call()


# K that ends inside a step, in its first one, on it, and NaN behind each row; few tiles and many, of both sizes
@pytest.mark.parametrize("M,N", [(300, 136), (1100, 3300), (2100, 4400)])
@pytest.mark.parametrize("K", [8, 32, 64, 72, 136, 200, 232, 328])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_ends_of_k(M, N, K, dt):
    x, w = R.values(M, K, dt, 7).cuda(), R.values(2 * N, K, dt, 8, K ** -0.5).cuda()
    check_forward(forward(x, w, dt, "silu", keep=False, pad=8), x, w, dt, "silu")


@pytest.mark.parametrize("act", list(R.ACTS))
@pytest.mark.parametrize("M", [1, 300])
def test_ends_of_the_activations(act, M):
    """Gates of -200 .. 200 (exponentials that overflow and vanish), zeros, and NaN kept to its own outputs."""
    N, K = 128, 128
    x, w = torch.zeros(M, K, dtype=torch.float64), torch.zeros(2 * N, K, dtype=torch.float64)
    x[:, 0], x[:, 1] = 1.0, 2.0
    w[:N, 0] = torch.linspace(-200, 200, N, dtype=torch.float64).float().double()
    w[N:, 1] = 1.5
    check_forward(forward(x, w, "f32", act), x, w, "f32", act)
    w[5, 3] = float("nan")
    h, gu = forward(x, w, "f32", act)
    assert bool(torch.isnan(h[:, 5]).all()) and bool(torch.isnan(gu[:, 5]).all())
    rest = [i for i in range(N) if i != 5]
    assert bool(torch.isfinite(h[:, rest]).all())


def backward(dh, gu, x, w, dt, act, wt=None, pad=0, off=0, beta=0.0, dw0=None, want="xwg", inplace=False):
    M, K = x.shape
    N = w.shape[0] // 2
    wt = wt or dt
    bh, bg = R.Buf(M, N, dt, pad, off, dh), R.Buf(M, 2 * N, dt, pad, off, gu)
    bx, bw = R.Buf(M, K, dt, pad, off, x), R.Buf(2 * N, K, dt, pad, off, w)
    dx, dw = R.Buf(M, K, dt, pad, off), R.Buf(2 * N, K, wt, pad, off, dw0)
    dgu = bg if inplace else R.Buf(M, 2 * N, dt, pad, off)
    vk.glu_backward_async(R.ENGINE[dt], R.ACTS[act], M, N, K, bh.ptr, bh.ld, bg.ptr, bg.ld, bx.ptr, bx.ld, bw.ptr,
                          bw.ld, dgu.ptr if "g" in want else None, dgu.ld, dx.ptr if "x" in want else None, dx.ld,
                          dw.ptr if "w" in want else None, dw.ld, R.ENGINE[wt], beta, stream=stream())
    for o in (dx, dw, dgu):
        o.check_around()
    return dx.get(), dw.get(), dgu.get()


def check_backward(got, dh, gu, x, w, dt, act, wt=None, beta=0.0, dw0=None, want="xwg"):
    N = w.shape[0] // 2
    wt = wt or dt
    g, u = gu[:, :N], gu[:, N:]
    a, da = R.act(act, g), R.act_slope(act, g)
    d = torch.cat((dh * u * da, dh * a), 1)
    # act' has terms of size 1 + |g| exp(-g^2 / 2) <= 2 whose sum may cancel
    ed = torch.cat(((dh * u).abs() * R.STEP * (2 + g.abs().clamp(max=16)), dh.abs() * R.STEP * (g.abs() + a.abs())), 1)
    ed = R.rounded(d, dt, ed)
    if "g" in want:
        R.close(got[2], d, ed, "dgu")
    if "x" in want:
        dx = d @ w
        R.close(got[0], dx, R.rounded(dx, dt, ed @ w.abs() + R.dot_bound(d.abs() + ed, w)), "dx")
    if "w" in want:
        old = torch.zeros_like(w) if dw0 is None else dw0
        dw = d.t() @ x + beta * old
        err = ed.t() @ x.abs() + R.dot_bound((d.abs() + ed).t(), x) + 4 * R.E * (beta * old).abs()
        R.close(got[1], dw, R.rounded(dw, wt, err), "dw")


def grad_inputs(M, N, K, dt, seed=20):
    x, w = R.values(M, K, dt, seed), R.values(2 * N, K, dt, seed + 1, K ** -0.5)
    return R.values(M, N, dt, seed + 2, 0.1), (x @ w.t()).to(R.TORCH[dt]).double(), x, w


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_backward(M, N, K, dt):
    args = grad_inputs(M, N, K, dt)
    check_backward(backward(*args, dt, "silu"), *args, dt, "silu")


@pytest.mark.parametrize("act", list(R.ACTS))
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_backward_forms(act, dt):
    """Each activation; single outputs, dgu in gu's place or in the workspace, fp32 accumulation, strides."""
    args = grad_inputs(70, 40, 64, dt)
    dw0 = R.values(80, 64, "f32", 30, 2.0)
    for kw in (dict(), dict(want="x"), dict(want="w"), dict(want="g"), dict(want="xw"), dict(inplace=True),
               dict(wt="f32", beta=0.5, dw0=dw0), dict(pad=8), dict(pad=3, off=1)):
        check_backward(backward(*args, dt, act, **kw), *args, dt, act,
                       **{k: v for k, v in kw.items() if k in ("wt", "beta", "dw0", "want")})


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gradients_against_differences(act):
    """<gradient, v> against central differences of the definition, h = 1e-4 (the kept projections in fp32)."""
    M, N, K, h = 5, 24, 40, 1e-4
    x, w, c = R.values(M, K, "f32", 41), R.values(2 * N, K, "f32", 42, 0.3), R.values(M, N, "f32", 43)

    def f(x, w):
        gu = x @ w.t()
        return float((R.act(act, gu[:, :N]) * gu[:, N:] * c).sum())
    dx, dw, _ = backward(c, (x @ w.t()), x, w, "f32", act)
    for i, (grad, at) in enumerate(((dx, x), (dw, w))):
        v = R.values(*at.shape, "f32", 50 + i)
        lo, hi = [x, w], [x, w]
        hi[i], lo[i] = at + h * v, at - h * v
        diff = (f(*hi) - f(*lo)) / (2 * h)
        assert abs(float((grad * v).sum()) - diff) <= 1e-5 * float((grad * v).abs().sum()) + 1e-6


def test_empty_batch():
    dw = R.Buf(20, 30, "f32", 2, values=torch.full((20, 30), 3.0))
    assert vk.glu_async(0, 0, 0, 10, 30, None, 30, None, 30, None, 10) == vk.OK
    for beta, want in ((0.5, 1.5), (0.0, 0.0)):
        vk.glu_backward_async(0, 0, 0, 10, 30, None, 10, None, 20, None, 30, None, 30, None, 0, None, 30, dw.ptr, dw.ld,
                              0, beta, stream=stream())
        assert bool((dw.get() == want).all())
    dw.check_around()


# sizes whose work is worth copies of the operands: K in no 16-byte units, M and N in no whole steps, together
# and alone; a misaligned x or w alone; the references in float64 on the GPU
LARGE = [(300, 600, 1501), (300, 600, 2701), (1100, 1001, 1003), (1030, 2051, 512), (1100, 1024, 1000), (129, 4099, 2048)]


@pytest.mark.parametrize("M,N,K", LARGE)
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_padded_operands(M, N, K, dt):
    x, w = R.values(M, K, dt, 60).cuda(), R.values(2 * N, K, dt, 61, K ** -0.5).cuda()
    check_forward(forward(x, w, dt, "silu"), x, w, dt, "silu")
    joined = N == 600 and (dt == "f32" or K == 2701)   # few tiles with a long K
    assert vk.last_kernel() == (vk.KERNEL_JOINED if joined else vk.KERNEL_FUSED)
    dh = R.values(M, N, dt, 62, 0.1).cuda()
    args = (dh, (x @ w.t()).to(R.TORCH[dt]).double(), x, w)
    dw0 = R.values(2 * N, K, "f32", 63).cuda()
    for kw in (dict(want="xw"), dict(), dict(want="xw", wt="f32", beta=0.5, dw0=dw0), dict(want="xw", pad=3, off=1)):
        check_backward(backward(*args, dt, "silu", **kw), *args, dt, "silu",
                       **{k: v for k, v in kw.items() if k in ("wt", "beta", "dw0", "want")})


def test_offsets_past_32_bits():
    """gu of 2.2e9 elements: the last rows and columns are right."""
    M, N, K = 70000, 16000, 128
    x, w = torch.randn(M, K, device="cuda").bfloat16(), (torch.randn(2 * N, K, device="cuda") * K ** -0.5).bfloat16()
    h, gu = (torch.empty(M, c, device="cuda", dtype=torch.bfloat16) for c in (N, 2 * N))
    vk.glu_async(vk.DT_BF16, vk.ACT_SILU, M, N, K, x.data_ptr(), K, w.data_ptr(), K, h.data_ptr(), N, gu.data_ptr(),
                 2 * N, stream=stream())
    for rows in (slice(0, 3), slice(M - 3, M)):
        check_forward((h[rows].double(), gu[rows].double()), x[rows].double(), w.double(), "bf16", "silu")
    dh = torch.randn(M, N, device="cuda").bfloat16()
    dx = torch.empty(M, K, device="cuda", dtype=torch.bfloat16)
    vk.glu_backward_async(vk.DT_BF16, vk.ACT_SILU, M, N, K, dh.data_ptr(), N, gu.data_ptr(), 2 * N, None, 0,
                          w.data_ptr(), K, gu.data_ptr(), 2 * N, dx.data_ptr(), K, None, 0, vk.DT_BF16, 0.0,
                          stream=stream())
    # dgu took gu's place: what it was, from x again
    for rows in (slice(0, 3), slice(M - 3, M)):
        pre = (x[rows].double() @ w.double().t()).bfloat16().double()
        check_backward((dx[rows].double(), None, gu[rows].double()), dh[rows].double(), pre, x[rows].double(),
                       w.double(), "bf16", "silu", want="x")


def test_graph_capture_and_workspace():
    """A fused forward pass needs no workspace: captured and replayed, equal to the eager result each time.  A
    backward pass without dgu needs one: refused under capture, nothing launched."""
    M, N, K = 300, 200, 256
    x, w = (torch.randn(r, K, device="cuda").half() for r in (M, 2 * N))
    h, gu, dx = (torch.zeros(M, c, device="cuda", dtype=torch.half) for c in (N, 2 * N, K))

    def call(s):
        return vk.glu_async(vk.DT_F16, vk.ACT_GELU, M, N, K, x.data_ptr(), K, w.data_ptr(), K, h.data_ptr(), N,
                            gu.data_ptr(), 2 * N, stream=s)
    call(stream())
    torch.cuda.synchronize()
    eager = h.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(stream())
        st = vk.glu_backward_async(vk.DT_F16, vk.ACT_GELU, M, N, K, h.data_ptr(), N, gu.data_ptr(), 2 * N, x.data_ptr(),
                                   K, w.data_ptr(), K, None, 0, dx.data_ptr(), K, None, 0, vk.DT_F16, 0.0,
                                   stream=stream(), check=False)
    assert st == vk.ERR_INIT
    for _ in range(3):
        h.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, eager)
        call(stream())
    assert not dx.any()
