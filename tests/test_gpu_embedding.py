"""vkblas_embedding_async and its gradient against the definition in float64: types, one token to several merged runs,
one class to many, a token in every row, padding, ids outside the vocabulary, strides, alignment, beta, equal bits."""
import pytest
import torch

import nn_ref as R
import train_ref as D
import vkblas_amd as vk

pytestmark = pytest.mark.gpu
PAD = D.PAD
TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")]


def stream():
    return torch.cuda.current_stream().cuda_stream


def tokens(M, V, seed, kind="usual"):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        return torch.full((M,), V // 2)
    if kind == "uniform":
        return torch.randint(0, V, (M,), generator=g)
    ids = (V ** torch.rand(M, generator=g, dtype=torch.float64) - 1).long().clamp(0, V - 1)
    ids[3::7] = PAD
    ids[0], ids[-1] = V - 1, 0
    return ids


def lookup(w, ids, dt, wt, scale, pad=0, off=0, pad_id=PAD):
    M, (V, N) = len(ids), w.shape
    bw, by, ti = R.Buf(V, N, wt, pad, off, w), R.Buf(M, N, dt, pad, off), ids.cuda()
    vk.embedding_async(R.ENGINE[dt], R.ENGINE[wt], M, V, N, ti.data_ptr(), pad_id, bw.ptr, bw.ld, scale, by.ptr, by.ld,
                       stream=stream())
    assert vk.last_kernel() == vk.KERNEL_EMBED
    by.check_around()
    return by.get()


def check_lookup(got, w, ids, dt, scale, pad_id=PAD):
    y = D.embedding(w, ids, scale, pad_id)
    assert torch.equal(torch.isnan(got), torch.isnan(y))
    R.close(got.nan_to_num(0), y.nan_to_num(0), R.rounded(y.nan_to_num(0), dt, R.E * y.nan_to_num(0).abs()), "y")
    assert bool((got[ids == pad_id] == 0).all())


SIZES = [(1, 1, 1), (1, 50, 64), (2, 7, 3), (5, 1000, 4096), (33, 300, 257), (200, 64, 512), (1003, 997, 515),
         (4096, 100, 72), (4097, 2000, 65)]


@pytest.mark.parametrize("M,V,N", SIZES)
@pytest.mark.parametrize("dt,wt", TYPES)
def test_forward(M, V, N, dt, wt):
    w, ids = R.values(V, N, wt, 1), tokens(M, V, 2)
    check_lookup(lookup(w, ids, dt, wt, 1.5), w, ids, dt, 1.5)


@pytest.mark.parametrize("dt,wt", TYPES)
@pytest.mark.parametrize("pad,off", [(8, 0), (4, 4), (1, 0), (3, 1)])
def test_forward_strides_padding_and_ids_outside(dt, wt, pad, off):
    w, ids = R.values(90, 130, wt, 1), tokens(70, 90, 2)
    check_lookup(lookup(w, ids, dt, wt, 0.37109375, pad, off), w, ids, dt, 0.37109375)
    ids[5], ids[6], ids[7], ids[8], ids[9] = 90, -2, 2 ** 40, -2 ** 63, 2 ** 32 + 3
    check_lookup(lookup(w, ids, dt, wt, 2.0, pad, off), w, ids, dt, 2.0)
    check_lookup(lookup(w, ids, dt, wt, 2.0, pad, off, pad_id=2 ** 40), w, ids, dt, 2.0, 2 ** 40)
    check_lookup(lookup(w, ids, dt, wt, 2.0, pad, off, pad_id=0), w, ids, dt, 2.0, 0)


def test_forward_copies_what_it_does_not_scale():
    """scale 1 and one type: bits as they are, infinities too."""
    w = R.values(40, 72, "f16", 1)
    w[3, 5], w[4, 6] = float("inf"), -float("inf")
    ids = tokens(100, 40, 2, "uniform")
    assert torch.equal(lookup(w, ids, "f16", "f16", 1.0), w[ids])


def gradient(dy, ids, V, dt, wt, scale, beta=0.0, dw0=None, pad=0, off=0, pad_id=PAD):
    M, N = dy.shape
    bd, bw, ti = R.Buf(M, N, dt, pad, off, dy), R.Buf(V, N, wt, pad, off, dw0), ids.cuda()
    vk.embedding_backward_async(R.ENGINE[dt], M, V, N, ti.data_ptr(), pad_id, bd.ptr, bd.ld, scale, bw.ptr, bw.ld,
                                R.ENGINE[wt], beta, stream=stream())
    assert vk.last_kernel() == vk.KERNEL_EMBED
    bw.check_around()
    return bw.get()


def check_gradient(got, dy, ids, V, wt, scale, beta=0.0, dw0=None, pad_id=PAD):
    dw, err = D.embedding_grad(dy, ids, V, scale, pad_id, beta, dw0)
    R.close(got, dw, R.rounded(dw, wt, err), "dw")
    return dw


# one launch (up to 2048 and 4096 rows), chunks of the sorted pairs, runs of 1024, merges of up to 16 and 64 of them, a
# second level of merges (past 65536)
GRAD_SIZES = SIZES + [(8, 3, 70), (9, 3, 70), (2047, 5, 24), (2048, 700, 72), (2049, 9, 8), (4095, 3, 8), (4097, 3, 8),
                      (6145, 1, 20), (8192, 5, 24), (12289, 100000, 8), (16385, 40, 264), (32768, 200, 16),
                      (32769, 3, 16), (65536, 3000, 16), (65537, 257, 9), (131073, 50, 8), (150001, 1000, 5),
                      (16384, 90, 8)]


@pytest.mark.parametrize("M,V,N", GRAD_SIZES)
@pytest.mark.parametrize("dt,wt", TYPES)
def test_gradient(M, V, N, dt, wt):
    dy, ids = R.values(M, N, dt, 1), tokens(M, V, 2)
    check_gradient(gradient(dy, ids, V, dt, wt, 1.5), dy, ids, V, wt, 1.5)


@pytest.mark.parametrize("kind", ["usual", "uniform"])
def test_gradient_of_more_tokens_than_a_launch_merges_at_once(kind):
    M, V, N = 4_300_001, 5000, 4
    dy, ids = R.values(M, N, "bf16", 1), tokens(M, V, 2, kind)
    check_gradient(gradient(dy, ids, V, "bf16", "f32", 0.5), dy, ids, V, "f32", 0.5)


@pytest.mark.parametrize("M,V,N", [(1, 40000, 1000), (3, 33000, 1025), (300, 70001, 520), (1024, 34000, 1000),
                                   (1025, 34000, 1000), (4096, 16400, 2050)])
@pytest.mark.parametrize("beta", [0.0, 1.0, 0.5])
def test_gradient_of_few_tokens_and_a_large_one(M, V, N, beta):
    """More bytes than the one launch takes: the sort of one run.  On the GPU."""
    dy, ids = R.values(M, N, "bf16", 1).cuda(), tokens(M, V, 2).cuda()
    dw0 = torch.linspace(-1, 1, V, dtype=torch.float32).double()[:, None].expand(V, N).contiguous().cuda()
    got = gradient(dy, ids, V, "bf16", "f32", 1.5, beta, dw0)
    dw, err = D.embedding_grad(dy, ids, V, 1.5, PAD, beta, dw0)
    R.close(got.cuda(), dw, R.rounded(dw, "f32", err), "dw")


@pytest.mark.parametrize("M,V,N", [(7, 5, 130), (100, 64, 257), (5000, 900, 72), (70000, 30, 24)])
@pytest.mark.parametrize("kind", ["one", "uniform", "usual"])
@pytest.mark.parametrize("dt,wt", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
def test_gradient_of_one_token_and_beta(M, V, N, kind, dt, wt):
    """Every row the same token; what dw held is kept (beta 1), scaled, or not read (NaN, beta 0)."""
    dy, ids = R.values(M, N, dt, 1), tokens(M, V, 2, kind)
    dw0 = R.values(V, N, wt, 3)
    for beta in (1.0, 0.5, -2.0):
        got = gradient(dy, ids, V, dt, wt, 0.5, beta, dw0)
        check_gradient(got, dy, ids, V, wt, 0.5, beta, dw0)
        if beta == 1.0:
            rest = torch.ones(V, dtype=torch.bool)
            rest[ids[ids >= 0]] = False
            assert torch.equal(got[rest], dw0[rest])
    got = gradient(dy, ids, V, dt, wt, 0.5, 0.0, torch.full_like(dw0, float("nan")))
    check_gradient(got, dy, ids, V, wt, 0.5)


@pytest.mark.parametrize("dt,wt", TYPES)
@pytest.mark.parametrize("pad,off", [(8, 0), (4, 4), (1, 0), (3, 1)])
def test_gradient_strides_padding_and_ids_outside(dt, wt, pad, off):
    """Rows of padding and of ids outside the vocabulary add nothing, whatever they hold."""
    M, V, N = 300, 77, 133
    dy, ids = R.values(M, N, dt, 1), tokens(M, V, 2)
    ids[5], ids[6], ids[7], ids[8], ids[9], ids[10] = V, -2, 2 ** 40, -2 ** 63, 2 ** 32 + 3, 2 ** 31
    clean = dy.clone()
    for m in range(M):
        if not 0 <= ids[m] < V:
            dy[m] = float("nan") if m % 2 else float("inf")
            clean[m] = 0
    check_gradient(gradient(dy, ids, V, dt, wt, 2.0, pad=pad, off=off), clean, ids, V, wt, 2.0)
    dw0 = R.values(V, N, wt, 3)
    check_gradient(gradient(dy, ids, V, dt, wt, 2.0, 1.0, dw0, pad, off), clean, ids, V, wt, 2.0, 1.0, dw0)
    every = torch.full((M,), PAD)
    assert torch.equal(gradient(dy, every, V, dt, wt, 2.0, 1.0, dw0, pad, off), dw0)
    assert bool((gradient(dy, every, V, dt, wt, 2.0, 0.0, dw0, pad, off) == 0).all())


@pytest.mark.parametrize("M", [1000, 20000])
def test_equal_calls_give_equal_bits(M):
    V, N = 500, 264
    dy, ids = R.values(M, N, "bf16", 1), tokens(M, V, 2)
    first = gradient(dy, ids, V, "bf16", "f32", 1.0)
    for _ in range(3):
        assert torch.equal(gradient(dy, ids, V, "bf16", "f32", 1.0), first)


def test_gradient_against_differences():
    """The map is linear: <dw, v> equals <dy, y(v)>."""
    M, V, N = 60, 17, 40
    dy, ids, v = R.values(M, N, "f32", 1), tokens(M, V, 2), R.values(V, N, "f32", 3)
    dw = gradient(dy, ids, V, "f32", "f32", 0.75)
    size = float((dy * D.embedding(v, ids, 0.75)).abs().sum())
    assert abs(float((dw * v).sum()) - float((dy * lookup(v, ids, "f32", "f32", 0.75)).sum())) <= (M + 8) * R.E * size


def test_empty_batch():
    dw = R.Buf(20, 30, "f16", 2, values=torch.full((20, 30), 3.0))
    for beta, want in ((1.0, 3.0), (0.5, 1.5), (0.0, 0.0)):
        vk.embedding_backward_async(vk.DT_F16, 0, 20, 30, None, PAD, None, 30, 1.0, dw.ptr, dw.ld, vk.DT_F16, beta,
                                    stream=stream())
        assert bool((dw.get() == want).all())
    dw.check_around()


def test_a_vocabulary_of_many_rows():
    """More rows than the fill has workgroups of 64."""
    M, V = 5000, 70_000_001
    ids = torch.randint(0, V, (M,), device="cuda")
    ids[0], ids[1], ids[2] = V - 1, 0, V - 1
    dy = torch.randn(M, 1, device="cuda")
    for beta in (0.0, 0.5):
        dw = torch.full((V, 1), 2.0, device="cuda")
        vk.embedding_backward_async(vk.DT_F32, M, V, 1, ids.data_ptr(), PAD, dy.data_ptr(), 1, 1.0, dw.data_ptr(), 1,
                                    vk.DT_F32, beta, stream=stream())
        want = torch.full((V, 1), 2.0 * beta, device="cuda", dtype=torch.float64).index_add(0, ids, dy.double())
        assert float((dw - want).abs().max()) <= 1e-5


def test_offsets_past_32_bits():
    """A vocabulary of 2.2e9 elements: the last rows are read and written where they are."""
    V, N = 540000, 4096
    w = torch.zeros(V, N, device="cuda", dtype=torch.bfloat16)
    ids = torch.tensor([V - 1, 3, V - 2, V - 1, 524288], device="cuda")
    dy = torch.randn(5, N, device="cuda").bfloat16()
    vk.embedding_backward_async(vk.DT_BF16, 5, V, N, ids.data_ptr(), PAD, dy.data_ptr(), N, 1.0, w.data_ptr(), N,
                                vk.DT_BF16, 0.0, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(w[V - 1], (dy[0].float() + dy[3].float()).bfloat16())
    assert torch.equal(w[524288], dy[4]) and torch.equal(w[3], dy[1]) and not w[4].any() and not w[V - 3].any()
    y = torch.empty(5, N, device="cuda", dtype=torch.bfloat16)
    vk.embedding_async(vk.DT_BF16, vk.DT_BF16, 5, V, N, ids.data_ptr(), PAD, w.data_ptr(), N, 1.0, y.data_ptr(), N,
                       stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(y, w[ids])


@pytest.mark.parametrize("dt,V", [("f32", 2 ** 24), ("bf16", 2 ** 25), ("bf16", 2 ** 25 - 4097)])
@pytest.mark.parametrize("beta", [0.0, 1.0, 0.5])
def test_the_one_launch_of_the_most_rows(dt, V, beta):
    """One column of a gradient of 64 MiB: as many rows as a workgroup lists.  On the GPU."""
    M = 4096
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, V, (M,), generator=g)
    ids[:40], ids[40], ids[41], ids[42] = V - 1, 0, PAD, V
    dy = R.values(M, 1, dt, 1).cuda()
    dw0 = torch.linspace(-1, 1, V, dtype=torch.float32, device="cuda").to(R.TORCH[dt]).double()[:, None]
    got = gradient(dy, ids, V, dt, dt, 0.5, beta, dw0)
    dw, err = D.embedding_grad(dy, ids.cuda(), V, 0.5, PAD, beta, dw0)
    R.close(got.cuda(), dw, R.rounded(dw, dt, err), "dw")
