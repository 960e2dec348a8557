"""vkblas_policy_loss_async and its gradient against the definition in float64: sizes around units and the small call,
reductions, masks that leave sequences or everything empty, NaN and infinities where nothing counts, ratios at their
bounds, no reference, advantages of a token and of a sequence, strides."""
import math

import pytest
import torch

import nn_ref as R
import train_ref as D
import vkblas_amd as vk

pytestmark = pytest.mark.gpu
LOW, HIGH, KL = D.f32(0.2), D.f32(0.28), D.f32(0.05)
REDUCE = {"tokens": vk.REDUCE_TOKENS, "sequences": vk.REDUCE_SEQUENCES, "sum": vk.REDUCE_SUM}


def stream():
    return torch.cuda.current_stream().cuda_stream


def inputs(B, T, seed=1, ref=True, per_token=True, masked=True, spread=0.2):
    g = torch.Generator().manual_seed(seed)
    old = (torch.rand(B, T, generator=g) + 1e-6).log()
    logp = old + spread * torch.randn(B, T, generator=g)
    r = old + 2 * spread * torch.randn(B, T, generator=g) if ref else None
    adv = torch.randn(B, T if per_token else 1, generator=g)
    mask = torch.ones(B, T, dtype=torch.uint8)
    if masked:
        mask = (torch.arange(T) < torch.randint(0, T + 1, (B, 1), generator=g)).to(torch.uint8) * 3
        mask[torch.rand(B, T, generator=g) < 0.1] = 0
        mask[0, 0] = 255
        mask[1::7] = 0
    return dict(logp=logp, old=old, ref=r, adv=adv, mask=mask, masked=masked)


class Call:
    """The inputs on the GPU: rows of T + pad floats, off elements past their alignment, NaN around them."""

    def __init__(self, i, pad=0, off=0):
        self.B, self.T = i["logp"].shape
        buf = lambda v: None if v is None else R.Buf(*v.shape, "f32", pad, off, v)
        self.bufs = [buf(i[k]) for k in ("logp", "old", "ref", "adv")]
        self.mask = torch.full((self.B * (self.T + pad) + off,), 1, dtype=torch.uint8, device="cuda")
        self.mask[off:].view(self.B, -1)[:, :self.T] = i["mask"].cuda()
        args = []
        for b in self.bufs[:3]:
            args += [b.ptr if b else None, b.ld if b else 0]
        a = self.bufs[3]
        args += [a.ptr, a.ld, int(a.cols > 1 or self.T == 1)]
        args += [self.mask.data_ptr() + off if i["masked"] else None, self.T + pad]
        self.args, self.pad, self.off = args, pad, off

    def loss(self, reduce="tokens", low=LOW, high=HIGH, kl=KL):
        stats, norm = R.Buf(1, 4, "f32"), R.Buf(1, self.B, "f32")
        vk.policy_loss_async(REDUCE[reduce], self.B, self.T, *self.args, low, high, kl, stats.ptr, norm.ptr,
                             stream=stream())
        assert vk.last_kernel() == vk.KERNEL_POLICY
        stats.check_around()
        norm.check_around()
        return stats.get()[0], norm.get()[0]

    def grad(self, norm, dloss, low=LOW, high=HIGH, kl=KL):
        out, n = R.Buf(self.B, self.T, "f32", self.pad, self.off), R.Buf(1, self.B, "f32", values=norm[None])
        dl = torch.tensor([dloss], dtype=torch.float32, device="cuda")
        vk.policy_loss_backward_async(self.B, self.T, *self.args, low, high, kl, n.ptr, dl.data_ptr(), out.ptr, out.ld,
                                      stream=stream())
        out.check_around()
        return out.get()


def exact(i):
    return [None if i[k] is None else i[k].double() for k in ("logp", "old", "ref", "adv")] + [i["mask"] != 0]


def err(i):
    """Relative error of a token's ratio and KL term: their arguments' rounding and a few operations."""
    logp, old, ref, adv, mask = exact(i)
    big = torch.where(mask, (logp - old).abs(), torch.zeros_like(logp)).max()
    if ref is not None:
        big = torch.maximum(big, torch.where(mask, (ref - logp).abs(), torch.zeros_like(logp)).max())
    return R.STEP * (4 + float(big))


def check_loss(got, i, reduce, low=LOW, high=HIGH, kl=KL):
    stats, size, norm = D.policy(*exact(i), low, high, kl, reduce)
    R.close(got[0], stats, err(i) * size + R.E * stats.abs(), "stats")
    R.close(got[1], norm, 2 * R.E * norm, "norm")


def check_grad(got, i, norm, dloss, low=LOW, high=HIGH, kl=KL):
    g, size = D.policy_grad(*exact(i), low, high, kl, norm, dloss)
    # the KL term's difference of two fp32 numbers is rounded once: e |d| <= size's own scale times e / slope of 1
    logp, _, ref, _, mask = exact(i)
    w = (norm * dloss).abs()[:, None]
    diff = 0 if ref is None else torch.where(mask, w * abs(kl) * R.E * (ref - logp).abs() * torch.exp(ref - logp),
                                             torch.zeros_like(logp))
    R.close(got, g, err(i) * size + diff, "dlogp")
    assert bool((got[i["mask"] == 0] == 0).all())


# units of 256 tokens, the small call of 64 of them (one workgroup) and past it, many units of a sequence
SIZES = [(1, 1), (1, 5), (3, 64), (8, 100), (2, 255), (2, 256), (2, 257), (64, 256), (65, 256), (63, 257), (1, 16384),
         (1, 16385), (16, 256), (17, 256), (15, 257), (2, 40001), (300, 700), (5000, 3), (1, 2000001),
         (9000, 5), (2500, 300), (70001, 2), (2049, 257), (2047, 257), (2048, 1025)]


@pytest.mark.parametrize("B,T", SIZES)
@pytest.mark.parametrize("reduce", REDUCE)
def test_loss_and_gradient(B, T, reduce):
    i = inputs(B, T, per_token=reduce != "sequences", ref=reduce != "sum")
    c = Call(i)
    got = c.loss(reduce)
    check_loss(got, i, reduce)
    check_grad(c.grad(got[1], 0.75), i, got[1], 0.75)


@pytest.mark.parametrize("B,T", [(5_000_000, 1), (1_100_000, 257)])
def test_more_sequences_than_workgroups(B, T):
    """Against the definition on the GPU, equal rows: sequences of equal tokens."""
    base = torch.linspace(-0.3, 0.3, 7, device="cuda").repeat(B // 7 + 1)[:B, None].expand(B, T).contiguous()
    zero, adv = torch.zeros(B, T, device="cuda"), torch.ones(B, 1, device="cuda")
    stats, norm = torch.empty(4, device="cuda"), torch.empty(B, device="cuda")
    vk.policy_loss_async(vk.REDUCE_SEQUENCES, B, T, base.data_ptr(), T, zero.data_ptr(), T, None, 0, adv.data_ptr(), 1,
                         0, None, 0, LOW, HIGH, 0.0, stats.data_ptr(), norm.data_ptr(), stream=stream())
    r = base[:, 0].double().exp()
    want = torch.stack([-r.clamp(max=1 + HIGH).mean(), 0 * r[0], (r > 1 + HIGH).double().mean(), r.mean()])
    assert float((stats.double() - want).abs().max()) <= 1e-6
    assert float((norm.double() * B * T - 1).abs().max()) <= 1e-6


@pytest.mark.parametrize("B,T", [(7, 130), (90, 301)])
@pytest.mark.parametrize("pad,off", [(0, 0), (4, 0), (1, 0), (3, 1)])
@pytest.mark.parametrize("masked", [True, False])
def test_strides_alignment_and_no_mask(B, T, pad, off, masked):
    i = inputs(B, T, masked=masked)
    c = Call(i, pad, off)
    got = c.loss("sequences")
    check_loss(got, i, "sequences")
    check_grad(c.grad(got[1], -2.0), i, got[1], -2.0)


@pytest.mark.parametrize("B,T", [(6, 40), (100, 400)])
@pytest.mark.parametrize("reduce", REDUCE)
def test_what_does_not_count_may_hold_anything(B, T, reduce):
    i = inputs(B, T)
    out = i["mask"] == 0
    clean = Call(i)
    want = clean.loss(reduce)
    grad = clean.grad(want[1], 1.0)
    for v in (float("nan"), float("inf"), -float("inf"), torch.finfo(torch.float32).min):
        for k in ("logp", "old", "ref", "adv"):
            i[k][out] = v
        c = Call(i)
        assert all(torch.equal(a, b) for a, b in zip(c.loss(reduce), want))
        assert torch.equal(c.grad(want[1], 1.0), grad)


@pytest.mark.parametrize("B,T", [(1, 3), (5, 300), (200, 200)])
@pytest.mark.parametrize("reduce", REDUCE)
def test_nothing_counts(B, T, reduce):
    i = inputs(B, T)
    i["mask"][:] = 0
    stats, norm = Call(i).loss(reduce)
    assert bool((stats == 0).all()) and bool((norm == 0).all())
    assert bool((Call(i).grad(norm, 1.0) == 0).all())


def test_ratios_at_their_bounds():
    """logp - old one unit to each side of log(1 + clip_high) and log(1 - clip_low), both signs of the advantage: the
    side is the exact one."""
    at = torch.tensor([math.log1p(HIGH), math.log1p(-LOW)], dtype=torch.float32)
    d = torch.stack([at] + [torch.nextafter(at, at + s) for s in (1.0, -1.0)]).flatten()
    # old of a far larger magnitude than the difference, so that an fp32 difference would round
    old = torch.stack((torch.zeros(6), torch.full((6,), -4096.0)))
    i = dict(logp=old + d, old=old, ref=None, mask=torch.ones(2, 6, dtype=torch.uint8), masked=True)
    for sign in (1.0, -1.0):
        i["adv"] = torch.full((2, 6), sign)
        c = Call(i)
        got = c.loss("sum")
        check_loss(got, i, "sum")
        assert float(got[0][2]) == float(D.policy(*exact(i), LOW, HIGH, KL, "sum")[0][2])
        check_grad(c.grad(got[1], 1.0), i, got[1], 1.0)


@pytest.mark.parametrize("low,high", [(0.0, 0.0), (1.0, 0.5), (3.0, 0.1), (float("inf"), float("inf")), (0.1, 1e30)])
@pytest.mark.parametrize("kl", [0.0, 2.5, -1.0])
def test_bounds_and_coefficients(low, high, kl):
    low, high = D.f32(low), D.f32(high)
    i = inputs(20, 50, spread=0.5)
    c = Call(i)
    got = c.loss("tokens", low, high, kl)
    check_loss(got, i, "tokens", low, high, kl)
    check_grad(c.grad(got[1], 1.0, low, high, kl), i, got[1], 1.0, low, high, kl)


def test_far_apart_policies():
    """Ratios that overflow are held by the bound for a positive advantage; kl_coef 0 leaves an infinite KL term out of
    the loss."""
    i = inputs(1, 4, masked=False)
    i["old"][:], i["logp"][:] = -200.0, 0.0
    i["ref"][:] = 200.0
    i["adv"][:] = 1.0
    c = Call(i)
    stats, norm = c.loss("tokens", kl=0.0)
    assert abs(float(stats[0]) + 1 + HIGH) < 1e-6 and math.isinf(stats[1]) and float(stats[2]) == 1.0
    assert bool((c.grad(norm, 1.0, kl=0.0) == 0).all())
    i["adv"][:] = -1.0
    assert float(Call(i).loss("tokens", kl=0.0)[0][0]) == float("inf")
    i["logp"][0, 2] = float("nan")
    stats, norm = Call(i).loss("tokens")
    assert math.isnan(stats[0])


def test_small_kl_terms_keep_their_digits():
    """exp(d) - d - 1 of d = 1e-4 is 5e-9: all of its bits, not those that a difference leaves."""
    i = inputs(4, 64, masked=False)
    i["old"] = i["logp"].clone()
    i["ref"] = i["logp"] + 1e-4
    c = Call(i)
    got = c.loss("tokens")
    ref = D.policy(*exact(i), LOW, HIGH, KL, "tokens")[0]
    assert abs(float(got[0][1] / ref[1]) - 1) < 1e-5


def test_gradient_against_differences():
    """Central differences of the definition, h = 1e-5, away from the bounds."""
    i = inputs(6, 30, spread=0.3)
    logp, old, ref, adv, mask = exact(i)
    ratio = torch.exp(logp - old)
    near = ((ratio - 1 + LOW).abs() < 1e-3) | ((ratio - 1 - HIGH).abs() < 1e-3)
    i["mask"][near] = 0
    mask = i["mask"] != 0
    c = Call(i)
    norm = c.loss("sequences")[1]
    got, h = c.grad(norm, 1.0), 1e-5
    up, down = (D.policy_terms(logp + s * h, old, ref, adv, LOW, HIGH, KL)[0] for s in (1, -1))
    diff = torch.where(mask, norm[:, None] * (up - down) / (2 * h), torch.zeros_like(up))
    assert float((got - diff).abs().max()) <= 1e-6 * float(diff.abs().max())


def test_gradient_in_place_of_logp():
    i = inputs(10, 333)
    c = Call(i)
    norm = c.loss()[1]
    want = c.grad(norm, 1.0)
    dl = torch.ones(1, device="cuda")
    n = norm.float().cuda()
    vk.policy_loss_backward_async(10, 333, *c.args, LOW, HIGH, KL, n.data_ptr(), dl.data_ptr(), c.bufs[0].ptr,
                                  c.bufs[0].ld, stream=stream())
    assert torch.equal(c.bufs[0].get(), want)


def test_equal_calls_give_equal_bits():
    c = Call(inputs(300, 700))
    first = c.loss()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(c.loss(), first))


def test_empty_batch():
    args = 0, 5, None, 5, None, 5, None, 0, None, 5, 1, None, 0, 0.2, 0.2, 0.0
    assert vk.policy_loss_async(0, *args, None, None) == vk.OK
    assert vk.policy_loss_backward_async(*args, None, None, None, 5) == vk.OK


# ---- ratios past fp32

def overflowing(B, T, per_token):
    """Tokens (or whole sequences) without an advantage whose ratio is past fp32's range, and the same with a ratio of
    1: they add the same to everything but the mean ratio."""
    i = inputs(B, T, per_token=per_token)
    i["mask"][-1] = 1
    none = torch.zeros(B, T, dtype=torch.bool)
    none[:, ::3] = True
    if not per_token:
        none[:] = False
        none[::2] = True
        none[-1] = True
    i["adv"][none if per_token else none[:, :1]] = 0.0
    i["adv"][0, 0] = -0.0 if none[0, 0] else i["adv"][0, 0]
    i["ref"][none], i["logp"][none] = 0.125, 0.0
    i["old"][none] = 0.0
    plain = dict(i, old=i["old"].clone())
    i["old"][none] = -200.0
    return i, plain


# the small call, units, a sequence a wave, a sequence a workgroup
OVERFLOW = [(1, 7), (20, 9000), (3000, 70), (300, 700)]


@pytest.mark.parametrize("B,T", OVERFLOW)
@pytest.mark.parametrize("reduce", REDUCE)
@pytest.mark.parametrize("per_token", [True, False])
def test_no_advantage_times_a_ratio_past_fp32_is_nothing(B, T, reduce, per_token):
    i, plain = overflowing(B, T, per_token)
    want, got = Call(plain).loss(reduce), Call(i).loss(reduce)
    check_loss(want, plain, reduce)
    assert torch.equal(got[0][:3], want[0][:3]) and math.isinf(got[0][3]) and torch.equal(got[1], want[1])
    grad = Call(plain).grad(want[1], 0.5)
    check_grad(grad, plain, want[1], 0.5)
    assert torch.equal(Call(i).grad(want[1], 0.5), grad)


@pytest.mark.parametrize("key,v", [("logp", math.nan), ("old", math.nan), ("adv", math.nan), ("old", -math.inf)])
def test_no_advantage_hides_no_nan(key, v):
    """A NaN reaches the loss through an advantage of 0 too, and so does 0 times an infinite difference."""
    i = inputs(2, 30, masked=False)
    i["adv"][1, 4] = 0.0
    i[key][1, 4] = v
    c = Call(i)
    stats, norm = c.loss("tokens", kl=0.0)
    assert math.isnan(stats[0])
    g = c.grad(norm, 1.0, kl=0.0)
    assert bool(torch.isnan(g[1, 4])) and int(torch.isnan(g).sum()) == 1


@pytest.mark.parametrize("shape", [(1, 7), (20, 9000)])
def test_a_loss_gradient_of_0_leaves_none(shape):
    """Whatever a token's ratio and KL term grow to; a NaN or an infinity among the inputs stays a NaN."""
    i = inputs(*shape, masked=False)
    i["logp"][:] = 0.0
    i["old"][0, ::2], i["ref"][0, 1::2] = -200.0, 200.0
    i["adv"][:] = -1.0
    norm = torch.ones(shape[0], dtype=torch.float64)
    assert bool(torch.isinf(Call(i).grad(norm, 1.0)[0]).all())
    assert bool((Call(i).grad(norm, 0.0) == 0).all())
    for key, v in (("logp", math.nan), ("old", -math.inf), ("ref", math.inf), ("adv", -math.inf)):
        j = {**i, key: i[key].clone()}
        j[key][0, 3] = v
        g = Call(j).grad(norm, 0.0)
        assert bool(torch.isnan(g[0, 3])) and int(torch.isnan(g).sum()) == 1 and bool((g.nan_to_num(0) == 0).all())


@pytest.mark.parametrize("B,T", [(20, 9000), (300, 9000), (1024, 8192), (1100, 8192), (2047, 3001)])
@pytest.mark.parametrize("reduce", REDUCE)
def test_units_of_many_sequences(B, T, reduce):
    """Several units each of a few to more sequences than the finish keeps the tokens of, some without any."""
    i = inputs(B, T, per_token=reduce != "sum")
    assert bool((i["mask"] == 0).all(1).any())
    c = Call(i)
    got = c.loss(reduce)
    check_loss(got, i, reduce)
    check_grad(c.grad(got[1], 0.75), i, got[1], 0.75)


def misjudged(bound, upper, n=64):
    """fp32 pairs whose exact difference lies on one side of the bound and whose fp32 difference on the other, and
    which of them are past it."""
    g = torch.Generator().manual_seed(3)
    # multiples of 2^-30, finer than the difference's own step
    small = -torch.randint(2 ** 21, 2 ** 24, (20000,), generator=g).float() * 2.0 ** -30
    near = (small.double() - abs(bound)).float()
    other = torch.cat((near, torch.nextafter(near, near + 1), torch.nextafter(near, near - 1)))
    small = small.repeat(3)
    logp, old = (small, other) if upper else (other, small)
    exact_diff = logp.double() - old.double()
    past = exact_diff > bound if upper else exact_diff < bound
    wrong = past != ((logp - old).double() > bound if upper else (logp - old).double() < bound)
    # (far from the bound against what float64's own exp and log are off by)
    pick = torch.nonzero(wrong & ((exact_diff - bound).abs() > 1e-11))[:n, 0]
    return logp[pick], old[pick], past[pick]


# bounds whose logarithm lies below and above the middle of a step of fp32: the fp32 difference falls short of it, or
# goes past it
@pytest.mark.parametrize("clip,upper,past", [(0.3, True, True), (0.2, True, False), (0.1, False, True),
                                             (0.3, False, False)])
def test_sides_that_an_fp32_difference_takes_wrongly(clip, upper, past):
    clip = D.f32(clip)
    logp, old, held = misjudged(math.log1p(clip if upper else -clip), upper)
    assert len(logp) >= 20 and bool((held == past).all())
    i = dict(logp=logp[None], old=old[None], ref=None, adv=torch.full((1, len(logp)), 1.0 if upper else -1.0),
             mask=torch.ones(1, len(logp), dtype=torch.uint8), masked=True)
    assert torch.equal(D.policy_terms(*exact(i)[:4], clip, clip, KL)[2][0], held)
    c = Call(i)
    stats, norm = c.loss("sum", clip, clip)
    assert float(stats[2]) == float(held.sum())
    assert torch.equal(c.grad(norm, 1.0, clip, clip)[0] == 0, held)
