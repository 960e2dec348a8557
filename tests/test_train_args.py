"""The operators of vkblas_train.h refuse what they cannot compute before anything is launched (CPU: the pointers are
never followed), and accept empty batches without a GPU where nothing is to be written."""
import os
import re

import pytest

import vkblas_amd as vk

P = 4096    # a pointer that no check follows
NAN, INF = float("nan"), float("inf")
POLICY = dict(B=4, T=8, logp=P, ldp=8, old_logp=P, ldo=8, ref_logp=P, ldr=8, adv=P, ldadv=8, adv_step=1, mask=P,
              ldmask=8, clip_low=0.2, clip_high=0.2, kl_coef=0.1)
DISTILL = dict(dtype=1, M=4, V=9, K=16, x=P, ldx=16, w=P, ldw=16, n_top=5, top=P, ldtop=5, t_dtype=0, t=P, ldt=5,
               temperature=2.0)
CALLS = {
    "embedding": (vk.embedding_async, dict(dtype=2, w_dtype=0, M=4, V=9, N=8, ids=P, pad_id=-1, w=P, ldw=8, scale=1.0,
                                           y=P, ldy=8)),
    "embedding_backward": (vk.embedding_backward_async,
                           dict(dtype=2, M=4, V=9, N=8, ids=P, pad_id=-1, dy=P, lddy=8, scale=1.0, dw=P, lddw=8,
                                dw_dtype=2)),
    "linear_distill": (vk.linear_distill_async, dict(DISTILL, loss=P, lse=P, z_top=P)),
    "linear_distill_backward": (vk.linear_distill_backward_async,
                                dict(DISTILL, lse=P, z_top=P, dloss=P, dx=P, lddx=16, dw=P, lddw=16, dw_dtype=1)),
    "policy_loss": (vk.policy_loss_async, dict(POLICY, reduce=1, stats=P, norm=P)),
    "policy_loss_backward": (vk.policy_loss_backward_async, dict(POLICY, norm=P, dloss=P, dlogp=P, lddp=8)),
}
BIG = 2 ** 31
BAD_DISTILL = [
    dict(dtype=3), dict(x=None), dict(w=None), dict(top=None), dict(t=None), dict(lse=None), dict(z_top=None),
    dict(V=0), dict(K=0), dict(M=BIG), dict(V=BIG), dict(K=BIG, ldx=BIG, ldw=BIG), dict(ldx=15), dict(ldw=15),
    dict(n_top=0),
    dict(n_top=vk.DISTILL_TOP + 1, ldtop=2000, ldt=2000), dict(ldtop=4), dict(ldt=4), dict(t_dtype=2), dict(t_dtype=-1),
    dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=NAN), dict(temperature=INF),
    dict(temperature=1e-44)]
BAD_POLICY = [
    dict(logp=None), dict(old_logp=None), dict(adv=None), dict(norm=None), dict(T=0), dict(B=BIG),
    dict(T=BIG, ldp=BIG, ldo=BIG, ldr=BIG, ldadv=BIG, ldmask=BIG, lddp=BIG), dict(ldp=7), dict(ldo=7), dict(ldr=7),
    dict(ldadv=7), dict(ldadv=0, adv_step=0), dict(adv_step=2), dict(ldmask=7), dict(clip_low=-0.1), dict(clip_low=NAN),
    dict(clip_high=-0.1), dict(clip_high=NAN), dict(kl_coef=NAN), dict(kl_coef=INF)]
BAD = {
    "embedding": [dict(dtype=3), dict(dtype=-1), dict(w_dtype=1), dict(w_dtype=4), dict(ids=None), dict(w=None),
                  dict(y=None), dict(V=0), dict(N=0), dict(M=BIG), dict(V=BIG), dict(N=BIG, ldw=BIG, ldy=BIG),
                  dict(ldw=7), dict(ldy=7), dict(pad_id=2 ** 63), dict(M=-1)],
    "embedding_backward": [dict(dtype=3), dict(dw_dtype=1), dict(ids=None), dict(dy=None), dict(dw=None), dict(V=0),
                           dict(N=0), dict(M=BIG), dict(V=BIG), dict(N=BIG, lddy=BIG, lddw=BIG), dict(lddy=7),
                           dict(lddw=7)],
    "linear_distill": BAD_DISTILL + [dict(loss=None)],
    "linear_distill_backward": BAD_DISTILL + [dict(dloss=None), dict(dw_dtype=2), dict(lddx=15), dict(lddw=15)],
    "policy_loss": [{k: v for k, v in b.items() if k != "lddp"} for b in BAD_POLICY] + [
        dict(reduce=-1), dict(reduce=3), dict(stats=None)],
    "policy_loss_backward": BAD_POLICY + [dict(dloss=None), dict(dlogp=None), dict(lddp=7)],
}


@pytest.mark.parametrize("op,bad", [(op, bad) for op in BAD for bad in BAD[op]], ids=str)
def test_refused(op, bad):
    fn, good = CALLS[op]
    assert fn(**{**good, **bad}, check=False) == vk.ERR_PARAM
    with pytest.raises(vk.VkblasError) as e:
        fn(**{**good, **bad})
    assert e.value.status == vk.ERR_PARAM


def test_an_empty_batch_or_no_output_is_no_error():
    for op, size, unused in (("embedding", "M", "ids"), ("linear_distill", "M", "x"), ("policy_loss", "B", "logp"),
                             ("policy_loss_backward", "B", "logp")):
        fn, good = CALLS[op]
        assert fn(**{**good, size: 0, unused: None}) == vk.OK
    fn, good = CALLS["linear_distill_backward"]
    assert fn(**{**good, "dx": None, "dw": None}) == vk.OK
    assert fn(**{**good, "dx": None, "dw": None, "M": 0}) == vk.OK
    fn, good = CALLS["embedding_backward"]
    assert fn(**{**good, "M": 0, "beta": 1.0}) == vk.OK


def test_leading_dimensions_of_what_is_not_there_are_not_checked():
    for op in ("policy_loss", "policy_loss_backward"):
        fn, good = CALLS[op]
        assert fn(**{**good, "B": 0, "ref_logp": None, "ldr": 0, "mask": None, "ldmask": 0}) == vk.OK
    fn, good = CALLS["linear_distill_backward"]
    assert fn(**{**good, "M": 0, "dw": None, "lddw": 0, "dw_dtype": 7, "dx": None, "lddx": 0}) == vk.OK


def test_header_symbols_are_exported():
    text = open(os.path.join(vk.REPO, "include", "vkblas_train.h")).read()
    names = set(re.findall(r"^vkblas_status_t (vkblas_\w+)\(", text, flags=re.M))
    assert names == {f"vkblas_{n}_async" for n in CALLS}
    assert all(hasattr(vk.load(), n) for n in names)
    assert int(re.search(r"#define VKBLAS_DISTILL_TOP (\d+)", text).group(1)) == vk.DISTILL_TOP


@pytest.mark.parametrize("op", ["linear_distill", "linear_distill_backward"])
def test_temperatures_that_leave_fp32(op):
    """log2(e) / T and T^2 have to be numbers: refused past that, taken up to it."""
    fn, good = CALLS[op]
    for t in (1e-45, 2.95e-39, 4.2e-39, 1.85e19, 1e30, 3e38):
        assert fn(**{**good, "temperature": t}, check=False) == vk.ERR_PARAM, t
        assert fn(**{**good, "temperature": t, "M": 0, "dw": None} if "dw" in good else
                  {**good, "temperature": t, "M": 0}, check=False) == vk.ERR_PARAM, t
    for t in (4.3e-39, 1e-20, 1e10, 1.84e19):
        assert fn(**{**good, "temperature": t, "M": 0, "dw": None} if "dw" in good else
                  {**good, "temperature": t, "M": 0}) == vk.OK, t
