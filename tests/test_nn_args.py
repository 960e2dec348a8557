"""The operators of vkblas_nn.h refuse what they cannot compute before anything is launched (CPU: the pointers
are never followed), and accept empty batches without a GPU where nothing is to be written."""
import os
import re

import pytest

import vkblas_amd as vk

P = 4096    # a pointer that no check follows

CALLS = {
    "layer_norm": (vk.layer_norm_async, dict(dtype=0, w_dtype=0, M=4, N=8, x=P, ldx=8, w=P, b=P, eps=1e-5, y=P, ldy=8)),
    "layer_norm_backward": (vk.layer_norm_backward_async,
                            dict(dtype=1, w_dtype=1, M=4, N=8, dy=P, lddy=8, x=P, ldx=8, w=P, mean=P, rstd=P, dx=P,
                                 lddx=8, dw=P, db=P, g_dtype=1)),
    "glu": (vk.glu_async, dict(dtype=2, act=0, M=4, N=8, K=16, x=P, ldx=16, w=P, ldw=16, h=P, ldh=8, gu=P, ldgu=16)),
    "glu_backward": (vk.glu_backward_async,
                     dict(dtype=1, act=1, M=4, N=8, K=16, dh=P, lddh=8, gu=P, ldgu=16, x=P, ldx=16, w=P, ldw=16, dgu=P,
                          lddgu=16, dx=P, lddx=16, dw=P, lddw=16, dw_dtype=0)),
    "linear_xent": (vk.linear_xent_async, dict(dtype=1, M=4, V=9, K=16, x=P, ldx=16, w=P, ldw=16, target=P,
                                               ignore_index=-100, loss=P, lse=P)),
    "linear_xent_backward": (vk.linear_xent_backward_async,
                             dict(dtype=1, M=4, V=9, K=16, x=P, ldx=16, w=P, ldw=16, target=P, ignore_index=-100,
                                  lse=P, dloss=P, dx=P, lddx=16, dw=P, lddw=16, dw_dtype=1)),
}
BIG = 2 ** 31
BAD = {
    "layer_norm": [dict(dtype=3), dict(dtype=-1), dict(w_dtype=1), dict(x=None), dict(y=None), dict(N=0), dict(M=BIG),
                   dict(N=BIG, ldx=BIG, ldy=BIG), dict(ldx=7), dict(ldy=7)],
    "layer_norm_backward": [dict(dtype=9), dict(w_dtype=2), dict(g_dtype=2), dict(dy=None), dict(x=None),
                            dict(mean=None), dict(rstd=None), dict(N=0), dict(lddy=7), dict(ldx=7), dict(lddx=7)],
    "glu": [dict(dtype=3), dict(act=4), dict(act=-1), dict(x=None), dict(w=None), dict(h=None), dict(N=0), dict(K=0),
            dict(ldx=15), dict(ldw=15), dict(ldh=7), dict(ldgu=15), dict(N=2 ** 30, ldh=2 ** 30, ldgu=BIG)],
    "glu_backward": [dict(dtype=3), dict(act=4), dict(dh=None), dict(gu=None), dict(x=None), dict(w=None),
                     dict(dw_dtype=2), dict(N=0), dict(K=0), dict(lddh=7), dict(ldgu=15), dict(ldx=15), dict(ldw=15),
                     dict(lddgu=15), dict(lddx=15), dict(lddw=15)],
    "linear_xent": [dict(dtype=3), dict(x=None), dict(w=None), dict(target=None), dict(lse=None), dict(V=0), dict(K=0),
                    dict(ldx=15), dict(ldw=15), dict(M=BIG), dict(V=BIG)],
    "linear_xent_backward": [dict(dtype=3), dict(x=None), dict(w=None), dict(target=None), dict(lse=None),
                             dict(dloss=None), dict(dw_dtype=2), dict(V=0), dict(K=0), dict(ldx=15), dict(ldw=15),
                             dict(lddx=15), dict(lddw=15)],
}


@pytest.mark.parametrize("op,bad", [(op, bad) for op in BAD for bad in BAD[op]], ids=str)
def test_refused(op, bad):
    fn, good = CALLS[op]
    assert fn(**{**good, **bad}, check=False) == vk.ERR_PARAM
    with pytest.raises(vk.VkblasError) as e:
        fn(**{**good, **bad})
    assert e.value.status == vk.ERR_PARAM


def test_an_empty_batch_or_no_output_is_no_error():
    for op in ("layer_norm", "glu", "linear_xent"):
        fn, good = CALLS[op]
        assert fn(**{**good, "M": 0, "x": None}) == vk.OK
    for op, none in (("layer_norm_backward", ("dx", "dw", "db")), ("glu_backward", ("dgu", "dx", "dw")),
                     ("linear_xent_backward", ("dx", "dw"))):
        fn, good = CALLS[op]
        assert fn(**{**good, **dict.fromkeys(none)}) == vk.OK
        assert fn(**{**good, **dict.fromkeys(none), "M": 0}) == vk.OK


def test_leading_dimensions_of_what_is_not_computed_are_not_checked():
    fn, good = CALLS["glu"]
    assert fn(**{**good, "M": 0, "gu": None, "ldgu": 0}) == vk.OK
    fn, good = CALLS["glu_backward"]
    assert fn(**{**good, "M": 0, "dw": None, "lddw": 0, "ldx": 0, "dgu": None, "lddgu": 0}) == vk.OK


def test_header_symbols_are_exported():
    text = open(os.path.join(vk.REPO, "include", "vkblas_nn.h")).read()
    names = set(re.findall(r"^vkblas_status_t (vkblas_\w+)\(", text, flags=re.M))
    assert len(names) == 6
    assert all(hasattr(vk.load(), n) for n in names)
