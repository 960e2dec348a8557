"""vkblas_amd -- MI355X-native (gfx950) implementation of vkblas's GEMM hot path.

The product is ``libvkblas_hipblas.so`` in this directory: the reference's
public C API (``include/vkblas.h``), its hipBLAS ABI entry points (an
``LD_PRELOAD`` drop-in for PyTorch-ROCm) and the stream-aware extension
(``include/vkblas_ext.h``), all running hand-written gfx950 HIP kernels.

This module is the Python host-side binding used by the tests, the benchmark
and ``__graft_entry__``: it loads the built library with ctypes and mirrors the
engine entry points (``vkblas_gemm_f32`` / ``vkblas_gemm_f16`` of the
reference's ``src/vkblas.h:27-77``) with the same argument meaning and status
codes.  There is no fallback: if the library is missing, loading raises.
The asynchronous GEMMs and the operators of ``include/vkblas_nn.h`` and
``include/vkblas_train.h`` (embedding, layer norm, gated projection, linear cross entropy
and distillation, policy loss, with their gradients; ``torch_nn`` wraps them for autograd)
go through ``_call`` (csrc/pycall.c), which converts their arguments natively; arguments it does not know, and every call of an
interpreter it is not built for, go through ctypes.
"""
from __future__ import annotations

import ctypes
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
LIB_NAME = "libvkblas_hipblas.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)
# the host dispatcher and kernels, opened by LIB_PATH's first call
ENGINE_PATH = os.path.join(HERE, "libvkblas_engine.so")

# vkblas_status_t (reference src/vkblas.h:6-12)
OK, ERR_INIT, ERR_IMPORT, ERR_PARAM, ERR_FALLBACK = 0, 1, 2, 3, 4
STATUS_NAMES = {0: "VKBLAS_OK", 1: "VKBLAS_ERR_INIT", 2: "VKBLAS_ERR_IMPORT", 3: "VKBLAS_ERR_PARAM",
                4: "VKBLAS_ERR_FALLBACK"}
# vkblas_op_t
OP_N, OP_T = 0, 1
# vkblas_dtype_t
DT_F32, DT_F16, DT_BF16 = 0, 1, 2
# vkblas_scalar_mode_t
SCALAR_HOST, SCALAR_DEV_F32, SCALAR_DEV_F16 = 0, 1, 2
# vkblas_act_t (include/vkblas_nn.h)
ACT_SILU, ACT_GELU, ACT_GELU_TANH, ACT_RELU = range(4)
# vkblas_reduce_t (include/vkblas_train.h)
REDUCE_TOKENS, REDUCE_SEQUENCES, REDUCE_SUM = range(3)
# the most entries of a row in linear_distill_async (VKBLAS_DISTILL_TOP)
DISTILL_TOP = 1024
# vkblas_path_t
PATH_NONE, PATH_TILE64, PATH_TILE128, PATH_TILE256, PATH_SPLITK, PATH_SKINNY, PATH_TAIL = range(7)
PATH_NAMES = {0: "none", 1: "tile64", 2: "tile128", 3: "tile256", 4: "splitk", 5: "skinny", 6: "tail"}


class VkblasError(RuntimeError):
    def __init__(self, status: int, what: str = "vkblas call"):
        super().__init__(f"{what} failed: {STATUS_NAMES.get(status, status)}")
        self.status = status


class Epilogue(ctypes.Structure):
    """vkblas_epilogue_t: C = alpha * op(A) op(B) + beta * c_in + bias[n]."""
    _fields_ = [("c_in", ctypes.c_void_p), ("ldc_in", ctypes.c_uint32), ("stride_c_in", ctypes.c_int64),
                ("bias", ctypes.c_void_p), ("bias_type", ctypes.c_int)]


class Plan(ctypes.Structure):
    _fields_ = [("path", ctypes.c_int), ("tile", ctypes.c_int), ("split", ctypes.c_uint32),
                ("k_per_split", ctypes.c_uint32), ("tail_rows", ctypes.c_uint32)]


def _ctypes_call(*args):
    return None


_lib = None
_native = _ctypes_call      # vkblas_amd._call.gemm_ex where load() finds it
_ex_addr = 0        # address of vkblas_gemm_ex_async

_u32, _i64, _f, _vp, _int = ctypes.c_uint32, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p, ctypes.c_int
_ENGINE_ARGS = [_int, _int, _u32, _u32, _u32, _f, _vp, _u32, _vp, _u32, _f, _vp, _u32, _u32, _i64, _i64, _i64]


# include/vkblas_nn.h and vkblas_train.h: the arguments of vkblas_<name>_async
_NN_ARGS = {
    "layer_norm": [_int, _int, _u32, _u32, _vp, _u32, _vp, _vp, _f, _vp, _u32, _vp, _vp, _vp],
    "layer_norm_backward": [_int, _int, _u32, _u32, _vp, _u32, _vp, _u32, _vp, _vp, _vp, _vp, _u32, _vp,
                                         _vp, _int, _f, _vp],
    "glu": [_int, _int, _u32, _u32, _u32, _vp, _u32, _vp, _u32, _vp, _u32, _vp, _u32, _vp],
    "glu_backward": [_int, _int, _u32, _u32, _u32, _vp, _u32, _vp, _u32, _vp, _u32, _vp, _u32, _vp, _u32,
                                  _vp, _u32, _vp, _u32, _int, _f, _vp],
    "linear_xent": [_int, _u32, _u32, _u32, _vp, _u32, _vp, _u32, _vp, _i64, _vp, _vp, _vp],
    "linear_xent_backward": [_int, _u32, _u32, _u32, _vp, _u32, _vp, _u32, _vp, _i64, _vp, _vp, _vp, _u32,
                                          _vp, _u32, _int, _f, _vp],
    "embedding": [_int, _int, _u32, _u32, _u32, _vp, _i64, _vp, _u32, _f, _vp, _u32, _vp],
    "embedding_backward": [_int, _u32, _u32, _u32, _vp, _i64, _vp, _u32, _f, _vp, _u32, _int, _f, _vp],
    "linear_distill": [_int, _u32, _u32, _u32, _vp, _u32, _vp, _u32, _u32, _vp, _u32, _int, _vp, _u32, _f, _vp, _vp,
                       _vp, _vp],
    "linear_distill_backward": [_int, _u32, _u32, _u32, _vp, _u32, _vp, _u32, _u32, _vp, _u32, _int, _vp, _u32, _f, _vp,
                                _vp, _vp, _vp, _u32, _vp, _u32, _int, _f, _vp],
    "policy_loss": [_int, _u32, _u32, _vp, _u32, _vp, _u32, _vp, _u32, _vp, _u32, _u32, _vp, _u32, _f, _f, _f, _vp, _vp,
                    _vp],
    "policy_loss_backward": [_u32, _u32, _vp, _u32, _vp, _u32, _vp, _u32, _vp, _u32, _u32, _vp, _u32, _f, _f, _f, _vp,
                             _vp, _vp, _u32, _vp],
}


# the kinds of those arguments, as _call.fits and _fits take them
_NN_KINDS = {name: "".join({_u32: "u", _int: "i", _i64: "l"}.get(t, ".") for t in args)
             for name, args in _NN_ARGS.items()}
_RANGES = {"u": (0, 2 ** 32 - 1), "i": (-2 ** 31, 2 ** 31 - 1), "l": (-2 ** 63, 2 ** 63 - 1)}
_nn_calls = {}      # by name: the native call, the function's address, the function


def _fits(kinds, *args) -> bool:
    """Whether the C types hold the whole numbers among args (_call.fits where that is not there)."""
    return all(_RANGES[k][0] <= a <= _RANGES[k][1] for k, a in zip(kinds, args) if k in _RANGES and isinstance(a, int))


_range_check = _fits


def build(jobs: int = 8) -> None:
    """Compile every HIP kernel for gfx950 and link libvkblas_hipblas.so."""
    subprocess.run(["make", "-s", "-C", HERE, f"-j{jobs}", "-B"], check=True)


def load():
    """Load the built library (raises if it has not been built)."""
    global _lib, _native, _ex_addr, _range_check, _nn_calls
    if _lib is not None:
        return _lib
    for path in (LIB_PATH, ENGINE_PATH):
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: run __graft_entry__.build() (make -C vkblas_amd)")
    L = ctypes.CDLL(LIB_PATH)
    for name in ("vkblas_gemm_f32", "vkblas_gemm_f16", "vkblas_gemm_bf16", "vkblas_gemm_bf16_hipblas"):
        fn = getattr(L, name)
        fn.argtypes = _ENGINE_ARGS
        fn.restype = _int
    L.vkblas_gemm_async.argtypes = [_int, _int, _int, _int, _u32, _u32, _u32, _f, _vp, _u32, _vp, _u32, _f, _vp,
                                    _u32, _u32, _i64, _i64, _i64, _int, _vp, _vp, _u32, _vp]
    L.vkblas_gemm_async.restype = _int
    L.vkblas_gemm_ex_async.argtypes = L.vkblas_gemm_async.argtypes[:-1] + [ctypes.POINTER(Epilogue), _vp]
    L.vkblas_gemm_ex_async.restype = _int
    L.vkblas_gemm_batched_async.argtypes = [_int, _int, _int, _int, _u32, _u32, _u32, _f, _vp, _u32, _vp, _u32, _f,
                                            _vp, _u32, _u32, _int, _vp, _vp, _vp]
    L.vkblas_gemm_batched_async.restype = _int
    L.vkblas_plan_gemm.argtypes = [_int, _int, _int, _int, _u32, _u32, _u32, _u32, _u32, _u32, _u32, _u32, _int,
                                   ctypes.POINTER(Plan)]
    L.vkblas_plan_gemm.restype = _int
    L.vkblas_last_path.restype = _int
    L.vkblas_set_override.argtypes = [_int, _int]
    L.vkblas_set_override.restype = _int
    L.vkblas_version.restype = ctypes.c_char_p
    L.vkblas_cache_invalidate_base.argtypes = [_vp]
    L.vkblas_cache_invalidate_base.restype = None
    L.vkblas_last_kernel.restype = _int
    L.vkblas_workspace_release.restype = _int
    L.vkblas_gemm_noalloc_async.argtypes = L.vkblas_gemm_async.argtypes
    L.vkblas_gemm_noalloc_async.restype = _int
    L.vkblas_noalloc_scratch_bytes.restype = ctypes.c_size_t
    try:
        from . import _call
    except ImportError:     # not built, or for another interpreter
        _call = None
        _range_check = _fits
    else:
        _range_check = getattr(_call, "fits", _fits)
        _native, _ex_addr = _call.gemm_ex, ctypes.cast(L.vkblas_gemm_ex_async, ctypes.c_void_p).value
    calls = {}          # published whole: another thread may look while this one loads
    for name, args in _NN_ARGS.items():
        fn = getattr(L, f"vkblas_{name}_async")
        fn.argtypes = args
        fn.restype = _int
        calls[name] = (getattr(_call, name, _ctypes_call), ctypes.cast(fn, ctypes.c_void_p).value, fn)
    _nn_calls = calls
    _lib = L
    return L


def version() -> str:
    return load().vkblas_version().decode()


def plan(ab_type, c_type, op_a, op_b, M, N, K, lda, ldb, ldc, batch=1, split_k=0, aligned=True) -> Plan:
    p = Plan()
    st = load().vkblas_plan_gemm(ab_type, c_type, op_a, op_b, M, N, K, lda, ldb, ldc, batch, split_k,
                                 1 if aligned else 0, ctypes.byref(p))
    if st != OK:
        raise VkblasError(st, "vkblas_plan_gemm")
    return p


def set_override(tile: int = -1, generic: bool = False) -> None:
    """Force a tile (-1 planner, 0: 64, 1: 128, 2: 256) / the generic kernel."""
    st = load().vkblas_set_override(tile, 1 if generic else 0)
    if st != OK:
        raise VkblasError(st, "vkblas_set_override")


def last_path() -> int:
    return load().vkblas_last_path()


# vkblas_kernel_t (include/vkblas_ext.h)
KERNEL_NONE, KERNEL_GENERIC, KERNEL_GENERIC_CHECKED, KERNEL_PIPE256, KERNEL_PIPE128, KERNEL_PIPE128_4, \
    KERNEL_SKINNY, KERNEL_WAVEK, KERNEL_DIRECT, KERNEL_FLOW, KERNEL_NORM, KERNEL_NORM_LONG, \
    KERNEL_JOINED, KERNEL_FUSED, KERNEL_FEW, KERNEL_EMBED, KERNEL_POLICY = range(17)


def workspace_release() -> None:
    """vkblas_workspace_release: free the per-stream partial buffers."""
    st = load().vkblas_workspace_release()
    if st != OK:
        raise VkblasError(st, "vkblas_workspace_release")


def last_kernel() -> int:
    """vkblas_kernel_t of the calling thread's most recent successful GEMM."""
    return load().vkblas_last_kernel()


def gemm_async(ab_type, c_type, op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch=1,
               stride_a=0, stride_b=0, stride_c=0, scalar_mode=SCALAR_HOST, alpha_dev=None, beta_dev=None,
               split_k=0, stream=None, check=True) -> int:
    """vkblas_gemm_async on raw device pointers (ints).  Row-major engine
    contract of src/vkblas.h:21-26.  Returns the status (raises if check)."""
    if _lib is None:
        load()
    st = _native(_ex_addr, ab_type, c_type, op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch,
                 stride_a, stride_b, stride_c, scalar_mode, alpha_dev, beta_dev, split_k, 0, None, 0, 0, None, 0,
                 stream)
    if st is None:
        st = _lib.vkblas_gemm_async(ab_type, c_type, op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc,
                                    batch, stride_a, stride_b, stride_c, scalar_mode, alpha_dev, beta_dev, split_k,
                                    stream)
    if check and st != OK:
        raise VkblasError(st, "vkblas_gemm_async")
    return st


def gemm_ex_async(ab_type, c_type, op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch=1,
                  stride_a=0, stride_b=0, stride_c=0, scalar_mode=SCALAR_HOST, alpha_dev=None, beta_dev=None,
                  split_k=0, c_in=None, ldc_in=0, stride_c_in=0, bias=None, bias_type=DT_F32, stream=None,
                  check=True) -> int:
    """vkblas_gemm_ex_async: gemm_async with a separate C input (c_in, beta's
    matrix) and a bias vector (one value per column n of C)."""
    if _lib is None:
        load()
    st = _native(_ex_addr, ab_type, c_type, op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch,
                 stride_a, stride_b, stride_c, scalar_mode, alpha_dev, beta_dev, split_k, 1, c_in, ldc_in,
                 stride_c_in, bias, bias_type, stream)
    if st is None:
        ep = Epilogue(c_in, ldc_in, stride_c_in, bias, bias_type)
        st = _lib.vkblas_gemm_ex_async(ab_type, c_type, op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc,
                                       batch, stride_a, stride_b, stride_c, scalar_mode, alpha_dev, beta_dev,
                                       split_k, ctypes.byref(ep), stream)
    if check and st != OK:
        raise VkblasError(st, "vkblas_gemm_ex_async")
    return st


def gemm_noalloc_async(ab_type, c_type, op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch=1,
                       stride_a=0, stride_b=0, stride_c=0, scalar_mode=SCALAR_HOST, alpha_dev=None, beta_dev=None,
                       split_k=0, stream=None, check=True) -> int:
    """vkblas_gemm_noalloc_async: gemm_async with the partials in the library's
    per-device scratch array (allocates nothing)."""
    st = load().vkblas_gemm_noalloc_async(ab_type, c_type, op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C,
                                          ldc, batch, stride_a, stride_b, stride_c, scalar_mode, alpha_dev, beta_dev,
                                          split_k, stream)
    if check and st != OK:
        raise VkblasError(st, "vkblas_gemm_noalloc_async")
    return st


def noalloc_scratch_bytes() -> int:
    return load().vkblas_noalloc_scratch_bytes()


def gemm_batched_async(ab_type, c_type, op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch,
                       scalar_mode=SCALAR_HOST, alpha_dev=None, beta_dev=None, stream=None, check=True) -> int:
    """vkblas_gemm_batched_async: A, B, C are device addresses of arrays of
    `batch` matrix pointers (pointer-array batched GEMM)."""
    st = load().vkblas_gemm_batched_async(ab_type, c_type, op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc,
                                          batch, scalar_mode, alpha_dev, beta_dev, stream)
    if check and st != OK:
        raise VkblasError(st, "vkblas_gemm_batched_async")
    return st


def _nn(name, check, *args) -> int:
    """A call of vkblas_nn.h or vkblas_train.h; its status (raises if check).  A number that its C type
    does not hold is refused like the sizes that the library refuses, not passed as what is left of it."""
    if not _nn_calls:
        load()
    native, addr, fn = _nn_calls[name]
    if not _range_check(_NN_KINDS[name], *args):
        st = ERR_PARAM
    else:
        st = native(addr, *args)
        if st is None:
            st = fn(*args)
    if check and st != OK:
        raise VkblasError(st, f"vkblas_{name}_async")
    return st


def layer_norm_async(dtype, w_dtype, M, N, x, ldx, w, b, eps, y, ldy, mean=None, rstd=None, stream=None,
                     check=True) -> int:
    """vkblas_layer_norm_async: y = (x - mean) * rstd * w + b over M rows of N;
    mean and rstd (M floats each) kept where given."""
    return _nn("layer_norm", check, dtype, w_dtype, M, N, x, ldx, w, b, eps, y, ldy, mean, rstd, stream)


def layer_norm_backward_async(dtype, w_dtype, M, N, dy, lddy, x, ldx, w, mean, rstd, dx, lddx, dw, db, g_dtype,
                              beta=0.0, stream=None, check=True) -> int:
    """vkblas_layer_norm_backward_async: dx, and dw and db (beta times what
    they held, plus the sums over the rows); each may be None."""
    return _nn("layer_norm_backward", check, dtype, w_dtype, M, N, dy, lddy, x, ldx, w, mean, rstd, dx,
               lddx, dw, db, g_dtype, beta, stream)


def glu_async(dtype, act, M, N, K, x, ldx, w, ldw, h, ldh, gu=None, ldgu=0, stream=None, check=True) -> int:
    """vkblas_glu_async: h = act(G) * U with [G | U] = x w^T (w is 2N x K, the
    gate's rows first); gu (M x 2N) receives [G | U] where given."""
    return _nn("glu", check, dtype, act, M, N, K, x, ldx, w, ldw, h, ldh, gu, ldgu, stream)


def glu_backward_async(dtype, act, M, N, K, dh, lddh, gu, ldgu, x, ldx, w, ldw, dgu, lddgu, dx, lddx, dw, lddw,
                       dw_dtype, beta=0.0, stream=None, check=True) -> int:
    """vkblas_glu_backward_async: dgu = [dG | dU], dx = dgu w and dw = beta dw
    + dgu^T x; each may be None."""
    return _nn("glu_backward", check, dtype, act, M, N, K, dh, lddh, gu, ldgu, x, ldx, w, ldw, dgu, lddgu,
               dx, lddx, dw, lddw, dw_dtype, beta, stream)


def linear_xent_async(dtype, M, V, K, x, ldx, w, ldw, target, ignore_index, loss, lse, stream=None,
                      check=True) -> int:
    """vkblas_linear_xent_async: each row's cross entropy (loss) and
    log-sum-exp (lse) of the logits x w^T, which are not kept."""
    return _nn("linear_xent", check, dtype, M, V, K, x, ldx, w, ldw, target, ignore_index, loss, lse,
               stream)


def linear_xent_backward_async(dtype, M, V, K, x, ldx, w, ldw, target, ignore_index, lse, dloss, dx, lddx, dw, lddw,
                               dw_dtype, beta=0.0, stream=None, check=True) -> int:
    """vkblas_linear_xent_backward_async: dx and dw = beta dw + D^T x from the
    rows' loss gradients; each may be None."""
    return _nn("linear_xent_backward", check, dtype, M, V, K, x, ldx, w, ldw, target, ignore_index, lse,
               dloss, dx, lddx, dw, lddw, dw_dtype, beta, stream)


def embedding_async(dtype, w_dtype, M, V, N, ids, pad_id, w, ldw, scale, y, ldy, stream=None, check=True) -> int:
    """vkblas_embedding_async: y[m] = scale * w[ids[m]], zeros where ids[m] is
    pad_id."""
    return _nn("embedding", check, dtype, w_dtype, M, V, N, ids, pad_id, w, ldw, scale, y, ldy, stream)


def embedding_backward_async(dtype, M, V, N, ids, pad_id, dy, lddy, scale, dw, lddw, dw_dtype, beta=0.0, stream=None,
                             check=True) -> int:
    """vkblas_embedding_backward_async: dw = beta dw + scale times the sums of
    each id's rows of dy."""
    return _nn("embedding_backward", check, dtype, M, V, N, ids, pad_id, dy, lddy, scale, dw, lddw, dw_dtype, beta,
               stream)


def linear_distill_async(dtype, M, V, K, x, ldx, w, ldw, n_top, top, ldtop, t_dtype, t, ldt, temperature, loss, lse,
                         z_top, stream=None, check=True) -> int:
    """vkblas_linear_distill_async: each row's distillation loss from the
    teacher's top logits t at the classes top (M x n_top, negative: absent),
    log-sum-exp of the tempered logits of x w^T, and z_top (M x n_top), those
    logits at the classes."""
    return _nn("linear_distill", check, dtype, M, V, K, x, ldx, w, ldw, n_top, top, ldtop, t_dtype, t, ldt, temperature,
               loss, lse, z_top, stream)


def linear_distill_backward_async(dtype, M, V, K, x, ldx, w, ldw, n_top, top, ldtop, t_dtype, t, ldt, temperature, lse,
                                  z_top, dloss, dx, lddx, dw, lddw, dw_dtype, beta=0.0, stream=None,
                                  check=True) -> int:
    """vkblas_linear_distill_backward_async: dx and dw = beta dw + D^T x from the
    rows' loss gradients; each may be None."""
    return _nn("linear_distill_backward", check, dtype, M, V, K, x, ldx, w, ldw, n_top, top, ldtop, t_dtype, t, ldt,
               temperature, lse, z_top, dloss, dx, lddx, dw, lddw, dw_dtype, beta, stream)


def policy_loss_async(reduce, B, T, logp, ldp, old_logp, ldo, ref_logp, ldr, adv, ldadv, adv_step, mask, ldmask,
                      clip_low, clip_high, kl_coef, stats, norm, stream=None, check=True) -> int:
    """vkblas_policy_loss_async: the clipped policy loss with a KL term of B
    sequences of T tokens; stats (4 floats): loss, KL term, bounds taken, ratio,
    by weight; norm (B floats): a token's weight."""
    return _nn("policy_loss", check, reduce, B, T, logp, ldp, old_logp, ldo, ref_logp, ldr, adv, ldadv, adv_step, mask,
               ldmask, clip_low, clip_high, kl_coef, stats, norm, stream)


def policy_loss_backward_async(B, T, logp, ldp, old_logp, ldo, ref_logp, ldr, adv, ldadv, adv_step, mask, ldmask,
                               clip_low, clip_high, kl_coef, norm, dloss, dlogp, lddp, stream=None, check=True) -> int:
    """vkblas_policy_loss_backward_async: dlogp from dloss (one float on the
    device) and norm."""
    return _nn("policy_loss_backward", check, B, T, logp, ldp, old_logp, ldo, ref_logp, ldr, adv, ldadv, adv_step, mask,
               ldmask, clip_low, clip_high, kl_coef, norm, dloss, dlogp, lddp, stream)


def gemm_f32(op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch=1, sa=0, sb=0, sc=0) -> int:
    """vkblas_gemm_f32 (reference src/vkblas.h:27-36); returns the status."""
    return load().vkblas_gemm_f32(op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch, sa, sb, sc)


def gemm_f16(op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch=1, sa=0, sb=0, sc=0) -> int:
    """vkblas_gemm_f16 (reference src/vkblas.h:68-77); returns the status."""
    return load().vkblas_gemm_f16(op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch, sa, sb, sc)


def gemm_bf16(op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch=1, sa=0, sb=0, sc=0) -> int:
    """vkblas_gemm_bf16 (reference src/vkblas.h:41-50); returns the status."""
    return load().vkblas_gemm_bf16(op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch, sa, sb, sc)


def gemm_bf16_hipblas(op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch=1, sa=0, sb=0, sc=0) -> int:
    """vkblas_gemm_bf16_hipblas (reference src/vkblas.h:55-64); returns the status."""
    return load().vkblas_gemm_bf16_hipblas(op_a, op_b, M, N, K, alpha, A, lda, B, ldb, beta, C, ldc, batch, sa, sb,
                                           sc)


def hipblas():
    """The library's hipBLAS entry points, typed for ctypes callers."""
    from . import hipblas_abi
    return hipblas_abi.bind(load())
