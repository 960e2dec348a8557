/*
 * pycall.c — the Python binding's calls without ctypes (module
 * vkblas_amd._call): vkblas_gemm_ex_async and the functions of vkblas_nn.h
 * and vkblas_train.h, and the check of those functions' numbers against their C types.
 *
 * A small call is bound by its launch on the host, and ctypes' conversion of
 * 25 arguments was the largest part of that: 3.1 us for vkblas_gemm_async and
 * 3.7 for vkblas_gemm_ex_async with its structure, of about 8 a call.  Here
 * the arguments are read from the interpreter's vector directly.
 *
 * Arguments are converted as the ctypes prototypes of vkblas_amd/__init__.py
 * do: integers modulo 2^32 or 2^64, pointers from an int or None, floats from a
 * float or an int.  Anything else (a ctypes object, a subclass) returns None
 * and the caller makes the call through ctypes, whose rules then apply.  The
 * GIL is released during the call, as ctypes releases it.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include "vkblas_train.h"

typedef vkblas_status_t (*gemm_ex_fn)(vkblas_dtype_t, vkblas_dtype_t, vkblas_op_t, vkblas_op_t, uint32_t, uint32_t,
                                      uint32_t, float, const void*, uint32_t, const void*, uint32_t, float, void*,
                                      uint32_t, uint32_t, int64_t, int64_t, int64_t, vkblas_scalar_mode_t,
                                      const void*, const void*, uint32_t, const vkblas_epilogue_t*, void*);

/* 1 and *v, or 0: not a plain int */
static int get_int(PyObject* o, unsigned long long* v) {
    if (!PyLong_CheckExact(o)) return 0;
    *v = PyLong_AsUnsignedLongLongMask(o);
    return !(*v == (unsigned long long)-1 && PyErr_Occurred());
}
static int get_ptr(PyObject* o, unsigned long long* v) {
    *v = 0;
    return o == Py_None || get_int(o, v);
}
static int get_float(PyObject* o, float* v) {
    if (PyFloat_CheckExact(o)) {
        *v = (float)PyFloat_AS_DOUBLE(o);
        return 1;
    }
    if (!PyLong_CheckExact(o)) return 0;
    const double d = PyLong_AsDouble(o);
    if (d == -1.0 && PyErr_Occurred()) return 0;
    *v = (float)d;
    return 1;
}

/* gemm_ex(address of vkblas_gemm_ex_async, its 23 arguments up to split_k,
 * use_epilogue, c_in, ldc_in, stride_c_in, bias, bias_type, stream) */
enum { NARGS = 31 };
static PyObject* gemm_ex(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    if (n != NARGS) return PyErr_Format(PyExc_TypeError, "gemm_ex takes %d arguments (%zd given)", (int)NARGS, n);
    /* i: int, p: pointer, f: float, in the order of the arguments */
    static const char kind[] = "piiiiiiifpipifpiiiiiippiipiipip";
    unsigned long long v[NARGS];
    float alpha = 0.0f, beta = 0.0f;
    for (int k = 0; k < NARGS; ++k) {
        const int ok = kind[k] == 'i' ? get_int(a[k], &v[k])
                     : kind[k] == 'p' ? get_ptr(a[k], &v[k]) : get_float(a[k], k == 8 ? &alpha : &beta);
        if (!ok) {
            PyErr_Clear();
            Py_RETURN_NONE;
        }
    }
    if (!v[0]) return PyErr_Format(PyExc_ValueError, "no function address");
    const gemm_ex_fn fn = (gemm_ex_fn)(uintptr_t)v[0];
    vkblas_epilogue_t ep = {(const void*)(uintptr_t)v[25], (uint32_t)v[26], (int64_t)v[27],
                            (const void*)(uintptr_t)v[28], (vkblas_dtype_t)(int)v[29]};
    int st;
    Py_BEGIN_ALLOW_THREADS
    st = (int)fn((vkblas_dtype_t)(int)v[1], (vkblas_dtype_t)(int)v[2], (vkblas_op_t)(int)v[3], (vkblas_op_t)(int)v[4],
                 (uint32_t)v[5], (uint32_t)v[6], (uint32_t)v[7], alpha, (const void*)(uintptr_t)v[9], (uint32_t)v[10],
                 (const void*)(uintptr_t)v[11], (uint32_t)v[12], beta, (void*)(uintptr_t)v[14], (uint32_t)v[15],
                 (uint32_t)v[16], (int64_t)v[17], (int64_t)v[18], (int64_t)v[19], (vkblas_scalar_mode_t)(int)v[20],
                 (const void*)(uintptr_t)v[21], (const void*)(uintptr_t)v[22], (uint32_t)v[23], v[24] ? &ep : NULL,
                 (void*)(uintptr_t)v[30]);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(st);
}

/* v[k] and f[] (the floats in order) from n arguments of these kinds; 1, or
 * 0 with *result set: an exception (NULL) or None */
static int get_args(const char* name, const char* kind, PyObject* const* a, Py_ssize_t n, unsigned long long* v,
                    float* f, PyObject** result) {
    *result = NULL;
    const Py_ssize_t want = (Py_ssize_t)strlen(kind);
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (%zd given)", name, want, n);
        return 0;
    }
    for (Py_ssize_t k = 0; k < n; ++k) {
        const int ok = kind[k] == 'i' ? get_int(a[k], &v[k]) : kind[k] == 'p' ? get_ptr(a[k], &v[k]) : get_float(a[k], f);
        if (!ok) {
            PyErr_Clear();
            Py_INCREF(Py_None);
            *result = Py_None;
            return 0;
        }
        if (kind[k] == 'f') ++f;
    }
    if (!v[0]) {
        PyErr_Format(PyExc_ValueError, "no function address");
        return 0;
    }
    return 1;
}

/* name(address of vkblas_<name>_async, its arguments): KIND starts with the
 * address; CALL is the call's argument list in terms of v[] and f[] */
#define P(k) ((void*)(uintptr_t)v[k])
#define U(k) ((uint32_t)v[k])
#define I(k) ((int)v[k])
#define NN_CALL(NAME, KIND, CALL)                                                                  \
    static PyObject* NAME(PyObject* self, PyObject* const* a, Py_ssize_t n) {                      \
        (void)self;                                                                                \
        unsigned long long v[sizeof(KIND)];                                                        \
        float f[3];                                                                                \
        PyObject* result;                                                                          \
        if (!get_args(#NAME, KIND, a, n, v, f, &result)) return result;                            \
        int st;                                                                                    \
        Py_BEGIN_ALLOW_THREADS                                                                     \
        st = (int)((__typeof__(&vkblas_##NAME##_async))(uintptr_t)v[0]) CALL;                      \
        Py_END_ALLOW_THREADS                                                                       \
        return PyLong_FromLong(st);                                                                \
    }

NN_CALL(layer_norm, "piiiipippfpippp",
        (I(1), I(2), U(3), U(4), P(5), U(6), P(7), P(8), f[0], P(10), U(11), P(12), P(13), P(14)))
NN_CALL(layer_norm_backward, "piiiipipippppippifp",
        (I(1), I(2), U(3), U(4), P(5), U(6), P(7), U(8), P(9), P(10), P(11), P(12), U(13), P(14), P(15), I(16), f[0],
         P(18)))
NN_CALL(glu, "piiiiipipipipip",
        (I(1), I(2), U(3), U(4), U(5), P(6), U(7), P(8), U(9), P(10), U(11), P(12), U(13), P(14)))
NN_CALL(glu_backward, "piiiiipipipipipipipiifp",
        (I(1), I(2), U(3), U(4), U(5), P(6), U(7), P(8), U(9), P(10), U(11), P(12), U(13), P(14), U(15), P(16), U(17),
         P(18), U(19), I(20), f[0], P(22)))
NN_CALL(linear_xent, "piiiipipipippp",
        (I(1), U(2), U(3), U(4), P(5), U(6), P(7), U(8), P(9), (int64_t)v[10], P(11), P(12), P(13)))
NN_CALL(linear_xent_backward, "piiiipipipipppipiifp",
        (I(1), U(2), U(3), U(4), P(5), U(6), P(7), U(8), P(9), (int64_t)v[10], P(11), P(12), P(13), U(14), P(15),
         U(16), I(17), f[0], P(19)))

NN_CALL(embedding, "piiiiipipifpip",
        (I(1), I(2), U(3), U(4), U(5), P(6), (int64_t)v[7], P(8), U(9), f[0], P(11), U(12), P(13)))
NN_CALL(embedding_backward, "piiiipipifpiifp",
        (I(1), U(2), U(3), U(4), P(5), (int64_t)v[6], P(7), U(8), f[0], P(10), U(11), I(12), f[1], P(14)))
NN_CALL(linear_distill, "piiiipipiipiipifpppp",
        (I(1), U(2), U(3), U(4), P(5), U(6), P(7), U(8), U(9), P(10), U(11), I(12), P(13), U(14), f[0], P(16), P(17),
         P(18), P(19)))
NN_CALL(linear_distill_backward, "piiiipipiipiipifppppipiifp",
        (I(1), U(2), U(3), U(4), P(5), U(6), P(7), U(8), U(9), P(10), U(11), I(12), P(13), U(14), f[0], P(16), P(17),
         P(18), P(19), U(20), P(21), U(22), I(23), f[1], P(25)))
NN_CALL(policy_loss, "piiipipipipiipifffppp",
        (I(1), U(2), U(3), P(4), U(5), P(6), U(7), P(8), U(9), P(10), U(11), U(12), P(13), U(14), f[0], f[1], f[2], P(18),
         P(19), P(20)))
NN_CALL(policy_loss_backward, "piipipipipiipifffpppip",
        (U(1), U(2), P(3), U(4), P(5), U(6), P(7), U(8), P(9), U(10), U(11), P(12), U(13), f[0], f[1], f[2], P(17), P(18),
         P(19), U(20), P(21)))

/* fits(kinds, arguments): whether the C types hold the whole numbers among
 * them; u: uint32_t, i: int, l: int64_t, anything else is not looked at */
static PyObject* fits(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    Py_ssize_t kinds = 0;
    const char* kind = n > 0 && PyUnicode_Check(a[0]) ? PyUnicode_AsUTF8AndSize(a[0], &kinds) : NULL;
    if (!kind || kinds != n - 1) {
        if (!PyErr_Occurred()) PyErr_Format(PyExc_TypeError, "fits takes the kinds of as many arguments as follow");
        return NULL;
    }
    for (Py_ssize_t k = 0; k < kinds; ++k) {
        PyObject* o = a[k + 1];
        if ((kind[k] != 'u' && kind[k] != 'i' && kind[k] != 'l') || !PyLong_Check(o)) continue;
        int past;
        const long long v = PyLong_AsLongLongAndOverflow(o, &past);
        if (past || (kind[k] == 'u' && (v < 0 || v > 0xffffffffll)) ||
            (kind[k] == 'i' && (v < INT32_MIN || v > INT32_MAX)))
            Py_RETURN_FALSE;
    }
    Py_RETURN_TRUE;
}

static PyMethodDef methods[] = {
                                {"fits", (PyCFunction)(void (*)(void))fits, METH_FASTCALL,
                                 "whether whole numbers lie in their C types' ranges"},
#define NN_METHOD(NAME) {#NAME, (PyCFunction)(void (*)(void))NAME, METH_FASTCALL, \
                         "vkblas_" #NAME "_async by address; None if an argument is not a plain int, float or None"}
                                NN_METHOD(layer_norm), NN_METHOD(layer_norm_backward), NN_METHOD(glu),
                                NN_METHOD(glu_backward), NN_METHOD(linear_xent), NN_METHOD(linear_xent_backward),
                                NN_METHOD(embedding), NN_METHOD(embedding_backward), NN_METHOD(linear_distill),
                                NN_METHOD(linear_distill_backward), NN_METHOD(policy_loss),
                                NN_METHOD(policy_loss_backward),
                                {"gemm_ex", (PyCFunction)(void (*)(void))gemm_ex, METH_FASTCALL,
                                 "vkblas_gemm_ex_async by address; None if an argument is not a plain int, float or None"},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_call", "calls of the binding", -1, methods,
                                    NULL, NULL, NULL, NULL};
PyMODINIT_FUNC PyInit__call(void) { return PyModule_Create(&module); }
