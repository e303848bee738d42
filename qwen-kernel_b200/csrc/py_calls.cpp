// The calls a decode step makes most often, as a CPython extension module over the C ABI (include/qk_moe.h).
//
// A call through ctypes converts eight arguments and looks three pointers up in Python: 2.4 us, as long as the host part of a
// kernel launch.  Here it is 0.4 us.  Arguments are what the ctypes signatures take; a pointer is None, an int, an object with
// data_ptr() (a torch tensor) or one with ptr (DevBuf).  Every function returns the C ABI's return code and runs without the GIL.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <tuple>
#include <type_traits>
#include <utility>

#include "../../include/qk_moe.h"

namespace {

PyObject *s_data_ptr, *s_ptr;   // interned names

bool pointer(PyObject* o, void** out) {
    if (PyLong_CheckExact(o)) { *out = PyLong_AsVoidPtr(o); return !PyErr_Occurred(); }
    if (o == Py_None) { *out = nullptr; return true; }
    PyObject* r = PyObject_CallMethodNoArgs(o, s_data_ptr);
    if (!r && PyErr_ExceptionMatches(PyExc_AttributeError)) {
        PyErr_Clear();
        r = PyObject_GetAttr(o, s_ptr);
        if (!r && PyErr_ExceptionMatches(PyExc_AttributeError)) { PyErr_Clear(); r = PyNumber_Long(o); }
    }
    if (!r) return false;
    if (r == Py_None) *out = nullptr;
    else *out = PyLong_AsVoidPtr(r);
    Py_DECREF(r);
    return !PyErr_Occurred();
}
bool u32(PyObject* o, uint32_t* out) {
    *out = (uint32_t)PyLong_AsUnsignedLongMask(o);
    return !PyErr_Occurred();
}
bool f32(PyObject* o, float* out) {
    *out = (float)PyFloat_AsDouble(o);
    return !PyErr_Occurred();
}
bool count(const char* name, Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, want, n);
    return false;
}
template <typename F>
PyObject* run(F f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

// (ctx, type, W, x, y, M, K, n)
PyObject* gemv(PyObject*, PyObject* const* a, Py_ssize_t n) {
    void *c, *w, *x, *y;
    uint32_t type, M, K, rows;
    if (!count("gemv", n, 8) || !pointer(a[0], &c) || !u32(a[1], &type) || !pointer(a[2], &w) || !pointer(a[3], &x) || !pointer(a[4], &y) ||
        !u32(a[5], &M) || !u32(a[6], &K) || !u32(a[7], &rows)) return nullptr;
    return run([&] { return qkm_gemv((qkm_ctx*)c, type, w, (const float*)x, (float*)y, M, K, rows); });
}
// (ctx, index, x, n, y)
template <int (*F)(qkm_ctx*, uint32_t, const float*, uint32_t, float*)>
PyObject* rows_call(PyObject*, PyObject* const* a, Py_ssize_t n) {
    void *c, *x, *y;
    uint32_t index, rows;
    if (!count("call", n, 5) || !pointer(a[0], &c) || !u32(a[1], &index) || !pointer(a[2], &x) || !u32(a[3], &rows) || !pointer(a[4], &y)) return nullptr;
    return run([&] { return F((qkm_ctx*)c, index, (const float*)x, rows, (float*)y); });
}
// (ctx, first, count, x, n, y)
template <int (*F)(qkm_ctx*, uint32_t, uint32_t, const float*, uint32_t, float*)>
PyObject* stack_call(PyObject*, PyObject* const* a, Py_ssize_t n) {
    void *c, *x, *y;
    uint32_t first, layers, rows;
    if (!count("call", n, 6) || !pointer(a[0], &c) || !u32(a[1], &first) || !u32(a[2], &layers) || !pointer(a[3], &x) || !u32(a[4], &rows) ||
        !pointer(a[5], &y)) return nullptr;
    return run([&] { return F((qkm_ctx*)c, first, layers, (const float*)x, rows, (float*)y); });
}
// (ctx, logits, n_rows, n, tok)
PyObject* argmax(PyObject*, PyObject* const* a, Py_ssize_t n) {
    void *c, *l, *t;
    uint32_t rows, len;
    if (!count("argmax", n, 5) || !pointer(a[0], &c) || !pointer(a[1], &l) || !u32(a[2], &rows) || !u32(a[3], &len) || !pointer(a[4], &t)) return nullptr;
    return run([&] { return qkm_argmax((qkm_ctx*)c, (const float*)l, rows, len, (uint32_t*)t); });
}
// (ctx, layer, resid, attn_out, w_post, w_next, n, eps, resid_out, xn_next)
PyObject* layer_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
    void *c, *p[6];
    uint32_t layer, rows;
    float eps;
    if (!count("layer_step", n, 10) || !pointer(a[0], &c) || !u32(a[1], &layer) || !pointer(a[2], &p[0]) || !pointer(a[3], &p[1]) || !pointer(a[4], &p[2]) ||
        !pointer(a[5], &p[3]) || !u32(a[6], &rows) || !f32(a[7], &eps) || !pointer(a[8], &p[4]) || !pointer(a[9], &p[5])) return nullptr;
    return run([&] {
        return qkm_moe_layer_step((qkm_ctx*)c, layer, (const float*)p[0], (const float*)p[1], (const float*)p[2], (const float*)p[3], rows, eps,
                                  (float*)p[4], (float*)p[5]);
    });
}

// Any C ABI call: pointers, 32-bit numbers and floats in the order of its parameters.
bool convert(PyObject* o, uint32_t* out) { return u32(o, out); }
bool convert(PyObject* o, float* out) { return f32(o, out); }
template <class T>
bool convert(PyObject* o, T** out) {
    void* p = nullptr;
    if (!pointer(o, &p)) return false;
    *out = (T*)p;
    return true;
}
template <auto F> struct Plain;
template <class... A, int (*F)(A...)>
struct Plain<F> {
    static PyObject* call(PyObject*, PyObject* const* a, Py_ssize_t n) { return with(a, n, std::index_sequence_for<A...>{}); }
    template <size_t... I>
    static PyObject* with(PyObject* const* a, Py_ssize_t n, std::index_sequence<I...>) {
        std::tuple<std::remove_const_t<A>...> v;
        if (!count("call", n, sizeof...(A)) || !(convert(a[I], &std::get<I>(v)) && ...)) return nullptr;
        return run([&] { return F(std::get<I>(v)...); });
    }
};

#define FAST(f) ((PyCFunction)(void (*)(void))(f))
PyMethodDef methods[] = {
    {"gemv", FAST(gemv), METH_FASTCALL, nullptr},
    {"moe_decode", FAST(rows_call<qkm_moe_decode>), METH_FASTCALL, nullptr},
    {"moe_prefill", FAST(rows_call<qkm_moe_prefill>), METH_FASTCALL, nullptr},
    {"dense_gemm", FAST(rows_call<qkm_dense_gemm>), METH_FASTCALL, nullptr},
    {"moe_decode_stack", FAST(stack_call<qkm_moe_decode_stack>), METH_FASTCALL, nullptr},
    {"moe_decode_stack_host", FAST(stack_call<qkm_moe_decode_stack_host>), METH_FASTCALL, nullptr},
    {"argmax", FAST(argmax), METH_FASTCALL, nullptr},
    {"moe_layer_step", FAST(layer_step), METH_FASTCALL, nullptr},
    {"fp8_quantize", FAST(Plain<qkm_fp8_quantize>::call), METH_FASTCALL, nullptr},
    {"fp8_gemm", FAST(Plain<qkm_fp8_gemm>::call), METH_FASTCALL, nullptr},
    {"moe_gateup_grouped_fp8", FAST(Plain<qkm_moe_gateup_grouped_fp8>::call), METH_FASTCALL, nullptr},
    {"moe_down_grouped_fp8", FAST(Plain<qkm_moe_down_grouped_fp8>::call), METH_FASTCALL, nullptr},
    {"moe_shared_gateup_fp8", FAST(Plain<qkm_moe_shared_gateup_fp8>::call), METH_FASTCALL, nullptr},
    {"moe_shared_down_fp8", FAST(Plain<qkm_moe_shared_down_fp8>::call), METH_FASTCALL, nullptr},
    {"moe_balance", FAST(Plain<qkm_moe_balance>::call), METH_FASTCALL, nullptr},
    {"moe_balance_grad", FAST(Plain<qkm_moe_balance_grad>::call), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "qkm_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_qkm_calls(void) {
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    s_ptr = PyUnicode_InternFromString("ptr");
    return s_data_ptr && s_ptr ? PyModule_Create(&module) : nullptr;
}
