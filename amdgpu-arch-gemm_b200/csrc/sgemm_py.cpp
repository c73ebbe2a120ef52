// _sgemm_native: the 8-bit calls of runner/api.py without ctypes in between (CPython extension module).
//
// A decode step makes hundreds of these calls, each for a kernel of a few microseconds; through ctypes a linear call costs the host 7 us,
// through this module about half.  The module only takes addresses and types from its arguments and calls the C ABI: what an
// argument must be is said in api.py, whose checks (`SgemmRunner._addr`, `_type_code`) are called for every argument that does not
// pass the quick test here, and raise or resolve it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "sgemm_runner.h"

namespace {

PyObject *s_data_ptr, *s_get_device, *s_dtype, *s_is_contiguous, *s_addr, *s_stride, *s_shape, *s_element_size;   // interned names
PyObject *g_codes = nullptr;       // dtype object -> type code (api._type_codes)
PyObject *g_type_code = nullptr;   // api._type_code

// One call's view of its runner: converts arguments one after the other, remembers the first failure.
struct Call {
    PyObject *runner;
    long device;
    bool ok = true;

    // type code of a tensor-like object by its dtype, -1 when unknown
    long code_of(PyObject *x) {
        PyObject *dtype = PyObject_GetAttr(x, s_dtype);
        if (!dtype) {
            PyErr_Clear();
            return -1;
        }
        PyObject *code = PyDict_GetItemWithError(g_codes, dtype);   // borrowed
        Py_DECREF(dtype);
        if (!code) {
            PyErr_Clear();
            return -1;
        }
        return PyLong_AsLong(code);
    }
    // address of an operand; `code`: the element type it must have, -1 any
    void *addr(PyObject *x, const char *name, long code) {
        if (!ok || x == Py_None) return nullptr;
        if (PyLong_CheckExact(x)) {
            void *p = PyLong_AsVoidPtr(x);
            if (!p && PyErr_Occurred()) ok = false;
            return p;
        }
        PyObject *r = PyObject_CallMethodNoArgs(x, s_get_device);
        bool quick = r && PyLong_Check(r) && PyLong_AsLong(r) == device;
        Py_XDECREF(r);
        if (quick && code >= 0) quick = code_of(x) == code;
        if (quick) {
            r = PyObject_CallMethodNoArgs(x, s_is_contiguous);
            quick = r == Py_True;
            Py_XDECREF(r);
        }
        PyErr_Clear();
        if (quick) {
            r = PyObject_CallMethodNoArgs(x, s_data_ptr);
        } else {
            PyObject *py_name = PyUnicode_FromString(name), *py_code = PyLong_FromLong(code);
            r = py_name && py_code ? PyObject_CallMethodObjArgs(runner, s_addr, x, py_name, py_code, nullptr) : nullptr;
            Py_XDECREF(py_name);
            Py_XDECREF(py_code);
        }
        void *p = r ? PyLong_AsVoidPtr(r) : nullptr;
        Py_XDECREF(r);
        if (PyErr_Occurred()) ok = false;
        return p;
    }
    // element type of a matrix: the one given, else its own
    int type(PyObject *x, PyObject *given) {
        if (!ok) return -1;
        if (given == Py_None) {
            const long code = code_of(x);
            if (code >= 0 && code <= 2) return (int)code;
        }
        PyObject *r = PyObject_CallFunctionObjArgs(g_type_code, x, given, nullptr);
        const long code = r ? PyLong_AsLong(r) : -1;
        Py_XDECREF(r);
        if (PyErr_Occurred()) ok = false;
        return (int)code;
    }
    // address of an operand of the type that another one has: its own where none is given, and then this one must have it too; a given one
    // holds for tensors of a known type, as it does for that other operand
    void *sibling(PyObject *x, const char *name, int of, PyObject *given) {
        if (given == Py_None) return addr(x, name, of);
        if (ok && x != Py_None && !PyLong_CheckExact(x)) type(x, given);
        return addr(x, name, -1);
    }
    uint32_t u32(PyObject *x) {
        if (!ok) return 0;
        const unsigned long long v = PyLong_Check(x) ? PyLong_AsUnsignedLongLong(x) : PyNumber_AsSsize_t(x, PyExc_OverflowError);
        if (PyErr_Occurred() || v > 0xFFFFFFFFull) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_OverflowError, "a size or leading dimension does not fit 32 bits");
            ok = false;
        }
        return (uint32_t)v;
    }
    // A leading dimension.  0: the distance of the rows of a tensor of two or more dimensions, else the columns lie one behind the other.
    // The rows' distance is that of the last dimension before the elements' that is longer than one: the stride of a dimension of
    // one says nothing (a contiguous (rows, 1, elements) may carry any there).  `type`: the element type where it was given in the call
    // (else None): the tensor may then be storage of another kind, whose strides are in its own elements.
    uint32_t ld(PyObject *given, PyObject *matrix, uint32_t rows, PyObject *type = Py_None, int code = -1) {
        const uint32_t v = u32(given), dense = rows ? rows : 1u;
        if (!ok || v || matrix == Py_None || PyLong_CheckExact(matrix)) return v ? v : dense;
        PyObject *r = PyObject_CallMethodNoArgs(matrix, s_stride);   // a tuple; an object without one is dense
        if (!r) {
            PyErr_Clear();
            return dense;
        }
        uint32_t pitch = dense;
        if (PyTuple_Check(r) && PyTuple_GET_SIZE(r) >= 2) {
            const Py_ssize_t last = PyTuple_GET_SIZE(r) - 2;
            long long wide = 1, narrow = 1;   // bytes of the tensor's elements and of the call's
            if (type != Py_None && code_of(matrix) != code) {
                wide = element_size(matrix);
                narrow = code == 0 ? 4 : 2;
            }
            const auto stride_of = [&](Py_ssize_t dim) -> long long {
                const long long bytes = PyLong_AsLongLong(PyTuple_GET_ITEM(r, dim)) * wide;
                return bytes % narrow ? -1 : bytes / narrow;
            };
            long long stride = stride_of(last);
            const bool fits = stride >= (long long)dense && stride <= 0xFFFFFFFFll;
            const Py_ssize_t dim = last > 0 || !fits ? row_dimension(matrix, last) : last;
            if (dim >= 0) stride = stride_of(dim);
            if (stride >= (long long)dense && stride <= 0xFFFFFFFFll) pitch = (uint32_t)stride;
            else if (dim < 0) pitch = dense;
            else {
                if (stride < 0) PyErr_SetString(PyExc_ValueError, "a tensor's rows are no whole number of the given type's elements apart");
                else PyErr_Format(PyExc_ValueError, "a tensor's rows are %lld elements apart, the call reads %u of each", stride, dense);
                ok = false;
            }
        }
        Py_DECREF(r);
        return pitch;
    }
    // the last dimension up to `last` that is longer than one, -1 if there is none
    Py_ssize_t row_dimension(PyObject *matrix, Py_ssize_t last) {
        PyObject *shape = PyObject_GetAttr(matrix, s_shape);
        Py_ssize_t d = last;
        if (shape && PyTuple_Check(shape) && PyTuple_GET_SIZE(shape) > last)
            while (d >= 0 && PyLong_AsLong(PyTuple_GET_ITEM(shape, d)) <= 1) --d;
        Py_XDECREF(shape);
        PyErr_Clear();
        return d;
    }
    long long element_size(PyObject *x) {
        PyObject *r = PyObject_CallMethodNoArgs(x, s_element_size);
        const long long v = r ? PyLong_AsLongLong(r) : 1;
        Py_XDECREF(r);
        PyErr_Clear();   // (an object without one: in elements of the call's type)
        return v > 0 ? v : 1;
    }
    float f32(PyObject *x) {
        if (!ok) return 0.0f;
        const double v = PyFloat_AsDouble(x);
        if (PyErr_Occurred()) ok = false;
        return (float)v;
    }
    int flag(PyObject *x) {
        const int v = ok ? PyObject_IsTrue(x) : 0;
        if (v < 0) ok = false;
        return v > 0;
    }
    void *ptr(PyObject *x) {
        if (!ok) return nullptr;
        void *p = PyLong_AsVoidPtr(x);
        if (PyErr_Occurred()) ok = false;
        return p;
    }
};

// Every function: (runner, handle, device, arguments in the order of the SgemmRunner method) -> status of the C call.  The C call runs without the
// interpreter's lock, as calls through ctypes do: a launch can wait for room in the queue, and the stream for another Python thread.
#define NATIVE_BEGIN(NAME, COUNT)                                                                        \
    PyObject *NAME(PyObject *, PyObject *const *v, Py_ssize_t n) {                                       \
        if (n != 3 + (COUNT)) {                                                                          \
            PyErr_Format(PyExc_TypeError, #NAME " takes %d arguments, not %zd", 3 + (COUNT), n);         \
            return nullptr;                                                                              \
        }                                                                                                \
        Call c{v[0], PyLong_AsLong(v[2])};                                                               \
        sgemm_handle *h = static_cast<sgemm_handle *>(c.ptr(v[1]));                                      \
        PyObject *const *a = v + 3;
#define NATIVE_END(CALL)                  \
        if (!c.ok) return nullptr;        \
        int rc;                           \
        Py_BEGIN_ALLOW_THREADS            \
        rc = (CALL);                      \
        Py_END_ALLOW_THREADS              \
        return PyLong_FromLong(rc);       \
    }

// w, w_scale, x, x_scale, y, m, n, k, bias, ldw, ldx, ldy, y_type, stream
NATIVE_BEGIN(i8_linear, 14)
    const auto *w = static_cast<const int8_t *>(c.addr(a[0], "w", 3));
    const auto *ws = static_cast<const float *>(c.addr(a[1], "w_scale", 0));
    const auto *x = static_cast<const int8_t *>(c.addr(a[2], "x", 3));
    const auto *xs = static_cast<const float *>(c.addr(a[3], "x_scale", 0));
    void *y = c.addr(a[4], "y", -1);
    const uint32_t m = c.u32(a[5]), tokens = c.u32(a[6]), k = c.u32(a[7]);
    const auto *bias = static_cast<const float *>(c.addr(a[8], "bias", 0));
    const int type = c.type(a[4], a[12]);
    const uint32_t ldw = c.ld(a[9], a[0], k), ldx = c.ld(a[10], a[2], k), ldy = c.ld(a[11], a[4], m, a[12], type);
    void *stream = c.ptr(a[13]);
NATIVE_END(sgemm_i8_linear(h, w, ws, x, xs, bias, y, type, m, tokens, k, ldw, ldx, ldy, stream))

// x, q, scale, k, n, pow2, ldx, ldq, x_type, stream
NATIVE_BEGIN(i8_quantize, 10)
    const void *x = c.addr(a[0], "x", -1);
    auto *q = static_cast<int8_t *>(c.addr(a[1], "q", 3));
    auto *s = static_cast<float *>(c.addr(a[2], "scale", 0));
    const uint32_t k = c.u32(a[3]), rows = c.u32(a[4]);
    const int pow2 = c.flag(a[5]);
    const int type = c.type(a[0], a[8]);
    const uint32_t ldx = c.ld(a[6], a[0], k, a[8], type), ldq = c.ld(a[7], a[1], k);
    void *stream = c.ptr(a[9]);
NATIVE_END(sgemm_i8_quantize(h, x, type, q, s, k, rows, ldx, ldq, pow2, stream))

// q, scale, out, k, n, ldq, ldo, out_type, stream
NATIVE_BEGIN(i8_restore, 9)
    const auto *q = static_cast<const int8_t *>(c.addr(a[0], "q", 3));
    const auto *s = static_cast<const float *>(c.addr(a[1], "scale", 0));
    void *out = c.addr(a[2], "out", -1);
    const uint32_t k = c.u32(a[3]), rows = c.u32(a[4]);
    const int type = c.type(a[2], a[7]);
    const uint32_t ldq = c.ld(a[5], a[0], k), ldo = c.ld(a[6], a[2], k, a[7], type);
    void *stream = c.ptr(a[8]);
NATIVE_END(sgemm_i8_restore(h, q, s, out, type, k, rows, ldq, ldo, stream))

// x, gamma, q, scale, k, n, residual, sum_out, eps, ldx, ldr, ldq, lds, x_type, stream
NATIVE_BEGIN(i8_rmsnorm, 15)
    const int type = c.type(a[0], a[13]);
    const void *x = c.addr(a[0], "x", -1), *g = c.sibling(a[1], "gamma", type, a[13]);
    auto *q = static_cast<int8_t *>(c.addr(a[2], "q", 3));
    auto *s = static_cast<float *>(c.addr(a[3], "scale", 0));
    const uint32_t k = c.u32(a[4]), rows = c.u32(a[5]);
    const void *res = c.sibling(a[6], "residual", type, a[13]);
    void *sum = c.sibling(a[7], "sum_out", type, a[13]);
    const float eps = c.f32(a[8]);
    const uint32_t ldx = c.ld(a[9], a[0], k, a[13], type), ldr = c.ld(a[10], a[6], k, a[13], type), ldq = c.ld(a[11], a[2], k),
                   lds = c.ld(a[12], a[7], k, a[13], type);
    void *stream = c.ptr(a[14]);
NATIVE_END(sgemm_i8_rmsnorm(h, x, res, g, type, eps, q, s, sum, k, rows, ldx, ldr, ldq, lds, stream))

// q, scale, dy, dw, m, n, tokens, c, alpha, beta, ldq, lddy, ldc, lddw, dy_type, dw_type, stream
NATIVE_BEGIN(i8_wgrad, 17)
    const auto *q = static_cast<const int8_t *>(c.addr(a[0], "q", 3));
    const auto *s = static_cast<const float *>(c.addr(a[1], "scale", 0));
    const void *dy = c.addr(a[2], "dy", -1);
    void *dw = c.addr(a[3], "dw", -1);
    const uint32_t m = c.u32(a[4]), channels = c.u32(a[5]), tokens = c.u32(a[6]);
    const int dy_type = c.type(a[2], a[14]), dw_type = c.type(a[3], a[15]);
    const void *prior = c.sibling(a[7], "c", dw_type, a[15]);
    const float alpha = c.f32(a[8]), beta = c.f32(a[9]);
    const uint32_t ldq = c.ld(a[10], a[0], m), lddy = c.ld(a[11], a[2], channels, a[14], dy_type), ldc = c.ld(a[12], a[7], m, a[15], dw_type),
                   lddw = c.ld(a[13], a[3], m, a[15], dw_type);
    void *stream = c.ptr(a[16]);
NATIVE_END(sgemm_i8_wgrad(h, q, s, dy, dy_type, prior, dw, dw_type, alpha, beta, m, channels, tokens, ldq, lddy, ldc, lddw, stream))

// pitch(matrix, row length): the leading dimension that the calls above take for a matrix
PyObject *pitch(PyObject *, PyObject *const *v, Py_ssize_t n) {
    if (n != 2) {
        PyErr_SetString(PyExc_TypeError, "pitch(matrix, row length)");
        return nullptr;
    }
    Call c{nullptr, -1};
    PyObject *zero = PyLong_FromLong(0);
    const uint32_t rows = c.u32(v[1]), ld = zero ? c.ld(zero, v[0], rows) : 0;
    Py_XDECREF(zero);
    return c.ok && zero ? PyLong_FromUnsignedLong(ld) : nullptr;
}

// setup(type codes by dtype, api._type_code)
PyObject *setup(PyObject *, PyObject *const *v, Py_ssize_t n) {
    if (n != 2 || !PyDict_Check(v[0]) || !PyCallable_Check(v[1])) {
        PyErr_SetString(PyExc_TypeError, "setup(dict, callable)");
        return nullptr;
    }
    Py_INCREF(v[0]);
    Py_XSETREF(g_codes, v[0]);
    Py_INCREF(v[1]);
    Py_XSETREF(g_type_code, v[1]);
    Py_RETURN_NONE;
}

#define NATIVE_METHOD(NAME) {#NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(NAME)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {
    NATIVE_METHOD(i8_linear), NATIVE_METHOD(i8_quantize), NATIVE_METHOD(i8_restore), NATIVE_METHOD(i8_rmsnorm), NATIVE_METHOD(i8_wgrad),
    NATIVE_METHOD(pitch), NATIVE_METHOD(setup), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_sgemm_native", "8-bit calls of runner.api without ctypes", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__sgemm_native(void) {
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    s_get_device = PyUnicode_InternFromString("get_device");
    s_dtype = PyUnicode_InternFromString("dtype");
    s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
    s_addr = PyUnicode_InternFromString("_addr");
    s_stride = PyUnicode_InternFromString("stride");
    s_shape = PyUnicode_InternFromString("shape");
    s_element_size = PyUnicode_InternFromString("element_size");
    if (!s_stride || !s_shape || !s_element_size || !s_data_ptr || !s_get_device || !s_dtype || !s_is_contiguous || !s_addr) return nullptr;
    return PyModule_Create(&g_module);
}
