// _sgemm_native: the 8-bit calls of runner/api.py without ctypes in between (CPython extension module).
//
// A decode step makes hundreds of these calls, each for a kernel of a few microseconds.  A linear call costs the host 3.2 us through this
// module, 3.1 with bare addresses; through ctypes 4.1 with addresses at hand, and the checks of the operands come on top.  The module only
// takes addresses, types, sizes and strides from its arguments and calls the C ABI: what an argument must be is said in api.py, whose
// checks (`SgemmRunner._addr`, `_type_code`) are called for every argument that does not pass the quick test here, and raise or resolve it.
//
// Tensors are read through DLPack's exchange of borrowed tensors (a table of C functions that a tensor type carries as
// `__dlpack_c_exchange_api__`): one C call for what six method calls told (with those a linear call cost 4.2 us).  Types without it are
// asked by name.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "sgemm_i8_params.hpp"
#include "sgemm_runner.h"

namespace {

PyObject *s_exchange, *s_addr, *s_shape, *s_stride, *s_element_size;   // interned names
PyObject *g_type_code = nullptr;                                       // api._type_code

// ---- DLPack 1.x as far as it is used here: a borrowed tensor, and the table of functions by which a type's objects are read
struct DlTensor {
    void *data;
    int32_t device_type, device_id;   // 1: host, 2: CUDA
    int32_t ndim;
    uint8_t code, bits;               // code 0: signed integer, 2: IEEE float, 4: bfloat
    uint16_t lanes;
    int64_t *shape, *strides;         // strides in elements
    uint64_t byte_offset;
};
struct DlExchange {
    uint32_t major, minor;
    void *previous;
    void *allocate, *managed_from_object, *managed_to_object;
    int (*borrow)(void *object, DlTensor *out);   // without synchronisation or a reference; shape and strides live as long as the object
    void *current_stream;
};
using Borrow = decltype(DlExchange::borrow);

// The function of an object's type, NULL where it has none.  The first few types met are kept (torch.Tensor, torch.nn.Parameter).
struct KnownType {
    PyTypeObject *type;
    Borrow borrow;
};
KnownType g_known[8];

Borrow borrow_of(PyObject *x) {
    KnownType *free = nullptr;
    for (KnownType &t : g_known) {
        if (t.type == Py_TYPE(x)) return t.borrow;
        if (!t.type && !free) free = &t;
    }
    Borrow found = nullptr;
    PyObject *capsule = PyObject_GetAttr(reinterpret_cast<PyObject *>(Py_TYPE(x)), s_exchange);
    if (capsule && PyCapsule_IsValid(capsule, "dlpack_exchange_api")) {
        const auto *api = static_cast<const DlExchange *>(PyCapsule_GetPointer(capsule, "dlpack_exchange_api"));
        if (api->major == 1) found = api->borrow;
    }
    Py_XDECREF(capsule);
    PyErr_Clear();
    if (free) {
        Py_INCREF(Py_TYPE(x));
        *free = KnownType{Py_TYPE(x), found};
    }
    return found;
}

// An operand: the object, its address and, of a tensor, how its elements lie.
struct Operand {
    static constexpr int kMost = 16;      // dimensions of one that is asked by name
    PyObject *x = nullptr;
    const char *name = "";
    void *p = nullptr;
    int ndim = -1;                        // -1: no tensor, or one that does not tell
    const int64_t *shape = nullptr, *stride = nullptr;
    int code = -1;                        // element type as the C ABI numbers it, -1: another one
    int64_t bytes = 0;                    // size of an element, 0: not known
    int64_t own[2 * kMost];

    Operand() = default;
    Operand(Operand &&) = delete;         // (shape may point into the object itself)

    bool contiguous() const {
        int64_t dense = 1;
        for (int d = 0; d < ndim; ++d)
            if (shape[d] == 0) return true;
        for (int d = ndim - 1; d >= 0; --d) {
            if (shape[d] != 1 && stride[d] != dense) return false;
            dense *= shape[d];
        }
        return true;
    }
    // elements from the first to the last one
    uint64_t extent() const {
        uint64_t n = 1;
        for (int d = 0; d < ndim; ++d) {
            if (shape[d] == 0) return 0;
            n += (uint64_t)(shape[d] - 1) * (uint64_t)stride[d];
        }
        return n;
    }
    // Fills in what the object tells about itself; true when it did so by DLPack (`t` then holds its device and address too).
    bool read(PyObject *object, DlTensor &t) {
        x = object;
        if (const Borrow borrow = borrow_of(x)) {
            if (borrow(x, &t) == 0 && t.strides) {
                ndim = t.ndim;
                shape = t.shape;
                stride = t.strides;
                bytes = (t.bits * t.lanes + 7) / 8;
                if (t.lanes == 1) code = t.code == 2 && t.bits == 32 ? 0 : t.code == 2 && t.bits == 16 ? 1 : t.code == 4 && t.bits == 16 ? 2 : t.code == 0 && t.bits == 8 ? 3 : -1;
                return true;
            }
            PyErr_Clear();
        }
        PyObject *sizes = PyObject_GetAttr(x, s_shape), *strides = sizes ? PyObject_CallMethodNoArgs(x, s_stride) : nullptr;
        if (strides && PyTuple_Check(sizes) && PyTuple_Check(strides) && PyTuple_GET_SIZE(sizes) == PyTuple_GET_SIZE(strides) && PyTuple_GET_SIZE(sizes) <= kMost) {
            const int n = (int)PyTuple_GET_SIZE(sizes);
            for (int d = 0; d < n; ++d) {
                own[d] = PyLong_AsLongLong(PyTuple_GET_ITEM(sizes, d));
                own[kMost + d] = PyLong_AsLongLong(PyTuple_GET_ITEM(strides, d));
            }
            if (!PyErr_Occurred()) {
                ndim = n;
                shape = own;
                stride = own + kMost;
                PyObject *size = PyObject_CallMethodNoArgs(x, s_element_size);   // (one without it has the call's elements)
                if (size) bytes = PyLong_AsLongLong(size);
                Py_XDECREF(size);
            }
        }
        Py_XDECREF(sizes);
        Py_XDECREF(strides);
        PyErr_Clear();
        return false;
    }
};

// One call's view of its runner: converts arguments one after the other, remembers the first failure.
struct Call {
    PyObject *runner;
    long device;
    bool ok = true;

    // an operand; `code`: the element type it must have, -1 any
    Operand &addr(Operand &o, PyObject *x, const char *name, long code) {
        o.x = x;
        o.name = name;
        if (!ok || x == Py_None) return o;
        if (PyLong_CheckExact(x)) {
            o.p = PyLong_AsVoidPtr(x);
            if (!o.p && PyErr_Occurred()) ok = false;
            return o;
        }
        DlTensor t;
        if (o.read(x, t) && (device < 0 ? t.device_type == 1 : t.device_type == 2 && t.device_id == device) && (code < 0 || o.code == code) && o.contiguous() &&
            t.data) {   // (a type may give no address, as wrappers without storage do: they say what is wrong when asked by name)
            o.p = static_cast<char *>(t.data) + t.byte_offset;
            return o;
        }
        PyObject *py_name = PyUnicode_FromString(name), *py_code = PyLong_FromLong(code);
        PyObject *r = py_name && py_code ? PyObject_CallMethodObjArgs(runner, s_addr, x, py_name, py_code, nullptr) : nullptr;
        Py_XDECREF(py_name);
        Py_XDECREF(py_code);
        o.p = r ? PyLong_AsVoidPtr(r) : nullptr;
        Py_XDECREF(r);
        if (PyErr_Occurred()) ok = false;
        return o;
    }
    // an operand of the type that another one has: its own where none is given, and then this one must have it too; a given one holds for
    // tensors of a known type, as it does for that other operand
    void sibling(Operand &o, PyObject *x, const char *name, int of, PyObject *given) {
        addr(o, x, name, given == Py_None ? of : -1);
        if (given != Py_None && x != Py_None && !PyLong_CheckExact(x)) type(o, given);
    }
    // element type of a matrix: the one given, else its own
    int type(const Operand &o, PyObject *given) {
        if (!ok) return -1;
        if (given == Py_None && o.code >= 0 && o.code <= 2) return o.code;
        PyObject *r = PyObject_CallFunctionObjArgs(g_type_code, o.x, given, nullptr);
        const long code = r ? PyLong_AsLong(r) : -1;
        Py_XDECREF(r);
        if (PyErr_Occurred()) ok = false;
        return (int)code;
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
    // A distance in the tensor's own elements, in elements of the call's type where that was given (the tensor may then be storage of another
    // kind): `code`, or -1 where the two are the same.  -1: no whole number.
    static int64_t in_elements(const Operand &o, int64_t distance, int code) {
        if (code < 0 || o.code == code || o.bytes <= 0) return distance;
        const int64_t size = code == 0 ? 4 : 2;
        return distance * o.bytes % size ? -1 : distance * o.bytes / size;
    }
    // A leading dimension.  0: the distance of the rows of a tensor of two or more dimensions, else the columns lie one behind the other.
    // The rows' distance is that of the last dimension before the elements' that is longer than one: the stride of a dimension of
    // one says nothing (a contiguous (rows, 1, elements) may carry any there); with all of them one a stride that fits is taken.
    uint32_t ld(PyObject *given, const Operand &o, uint32_t rows, int code = -1) {
        const uint32_t v = u32(given), dense = rows ? rows : 1u;
        if (!ok || v || o.ndim < 2) return v ? v : dense;
        const auto fits = [&](int64_t stride) { return stride >= (int64_t)dense && stride <= 0xFFFFFFFFll; };
        int dim = o.ndim - 2;
        int64_t stride = in_elements(o, o.stride[dim], code);
        if (dim > 0 || !fits(stride)) {
            while (dim >= 0 && o.shape[dim] <= 1) --dim;
            if (dim < 0) return fits(stride) ? (uint32_t)stride : dense;
            stride = in_elements(o, o.stride[dim], code);
        }
        if (fits(stride)) return (uint32_t)stride;
        if (stride < 0) PyErr_SetString(PyExc_ValueError, "a tensor's rows are no whole number of the given type's elements apart");
        else PyErr_Format(PyExc_ValueError, "a tensor's rows are %lld elements apart, the call reads %u of each", (long long)stride, dense);
        ok = false;
        return dense;
    }
    // A matrix of `rows` rows of `length` elements `ld` apart must end inside its tensor, a vector is one row; `code` as in ld().  (What a call
    // does not touch has no rows; an `ld` below `length` is refused by the call itself.)
    void extent(const Operand &o, uint32_t rows, uint32_t ld, uint32_t length, int code = -1) {
        if (!ok || o.ndim < 0 || rows == 0 || length == 0 || ld < length) return;
        const uint64_t need = (uint64_t)(rows - 1) * ld + length;
        uint64_t have = o.extent();
        if (code >= 0 && o.code != code && o.bytes > 0) have = have * (uint64_t)o.bytes / (code == 0 ? 4 : 2);
        if (have >= need) {
            if (!o.p) {   // NULL would be an operand that was left out
                PyErr_Format(PyExc_ValueError, "%s has no storage", o.name);
                ok = false;
            }
            return;
        }
        PyErr_Format(PyExc_ValueError, "%s holds %llu elements, the call reaches over %llu", o.name, (unsigned long long)have, (unsigned long long)need);
        ok = false;
    }
    void extent(const Operand &vector, uint32_t length) { extent(vector, 1, length, length); }
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

template <typename T> T *as(const Operand &o) { return static_cast<T *>(o.p); }
// the element type that was given, -1 where none was: a tensor then has the call's
int given(PyObject *type, int code) { return type == Py_None ? -1 : code; }

// w, w_scale, x, x_scale, y, m, n, k, bias, ldw, ldx, ldy, y_type, stream
NATIVE_BEGIN(i8_linear, 14)
    Operand w, ws, x, xs, y, bias;
    c.addr(w, a[0], "w", 3);
    c.addr(ws, a[1], "w_scale", 0);
    c.addr(x, a[2], "x", 3);
    c.addr(xs, a[3], "x_scale", 0);
    c.addr(y, a[4], "y", -1);
    c.addr(bias, a[8], "bias", 0);
    const uint32_t m = c.u32(a[5]), tokens = c.u32(a[6]), k = c.u32(a[7]);
    const int type = c.type(y, a[12]), y_given = given(a[12], type);
    const uint32_t ldw = c.ld(a[9], w, k), ldx = c.ld(a[10], x, k), ldy = c.ld(a[11], y, m, y_given);
    if (m && tokens && k <= I8_MAX_K) {
        c.extent(w, m, ldw, k);
        c.extent(ws, m);
        c.extent(x, tokens, ldx, k);
        c.extent(xs, tokens);
        c.extent(y, tokens, ldy, m, y_given);
        c.extent(bias, m);
    }
    void *stream = c.ptr(a[13]);
NATIVE_END(sgemm_i8_linear(h, as<int8_t>(w), as<float>(ws), as<int8_t>(x), as<float>(xs), as<float>(bias), y.p, type, m, tokens, k, ldw, ldx, ldy, stream))

// x, q, scale, k, n, pow2, ldx, ldq, x_type, stream
NATIVE_BEGIN(i8_quantize, 10)
    Operand x, q, s;
    c.addr(x, a[0], "x", -1);
    c.addr(q, a[1], "q", 3);
    c.addr(s, a[2], "scale", 0);
    const uint32_t k = c.u32(a[3]), rows = c.u32(a[4]);
    const int pow2 = c.flag(a[5]), type = c.type(x, a[8]), x_given = given(a[8], type);
    const uint32_t ldx = c.ld(a[6], x, k, x_given), ldq = c.ld(a[7], q, k);
    c.extent(x, rows, ldx, k, x_given);
    c.extent(q, rows, ldq, k);
    c.extent(s, rows);
    void *stream = c.ptr(a[9]);
NATIVE_END(sgemm_i8_quantize(h, x.p, type, as<int8_t>(q), as<float>(s), k, rows, ldx, ldq, pow2, stream))

// q, scale, out, k, n, ldq, ldo, out_type, stream
NATIVE_BEGIN(i8_restore, 9)
    Operand q, s, out;
    c.addr(q, a[0], "q", 3);
    c.addr(s, a[1], "scale", 0);
    c.addr(out, a[2], "out", -1);
    const uint32_t k = c.u32(a[3]), rows = c.u32(a[4]);
    const int type = c.type(out, a[7]), out_given = given(a[7], type);
    const uint32_t ldq = c.ld(a[5], q, k), ldo = c.ld(a[6], out, k, out_given);
    c.extent(q, rows, ldq, k);
    c.extent(s, k ? rows : 0);
    c.extent(out, rows, ldo, k, out_given);
    void *stream = c.ptr(a[8]);
NATIVE_END(sgemm_i8_restore(h, as<int8_t>(q), as<float>(s), out.p, type, k, rows, ldq, ldo, stream))

// x, gamma, q, scale, k, n, residual, sum_out, eps, ldx, ldr, ldq, lds, x_type, stream
NATIVE_BEGIN(i8_rmsnorm, 15)
    Operand x, g, q, s, res, sum;
    c.addr(x, a[0], "x", -1);
    const int type = c.type(x, a[13]), x_given = given(a[13], type);
    c.sibling(g, a[1], "gamma", type, a[13]);
    c.addr(q, a[2], "q", 3);
    c.addr(s, a[3], "scale", 0);
    c.sibling(res, a[6], "residual", type, a[13]);
    c.sibling(sum, a[7], "sum_out", type, a[13]);
    const uint32_t k = c.u32(a[4]), rows = c.u32(a[5]);
    const float eps = c.f32(a[8]);
    const uint32_t ldx = c.ld(a[9], x, k, x_given), ldr = c.ld(a[10], res, k, x_given), ldq = c.ld(a[11], q, k), lds = c.ld(a[12], sum, k, x_given);
    c.extent(x, rows, ldx, k, x_given);
    c.extent(g, rows ? 1 : 0, k, k, x_given);
    c.extent(q, rows, ldq, k);
    c.extent(s, rows);
    c.extent(res, rows, ldr, k, x_given);
    c.extent(sum, rows, lds, k, x_given);
    void *stream = c.ptr(a[14]);
NATIVE_END(sgemm_i8_rmsnorm(h, x.p, res.p, g.p, type, eps, as<int8_t>(q), as<float>(s), sum.p, k, rows, ldx, ldr, ldq, lds, stream))

// q, scale, dy, dw, m, n, tokens, c, alpha, beta, ldq, lddy, ldc, lddw, dy_type, dw_type, stream
NATIVE_BEGIN(i8_wgrad, 17)
    Operand q, s, dy, dw, prior;
    c.addr(q, a[0], "q", 3);
    c.addr(s, a[1], "scale", 0);
    c.addr(dy, a[2], "dy", -1);
    c.addr(dw, a[3], "dw", -1);
    const uint32_t m = c.u32(a[4]), channels = c.u32(a[5]), tokens = c.u32(a[6]);
    const int dy_type = c.type(dy, a[14]), dw_type = c.type(dw, a[15]), dy_given = given(a[14], dy_type), dw_given = given(a[15], dw_type);
    c.sibling(prior, a[7], "c", dw_type, a[15]);
    const float alpha = c.f32(a[8]), beta = c.f32(a[9]);
    const uint32_t ldq = c.ld(a[10], q, m), lddy = c.ld(a[11], dy, channels, dy_given), ldc = c.ld(a[12], prior, m, dw_given),
                   lddw = c.ld(a[13], dw, m, dw_given);
    if (m && channels) {
        c.extent(q, tokens, ldq, m);
        c.extent(s, tokens);
        c.extent(dy, tokens, lddy, channels, dy_given);
        c.extent(dw, channels, lddw, m, dw_given);
        if (beta != 0.0f) c.extent(prior, channels, ldc, m, dw_given);
    }
    void *stream = c.ptr(a[16]);
NATIVE_END(sgemm_i8_wgrad(h, as<int8_t>(q), as<float>(s), dy.p, dy_type, prior.p, dw.p, dw_type, alpha, beta, m, channels, tokens, ldq, lddy, ldc, lddw, stream))

// pitch(matrix, row length): the leading dimension that the calls above take for a matrix
PyObject *pitch(PyObject *, PyObject *const *v, Py_ssize_t n) {
    if (n != 2) {
        PyErr_SetString(PyExc_TypeError, "pitch(matrix, row length)");
        return nullptr;
    }
    Call c{nullptr, -1};
    Operand o;
    DlTensor t;
    o.read(v[0], t);
    PyObject *zero = PyLong_FromLong(0);
    const uint32_t rows = c.u32(v[1]), ld = zero ? c.ld(zero, o, rows) : 0;
    Py_XDECREF(zero);
    return c.ok && zero ? PyLong_FromUnsignedLong(ld) : nullptr;
}

// setup(api._type_code)
PyObject *setup(PyObject *, PyObject *const *v, Py_ssize_t n) {
    if (n != 1 || !PyCallable_Check(v[0])) {
        PyErr_SetString(PyExc_TypeError, "setup(callable)");
        return nullptr;
    }
    Py_INCREF(v[0]);
    Py_XSETREF(g_type_code, v[0]);
    Py_RETURN_NONE;
}

#define NATIVE_METHOD(NAME) {#NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(NAME)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {
    NATIVE_METHOD(i8_linear), NATIVE_METHOD(i8_quantize), NATIVE_METHOD(i8_restore), NATIVE_METHOD(i8_rmsnorm), NATIVE_METHOD(i8_wgrad),
    NATIVE_METHOD(pitch), NATIVE_METHOD(setup), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_sgemm_native", "8-bit calls of runner.api without ctypes", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__sgemm_native(void) {
    s_exchange = PyUnicode_InternFromString("__dlpack_c_exchange_api__");
    s_addr = PyUnicode_InternFromString("_addr");
    s_shape = PyUnicode_InternFromString("shape");
    s_stride = PyUnicode_InternFromString("stride");
    s_element_size = PyUnicode_InternFromString("element_size");
    if (!s_exchange || !s_addr || !s_shape || !s_stride || !s_element_size) return nullptr;
    return PyModule_Create(&g_module);
}
