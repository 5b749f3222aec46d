// CPython module nne_pycall: the calls of a decode or prefill step from Python
// to the C ABI (include/nne_attn.h) without ctypes.
//
// A small call's GPU time is 6-13 us; converting its 18-25 arguments through
// ctypes took 4-5 us of host time and building its shape arrays 3 us more, so a
// loop of such calls ran at the host's pace.  Here the arguments are read
// straight from Python ints and tuples.  Host time per call: a prefill of 256
// rows 15.4 -> 8.3 us (10.5 with ctypes on plain addresses), a decode step of one
// sequence 19.2 -> 9.7 (12.7).
//
// Each function takes the address of its ABI function first (the package loads
// the library and owns it) and returns the ABI's status.  Shapes and strides
// are tuples of 4 ints, device pointers ints or None, host arrays any object
// with a contiguous buffer or None, a workspace the tuple (records,
// records_bytes, counters, n_counters) or None.
//
// The *_t functions take the tensors themselves and read what the call needs from them
// here; they return None, with nothing done, where a tensor is not of the type, device
// or shape that the call needs, and the package's own checks then say which.  Host time
// of a step's head norm 9.9 -> 9.1 us, of an append 5.6 -> 5.2 (an attention call, with
// two tensors fewer, gained nothing).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "nne_attn.h"

namespace {

// Reads the arguments in order; after the first bad one the error is set and
// every later read returns zeros.
struct Args {
    PyObject* const* a;
    Py_ssize_t n, i = 0;
    bool ok = true;
    Py_buffer host[2];
    int n_host = 0;

    Args(PyObject* const* args, Py_ssize_t count) : a(args), n(count) {}
    ~Args() {
        for (int k = 0; k < n_host; ++k) PyBuffer_Release(&host[k]);
    }
    PyObject* next() {
        if (!ok) return nullptr;
        if (i < n) return a[i++];
        PyErr_SetString(PyExc_TypeError, "nne_pycall: too few arguments");
        ok = false;
        return nullptr;
    }
    int64_t integer() {
        PyObject* o = next();
        if (!o) return 0;
        const long long v = PyLong_AsLongLong(o);
        if (v == -1 && PyErr_Occurred()) ok = false;
        return v;
    }
    template <typename T>
    T* pointer() {
        PyObject* o = next();
        if (!o || o == Py_None) return nullptr;
        void* p = PyLong_AsVoidPtr(o);
        if (!p && PyErr_Occurred()) ok = false;
        return static_cast<T*>(p);
    }
    float real() {
        PyObject* o = next();
        if (!o) return 0.f;
        const double v = PyFloat_AsDouble(o);
        if (v == -1.0 && PyErr_Occurred()) ok = false;
        return (float)v;
    }
    void ints(PyObject* o, int64_t* out) {
        if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) {
            PyErr_SetString(PyExc_TypeError, "nne_pycall: expected a tuple of 4 ints");
            ok = false;
            return;
        }
        for (int k = 0; k < 4; ++k) {
            out[k] = PyLong_AsLongLong(PyTuple_GET_ITEM(o, k));
            if (out[k] == -1 && PyErr_Occurred()) { ok = false; return; }
        }
    }
    struct Dims { int64_t v[4] = {0, 0, 0, 0}; };
    Dims dims() {
        Dims d;
        if (PyObject* o = next()) ints(o, d.v);
        return d;
    }
    int32_t* host_array() {
        PyObject* o = next();
        if (!o || o == Py_None) return nullptr;
        if (PyObject_GetBuffer(o, &host[n_host], PyBUF_SIMPLE) != 0) {
            ok = false;
            return nullptr;
        }
        return static_cast<int32_t*>(host[n_host++].buf);
    }
    nne_workspace_t ws_store;
    const nne_workspace_t* workspace() {
        PyObject* o = next();
        if (!o || o == Py_None) return nullptr;
        int64_t v[4] = {0, 0, 0, 0};
        ints(o, v);
        ws_store.records = reinterpret_cast<void*>((uintptr_t)v[0]);
        ws_store.records_bytes = (uint64_t)v[1];
        ws_store.counters = reinterpret_cast<uint32_t*>((uintptr_t)v[2]);
        ws_store.n_counters = (uint64_t)v[3];
        return &ws_store;
    }
    bool done() {
        if (ok && i != n) {
            PyErr_SetString(PyExc_TypeError, "nne_pycall: too many arguments");
            ok = false;
        }
        return ok;
    }
};

PyObject *g_dtype, *g_get_device, *g_shape, *g_stride, *g_data_ptr;    // interned names

bool make_names() {
    return (g_dtype = PyUnicode_InternFromString("dtype")) && (g_get_device = PyUnicode_InternFromString("get_device")) &&
           (g_shape = PyUnicode_InternFromString("shape")) && (g_stride = PyUnicode_InternFromString("stride")) &&
           (g_data_ptr = PyUnicode_InternFromString("data_ptr"));
}

// The int that a method without arguments returns.
bool int_of(PyObject* o, PyObject* method, int64_t& v) {
    PyObject* r = PyObject_CallMethodNoArgs(o, method);
    if (!r) return false;
    v = PyLong_AsLongLong(r);
    Py_DECREF(r);
    return !(v == -1 && PyErr_Occurred());
}

// A tensor of up to 4 dims.  read() is false on an error (set) and on a tensor of
// another type or device, or more dims (`fits` false, no error).
struct Tensor {
    float* p = nullptr;
    int64_t shape[4] = {0, 0, 0, 0}, stride[4] = {0, 0, 0, 0};
    Py_ssize_t dims = 0;
    bool fits = false;

    static Py_ssize_t tuple_of(PyObject* t, int64_t* out) {
        if (!t) return -1;
        Py_ssize_t n = PyTuple_Check(t) ? PyTuple_GET_SIZE(t) : -1;
        if (n < 0) PyErr_SetString(PyExc_TypeError, "nne_pycall: expected a tensor");
        for (Py_ssize_t k = 0; k < n && k < 4; ++k) {
            out[k] = PyLong_AsLongLong(PyTuple_GET_ITEM(t, k));
            if (out[k] == -1 && PyErr_Occurred()) { n = -1; break; }
        }
        Py_DECREF(t);
        return n;
    }
    // address: its address alone.
    bool read(PyObject* o, PyObject* dtype, int64_t index, bool address = false) {
        PyObject* d = PyObject_GetAttr(o, g_dtype);
        if (!d) return false;
        const bool type = d == dtype;
        Py_DECREF(d);
        if (!type) return false;
        int64_t dev, at;
        if (!int_of(o, g_get_device, dev)) return false;
        if (dev != index) return false;
        if (!address) {
            dims = tuple_of(PyObject_GetAttr(o, g_shape), shape);
            if (dims < 0 || dims > 4) return false;
            if (tuple_of(PyObject_CallMethodNoArgs(o, g_stride), stride) != dims) return false;
        }
        if (!int_of(o, g_data_ptr, at)) return false;
        p = reinterpret_cast<float*>((uintptr_t)at);
        return fits = true;
    }
    bool is(const Tensor& t) const {
        return dims == t.dims && shape[0] == t.shape[0] && shape[1] == t.shape[1] && shape[2] == t.shape[2] &&
               shape[3] == t.shape[3];
    }
    bool vector(int64_t n) const { return dims == 1 && shape[0] == n && (stride[0] == 1 || n <= 1); }
};

// What the *_t functions read beside Args: tensors of one type on one GPU, None where
// allowed; `fits` falls where one is another.
struct TensorArgs : Args {
    PyObject* f32;
    int64_t index = 0;
    bool fits = true;

    TensorArgs(PyObject* const* args, Py_ssize_t count) : Args(args, count), f32(nullptr) {}
    void types() {
        f32 = next();
        index = integer();
    }
    Tensor tensor(bool optional = false) { return typed(f32, optional); }
    Tensor table() { return typed(f32, true, true); }
    Tensor typed(PyObject* dtype, bool optional, bool address = false) {
        Tensor t;
        PyObject* o = next();
        if (!o || !fits || (optional && o == Py_None)) return t;
        if (!t.read(o, dtype, index, address)) {
            if (PyErr_Occurred()) ok = false;
            fits = false;
        }
        return t;
    }
    // A host array of n int32, or None.
    const int32_t* ints_of(int64_t n) {
        PyObject* o = next();
        if (!o || !fits || o == Py_None) return nullptr;
        if (PyObject_GetBuffer(o, &host[n_host], PyBUF_ND | PyBUF_FORMAT) != 0) {
            PyErr_Clear();               // (strided, or no buffer)
            fits = false;
            return nullptr;
        }
        const Py_buffer& b = host[n_host++];
        if (b.ndim != 1 || b.shape[0] != n || b.itemsize != 4 || !b.format || b.format[0] != 'i' || b.format[1]) {
            fits = false;
            return nullptr;
        }
        return static_cast<const int32_t*>(b.buf);
    }
};

template <typename F>
F* function(Args& a) {
    F* f = reinterpret_cast<F*>(a.pointer<void>());
    if (a.ok && !f) {
        PyErr_SetString(PyExc_ValueError, "nne_pycall: null function");
        a.ok = false;
    }
    return f;
}

PyObject* flash(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n);
    auto* f = function<decltype(nne_flash_attention_forward_ws)>(a);
    auto* q = a.pointer<const float>();
    const auto qs = a.dims(), qst = a.dims();
    auto* k = a.pointer<const float>();
    const auto ks = a.dims(), kst = a.dims();
    auto* v = a.pointer<const float>();
    const auto vs = a.dims(), vst = a.dims();
    auto* o = a.pointer<float>();
    const auto ost = a.dims();
    const int causal = (int)a.integer(), has_scale = (int)a.integer();
    const float scale = a.real();
    const int64_t br = a.integer(), bc = a.integer();
    const nne_workspace_t* ws = a.workspace();
    void* stream = a.pointer<void>();
    if (!a.done()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(q, qs.v, qst.v, k, ks.v, kst.v, v, vs.v, vst.v, o, ost.v, causal, has_scale, scale, br, bc,
           ws, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n);
    auto* f = function<decltype(nne_attention_forward_ws)>(a);
    auto* q = a.pointer<const float>();
    const auto qs = a.dims(), qst = a.dims();
    auto* k = a.pointer<const float>();
    const auto ks = a.dims(), kst = a.dims();
    auto* v = a.pointer<const float>();
    const auto vs = a.dims(), vst = a.dims();
    auto* o = a.pointer<float>();
    const auto ost = a.dims();
    const int causal = (int)a.integer();
    const int64_t q_offset = a.integer();
    const int has_scale = (int)a.integer();
    const float scale = a.real();
    const nne_workspace_t* ws = a.workspace();
    void* stream = a.pointer<void>();
    if (!a.done()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(q, qs.v, qst.v, k, ks.v, kst.v, v, vs.v, vst.v, o, ost.v, causal, q_offset, has_scale, scale,
           ws, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject* decode_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n);
    auto* f = function<decltype(nne_decode_attention)>(a);
    auto* q = a.pointer<const float>();
    const auto qst = a.dims();
    auto *kc = a.pointer<const float>(), *vc = a.pointer<const float>();
    auto* lens = a.pointer<const int32_t>();
    const int32_t* lens_host = a.host_array();
    auto* o = a.pointer<float>();
    const auto ost = a.dims();
    const int64_t B = a.integer(), Hq = a.integer(), Hkv = a.integer(), cap = a.integer(), d = a.integer();
    const int has_scale = (int)a.integer();
    const float scale = a.real();
    const nne_workspace_t* ws = a.workspace();
    void* stream = a.pointer<void>();
    if (!a.done()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(q, qst.v, kc, vc, lens, lens_host, o, ost.v, B, Hq, Hkv, cap, d, has_scale, scale, ws, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject* decode_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n);
    auto* f = function<decltype(nne_decode_step)>(a);
    auto* q = a.pointer<const float>();
    const auto qst = a.dims();
    auto *kc = a.pointer<float>(), *vc = a.pointer<float>();
    auto* lens = a.pointer<int32_t>();
    int32_t* lens_host = a.host_array();
    auto* kn = a.pointer<const float>();
    const auto knst = a.dims();
    auto* vn = a.pointer<const float>();
    const auto vnst = a.dims();
    auto* o = a.pointer<float>();
    const auto ost = a.dims();
    const int64_t B = a.integer(), Hq = a.integer(), Hkv = a.integer(), cap = a.integer(), d = a.integer();
    const int has_scale = (int)a.integer();
    const float scale = a.real();
    const nne_workspace_t* ws = a.workspace();
    void* stream = a.pointer<void>();
    if (!a.done()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(q, qst.v, kc, vc, lens, lens_host, kn, knst.v, vn, vnst.v, o, ost.v, B, Hq, Hkv, cap, d,
           has_scale, scale, ws, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject* qkv_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n);
    auto* f = function<decltype(nne_qkv_rope_ws)>(a);
    auto* x = a.pointer<const float>();
    const int64_t x_rs = a.integer();
    auto* w = a.pointer<const float>();
    auto *bq = a.pointer<const float>(), *bk = a.pointer<const float>(), *bv = a.pointer<const float>();
    auto *cos = a.pointer<const float>(), *sin = a.pointer<const float>();
    const int64_t max_seq = a.integer(), table_d = a.integer();
    auto* pos = a.pointer<const int32_t>();
    const int32_t* pos_host = a.host_array();
    auto *q = a.pointer<float>(), *k = a.pointer<float>(), *v = a.pointer<float>();
    const int64_t B = a.integer(), C = a.integer(), Hq = a.integer(), Hkv = a.integer(), d = a.integer();
    const nne_workspace_t* ws = a.workspace();
    void* stream = a.pointer<void>();
    if (!a.done()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(x, x_rs, w, bq, bk, bv, cos, sin, max_seq, table_d, pos, pos_host, q, k, v, B, C, Hq, Hkv, d,
           ws, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject* qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n);
    auto* f = function<decltype(nne_qk_norm_rope)>(a);
    auto* q = a.pointer<const float>();
    const auto qs = a.dims(), qst = a.dims();
    auto* qo = a.pointer<float>();
    const auto qot = a.dims();
    auto* k = a.pointer<const float>();
    const auto ks = a.dims(), kst = a.dims();
    auto* ko = a.pointer<float>();
    const auto kot = a.dims();
    auto *qw = a.pointer<const float>(), *kw = a.pointer<const float>();
    const int has_norm = (int)a.integer();
    const float eps = a.real();
    auto *cos = a.pointer<const float>(), *sin = a.pointer<const float>();
    const int64_t max_seq = a.integer(), table_d = a.integer();
    auto* start = a.pointer<const int32_t>();
    const int32_t* start_host = a.host_array();
    auto* depths = a.pointer<const int32_t>();
    const int32_t* depths_host = a.host_array();
    void* stream = a.pointer<void>();
    if (!a.done()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(q, qs.v, qst.v, qo, qot.v, k, ks.v, kst.v, ko, kot.v, qw, kw, has_norm, eps, cos, sin, max_seq, table_d,
           start, start_host, depths, depths_host, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject* qk_norm_rope_t(PyObject*, PyObject* const* args, Py_ssize_t n) {
    TensorArgs a(args, n);
    auto* f = function<decltype(nne_qk_norm_rope)>(a);
    a.types();
    PyObject* i32 = a.next();
    const Tensor q = a.tensor(), qo = a.tensor(), k = a.tensor(true), ko = a.tensor(true), qw = a.tensor(true),
                 kw = a.tensor(true);
    const int has_norm = (int)a.integer();
    const float eps = a.real();
    const Tensor cos = a.table(), sin = a.table();
    const int64_t max_seq = a.integer(), table_d = a.integer();
    const Tensor start = a.typed(i32, true);
    const int32_t* start_host = a.ints_of(q.shape[0]);
    auto* depths = a.pointer<const int32_t>();
    const int32_t* depths_host = a.host_array();
    void* stream = a.pointer<void>();
    if (!a.done()) return nullptr;
    const int64_t d = q.shape[3];
    if (!a.fits || q.dims != 4 || !qo.is(q) || (k.fits ? k.dims != 4 || !ko.is(k) : ko.fits) ||
        (qw.fits && !qw.vector(d)) || (kw.fits && !kw.vector(d)) ||
        (cos.fits && (!start.fits || !start.vector(q.shape[0]) || !start_host)))
        Py_RETURN_NONE;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(q.p, q.shape, q.stride, qo.p, qo.stride, k.p, k.shape, k.stride, ko.p, ko.stride, qw.p, kw.p, has_norm, eps,
           cos.p, sin.p, max_seq, table_d, reinterpret_cast<const int32_t*>(start.p), start_host, depths, depths_host,
           stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject* paged_append_t(PyObject*, PyObject* const* args, Py_ssize_t n) {
    TensorArgs a(args, n);
    auto* f = function<decltype(nne_paged_append)>(a);
    a.types();
    auto* cache = a.pointer<const nne_paged_cache_t>();
    const Tensor k = a.tensor(), v = a.tensor();
    auto* counts = a.pointer<const int32_t>();
    const int32_t* counts_host = a.host_array();
    auto* depths = a.pointer<const int32_t>();
    const int32_t* depths_host = a.host_array();
    const Tensor cos = a.table(), sin = a.table();
    const int64_t max_seq = a.integer(), table_d = a.integer();
    void* stream = a.pointer<void>();
    if (!a.done()) return nullptr;
    if (!a.fits || !cache || k.dims != 4 || !v.is(k) || k.shape[0] != cache->B || k.shape[1] != cache->Hkv ||
        k.shape[3] != cache->d)
        Py_RETURN_NONE;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(cache, k.p, k.stride, v.p, v.stride, k.shape[2], counts, counts_host, depths, depths_host, cos.p, sin.p,
           max_seq, table_d, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject* paged_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n);
    auto* f = function<decltype(nne_paged_append)>(a);
    auto* cache = a.pointer<const nne_paged_cache_t>();
    auto* k = a.pointer<const float>();
    const auto kst = a.dims();
    auto* v = a.pointer<const float>();
    const auto vst = a.dims();
    const int64_t T = a.integer();
    auto* counts = a.pointer<const int32_t>();
    const int32_t* counts_host = a.host_array();
    auto* depths = a.pointer<const int32_t>();
    const int32_t* depths_host = a.host_array();
    auto *cos = a.pointer<const float>(), *sin = a.pointer<const float>();
    const int64_t max_seq = a.integer(), table_d = a.integer();
    void* stream = a.pointer<void>();
    if (!a.done()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(cache, k, kst.v, v, vst.v, T, counts, counts_host, depths, depths_host, cos, sin, max_seq, table_d, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n);
    auto* f = function<decltype(nne_paged_attention)>(a);
    auto* cache = a.pointer<const nne_paged_cache_t>();
    auto* q = a.pointer<const float>();
    const auto qst = a.dims();
    auto* o = a.pointer<float>();
    const auto ost = a.dims();
    const int64_t Hq = a.integer(), T = a.integer();
    auto* counts = a.pointer<const int32_t>();
    const int32_t* counts_host = a.host_array();
    auto* parents = a.pointer<const int32_t>();
    const int32_t* parents_host = a.host_array();
    const int has_scale = (int)a.integer();
    const float scale = a.real();
    const nne_workspace_t* ws = a.workspace();
    void* stream = a.pointer<void>();
    if (!a.done()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(cache, q, qst.v, o, ost.v, Hq, T, counts, counts_host, parents, parents_host, has_scale, scale, ws, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject* paged_commit(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n);
    auto* f = function<decltype(nne_paged_commit)>(a);
    auto* cache = a.pointer<const nne_paged_cache_t>();
    const int64_t layers = a.integer(), stride = a.integer();
    auto* counts = a.pointer<const int32_t>();
    const int32_t* counts_host = a.host_array();
    auto* paths = a.pointer<const int32_t>();
    const int32_t* paths_host = a.host_array();
    const int64_t J = a.integer();
    const nne_workspace_t* ws = a.workspace();
    void* stream = a.pointer<void>();
    if (!a.done()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(cache, layers, stride, counts, counts_host, paths, paths_host, J, ws, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

#define NNE_METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {NNE_METHOD(flash), NNE_METHOD(attention), NNE_METHOD(decode_attention),
                         NNE_METHOD(decode_step), NNE_METHOD(qkv_rope), NNE_METHOD(qk_norm_rope),
                         NNE_METHOD(paged_append), NNE_METHOD(paged_attention), NNE_METHOD(paged_commit),
                         NNE_METHOD(qk_norm_rope_t), NNE_METHOD(paged_append_t), {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "nne_pycall", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_nne_pycall(void) { return make_names() ? PyModule_Create(&module) : nullptr; }
