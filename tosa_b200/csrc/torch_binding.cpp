// The calls of tosa_b200/attention.py on torch tensors: checks of arguments, allocation of results and the
// C entry points, in one native step. The kernels of a small call take 3 to 10 us on the GPU; checked and
// called from Python through ctypes such a call took 7 to 25 us of the host.
//
// A CPython module without pybind: functions take positional arguments (METH_FASTCALL) and raise the
// TbError class given to init().
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <string>

#include "../../include/tosa_b200.h"

namespace {

PyObject* g_error = nullptr;  // TbError(status, message)

struct Refused {};  // a Python exception is set

[[noreturn]] void refuse(int status, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    PyObject* e = g_error ? PyObject_CallFunction(g_error, "is", status, buf) : nullptr;
    if (e) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    } else if (!PyErr_Occurred()) {
        PyErr_SetString(PyExc_RuntimeError, buf);
    }
    throw Refused{};
}

// Calls the library with the interpreter unlocked (a launch can wait for room in the stream's queue).
template <class F>
void call(at::Device device, F f) {
    c10::OptionalDeviceGuard guard;
    if (device.is_cuda()) guard.reset_device(device);
    PyThreadState* state = PyEval_SaveThread();
    const tb_status st = f();
    PyEval_RestoreThread(state);
    if (st != TB_OK) refuse(st, "%s", tb_last_error());
}

std::string shape_of(const at::Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}

const at::Tensor& tensor(const char* op, const char* name, PyObject* o) {
    if (!THPVariable_Check(o)) refuse(TB_ERR_INVALID_ARGUMENT, "%s: %s is not a tensor", op, name);
    return THPVariable_Unpack(o);
}

int dtype_code(const char* op, at::ScalarType t) {
    if (t == at::kBFloat16) return TB_DT_BF16;
    if (t == at::kHalf) return TB_DT_FP16;
    refuse(TB_ERR_DTYPE_MISMATCH, "%s: unsupported type %s (float16 or bfloat16)", op, c10::toString(t));
}

struct Heads {
    void* p;
    int64_t rows, heads, dim, row_stride, head_stride;
};

// A [rows, heads, head_dim] tensor whose heads are contiguous; -1: any number.
Heads heads(const char* op, const char* name, const at::Tensor& t, at::ScalarType type, at::Device device, int64_t rows = -1,
            int64_t n = -1, int64_t dim = -1) {
    if (t.scalar_type() != type)
        refuse(TB_ERR_DTYPE_MISMATCH, "%s: %s is %s, not %s", op, name, c10::toString(t.scalar_type()), c10::toString(type));
    if (t.device() != device)
        refuse(TB_ERR_INVALID_ARGUMENT, "%s: %s is on %s, not on %s", op, name, t.device().str().c_str(), device.str().c_str());
    if (t.dim() != 3 || (rows >= 0 && t.size(0) != rows) || (n >= 0 && t.size(1) != n) || (dim >= 0 && t.size(2) != dim))
        refuse(TB_ERR_SHAPE_MISMATCH, "%s: %s has shape %s", op, name, shape_of(t).c_str());
    if (t.requires_grad() && c10::GradMode::is_enabled())
        refuse(TB_ERR_INVALID_ARGUMENT, "%s: %s requires a gradient, and there is none (torch.no_grad() or %s.detach())", op, name, name);
    if (t.stride(2) != 1) refuse(TB_ERR_SHAPE_MISMATCH, "%s: the last dimension of %s must be contiguous", op, name);
    // the stride of a dimension of one element says nothing
    return Heads{t.data_ptr(), t.size(0), t.size(1), t.size(2), t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2),
                 t.size(1) > 1 ? t.stride(1) : t.size(2)};
}

struct Index {
    const int32_t* p;
    int32_t n;
};

// A contiguous int32 vector; -1: of any length.
Index index(const char* op, const char* name, PyObject* o, at::Device device, int64_t n = -1) {
    const at::Tensor& t = tensor(op, name, o);
    if (t.scalar_type() != at::kInt || t.dim() != 1 || (n >= 0 && t.size(0) != n) || !t.is_contiguous() || t.size(0) > INT32_MAX) {
        if (n >= 0) refuse(TB_ERR_SHAPE_MISMATCH, "%s: %s must be a contiguous int32 vector of %lld", op, name, static_cast<long long>(n));
        refuse(TB_ERR_SHAPE_MISMATCH, "%s: %s must be a contiguous int32 vector", op, name);
    }
    if (t.device() != device)
        refuse(TB_ERR_INVALID_ARGUMENT, "%s: %s is on %s, not on %s", op, name, t.device().str().c_str(), device.str().c_str());
    return Index{static_cast<const int32_t*>(t.data_ptr()), static_cast<int32_t>(t.size(0))};
}

at::Tensor sums(const char* op, PyObject* o, int64_t rows, int64_t columns, at::Device device) {
    if (o == Py_None) return at::empty({rows, columns}, at::TensorOptions(at::kFloat).device(device));
    const at::Tensor& t = tensor(op, "lse", o);
    if (t.scalar_type() != at::kFloat || t.dim() != 2 || t.size(0) != rows || t.size(1) != columns || !t.is_contiguous() || t.device() != device)
        refuse(TB_ERR_SHAPE_MISMATCH, "%s: lse must be contiguous float32 of (%lld, %lld)", op, static_cast<long long>(rows),
               static_cast<long long>(columns));
    return t;
}

float scale_of(PyObject* o, int64_t dim) {
    if (o == Py_None) return static_cast<float>(1.0 / std::sqrt(static_cast<double>(dim)));
    const double x = PyFloat_AsDouble(o);
    if (PyErr_Occurred()) throw Refused{};
    return static_cast<float>(x);
}

// A handle of the Python side: the object's `h`, a ctypes pointer.
void* handle(const char* op, PyObject* o) {
    PyObject* h = PyObject_GetAttrString(o, "h");
    PyObject* v = h && h != Py_None ? PyObject_GetAttrString(h, "value") : nullptr;
    void* p = v && v != Py_None ? PyLong_AsVoidPtr(v) : nullptr;
    Py_XDECREF(v);
    Py_XDECREF(h);
    if (PyErr_Occurred()) throw Refused{};
    if (!p) refuse(TB_ERR_INVALID_ARGUMENT, "%s: the handle is closed", op);
    return p;
}

// A cache's handle, which points into its context.
tb_cache* cache_handle(const char* op, PyObject* o) {
    PyObject* context = PyObject_GetAttrString(o, "ctx");
    if (!context) throw Refused{};
    PyObject* h = PyObject_GetAttrString(context, "h");
    const bool closed = h == Py_None;
    const bool missing = h == nullptr;
    Py_XDECREF(h);
    Py_DECREF(context);
    if (missing) throw Refused{};
    if (closed) refuse(TB_ERR_INVALID_ARGUMENT, "%s: the cache's context is closed", op);
    return static_cast<tb_cache*>(handle(op, o));
}

// A call's tensors (all on `device`) have to be on the context's device: elsewhere the kernel would use addresses that are not its own.
void on_device_of(const char* op, PyObject* context, at::Device device) {
    if (!device.is_cuda()) refuse(TB_ERR_INVALID_ARGUMENT, "%s: the tensors are on %s, not on a CUDA device", op, device.str().c_str());
    PyObject* o = PyObject_GetAttrString(context, "device");
    const long long own = o ? PyLong_AsLongLong(o) : -1;
    Py_XDECREF(o);
    if (PyErr_Occurred()) throw Refused{};
    if (own != device.index())
        refuse(TB_ERR_INVALID_ARGUMENT, "%s: the tensors are on %s, the context is on device %lld", op, device.str().c_str(), own);
}

// The stream of a call: the current one, or the given cudaStream_t.
void* stream_of(PyObject* o, at::Device device) {
    if (o != Py_None) {
        void* p = PyLong_AsVoidPtr(o);
        if (PyErr_Occurred()) throw Refused{};
        return p;
    }
    return device.is_cuda() ? c10::cuda::getCurrentCUDAStream(device.index()).stream() : nullptr;
}

long long number(PyObject* o) {
    const long long x = PyLong_AsLongLong(o);
    if (x == -1 && PyErr_Occurred()) throw Refused{};
    return x;
}

int32_t layer_of(const char* op, PyObject* o) {
    const long long x = number(o);
    if (x < 0 || x > INT32_MAX) refuse(TB_ERR_SHAPE_MISMATCH, "%s: layer %lld", op, x);
    return static_cast<int32_t>(x);
}

PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
    PyObject* x = THPVariable_Wrap(a);
    PyObject* y = x ? THPVariable_Wrap(b) : nullptr;
    PyObject* r = y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return r;
}

template <class F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F f) {
    if (got != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, got);
        return nullptr;
    }
    try {
        return f();
    } catch (const Refused&) {
        return nullptr;
    } catch (const std::exception& e) {  // torch's own errors, out of memory among them
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyObject* none() { Py_RETURN_NONE; }

// (ctx, q, k, v, cu_q, cu_k, causal, scale, out, lse, stream)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 11, [&]() -> PyObject* {
        const char* op = "attention";
        const at::Tensor& q = tensor(op, "q", a[1]);
        const at::ScalarType type = q.scalar_type();
        const at::Device device = q.device();
        const int code = dtype_code(op, type);
        const Heads hq = heads(op, "q", q, type, device);
        const Heads hk = heads(op, "k", tensor(op, "k", a[2]), type, device, -1, -1, hq.dim);
        const Heads hv = heads(op, "v", tensor(op, "v", a[3]), type, device, hk.rows, hk.heads, hq.dim);
        const Index cq = index(op, "cu_q", a[4], device);
        const Index ck = index(op, "cu_k", a[5], device, cq.n);
        if (cq.n < 1) refuse(TB_ERR_SHAPE_MISMATCH, "%s: cu_q needs batch + 1 offsets", op);
        const int causal = PyObject_IsTrue(a[6]);
        if (causal < 0) throw Refused{};
        const float scale = scale_of(a[7], hq.dim);
        const at::Tensor out = a[8] == Py_None ? at::empty({hq.rows, hq.heads, hq.dim}, at::TensorOptions(type).device(device))
                                               : tensor(op, "out", a[8]);
        const Heads ho = heads(op, "out", out, type, device, hq.rows, hq.heads, hq.dim);
        const at::Tensor lse = sums(op, a[9], hq.heads, hq.rows, device);
        if (hq.heads > INT32_MAX || hk.heads > INT32_MAX) refuse(TB_ERR_NOT_ACCELERATED, "%s: too many heads", op);
        const tb_attention_desc d{code, cq.n - 1, static_cast<int32_t>(hq.heads), static_cast<int32_t>(hk.heads),
                                  static_cast<int32_t>(hq.dim), causal, scale, hq.rows, hk.rows, hq.row_stride, hq.head_stride,
                                  hk.row_stride, hk.head_stride, hv.row_stride, hv.head_stride, ho.row_stride, ho.head_stride};
        auto* h = static_cast<tb_context*>(handle(op, a[0]));
        on_device_of(op, a[0], device);
        void* st = stream_of(a[10], device);
        call(device, [&] { return tb_attention(h, &d, hq.p, hk.p, hv.p, cq.p, ck.p, ho.p,
                           static_cast<float*>(lse.data_ptr()), st); });
        return pair(out, lse);
    });
}

// (cache, k_pages, layer, slots, offsets, k, v, stream)
PyObject* cache_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&]() -> PyObject* {
        const char* op = "cache write";
        const at::Tensor& pages = tensor(op, "k_pages", a[1]);
        const at::Device device = pages.device();
        const int32_t layer = layer_of(op, a[2]);
        const Index slots = index(op, "slots", a[3], device);
        const Index offsets = index(op, "offsets", a[4], device, static_cast<int64_t>(slots.n) + 1);
        const Heads k = heads(op, "k", tensor(op, "k", a[5]), pages.scalar_type(), device, -1, pages.size(2), pages.size(4));
        const Heads v = heads(op, "v", tensor(op, "v", a[6]), pages.scalar_type(), device, k.rows, pages.size(2), pages.size(4));
        tb_cache* h = cache_handle(op, a[0]);
        void* st = stream_of(a[7], device);
        call(device, [&] { return tb_cache_write(h, layer, slots.p, offsets.p, slots.n, k.rows, k.p, k.row_stride,
                             k.head_stride, v.p, v.row_stride, v.head_stride, st); });
        return none();
    });
}

// (cache, k_pages, layer, slots, q, scale, out, lse, stream)
PyObject* cache_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 9, [&]() -> PyObject* {
        const char* op = "cache attend";
        const at::Tensor& pages = tensor(op, "k_pages", a[1]);
        const at::Device device = pages.device();
        const at::ScalarType type = pages.scalar_type();
        const int32_t layer = layer_of(op, a[2]);
        const Index slots = index(op, "slots", a[3], device);
        const Heads q = heads(op, "q", tensor(op, "q", a[4]), type, device, slots.n, -1, pages.size(4));
        if (q.heads > INT32_MAX) refuse(TB_ERR_NOT_ACCELERATED, "%s: too many heads", op);
        const float scale = scale_of(a[5], q.dim);
        const at::Tensor out = a[6] == Py_None ? at::empty({q.rows, q.heads, q.dim}, at::TensorOptions(type).device(device))
                                               : tensor(op, "out", a[6]);
        const Heads ho = heads(op, "out", out, type, device, q.rows, q.heads, q.dim);
        const at::Tensor lse = sums(op, a[7], q.rows, q.heads, device);
        tb_cache* h = cache_handle(op, a[0]);
        void* st = stream_of(a[8], device);
        call(device, [&] { return tb_cache_attend(h, layer, slots.p, slots.n, static_cast<int32_t>(q.heads), scale,
                              q.p, q.row_stride, q.head_stride, ho.p, ho.row_stride, ho.head_stride,
                              static_cast<float*>(lse.data_ptr()), st); });
        return pair(out, lse);
    });
}

// (cache, k_pages, slots, counts or None, stream)
PyObject* cache_reserve(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 5, [&]() -> PyObject* {
        const char* op = "cache reserve";
        const at::Device device = tensor(op, "k_pages", a[1]).device();
        const Index slots = index(op, "slots", a[2], device);
        const int32_t* counts = a[3] == Py_None ? nullptr : index(op, "counts", a[3], device, slots.n).p;
        tb_cache* h = cache_handle(op, a[0]);
        void* st = stream_of(a[4], device);
        call(device, [&] { return tb_cache_reserve(h, slots.p, counts, slots.n, st); });
        return none();
    });
}

// (cache, k_pages, slots, stream)
PyObject* cache_free(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 4, [&]() -> PyObject* {
        const char* op = "cache free";
        const at::Device device = tensor(op, "k_pages", a[1]).device();
        const Index slots = index(op, "slots", a[2], device);
        tb_cache* h = cache_handle(op, a[0]);
        void* st = stream_of(a[3], device);
        call(device, [&] { return tb_cache_free(h, slots.p, slots.n, st); });
        return none();
    });
}

// (cache, k_pages, parents, children, stream)
PyObject* cache_fork(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 5, [&]() -> PyObject* {
        const char* op = "cache fork";
        const at::Device device = tensor(op, "k_pages", a[1]).device();
        const Index parents = index(op, "parents", a[2], device);
        const Index children = index(op, "children", a[3], device, parents.n);
        tb_cache* h = cache_handle(op, a[0]);
        void* st = stream_of(a[4], device);
        call(device, [&] { return tb_cache_fork(h, parents.p, children.p, parents.n, st); });
        return none();
    });
}

// (cache, k_pages, src, dst, stream)
PyObject* cache_copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 5, [&]() -> PyObject* {
        const char* op = "cache copy_pages";
        const at::Device device = tensor(op, "k_pages", a[1]).device();
        const Index src = index(op, "src", a[2], device);
        const Index dst = index(op, "dst", a[3], device, src.n);
        tb_cache* h = cache_handle(op, a[0]);
        void* st = stream_of(a[4], device);
        call(device, [&] { return tb_cache_copy_pages(h, src.p, dst.p, src.n, st); });
        return none();
    });
}

// (cache, page_table, refs, page_table_out or None, refs_out or None, stream)
PyObject* cache_compact(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 6, [&]() -> PyObject* {
        const char* op = "cache compact";
        const at::Device device = tensor(op, "page_table", a[1]).device();
        int32_t* to[2] = {nullptr, nullptr};
        const char* names[2] = {"page_table", "refs"};
        for (int i = 0; i < 2; ++i) {
            if (a[3 + i] == Py_None) continue;
            const at::Tensor &t = tensor(op, names[i], a[3 + i]), &own = tensor(op, names[i], a[1 + i]);
            if (t.scalar_type() != at::kInt || t.sizes() != own.sizes() || !t.is_contiguous() || t.device() != device)
                refuse(TB_ERR_SHAPE_MISMATCH, "%s: %s must be like the cache's own", op, names[i]);
            to[i] = static_cast<int32_t*>(t.data_ptr());
        }
        tb_cache* h = cache_handle(op, a[0]);
        void* st = stream_of(a[5], device);
        call(device, [&] { return tb_cache_compact(h, to[0], to[1], st); });
        return none();
    });
}

PyObject* init(PyObject*, PyObject* error) {
    Py_INCREF(error);
    Py_XSETREF(g_error, error);
    Py_RETURN_NONE;
}

#define TB_FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"init", init, METH_O, nullptr}, TB_FAST(attention), TB_FAST(cache_write), TB_FAST(cache_attend),
                         TB_FAST(cache_reserve), TB_FAST(cache_free), TB_FAST(cache_fork), TB_FAST(cache_copy_pages),
                         TB_FAST(cache_compact), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding() { return PyModule_Create(&module); }
