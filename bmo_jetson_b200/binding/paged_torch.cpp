// paged_torch.cpp -- the paged cache's calls (include/bmo_kernels.h) on torch
// tensors, for bmo_jetson_b200/paged.py: checks each tensor, takes torch's
// current stream and calls the library through the addresses given to bind().
//
// A decode step makes a few of these calls a layer on kernels of a few
// microseconds, so the checks are done here: in Python they and the
// conversion of some 17 arguments took 4 us of a call, here they take 0.5.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "bmo_kernels.h"

namespace {

decltype(&bmo_k_paged_plan) g_plan;
decltype(&bmo_k_paged_append) g_append;
decltype(&bmo_k_paged_read) g_read;
decltype(&bmo_k_paged_attention) g_attention;

// Thrown after the Python error is set.
struct Raised {};

[[noreturn]] void refuse(const char *name, const char *what) {
    PyErr_Format(PyExc_ValueError, "%s: %s", name, what);
    throw Raised{};
}

const at::Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) refuse(name, "a tensor");
    return THPVariable_Unpack(o);
}

void on_device(const at::Tensor &t, const char *name, int dev) {
    if (!t.is_cuda() || t.get_device() != dev) refuse(name, "a tensor on the cache's GPU");
}

// A dense int32 tensor; numel < 0: of any size.  None where it may be: null.
int32_t *ints(PyObject *o, const char *name, int dev, int64_t numel, bool optional = false) {
    if (optional && o == Py_None) return nullptr;
    const at::Tensor &t = tensor(o, name);
    on_device(t, name, dev);
    if (t.scalar_type() != at::kInt || !t.is_contiguous()) refuse(name, "a contiguous int32 tensor");
    if (numel >= 0 && t.numel() != numel) refuse(name, "a tensor of another size");
    return static_cast<int32_t *>(t.data_ptr());
}

int act_type(const at::Tensor &t, const char *name) {
    switch (t.scalar_type()) {
        case at::kFloat: return BMO_ACT_F32;
        case at::kHalf: return BMO_ACT_F16;
        case at::kBFloat16: return BMO_ACT_BF16;
        default: refuse(name, "float32, float16 or bfloat16");
    }
}

struct Rows {
    void *p;
    long long stride;
};
// [n, heads, head_dim] rows whose heads are dense.
Rows rows(PyObject *o, const char *name, int dev, int64_t n, int64_t heads, int64_t head_dim, at::ScalarType type) {
    const at::Tensor &t = tensor(o, name);
    on_device(t, name, dev);
    if (t.scalar_type() != type) refuse(name, "a tensor of another type than the first");
    if (t.dim() != 3 || t.size(0) != n || t.size(1) != heads || t.size(2) != head_dim)
        refuse(name, "[n, heads, head_dim] of another shape");
    if (t.stride(2) != 1 || (heads > 1 && t.stride(1) != head_dim)) refuse(name, "the heads of a row are contiguous");
    return {t.data_ptr(), t.stride(0)};
}

long long integer(PyObject *o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}
int layer_of(PyObject *o) {
    const long long v = integer(o);
    return v < 0 || v > INT32_MAX ? -1 : static_cast<int>(v);  // the library refuses -1
}
// 0 has a meaning of its own in theta and scale: what rounds to it is refused.
float number(PyObject *o, const char *name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    const float f = static_cast<float>(v);
    if (f == 0.0f && v != 0.0) refuse(name, "too small for float32");
    return f;
}
int count(int64_t n, const char *name) {
    if (n > INT32_MAX) refuse(name, "too many rows");
    return static_cast<int>(n);
}

PyObject *result(int rc, const char *what) {
    if (rc != 0) return PyErr_Format(PyExc_RuntimeError, "%s rc=%d", what, rc);
    Py_RETURN_NONE;
}

// Runs body(stream) on the device; C++ exceptions do not reach Python.
template <class Body>
PyObject *call(PyObject *dev_arg, Py_ssize_t got, Py_ssize_t want, const char *what, Body body) {
    if (got != want) return PyErr_Format(PyExc_TypeError, "%s: %zd arguments, got %zd", what, want, got);
    try {
        const int dev = static_cast<int>(integer(dev_arg));
        c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
        void *stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
        return result(body(dev, stream), what);
    } catch (const Raised &) {
        return nullptr;
    } catch (const std::exception &e) {
        return PyErr_Format(PyExc_RuntimeError, "%s: %s", what, e.what());
    }
}

// plan(book, device, n_new, slot, pos, req, offsets, lens_out, state_out)
PyObject *plan(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(n > 1 ? a[1] : nullptr, n, 9, "bmo_k_paged_plan", [&](int dev, void *stream) {
        const auto *book = reinterpret_cast<const bmo_page_book *>(integer(a[0]));
        const int64_t most = tensor(a[3], "slot").numel();
        int32_t *lens = ints(a[7], "lens_out", dev, book->n_req, true), *state = ints(a[8], "state_out", dev, 4, true);
        return g_plan(book, ints(a[2], "n_new", dev, book->n_req), count(most, "slot"), ints(a[3], "slot", dev, -1),
                      ints(a[4], "pos", dev, most), ints(a[5], "req", dev, most),
                      ints(a[6], "offsets", dev, book->n_req + 1), lens ? lens : book->lens, state ? state : book->state,
                      stream);
    });
}

// append(cache, device, layer, k, v, slot, pos, q, q_out, theta, status)
PyObject *append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(n > 1 ? a[1] : nullptr, n, 11, "bmo_k_paged_append", [&](int dev, void *stream) {
        const auto *c = reinterpret_cast<const bmo_paged_kv *>(integer(a[0]));
        const int64_t tokens = tensor(a[5], "slot").numel();
        const at::Tensor &key = tensor(a[3], "k");
        const int act = act_type(key, "k");
        const auto type = key.scalar_type();
        const Rows k = rows(a[3], "k", dev, tokens, c->n_kv_heads, c->head_dim, type);
        const Rows v = rows(a[4], "v", dev, tokens, c->n_kv_heads, c->head_dim, type);
        Rows q{nullptr, 0}, qo{nullptr, 0};
        int64_t heads = 0;
        const float theta = number(a[9], "theta");
        if (a[7] != Py_None && theta == 0.0f) refuse("theta", "above 0 where q is to be rotated");
        if (a[7] == Py_None && a[8] != Py_None) refuse("q_out", "without q");
        if (a[7] != Py_None) {
            const at::Tensor &query = tensor(a[7], "q");
            if (query.dim() != 3) refuse("q", "[n, heads, head_dim]");
            heads = query.size(1);
            q = rows(a[7], "q", dev, tokens, heads, c->head_dim, type);
            qo = rows(a[8], "q_out", dev, tokens, heads, c->head_dim, type);
        }
        return g_append(c, layer_of(a[2]), count(tokens, "slot"), k.p, k.stride, v.p, v.stride, ints(a[5], "slot", dev, -1),
                        ints(a[6], "pos", dev, tokens, true), theta, q.p, q.stride,
                        count(heads, "q"), qo.p, qo.stride, act, ints(a[10], "status", dev, 1, true), stream);
    });
}

// read(cache, device, layer, slot, k_out, v_out, status)
PyObject *read(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(n > 1 ? a[1] : nullptr, n, 7, "bmo_k_paged_read", [&](int dev, void *stream) {
        const auto *c = reinterpret_cast<const bmo_paged_kv *>(integer(a[0]));
        const int64_t tokens = tensor(a[3], "slot").numel();
        const at::Tensor &key = tensor(a[4], "k_out");
        const int act = act_type(key, "k_out");
        const Rows k = rows(a[4], "k_out", dev, tokens, c->n_kv_heads, c->head_dim, key.scalar_type());
        const Rows v = rows(a[5], "v_out", dev, tokens, c->n_kv_heads, c->head_dim, key.scalar_type());
        if (!key.is_contiguous()) refuse("k_out", "contiguous");
        if (!tensor(a[5], "v_out").is_contiguous()) refuse("v_out", "contiguous");
        return g_read(c, layer_of(a[2]), count(tokens, "slot"), ints(a[3], "slot", dev, -1), k.p, v.p, act,
                      ints(a[6], "status", dev, 1, true), stream);
    });
}

// attention(cache, device, layer, q, out, rows, row_lens, scale, lse, status, scratch, scratch_bytes)
PyObject *attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return call(n > 1 ? a[1] : nullptr, n, 12, "bmo_k_paged_attention", [&](int dev, void *stream) {
        const auto *c = reinterpret_cast<const bmo_paged_kv *>(integer(a[0]));
        const at::Tensor &query = tensor(a[3], "q");
        if (query.dim() != 3) refuse("q", "[n, heads, head_dim]");
        const int64_t tokens = query.size(0), heads = query.size(1);
        if (heads == 0 || heads % c->n_kv_heads) refuse("q", "a multiple of the key heads");
        const int act = act_type(query, "q");
        const Rows q = rows(a[3], "q", dev, tokens, heads, c->head_dim, query.scalar_type());
        const Rows out = rows(a[4], "out", dev, tokens, heads, c->head_dim, query.scalar_type());
        float *lse = nullptr;
        if (a[8] != Py_None) {
            const at::Tensor &t = tensor(a[8], "lse");
            on_device(t, "lse", dev);
            if (t.scalar_type() != at::kFloat || !t.is_contiguous() || t.dim() != 2 || t.size(0) != tokens || t.size(1) != heads)
                refuse("lse", "a contiguous float32 tensor [n, heads]");
            lse = static_cast<float *>(t.data_ptr());
        }
        return g_attention(c, layer_of(a[2]), count(tokens, "q"), q.p, q.stride, count(heads, "q"),
                           ints(a[5], "rows", dev, tokens, true), ints(a[6], "row_lens", dev, tokens, true),
                           number(a[7], "scale"), out.p, out.stride, lse, act,
                           ints(a[9], "status", dev, 1, true), reinterpret_cast<void *>(integer(a[10])),
                           static_cast<size_t>(integer(a[11])), stream);
    });
}

// bind(plan, append, read, attention): the entries' addresses
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 4) return PyErr_Format(PyExc_TypeError, "bind: 4 addresses");
    try {
        g_plan = reinterpret_cast<decltype(g_plan)>(integer(a[0]));
        g_append = reinterpret_cast<decltype(g_append)>(integer(a[1]));
        g_read = reinterpret_cast<decltype(g_read)>(integer(a[2]));
        g_attention = reinterpret_cast<decltype(g_attention)>(integer(a[3]));
    } catch (const Raised &) {
        return nullptr;
    }
    Py_RETURN_NONE;
}

#define BMO_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {BMO_METHOD(bind), BMO_METHOD(plan), BMO_METHOD(append), BMO_METHOD(read), BMO_METHOD(attention),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged() { return PyModule_Create(&module); }
