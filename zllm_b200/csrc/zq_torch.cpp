// Native half of the host mirror (zllm_b200/backend.py): the operators a decode step calls per projection, from Python objects
// straight to the C ABI.
//
// A decode projection of a small model runs for about 4 us on the GPU; building its ctypes arguments, reading the weight's
// shape through the ABI and allocating the output from Python took 6 us on top of the launch itself (10.1 us per call of a
// 1536 -> 512 projection, 3.8 us of them inside zq_linear).  Here a call costs one argument walk and one allocation from
// torch's caching allocator.  Checks, errors and results are those of the Python methods that call in.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <ATen/detail/CUDAHooksInterface.h>
#include <ATen/record_function.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <vector>

#include "../../include/zq_b200.h"

namespace {

PyObject *g_failure = nullptr;  // zllm_b200.ffi.ZqFailure
PyObject *s_handle, *s_rows, *s_cols;

struct PyError {};  // a Python exception is set

[[noreturn]] void fail(int code, const std::string &message) {
    PyObject *e = PyObject_CallFunction(g_failure, "is", code, message.c_str());
    if (e) {
        PyErr_SetObject(g_failure, e);
        Py_DECREF(e);
    }
    throw PyError();
}
void check(int rc, const zq_error &err) {
    if (rc) fail(rc, err.message);
}
[[noreturn]] void type_error(const std::string &message) {
    PyErr_SetString(PyExc_TypeError, message.c_str());
    throw PyError();
}

size_t attr_size(PyObject *o, PyObject *name) {
    PyObject *v = PyObject_GetAttr(o, name);
    if (!v) throw PyError();
    const size_t r = PyLong_AsSize_t(v);
    Py_DECREF(v);
    if (r == (size_t)-1 && PyErr_Occurred()) throw PyError();
    return r;
}
struct WeightRef {
    zq_weight *h;
    size_t rows, cols;
};
WeightRef weight_of(PyObject *o) { return {reinterpret_cast<zq_weight *>(attr_size(o, s_handle)), attr_size(o, s_rows), attr_size(o, s_cols)}; }

zq_ctx *ctx_of(PyObject *o) {
    void *p = PyLong_AsVoidPtr(o);
    if (!p && PyErr_Occurred()) throw PyError();
    return reinterpret_cast<zq_ctx *>(p);
}
at::Tensor tensor_of(PyObject *o) {
    if (!THPVariable_Check(o)) type_error("a tensor is expected, got " + std::string(Py_TYPE(o)->tp_name));
    return THPVariable_Unpack(o);
}
bool is_none(PyObject *o) { return o == Py_None; }
int zq_dtype(at::ScalarType t) { return t == at::kFloat ? ZQ_F32 : t == at::kHalf ? ZQ_F16 : t == at::kBFloat16 ? ZQ_BF16 : -1; }
std::string dtype_name(at::ScalarType t) {
    std::string n = at::toString(t);
    const char *known = t == at::kDouble ? "torch.float64" : t == at::kLong ? "torch.int64" : t == at::kInt ? "torch.int32" : t == at::kByte ? "torch.uint8" : t == at::kChar ? "torch.int8" : t == at::kBool ? "torch.bool" : nullptr;
    return known ? known : "torch." + n;
}
int in_dtype(const at::Tensor &x) {
    const int d = zq_dtype(x.scalar_type());
    if (d < 0) type_error("unsupported activation dtype " + dtype_name(x.scalar_type()));
    return d;
}
at::ScalarType dtype_of(PyObject *o) {
    if (!THPDtype_Check(o)) type_error("a torch dtype is expected");
    return reinterpret_cast<THPDtype *>(o)->scalar_type;
}
// out_dtype, or the input's dtype when it is None; KeyError for a dtype the library does not write
at::ScalarType out_dtype_of(PyObject *o, at::ScalarType fallback) {
    const at::ScalarType t = is_none(o) ? fallback : dtype_of(o);
    if (zq_dtype(t) < 0) {
        if (is_none(o)) type_error("unsupported activation dtype " + dtype_name(t));
        PyErr_SetObject(PyExc_KeyError, o);
        throw PyError();
    }
    return t;
}
size_t rows_of(const at::Tensor &x, size_t cols) {
    const int64_t last = x.dim() ? x.size(-1) : 1;
    if (cols == 0 || (size_t)last != cols) fail(1, "linear input cols=" + std::to_string(last) + ", weight cols=" + std::to_string(cols));
    return (size_t)x.numel() / cols;
}
// Other threads run while torch allocates (which may wait for the device) and inside the ABI (workspace growth, host-buffer calls).
struct NoGil {
    PyThreadState *s = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(s); }
};
// without the GIL.  On the GPU from torch's allocator directly (0.4 us instead of the 0.8 of at::empty), by way of its hooks, so that this library
// needs no CUDA build of torch to load, unless something is on that would see the call (dispatch modes, tracing, function transforms, autocast, the callbacks of
// profilers) or fill the tensor.
at::Tensor new_tensor(const at::Tensor &like, at::IntArrayRef size, at::ScalarType t) {
    const bool watched = !(c10::impl::tls_local_dispatch_key_set().included_ - c10::default_included_set).empty() || at::getStepCallbacksUnlessEmpty(at::RecordScope::FUNCTION).has_value();
    if (like.is_cuda() && !watched && !at::globalContext().deterministicAlgorithms()) {
        const c10::DeviceGuard on(like.device());
        return at::Tensor(at::detail::empty_generic(size, at::detail::getCUDAHooks().getCUDADeviceAllocator(), c10::DispatchKeySet(c10::DispatchKey::CUDA), t, std::nullopt));
    }
    return at::empty(size, like.options().dtype(t));
}
at::Tensor new_rows(const at::Tensor &like, size_t m, size_t n, at::ScalarType t) {
    const int64_t size[2] = {(int64_t)m, (int64_t)n};
    return new_tensor(like, size, t);
}
at::Tensor contiguous(const at::Tensor &t) {
    if (t.is_contiguous()) return t;
    NoGil g;
    return t.contiguous();
}
at::Tensor as_f32(const at::Tensor &t) {
    if (t.scalar_type() == at::kFloat) return t;
    NoGil g;
    return t.to(at::kFloat);
}

template <class Fn> PyObject *guarded(Fn fn) {
    try {
        return fn();
    } catch (const PyError &) {
        return nullptr;
    } catch (...) {  // torch's own errors become the exceptions torch raises from Python (an allocation that fails: torch.OutOfMemoryError)
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}
template <class Tensors> PyObject *wrap_list(Tensors &ys) {
    PyObject *out = PyList_New((Py_ssize_t)ys.size());
    if (!out) throw PyError();
    for (size_t i = 0; i < ys.size(); ++i) PyList_SET_ITEM(out, (Py_ssize_t)i, THPVariable_Wrap(std::move(ys[i])));  // None for one that was never made
    return out;
}
// The items of a sequence for the time of a call.
struct Items {
    PyObject *fast;
    Items(PyObject *seq) : fast(PySequence_Fast(seq, "a sequence is expected")) {
        if (!fast) throw PyError();
    }
    ~Items() { Py_DECREF(fast); }
    size_t size() const { return (size_t)PySequence_Fast_GET_SIZE(fast); }
    PyObject *operator[](size_t i) const { return PySequence_Fast_GET_ITEM(fast, (Py_ssize_t)i); }
};

// KeyError(x.dtype): what a batch raises for inputs the library does not read
[[noreturn]] void dtype_key_error(PyObject *x) {
    PyObject *dtype = PyObject_GetAttrString(x, "dtype");
    if (dtype) {
        PyErr_SetObject(PyExc_KeyError, dtype);
        Py_DECREF(dtype);
    }
    throw PyError();
}

// linear(ctx, x, weight, out_dtype, residual)
PyObject *py_linear(PyObject *, PyObject *const *a, Py_ssize_t) {
    return guarded([&]() -> PyObject * {
        zq_ctx *ctx = ctx_of(a[0]);
        const at::Tensor x = contiguous(tensor_of(a[1]));
        const WeightRef w = weight_of(a[2]);
        const size_t m = rows_of(x, w.cols);
        const at::ScalarType od = out_dtype_of(a[3], x.scalar_type());
        at::Tensor y, r;
        if (!is_none(a[4])) {
            r = contiguous(tensor_of(a[4]));
            if ((size_t)r.numel() != m * w.rows || r.scalar_type() != od) fail(1, "residual shape/dtype mismatch: " + std::to_string(r.numel()) + " values of " + dtype_name(r.scalar_type()) + " vs " + std::to_string(m * w.rows) + " of " + dtype_name(od));
        }
        const int xd = in_dtype(x);
        zq_error err;
        int rc;
        {
            NoGil g;
            y = new_rows(x, m, w.rows, od);
            rc = zq_linear(ctx, w.h, x.data_ptr(), xd, m, y.data_ptr(), zq_dtype(od), r.defined() ? r.data_ptr() : nullptr, &err);
        }
        check(rc, err);
        return THPVariable_Wrap(std::move(y));
    });
}

// linear_batch(ctx, jobs, out_dtype)
PyObject *py_linear_batch(PyObject *, PyObject *const *a, Py_ssize_t) {
    return guarded([&]() -> PyObject * {
        zq_ctx *ctx = ctx_of(a[0]);
        Items jobs(a[1]);
        const size_t n = jobs.size();
        std::vector<zq_linear_job> arr(n);
        std::vector<at::Tensor> ys(n), inputs(n), keep;
        std::vector<size_t> rows(n);
        at::ScalarType xt = at::kFloat, od = at::kFloat;
        for (size_t i = 0; i < n; ++i) {
            Items job(jobs[i]);
            if (job.size() < 2) type_error("linear_batch: a job is (x, weight[, residual]) or (x, gate, up, \"gated\") or (x, weight, residual, \"row\")");
            bool gated = false, row = false;
            if (job.size() == 4 && PyUnicode_Check(job[3])) {
                gated = PyUnicode_CompareWithASCIIString(job[3], "gated") == 0;
                row = PyUnicode_CompareWithASCIIString(job[3], "row") == 0;
            }
            const at::Tensor x = contiguous(tensor_of(job[0]));
            const WeightRef w = weight_of(job[1]);
            const size_t m = rows_of(x, w.cols);
            if (i == 0) {
                xt = x.scalar_type();
                if (zq_dtype(xt) < 0) dtype_key_error(job[0]);
                od = out_dtype_of(a[2], xt);
            }
            if (x.scalar_type() != xt) type_error("linear_batch: all inputs must share one dtype");
            zq_linear_job &j = arr[i];
            j = {};
            j.w = w.h;
            j.w_up = gated ? weight_of(job[2]).h : nullptr;
            j.dev_x = x.data_ptr();
            j.m = m;
            rows[i] = w.rows;
            inputs[i] = x;
            if ((job.size() == 3 || row) && !is_none(job[2])) {
                const at::Tensor r = contiguous(tensor_of(job[2]));
                j.dev_residual = r.data_ptr();
                keep.push_back(r);
            }
            j.flags = row ? ZQ_JOB_ROW_PARALLEL : 0;
        }
        if (n) {
            zq_error err;
            int rc;
            {
                NoGil g;
                for (size_t i = 0; i < n; ++i) {
                    ys[i] = new_rows(inputs[i], arr[i].m, rows[i], od);
                    arr[i].dev_y = ys[i].data_ptr();
                }
                rc = zq_linear_batch(ctx, arr.data(), n, zq_dtype(xt), zq_dtype(od), &err);
            }
            check(rc, err);
        }
        return wrap_list(ys);
    });
}

// linear_multi(ctx, x, weights, out_dtype, norm_weight | None, eps, weight_offset)
PyObject *py_linear_multi(PyObject *, PyObject *const *a, Py_ssize_t) {
    return guarded([&]() -> PyObject * {
        zq_ctx *ctx = ctx_of(a[0]);
        const at::Tensor x = contiguous(tensor_of(a[1]));
        Items ws(a[2]);
        const size_t n = ws.size();
        if (!n) {
            PyErr_SetString(PyExc_IndexError, "no weights given");
            throw PyError();
        }
        c10::SmallVector<const zq_weight *, 4> wh(n);
        c10::SmallVector<at::Tensor, 4> ys(n);
        c10::SmallVector<void *, 4> yp(n);
        c10::SmallVector<size_t, 4> rows(n);
        const size_t cols = weight_of(ws[0]).cols, m = rows_of(x, cols);
        at::Tensor norm;
        if (!is_none(a[4])) {
            norm = as_f32(contiguous(tensor_of(a[4])));
            if ((size_t)norm.numel() != cols) fail(1, "norm weight has " + std::to_string(norm.numel()) + " elements, input width is " + std::to_string(cols));
        }
        const at::ScalarType od = out_dtype_of(a[3], x.scalar_type());
        for (size_t i = 0; i < n; ++i) {
            const WeightRef w = weight_of(ws[i]);
            wh[i] = w.h;
            rows[i] = w.rows;
        }
        const int xd = in_dtype(x);
        const double eps = PyFloat_AsDouble(a[5]), offset = PyFloat_AsDouble(a[6]);
        if (PyErr_Occurred()) throw PyError();
        zq_error err;
        int rc;
        {
            NoGil g;
            for (size_t i = 0; i < n; ++i) {
                ys[i] = new_rows(x, m, rows[i], od);
                yp[i] = ys[i].data_ptr();
            }
            rc = norm.defined() ? zq_rmsnorm_linear(ctx, wh.data(), n, x.data_ptr(), xd, m, norm.data_ptr<float>(), (float)eps, (float)offset, yp.data(), zq_dtype(od), &err)
                                : zq_linear_multi(ctx, wh.data(), n, x.data_ptr(), xd, m, yp.data(), zq_dtype(od), &err);
        }
        check(rc, err);
        return wrap_list(ys);
    });
}

// gated(ctx, x, gate, up, down | None, out_dtype, residual)
PyObject *py_gated(PyObject *, PyObject *const *a, Py_ssize_t) {
    return guarded([&]() -> PyObject * {
        zq_ctx *ctx = ctx_of(a[0]);
        const at::Tensor x = contiguous(tensor_of(a[1]));
        const WeightRef gate = weight_of(a[2]), up = weight_of(a[3]);
        const bool mlp = !is_none(a[4]);
        const WeightRef down = mlp ? weight_of(a[4]) : WeightRef{nullptr, gate.rows, 0};
        const size_t m = rows_of(x, gate.cols);
        const at::ScalarType od = out_dtype_of(a[5], x.scalar_type());
        at::Tensor y, r;
        if (!is_none(a[6])) r = contiguous(tensor_of(a[6]));
        const int xd = in_dtype(x);
        zq_error err;
        int rc;
        {
            NoGil g;
            y = new_rows(x, m, down.rows, od);
            rc = mlp ? zq_gated_mlp(ctx, gate.h, up.h, down.h, x.data_ptr(), xd, m, y.data_ptr(), zq_dtype(od), r.defined() ? r.data_ptr() : nullptr, &err)
                     : zq_gated_silu(ctx, gate.h, up.h, x.data_ptr(), xd, m, y.data_ptr(), zq_dtype(od), &err);
        }
        check(rc, err);
        return THPVariable_Wrap(std::move(y));
    });
}

// rope(ctx, query, key | None, num_heads, num_kv_heads, rotary_dim, position, cos, sin, interleaved, suffix)
PyObject *py_rope(PyObject *, PyObject *const *a, Py_ssize_t) {
    return guarded([&]() -> PyObject * {
        zq_ctx *ctx = ctx_of(a[0]);
        const at::Tensor q = tensor_of(a[1]);
        at::Tensor k;
        if (!is_none(a[2])) k = tensor_of(a[2]);
        long v[6];
        const int at_[6] = {3, 4, 5, 6, 9, 10};
        for (int i = 0; i < 6; ++i) {
            v[i] = i < 4 ? PyLong_AsLong(a[at_[i]]) : PyObject_IsTrue(a[at_[i]]);
            if (v[i] == -1 && PyErr_Occurred()) throw PyError();
        }
        const int64_t rows = q.dim() > 1 ? q.size(0) : 1;
        if (rows == 0 || v[0] == 0) {
            PyErr_SetString(PyExc_ZeroDivisionError, "rope: no rows or no heads");
            throw PyError();
        }
        const int64_t head_dim = q.numel() / rows / v[0];
        if (k.defined() && (k.scalar_type() != q.scalar_type() || k.numel() != rows * v[1] * head_dim)) fail(1, "rope: key shape or dtype does not match the query's");
        const at::Tensor c = as_f32(contiguous(tensor_of(a[7]))), s = as_f32(contiguous(tensor_of(a[8])));
        if (c.numel() != s.numel()) fail(1, "rope: cos and sin tables differ in length (" + std::to_string(c.numel()) + " / " + std::to_string(s.numel()) + ")");
        const int d = in_dtype(q);
        zq_error err;
        int rc;
        {
            NoGil g;
            rc = zq_rope_qk(ctx, q.data_ptr(), (size_t)v[0], k.defined() ? k.data_ptr() : nullptr, k.defined() ? (size_t)v[1] : 0, d, (size_t)rows, (size_t)head_dim, (size_t)v[2], (int)v[4], (int)v[5], (size_t)v[3],
                            c.data_ptr<float>(), s.data_ptr<float>(), (size_t)c.numel(), &err);
        }
        check(rc, err);
        Py_RETURN_NONE;
    });
}

// gather_rows(ctx, weight, row_ids, dtype): row_ids on the weight's device, int32, contiguous
PyObject *py_gather_rows(PyObject *, PyObject *const *a, Py_ssize_t) {
    return guarded([&]() -> PyObject * {
        zq_ctx *ctx = ctx_of(a[0]);
        const WeightRef w = weight_of(a[1]);
        const at::Tensor ids = tensor_of(a[2]);
        const at::ScalarType t = dtype_of(a[3]);
        zq_error err;
        int rc;
        at::Tensor y;
        {
            NoGil g;
            y = new_rows(ids, (size_t)ids.numel(), w.cols, t);
            rc = zq_gather_rows(ctx, w.h, reinterpret_cast<const uint32_t *>(ids.data_ptr<int>()), (size_t)ids.numel(), y.data_ptr(), zq_dtype(t), &err);
        }
        check(rc, err);
        return THPVariable_Wrap(std::move(y));
    });
}

// linear_host_batch(ctx, jobs): (x, weight, y) with x and y buffers of f32 or f16
PyObject *py_linear_host_batch(PyObject *, PyObject *const *a, Py_ssize_t) {
    return guarded([&]() -> PyObject * {
        zq_ctx *ctx = ctx_of(a[0]);
        Items jobs(a[1]);
        const size_t n = jobs.size();
        std::vector<zq_linear_host_job> arr(n);
        struct View {
            Py_buffer b;
            bool held = false;
            ~View() {
                if (held) PyBuffer_Release(&b);
            }
        };
        std::vector<View> views(2 * n);
        int dt[2] = {ZQ_F32, ZQ_F32};
        for (size_t i = 0; i < n; ++i) {
            Items job(jobs[i]);
            if (job.size() != 3) type_error("linear_host_batch: a job is (x, weight, y)");
            const WeightRef w = weight_of(job[1]);
            for (int k = 0; k < 2; ++k) {
                View &v = views[2 * i + k];
                if (PyObject_GetBuffer(job[2 * k], &v.b, PyBUF_FORMAT | PyBUF_STRIDES)) throw PyError();
                v.held = true;
                if (i == 0) {
                    const char *f = v.b.format ? v.b.format : "";
                    dt[k] = !strcmp(f, "f") ? ZQ_F32 : !strcmp(f, "e") ? ZQ_F16 : -1;
                    if (dt[k] < 0) {
                        PyErr_SetString(PyExc_KeyError, f);
                        throw PyError();
                    }
                }
            }
            if (w.cols == 0) fail(4, "linear_host_batch: the weight was released");
            arr[i] = {w.h, views[2 * i].b.buf, (size_t)(views[2 * i].b.len / views[2 * i].b.itemsize) / w.cols, views[2 * i + 1].b.buf};
        }
        if (!n) {
            PyErr_SetString(PyExc_IndexError, "list index out of range");
            throw PyError();
        }
        zq_error err;
        int rc;
        {
            NoGil g;
            rc = zq_linear_host_batch(ctx, arr.data(), n, dt[0], dt[1], &err);
        }
        check(rc, err);
        Py_RETURN_NONE;
    });
}

// ---- drafted tokens over a paged cache.  Tensors of these operators are checked for their device too: (ctx, device index, ...).
int device_of(PyObject *o) {
    const long d = PyLong_AsLong(o);
    if (d == -1 && PyErr_Occurred()) throw PyError();
    return (int)d;
}
at::Tensor on_device(PyObject *o, int device, const char *what) {
    at::Tensor t = tensor_of(o);
    if (!t.is_cuda() || t.get_device() != device) fail(4, std::string(what) + " is not on the context's device cuda:" + std::to_string(device));
    return t;
}
std::string sizes_of(const at::Tensor &t) {
    std::string s = "[";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "]";
}
// A tensor of plain values: its type and how many it holds.
at::Tensor values(PyObject *o, int device, const char *what, at::ScalarType type, int64_t count) {
    at::Tensor t = on_device(o, device, what);
    if (t.scalar_type() != type) type_error(std::string(what) + " is " + dtype_name(type) + ", not " + dtype_name(t.scalar_type()));
    if (t.numel() != count) fail(1, std::string(what) + " of shape " + sizes_of(t) + ": " + std::to_string(count) + " values are needed");
    return contiguous(t);
}
// Rows of [heads, head_dim] values at one distance: the tensor itself, or a dense copy where its strides are others.
struct Rows {
    at::Tensor t;
    int64_t rows, heads, dim, stride;
};
Rows rows_3d(PyObject *o, int device, const char *what) {
    Rows r{on_device(o, device, what), 1, 0, 0, 0};
    if (r.t.dim() < 3) fail(1, std::string(what) + " of shape " + sizes_of(r.t) + ": [..., heads, head_dim] is needed");
    const int64_t n = r.t.dim();
    r.heads = r.t.size(n - 2);
    r.dim = r.t.size(n - 1);
    for (int64_t i = 0; i < n - 2; ++i) r.rows *= r.t.size(i);
    if (r.rows == 0 || r.heads == 0 || r.dim == 0) fail(1, std::string(what) + " of shape " + sizes_of(r.t) + " is empty");
    bool one = (r.dim == 1 || r.t.stride(n - 1) == 1) && (r.heads == 1 || r.t.stride(n - 2) == r.dim);
    int64_t step = r.heads * r.dim, inner = 1;  // the leading dimensions as one; a single row needs no distance
    bool seen = false;                          // a dimension of more than one row, whose stride may be 0 (expanded)
    for (int64_t i = n - 3; i >= 0 && one; --i) {
        if (r.t.size(i) == 1) continue;
        if (!seen) step = r.t.stride(i);
        else one = r.t.stride(i) == step * inner;
        seen = true;
        inner *= r.t.size(i);
    }
    if (!one || step < r.heads * r.dim) {
        r.t = contiguous(r.t);
        step = r.heads * r.dim;
    }
    r.stride = step;
    return r;
}
struct Cache {
    at::Tensor k, v, blocks, lens;
    zq_kv_cache c;
};
Cache cache_of(PyObject *k, PyObject *v, PyObject *blocks, PyObject *lens, int device, bool layers) {
    Cache s;
    s.k = on_device(k, device, "k_pages");
    s.v = on_device(v, device, "v_pages");
    const int64_t n = s.k.dim();
    if (n != 4 && !(layers && n == 5)) fail(1, "k_pages of shape " + sizes_of(s.k) + ": [pages, page_size, heads, head_dim] is needed" + (layers ? ", or that behind a dimension of layers" : ""));
    if (s.k.scalar_type() != s.v.scalar_type()) type_error("k_pages is " + dtype_name(s.k.scalar_type()) + " and v_pages " + dtype_name(s.v.scalar_type()));
    bool alike = s.k.sizes() == s.v.sizes();
    for (int64_t i = 0; alike && i < n; ++i) alike = s.k.size(i) == 1 || s.k.stride(i) == s.v.stride(i);  // a dimension of one has any stride
    if (!alike) fail(1, "k_pages and v_pages differ in shape or strides: " + sizes_of(s.k) + ", " + sizes_of(s.v));
    if (s.k.numel() == 0) fail(1, "k_pages of shape " + sizes_of(s.k) + " is empty");
    const int64_t heads = s.k.size(n - 2), dim = s.k.size(n - 1), size = s.k.size(n - 3);
    if ((dim > 1 && s.k.stride(n - 1) != 1) || (heads > 1 && s.k.stride(n - 2) != dim) || (size > 1 && s.k.stride(n - 3) != heads * dim)) fail(1, "a page of the cache is not dense");
    s.blocks = on_device(blocks, device, "block_table");
    if (s.blocks.scalar_type() != at::kInt) type_error("block_table is torch.int32, not " + dtype_name(s.blocks.scalar_type()));
    if (s.blocks.dim() != 2 || s.blocks.numel() == 0) fail(1, "block_table of shape " + sizes_of(s.blocks) + ": [sequences, blocks] is needed");
    s.blocks = contiguous(s.blocks);
    s.lens = values(lens, device, "context_lens", at::kInt, s.blocks.size(0));
    const int64_t pages = s.k.size(n - 4), page = size * heads * dim, page_stride = pages > 1 ? s.k.stride(n - 4) : page;
    if (page_stride < page) fail(1, "the pages of the cache overlap");
    const int64_t n_layers = n == 5 ? s.k.size(0) : 1;
    const int64_t layer_stride = n_layers > 1 ? s.k.stride(0) : 0;
    if (n_layers > 1 && layer_stride < page) fail(1, "the layers of the cache overlap");
    s.c = {s.k.data_ptr(), s.v.data_ptr(), zq_dtype(s.k.scalar_type()), (size_t)pages, (size_t)size, (size_t)heads, (size_t)dim, (size_t)page_stride, (size_t)n_layers, (size_t)layer_stride,
           s.blocks.data_ptr<int>(), (size_t)s.blocks.size(0), (size_t)s.blocks.size(1), s.lens.data_ptr<int>()};
    return s;
}
at::Tensor optional_lens(PyObject *o, int device, const char *what, int64_t count) { return is_none(o) ? at::Tensor() : values(o, device, what, at::kInt, count); }
const int32_t *ints_or_null(const at::Tensor &t) { return t.defined() ? t.data_ptr<int>() : nullptr; }
bool truth(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PyError();
    return v != 0;
}
double number(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PyError();
    return v;
}

// parents: [rows] for all sequences or [sequences, rows]
struct Parents {
    at::Tensor t;
    bool shared;
};
Parents parents_of(PyObject *o, int device, int64_t batch, int64_t rows) {
    at::Tensor t = on_device(o, device, "parents");
    if (t.scalar_type() != at::kInt) type_error("parents is torch.int32, not " + dtype_name(t.scalar_type()));
    const bool shared = t.dim() == 1;
    if ((t.dim() != 1 && t.dim() != 2) || t.size(-1) != rows || (!shared && t.size(0) != batch)) fail(1, "parents of shape " + sizes_of(t) + " for " + std::to_string(batch) + " sequences of " + std::to_string(rows) + " rows");
    return {contiguous(t), shared};
}

// draft_tree(ctx, device, parents, context_lens, draft_lens | None) -> positions, mask
PyObject *py_draft_tree(PyObject *, PyObject *const *a, Py_ssize_t) {
    return guarded([&]() -> PyObject * {
        zq_ctx *ctx = ctx_of(a[0]);
        const int device = device_of(a[1]);
        const at::Tensor lens = on_device(a[3], device, "context_lens"), given = on_device(a[2], device, "parents");
        const int64_t batch = lens.numel(), rows = given.dim() ? given.size(-1) : 0;
        const Parents parents = parents_of(a[2], device, batch, rows);
        const at::Tensor context = values(a[3], device, "context_lens", at::kInt, batch), drafted = optional_lens(a[4], device, "draft_lens", batch);
        std::vector<at::Tensor> out(2);
        zq_error err;
        int rc;
        {
            NoGil g;
            out[0] = new_tensor(context, {batch, rows}, at::kInt);
            out[1] = new_tensor(context, {batch, rows, (rows + 63) / 64}, at::kLong);
            rc = zq_draft_tree(ctx, parents.t.data_ptr<int>(), parents.shared, (size_t)batch, (size_t)rows, context.data_ptr<int>(), ints_or_null(drafted), out[0].data_ptr<int>(), reinterpret_cast<uint64_t *>(out[1].data_ptr<int64_t>()), &err);
        }
        check(rc, err);
        return wrap_list(out);
    });
}

// rope_rows(ctx, device, query, key | None, positions, inv_freq, interleaved, suffix, factor, inverse) -> query, key
PyObject *py_rope_rows(PyObject *, PyObject *const *a, Py_ssize_t) {
    return guarded([&]() -> PyObject * {
        zq_ctx *ctx = ctx_of(a[0]);
        const int device = device_of(a[1]);
        const Rows q = rows_3d(a[2], device, "query");
        Rows k{};
        if (!is_none(a[3])) {
            k = rows_3d(a[3], device, "key");
            if (k.rows != q.rows || k.dim != q.dim || k.t.scalar_type() != q.t.scalar_type()) fail(1, "rope_rows: key of shape " + sizes_of(k.t) + " or its dtype does not match the query's " + sizes_of(q.t));
        }
        const int d = in_dtype(q.t);
        const at::Tensor positions = values(a[4], device, "positions", at::kInt, q.rows);
        const at::Tensor freq = on_device(a[5], device, "inv_freq");
        const at::Tensor inv_freq = values(a[5], device, "inv_freq", at::kFloat, freq.numel());
        const bool interleaved = truth(a[6]), suffix = truth(a[7]), inverse = truth(a[9]);
        const float factor = (float)number(a[8]);
        std::vector<at::Tensor> out(2);
        zq_error err;
        int rc;
        {
            NoGil g;
            out[0] = new_tensor(q.t, q.t.sizes(), q.t.scalar_type());
            if (k.t.defined()) out[1] = new_tensor(k.t, k.t.sizes(), k.t.scalar_type());
            rc = zq_rope_rows(ctx, q.t.data_ptr(), (size_t)q.heads, (size_t)q.stride, k.t.defined() ? k.t.data_ptr() : nullptr, (size_t)k.heads, (size_t)k.stride, d, (size_t)q.rows, (size_t)q.dim, (size_t)(2 * inv_freq.numel()), interleaved, suffix,
                              positions.data_ptr<int>(), inv_freq.data_ptr<float>(), factor, inverse, out[0].data_ptr(), k.t.defined() ? out[1].data_ptr() : nullptr, &err);
        }
        check(rc, err);
        return wrap_list(out);
    });
}

// rope_append(ctx, device, query, key, value, k_pages, v_pages, block_table, context_lens, positions, inv_freq, draft_lens | None, interleaved, suffix, factor) -> query
PyObject *py_rope_append(PyObject *, PyObject *const *a, Py_ssize_t) {
    return guarded([&]() -> PyObject * {
        zq_ctx *ctx = ctx_of(a[0]);
        const int device = device_of(a[1]);
        const Rows q = rows_3d(a[2], device, "query"), k = rows_3d(a[3], device, "key"), v = rows_3d(a[4], device, "value");
        const Cache cache = cache_of(a[5], a[6], a[7], a[8], device, false);
        const int64_t batch = (int64_t)cache.c.batch;
        if (q.rows % batch || k.rows != q.rows || v.rows != q.rows) fail(1, "rope_append: " + std::to_string(q.rows) + " / " + std::to_string(k.rows) + " / " + std::to_string(v.rows) + " rows for " + std::to_string(batch) + " sequences");
        if (q.dim != (int64_t)cache.c.head_dim || k.dim != q.dim || v.dim != q.dim || k.heads != (int64_t)cache.c.heads || v.heads != k.heads) fail(1, "rope_append: heads of key " + sizes_of(k.t) + " or value " + sizes_of(v.t) + " are not the cache's " + sizes_of(cache.k));
        if (q.t.scalar_type() != cache.k.scalar_type() || k.t.scalar_type() != q.t.scalar_type() || v.t.scalar_type() != q.t.scalar_type()) type_error("rope_append: query, key and value have the cache's dtype " + dtype_name(cache.k.scalar_type()));
        const at::Tensor positions = values(a[9], device, "positions", at::kInt, q.rows);
        const at::Tensor freq = on_device(a[10], device, "inv_freq");
        const at::Tensor inv_freq = values(a[10], device, "inv_freq", at::kFloat, freq.numel()), drafted = optional_lens(a[11], device, "draft_lens", batch);
        const bool interleaved = truth(a[12]), suffix = truth(a[13]);
        const float factor = (float)number(a[14]);
        at::Tensor out;
        zq_error err;
        int rc;
        {
            NoGil g;
            out = new_tensor(q.t, q.t.sizes(), q.t.scalar_type());
            rc = zq_rope_append(ctx, q.t.data_ptr(), (size_t)q.heads, (size_t)q.stride, k.t.data_ptr(), (size_t)k.stride, v.t.data_ptr(), (size_t)v.stride, (size_t)(q.rows / batch), &cache.c, ints_or_null(drafted), (size_t)(2 * inv_freq.numel()),
                                interleaved, suffix, positions.data_ptr<int>(), inv_freq.data_ptr<float>(), factor, out.data_ptr(), &err);
        }
        check(rc, err);
        return THPVariable_Wrap(std::move(out));
    });
}

// tree_attention(ctx, device, query, k_pages, v_pages, block_table, context_lens, mask | None, draft_lens | None, scale | None) -> rows
PyObject *py_tree_attention(PyObject *, PyObject *const *a, Py_ssize_t) {
    return guarded([&]() -> PyObject * {
        zq_ctx *ctx = ctx_of(a[0]);
        const int device = device_of(a[1]);
        Rows q = rows_3d(a[2], device, "query");
        if (q.stride % 8 || (reinterpret_cast<uintptr_t>(q.t.data_ptr()) & 15)) {  // the kernels read whole words, the fast one 16 bytes
            NoGil g;
            q.t = q.t.clone(at::MemoryFormat::Contiguous);
            q.stride = q.heads * q.dim;
        }
        const Cache cache = cache_of(a[3], a[4], a[5], a[6], device, false);
        const int64_t batch = (int64_t)cache.c.batch, rows = q.rows / batch;
        if (q.rows % batch || q.dim != (int64_t)cache.c.head_dim) fail(1, "tree_attention: query of shape " + sizes_of(q.t) + " for " + std::to_string(batch) + " sequences of a cache of " + sizes_of(cache.k));
        if (q.t.scalar_type() != cache.k.scalar_type()) type_error("tree_attention: the query has the cache's dtype " + dtype_name(cache.k.scalar_type()) + ", not " + dtype_name(q.t.scalar_type()));
        at::Tensor mask;
        if (!is_none(a[7])) mask = values(a[7], device, "mask", at::kLong, batch * rows * ((rows + 63) / 64));
        const at::Tensor drafted = optional_lens(a[8], device, "draft_lens", batch);
        const float scale = is_none(a[9]) ? (float)(1.0 / std::sqrt((double)q.dim)) : (float)number(a[9]);
        at::Tensor out;
        zq_error err;
        int rc;
        {
            NoGil g;
            out = new_tensor(q.t, q.t.sizes(), q.t.scalar_type());
            rc = zq_tree_attention(ctx, q.t.data_ptr(), (size_t)q.heads, (size_t)q.stride, (size_t)rows, &cache.c, mask.defined() ? reinterpret_cast<const uint64_t *>(mask.data_ptr<int64_t>()) : nullptr, ints_or_null(drafted), scale, out.data_ptr(),
                                   &err);
        }
        check(rc, err);
        return THPVariable_Wrap(std::move(out));
    });
}

// verify_draft(ctx, device, logits, tokens, parents, accept_u, sample_u, temperature, draft_logits | None, draft_lens | None) -> path, accepted, token
PyObject *py_verify_draft(PyObject *, PyObject *const *a, Py_ssize_t) {
    return guarded([&]() -> PyObject * {
        zq_ctx *ctx = ctx_of(a[0]);
        const int device = device_of(a[1]);
        const at::Tensor logits = contiguous(on_device(a[2], device, "logits"));
        if (logits.dim() != 3 || logits.numel() == 0) fail(1, "logits of shape " + sizes_of(logits) + ": [sequences, rows, vocabulary] is needed");
        const int64_t batch = logits.size(0), rows = logits.size(1);
        const int d = in_dtype(logits);
        const at::Tensor tokens = values(a[3], device, "tokens", at::kInt, batch * rows);
        const Parents parents = parents_of(a[4], device, batch, rows);
        const at::Tensor accept_u = values(a[5], device, "accept_u", at::kFloat, batch * rows), sample_u = values(a[6], device, "sample_u", at::kFloat, batch), heat = values(a[7], device, "temperature", at::kFloat, batch);
        at::Tensor draft;
        if (!is_none(a[8])) {
            draft = values(a[8], device, "draft_logits", logits.scalar_type(), logits.numel());
            if (tensor_of(a[8]).sizes() != logits.sizes()) fail(1, "draft_logits of shape " + sizes_of(draft) + " for logits of " + sizes_of(logits));
        }
        const at::Tensor drafted = optional_lens(a[9], device, "draft_lens", batch);
        std::vector<at::Tensor> out(3);
        zq_error err;
        int rc;
        {
            NoGil g;
            out[0] = new_tensor(logits, {batch, rows}, at::kInt);
            out[1] = new_tensor(logits, {batch}, at::kInt);
            out[2] = new_tensor(logits, {batch}, at::kInt);
            rc = zq_verify_draft(ctx, logits.data_ptr(), draft.defined() ? draft.data_ptr() : nullptr, d, (size_t)batch, (size_t)rows, (size_t)logits.size(2), tokens.data_ptr<int>(), parents.t.data_ptr<int>(), parents.shared, accept_u.data_ptr<float>(),
                                 sample_u.data_ptr<float>(), heat.data_ptr<float>(), ints_or_null(drafted), out[0].data_ptr<int>(), out[1].data_ptr<int>(), out[2].data_ptr<int>(), &err);
        }
        check(rc, err);
        return wrap_list(out);
    });
}

// cache_keep_path(ctx, device, k_pages, v_pages, block_table, context_lens, path, accepted)
PyObject *py_cache_keep_path(PyObject *, PyObject *const *a, Py_ssize_t) {
    return guarded([&]() -> PyObject * {
        zq_ctx *ctx = ctx_of(a[0]);
        const int device = device_of(a[1]);
        const Cache cache = cache_of(a[2], a[3], a[4], a[5], device, true);
        const at::Tensor given = on_device(a[6], device, "path");
        if (given.dim() != 2 || given.size(0) != (int64_t)cache.c.batch) fail(1, "path of shape " + sizes_of(given) + " for " + std::to_string(cache.c.batch) + " sequences");
        const at::Tensor path = values(a[6], device, "path", at::kInt, given.numel()), accepted = values(a[7], device, "accepted", at::kInt, (int64_t)cache.c.batch);
        zq_error err;
        int rc;
        {
            NoGil g;
            rc = zq_cache_keep_path(ctx, &cache.c, path.data_ptr<int>(), (size_t)path.size(1), accepted.data_ptr<int>(), &err);
        }
        check(rc, err);
        Py_RETURN_NONE;
    });
}

PyObject *py_setup(PyObject *, PyObject *failure) {
    Py_INCREF(failure);
    Py_XSETREF(g_failure, failure);
    Py_RETURN_NONE;
}

template <Py_ssize_t N, PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)> PyObject *counted(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", N, n);
        return nullptr;
    }
    return F(self, a, n);
}
#define ZQ_FAST(name, n, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&counted<n, fn>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    ZQ_FAST("linear", 5, py_linear), ZQ_FAST("linear_batch", 3, py_linear_batch), ZQ_FAST("linear_multi", 7, py_linear_multi), ZQ_FAST("gated", 7, py_gated),
    ZQ_FAST("rope", 11, py_rope), ZQ_FAST("gather_rows", 4, py_gather_rows), ZQ_FAST("linear_host_batch", 2, py_linear_host_batch),
    ZQ_FAST("draft_tree", 5, py_draft_tree), ZQ_FAST("rope_rows", 10, py_rope_rows), ZQ_FAST("rope_append", 15, py_rope_append), ZQ_FAST("tree_attention", 10, py_tree_attention), ZQ_FAST("verify_draft", 10, py_verify_draft),
    ZQ_FAST("cache_keep_path", 8, py_cache_keep_path), {"setup", py_setup, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_zq_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__zq_torch() {
    s_handle = PyUnicode_InternFromString("_h");
    s_rows = PyUnicode_InternFromString("_rows");
    s_cols = PyUnicode_InternFromString("_cols");
    return PyModule_Create(&module);
}
