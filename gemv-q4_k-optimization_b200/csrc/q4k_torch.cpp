// q4k_torch.cpp -- native front-end of the per-request entries for torch
// tensors (Python module _q4k_torch, used by __init__.py).
//
// These calls run many times per token and take a few microseconds on the
// device; checking tensors, allocating outputs and filling the C structs from
// Python took 12-16 us of host time per call, here it takes about one beside
// the launch. The module holds no pointers into libq4k_gemv.so of its own:
// bind() hands it the loaded library's entries, so another build of the
// library can be put in its place.
#include "q4k_gemv.h"

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/Functions.h>

#include <cstdarg>
#include <cstdio>
#include <exception>
#include <optional>
#include <string>

namespace {

// ---- the library's entries, and the error class ------------------------------
decltype(&q4k_lora_batch) g_lora = nullptr;
decltype(&q4k_lora_workspace_bytes) g_lora_bytes = nullptr;
decltype(&q4k_rope_multi) g_rope = nullptr;
decltype(&q4k_logits_process) g_logits = nullptr;
decltype(&q4k_last_error) g_last_error = nullptr;
PyObject *g_error = nullptr;  // Q4KError(status, message)

struct Refused {  // becomes a Q4KError
    int status;
    std::string message;
};
struct PythonError {};  // a Python exception is set

[[noreturn]] void refuse(const char *fmt, ...) {
    char buf[400];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    throw Refused{Q4K_EINVAL, buf};
}
void check(int status) {
    if (status != Q4K_OK) throw Refused{status, g_last_error()};
}

// Runs f() and turns what it throws into a Python exception.
template <typename F> PyObject *guarded(F f) {
    try {
        if (g_error == nullptr) refuse("bind() has not been called");
        return f();
    } catch (const Refused &r) {
        PyObject *e = PyObject_CallFunction(g_error, "is", r.status, r.message.c_str());
        if (e != nullptr) {
            PyErr_SetObject(g_error, e);
            Py_DECREF(e);
        }
    } catch (const PythonError &) {
    } catch (...) {  // torch's own, such as an allocation that does not fit
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

// ---- tensors -------------------------------------------------------------------
std::string shape_of(const at::Tensor &t) {
    std::string s = "(";
    for (int64_t d : t.sizes()) s += std::to_string(d) + ", ";
    return s + ") " + c10::toString(t.scalar_type()) + " on " + t.device().str();
}
bool none(PyObject *o) { return o == nullptr || o == Py_None; }

const at::Tensor &tensor(PyObject *o, const char *name) {
    if (o == nullptr || !THPVariable_Check(o)) refuse("%s: a tensor expected", name);
    return THPVariable_Unpack(o);
}
// The tensor's CUDA device (there is no CPU fallback).
int device_of(const at::Tensor &t, const char *name) {
    if (!t.is_cuda()) refuse("%s: not a CUDA tensor (there is no CPU fallback)", name);
    return t.get_device();
}
// A tensor of `ndim` dimensions on `device`, the last one contiguous.
const at::Tensor &dense(PyObject *o, const char *name, int64_t ndim, int device, std::optional<at::ScalarType> type) {
    const at::Tensor &t = tensor(o, name);
    if (t.dim() != ndim || !t.is_cuda() || t.get_device() != device || (type && t.scalar_type() != *type))
        refuse("%s: %lld-d %s on cuda:%d expected, got %s", name, (long long)ndim, type ? c10::toString(*type) : "tensor",
               device, shape_of(t).c_str());
    if (t.stride(ndim - 1) != 1 && t.size(ndim - 1) > 1) refuse("%s: the last dimension is not contiguous", name);
    return t;
}
// Address of n contiguous values; None: NULL.
template <typename P> const P *flat(PyObject *o, const char *name, at::ScalarType type, int64_t n, int device) {
    if (none(o)) return nullptr;
    const at::Tensor &t = tensor(o, name);
    if (t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1) || t.scalar_type() != type || !t.is_cuda() ||
        t.get_device() != device)
        refuse("%s: %lld contiguous values of %s on cuda:%d expected, got %s", name, (long long)n, c10::toString(type), device,
               shape_of(t).c_str());
    return static_cast<const P *>(t.data_ptr());
}
int type_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return Q4K_TYPE_F32;
        case at::kHalf: return Q4K_TYPE_F16;
        case at::kBFloat16: return Q4K_TYPE_BF16;
        default: refuse("type %s is not float32, float16 or bfloat16", c10::toString(t));
    }
}
// Columns of n values: (ncols, n), or one column (n).
struct Columns {
    int64_t ncols, n, stride;
    void *p;
};
Columns columns(PyObject *o, const char *name, int device) {
    const bool one = tensor(o, name).dim() == 1;
    const at::Tensor &t = dense(o, name, one ? 1 : 2, device, at::kFloat);
    if (one) return {1, t.size(0), t.size(0), t.data_ptr()};
    return {t.size(0), t.size(1), t.stride(0), t.data_ptr()};
}

// The stream a call runs on (None: the device's current one, else a handle);
// outputs and scratch are allocated for it, with the tensors' device current.
struct Where {
    c10::cuda::OptionalCUDAGuard device;
    c10::cuda::OptionalCUDAStreamGuard given;
    q4k_stream_t stream;

    Where(int index, PyObject *handle) {
        if (c10::cuda::current_device() != index) device.set_index(static_cast<c10::DeviceIndex>(index));
        c10::cuda::CUDAStream s = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index));
        if (!none(handle)) {
            void *h = PyLong_AsVoidPtr(handle);
            if (PyErr_Occurred()) throw PythonError{};
            if (h != static_cast<void *>(s.stream())) {
                s = c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(h), static_cast<c10::DeviceIndex>(index));
                given.reset_stream(s);
            }
        }
        stream = reinterpret_cast<q4k_stream_t>(s.stream());
    }
};
at::Tensor fresh(const at::Tensor &like, at::IntArrayRef shape, at::ScalarType type) {
    return at::empty(shape, like.options().dtype(type).memory_format(c10::nullopt).requires_grad(c10::nullopt));
}
// `out` as given, or a new tensor; an owned reference.
PyObject *owned(PyObject *given, at::Tensor made) {
    if (!none(given)) {
        Py_INCREF(given);
        return given;
    }
    return THPVariable_Wrap(std::move(made));
}

// References dropped at the end of a scope.
struct Refs {
    PyObject *v[Q4K_MAX_TASKS] = {};
    int n = 0;
    ~Refs() {
        for (int i = 0; i < n; ++i) Py_XDECREF(v[i]);
    }
};

// ---- lora ------------------------------------------------------------------------
struct LoraCall {
    q4k_lora_task task[Q4K_MAX_TASKS];
    int n = 0, device = -1;
    int64_t ncols = 0;
};

// One task; out None: allocated by the caller's `where`. Returns an owned output.
PyObject *add_task(LoraCall &c, std::optional<Where> &where, PyObject *stream, PyObject *x, PyObject *A, PyObject *B,
                   PyObject *base, PyObject *ranks, PyObject *scales, PyObject *out) {
    if (c.n == Q4K_MAX_TASKS) refuse("more than %d tasks", Q4K_MAX_TASKS);
    const at::Tensor &xt = tensor(x, "x");
    const int dev = device_of(xt, "x");
    const Columns xc = columns(x, "x", dev);
    if (c.n == 0) {
        c.device = dev;
        c.ncols = xc.ncols;
        where.emplace(dev, stream);
    } else if (dev != c.device || xc.ncols != c.ncols) {
        refuse("the tasks' columns or devices differ");
    }
    if (c.ncols > INT_MAX) refuse("too many columns");
    const at::Tensor &a = dense(A, "A", 3, dev, std::nullopt), &b = dense(B, "B", 3, dev, a.scalar_type());
    const int64_t slots = a.size(0), rank = a.size(1), nrows = b.size(1);
    if (a.size(2) != xc.n || b.size(0) != slots || b.size(2) != rank || slots > INT_MAX || rank > INT_MAX)
        refuse("A %s and B %s do not fit x %s", shape_of(a).c_str(), shape_of(b).c_str(), shape_of(xt).c_str());
    q4k_lora_task &t = c.task[c.n];
    t = {};
    t.x = static_cast<const float *>(xc.p);
    t.A = a.data_ptr();
    t.B = b.data_ptr();
    t.ranks = flat<int32_t>(ranks, "ranks", at::kInt, slots, dev);
    t.scales = flat<float>(scales, "scales", at::kFloat, slots, dev);
    t.K = xc.n;
    t.nrows = nrows;
    t.stride_col_x = xc.stride;
    t.stride_a_slot = a.stride(0);
    t.stride_a_row = a.stride(1);
    t.stride_b_slot = b.stride(0);
    t.stride_b_row = b.stride(1);
    t.slots = static_cast<int>(slots);
    t.rank = static_cast<int>(rank);
    t.type = type_of(a.scalar_type());
    if (!none(base)) {
        const Columns bc = columns(base, "base", dev);
        if (bc.ncols != c.ncols || bc.n != nrows)
            refuse("base %s: (%lld, %lld) expected", shape_of(tensor(base, "base")).c_str(), (long long)c.ncols, (long long)nrows);
        t.base = static_cast<const float *>(bc.p);
        t.stride_col_base = bc.stride;
    }
    at::Tensor made;
    if (none(out)) {
        made = fresh(xt, {c.ncols, nrows}, at::kFloat);
        t.dst = static_cast<float *>(made.data_ptr());
        t.stride_col_dst = nrows;
    } else {
        const Columns oc = columns(out, "out", dev);
        if (oc.ncols != c.ncols || oc.n != nrows)
            refuse("out %s: (%lld, %lld) expected", shape_of(tensor(out, "out")).c_str(), (long long)c.ncols, (long long)nrows);
        t.dst = static_cast<float *>(oc.p);
        t.stride_col_dst = oc.stride;
    }
    ++c.n;
    return owned(out, std::move(made));
}

// The call itself: ids, and a workspace where the library wants one (ws None:
// scratch of this call's own, so that calls on several streams or in several
// graphs share nothing; else a Workspace: ensure(bytes) and buf, a tensor on the tasks' device).
void run_tasks(const q4k_lora_task *tasks, int n, int64_t ncols, int device, PyObject *ids, PyObject *ws, const Where &where) {
    const int32_t *idp = flat<int32_t>(ids, "ids", at::kInt, ncols, device);
    if (idp == nullptr && ncols > 0) refuse("ids: %lld device ints expected", (long long)ncols);
    const size_t need = g_lora_bytes(tasks, n, static_cast<int>(ncols));
    void *p = nullptr;
    at::Tensor scratch;
    if (need > 0) {
        if (none(ws)) {
            scratch = fresh(THPVariable_Unpack(ids), {static_cast<int64_t>(need)}, at::kByte);
            p = scratch.data_ptr();
        } else {
            PyObject *r = PyObject_CallMethod(ws, "ensure", "n", static_cast<Py_ssize_t>(need));
            if (r == nullptr) throw PythonError{};
            Py_DECREF(r);
            Refs hold;
            if ((hold.v[0] = PyObject_GetAttrString(ws, "buf")) == nullptr) throw PythonError{};
            hold.n = 1;
            const at::Tensor &buf = tensor(hold.v[0], "ws.buf");
            if (!buf.is_cuda() || buf.get_device() != device)
                refuse("ws: a workspace on cuda:%d expected, got %s", device, shape_of(buf).c_str());
            p = buf.data_ptr();
        }
    }
    check(g_lora(tasks, n, static_cast<int>(ncols), idp, p, need, where.stream));
}

// lora_add(x, A, B, ids, base, ranks, scales, out, ws, stream)
PyObject *py_lora_add(PyObject *, PyObject *const *v, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 10) refuse("lora_add: 10 arguments");
        LoraCall c;
        std::optional<Where> where;
        Refs out;
        out.v[0] = add_task(c, where, v[9], v[0], v[1], v[2], v[4], v[5], v[6], v[7]);
        out.n = 1;
        run_tasks(c.task, 1, c.ncols, c.device, v[3], v[8], *where);
        out.n = 0;
        return out.v[0];
    });
}

// Tasks from a sequence of dicts; outputs as owned references.
void add_items(LoraCall &c, std::optional<Where> &where, Refs &out, PyObject *items, PyObject *stream) {
    static PyObject *keys[7] = {};
    static const char *names[7] = {"x", "A", "B", "base", "ranks", "scales", "out"};
    for (int i = 0; i < 7; ++i)
        if (keys[i] == nullptr && (keys[i] = PyUnicode_InternFromString(names[i])) == nullptr) throw PythonError{};
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(items);
    if (n > Q4K_MAX_TASKS) refuse("more than %d tasks", Q4K_MAX_TASKS);
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject *it = PySequence_Fast_GET_ITEM(items, i), *f[7];
        if (!PyDict_Check(it)) refuse("a task is a dict");
        for (int k = 0; k < 7; ++k) {
            f[k] = PyDict_GetItemWithError(it, keys[k]);
            if (f[k] == nullptr && PyErr_Occurred()) throw PythonError{};
        }
        out.v[out.n] = add_task(c, where, stream, f[0], f[1], f[2], f[3], f[4], f[5], f[6]);
        ++out.n;
    }
}

// lora_batch(items, ids, ws, stream) -> outputs
PyObject *py_lora_batch(PyObject *, PyObject *const *v, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 4) refuse("lora_batch: 4 arguments");
        PyObject *items = PySequence_Fast(v[0], "tasks: a sequence of dicts");
        if (items == nullptr) throw PythonError{};
        LoraCall c;
        std::optional<Where> where;
        Refs out, hold;
        hold.v[hold.n++] = items;
        add_items(c, where, out, items, v[3]);
        if (c.n > 0) run_tasks(c.task, c.n, c.ncols, c.device, v[1], v[2], *where);
        PyObject *list = PyList_New(out.n);
        if (list == nullptr) throw PythonError{};
        for (int i = 0; i < out.n; ++i) PyList_SET_ITEM(list, i, out.v[i]);
        out.n = 0;
        return list;
    });
}

// lora_pack(items) -> the tasks' bytes
PyObject *py_lora_pack(PyObject *, PyObject *const *v, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 1) refuse("lora_pack: 1 argument");
        PyObject *items = PySequence_Fast(v[0], "tasks: a sequence of dicts");
        if (items == nullptr) throw PythonError{};
        LoraCall c;
        std::optional<Where> where;
        Refs out, hold;
        hold.v[hold.n++] = items;
        add_items(c, where, out, items, nullptr);
        return PyBytes_FromStringAndSize(reinterpret_cast<const char *>(c.task), c.n * sizeof(q4k_lora_task));
    });
}

// lora_run(tasks' bytes (buffer), ids, ws, stream, the tasks' columns, their device)
PyObject *py_lora_run(PyObject *, PyObject *const *v, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 6) refuse("lora_run: 6 arguments");
        const int64_t ncols = PyLong_AsLongLong(v[4]), device = PyLong_AsLongLong(v[5]);
        if (PyErr_Occurred()) throw PythonError{};
        Py_buffer buf;
        if (PyObject_GetBuffer(v[0], &buf, PyBUF_SIMPLE) != 0) throw PythonError{};
        struct Release {
            Py_buffer *b;
            ~Release() { PyBuffer_Release(b); }
        } release{&buf};
        const Py_ssize_t count = buf.len / static_cast<Py_ssize_t>(sizeof(q4k_lora_task));
        if (buf.len % static_cast<Py_ssize_t>(sizeof(q4k_lora_task)) != 0 || count > Q4K_MAX_TASKS)
            refuse("tasks: %lld bytes are not up to %d tasks", (long long)buf.len, Q4K_MAX_TASKS);
        if (count == 0) Py_RETURN_NONE;
        const int dev = device_of(tensor(v[1], "ids"), "ids");
        if (dev != device) refuse("ids: on cuda:%d, the tasks' tensors are on cuda:%lld", dev, (long long)device);
        Where where(dev, v[3]);
        run_tasks(static_cast<const q4k_lora_task *>(buf.buf), static_cast<int>(count), ncols, dev, v[1], v[2], where);
        Py_RETURN_NONE;
    });
}

// ---- rope ------------------------------------------------------------------------
// rope(x or sequence, pos, inv_freq, sections, layout, order, scale, dtype, out, stream)
PyObject *py_rope(PyObject *, PyObject *const *v, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 10) refuse("rope: 10 arguments");
        const bool single = THPVariable_Check(v[0]);
        Refs hold, made;
        PyObject *xs = nullptr, *os = nullptr;
        int count = 1;
        if (!single) {
            if ((xs = PySequence_Fast(v[0], "x: a tensor or a sequence of tensors")) == nullptr) throw PythonError{};
            hold.v[hold.n++] = xs;
            count = static_cast<int>(PySequence_Fast_GET_SIZE(xs));
            if (count < 1 || count > Q4K_MAX_ROPE_TENSORS) refuse("1 to %d tensors expected", Q4K_MAX_ROPE_TENSORS);
            if (!none(v[8])) {
                if ((os = PySequence_Fast(v[8], "out: as many tensors as x")) == nullptr) throw PythonError{};
                hold.v[hold.n++] = os;
                if (PySequence_Fast_GET_SIZE(os) != count) refuse("out: as many tensors as x expected");
            }
        }
        auto x_of = [&](int i) { return single ? v[0] : PySequence_Fast_GET_ITEM(xs, i); };
        auto out_of = [&](int i) { return single ? v[8] : os != nullptr ? PySequence_Fast_GET_ITEM(os, i) : nullptr; };
        const at::Tensor &first = tensor(x_of(0), "x");
        const int dev = device_of(first, "x");
        const at::Tensor &x0 = dense(x_of(0), "x", 3, dev, at::kFloat);
        const int64_t ncols = x0.size(0), dim = x0.size(2);
        at::ScalarType type = at::kFloat;
        if (!none(v[7])) {
            if (!THPDtype_Check(v[7])) refuse("dtype: a torch dtype expected");
            type = reinterpret_cast<THPDtype *>(v[7])->scalar_type;
        } else if (!none(out_of(0))) {
            type = tensor(out_of(0), "out").scalar_type();
        }
        const int kind = type_of(type);
        if (ncols > INT_MAX || dim > INT_MAX) refuse("x %s: too large", shape_of(x0).c_str());
        Where where(dev, v[9]);
        q4k_rope_tensor t[Q4K_MAX_ROPE_TENSORS];
        for (int i = 0; i < count; ++i) {
            const at::Tensor &x = dense(x_of(i), "x", 3, dev, at::kFloat);
            if (x.size(0) != ncols || x.size(2) != dim || x.size(1) > INT_MAX)
                refuse("x %s: (%lld, heads, %lld) expected", shape_of(x).c_str(), (long long)ncols, (long long)dim);
            at::Tensor fresh_out;
            PyObject *given = out_of(i);
            if (none(given)) fresh_out = fresh(x, x.sizes(), type);
            const at::Tensor &o = none(given) ? fresh_out : dense(given, "out", 3, dev, type);
            if (o.sizes() != x.sizes()) refuse("out %s: x's shape expected", shape_of(o).c_str());
            t[i] = {static_cast<const float *>(x.data_ptr()), o.data_ptr(), x.stride(0), x.stride(1), o.stride(0), o.stride(1),
                    static_cast<int>(x.size(1))};
            made.v[i] = owned(given, std::move(fresh_out));
            ++made.n;
        }
        int sections[Q4K_MAX_ROPE_AXES], axes;
        {
            PyObject *s = PySequence_Fast(v[3], "sections: a sequence of whole numbers");
            if (s == nullptr) throw PythonError{};
            hold.v[hold.n++] = s;
            axes = static_cast<int>(PySequence_Fast_GET_SIZE(s));
            if (axes < 1 || axes > Q4K_MAX_ROPE_AXES) refuse("1 to %d sections expected", Q4K_MAX_ROPE_AXES);
            for (int i = 0; i < axes; ++i) {
                const long v = PyLong_AsLong(PySequence_Fast_GET_ITEM(s, i));
                if (v == -1 && PyErr_Occurred()) throw PythonError{};
                if (v < 0 || v > Q4K_MAX_ROPE_DIM) refuse("sections[%d]=%ld outside 0..%d", i, v, Q4K_MAX_ROPE_DIM);
                sections[i] = static_cast<int>(v);
            }
        }
        const at::Tensor &pos = dense(v[1], "pos", 2, dev, at::kInt);
        if (pos.size(0) != axes || pos.size(1) != ncols)
            refuse("pos %s: (%d, %lld) expected", shape_of(pos).c_str(), axes, (long long)ncols);
        const int64_t half = tensor(v[2], "inv_freq").numel();
        if (half > Q4K_MAX_ROPE_DIM / 2) refuse("inv_freq: at most %d values", Q4K_MAX_ROPE_DIM / 2);
        const double *inv = flat<double>(v[2], "inv_freq", at::kDouble, half, dev);
        const int layout = static_cast<int>(PyLong_AsLong(v[4])), order = static_cast<int>(PyLong_AsLong(v[5]));
        const double scale = PyFloat_AsDouble(v[6]);
        if (PyErr_Occurred()) throw PythonError{};
        check(g_rope(t, count, static_cast<int>(ncols), static_cast<int>(dim), static_cast<int>(2 * half),
                     static_cast<const int32_t *>(pos.data_ptr()), pos.stride(0), inv, sections, axes, order, layout,
                     static_cast<float>(scale), kind, where.stream));
        if (single) {
            made.n = 0;
            return made.v[0];
        }
        PyObject *list = PyList_New(count);
        if (list == nullptr) throw PythonError{};
        for (int i = 0; i < count; ++i) PyList_SET_ITEM(list, i, made.v[i]);
        made.n = 0;
        return list;
    });
}

// ---- logits ----------------------------------------------------------------------
// logits(logits, history, history_len, penalties, bias_tokens, bias_values, bias_offsets, mask, mask_rows, out, pick,
//        stream) -> out, or (out, token, lse)
PyObject *py_logits(PyObject *, PyObject *const *v, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 12) refuse("logits: 12 arguments");
        const at::Tensor &lt = tensor(v[0], "logits");
        const int dev = device_of(lt, "logits");
        const Columns lc = columns(v[0], "logits", dev);
        if (lc.ncols > INT_MAX) refuse("too many columns");
        Where where(dev, v[11]);
        q4k_logits_args a = {};
        a.logits = static_cast<const float *>(lc.p);
        a.nvocab = lc.n;
        a.stride_col = lc.stride;
        at::Tensor made;
        if (none(v[9])) {
            made = fresh(lt, lt.sizes(), at::kFloat);
            a.dst = static_cast<float *>(made.data_ptr());
            a.stride_col_dst = lc.n;
        } else {
            const Columns oc = columns(v[9], "out", dev);
            if (oc.ncols != lc.ncols || oc.n != lc.n) refuse("out %s: logits' shape expected", shape_of(tensor(v[9], "out")).c_str());
            a.dst = static_cast<float *>(oc.p);
            a.stride_col_dst = oc.stride;
        }
        if (!none(v[1])) {
            const at::Tensor &h = dense(v[1], "history", 2, dev, at::kInt);
            if (none(v[3])) refuse("history and penalties go together");
            if (h.size(0) != lc.ncols) refuse("history %s: %lld rows expected", shape_of(h).c_str(), (long long)lc.ncols);
            const at::Tensor &p = dense(v[3], "penalties", 2, dev, at::kFloat);
            if (p.size(0) != lc.ncols || p.size(1) != 3 || !p.is_contiguous())
                refuse("penalties %s: (%lld, 3) contiguous expected", shape_of(p).c_str(), (long long)lc.ncols);
            a.history = static_cast<const int32_t *>(h.data_ptr());
            a.history_len = flat<int32_t>(v[2], "history_len", at::kInt, lc.ncols, dev);
            a.penalties = static_cast<const float *>(p.data_ptr());
            a.max_history = h.size(1);
            a.stride_history = h.stride(0);
        } else if (!none(v[2]) || !none(v[3])) {
            refuse("history and penalties go together");
        }
        if (!none(v[4])) {
            if (none(v[5]) || none(v[6])) refuse("bias_tokens, bias_values and bias_offsets go together");
            a.n_bias = tensor(v[4], "bias_tokens").numel();
            a.bias_tokens = flat<int32_t>(v[4], "bias_tokens", at::kInt, a.n_bias, dev);
            a.bias_values = flat<float>(v[5], "bias_values", at::kFloat, a.n_bias, dev);
            a.bias_offsets = flat<int32_t>(v[6], "bias_offsets", at::kInt, lc.ncols + 1, dev);
        } else if (!none(v[5]) || !none(v[6])) {
            refuse("bias_tokens, bias_values and bias_offsets go together");
        }
        if (!none(v[7])) {
            const at::Tensor &m = dense(v[7], "mask", 2, dev, std::nullopt);
            if ((m.scalar_type() != at::kInt && m.scalar_type() != at::kUInt32) || m.size(1) != (lc.n + 31) / 32 ||
                m.size(0) > INT_MAX)
                refuse("mask %s: (masks, %lld) int32 expected", shape_of(m).c_str(), (long long)((lc.n + 31) / 32));
            a.mask = static_cast<const uint32_t *>(m.data_ptr());
            a.n_masks = static_cast<int>(m.size(0));
            a.stride_mask = m.stride(0);
            a.mask_rows = flat<int32_t>(v[8], "mask_rows", at::kInt, lc.ncols, dev);
        } else if (!none(v[8])) {
            refuse("mask_rows without a mask");
        }
        const int pick = PyObject_IsTrue(v[10]);
        if (pick < 0) throw PythonError{};
        at::Tensor token, lse;
        if (pick) {
            token = fresh(lt, {lc.ncols}, at::kInt);
            lse = fresh(lt, {lc.ncols}, at::kFloat);
            a.token = static_cast<int32_t *>(token.data_ptr());
            a.lse = static_cast<float *>(lse.data_ptr());
        }
        check(g_logits(&a, static_cast<int>(lc.ncols), where.stream));
        PyObject *out = owned(v[9], std::move(made));
        if (!pick) return out;
        return Py_BuildValue("(NNN)", out, THPVariable_Wrap(std::move(token)), THPVariable_Wrap(std::move(lse)));
    });
}

// bind(error class, addresses of q4k_last_error, q4k_lora_batch, q4k_lora_workspace_bytes, q4k_rope_multi,
//      q4k_logits_process)
PyObject *py_bind(PyObject *, PyObject *const *v, Py_ssize_t n) {
    if (n != 6) {
        PyErr_SetString(PyExc_TypeError, "bind: 6 arguments");
        return nullptr;
    }
    void *f[5];
    for (int i = 0; i < 5; ++i) f[i] = PyLong_AsVoidPtr(v[i + 1]);
    if (PyErr_Occurred()) return nullptr;
    g_last_error = reinterpret_cast<decltype(g_last_error)>(f[0]);
    g_lora = reinterpret_cast<decltype(g_lora)>(f[1]);
    g_lora_bytes = reinterpret_cast<decltype(g_lora_bytes)>(f[2]);
    g_rope = reinterpret_cast<decltype(g_rope)>(f[3]);
    g_logits = reinterpret_cast<decltype(g_logits)>(f[4]);
    Py_INCREF(v[0]);
    Py_XDECREF(g_error);
    g_error = v[0];
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"bind", FAST(py_bind)},
                         {"lora_add", FAST(py_lora_add)},
                         {"lora_batch", FAST(py_lora_batch)},
                         {"lora_pack", FAST(py_lora_pack)},
                         {"lora_run", FAST(py_lora_run)},
                         {"rope", FAST(py_rope)},
                         {"logits", FAST(py_logits)},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_q4k_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__q4k_torch(void) { return PyModule_Create(&module); }
