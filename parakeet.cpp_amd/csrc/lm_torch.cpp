// lm_torch.cpp -- the calls of parakeet_lm.h for torch tensors (_lm_torch.so, used by lm.py).
//
// The same calls as lm.py makes through ctypes, with the tensors' shapes, types and strides read in C++: a decode step of
// a small model is a row of short kernels, and reading a dozen tensors from Python takes longer than the kernel runs
// (a plan of one request: 8.2 us a call through ctypes, 4.1 here, 3.2 of them on the GPU).  Each function takes all its arguments
// by position (lm.py has the public signatures) and returns the library's status.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/Functions.h>
#include <ATen/core/Tensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <cmath>
#include <limits>
#include <string>
#include <vector>

#include "parakeet_lm.h"

namespace {

struct Refused {            // an argument that the call does not take: a Python exception
    PyObject *kind;
    std::string what;
};
[[noreturn]] void value_error(std::string what) { throw Refused{PyExc_ValueError, std::move(what)}; }
[[noreturn]] void type_error(std::string what) { throw Refused{PyExc_TypeError, std::move(what)}; }

std::string shape_text(c10::IntArrayRef s) {
    std::string t = "(";
    for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + ")";
}

// One call's arguments: all tensors on one GPU, which is made current, and the stream.
struct Call {
    PyObject *const *args;
    c10::Device device{c10::kCPU};
    bool first = true;

    explicit Call(PyObject *const *a) : args(a) {}

    const at::Tensor &tensor(int i, const char *what) {
        if (!THPVariable_Check(args[i])) type_error(std::string(what) + ": not a tensor");
        const at::Tensor &t = THPVariable_Unpack(args[i]);
        if (first) {
            if (!t.is_cuda()) value_error("tensors have to be on the GPU");
            device = t.device(), first = false;
        } else if (t.device() != device) {
            value_error("arrays on " + device.str() + " and on " + t.device().str());
        }
        if (t.requires_grad() && c10::GradMode::is_enabled())
            value_error(std::string(what) + " requires a gradient, and these operators have none: call them under torch.no_grad()");
        return t;
    }
    bool none(int i) const { return args[i] == Py_None; }
    long long whole(int i) const {
        const long long v = PyLong_AsLongLong(args[i]);
        if (v == -1 && PyErr_Occurred()) throw Refused{nullptr, ""};
        return v;
    }
    int32_t whole32(int i, const char *what) const {
        const long long v = whole(i);
        if (v < std::numeric_limits<int32_t>::min() || v > std::numeric_limits<int32_t>::max()) value_error(std::string(what) + ": out of range");
        return (int32_t)v;
    }
    void *stream(int i) const {
        if (!none(i)) {
            void *given = PyLong_AsVoidPtr(args[i]);
            if (!given && PyErr_Occurred()) throw Refused{nullptr, ""};
            return given;
        }
        return (void *)c10::hip::getCurrentHIPStream(device.index()).stream();
    }
    // a contiguous array of this type and shape
    void *array(int i, const char *what, at::ScalarType type, std::initializer_list<int64_t> shape) {
        const at::Tensor &t = tensor(i, what);
        if (t.scalar_type() != type) type_error(std::string(what) + ": " + c10::toString(t.scalar_type()) + ", expected " + c10::toString(type));
        if (t.sizes() != c10::IntArrayRef(shape))
            value_error(std::string(what) + ": shape " + shape_text(t.sizes()) + ", expected " + shape_text(c10::IntArrayRef(shape)));
        if (!t.is_contiguous()) value_error(std::string(what) + ": not contiguous");
        return t.data_ptr();
    }
    int32_t *i32(int i, const char *what, std::initializer_list<int64_t> shape) { return (int32_t *)array(i, what, at::kInt, shape); }
    int32_t *i32_or(int i, const char *what, std::initializer_list<int64_t> shape) { return none(i) ? nullptr : i32(i, what, shape); }
    float *f32(int i, const char *what, std::initializer_list<int64_t> shape) { return (float *)array(i, what, at::kFloat, shape); }
    float *f32_or(int i, const char *what, std::initializer_list<int64_t> shape) { return none(i) ? nullptr : f32(i, what, shape); }

    int32_t dtype(const at::Tensor &t, const char *what) const {
        if (t.scalar_type() == at::kFloat) return PK_DTYPE_F32;
        if (t.scalar_type() == at::kHalf) return PK_DTYPE_F16;
        if (t.scalar_type() == at::kBFloat16) return PK_DTYPE_BF16;
        type_error(std::string(what) + ": " + c10::toString(t.scalar_type()) + " (f32, f16 or bf16)");
    }
    const at::Tensor &table(int i, int64_t &stride) {
        const at::Tensor &t = tensor(i, "table");
        if (t.scalar_type() != at::kInt) type_error(std::string("table: ") + c10::toString(t.scalar_type()) + " (int32)");
        if (t.dim() != 2) value_error("table: shape " + shape_text(t.sizes()) + ", expected [requests, width]");
        if (t.size(1) > 1 && t.stride(1) != 1) value_error("table: the last axis is not adjacent");
        stride = t.stride(0);
        return t;
    }
    const at::Tensor &heads(int i, const char *what) {
        const at::Tensor &t = tensor(i, what);
        if (t.dim() != 3) value_error(std::string(what) + ": shape " + shape_text(t.sizes()) + ", expected [rows, heads, head_dim]");
        if (t.stride(2) != 1) value_error(std::string(what) + ": channels are not adjacent");
        return t;
    }
    struct Cache {
        void *ptr;
        int64_t page_stride, pages, heads, dim;
    };
    Cache cache(int i, int64_t page) {
        const at::Tensor &t = tensor(i, "cache");
        if (t.scalar_type() != at::kByte) type_error(std::string("cache of ") + c10::toString(t.scalar_type()) + " (uint8)");
        if (t.dim() != 3 || page <= 0 || t.size(2) * 16 % (page * 17) || t.stride(2) != 1 || (t.size(1) > 1 && t.stride(1) != t.size(2)))
            value_error("cache of shape " + shape_text(t.sizes()) + ": expected kv4_shape(...) for pages of " + std::to_string(page) +
                        " tokens, the records of a page adjacent");
        return {t.data_ptr(), t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2), t.size(0), t.size(1), t.size(2) * 16 / (page * 17)};
    }
    Cache cache8(int i, int64_t page) {
        const at::Tensor &t = tensor(i, "cache");
        if (t.scalar_type() != at::kByte) type_error(std::string("cache of ") + c10::toString(t.scalar_type()) + " (uint8)");
        if (t.dim() != 3 || page <= 0 || t.size(2) * 2 <= page || (t.size(2) * 2 - page) % (4 * page) || t.stride(2) != 1 ||
            (t.size(1) > 1 && t.stride(1) != t.size(2)))
            value_error("cache of shape " + shape_text(t.sizes()) + ": expected kv8_shape(...) for pages of " + std::to_string(page) +
                        " tokens, the records of a page adjacent");
        return {t.data_ptr(), t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2), t.size(0), t.size(1), (t.size(2) * 2 - page) / (4 * page)};
    }
    bool flag(int i) const {
        const int v = PyObject_IsTrue(args[i]);
        if (v < 0) throw Refused{nullptr, ""};
        return v != 0;
    }
    float real(int i) const {
        const double v = PyFloat_AsDouble(args[i]);
        if (PyErr_Occurred()) throw Refused{nullptr, ""};
        return (float)v;
    }
    // rows that are normed and rotated, their results and weights
    struct Turned {
        const void *x;
        void *y;
        const float *weight;
        int64_t x_row, x_head, y_row, y_head, n, heads, dim;
        at::ScalarType type;
    };
    Turned turned(int ix, int iy, int iw, const char *what) {
        const std::string out = std::string(what) + "_out", w = std::string(what) + "_weight";
        const at::Tensor &x = heads(ix, what);
        if (none(iy)) value_error(out + ": missing");
        const at::Tensor &y = heads(iy, out.c_str());
        if (x.scalar_type() != y.scalar_type() || x.sizes() != y.sizes())
            value_error(std::string(what) + " " + shape_text(x.sizes()) + " " + c10::toString(x.scalar_type()) + ", " + out + " " + shape_text(y.sizes()) +
                        " " + c10::toString(y.scalar_type()));
        if ((x.size(1) > 1 && y.stride(1) < x.size(2)) || (x.size(0) > 1 && y.stride(0) < x.size(2))) value_error(out + ": rows overlap");
        return {x.data_ptr(), y.data_ptr(), f32_or(iw, w.c_str(), {x.size(2)}), x.stride(0), x.stride(1), y.stride(0), y.stride(1),
                x.size(0), x.size(1), x.size(2), x.scalar_type()};
    }
    // the norm's and the rotation's settings of a descriptor
    template <class Desc>
    void turn(Desc &d, int ipos, int iinv, int ieps, int iinterleaved, int64_t n) {
        d.pos = i32_or(ipos, "pos", {n});
        if (!none(iinv)) {
            const at::Tensor &t = tensor(iinv, "inv_freq");
            if (t.dim() != 1) value_error("inv_freq has one axis");
            d.inv_freq = f32(iinv, "inv_freq", {t.size(0)});
            if (t.size(0) > 4096) value_error("inv_freq: out of range");
            d.rot_dim = (int32_t)(2 * t.size(0));
        }
        d.norm = !none(ieps), d.eps = none(ieps) ? 0.0f : real(ieps), d.interleaved = flag(iinterleaved);
    }
};

int32_t narrow(int64_t v, const char *what) {
    if (v > std::numeric_limits<int32_t>::max()) value_error(std::string(what) + ": over 2^31");
    return (int32_t)v;
}

// Workspaces by kind of call, device and stream, and by capture where a graph is being captured: a graph has its own and
// zeroes it whenever it is replayed, so it may be replayed before, after and beside other graphs and eager calls.  They only
// grow, and one that was handed out is never freed: a captured graph may hold it.
constexpr int64_t kEager = -1;
struct Workspace {
    int kind, device;
    void *stream;
    int64_t capture;        // the capture's number, or kEager
    int64_t bytes;
    at::Tensor t;
};
std::vector<Workspace> &workspaces() {
    static auto *all = new std::vector<Workspace>;      // not destroyed at exit: the runtime may be gone by then
    return *all;
}

int64_t capture_of(void *stream) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    const hipError_t e = hipStreamGetCaptureInfo((hipStream_t)stream, &status, &id);
    if (e != hipSuccess) throw Refused{PyExc_RuntimeError, std::string("hipStreamGetCaptureInfo: ") + hipGetErrorString(e)};
    return status == hipStreamCaptureStatusNone ? kEager : (int64_t)(id & 0x7FFFFFFFFFFFFFFFull);
}

// Makes a stream torch's current one.
struct CurrentStream {
    c10::hip::HIPStream before;
    CurrentStream(void *stream, c10::DeviceIndex device) : before(c10::hip::getCurrentHIPStream(device)) {
        if ((void *)before.stream() != stream) c10::hip::setCurrentHIPStream(c10::hip::getStreamFromExternal((hipStream_t)stream, device));
    }
    ~CurrentStream() { c10::hip::setCurrentHIPStream(before); }
};

void workspace(Call &c, int given, int kind, void *stream, int64_t wanted, void *&ptr, int64_t &bytes) {
    if (!c.none(given)) {
        const at::Tensor &t = c.tensor(given, "workspace");
        if (t.scalar_type() != at::kByte || !t.is_contiguous()) type_error("workspace: not contiguous uint8");
        ptr = t.data_ptr(), bytes = t.numel();
        return;
    }
    ptr = nullptr, bytes = 0;
    if (wanted == 0) return;
    auto &all = workspaces();
    const int64_t capture = capture_of(stream);
    for (auto w = all.rbegin(); w != all.rend(); ++w)
        if (w->kind == kind && w->device == c.device.index() && w->stream == stream && w->capture == capture) {
            if (w->bytes < wanted) break;
            ptr = w->t.data_ptr(), bytes = w->bytes;
            return;
        }
    int64_t size = 1 << 20;
    while (size < wanted) size *= 2;
    const CurrentStream here(stream, c.device.index());      // zeroed in the order of the calls that use it
    at::Tensor t = at::zeros({size}, at::TensorOptions().dtype(at::kByte).device(c.device));
    ptr = t.data_ptr(), bytes = size;
    all.push_back({kind, (int)c.device.index(), stream, capture, size, std::move(t)});
}

// f(call) -> status, with its C++ exceptions turned into Python's
template <class F>
PyObject *guarded(PyObject *const *args, Py_ssize_t n, Py_ssize_t expected, F f) {
    if (n != expected) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, expected %zd", n, expected);
        return nullptr;
    }
    try {
        Call c(args);
        return PyLong_FromLong(f(c));
    } catch (const Refused &r) {
        if (r.kind) PyErr_SetString(r.kind, r.what.c_str());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

PyObject *kv_plan(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded(args, n, 13, [](Call &c) {
        pk_kv_plan_desc d{};
        const at::Tensor &table = c.table(2, d.table_stride);
        const int64_t B = table.size(0);
        const at::Tensor &ring = c.tensor(3, "ring"), &slots = c.tensor(10, "slots");
        if (ring.dim() != 1 || slots.dim() != 1) value_error("ring and slots have one axis");
        d.old_len = c.i32(0, "old_len", {B}), d.new_len = c.i32(1, "new_len", {B});
        d.table = (int32_t *)table.data_ptr(), d.ring = c.i32(3, "ring", {ring.size(0)}), d.state = c.i32(4, "state", {2});
        d.page = c.whole32(5, "page");
        d.state_out = c.i32(6, "state_out", {2}), d.lens = c.i32(7, "lens", {B}), d.ok = c.i32(8, "ok", {B});
        d.first = c.i32(9, "first", {B + 1}), d.slots = c.i32(10, "slots", {slots.size(0)});
        d.pos = c.i32_or(11, "pos", {slots.size(0)});
        d.requests = narrow(B, "requests"), d.width = narrow(table.size(1), "table"), d.n_pages = narrow(ring.size(0), "ring");
        d.n_tokens = narrow(slots.size(0), "slots");
        const c10::DeviceGuard guard(c.device);
        return pk_kv_plan(&d, c.stream(12));
    });
}

template <int (*Entry)(const pk_kv4_rows_desc *, void *), Call::Cache (Call::*Layout)(int, int64_t) = &Call::cache>
int rows(Call &c, int ik, int iv, int islots, int icache) {
    pk_kv4_rows_desc d{};
    d.page = c.whole32(4, "page");
    const at::Tensor &k = c.heads(ik, "k"), &v = c.heads(iv, "v");
    const auto cache = (c.*Layout)(icache, d.page);
    if (k.scalar_type() != v.scalar_type() || k.sizes() != v.sizes())
        value_error("k " + shape_text(k.sizes()) + " " + c10::toString(k.scalar_type()) + ", v " + shape_text(v.sizes()) + " " + c10::toString(v.scalar_type()));
    if (k.size(1) != cache.heads || k.size(2) != cache.dim)
        value_error("rows of " + std::to_string(k.size(1)) + " heads of " + std::to_string(k.size(2)) + ", a cache of " +
                    std::to_string(cache.heads) + " heads of " + std::to_string(cache.dim));
    d.dtype = c.dtype(k, "k");
    d.k = k.data_ptr(), d.v = v.data_ptr(), d.slots = c.i32(islots, "slots", {k.size(0)}), d.cache = cache.ptr;
    d.k_row = k.stride(0), d.k_head = k.stride(1), d.v_row = v.stride(0), d.v_head = v.stride(1), d.page_stride = cache.page_stride;
    d.n_rows = narrow(k.size(0), "rows"), d.heads = narrow(cache.heads, "heads"), d.head_dim = narrow(cache.dim, "head_dim");
    d.n_pages = narrow(cache.pages, "pages");
    const c10::DeviceGuard guard(c.device);
    return Entry(&d, c.stream(5));
}
PyObject *kv4_store(PyObject *, PyObject *const *args, Py_ssize_t n) {      // k, v, slots, cache, page, stream
    return guarded(args, n, 6, [](Call &c) { return rows<pk_kv4_store>(c, 0, 1, 2, 3); });
}
PyObject *kv4_load(PyObject *, PyObject *const *args, Py_ssize_t n) {       // cache, slots, k, v, page, stream
    return guarded(args, n, 6, [](Call &c) { return rows<pk_kv4_load>(c, 2, 3, 1, 0); });
}

template <int (*Entry)(const pk_kv4_attend_desc *, void *), int (*Wanted)(const pk_kv4_attend_desc *, int64_t *), Call::Cache (Call::*Layout)(int, int64_t)>
PyObject *attend(PyObject *const *args, Py_ssize_t n, int kind) {
    return guarded(args, n, 14, [kind](Call &c) {
        pk_kv4_attend_desc d{};
        const at::Tensor &q = c.heads(0, "q"), &out = c.heads(4, "out");
        d.page = c.whole32(5, "page");
        const auto cache = (c.*Layout)(1, d.page);
        const at::Tensor &table = c.table(2, d.table_stride);
        if (out.scalar_type() != q.scalar_type() || out.sizes() != q.sizes())
            value_error("q " + shape_text(q.sizes()) + ", out " + shape_text(out.sizes()) + " " + c10::toString(out.scalar_type()));
        const int64_t rows = q.size(0), heads = q.size(1), dim = q.size(2), B = table.size(0), width = table.size(1);
        if (dim != cache.dim || cache.heads == 0 || heads % cache.heads)
            value_error(std::to_string(heads) + " query heads of " + std::to_string(dim) + ", a cache of " + std::to_string(cache.heads) +
                        " heads of " + std::to_string(cache.dim));
        if ((heads > 1 && out.stride(1) < dim) || (rows > 1 && out.stride(0) < dim)) value_error("out: rows overlap");
        d.q = q.data_ptr(), d.out = out.data_ptr(), d.cache = cache.ptr, d.table = (const int32_t *)table.data_ptr();
        d.lens = c.i32(3, "lens", {B}), d.first = c.i32_or(6, "first", {B + 1});
        d.max_new = c.whole32(7, "max_new");
        constexpr int64_t kMost = std::numeric_limits<int32_t>::max() - 4096;
        d.max_len = c.none(8) ? (int32_t)std::min<int64_t>(width * d.page, kMost) : c.whole32(8, "max_len");
        if (c.none(9)) {
            d.scale = 1.0f / std::sqrt((float)dim);
        } else {
            d.scale = (float)PyFloat_AsDouble(c.args[9]);
            if (PyErr_Occurred()) throw Refused{nullptr, ""};
        }
        d.window = c.whole32(10, "window"), d.lse = c.f32_or(11, "lse", {rows, heads});
        d.q_row = q.stride(0), d.q_head = q.stride(1), d.out_row = out.stride(0), d.out_head = out.stride(1);
        d.page_stride = cache.page_stride;
        d.n_rows = narrow(rows, "rows"), d.requests = narrow(B, "requests"), d.heads = narrow(heads, "heads");
        d.kv_heads = narrow(cache.heads, "heads"), d.head_dim = narrow(dim, "head_dim"), d.dtype = c.dtype(q, "q");
        d.n_pages = narrow(cache.pages, "pages"), d.width = narrow(width, "table");
        const c10::DeviceGuard guard(c.device);
        void *stream = c.stream(13);
        int64_t wanted = 0;
        if (const int rc = Wanted(&d, &wanted)) return rc;
        workspace(c, 12, kind, stream, wanted, d.workspace, d.workspace_bytes);
        return Entry(&d, stream);
    });
}
PyObject *kv4_attend(PyObject *, PyObject *const *args, Py_ssize_t n) { return attend<pk_kv4_attend, pk_kv4_attend_workspace, &Call::cache>(args, n, 0); }
PyObject *kv8_attend(PyObject *, PyObject *const *args, Py_ssize_t n) { return attend<pk_kv8_attend, pk_kv8_attend_workspace, &Call::cache8>(args, n, 2); }

PyObject *sample(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded(args, n, 11, [](Call &c) {
        pk_sample_desc d{};
        const at::Tensor &x = c.tensor(0, "logits");
        if (x.dim() != 2) value_error("logits: shape " + shape_text(x.sizes()) + ", expected [rows, vocab]");
        if (x.size(1) > 1 && x.stride(1) != 1) value_error("logits: the last axis is not adjacent");
        const int64_t B = x.size(0);
        d.logits = x.data_ptr(), d.logits_row = x.stride(0), d.dtype = c.dtype(x, "logits");
        d.rows = narrow(B, "rows"), d.vocab = narrow(x.size(1), "vocab");
        d.u = c.f32(1, "u", {B}), d.token = c.i32(2, "token", {B});
        d.temperature = c.f32_or(3, "temperature", {B}), d.top_k = c.i32_or(4, "top_k", {B}), d.top_p = c.f32_or(5, "top_p", {B});
        d.min_p = c.f32_or(6, "min_p", {B}), d.prob = c.f32_or(7, "prob", {B}), d.kept = c.i32_or(8, "kept", {B});
        const c10::DeviceGuard guard(c.device);
        void *stream = c.stream(10);
        int64_t wanted = 0;
        if (const int rc = pk_sample_workspace(&d, &wanted)) return rc;
        workspace(c, 9, 1, stream, wanted, d.workspace, d.workspace_bytes);
        return pk_sample(&d, stream);
    });
}

PyObject *kv8_load(PyObject *, PyObject *const *args, Py_ssize_t n) {       // cache, slots, k, v, page, stream
    return guarded(args, n, 6, [](Call &c) { return rows<pk_kv8_load, &Call::cache8>(c, 2, 3, 1, 0); });
}

PyObject *qk_rope(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded(args, n, 11, [](Call &c) {
        pk_qk_rope_desc d{};
        const auto q = c.turned(0, 1, 7, "q");
        d.q = q.x, d.q_out = q.y, d.q_weight = q.weight, d.q_row = q.x_row, d.q_head = q.x_head, d.q_out_row = q.y_row, d.q_out_head = q.y_head;
        d.dtype = c.dtype(c.tensor(0, "q"), "q");
        if (!c.none(4)) {
            const auto k = c.turned(4, 5, 8, "k");
            if (k.type != q.type || k.n != q.n || k.dim != q.dim) value_error("k: rows of another number, size or type than q's");
            d.k = k.x, d.k_out = k.y, d.k_weight = k.weight, d.k_row = k.x_row, d.k_head = k.x_head, d.k_out_row = k.y_row, d.k_out_head = k.y_head;
            d.kv_heads = narrow(k.heads, "heads");
        }
        c.turn(d, 2, 3, 6, 9, q.n);
        d.n_rows = narrow(q.n, "rows"), d.heads = narrow(q.heads, "heads"), d.head_dim = narrow(q.dim, "head_dim");
        const c10::DeviceGuard guard(c.device);
        return pk_qk_rope(&d, c.stream(10));
    });
}

PyObject *kv8_append(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded(args, n, 14, [](Call &c) {
        pk_kv8_append_desc d{};
        d.page = c.whole32(4, "page");
        const at::Tensor &k = c.heads(0, "k"), &v = c.heads(1, "v");
        const auto cache = c.cache8(3, d.page);
        if (k.scalar_type() != v.scalar_type() || k.sizes() != v.sizes())
            value_error("k " + shape_text(k.sizes()) + " " + c10::toString(k.scalar_type()) + ", v " + shape_text(v.sizes()) + " " + c10::toString(v.scalar_type()));
        if (k.size(1) != cache.heads || k.size(2) != cache.dim)
            value_error("rows of " + std::to_string(k.size(1)) + " heads of " + std::to_string(k.size(2)) + ", a cache of " +
                        std::to_string(cache.heads) + " heads of " + std::to_string(cache.dim));
        d.dtype = c.dtype(k, "k");
        d.k = k.data_ptr(), d.v = v.data_ptr(), d.slots = c.i32(2, "slots", {k.size(0)}), d.cache = cache.ptr;
        d.k_row = k.stride(0), d.k_head = k.stride(1), d.v_row = v.stride(0), d.v_head = v.stride(1), d.page_stride = cache.page_stride;
        d.k_weight = c.f32_or(8, "k_weight", {k.size(2)});
        if (!c.none(9)) {
            const auto q = c.turned(9, 10, 11, "q");
            if (q.type != k.scalar_type() || q.n != k.size(0) || q.dim != k.size(2)) value_error("q: rows of another number, size or type than k's");
            d.q = q.x, d.q_out = q.y, d.q_weight = q.weight, d.q_row = q.x_row, d.q_head = q.x_head, d.q_out_row = q.y_row, d.q_out_head = q.y_head;
            d.heads = narrow(q.heads, "heads");
        }
        c.turn(d, 5, 6, 7, 12, k.size(0));
        d.n_rows = narrow(k.size(0), "rows"), d.kv_heads = narrow(cache.heads, "heads"), d.head_dim = narrow(cache.dim, "head_dim");
        d.n_pages = narrow(cache.pages, "pages");
        const c10::DeviceGuard guard(c.device);
        return pk_kv8_append(&d, c.stream(13));
    });
}

PyObject *verify(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded(args, n, 16, [](Call &c) {
        pk_verify_desc d{};
        const at::Tensor &x = c.tensor(0, "logits"), &first = c.tensor(2, "first");
        auto rows2 = [](const at::Tensor &t, const char *what) {
            if (t.dim() != 2) value_error(std::string(what) + ": shape " + shape_text(t.sizes()) + ", expected [rows, vocab]");
            if (t.size(1) > 1 && t.stride(1) != 1) value_error(std::string(what) + ": the last axis is not adjacent");
        };
        rows2(x, "logits");
        if (first.dim() != 1 || first.size(0) < 1) value_error("first: shape " + shape_text(first.sizes()) + ", expected [requests + 1]");
        const int64_t N = x.size(0), B = first.size(0) - 1;
        d.logits = x.data_ptr(), d.logits_row = x.stride(0), d.dtype = c.dtype(x, "logits");
        if (!c.none(8)) {
            const at::Tensor &y = c.tensor(8, "draft");
            rows2(y, "draft");
            if (y.scalar_type() != x.scalar_type() || y.sizes() != x.sizes())
                value_error("logits " + shape_text(x.sizes()) + ", draft " + shape_text(y.sizes()) + " " + c10::toString(y.scalar_type()));
            d.draft = y.data_ptr(), d.draft_row = y.stride(0);
        }
        d.tokens = c.i32(1, "tokens", {N}), d.first = c.i32(2, "first", {B + 1}), d.u = c.f32(3, "u", {N}), d.u_draw = c.f32(4, "u_draw", {B});
        d.out = c.i32(5, "out", {N}), d.accepted = c.i32(6, "accepted", {B});
        d.n_rows = narrow(N, "rows"), d.requests = narrow(B, "requests"), d.vocab = narrow(x.size(1), "vocab");
        d.max_new = c.none(7) ? d.n_rows : c.whole32(7, "max_new");
        d.temperature = c.f32_or(9, "temperature", {B}), d.draft_temperature = c.f32_or(10, "draft_temperature", {B});
        d.lens = c.i32_or(11, "lens", {B}), d.lens_out = c.i32_or(12, "lens_out", {B}), d.prob = c.f32_or(13, "prob", {N});
        const c10::DeviceGuard guard(c.device);
        void *stream = c.stream(15);
        int64_t wanted = 0;
        if (const int rc = pk_verify_workspace(&d, &wanted)) return rc;
        workspace(c, 14, 3, stream, wanted, d.workspace, d.workspace_bytes);
        return pk_verify(&d, stream);
    });
}

PyMethodDef methods[] = {{"kv_plan", (PyCFunction)(void (*)(void))kv_plan, METH_FASTCALL, nullptr},
                         {"kv4_store", (PyCFunction)(void (*)(void))kv4_store, METH_FASTCALL, nullptr},
                         {"kv4_load", (PyCFunction)(void (*)(void))kv4_load, METH_FASTCALL, nullptr},
                         {"kv4_attend", (PyCFunction)(void (*)(void))kv4_attend, METH_FASTCALL, nullptr},
                         {"sample", (PyCFunction)(void (*)(void))sample, METH_FASTCALL, nullptr},
                         {"qk_rope", (PyCFunction)(void (*)(void))qk_rope, METH_FASTCALL, nullptr},
                         {"kv8_append", (PyCFunction)(void (*)(void))kv8_append, METH_FASTCALL, nullptr},
                         {"kv8_load", (PyCFunction)(void (*)(void))kv8_load, METH_FASTCALL, nullptr},
                         {"kv8_attend", (PyCFunction)(void (*)(void))kv8_attend, METH_FASTCALL, nullptr},
                         {"verify", (PyCFunction)(void (*)(void))verify, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module{PyModuleDef_HEAD_INIT, "_lm_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__lm_torch() { return PyModule_Create(&module); }
