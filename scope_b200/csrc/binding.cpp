// CPython binding of the paged cache's entries: checks a call's tensors, allocates its outputs on the current stream's
// device and calls the C ABI.
//
// A step of a server makes one of these calls per layer, each of a few microseconds on the device, so what the host
// spends on a call counts as much as the kernel: reading some thirty tensor attributes through Python and converting
// twenty arguments with ctypes took 15 to 20 us a call, this takes 5 to 8.  The functions take positional arguments
// only; scope_b200/paged.py has their signatures and documentation.  The C ABI's functions are handed over by address
// (setup), so this module serves whichever build of the library the package loaded.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <string>

#include "scope_b200.h"

namespace {

decltype(&ws_last_error) p_last_error;
decltype(&ws_paged_slots) p_paged_slots;
decltype(&ws_paged_release) p_paged_release;
decltype(&ws_rope_append) p_rope_append;
decltype(&ws_paged_decode) p_paged_decode;
size_t g_slots_ws, g_decode_ws;   // workspace sizes (they do not depend on the call)
PyObject *g_error, *g_pool_get, *g_pool_bufs, *g_step;   // ScopeError, workspaces.get, its dict, PagedStep

struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};
struct PythonError {};   // a Python exception is set

[[noreturn]] void refuse(const char* what, const std::string& why) { throw Refused(std::string(what) + ": " + why); }

bool is_tensor(PyObject* o) { return THPVariable_Check(o); }
const at::Tensor& tensor(const char* what, const char* name, PyObject* o) {
    if (!is_tensor(o)) refuse(what, std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}
int64_t integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw PythonError();
    return v;
}

bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PythonError();
    return v;
}

bool unit(const at::Tensor& t, int d) { return t.size(d) <= 1 || t.stride(d) == 1; }
std::string on(const at::Device& dev) { return dev.str(); }

int half_of(at::ScalarType t) {
    return t == at::kBFloat16 ? WS_DTYPE_BF16 : t == at::kHalf ? WS_DTYPE_F16 : -1;
}

// A contiguous tensor of this type and number of dimensions on `dev`.
void want(const char* what, const char* name, const at::Tensor& t, at::ScalarType type, int dim, const at::Device& dev) {
    if (t.scalar_type() != type || t.dim() != dim || t.device() != dev || !t.is_contiguous())
        refuse(what, std::string(name) + " must be a contiguous " + c10::toString(type) + " tensor of " + std::to_string(dim) +
                         " dimension(s) on " + on(dev));
}
void want_table(const char* what, const at::Tensor& t, int64_t B, const at::Device& dev) {
    if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) != B || (t.numel() > 1 && !unit(t, 1)) || t.device() != dev)
        refuse(what, "page_table must be int32 [" + std::to_string(B) + ", pages] on " + on(dev) +
                         " with unit stride on the pages");
}
void want_rows(const char* what, const char* name, const at::Tensor& t, at::ScalarType type, int64_t N, const at::Device& dev) {
    if (t.scalar_type() != type || t.dim() != 3 || t.device() != dev || t.size(0) != N || !unit(t, 2))
        refuse(what, std::string(name) + " must be " + c10::toString(type) + " [" + std::to_string(N) + ", heads, D] on " +
                         on(dev) + " with unit stride on the head dim");
}
// A new contiguous tensor on the current stream's allocator, without the dispatcher's round (0.5 us a tensor).
at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const at::Device& dev) {
    return at::detail::empty_cuda(shape, type, dev, std::nullopt);
}
// `given` when it is a tensor of this shape and type, else a new one.
at::Tensor output(const char* what, const char* name, PyObject* given, at::IntArrayRef shape, at::ScalarType type,
                  const at::Device& dev) {
    if (given == Py_None) return fresh(shape, type, dev);
    const at::Tensor& t = tensor(what, name, given);
    if (t.scalar_type() != type || t.sizes() != shape || !t.is_contiguous() || t.device() != dev)
        refuse(what, std::string(name) + " must be a contiguous " + c10::toString(type) + " tensor of the result's shape on " + on(dev));
    return t;
}

// A given output may be the input that it replaces (`same`), whole, and shares no memory with the others: the kernels read
// those while they write it.
void want_apart(const at::Tensor& out, const at::Tensor& same, std::initializer_list<const at::Tensor*> others) {
    at::assert_no_internal_overlap(out);
    at::assert_no_partial_overlap(out, same);
    for (const at::Tensor* t : others)
        if (t->defined()) at::assert_no_overlap(out, *t);
}

// The workspace of this device and stream, from the package's pool, which never frees one: a captured launch keeps the
// address.
struct Workspace {
    void* ptr;
    size_t bytes;
};
Workspace workspace(size_t bytes, const at::Device& dev, void* stream) {
    PyObject* key = Py_BuildValue("(iK)", (int)dev.index(), (unsigned long long)(uintptr_t)stream);
    if (!key) throw PythonError();
    PyObject* buf = PyDict_GetItem(g_pool_bufs, key);   // borrowed
    Py_DECREF(key);
    if (buf && (size_t)THPVariable_Unpack(buf).numel() >= bytes) {
        const at::Tensor& t = THPVariable_Unpack(buf);
        return {t.data_ptr(), (size_t)t.numel()};
    }
    PyObject* d = THPDevice_New(dev);
    buf = d ? PyObject_CallFunction(g_pool_get, "nO", (Py_ssize_t)bytes, d) : nullptr;
    Py_XDECREF(d);
    if (!buf) throw PythonError();
    const at::Tensor t = THPVariable_Unpack(buf);
    Py_DECREF(buf);   // the pool keeps it
    return {t.data_ptr(), (size_t)t.numel()};
}

void check(int rc, const char* what) {
    if (rc == WS_OK) return;
    PyErr_Format(g_error, "%s failed (status %d): %s", what, rc, p_last_error());
    throw PythonError();
}

template <typename T>
T* data(const at::Tensor& t) {
    return static_cast<T*>(t.data_ptr());
}

// Runs a call: C++ exceptions become Python ones, and none leaves the entry.
template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want_n, F&& f) {
    if (n != want_n) {
        PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
        return nullptr;
    }
    try {
        return f();
    } catch (const PythonError&) {
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// ---- pages and slots

struct Books {
    at::Device dev{at::kCPU};
    int64_t B = 0;
};
Books bookkeeping(const char* what, const at::Tensor& lens, const at::Tensor& other, const char* name, at::ScalarType type,
                  const at::Tensor& table, const at::Tensor& free_pages, const at::Tensor& ring) {
    if (!lens.is_cuda()) refuse(what, "CUDA tensors required (there is no CPU path)");
    const Books b{lens.device(), lens.numel()};
    want(what, "seq_lens", lens, at::kInt, 1, b.dev);
    want(what, name, other, type, 1, b.dev);
    want_table(what, table, b.B, b.dev);
    want(what, "free_pages", free_pages, at::kInt, 1, b.dev);
    want(what, "ring", ring, at::kInt, 1, b.dev);
    if (other.numel() != b.B || ring.numel() != 3)
        refuse(what, std::string(name) + " must hold one entry per request, and ring three");
    if (b.B > INT32_MAX || table.size(1) > INT32_MAX || free_pages.numel() > INT32_MAX) refuse(what, "bad shape");
    return b;
}

// seq_lens, new_lens, page_table, free_pages, ring, page_size, n_tokens, seq_lens_out, ring_out
PyObject* paged_slots(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 9, [&]() -> PyObject* {
        const char* what = "paged_slots";
        const at::Tensor &lens = tensor(what, "seq_lens", a[0]), &added = tensor(what, "new_lens", a[1]),
                         &table = tensor(what, "page_table", a[2]), &pages = tensor(what, "free_pages", a[3]),
                         &ring = tensor(what, "ring", a[4]);
        const Books b = bookkeeping(what, lens, added, "new_lens", at::kInt, table, pages, ring);
        const int64_t page_size = integer(a[5]), N = integer(a[6]);
        if (page_size < 1 || page_size > INT32_MAX || N < 0) refuse(what, "bad shape");
        const c10::cuda::OptionalCUDAGuard guard(b.dev);
        const at::Tensor lens_out = output(what, "seq_lens_out", a[7], {b.B}, at::kInt, b.dev);
        const at::Tensor ring_out = output(what, "ring_out", a[8], {3}, at::kInt, b.dev);
        if (a[7] != Py_None) want_apart(lens_out, lens, {&added, &table, &pages, &ring, &ring_out});
        if (a[8] != Py_None) want_apart(ring_out, ring, {&lens, &added, &table, &pages});
        const at::Tensor slots = fresh({N}, at::kLong, b.dev), positions = fresh({N}, at::kInt, b.dev);
        const at::Tensor cu = fresh({b.B + 1}, at::kInt, b.dev);
        void* stream = c10::cuda::getCurrentCUDAStream(b.dev.index()).stream();
        const Workspace ws = workspace(g_slots_ws, b.dev, stream);
        check(p_paged_slots(data<int32_t>(lens), data<int32_t>(added), (int)b.B, data<int32_t>(table), table.stride(0),
                            (int)table.size(1), data<int32_t>(pages), (int)pages.numel(), data<int32_t>(ring), (int)page_size,
                            N, data<int64_t>(slots), data<int32_t>(positions), data<int32_t>(cu), data<int32_t>(lens_out),
                            data<int32_t>(ring_out), ws.ptr, ws.bytes, stream),
              "ws_paged_slots");
        PyObject* out = PyTuple_New(5);
        if (!out) return nullptr;
        PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(slots));
        PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(positions));
        PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(cu));
        PyTuple_SET_ITEM(out, 3, THPVariable_Wrap(lens_out));
        PyTuple_SET_ITEM(out, 4, THPVariable_Wrap(ring_out));
        PyObject* step = PyObject_CallObject(g_step, out);
        Py_DECREF(out);
        return step;
    });
}

// seq_lens, done, page_table, free_pages, ring, page_size, seq_lens_out, ring_out
PyObject* paged_release(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&]() -> PyObject* {
        const char* what = "paged_release";
        const at::Tensor &lens = tensor(what, "seq_lens", a[0]), &done = tensor(what, "done", a[1]),
                         &table = tensor(what, "page_table", a[2]), &pages = tensor(what, "free_pages", a[3]),
                         &ring = tensor(what, "ring", a[4]);
        const Books b = bookkeeping(what, lens, done, "done", at::kBool, table, pages, ring);
        const int64_t page_size = integer(a[5]);
        if (page_size < 1 || page_size > INT32_MAX) refuse(what, "bad shape");
        const c10::cuda::OptionalCUDAGuard guard(b.dev);
        const at::Tensor lens_out = output(what, "seq_lens_out", a[6], {b.B}, at::kInt, b.dev);
        const at::Tensor ring_out = output(what, "ring_out", a[7], {3}, at::kInt, b.dev);
        if (a[6] != Py_None) want_apart(lens_out, lens, {&done, &table, &pages, &ring, &ring_out});
        if (a[7] != Py_None) want_apart(ring_out, ring, {&lens, &done, &table, &pages});
        void* stream = c10::cuda::getCurrentCUDAStream(b.dev.index()).stream();
        const Workspace ws = workspace(g_slots_ws, b.dev, stream);
        check(p_paged_release(data<int32_t>(lens), static_cast<uint8_t*>(done.data_ptr()), (int)b.B, data<int32_t>(table),
                              table.stride(0), (int)table.size(1), data<int32_t>(pages), (int)pages.numel(),
                              data<int32_t>(ring), (int)page_size, data<int32_t>(lens_out), data<int32_t>(ring_out), ws.ptr,
                              ws.bytes, stream),
              "ws_paged_release");
        PyObject* out = PyTuple_New(2);
        if (!out) return nullptr;
        PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(lens_out));
        PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(ring_out));
        return out;
    });
}

// ---- rotary positions.  axis_map: None (one axis) or the 32 bytes of rope_axis_map; axes: their number.
ws_rope rope_of(const char* what, PyObject* positions, PyObject* cos_sin, int64_t N, const at::Device& dev, PyObject* axis_map,
                PyObject* axes, PyObject* pairs, bool inverse) {
    const at::Tensor &pos = tensor(what, "positions", positions), &table = tensor(what, "cos_sin", cos_sin);
    if (table.scalar_type() != at::kFloat || table.dim() != 2 || !table.is_contiguous() || table.device() != dev)
        refuse(what, "cos_sin must be contiguous fp32 [max_pos, rope_dim] on " + on(dev));
    ws_rope r;
    memset(&r, 0, sizeof(r));
    const char* style = PyUnicode_Check(pairs) ? PyUnicode_AsUTF8(pairs) : nullptr;
    if (!style || (strcmp(style, "half") && strcmp(style, "adjacent"))) refuse(what, "pairs must be 'half' or 'adjacent'");
    r.adjacent = style[0] == 'a';
    r.n_axes = axis_map == Py_None ? 1 : (int)integer(axes);
    const bool i64 = pos.scalar_type() == at::kLong;
    const bool rows = pos.dim() == 2 && pos.size(0) == r.n_axes && pos.size(1) == N;
    if ((!i64 && pos.scalar_type() != at::kInt) || pos.device() != dev ||
        !(rows || (r.n_axes == 1 && pos.dim() == 1 && pos.size(0) == N)) || !unit(pos, pos.dim() - 1))
        refuse(what, "positions must be int32 or int64 [" + std::to_string(N) + "], or [" + std::to_string(r.n_axes) + ", " +
                         std::to_string(N) + "], on " + on(dev) + ", unit stride");
    if (axis_map != Py_None) {
        if (!PyBytes_Check(axis_map) || PyBytes_GET_SIZE(axis_map) != sizeof(r.axis_map)) refuse(what, "bad axis map");
        memcpy(r.axis_map, PyBytes_AS_STRING(axis_map), sizeof(r.axis_map));
    }
    r.positions = pos.data_ptr();
    r.cos_sin = data<float>(table);
    r.axis_stride = rows ? pos.stride(0) : 0;
    r.max_pos = table.size(0);
    r.positions_i64 = i64;
    r.rope_dim = (int)std::min<int64_t>(table.size(1), INT32_MAX);
    r.inverse = inverse;
    return r;
}

// x, positions, cos_sin, axis_map, axes, pairs, inverse, out
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&]() -> PyObject* {
        const char* what = "rope";
        const at::Tensor& x = tensor(what, "x", a[0]);
        if (!x.is_cuda()) refuse(what, "CUDA tensors required (there is no CPU path)");
        const at::Device dev = x.device();
        const int type = half_of(x.scalar_type());
        if (type < 0) refuse(what, "x must be bf16 or fp16");
        if (x.dim() != 3) refuse(what, "x must be [N, heads, D]");
        const int64_t N = x.size(0);
        want_rows(what, "x", x, x.scalar_type(), N, dev);
        if (x.size(1) > INT32_MAX || x.size(2) > INT32_MAX) refuse(what, "bad shape");
        const ws_rope r = rope_of(what, a[1], a[2], N, dev, a[3], a[4], a[5], truth(a[6]));
        const c10::cuda::OptionalCUDAGuard guard(dev);
        at::Tensor out;
        if (a[7] == Py_None) {
            out = fresh(x.sizes(), x.scalar_type(), dev);
        } else {
            out = tensor(what, "out", a[7]);
            want_rows(what, "out", out, x.scalar_type(), N, dev);
            if (out.sizes() != x.sizes()) refuse(what, "out must have x's shape");
            want_apart(out, x, {});
        }
        void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
        check(p_rope_append(&r, x.data_ptr(), x.stride(0), x.stride(1), (int)x.size(1), (int)x.size(2), out.data_ptr(),
                            out.stride(0), out.stride(1), nullptr, 0, 0, nullptr, 0, 0, type, N, nullptr, nullptr, stream),
              "ws_rope_append");
        return THPVariable_Wrap(out);
    });
}

// ---- the pool
ws_paged_kv pool_of(const char* what, PyObject* k_pages, PyObject* v_pages, PyObject* k_scales, PyObject* v_scales,
                    const at::Device& dev) {
    const at::Tensor &k = tensor(what, "k_pages", k_pages), &v = tensor(what, "v_pages", v_pages);
    const at::ScalarType type = k.scalar_type();
    const bool i8 = type == at::kChar;
    if (!i8 && half_of(type) < 0) refuse(what, "the pool must be bf16, fp16 or int8");
    if (k.dim() != 4 || v.dim() != 4 || k.size(0) != v.size(0) || k.size(1) != v.size(1) || k.size(2) != v.size(2) ||
        v.scalar_type() != type || k.device() != dev || v.device() != dev)
        refuse(what, "k_pages, v_pages must be [n_pages, page_size, Hkv, D] of one type on " + on(dev));
    if (k.stride(3) != 1 || v.stride(3) != 1) refuse(what, "unit stride on the head dim required");
    ws_paged_kv p;
    memset(&p, 0, sizeof(p));
    for (int d = 1; d < 4; ++d)
        if (k.size(d) > INT32_MAX || v.size(d) > INT32_MAX) refuse(what, "bad pool shape");
    if (i8) {
        if (k_scales == Py_None || v_scales == Py_None) refuse(what, "an int8 pool needs k_scales and v_scales");
        const at::Tensor &ks = tensor(what, "k_scales", k_scales), &vs = tensor(what, "v_scales", v_scales);
        for (const at::Tensor* s : {&ks, &vs})
            if (s->scalar_type() != at::kFloat || s->dim() != 3 || s->size(0) != k.size(0) || s->size(1) != k.size(1) ||
                s->size(2) != k.size(2) || s->device() != dev)
                refuse(what, "scales must be fp32 [n_pages, page_size, Hkv] on " + on(dev));
        p.k_scales = data<float>(ks), p.v_scales = data<float>(vs);
        p.ks_stride_page = ks.stride(0), p.ks_stride_tok = ks.stride(1), p.ks_stride_head = ks.stride(2);
        p.vs_stride_page = vs.stride(0), p.vs_stride_tok = vs.stride(1), p.vs_stride_head = vs.stride(2);
    } else if (k_scales != Py_None || v_scales != Py_None) {
        refuse(what, "scales belong to an int8 pool");
    }
    p.k = k.data_ptr(), p.v = v.data_ptr();
    p.n_pages = k.size(0);
    p.k_stride_page = k.stride(0), p.k_stride_tok = k.stride(1), p.k_stride_head = k.stride(2);
    p.v_stride_page = v.stride(0), p.v_stride_tok = v.stride(1), p.v_stride_head = v.stride(2);
    p.page_size = (int)k.size(1), p.Hkv = (int)k.size(2), p.Dk = (int)k.size(3), p.Dv = (int)v.size(3);
    p.dtype = i8 ? WS_DTYPE_I8 : half_of(type);
    return p;
}

// q, k, v, positions, cos_sin, slots, k_pages, v_pages, k_scales, v_scales, axis_map, axes, pairs, q_out
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 14, [&]() -> PyObject* {
        const char* what = "rope_append";
        const at::Tensor &k = tensor(what, "k", a[1]), &v = tensor(what, "v", a[2]), &slots = tensor(what, "slots", a[5]);
        if (!k.is_cuda()) refuse(what, "CUDA tensors required (there is no CPU path)");
        const at::Device dev = k.device();
        const at::ScalarType st = k.scalar_type();
        const int type = half_of(st);
        if (type < 0) refuse(what, "q, k, v must be bf16 or fp16");
        if (k.dim() != 3) refuse(what, "k must be [N, Hkv, Dk]");
        const int64_t N = k.size(0);
        want_rows(what, "k", k, st, N, dev);
        want_rows(what, "v", v, st, N, dev);
        const ws_paged_kv p = pool_of(what, a[6], a[7], a[8], a[9], dev);
        for (int i = 6; i < 10; ++i)
            if (a[i] != Py_None) at::assert_no_internal_overlap(THPVariable_Unpack(a[i]));
        if (k.size(1) != p.Hkv || v.size(1) != p.Hkv || k.size(2) != p.Dk || v.size(2) != p.Dv)
            refuse(what, "k, v must be [N, " + std::to_string(p.Hkv) + ", " + std::to_string(p.Dk) + "] and [N, " +
                             std::to_string(p.Hkv) + ", " + std::to_string(p.Dv) + "] as the pool is");
        want(what, "slots", slots, at::kLong, 1, dev);
        if (slots.numel() != N) refuse(what, "slots must hold one entry per token");
        if ((a[3] == Py_None) != (a[4] == Py_None)) refuse(what, "positions and cos_sin: both or neither");
        ws_rope r;
        const bool turn = a[4] != Py_None;
        if (turn) r = rope_of(what, a[3], a[4], N, dev, a[10], a[11], a[12], false);
        const c10::cuda::OptionalCUDAGuard guard(dev);
        at::Tensor q, out;
        if (a[0] != Py_None) {
            q = tensor(what, "q", a[0]);
            want_rows(what, "q", q, st, N, dev);
            if (q.size(2) != p.Dk || q.size(1) > INT32_MAX) refuse(what, "q must be [N, H, " + std::to_string(p.Dk) + "]");
            if (a[13] == Py_None) {
                out = fresh(q.sizes(), st, dev);
            } else {
                out = tensor(what, "q_out", a[13]);
                want_rows(what, "q_out", out, st, N, dev);
                if (out.sizes() != q.sizes()) refuse(what, "q_out must have q's shape");
                want_apart(out, q, {&k, &v});
            }
        } else if (a[13] != Py_None) {
            refuse(what, "q_out without q");
        }
        const bool has = q.defined();
        void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
        check(p_rope_append(turn ? &r : nullptr, has ? q.data_ptr() : nullptr, has ? q.stride(0) : 0, has ? q.stride(1) : 0,
                            has ? (int)q.size(1) : 0, p.Dk, has ? out.data_ptr() : nullptr, has ? out.stride(0) : 0,
                            has ? out.stride(1) : 0, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                            v.stride(1), type, N, data<int64_t>(slots), &p, stream),
              "ws_rope_append");
        if (!has) Py_RETURN_NONE;
        return THPVariable_Wrap(out);
    });
}

// q, k_pages, v_pages, page_table, seq_lens, scale, window, k_scales, v_scales, out, lse
PyObject* paged_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 11, [&]() -> PyObject* {
        const char* what = "paged_decode";
        const at::Tensor &q = tensor(what, "q", a[0]), &table = tensor(what, "page_table", a[3]),
                         &lens = tensor(what, "seq_lens", a[4]);
        if (!q.is_cuda()) refuse(what, "CUDA tensors required (there is no CPU path)");
        const at::Device dev = q.device();
        const at::ScalarType st = q.scalar_type();
        const int type = half_of(st);
        if (type < 0 || q.dim() != 3 || !unit(q, 2))
            refuse(what, "q must be bf16 or fp16 [B, H, Dk] with unit stride on the head dim");
        const int64_t B = q.size(0), H = q.size(1);
        const ws_paged_kv p = pool_of(what, a[1], a[2], a[7], a[8], dev);
        if (p.dtype != type && p.dtype != WS_DTYPE_I8) refuse(what, "the pool must hold q's type or int8");
        if (q.size(2) != p.Dk || p.Hkv < 1 || H < 1 || H % p.Hkv) refuse(what, "q must be [B, Hkv * G, Dk]");
        if (B > INT32_MAX || H > INT32_MAX) refuse(what, "bad shape");
        want_table(what, table, B, dev);
        want(what, "seq_lens", lens, at::kInt, 1, dev);
        if (lens.numel() != B) refuse(what, "seq_lens must hold one entry per request");
        const double scale = PyFloat_AsDouble(a[5]);
        if (scale == -1.0 && PyErr_Occurred()) throw PythonError();
        const int64_t window = integer(a[6]);
        if (window < 0) refuse(what, "window must not be negative");
        const c10::cuda::OptionalCUDAGuard guard(dev);
        const at::Tensor out = output(what, "out", a[9], {B, H, p.Dv}, st, dev);
        const at::Tensor lse = output(what, "lse", a[10], {B, H}, at::kFloat, dev);
        for (const at::Tensor* t : {&q, &table, &lens}) {
            if (a[9] != Py_None) at::assert_no_overlap(out, *t);
            if (a[10] != Py_None) at::assert_no_overlap(lse, *t);
        }
        void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
        const Workspace ws = workspace(g_decode_ws, dev, stream);
        check(p_paged_decode(q.data_ptr(), q.stride(0), q.stride(1), type, (int)B, (int)(H / p.Hkv), &p, data<int32_t>(table),
                             table.stride(0), (int)std::min<int64_t>(table.size(1), INT32_MAX), data<int32_t>(lens),
                             (int)std::min<int64_t>(window, INT32_MAX), (float)scale, out.data_ptr(), data<float>(lse), ws.ptr,
                             ws.bytes, stream),
              "ws_paged_decode");
        PyObject* r = PyTuple_New(2);
        if (!r) return nullptr;
        PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(out));
        PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(lse));
        return r;
    });
}

// bytes, device index: a zeroed buffer made while the current stream is being captured, but outside of the capture: on
// another stream, and with the capture's ban on allocations lifted for this thread meanwhile.
PyObject* zeros_outside_capture(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 2, [&]() -> PyObject* {
        const int64_t bytes = integer(a[0]), index = integer(a[1]);
        const at::Device dev(at::kCUDA, (c10::DeviceIndex)index);
        const c10::cuda::OptionalCUDAGuard guard(dev);
        const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
        c10::cuda::CUDAStream side = c10::cuda::getStreamFromPool(false, dev.index());
        for (int i = 0; i < 64; ++i) {   // the captured stream may be of the pool too
            const c10::cuda::CUDAStreamGuard on_side(side);
            if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) {
                const at::Tensor t = at::zeros({bytes}, at::TensorOptions().dtype(at::kByte).device(dev));
                side.synchronize();
                return THPVariable_Wrap(t);
            }
            side = c10::cuda::getStreamFromPool(false, dev.index());
        }
        refuse("workspace", "no stream that is not being captured");
    });
}

// (addresses of ws_last_error, ws_paged_slots, ws_paged_release, ws_rope_append, ws_paged_decode; the two workspace
// sizes; ScopeError, workspaces.get, the pool's dict, PagedStep)
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 11, [&]() -> PyObject* {
        auto address = [&](int i) { return reinterpret_cast<void*>((uintptr_t)integer(a[i])); };
        p_last_error = reinterpret_cast<decltype(p_last_error)>(address(0));
        p_paged_slots = reinterpret_cast<decltype(p_paged_slots)>(address(1));
        p_paged_release = reinterpret_cast<decltype(p_paged_release)>(address(2));
        p_rope_append = reinterpret_cast<decltype(p_rope_append)>(address(3));
        p_paged_decode = reinterpret_cast<decltype(p_paged_decode)>(address(4));
        g_slots_ws = (size_t)integer(a[5]), g_decode_ws = (size_t)integer(a[6]);
        PyObject** keep[4] = {&g_error, &g_pool_get, &g_pool_bufs, &g_step};
        for (int i = 0; i < 4; ++i) {
            Py_INCREF(a[7 + i]);
            Py_XDECREF(*keep[i]);
            *keep[i] = a[7 + i];
        }
        Py_RETURN_NONE;
    });
}

#define ENTRY(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(setup), ENTRY(zeros_outside_capture), ENTRY(paged_slots), ENTRY(paged_release), ENTRY(rope), ENTRY(rope_append),
                         ENTRY(paged_decode), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
