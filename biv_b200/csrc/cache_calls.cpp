// The Python calls of the paged cache: torch tensors in, one of the C ABI's bivmoe_cache_* calls out.
//
// A decode step makes these calls for every layer, and their kernels take three to ten microseconds: with
// the checks and the argument structs in Python, through ctypes, a call took 11 to 15, all of it host
// time.  Here it takes 4 to 6.  Nothing is computed here: shapes, types and devices are looked at, outputs
// allocated, and the functions of libbivmoe.so called by the addresses that cache.py hands over.
#include <Python.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>

#include "../../include/bivmoe.h"

namespace {

struct Geometry {
    bivmoe_cache* cache;
    int (*extend)(bivmoe_cache*, const bivmoe_extend_args*, void*);
    int (*store)(bivmoe_cache*, const bivmoe_store_args*, void*);
    int (*attend)(bivmoe_cache*, const bivmoe_attend_args*, void*);
    int device, n_head, n_head_kv, head_dim, page_size, ggml_type, axes;
    at::ScalarType type;
    float scale;
};
constexpr const char* kName = "biv_b200.cache";

// a wrong argument: ValueError with this text
struct Wrong { std::string text; };

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) throw Wrong{std::string(what) + ": a tensor is wanted"};
    return THPVariable_Unpack(o);
}
bool here(const Geometry& g, const at::Tensor& t) { return t.is_cuda() && t.get_device() == g.device; }

template <class T> T* list(const Geometry& g, PyObject* o, const char* what, int64_t n) {
    constexpr auto type = sizeof(T) == 8 ? at::kLong : at::kInt;
    const at::Tensor& t = tensor(o, what);
    if (t.scalar_type() != type || !here(g, t) || !t.is_contiguous() || t.numel() < n)
        throw Wrong{std::string(what) + ": " + std::to_string(n) + " contiguous " + (sizeof(T) == 8 ? "int64" : "int32") +
                    " on the cache's device are wanted"};
    return (T*)t.data_ptr();
}
struct Table { int32_t* data; int64_t stride; int32_t width; };
Table table(const Geometry& g, PyObject* o, int64_t n_seq) {
    const at::Tensor& t = tensor(o, "table");
    if (t.scalar_type() != at::kInt || !here(g, t) || t.dim() != 2 || t.size(0) < n_seq || (t.size(1) > 1 && t.stride(1) != 1) ||
        t.size(1) > INT32_MAX)
        throw Wrong{"table: [n_seq, pages] int32 with neighbouring pages is wanted"};
    return {(int32_t*)t.data_ptr(), t.stride(0), (int32_t)t.size(1)};
}
// A dimension's stride; where there is one place or none, which torch may give any stride, `dense`.
int64_t stride(const at::Tensor& t, int dim, int64_t dense) { return t.size(dim) > 1 ? t.stride(dim) : dense; }
bivmoe_pool pool(const Geometry& g, PyObject* o, const char* what) {
    const at::Tensor& t = tensor(o, what);
    if (t.scalar_type() != g.type || !here(g, t) || t.dim() != 4 || t.size(1) != g.page_size || t.size(2) != g.n_head_kv ||
        t.size(3) != g.head_dim || t.stride(3) != 1)
        throw Wrong{std::string(what) + ": [pages, " + std::to_string(g.page_size) + ", " + std::to_string(g.n_head_kv) + ", " +
                    std::to_string(g.head_dim) + "] of the cache's type is wanted"};
    const int64_t token = (int64_t)g.n_head_kv * g.head_dim;
    return {t.data_ptr(), stride(t, 0, g.page_size * token), stride(t, 1, token), stride(t, 2, g.head_dim), t.size(0)};
}
bivmoe_rows rows(const Geometry& g, const at::Tensor& t, const char* what, int heads, int64_t n, int ggml_type) {
    if (!here(g, t) || t.dim() != 3 || t.size(0) != n || t.size(1) != heads || t.size(2) != g.head_dim || t.stride(2) != 1)
        throw Wrong{std::string(what) + ": [tokens, " + std::to_string(heads) + ", " + std::to_string(g.head_dim) +
                    "] rows on the cache's device are wanted"};
    return {t.data_ptr(), stride(t, 0, (int64_t)heads * g.head_dim), stride(t, 1, g.head_dim), ggml_type, 0};
}
int32_t count(int64_t n, const char* what) {
    if (n < 0 || n > INT32_MAX) throw Wrong{std::string(what) + ": out of range"};
    return (int32_t)n;
}
int64_t whole(PyObject* o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
int32_t whole32(PyObject* o, const char* what) {
    const int64_t v = whole(o);
    if (v < INT32_MIN || v > INT32_MAX) throw Wrong{std::string(what) + ": out of range"};
    return (int32_t)v;
}
at::Tensor fresh(const Geometry& g, at::IntArrayRef shape, at::ScalarType type) {
    return at::empty(shape, at::TensorOptions().dtype(type).device(at::Device(at::kCUDA, (c10::DeviceIndex)g.device)));
}
// `n` values of a type from place `offset` on (in values of it) of a tensor's memory, without the
// dispatcher's way to a view (six of them took longer than the launch)
at::Tensor share(const at::Tensor& room, at::ScalarType type, int64_t offset, int64_t n) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(room.storage()), room.key_set(), at::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_storage_offset(offset);
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    return t;
}
// the rows' own layout where there is none given: [n, n_head, head_dim] of the cache's type
at::Tensor out_rows(const Geometry& g, PyObject* o, int64_t n) {
    if (o == Py_None) return fresh(g, {n, g.n_head, g.head_dim}, g.type);
    const at::Tensor& t = tensor(o, "out");
    if (t.scalar_type() != g.type) throw Wrong{"out: the cache's type is wanted"};
    return t;
}
void* stream(const Geometry& g) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)g.device).stream(); }

Geometry* geometry(PyObject* const* args, Py_ssize_t n, Py_ssize_t wanted) {
    if (n != wanted) throw Wrong{"wrong number of arguments"};
    auto* g = (Geometry*)PyCapsule_GetPointer(args[0], kName);
    if (!g) throw python_error();
    return g;
}

// A call's body: what it returns, or the library's status as a whole number, or an exception.
template <class F> PyObject* guarded(F f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Wrong& w) {
        PyErr_SetString(PyExc_ValueError, w.text.c_str());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// (cache, extend, store, attend: addresses; device, n_head, n_head_kv, head_dim, page_size, ggml_type, axes)
PyObject* make(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 11) throw Wrong{"wrong number of arguments"};
        auto* g = new Geometry();
        g->cache = (bivmoe_cache*)whole(a[0]);
        g->extend = (decltype(g->extend))whole(a[1]);
        g->store = (decltype(g->store))whole(a[2]);
        g->attend = (decltype(g->attend))whole(a[3]);
        int* fields[] = {&g->device, &g->n_head, &g->n_head_kv, &g->head_dim, &g->page_size, &g->ggml_type, &g->axes};
        for (int i = 0; i < 7; i++) *fields[i] = (int)whole(a[4 + i]);
        g->type = g->ggml_type == BIVMOE_F16 ? at::kHalf : at::kBFloat16;
        g->scale = (float)(1.0 / std::sqrt((double)g->head_dim));
        return PyCapsule_New(g, kName, [](PyObject* c) { delete (Geometry*)PyCapsule_GetPointer(c, kName); });
    });
}

// (geometry, past, added, held or None, free_pages, free_count, table, n_tokens, out or None)
PyObject* extend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const Geometry& g = *geometry(a, n, 9);
        bivmoe_extend_args x{};
        const int64_t n_seq = tensor(a[1], "past").numel(), n_tokens = whole(a[7]);
        x.n_seq = count(n_seq, "past");
        x.n_tokens = count(n_tokens, "n_tokens");
        x.past = list<int32_t>(g, a[1], "past", n_seq);
        x.added = list<int32_t>(g, a[2], "added", n_seq);
        x.held = a[3] == Py_None ? nullptr : list<int32_t>(g, a[3], "held", n_seq);
        x.free_pages = list<int32_t>(g, a[4], "free_pages", 0);
        x.n_free = count(THPVariable_Unpack(a[4]).numel(), "free_pages");
        x.free_count = list<int32_t>(g, a[5], "free_count", 1);
        const Table t = table(g, a[6], n_seq);
        x.table = t.data; x.table_stride = t.stride; x.table_width = t.width;
        at::Tensor out[6];                        // length, first, slots, positions, left, held
        if (a[8] == Py_None) {
            // one allocation: the slots, then the lists of int32
            const int64_t ints = 3 * n_seq + 3 + n_tokens;
            const at::Tensor room = fresh(g, {n_tokens + (ints + 1) / 2}, at::kLong);
            out[2] = share(room, at::kLong, 0, n_tokens);
            int64_t at = 2 * n_tokens;
            auto part = [&](int64_t k) { at += k; return share(room, at::kInt, at - k, k); };
            out[0] = part(n_seq); out[1] = part(n_seq + 1); out[4] = part(2); out[5] = part(n_seq); out[3] = part(n_tokens);
            x.length = (int32_t*)out[0].data_ptr(); x.first = (int32_t*)out[1].data_ptr(); x.slots = (int64_t*)out[2].data_ptr();
            x.positions = (int32_t*)out[3].data_ptr(); x.left = (int32_t*)out[4].data_ptr(); x.held_out = (int32_t*)out[5].data_ptr();
        } else {
            if (!PyTuple_Check(a[8]) || PyTuple_GET_SIZE(a[8]) != 6) throw Wrong{"out: a Step is wanted"};
            PyObject** o = &PyTuple_GET_ITEM(a[8], 0);
            x.length = list<int32_t>(g, o[0], "length", n_seq);
            x.first = list<int32_t>(g, o[1], "first", n_seq + 1);
            x.slots = list<int64_t>(g, o[2], "slots", n_tokens);
            x.positions = list<int32_t>(g, o[3], "positions", n_tokens);
            x.left = list<int32_t>(g, o[4], "left", 2);
            x.held_out = list<int32_t>(g, o[5], "held", n_seq);
        }
        if (const int code = g.extend(g.cache, &x, stream(g))) return PyLong_FromLong(code);
        if (a[8] != Py_None) { Py_INCREF(a[8]); return a[8]; }
        PyObject* r = PyTuple_New(6);
        if (!r) throw python_error();
        for (int i = 0; i < 6; i++) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(std::move(out[i])));
        return r;
    });
}

// (geometry, q, k, v, k_pool, v_pool, slots, positions or None, out or None)
PyObject* store(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        const Geometry& g = *geometry(a, n_args, 9);
        const at::Tensor &q = tensor(a[1], "q"), &k = tensor(a[2], "k"), &v = tensor(a[3], "v");
        const auto type = q.scalar_type();
        const int ty = type == at::kFloat ? BIVMOE_F32 : type == at::kHalf ? BIVMOE_F16 : type == at::kBFloat16 ? BIVMOE_BF16 : -1;
        if (ty < 0 || k.scalar_type() != type || v.scalar_type() != type)
            throw Wrong{"q, k and v: rows of one type, float32, float16 or bfloat16, are wanted"};
        if (q.dim() != 3) throw Wrong{"q: [tokens, heads, head_dim] rows are wanted"};
        const int64_t n = q.size(0);
        bivmoe_store_args x{};
        x.n_tokens = count(n, "q");
        x.q = rows(g, q, "q", g.n_head, n, ty);
        x.k = rows(g, k, "k", g.n_head_kv, n, ty);
        x.v = rows(g, v, "v", g.n_head_kv, n, ty);
        x.k_pool = pool(g, a[4], "k_pool");
        x.v_pool = pool(g, a[5], "v_pool");
        x.slots = list<int64_t>(g, a[6], "slots", n);
        if (g.axes) {
            const at::Tensor* p = a[7] == Py_None ? nullptr : &tensor(a[7], "positions");
            if (!p || p->scalar_type() != at::kInt || !here(g, *p) || p->numel() != g.axes * n || p->dim() < 1 || p->dim() > 2 ||
                (n > 1 && p->stride(-1) != 1) || (p->dim() == 2 && p->size(0) != g.axes) || (p->dim() == 1 && g.axes > 1))
                throw Wrong{"positions: [" + std::to_string(g.axes) + ", n] int32 on the cache's device are wanted"};
            x.positions = (int32_t*)p->data_ptr();
            x.positions_stride = p->dim() == 2 ? p->stride(0) : n;
        }
        at::Tensor out = out_rows(g, a[8], n);
        x.q_out = rows(g, out, "out", g.n_head, n, g.ggml_type);
        if (const int code = g.store(g.cache, &x, stream(g))) return PyLong_FromLong(code);
        return THPVariable_Wrap(std::move(out));
    });
}

// (geometry, q, k_pool, v_pool, table, first, length, max_new, scale or None, window, sinks, out or None)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        const Geometry& g = *geometry(a, n_args, 12);
        const at::Tensor& q = tensor(a[1], "q");
        if (q.scalar_type() != g.type || q.dim() != 3) throw Wrong{"q: [tokens, heads, head_dim] rows of the cache's type are wanted"};
        const int64_t n = q.size(0), n_seq = tensor(a[6], "length").numel();
        bivmoe_attend_args x{};
        x.n_tokens = count(n, "q");
        x.n_seq = count(n_seq, "length");
        x.q = rows(g, q, "q", g.n_head, n, g.ggml_type);
        x.k_pool = pool(g, a[2], "k_pool");
        x.v_pool = pool(g, a[3], "v_pool");
        const Table t = table(g, a[4], n_seq);
        x.table = t.data; x.table_stride = t.stride; x.table_width = t.width;
        x.first = list<int32_t>(g, a[5], "first", n_seq + 1);
        x.length = list<int32_t>(g, a[6], "length", n_seq);
        x.max_new = whole32(a[7], "max_new");
        x.scale = g.scale;
        if (a[8] != Py_None) {
            x.scale = (float)PyFloat_AsDouble(a[8]);
            if (PyErr_Occurred()) throw python_error();
        }
        x.window = whole32(a[9], "window");
        x.sinks = whole32(a[10], "sinks");
        at::Tensor out = out_rows(g, a[11], n);
        x.out = rows(g, out, "out", g.n_head, n, g.ggml_type);
        if (const int code = g.attend(g.cache, &x, stream(g))) return PyLong_FromLong(code);
        return THPVariable_Wrap(std::move(out));
    });
}

PyMethodDef methods[] = {{"make", (PyCFunction)(void (*)())make, METH_FASTCALL, nullptr},
                         {"extend", (PyCFunction)(void (*)())extend, METH_FASTCALL, nullptr},
                         {"store", (PyCFunction)(void (*)())store, METH_FASTCALL, nullptr},
                         {"attend", (PyCFunction)(void (*)())attend, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_cache_calls", "The Python calls of the paged cache.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__cache_calls() { return PyModule_Create(&module_def); }
