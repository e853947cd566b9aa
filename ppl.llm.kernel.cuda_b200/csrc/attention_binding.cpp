// What the Python binding of rotary positions, the paged cache and decode attention does on every call: tensors are checked, the argument
// block is filled in, the C entry point is called with the interpreter released.  Compiled, because the same in Python took 1.7 to
// 3.7 us a call, more than the smallest of these kernels; now it takes 0.4 to 0.6 (a 16-token rotation, call after call: 7.5 -> 4.3 us).  Each function takes the address of its entry point, the stream and the device
// that the tensors must be on (-1: memory of the host), and returns the entry point's code; a tensor that does not fit is a ValueError.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/pplb200_attention.h"

namespace {

struct Refused {}; // the Python error is set

[[noreturn]] void refuse(const char* format, const char* name, long long a = 0, long long b = 0, long long c = 0) {
    PyErr_Format(PyExc_ValueError, format, name, a, b, c);
    throw Refused();
}
const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
        throw Refused();
    }
    return THPVariable_Unpack(o);
}
bool on(const at::Tensor& t, int64_t device) { return t.device().index() == device && (device < 0 || t.is_cuda()); }

int64_t integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused();
    return v;
}
int32_t small_integer(PyObject* o) {
    const int64_t v = integer(o);
    if (v != (int32_t)v) {
        PyErr_SetString(PyExc_OverflowError, "the number does not fit 32 bits");
        throw Refused();
    }
    return (int32_t)v;
}
int32_t truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Refused();
    return v;
}
void* address(PyObject* o) {
    void* p = PyLong_AsVoidPtr(o);
    if (!p && PyErr_Occurred()) throw Refused();
    return p;
}
float real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused();
    return (float)v;
}

// fp16 [tokens, heads, head_dim] whose heads are contiguous; tokens < 0, head_dim < 0: the first tensor tells
struct Rows {
    void* data = nullptr;
    int64_t stride = 0;
    int32_t heads = 0;
};
Rows rows(PyObject* o, const char* name, int64_t& tokens, int64_t& head_dim, int64_t device) {
    const at::Tensor& t = tensor(o, name);
    const bool fits = t.dim() == 3 && t.scalar_type() == at::kHalf && on(t, device) && (tokens < 0 || t.size(0) == tokens) &&
                      (head_dim < 0 || t.size(2) == head_dim) && t.stride(2) == 1 && (t.size(1) <= 1 || t.stride(1) == t.size(2)) && t.size(1) <= INT32_MAX;
    if (!fits)
        refuse(tokens < 0 ? "%s must be fp16 [tokens, heads, dimensions] on the current device, the heads of a token contiguous"
                          : "%s must be fp16 [%lld, heads, %lld] on the current device %lld, the heads of a token contiguous", name, tokens, head_dim, device);
    tokens = t.size(0);
    head_dim = t.size(2);
    return {t.data_ptr(), t.stride(0), (int32_t)t.size(1)};
}
void same_heads(const Rows& a, const Rows& b, const char* name) {
    if (a.heads != b.heads) refuse("%s must have %lld heads, got %lld", name, a.heads, b.heads);
}
void* indices(PyObject* o, const char* name, int64_t tokens, int64_t device) {
    const at::Tensor& t = tensor(o, name);
    if (t.dim() != 1 || t.size(0) != tokens || t.scalar_type() != at::kLong || (tokens > 1 && t.stride(0) != 1) || !on(t, device))
        refuse("%s must be a contiguous int64 [%lld] tensor on the current device %lld", name, tokens, device);
    return t.data_ptr();
}

// (address of the turns, device, rotary_dim, magnitude) of a RotaryTable
struct Table {
    const uint64_t* turns;
    int32_t rotary_dim;
    float magnitude;
};
Table table_of(PyObject* o, int64_t device) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) refuse("%s is needed", "a rotary table");
    if (integer(PyTuple_GET_ITEM(o, 1)) != device) refuse("%s is not on the current device", "the rotary table");
    return {(const uint64_t*)address(PyTuple_GET_ITEM(o, 0)), small_integer(PyTuple_GET_ITEM(o, 2)), real(PyTuple_GET_ITEM(o, 3))};
}
// (pplb200_kv_cache as bytes, device) of a PagedKVCache
const pplb200_kv_cache* cache_of(PyObject* o, int64_t device) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2 || !PyBytes_Check(PyTuple_GET_ITEM(o, 0)) || PyBytes_GET_SIZE(PyTuple_GET_ITEM(o, 0)) != (Py_ssize_t)sizeof(pplb200_kv_cache))
        refuse("%s is needed", "a cache");
    if (integer(PyTuple_GET_ITEM(o, 1)) != device) refuse("%s is not on the current device", "the cache");
    return (const pplb200_kv_cache*)PyBytes_AS_STRING(PyTuple_GET_ITEM(o, 0));
}

// body(): fills in the block and gives what is to be called with the interpreter released
template <class F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F body) {
    if (given != wanted) {
        PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", wanted, given);
        return nullptr;
    }
    try {
        auto call = body();
        int32_t rc;
        Py_BEGIN_ALLOW_THREADS
        rc = call();
        Py_END_ALLOW_THREADS
        return PyLong_FromLong(rc);
    } catch (const Refused&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    }
    return nullptr;
}

// entry, stream, device, q | None, k | None, positions, table, interleaved, q_out, k_out
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 10, [&] {
        auto* const entry = (decltype(&pplb200_rotary_fp16))address(a[0]);
        const pplb200_stream_t stream = (pplb200_stream_t)address(a[1]);
        const int64_t device = integer(a[2]);
        int64_t tokens = -1, dim = -1;
        Rows q, k, qo, ko;
        if (a[3] != Py_None) {
            q = rows(a[3], "q", tokens, dim, device);
            qo = rows(a[8], "q_out", tokens, dim, device);
            same_heads(q, qo, "q_out");
        }
        if (a[4] != Py_None) {
            k = rows(a[4], "k", tokens, dim, device);
            ko = rows(a[9], "k_out", tokens, dim, device);
            same_heads(k, ko, "k_out");
        }
        if (tokens < 0) refuse("neither %s nor k is given", "q");
        const Table t = table_of(a[6], device);
        pplb200_rotary_args args = {};
        args.q = q.data; args.k = k.data; args.q_out = qo.data; args.k_out = ko.data;
        args.positions = (const int64_t*)indices(a[5], "positions", tokens, device);
        args.turns = t.turns;
        args.tokens = tokens;
        args.q_stride = q.stride; args.k_stride = k.stride; args.q_out_stride = qo.stride; args.k_out_stride = ko.stride;
        args.q_heads = q.heads; args.k_heads = k.heads;
        if (dim > INT32_MAX) refuse("%s: too many dimensions", "q");
        args.head_dim = (int32_t)dim; args.rotary_dim = t.rotary_dim; args.interleaved = truth(a[7]); args.magnitude = t.magnitude;
        return [=] { return entry(stream, &args); };
    });
}

// entry, stream, device, cache, q | None, k, v, positions, slots, table | None, interleaved, q_out
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 12, [&] {
        auto* const entry = (decltype(&pplb200_kv_cache_write_fp16))address(a[0]);
        const pplb200_stream_t stream = (pplb200_stream_t)address(a[1]);
        const int64_t device = integer(a[2]);
        const pplb200_kv_cache* const cache = cache_of(a[3], device);
        int64_t tokens = -1, dim = -1;
        const Rows k = rows(a[5], "k", tokens, dim, device), v = rows(a[6], "v", tokens, dim, device);
        if (k.heads != cache->kv_heads || v.heads != cache->kv_heads || dim != cache->head_dim)
            refuse("%s must have the cache's %lld heads of %lld dimensions", "k and v", cache->kv_heads, cache->head_dim);
        pplb200_kv_write_args args = {};
        args.k = k.data; args.v = v.data;
        args.k_stride = k.stride; args.v_stride = v.stride;
        args.tokens = tokens;
        args.slots = (const int64_t*)indices(a[8], "slots", tokens, device);
        args.magnitude = 1.0f;
        if (a[9] != Py_None) {
            const Table t = table_of(a[9], device);
            if (a[4] != Py_None) {
                const Rows q = rows(a[4], "q", tokens, dim, device), qo = rows(a[11], "q_out", tokens, dim, device);
                same_heads(q, qo, "q_out");
                args.q = q.data; args.q_out = qo.data;
                args.q_stride = q.stride; args.q_out_stride = qo.stride;
                args.q_heads = q.heads;
            }
            args.positions = (const int64_t*)indices(a[7], "positions", tokens, device);
            args.turns = t.turns; args.rotary_dim = t.rotary_dim; args.magnitude = t.magnitude;
            args.interleaved = truth(a[10]);
        }
        return [=] { return entry(stream, cache, &args); };
    });
}

// entry, stream, device, cache, slots, k_out, v_out
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 7, [&] {
        auto* const entry = (decltype(&pplb200_kv_cache_read_fp16))address(a[0]);
        const pplb200_stream_t stream = (pplb200_stream_t)address(a[1]);
        const int64_t device = integer(a[2]);
        const pplb200_kv_cache* const cache = cache_of(a[3], device);
        const at::Tensor& s = tensor(a[4], "slots");
        const int64_t tokens = s.dim() == 1 ? s.size(0) : -1;
        const int64_t* const slots = (const int64_t*)indices(a[4], "slots", tokens, device);
        void* out[2];
        for (int i = 0; i < 2; ++i) {
            const char* const name = i ? "v_out" : "k_out";
            const at::Tensor& t = tensor(a[5 + i], name);
            if (t.dim() != 3 || t.size(0) != tokens || t.size(1) != cache->kv_heads || t.size(2) != cache->head_dim || t.scalar_type() != at::kHalf || !t.is_contiguous() || !on(t, device))
                refuse("%s must be contiguous fp16 [%lld, %lld, %lld] on the current device", name, tokens, cache->kv_heads, cache->head_dim);
            out[i] = t.data_ptr();
        }
        void *const k = out[0], *const v = out[1];
        return [=] { return entry(stream, cache, slots, tokens, k, v); };
    });
}

// entry, stream, device, cache, (q_heads, max_batch, max_pages, ws, ws_bytes, window, scale), q, pages, lengths, out, lse | None
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 10, [&] {
        auto* const entry = (decltype(&pplb200_paged_decode_attention_fp16))address(a[0]);
        const pplb200_stream_t stream = (pplb200_stream_t)address(a[1]);
        const int64_t device = integer(a[2]);
        const pplb200_kv_cache* const cache = cache_of(a[3], device);
        if (!PyTuple_Check(a[4]) || PyTuple_GET_SIZE(a[4]) != 7) refuse("%s is needed", "an attention object");
        auto own = [&](int i) { return PyTuple_GET_ITEM(a[4], i); };
        const int32_t q_heads = small_integer(own(0));
        const int64_t max_batch = integer(own(1)), max_pages = integer(own(2));
        int64_t batch = -1, dim = cache->head_dim;
        const at::Tensor& first = tensor(a[5], "q");
        if (first.dim() == 3) batch = first.size(0);
        const Rows q = rows(a[5], "q", batch, dim, device), out = rows(a[8], "out", batch, dim, device);
        if (q.heads != q_heads || out.heads != q_heads || batch > max_batch) refuse("%s must be at most %lld sequences of %lld heads", "q and out", max_batch, q_heads);
        const at::Tensor& pages = tensor(a[6], "pages");
        if (pages.dim() != 2 || pages.size(0) != batch || pages.size(1) > max_pages || (pages.size(1) > 1 && pages.stride(1) != 1) || pages.scalar_type() != at::kInt || !on(pages, device))
            refuse("%s must be int32 [%lld, at most %lld] with contiguous rows on the current device", "pages", batch, max_pages);
        const at::Tensor& lengths = tensor(a[7], "lengths");
        if (lengths.dim() != 1 || lengths.size(0) != batch || (batch > 1 && lengths.stride(0) != 1) || lengths.scalar_type() != at::kInt || !on(lengths, device))
            refuse("%s must be a contiguous int32 [%lld] tensor on the current device", "lengths", batch);
        pplb200_paged_attention_args args = {};
        if (a[9] != Py_None) {
            const at::Tensor& lse = tensor(a[9], "lse");
            if (lse.dim() != 2 || lse.size(0) != batch || lse.size(1) != q_heads || lse.scalar_type() != at::kFloat || !lse.is_contiguous() || !on(lse, device))
                refuse("%s must be contiguous fp32 [%lld, %lld] on the current device", "lse", batch, q_heads);
            args.optional_lse = (float*)lse.data_ptr();
        }
        args.q = q.data; args.out = out.data;
        args.pages = (const int32_t*)pages.data_ptr(); args.lengths = (const int32_t*)lengths.data_ptr();
        args.ws = address(own(3)); args.ws_bytes = integer(own(4));
        args.batch = batch; args.pages_per_sequence = pages.size(1); args.pages_stride = pages.stride(0);
        args.q_stride = q.stride; args.out_stride = out.stride;
        args.q_heads = q_heads; args.window = small_integer(own(5)); args.scale = real(own(6));
        return [=] { return entry(stream, cache, &args); };
    });
}

PyMethodDef methods[] = {{"rotary", (PyCFunction)(void (*)(void))rotary, METH_FASTCALL, nullptr},
                         {"write", (PyCFunction)(void (*)(void))write, METH_FASTCALL, nullptr},
                         {"read", (PyCFunction)(void (*)(void))read, METH_FASTCALL, nullptr},
                         {"attend", (PyCFunction)(void (*)(void))attend, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "pplb200_attention_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit_pplb200_attention_binding() { return PyModule_Create(&module); }
