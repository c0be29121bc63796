// tensors.cc - the entry points of the paged caches and of the log
// probabilities for torch tensors, as a CPython extension (fyodor_b200/_tensors.so).
//
// A decode step calls them thousands of times a second on kernels of a few
// microseconds; through ctypes the checks and conversions of a dozen tensors
// took 8 microseconds of Python a call, here under one. Nothing is computed in
// this file: it checks tensors, takes their addresses and torch's current
// stream, and calls the C entry points of libfyodor_b200.so, whose addresses
// the package hands over once (bind()).
#include <Python.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include "fyodor_b200.h"

namespace {

struct {
    decltype(&fyb_kv_blocks) kv_blocks;
    decltype(&fyb_kv_release) kv_release;
    decltype(&fyb_rope) rope;
    decltype(&fyb_kv8_append) append;
    decltype(&fyb_kv8_read) read;
    decltype(&fyb_kv8_attention) attention;
    decltype(&fyb_kv4_append) append4;
    decltype(&fyb_kv4_read) read4;
    decltype(&fyb_kv4_attention) attention4;
    decltype(&fyb_logprobs) logprobs;
} entry;

struct Refused {};  // a Python exception is set

[[noreturn]] void refuse(const char *name, const char *what)
{
    PyErr_Format(PyExc_ValueError, "%s %s", name, what);
    throw Refused();
}

// The cache handle: what the Python object (KV8Handle, KV4Handle) holds the address of.
template <typename Cache> struct CacheHandle {
    Cache cache;
    int32_t device;
};

// One call: its device, taken from the cache or the first tensor seen.
struct Call {
    int device = -1;
    void on(int d, const char *name)
    {
        if (device < 0) {
            if (d != c10::cuda::current_device()) refuse(name, "is not on the current CUDA device");
            device = d;
        } else if (d != device) {
            refuse(name, "is on another device than the tensors before it");
        }
    }
    const at::Tensor &tensor(PyObject *o, const char *name)
    {
        if (!THPVariable_Check(o)) refuse(name, "has to be a tensor");
        const at::Tensor &t = THPVariable_Unpack(o);
        if (!t.is_cuda()) refuse(name, "has to be on the GPU");
        on(t.get_device(), name);
        return t;
    }
    template <typename Cache> const Cache *cache(PyObject *o)
    {
        const CacheHandle<Cache> *h = static_cast<const CacheHandle<Cache> *>(PyLong_AsVoidPtr(o));
        if (PyErr_Occurred()) throw Refused();
        if (!h) refuse("cache", "has no address");
        on(h->device, "cache");
        return &h->cache;
    }
    // a contiguous tensor of `kind` with `least` elements at least
    void *flat(PyObject *o, const char *name, at::ScalarType kind, int64_t least = 0)
    {
        const at::Tensor &t = tensor(o, name);
        if (t.scalar_type() != kind) refuse(name, "has another element type than it has to have");
        if (!t.is_contiguous()) refuse(name, "has to be contiguous");
        if (t.numel() < least) refuse(name, "has too few elements");
        return t.data_ptr();
    }
    int32_t *ints(PyObject *o, const char *name, int64_t least = 0)
    {
        return static_cast<int32_t *>(flat(o, name, at::kInt, least));
    }
    uint32_t *error(PyObject *o) { return o == Py_None ? nullptr : reinterpret_cast<uint32_t *>(ints(o, "error", 1)); }
    void *stream(PyObject *o)
    {
        if (o != Py_None) {
            void *s = PyLong_AsVoidPtr(o);
            if (PyErr_Occurred()) throw Refused();
            return s;
        }
        return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    }
};

// Rows [rows][heads][head_dim] whose heads are contiguous.
struct Rows {
    void *p = nullptr;
    int64_t rows = 0, heads = 0, dim = 0, stride = 0;
    at::ScalarType kind = at::kFloat;
};
Rows rows_of(Call &c, PyObject *o, const char *name)
{
    const at::Tensor &t = c.tensor(o, name);
    if (t.dim() != 3) refuse(name, "has to be [rows][heads][head_dim]");
    Rows r{t.data_ptr(), t.size(0), t.size(1), t.size(2), t.stride(0), t.scalar_type()};
    if ((t.stride(2) != 1 && r.dim > 1) || (t.stride(1) != r.dim && r.heads > 1))
        refuse(name, "has to have the heads of a row contiguous");
    if (r.rows < 2) r.stride = r.heads * r.dim;
    if (r.stride < 0) refuse(name, "has a negative stride");
    return r;
}
uint32_t type_of(at::ScalarType kind, const char *name)
{
    if (kind == at::kFloat) return 0;
    if (kind == at::kHalf) return 1;
    if (kind == at::kBFloat16) return 30;
    refuse(name, "has to be float32, float16 or bfloat16");
}
uint32_t type_of(const Rows &r, const char *name) { return type_of(r.kind, name); }
void alike(const Rows &a, const Rows &b, const char *name)
{
    if (a.rows != b.rows || a.dim != b.dim || a.kind != b.kind) refuse(name, "has other rows, head_dim or type than it has to have");
}

int64_t number(PyObject *o)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused();
    return v;
}
uint32_t u32(PyObject *o, const char *name)
{
    const int64_t v = number(o);
    if (v < 0 || v > 0xffffffffll) refuse(name, "is out of range");
    return (uint32_t)v;
}

fyb_rope_desc rope_desc(Call &c, PyObject *cos, PyObject *sin, PyObject *layout)
{
    fyb_rope_desc d;
    d.cos_table = static_cast<const float *>(c.flat(cos, "cos", at::kFloat));
    d.sin_table = static_cast<const float *>(c.flat(sin, "sin", at::kFloat));
    const at::Tensor &a = THPVariable_Unpack(cos), &b = THPVariable_Unpack(sin);
    if (a.dim() != 2 || b.dim() != 2 || a.size(0) != b.size(0) || a.size(1) != b.size(1) || a.size(0) > 0x7fffffff ||
        a.size(1) > 0x3fffffff)
        refuse("cos and sin", "have to be [positions][dims / 2], of one shape");
    d.table_rows = (uint32_t)a.size(0);
    d.dims = (uint32_t)a.size(1) * 2;
    const char *l = PyUnicode_Check(layout) ? PyUnicode_AsUTF8(layout) : "";
    if (!l) throw Refused();
    if (l[0] == 'i' && !strcmp(l, "interleaved")) d.layout = FYB_ROPE_INTERLEAVED;
    else if (!strcmp(l, "half")) d.layout = FYB_ROPE_HALF;
    else refuse("layout", "is 'interleaved' or 'half'");
    return d;
}

PyObject *answer(int r, const char *what)
{
    if (r == 0) Py_RETURN_NONE;
    if (r == -1) PyErr_Format(PyExc_ValueError, "%s refused its arguments", what);
    else PyErr_Format(PyExc_RuntimeError, "%s failed to launch (%d)", what, r);
    return nullptr;
}

template <typename F> PyObject *guarded(Py_ssize_t n, Py_ssize_t want, F f)
{
    if (n != want) return PyErr_Format(PyExc_TypeError, "%zd arguments given, %zd taken", n, want);
    try {
        return f();
    } catch (const Refused &) {
        return nullptr;
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyObject *kv_blocks(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 14, [&] {
        Call c;
        const at::Tensor &lengths = c.tensor(a[0], "lengths");
        const int64_t req = lengths.numel();
        const at::Tensor &table = c.tensor(a[2], "table");
        if (table.dim() != 2 || table.size(0) != req) refuse("table", "has to be [requests][blocks]");
        const int64_t rows = c.tensor(a[9], "slots").numel();
        if (req > 0x7fffffff || rows > 0x7fffffff) refuse("lengths or slots", "has too many elements");
        return answer(entry.kv_blocks(c.ints(a[0], "lengths"), c.ints(a[1], "new_tokens", req), (uint32_t)req,
                                      c.ints(a[2], "table"), (size_t)table.size(1), u32(a[5], "block_size"),
                                      c.ints(a[3], "free_list"), c.ints(a[4], "free_count", 1),
                                      c.ints(a[6], "lengths_out", req), c.ints(a[7], "free_count_out", 1),
                                      c.ints(a[8], "row_start", req + 1), c.ints(a[9], "slots"),
                                      c.ints(a[10], "positions", rows), c.ints(a[11], "row_request", rows),
                                      (uint32_t)rows, c.ints(a[12], "status", req), c.stream(a[13])),
                      "fyb_kv_blocks");
    });
}

PyObject *kv_release(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 7, [&] {
        Call c;
        const int64_t req = c.tensor(a[0], "lengths").numel();
        const at::Tensor &table = c.tensor(a[2], "table");
        if (table.dim() != 2 || table.size(0) != req) refuse("table", "has to be [requests][blocks]");
        const int64_t free = c.tensor(a[3], "free_list").numel();
        if (req > 0x7fffffff || free > 0x7fffffff) refuse("lengths or free_list", "has too many elements");
        return answer(entry.kv_release(c.ints(a[0], "lengths"), c.ints(a[1], "keep", req), (uint32_t)req,
                                       c.ints(a[2], "table"), (size_t)table.size(1), u32(a[5], "block_size"),
                                       c.ints(a[3], "free_list"), c.ints(a[4], "free_count", 1), (uint32_t)free,
                                       c.stream(a[6])),
                      "fyb_kv_release");
    });
}

// (q, k, positions, cos, sin, layout, q_out, k_out, error, stream)
PyObject *rope(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 10, [&] {
        Call c;
        const Rows q = rows_of(c, a[0], "q"), qo = rows_of(c, a[6], "q_out");
        alike(q, qo, "q_out");
        if (qo.heads != q.heads) refuse("q_out", "has other heads than q");
        Rows k, ko;
        if (a[1] != Py_None) {
            k = rows_of(c, a[1], "k");
            ko = rows_of(c, a[7], "k_out");
            alike(q, k, "k");
            alike(q, ko, "k_out");
            if (ko.heads != k.heads) refuse("k_out", "has other heads than k");
        }
        if (q.heads > 65536 || k.heads > 65536 || q.dim > 65536) refuse("q or k", "has too many heads or dimensions");
        const fyb_rope_desc d = rope_desc(c, a[3], a[4], a[5]);
        return answer(entry.rope(&d, c.ints(a[2], "positions", q.rows), (size_t)q.rows, (uint32_t)q.dim, type_of(q, "q"),
                                 q.p, (size_t)q.stride, qo.p, (size_t)qo.stride, (uint32_t)q.heads, k.p,
                                 (size_t)k.stride, ko.p, (size_t)ko.stride, (uint32_t)k.heads, c.error(a[8]),
                                 c.stream(a[9])),
                      "fyb_rope");
    });
}

// (cache, k, v, slots, positions, cos, sin, layout, q, q_out, error, stream)
template <typename Cache, typename Entry> PyObject *append_of(Entry entry, const char *what, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 12, [&] {
        Call c;
        const Cache *cache = c.cache<Cache>(a[0]);
        const Rows k = rows_of(c, a[1], "k"), v = rows_of(c, a[2], "v");
        alike(k, v, "v");
        if (k.heads != cache->kv_heads || v.heads != cache->kv_heads || k.dim != cache->head_dim)
            refuse("k or v", "has other heads or head_dim than the cache");
        const int32_t *slots = c.ints(a[3], "slots", k.rows), *positions = nullptr;
        fyb_rope_desc d;
        const bool turn = a[5] != Py_None;
        if (turn) {
            d = rope_desc(c, a[5], a[6], a[7]);
            positions = c.ints(a[4], "positions", k.rows);
        }
        Rows q, qo;
        if (a[8] != Py_None) {
            if (!turn) refuse("q", "needs cos and sin");
            q = rows_of(c, a[8], "q");
            qo = rows_of(c, a[9], "q_out");
            alike(k, q, "q");
            alike(k, qo, "q_out");
            if (q.heads != qo.heads || q.heads > 65536) refuse("q_out", "has other heads than q");
        }
        return answer(entry(cache, slots, (size_t)k.rows, type_of(k, "k"), k.p, (size_t)k.stride, v.p,
                                   (size_t)v.stride, turn ? &d : nullptr, positions, q.p, (size_t)q.stride, qo.p,
                                   (size_t)qo.stride, (uint32_t)q.heads, c.error(a[10]), c.stream(a[11])),
                      what);
    });
}

// (cache, slots, k_out, v_out, error, stream)
template <typename Cache, typename Entry> PyObject *read_of(Entry entry, const char *what, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 6, [&] {
        Call c;
        const Cache *cache = c.cache<Cache>(a[0]);
        const int64_t rows = c.tensor(a[1], "slots").numel(), need = rows * cache->kv_heads * cache->head_dim;
        const int32_t *slots = c.ints(a[1], "slots");
        float *k = static_cast<float *>(c.flat(a[2], "k_out", at::kFloat, need));
        float *v = static_cast<float *>(c.flat(a[3], "v_out", at::kFloat, need));
        return answer(entry(cache, slots, (size_t)rows, k, v, c.error(a[4]), c.stream(a[5])), what);
    });
}

// (cache, q, lengths, table, out, workspace, row_start, most_rows, scale, error, stream)
template <typename Cache, typename Entry> PyObject *attention_of(Entry entry, const char *what, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 11, [&] {
        Call c;
        const Cache *cache = c.cache<Cache>(a[0]);
        const Rows q = rows_of(c, a[1], "q"), out = rows_of(c, a[4], "out");
        alike(q, out, "out");
        if (q.heads != out.heads || q.dim != cache->head_dim || q.heads > 0x7fffffff)
            refuse("q or out", "has other heads or head_dim than it has to have");
        const int64_t req = c.tensor(a[2], "lengths").numel();
        const at::Tensor &table = c.tensor(a[3], "table");
        if (table.dim() != 2 || table.size(0) != req || req > 0x7fffffff) refuse("table", "has to be [requests][blocks]");
        const at::Tensor &ws = c.tensor(a[5], "workspace");
        if (!ws.is_contiguous()) refuse("workspace", "has to be contiguous");
        const double scale = a[8] == Py_None ? 1.0 / std::sqrt((double)cache->head_dim) : PyFloat_AsDouble(a[8]);
        if (PyErr_Occurred()) throw Refused();
        return answer(entry(cache, c.ints(a[2], "lengths"),
                                      a[6] == Py_None ? nullptr : c.ints(a[6], "row_start", req + 1), (uint32_t)req,
                                      u32(a[7], "most_rows"), (size_t)q.rows, c.ints(a[3], "table"),
                                      (size_t)table.size(1), type_of(q, "q"), q.p, (size_t)q.stride, out.p,
                                      (size_t)out.stride, (uint32_t)q.heads, (float)scale, ws.data_ptr(),
                                      (size_t)ws.nbytes(), c.error(a[9]), c.stream(a[10])),
                      what);
    });
}

#define CACHE_METHODS(name) \
    PyObject *name(PyObject *, PyObject *const *a, Py_ssize_t n) { return name##_of<fyb_kv8_cache>(entry.name, "fyb_kv8_" #name, a, n); } \
    PyObject *name##4(PyObject *, PyObject *const *a, Py_ssize_t n) { return name##_of<fyb_kv4_cache>(entry.name##4, "fyb_kv4_" #name, a, n); }
CACHE_METHODS(append)
CACHE_METHODS(read)
CACHE_METHODS(attention)

// (logits, tokens, logprob, entropy, rank, top_tokens, top_logprobs, workspace, error, stream)
PyObject *logprobs(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 10, [&] {
        Call c;
        const at::Tensor &x = c.tensor(a[0], "logits");
        if (x.dim() != 2 || (x.stride(1) != 1 && x.size(1) > 1)) refuse("logits", "has to be [rows][vocabulary], a row's logits contiguous");
        const int64_t rows = x.size(0), values = x.size(1), stride = rows < 2 ? values : x.stride(0);
        if (stride < values || values > 0x7fffffff) refuse("logits", "has overlapping rows or too many logits in one");
        auto floats = [&](PyObject *o, const char *name, int64_t least) {
            return o == Py_None ? nullptr : static_cast<float *>(c.flat(o, name, at::kFloat, least));
        };
        auto ints = [&](PyObject *o, const char *name, int64_t least) { return o == Py_None ? nullptr : c.ints(o, name, least); };
        int64_t top = 0;
        if (a[5] != Py_None) {
            const at::Tensor &t = c.tensor(a[5], "top_tokens");
            if (t.dim() != 2 || t.size(0) != rows || t.size(1) > 0x7fffffff) refuse("top_tokens", "has to be [rows][top]");
            top = t.size(1);
        }
        if (a[6] != Py_None) {  // not without tokens, nor of another width: it would be left, or filled in other places
            const at::Tensor &t = c.tensor(a[6], "top_logprobs");
            if ((t.dim() == 2 && t.size(1) != top) || (!top && t.numel())) refuse("top_logprobs", "has to be [rows][top], with top_tokens");
        }
        const at::Tensor &ws = c.tensor(a[7], "workspace");
        if (!ws.is_contiguous()) refuse("workspace", "has to be contiguous");
        return answer(entry.logprobs(type_of(x.scalar_type(), "logits"), x.data_ptr(), (size_t)stride, (size_t)rows,
                                     (uint32_t)values, ints(a[1], "tokens", rows), floats(a[2], "logprob", rows),
                                     ints(a[4], "rank", rows), floats(a[3], "entropy", rows), (uint32_t)top,
                                     top ? ints(a[5], "top_tokens", rows * top) : nullptr,
                                     top ? floats(a[6], "top_logprobs", rows * top) : nullptr, ws.data_ptr(),
                                     (size_t)ws.nbytes(), c.error(a[8]), c.stream(a[9])),
                      "fyb_logprobs");
    });
}

// Addresses of the C entry points, in the order of `entry`.
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    return guarded(n, 10, [&]() -> PyObject * {
        void **e = reinterpret_cast<void **>(&entry);
        for (int i = 0; i < 10; ++i) {
            e[i] = PyLong_AsVoidPtr(a[i]);
            if (PyErr_Occurred()) throw Refused();
        }
        Py_RETURN_NONE;
    });
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(kv_blocks), METHOD(kv_release), METHOD(rope), METHOD(append), METHOD(read),
                         METHOD(attention), METHOD(append4), METHOD(read4), METHOD(attention4), METHOD(logprobs), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) { return PyModule_Create(&module); }
