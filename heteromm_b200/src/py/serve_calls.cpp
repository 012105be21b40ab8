// serve_calls.cpp — the serving entry points called with torch tensors: checks of the
// arguments, outputs and scratch memory from torch's allocator, the current stream, the
// call.  A serving step makes a call per layer, on the host's critical path when few
// tokens are decoded: through ctypes and checks in Python a call took 21 us of the host
// (6.5 of them the two launches), more than the kernels of a small step; here 8.
//
// Positional arguments only, in the order that serve.py documents and passes.  The C entry
// points come as addresses (bind), so that the library is the one that _abi loads.
#include <Python.h>

#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <ATen/ops/empty.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <sstream>
#include <utility>

#include "heteromm_cuda.h"

namespace {

using at::ScalarType;
using at::Tensor;

// ------------------------------------------------------------ the C library

struct Entry {
    decltype(&hmm_paged_kv_append) append;
    decltype(&hmm_paged_attention) attention;
    decltype(&hmm_paged_attention_workspace_size) attention_workspace;
    decltype(&hmm_paged_state_workspace_size) state_workspace;
    decltype(&hmm_paged_copy_pages) copy;
    decltype(&hmm_paged_free) free;
    decltype(&hmm_paged_fork) fork;
    decltype(&hmm_paged_grow) grow;
    decltype(&hmm_paged_compact) compact;
    decltype(&hmm_status_read) status_read;
    decltype(&hmm_paged_quant_append) quant_append;
    decltype(&hmm_paged_quant_read) quant_read;
    decltype(&hmm_paged_quant_attention) quant_attention;
    decltype(&hmm_paged_quant_window_attention_workspace_size) quant_attention_workspace;
    decltype(&hmm_paged_prefix_attention) prefix_attention;
    decltype(&hmm_paged_prefix_attention_workspace_size) prefix_attention_workspace;
    decltype(&hmm_paged_quant_prefix_attention) quant_prefix_attention;
    decltype(&hmm_paged_quant_prefix_attention_workspace_size) quant_prefix_attention_workspace;
};
Entry hmm_fn{};
PyObject* raise_error = nullptr;   // (entry point's name, status): raises HmmError

// (addresses in Entry's order, raise)
PyObject* bind(PyObject*, PyObject* args) {
    PyObject *addresses, *raise;
    if (!PyArg_ParseTuple(args, "O!O", &PyTuple_Type, &addresses, &raise)) return nullptr;
    constexpr Py_ssize_t n = sizeof(Entry) / sizeof(void*);
    void* p[n];
    if (PyTuple_GET_SIZE(addresses) != n) {
        PyErr_Format(PyExc_ValueError, "%zd addresses, not %zd", n, PyTuple_GET_SIZE(addresses));
        return nullptr;
    }
    for (Py_ssize_t i = 0; i < n; ++i) {
        p[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(addresses, i));
        if (!p[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a null address");
            return nullptr;
        }
    }
    memcpy(&hmm_fn, p, sizeof hmm_fn);
    Py_INCREF(raise);
    raise_error = raise;
    Py_RETURN_NONE;
}

// Raises what a C entry point answered.
void check(hmm_status_t s, const char* name) {
    if (s == HMM_OK) return;
    PyObject* r = PyObject_CallFunction(raise_error, "si", name, (int)s);
    Py_XDECREF(r);
    throw python_error();
}

// A C entry point without the interpreter's lock: a launch waits when the stream's queue is full.
template <typename F>
hmm_status_t unlocked(F&& f) {
    hmm_status_t s;
    Py_BEGIN_ALLOW_THREADS s = f();
    Py_END_ALLOW_THREADS return s;
}

// ------------------------------------------------------------ arguments

// A refusal, raised as `type`.
struct Refused : torch::PyTorchError {
    PyObject* type;
    template <typename... A>
    Refused(PyObject* type, const char* fmt, const A&... args) : type(type) {
        char text[512];
        if constexpr (sizeof...(A) == 0) {
            msg = fmt;
        } else {
            snprintf(text, sizeof text, fmt, args...);
            msg = text;
        }
    }
    PyObject* python_type() override { return type; }
};
template <typename... A>
Refused value_error(const char* fmt, const A&... args) { return Refused(PyExc_ValueError, fmt, args...); }
template <typename... A>
Refused type_error(const char* fmt, const A&... args) { return Refused(PyExc_TypeError, fmt, args...); }

std::string name_of(ScalarType t) { return std::string("torch.") + torch::getTHPDtype(t)->name; }

const Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

const Tensor& on_gpu(PyObject* o, const char* name) {
    const Tensor* t = tensor(o);
    if (!t || !t->is_cuda()) throw value_error("%s must be a CUDA tensor", name);
    return *t;
}

const Tensor& typed(PyObject* o, const char* name, ScalarType dtype, int dev) {
    const Tensor& t = on_gpu(o, name);
    if (t.scalar_type() != dtype)
        throw type_error("%s must be %s, got %s", name, name_of(dtype).c_str(),
                               name_of(t.scalar_type()).c_str());
    if (t.get_device() != dev)
        throw value_error("%s is on cuda:%d, the others are on cuda:%d", name, (int)t.get_device(), dev);
    return t;
}

void shaped(const Tensor& t, const char* name, at::IntArrayRef shape) {
    if (t.sizes() == shape) return;
    std::ostringstream need, got;
    need << shape;
    got << t.sizes();
    throw value_error("%s must be %s, got %s", name, need.str().c_str(), got.str().c_str());
}

// A contiguous tensor of this dtype, device and (where given) shape.
const Tensor& dense(PyObject* o, const char* name, ScalarType dtype, int dev) {
    const Tensor& t = typed(o, name, dtype, dev);
    if (!t.is_contiguous()) throw value_error("%s must be contiguous", name);
    return t;
}
const Tensor& dense(PyObject* o, const char* name, ScalarType dtype, int dev, at::IntArrayRef shape) {
    const Tensor& t = dense(o, name, dtype, dev);
    shaped(t, name, shape);
    return t;
}
const int32_t* ints(PyObject* o, const char* name, int dev, at::IntArrayRef shape) {
    return (const int32_t*)dense(o, name, at::kInt, dev, shape).data_ptr();
}
const Tensor& int_vector(PyObject* o, const char* name, int dev) {
    const Tensor& t = dense(o, name, at::kInt, dev);
    if (t.dim() != 1) throw value_error("%s must be a vector", name);
    return t;
}

int64_t whole(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
double real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}

// Packed rows [n_tokens, heads, D]: strides in elements.
struct Rows {
    void* p = nullptr;
    int64_t token = 0, head = 0;
};

Rows rows(PyObject* o, const char* name, ScalarType dtype, int dev, at::IntArrayRef shape) {
    const Tensor& t = typed(o, name, dtype, dev);
    shaped(t, name, shape);
    if (t.stride(2) != 1 && shape[2] > 1) throw value_error("%s: the last dimension must be contiguous", name);
    return Rows{t.data_ptr(), t.stride(0), t.stride(1)};
}

struct Cache {
    hmm_paged_cache_t c;
    ScalarType dtype;
    int dev;
};

struct Four {
    int64_t n[4], st[4];
};

Four four(const Tensor& t, const char* name) {
    Four f;
    if (t.dim() == 3) {   // one head
        f = Four{{t.size(0), 1, t.size(1), t.size(2)},
                 {t.stride(0), t.size(1) * t.stride(1), t.stride(1), t.stride(2)}};
    } else if (t.dim() == 4) {
        for (int i = 0; i < 4; ++i) {
            f.n[i] = t.size(i);
            f.st[i] = t.stride(i);
        }
    } else {
        throw value_error("%s must be [n_pages, n_kv_heads, page_tokens, D]", name);
    }
    if (f.st[3] != 1 && f.n[3] > 1) throw value_error("%s: the last dimension must be contiguous", name);
    return f;
}

int32_t code_of(ScalarType t, const char* name) {   // int16: bf16 bit patterns
    if (t == at::kBFloat16 || t == at::kShort) return HMM_DTYPE_BF16;
    if (t == at::kHalf) return HMM_DTYPE_F16;
    throw type_error("%s must be bfloat16, float16 or int16 (bf16 bits), got %s", name, name_of(t).c_str());
}

Cache cache(PyObject* k_pages, PyObject* v_pages) {
    const Tensor &k = on_gpu(k_pages, "k_pages"), &v = on_gpu(v_pages, "v_pages");
    const Four a = four(k, "k_pages"), b = four(v, "v_pages");
    const int32_t code = code_of(k.scalar_type(), "k_pages");
    if (!std::equal(a.n, a.n + 4, b.n) || v.scalar_type() != k.scalar_type() || v.get_device() != k.get_device())
        throw value_error("k_pages and v_pages differ in shape, dtype or device");
    return Cache{{k.data_ptr(), v.data_ptr(), a.n[0], a.n[1], a.n[2], a.n[3], a.st[0], a.st[1], a.st[2], b.st[0],
                  b.st[1], b.st[2], code},
                 k.scalar_type(), (int)k.get_device()};
}

// A cache held in 8 bits: [n_pages, n_kv_heads, page_tokens, D + D / 32], a block per page and head.
struct QuantCache {
    hmm_paged_quant_t c;
    int dev;
};

QuantCache quant_cache(PyObject* k_pages, PyObject* v_pages) {
    const Tensor &k = on_gpu(k_pages, "k_pages"), &v = on_gpu(v_pages, "v_pages");
    const ScalarType t = k.scalar_type();
    if (t != at::kFloat8_e4m3fn && t != at::kChar)
        throw type_error("k_pages must be float8_e4m3fn or int8, got %s", name_of(t).c_str());
    if (v.scalar_type() != t || v.sizes() != k.sizes() || v.get_device() != k.get_device())
        throw value_error("k_pages and v_pages differ in shape, dtype or device");
    const Four a = four(k, "k_pages"), b = four(v, "v_pages");
    if (a.n[3] == 0 || a.n[3] % 33 != 0)
        throw value_error("k_pages must be [n_pages, n_kv_heads, page_tokens, D + D / 32], got rows of %d", (int)a.n[3]);
    for (const Four* f : {&a, &b})
        if (f->n[2] > 1 && f->st[2] != f->n[3])
            throw value_error("%s: a page and head must be one block of memory", f == &a ? "k_pages" : "v_pages");
    return QuantCache{{k.data_ptr(), v.data_ptr(), a.n[0], a.n[1], a.n[2], a.n[3] / 33 * 32, a.st[0], a.st[1], b.st[0],
                       b.st[1], t == at::kChar ? HMM_DTYPE_I8 : HMM_DTYPE_E4M3},
                      (int)k.get_device()};
}

// What the checks ask of a cache whose vectors are of this type, the one of `name`.
Cache of_quant(const QuantCache& q, ScalarType dtype, const char* name) {
    Cache c{};
    c.c.n_kv_heads = q.c.n_kv_heads;
    c.c.D = q.c.D;
    c.c.dtype = code_of(dtype, name);
    c.dtype = dtype;
    c.dev = q.dev;
    return c;
}

const Tensor& page_table(PyObject* o, int dev) {
    const Tensor& t = dense(o, "page_table", at::kInt, dev);
    if (t.dim() != 2) throw value_error("page_table must be [n_seq, pages_per_seq]");
    return t;
}

hmm_paged_batch_t batch(PyObject* table, PyObject* cu_new, PyObject* kv_len, int64_t n_tokens, int dev) {
    const Tensor& t = page_table(table, dev);
    const int64_t n = t.size(0);
    return hmm_paged_batch_t{(const int32_t*)t.data_ptr(), n, t.size(1), ints(cu_new, "cu_new", dev, {n + 1}),
                             n_tokens, ints(kv_len, "kv_len", dev, {n})};
}

// ------------------------------------------------------------ memory, stream, status

Tensor empty(at::IntArrayRef shape, ScalarType dtype, int dev) {
    return at::empty(shape, at::TensorOptions(dtype).device(at::kCUDA, (at::DeviceIndex)dev));
}

// Scratch memory for this call: the allocator hands it on in the stream's order, and to a
// graph from its pool.
c10::DataPtr scratch(size_t bytes) { return c10::cuda::CUDACachingAllocator::get()->allocate(std::max<size_t>(bytes, 16)); }

// The caller's status word; or with None one of the call's own, which it waits for.
struct Status {
    int32_t* p;
    bool waits;
    c10::DataPtr own;
};

Status status_word(PyObject* o, int dev, cudaStream_t st) {
    if (o == Py_None) {
        c10::DataPtr own = scratch(4);
        int32_t* p = (int32_t*)own.get();
        C10_CUDA_CHECK(cudaMemsetAsync(p, 0, 4, st));
        return Status{p, true, std::move(own)};
    }
    const Tensor& t = typed(o, "status", at::kInt, dev);
    if (t.numel() == 0) throw value_error("status must hold a value");
    return Status{(int32_t*)t.data_ptr(), false, {}};
}

void finish(hmm_status_t s, const char* name, const Status& status, cudaStream_t st) {
    check(s, name);
    if (status.waits) check(unlocked([&] { return hmm_fn.status_read(status.p, st); }), name);
}

// The first argument that is a CUDA tensor decides the device; the checks do the rest.
struct Place {
    c10::cuda::OptionalCUDAGuard guard;
    cudaStream_t stream;
    explicit Place(int dev) {
        if (dev != c10::cuda::current_device()) guard.set_index((c10::DeviceIndex)dev);
        stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    }
};

void arguments(Py_ssize_t got, Py_ssize_t need) {
    if (got != need) throw type_error("%d arguments, not %d", (int)need, (int)got);
}

// ------------------------------------------------------------ entry points

// q, k_pages, v_pages, page_table, cu_new, kv_len, causal, window, sinks, scale, max_new,
// return_lse, out, status
// (QUANT: over a cache held in 8 bits)
template <bool QUANT>
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    arguments(n_args, 14);
    const Tensor& q = on_gpu(a[0], "q");
    QuantCache qc{};
    const Cache c = QUANT ? of_quant(qc = quant_cache(a[1], a[2]), q.scalar_type(), "q") : cache(a[1], a[2]);
    if (q.dim() != 3) throw value_error("q must be [n_tokens, n_heads, D]");
    const int64_t n_tokens = q.size(0), heads = q.size(1), d = q.size(2);
    if (d != c.c.D) throw value_error("q has heads of %d, the cache of %d", (int)d, (int)c.c.D);
    const Rows qr = rows(a[0], "q", c.dtype, c.dev, q.sizes());
    const hmm_paged_batch_t b = batch(a[3], a[4], a[5], n_tokens, c.dev);
    const bool with_lse = truth(a[11]), causal = truth(a[6]);
    const int64_t window = whole(a[7]), sinks = whole(a[8]), max_new = whole(a[10]);
    const float scale = a[9] == Py_None ? (float)std::pow((double)d, -0.5) : (float)real(a[9]);
    const Place at(c.dev);
    Tensor out = a[12] == Py_None ? empty(q.sizes(), c.dtype, c.dev) : dense(a[12], "out", c.dtype, c.dev, q.sizes());
    Tensor lse;
    if (with_lse) lse = empty({n_tokens, heads}, at::kFloat, c.dev);
    const Status status = status_word(a[13], c.dev, at.stream);
    const size_t bytes = QUANT ? hmm_fn.quant_attention_workspace(b.n_seq, n_tokens, heads, c.c.n_kv_heads, d,
                                                                  b.pages_per_seq * qc.c.page_tokens, max_new, window)
                               : hmm_fn.attention_workspace(b.n_seq, n_tokens, heads, c.c.n_kv_heads, d);
    const c10::DataPtr ws = scratch(bytes);
    finish(unlocked([&] {
               if constexpr (QUANT)
                   return hmm_fn.quant_attention(&qc.c, &b, c.c.dtype, qr.p, qr.token, qr.head, heads, scale, causal, window,
                                                 sinks, max_new, out.data_ptr(), with_lse ? lse.data_ptr<float>() : nullptr,
                                                 status.p, ws.get(), bytes, at.stream);
               return hmm_fn.attention(&c.c, &b, qr.p, qr.token, qr.head, heads, scale, causal, window, sinks, max_new,
                                       out.data_ptr(), with_lse ? lse.data_ptr<float>() : nullptr, status.p, ws.get(),
                                       bytes, at.stream);
           }),
           QUANT ? "hmm_paged_quant_attention" : "hmm_paged_attention", status, at.stream);
    if (!with_lse) return THPVariable_Wrap(std::move(out));
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(lse)));
    END_HANDLE_TH_ERRORS
}

// q, k_pages, v_pages, page_table, cu_new, kv_len, cu_group, prefix_len, scale, max_new,
// return_lse, out, status; the dtype of k_pages says which cache it is
PyObject* prefix_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    arguments(n_args, 13);
    const Tensor& q = on_gpu(a[0], "q");
    const ScalarType pt = on_gpu(a[1], "k_pages").scalar_type();
    const bool quant = pt == at::kFloat8_e4m3fn || pt == at::kChar;
    QuantCache qc{};
    const Cache c = quant ? of_quant(qc = quant_cache(a[1], a[2]), q.scalar_type(), "q") : cache(a[1], a[2]);
    if (q.dim() != 3) throw value_error("q must be [n_tokens, n_heads, D]");
    const int64_t n_tokens = q.size(0), heads = q.size(1), d = q.size(2);
    if (d != c.c.D) throw value_error("q has heads of %d, the cache of %d", (int)d, (int)c.c.D);
    const Rows qr = rows(a[0], "q", c.dtype, c.dev, q.sizes());
    const hmm_paged_batch_t b = batch(a[3], a[4], a[5], n_tokens, c.dev);
    const Tensor& prefix = int_vector(a[7], "prefix_len", c.dev);
    const int64_t groups = prefix.size(0);
    const int32_t* cu_group = ints(a[6], "cu_group", c.dev, {groups + 1});
    const float scale = a[8] == Py_None ? (float)std::pow((double)d, -0.5) : (float)real(a[8]);
    if (whole(a[9]) < 0) throw value_error("max_new must be >= 0");
    const bool with_lse = truth(a[10]);
    const Place at(c.dev);
    Tensor out = a[11] == Py_None ? empty(q.sizes(), c.dtype, c.dev) : dense(a[11], "out", c.dtype, c.dev, q.sizes());
    Tensor lse;
    if (with_lse) lse = empty({n_tokens, heads}, at::kFloat, c.dev);
    float* lp = with_lse ? lse.data_ptr<float>() : nullptr;
    const Status status = status_word(a[12], c.dev, at.stream);
    const size_t bytes = quant ? hmm_fn.quant_prefix_attention_workspace(b.n_seq, n_tokens, groups, heads, c.c.n_kv_heads, d,
                                                                         b.pages_per_seq * qc.c.page_tokens)
                               : hmm_fn.prefix_attention_workspace(b.n_seq, n_tokens, groups, heads, c.c.n_kv_heads, d);
    const c10::DataPtr ws = scratch(bytes);
    const int32_t* pl = (const int32_t*)prefix.data_ptr();
    finish(unlocked([&] {
               return quant ? hmm_fn.quant_prefix_attention(&qc.c, &b, c.c.dtype, cu_group, pl, groups, qr.p, qr.token, qr.head,
                                                            heads, scale, out.data_ptr(), lp, status.p, ws.get(), bytes,
                                                            at.stream)
                            : hmm_fn.prefix_attention(&c.c, &b, cu_group, pl, groups, qr.p, qr.token, qr.head, heads, scale,
                                                      out.data_ptr(), lp, status.p, ws.get(), bytes, at.stream);
           }),
           quant ? "hmm_paged_quant_prefix_attention" : "hmm_paged_prefix_attention", status, at.stream);
    if (!with_lse) return THPVariable_Wrap(std::move(out));
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(lse)));
    END_HANDLE_TH_ERRORS
}

// q, k, v, k_pages, v_pages, page_table, cu_new, kv_len, rope, q_weight, k_weight, eps,
// interleaved, positions, out, status
// (QUANT: into a cache held in 8 bits, whose vectors are of k's type)
template <bool QUANT>
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    arguments(n_args, 16);
    const Tensor& k = on_gpu(a[1], "k");
    if (k.dim() != 3) throw value_error("k must be [n_tokens, n_kv_heads, D]");
    QuantCache qc{};
    const Cache c = QUANT ? of_quant(qc = quant_cache(a[3], a[4]), k.scalar_type(), "k") : cache(a[3], a[4]);
    const int64_t d = c.c.D, hk = c.c.n_kv_heads;
    const int64_t n_tokens = k.size(0);
    const Rows kr = rows(a[1], "k", c.dtype, c.dev, {n_tokens, hk, d}),
               vr = rows(a[2], "v", c.dtype, c.dev, {n_tokens, hk, d});
    const Place at(c.dev);
    int64_t heads = 0;
    Rows qr, outr;
    Tensor out;
    if (a[0] != Py_None) {
        const Tensor& q = on_gpu(a[0], "q");
        if (q.dim() != 3) throw value_error("q must be [n_tokens, n_heads, D]");
        heads = q.size(1);
        qr = rows(a[0], "q", c.dtype, c.dev, {n_tokens, heads, d});
        if (a[14] == Py_None) {
            out = empty({n_tokens, heads, d}, c.dtype, c.dev);
            outr = Rows{out.data_ptr(), heads * d, d};
        } else {
            outr = rows(a[14], "out", c.dtype, c.dev, {n_tokens, heads, d});
        }
    }
    const hmm_paged_batch_t b = batch(a[5], a[6], a[7], n_tokens, c.dev);
    int wdt = -1;
    const void* w[2] = {nullptr, nullptr};
    for (int i = 0; i < 2; ++i) {
        if (a[9 + i] == Py_None) continue;
        const Tensor* t = tensor(a[9 + i]);
        if (!t || (t->scalar_type() != c.dtype && t->scalar_type() != at::kFloat))
            throw type_error("norm weights must be torch.float32 or %s", name_of(c.dtype).c_str());
        const int own = t->scalar_type() == at::kFloat ? HMM_DTYPE_F32 : c.c.dtype;
        if (wdt >= 0 && own != wdt) throw type_error("q_weight and k_weight must be of one dtype");
        wdt = own;
        w[i] = dense(a[9 + i], i == 0 ? "q_weight" : "k_weight", t->scalar_type(), c.dev, {d}).data_ptr();
    }
    const float* rope = nullptr;
    int64_t n_pos = 0, rotary = 0;
    if (a[8] != Py_None) {
        const Tensor& r = dense(a[8], "rope", at::kFloat, c.dev);
        if (r.dim() != 3 || r.size(2) != 2) throw value_error("rope must be [n_pos, pairs, 2]");
        // (an array of nothing has no address, which would read as no rotation)
        if (r.numel() == 0 && n_tokens > 0) throw value_error("rope is empty; None is no rotation");
        rope = (const float*)r.data_ptr();
        n_pos = r.size(0);
        rotary = 2 * r.size(1);
    }
    const int32_t* positions = a[13] == Py_None ? nullptr : ints(a[13], "positions", c.dev, {n_tokens});
    const float eps = (float)real(a[11]);
    const bool interleaved = truth(a[12]);
    const Status status = status_word(a[15], c.dev, at.stream);
    finish(unlocked([&] {
               if constexpr (QUANT)
                   return hmm_fn.quant_append(&qc.c, &b, c.c.dtype, qr.p, qr.token, qr.head, heads, kr.p, kr.token, kr.head,
                                              vr.p, vr.token, vr.head, w[0], w[1], wdt, eps, rope, n_pos, rotary, interleaved,
                                              positions, outr.p, outr.token, outr.head, status.p, at.stream);
               return hmm_fn.append(&c.c, &b, qr.p, qr.token, qr.head, heads, kr.p, kr.token, kr.head, vr.p, vr.token,
                                    vr.head, w[0], w[1], wdt, eps, rope, n_pos, rotary, interleaved, positions, outr.p,
                                    outr.token, outr.head, status.p, at.stream);
           }),
           QUANT ? "hmm_paged_quant_append" : "hmm_paged_kv_append", status, at.stream);
    if (out.defined()) return THPVariable_Wrap(std::move(out));
    Py_INCREF(a[14]);
    return a[14];
    END_HANDLE_TH_ERRORS
}

// k_pages, v_pages, page_table, cu, kv_len, n_rows, dtype, out, status
PyObject* quant_read(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    arguments(n_args, 9);
    const QuantCache c = quant_cache(a[0], a[1]);
    const int64_t n_rows = whole(a[5]);
    if (n_rows < 0) throw value_error("n_rows must be >= 0, got %lld", (long long)n_rows);
    if (!THPDtype_Check(a[6])) throw type_error("dtype must be a torch.dtype");
    const ScalarType t = ((THPDtype*)a[6])->scalar_type;
    if (t != at::kBFloat16 && t != at::kHalf && t != at::kFloat)
        throw type_error("dtype must be torch.bfloat16, torch.float16 or torch.float32, got %s", name_of(t).c_str());
    const hmm_paged_batch_t b = batch(a[2], a[3], a[4], n_rows, c.dev);
    const Place at(c.dev);
    const int64_t shape[3] = {n_rows, c.c.n_kv_heads, c.c.D};
    THPObjectPtr out[2];
    void* p[2];
    if (a[7] == Py_None) {
        for (int i = 0; i < 2; ++i) {
            Tensor x = empty(shape, t, c.dev);
            p[i] = x.data_ptr();
            out[i] = THPObjectPtr(THPVariable_Wrap(std::move(x)));
            if (!out[i]) throw python_error();
        }
    } else {
        const THPObjectPtr list(PySequence_Tuple(a[7]));
        if (!list) throw python_error();
        if (PyTuple_GET_SIZE(list.get()) != 2) throw value_error("out must hold 2 tensors");
        for (int i = 0; i < 2; ++i) {
            out[i] = THPObjectPtr(Py_NewRef(PyTuple_GET_ITEM(list.get(), i)));
            p[i] = dense(out[i].get(), i == 0 ? "out k" : "out v", t, c.dev, shape).data_ptr();
        }
    }
    const Status status = status_word(a[8], c.dev, at.stream);
    const int dtype = t == at::kBFloat16 ? HMM_DTYPE_BF16 : t == at::kHalf ? HMM_DTYPE_F16 : HMM_DTYPE_F32;
    finish(unlocked([&] { return hmm_fn.quant_read(&c.c, &b, dtype, p[0], p[1], status.p, at.stream); }),
           "hmm_paged_quant_read", status, at.stream);
    return Py_BuildValue("(NN)", out[0].release(), out[1].release());
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------ pages

// [(n_layers,) n_pages, ...] arrays whose pages (all but the leading dimensions) are one
// block of memory; strides in bytes.
struct Pages {
    void* p;
    int64_t layers, layer, n, page, size;
};

Pages pages(const Tensor& t, const char* name) {
    const int64_t b = t.element_size(), dims = t.dim();
    if (dims < 3 || dims > 5)
        throw value_error("%s must be [(n_layers,) n_pages, (n_kv_heads,) page_tokens, D]", name);
    const int64_t lead = dims == 5;
    std::pair<int64_t, int64_t> in[4];   // (stride, size) of a page's dimensions
    int m = 0;
    for (int64_t i = 1 + lead; i < dims; ++i) {   // by stride
        int at = m++;
        for (; at > 0 && in[at - 1].first > t.stride(i); --at) in[at] = in[at - 1];
        in[at] = {t.stride(i), t.size(i)};
    }
    int64_t need = 1;
    for (int i = 0; i < m; ++i) {
        if (in[i].second == 1) continue;
        if (in[i].first != need) throw value_error("%s: a page must be one block of memory", name);
        need *= in[i].second;
    }
    return Pages{t.data_ptr(), lead ? t.size(0) : 1, lead ? t.stride(0) * b : 0, t.size(lead), t.stride(lead) * b,
                 need * b};
}

hmm_page_store_t store(PyObject* k_pages, PyObject* v_pages, int* dev) {
    const Tensor &k = on_gpu(k_pages, "k_pages"), &v = on_gpu(v_pages, "v_pages");
    const Pages a = pages(k, "k_pages"), b = pages(v, "v_pages");
    if (k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type() || k.get_device() != v.get_device())
        throw value_error("k_pages and v_pages differ in shape, dtype or device");
    *dev = (int)k.get_device();
    return hmm_page_store_t{a.p, b.p, a.n, a.size, a.layers, a.page, a.layer, b.page, b.layer};
}

// The state's old arrays and its new ones: fresh, or those of `out`.
struct State {
    hmm_paged_state_t s{};
    THPObjectPtr fresh[3];   // the result's entries (given back if a check throws here too)
    int count = 0;
    State(PyObject* table, PyObject* refs, PyObject* kv_len, PyObject* out, int dev) {
        static const char* const names[3] = {"out page_table", "out refs", "out kv_len"};
        const Tensor& t = page_table(table, dev);
        const Tensor& r = dense(refs, "refs", at::kInt, dev);
        if (r.dim() != 1) throw value_error("refs must be [n_pages]");
        const Tensor* old[3] = {&t, &r, nullptr};
        count = 2;
        if (kv_len) old[count++] = &dense(kv_len, "kv_len", at::kInt, dev, {t.size(0)});
        int32_t* to[3] = {nullptr, nullptr, nullptr};
        if (out == Py_None) {
            for (int i = 0; i < count; ++i) {
                Tensor x = empty(old[i]->sizes(), at::kInt, dev);
                to[i] = (int32_t*)x.data_ptr();
                fresh[i] = THPObjectPtr(THPVariable_Wrap(std::move(x)));
                if (!fresh[i]) throw python_error();
            }
        } else {
            const THPObjectPtr list(PySequence_Tuple(out));
            if (!list) throw python_error();
            if (PyTuple_GET_SIZE(list.get()) != count) throw value_error("out must hold %d tensors", count);
            for (int i = 0; i < count; ++i) {
                fresh[i] = THPObjectPtr(Py_NewRef(PyTuple_GET_ITEM(list.get(), i)));
                to[i] = (int32_t*)dense(fresh[i].get(), names[i], at::kInt, dev, old[i]->sizes()).data_ptr();
            }
        }
        s = hmm_paged_state_t{(const int32_t*)t.data_ptr(), (const int32_t*)r.data_ptr(),
                              kv_len ? (const int32_t*)old[2]->data_ptr() : nullptr, to[0], to[1], to[2], t.size(0),
                              t.size(1), r.size(0)};
    }
    // (page_table, refs[, kv_len][, more]); takes the references.
    PyObject* result(PyObject* more = nullptr) {
        PyObject* r = PyTuple_New(count + (more != nullptr));
        if (!r) throw python_error();
        for (int i = 0; i < count; ++i) PyTuple_SET_ITEM(r, i, fresh[i].release());
        if (more) PyTuple_SET_ITEM(r, count, more);
        return r;
    }
};

// k_pages, v_pages, src, dst, status
PyObject* copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    arguments(n_args, 5);
    int dev;
    const hmm_page_store_t p = store(a[0], a[1], &dev);
    const Tensor& src = int_vector(a[2], "src", dev);
    const int32_t* dst = ints(a[3], "dst", dev, src.sizes());
    const Place at(dev);
    const Status status = status_word(a[4], dev, at.stream);
    const c10::DataPtr ws = scratch(4);
    finish(unlocked([&] {
               return hmm_fn.copy(&p, (const int32_t*)src.data_ptr(), dst, src.size(0), status.p, ws.get(), 4,
                                  at.stream);
           }),
           "hmm_paged_copy_pages", status, at.stream);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// page_table, refs, kv_len, seqs, out, status
PyObject* free_(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    arguments(n_args, 6);
    const int dev = (int)on_gpu(a[0], "page_table").get_device();
    const Place at(dev);
    State s(a[0], a[1], a[2], a[4], dev);
    const Tensor& seqs = int_vector(a[3], "seqs", dev);
    const Status status = status_word(a[5], dev, at.stream);
    const size_t bytes = hmm_fn.state_workspace(s.s.n_seq, s.s.n_pages);
    const c10::DataPtr ws = scratch(bytes);
    finish(unlocked([&] {
               return hmm_fn.free(&s.s, (const int32_t*)seqs.data_ptr(), seqs.size(0), status.p, ws.get(), bytes,
                                  at.stream);
           }),
           "hmm_paged_free", status, at.stream);
    return s.result();
    END_HANDLE_TH_ERRORS
}

// page_table, refs, kv_len, src, dst, k_pages, v_pages, out, status
PyObject* fork_(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    arguments(n_args, 9);
    int dev;
    const hmm_page_store_t p = store(a[5], a[6], &dev);
    const int64_t page_tokens = tensor(a[5])->size(-2);
    const Place at(dev);
    State s(a[0], a[1], a[2], a[7], dev);
    const Tensor& src = int_vector(a[3], "src", dev);
    const int32_t* dst = ints(a[4], "dst", dev, src.sizes());
    const Status status = status_word(a[8], dev, at.stream);
    const size_t bytes = hmm_fn.state_workspace(s.s.n_seq, s.s.n_pages);
    const c10::DataPtr ws = scratch(bytes);
    finish(unlocked([&] {
               return hmm_fn.fork(&s.s, &p, page_tokens, (const int32_t*)src.data_ptr(), dst, src.size(0), status.p,
                                  ws.get(), bytes, at.stream);
           }),
           "hmm_paged_fork", status, at.stream);
    return s.result();
    END_HANDLE_TH_ERRORS
}

// page_table, refs, kv_len, n_new, page_tokens, out, status
PyObject* grow(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    arguments(n_args, 7);
    const int dev = (int)on_gpu(a[0], "page_table").get_device();
    const Place at(dev);
    State s(a[0], a[1], a[2], a[5], dev);
    const int32_t* n_new = ints(a[3], "n_new", dev, {s.s.n_seq});
    const int64_t page_tokens = whole(a[4]);
    const Status status = status_word(a[6], dev, at.stream);
    const size_t bytes = hmm_fn.state_workspace(s.s.n_seq, s.s.n_pages);
    const c10::DataPtr ws = scratch(bytes);
    finish(unlocked([&] { return hmm_fn.grow(&s.s, page_tokens, n_new, status.p, ws.get(), bytes, at.stream); }),
           "hmm_paged_grow", status, at.stream);
    return s.result();
    END_HANDLE_TH_ERRORS
}

// page_table, refs, k_pages, v_pages, out, status
PyObject* compact(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    arguments(n_args, 6);
    int dev;
    const hmm_page_store_t p = store(a[2], a[3], &dev);
    const Place at(dev);
    State s(a[0], a[1], nullptr, a[4], dev);
    Tensor live = empty({1}, at::kInt, dev);
    const Status status = status_word(a[5], dev, at.stream);
    const size_t bytes = hmm_fn.state_workspace(s.s.n_seq, s.s.n_pages);
    const c10::DataPtr ws = scratch(bytes);
    finish(unlocked([&] {
               return hmm_fn.compact(&s.s, &p, (int32_t*)live.data_ptr(), status.p, ws.get(), bytes, at.stream);
           }),
           "hmm_paged_compact", status, at.stream);
    PyObject* more = THPVariable_Wrap(std::move(live));
    if (!more) throw python_error();
    return s.result(more);
    END_HANDLE_TH_ERRORS
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr},
                         {"attention", FAST(attention<false>)},
                         {"append", FAST(append<false>)},
                         {"quant_append", FAST(append<true>)},
                         {"quant_read", FAST(quant_read)},
                         {"quant_attention", FAST(attention<true>)},
                         {"prefix_attention", FAST(prefix_attention)},
                         {"copy_pages", FAST(copy_pages)},
                         {"free", FAST(free_)},
                         {"fork", FAST(fork_)},
                         {"grow", FAST(grow)},
                         {"compact", FAST(compact)},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "heteromm_serve_calls", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_heteromm_serve_calls() { return PyModule_Create(&module); }
