// Python -> C calls of the decode and prefill path without ctypes.
//
// A decode step of a small batch is a few dozen kernels of a few microseconds each, so what Python spends per call is
// what the GPU waits for: through ctypes one Engine.decode_layer call cost 8.4 us of host time (attribute look-ups of
// four tensors, the stream object, argument conversion), of which the launch itself is about 2.  Here a call is one
// METH_FASTCALL function that reads tensors and the current stream through torch's C++ interface and calls the library
// function with the interpreter lock released, as ctypes does.
//
// Every function is made by one template from the declaration in triebwerk_b200.h: pointer parameters take a tensor
// (CUDA, contiguous), None or an address, int parameters a number; a trailing tq_stream_t is torch's current stream.
// They return the status (launchers: that of tq_last_compat_status()).  No C++ exception leaves them.
//
// The calls over paged caches take shapes and strides from the tensors themselves: each has a function that checks them
// (types, sizes, the current device) and makes the C call.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <exception>
#include <tuple>
#include <type_traits>
#include <utility>

#include "../../include/triebwerk_b200.h"

namespace {

// What the tensors of a call must be beside CUDA and contiguous.
enum class Need { Any, Half };

bool tensor_address(PyObject* o, Need need, void** out) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || !t.is_contiguous() || (need == Need::Half && t.scalar_type() != at::kHalf)) {
        PyErr_SetString(PyExc_AssertionError, need == Need::Half ? "device, contiguous fp16 tensors only" : "device, contiguous tensors only");
        return false;
    }
    *out = t.data_ptr();
    return true;
}

template <typename T>
bool convert(PyObject* o, Need need, T* out) {
    if constexpr (std::is_pointer_v<T>) {
        void* p = nullptr;
        if (THPVariable_Check(o)) {
            if (!tensor_address(o, need, &p)) return false;
        } else if (o != Py_None) {
            p = PyLong_AsVoidPtr(o);
            if (PyErr_Occurred()) return false;
        }
        *out = (T)p;
        return true;
    } else {
        const long long v = PyLong_AsLongLong(o);
        if (v == -1 && PyErr_Occurred()) return false;
        *out = (T)v;
        return true;
    }
}

template <auto Fn, Need need>
struct Call;

template <typename R, typename... A, R (*Fn)(A...), Need need>
struct Call<Fn, need> {
    static constexpr size_t N = sizeof...(A) - 1;  // the last parameter is the stream

    template <size_t... I>
    static PyObject* go(PyObject* const* args, std::index_sequence<I...>) {
        std::tuple<std::decay_t<A>...> v{};
        try {
            if (!(convert(args[I], need, &std::get<I>(v)) && ...)) return nullptr;
            std::get<N>(v) = (tq_stream_t)c10::cuda::getCurrentCUDAStream().stream();
        } catch (const std::exception& e) {  // torch throws: a machine without a GPU, a tensor without memory of its own
            PyErr_SetString(PyExc_RuntimeError, e.what());
            return nullptr;
        }
        int status = 0;
        Py_BEGIN_ALLOW_THREADS
        try {
            if constexpr (std::is_void_v<R>) {
                std::apply(Fn, v);
                status = tq_last_compat_status();
            } else {
                status = std::apply(Fn, v);
            }
        } catch (const std::exception&) {  // (the library's own containers)
            status = TQ_ERR_NOMEM;
        }
        Py_END_ALLOW_THREADS
        return PyLong_FromLong(status);
    }
    static PyObject* py(PyObject*, PyObject* const* args, Py_ssize_t n) {
        if (n != (Py_ssize_t)N) {
            PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", (Py_ssize_t)N, n);
            return nullptr;
        }
        return go(args, std::make_index_sequence<N>{});
    }
};

// ---- paged caches -------------------------------------------------------------------------------------------------------
struct Refused {
    const char* what;
};
void need(bool ok, const char* what) {
    if (!ok) throw Refused{what};
}
// Argument i as a tensor of `type` on the current device; an empty one for None where that is allowed.
struct Args {
    PyObject* const* a;
    int device;
    const at::Tensor& tensor(int i, at::ScalarType type, const char* what) const {
        need(THPVariable_Check(a[i]), what);
        const at::Tensor& t = THPVariable_Unpack(a[i]);
        need(t.is_cuda() && t.device().index() == device, "tensors on the current CUDA device only");
        need(t.scalar_type() == type, what);
        return t;
    }
    // contiguous, of n elements (or any number: n < 0)
    const at::Tensor& flat(int i, at::ScalarType type, long long n, const char* what) const {
        const at::Tensor& t = tensor(i, type, what);
        need(t.is_contiguous() && (n < 0 || t.numel() == n), what);
        return t;
    }
    int number(int i) const {
        const long long v = PyLong_AsLongLong(a[i]);
        need(!(v == -1 && PyErr_Occurred()) && v >= INT_MIN && v <= INT_MAX, "a whole number of 32 bits");
        return (int)v;
    }
};
// Rows of a 2-D tensor whose elements lie side by side: how far apart they begin.
int row_stride(const at::Tensor& t, const char* what) {
    need(t.dim() == 2 && (t.numel() == 0 || t.size(1) <= 1 || t.stride(1) == 1), what);  // (an empty one may have any strides)
    const long long s = t.size(0) <= 1 ? std::max<long long>(t.size(1), 1) : t.stride(0);
    need(s >= t.size(1) && s <= INT_MAX && t.size(0) <= INT_MAX, what);
    return (int)s;
}
template <typename Body>
PyObject* paged_call(PyObject* const* args, Py_ssize_t n, Py_ssize_t wanted, Body body) {
    if (n != wanted) {
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", wanted, n);
        return nullptr;
    }
    try {
        const Args a{args, (int)c10::cuda::current_device()};
        return PyLong_FromLong(body(a, (tq_stream_t)c10::cuda::getCurrentCUDAStream().stream()));
    } catch (const Refused& r) {
        PyErr_Clear();
        PyErr_SetString(PyExc_AssertionError, r.what);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}
template <typename Call>
int unlocked(Call call) {
    int status = 0;
    Py_BEGIN_ALLOW_THREADS
    try {
        status = call();
    } catch (const std::exception&) {
        status = TQ_ERR_NOMEM;
    }
    Py_END_ALLOW_THREADS
    return status;
}

PyObject* page_plan(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return paged_call(args, n, 12, [](const Args& a, tq_stream_t s) {
        const at::Tensor& table = a.tensor(0, at::kInt, "block_table: int32 [requests, pages]");
        const int stride = row_stride(table, "block_table: int32 [requests, pages], rows of neighbouring elements");
        const int G = (int)table.size(0), width = (int)table.size(1);
        const at::Tensor& stack = a.flat(1, at::kInt, -1, "free_pages: int32, contiguous");
        need(stack.numel() <= INT_MAX, "free_pages: fewer than 2^31");
        int* const count = a.flat(2, at::kInt, 1, "free_count: int32 [1]").data_ptr<int>();
        int* const count_out = a.flat(3, at::kInt, 1, "free_count_out: int32 [1]").data_ptr<int>();
        int* const context = a.flat(4, at::kInt, G, "context_lens: int32 [requests]").data_ptr<int>();
        int* const fresh = a.flat(5, at::kInt, G, "new_tokens: int32 [requests]").data_ptr<int>();
        const unsigned char* ended = nullptr;
        if (a.a[6] != Py_None) {
            need(THPVariable_Check(a.a[6]), "finished: bool or uint8 [requests], or None");
            const bool flag = THPVariable_Unpack(a.a[6]).scalar_type() == at::kBool;
            ended = (const unsigned char*)a.flat(6, flag ? at::kBool : at::kByte, G, "finished: bool or uint8 [requests], or None").data_ptr();
        }
        const int page_size = a.number(7);
        int* const lens = a.flat(8, at::kInt, G, "seq_lens: int32 [requests]").data_ptr<int>();
        int* const start = a.flat(9, at::kInt, G + 1ll, "query_start: int32 [requests + 1]").data_ptr<int>();
        const at::Tensor& slots = a.flat(10, at::kLong, -1, "slots: int64, contiguous");
        need(slots.numel() <= INT_MAX, "slots: fewer than 2^31");
        int* positions = nullptr;
        if (a.a[11] != Py_None) positions = a.flat(11, at::kInt, slots.numel(), "positions: int32, as many as slots, or None").data_ptr<int>();
        int* const t = table.data_ptr<int>();
        int* const f = stack.data_ptr<int>();
        long long* const sl = (long long*)slots.data_ptr();
        return unlocked([&] {
            return tq_page_plan(t, stride, width, f, count, count_out, (int)stack.numel(), page_size, context, fresh, ended, G, lens, start, sl, positions,
                                (int)slots.numel(), s);
        });
    });
}

// The four cache arrays from argument i on: codes and norms of K, codes and norms of V (in the order that `order` names).
struct CacheArgs {
    uint8_t *ck, *cv;
    void *kn, *vn;
    long long rows;
};
CacheArgs cache_arrays(const Args& a, int ck, int kn, int cv, int vn, int Hkv, int bits) {
    need(Hkv > 0 && (bits == 2 || bits == 4), "num_kv_heads above 0, bits 2 or 4");
    CacheArgs c{};
    auto array = [&](int i, at::ScalarType type, long long row, const char* what) {
        const at::Tensor& t = a.flat(i, type, -1, what);
        need(t.dim() == 2 && t.size(1) == row && (c.rows == 0 || t.size(0) == c.rows) && t.size(0) > 0, what);
        c.rows = t.size(0);
        return t.data_ptr();
    };
    c.ck = (uint8_t*)array(ck, at::kByte, Hkv * 16ll * bits, "K codes: uint8 [rows, num_kv_heads * 16 * bits], contiguous");
    c.cv = (uint8_t*)array(cv, at::kByte, Hkv * 16ll * bits, "V codes: as K's");
    c.kn = array(kn, at::kHalf, Hkv, "K norms: fp16 [rows, num_kv_heads], contiguous");
    c.vn = array(vn, at::kHalf, Hkv, "V norms: as K's");
    return c;
}
const void* rotation_of(const Args& a, int i) { return a.flat(i, at::kHalf, 128 * 128, "rotation: fp16 [128, 128]").data_ptr(); }

// k, v [T, num_kv_heads * 128] with one stride, slots [T]
template <auto Fn, int First, int Cache>  // First: argument of k; Cache: of the K codes
PyObject* paged_rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return paged_call(args, n, 10, [](const Args& a, tq_stream_t s) {
        const int Hkv = a.number(8), bits = a.number(9);
        const CacheArgs c = cache_arrays(a, Cache, Cache + 1, Cache + 2, Cache + 3, Hkv, bits);
        const at::Tensor& k = a.tensor(First, at::kHalf, "K: fp16 [tokens, num_kv_heads * 128]");
        const at::Tensor& v = a.tensor(First + 1, at::kHalf, "V: fp16 [tokens, num_kv_heads * 128]");
        const int ks = row_stride(k, "K: fp16 [tokens, num_kv_heads * 128], rows of neighbouring elements"), vs = row_stride(v, "V: as K");
        const int T = (int)k.size(0);
        need(k.size(1) == Hkv * 128ll && v.size(1) == k.size(1) && v.size(0) == T && (T <= 1 || ks == vs), "K and V: [tokens, num_kv_heads * 128], one stride for both");
        const void* const R = rotation_of(a, 6);
        const long long* const slots = (const long long*)a.flat(7, at::kLong, T, "slots: int64 [tokens]").data_ptr();
        void* const kp = k.data_ptr();
        void* const vp = v.data_ptr();
        return unlocked([&] {
            if constexpr (First == 4) return Fn(c.ck, c.kn, c.cv, c.vn, kp, vp, R, slots, c.rows, T, Hkv, 128, ks, bits, s);
            else return Fn(kp, vp, c.ck, c.kn, c.cv, c.vn, R, slots, c.rows, T, Hkv, 128, ks, bits, s);
        });
    });
}

struct AttentionArgs {
    CacheArgs c;
    const void *q, *R;
    void *out, *ws;
    const int *table, *lens;
    int T, G, stride, width, q_stride, out_stride, H, Hkv, bits, page, pages;
    size_t ws_bytes;
};
// out, q, ck, cv, kn, vn, rotation, block_table, seq_lens, then from `at` on: page_size, num_heads, num_kv_heads, bits, workspace
AttentionArgs attention_args(const Args& a, int at) {
    AttentionArgs p{};
    p.page = a.number(at); p.H = a.number(at + 1); p.Hkv = a.number(at + 2); p.bits = a.number(at + 3);
    need(p.H > 0 && p.page > 0, "num_heads and page_size above 0");
    p.c = cache_arrays(a, 2, 4, 3, 5, p.Hkv, p.bits);
    need(p.c.rows % p.page == 0 && p.c.rows / p.page <= INT_MAX, "cache arrays: whole pages");
    p.pages = (int)(p.c.rows / p.page);
    const at::Tensor& out = a.tensor(0, at::kHalf, "out: fp16 [tokens, num_heads * 128]");
    const at::Tensor& q = a.tensor(1, at::kHalf, "q: fp16 [tokens, num_heads * 128]");
    p.q_stride = row_stride(q, "q: fp16 [tokens, num_heads * 128], rows of neighbouring elements");
    p.out_stride = row_stride(out, "out: fp16 [tokens, num_heads * 128], rows of neighbouring elements");
    p.T = (int)q.size(0);
    need(q.size(1) == p.H * 128ll && out.size(1) == q.size(1) && out.size(0) == p.T, "q and out: [tokens, num_heads * 128]");
    p.q = q.data_ptr();
    p.out = out.data_ptr();
    p.R = rotation_of(a, 6);
    const at::Tensor& table = a.tensor(7, at::kInt, "block_table: int32 [requests, pages]");
    p.stride = row_stride(table, "block_table: int32 [requests, pages], rows of neighbouring elements");
    p.G = (int)table.size(0);
    p.width = (int)table.size(1);
    p.table = table.data_ptr<int>();
    p.lens = a.flat(8, at::kInt, p.G, "seq_lens: int32 [requests]").data_ptr<int>();
    const at::Tensor& ws = a.flat(at + 4, at::kByte, -1, "workspace: uint8, contiguous");
    p.ws = ws.data_ptr();
    p.ws_bytes = (size_t)ws.numel();
    return p;
}
PyObject* paged_decode_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return paged_call(args, n, 14, [](const Args& a, tq_stream_t s) {
        const AttentionArgs p = attention_args(a, 9);
        need(p.T == p.G, "one query token per row of the block table");
        return unlocked([&] {
            return tq_paged_decode_attention(p.out, p.q, p.c.ck, p.c.cv, p.c.kn, p.c.vn, p.R, p.table, p.stride, p.width, p.lens, p.pages, p.page, p.G, p.H,
                                             p.Hkv, 128, p.q_stride, p.out_stride, p.bits, p.ws, p.ws_bytes, s);
        });
    });
}

PyObject* paged_prefill_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return paged_call(args, n, 15, [](const Args& a, tq_stream_t s) {
        const AttentionArgs p = attention_args(a, 10);
        const int* const start = a.flat(9, at::kInt, p.G + 1ll, "query_start: int32 [requests + 1]").data_ptr<int>();
        return unlocked([&] {
            return tq_paged_prefill_attention(p.out, p.q, p.c.ck, p.c.cv, p.c.kn, p.c.vn, p.R, p.table, p.stride, p.width, p.lens, start, p.pages, p.page, p.T,
                                              p.G, p.H, p.Hkv, 128, p.q_stride, p.out_stride, p.bits, p.ws, p.ws_bytes, s);
        });
    });
}

#define TQ_CALL(name, need) {#name, (PyCFunction)(void (*)(void))Call<&name, need>::py, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    TQ_CALL(tq_engine_decode_layer, Need::Half),
    TQ_CALL(tq_engine_decode_step, Need::Half),
    TQ_CALL(tq_engine_prefill_layer, Need::Half),
    TQ_CALL(tq_engine_prefill_layer_batch, Need::Half),
    TQ_CALL(tq_engine_prefill_append, Need::Any),
    TQ_CALL(tq_engine_prefill_append_batch, Need::Any),
    TQ_CALL(launch_turbo_kv_quantize, Need::Any),
    TQ_CALL(launch_turbo_kv_quantize_batch, Need::Any),
    TQ_CALL(launch_turbo_gqa_attention_batch, Need::Any),
    TQ_CALL(launch_turbo_gqa_attention, Need::Any),
    TQ_CALL(launch_turbo_gqa_prefill_attention, Need::Any),
    TQ_CALL(launch_kv_cache_write_batch, Need::Any),
    TQ_CALL(launch_gqa_attention_batch, Need::Any),
    TQ_CALL(launch_gqa_attention, Need::Any),
    TQ_CALL(launch_gqa_prefill_attention, Need::Any),
    {"page_plan", (PyCFunction)(void (*)(void))page_plan, METH_FASTCALL, nullptr},
    {"paged_append", (PyCFunction)(void (*)(void))paged_rows<&tq_paged_append, 4, 0>, METH_FASTCALL, nullptr},
    {"paged_read", (PyCFunction)(void (*)(void))paged_rows<&tq_paged_read, 0, 2>, METH_FASTCALL, nullptr},
    {"paged_prefill_attention", (PyCFunction)(void (*)(void))paged_prefill_attention, METH_FASTCALL, nullptr},
    {"paged_decode_attention", (PyCFunction)(void (*)(void))paged_decode_attention, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hostcall", "Library calls on tensors and the current stream.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__hostcall(void) { return PyModule_Create(&module); }
