// ztq_py.cc -- Python entry points of the decode-step operators (module ztensor_b200._step).
//
// The same checks as a Python wrapper would make, and the call of the C-ABI launcher, in one native function per operator: a
// step makes several such calls per layer, and a dozen attribute look-ups per tensor cost more than the launch itself
// (plan of a step: 11.7 us through ctypes).  Arguments come by position from ztensor_b200/kernels.py, which documents them.
// Errors: ValueError for a tensor of the wrong type, shape, layout or device, RuntimeError with the launcher's code.
#include <Python.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <sstream>
#include <string>

#include "../../include/ztq.h"

namespace {

struct Refused {
    std::string what;
};

[[noreturn]] void refuse(const char* name, const std::string& wanted, const at::Tensor& t) {
    std::ostringstream s;
    s << name << ": " << wanted << " expected, got " << t.dtype() << " " << t.sizes() << ", strides " << t.strides() << " on " << t.device();
    throw Refused{s.str()};
}

struct Call {
    PyObject* const* args;
    Py_ssize_t n;
    int device;
    Call(PyObject* const* a, Py_ssize_t count, Py_ssize_t wanted) : args(a), n(count), device(-2) {
        if (n != wanted) throw Refused{"wrong number of arguments"};
        c10::DeviceIndex d = 0;
        if (c10::cuda::GetDevice(&d) == cudaSuccess) device = d;       // else no tensor is on it
        else cudaGetLastError();
    }
    bool none(int i) const { return args[i] == Py_None; }
    long long integer(int i) const {
        const long long v = PyLong_AsLongLong(args[i]);
        if (v == -1 && PyErr_Occurred()) throw python_error();
        return v;
    }
    int small(int i, const char* name) const {
        const long long v = integer(i);
        if (v < -0x7fffffffll - 1 || v > 0x7fffffffll) throw Refused{std::string(name) + ": out of range"};
        return (int)v;
    }
    const at::Tensor& tensor(int i, const char* name) const {
        if (!THPVariable_Check(args[i])) throw Refused{std::string(name) + ": a tensor expected"};
        return THPVariable_Unpack(args[i]);
    }
    void here(const at::Tensor& t, const char* name) const {
        if (!t.is_cuda() || t.get_device() != device) refuse(name, "a tensor on the current CUDA device", t);
    }
    // A contiguous tensor of this type and these extents (rank 1 or 2 or 3); NULL for None where that is allowed.
    template <typename T>
    T* flat(int i, const char* name, at::ScalarType type, at::IntArrayRef shape, bool optional = false) const {
        if (optional && none(i)) return nullptr;
        const at::Tensor& t = tensor(i, name);
        if (t.scalar_type() != type || t.sizes() != shape || !t.is_contiguous()) {
            std::ostringstream s;
            s << "contiguous " << type << " " << shape;
            refuse(name, s.str(), t);
        }
        here(t, name);
        return static_cast<T*>(t.data_ptr());
    }
    // [tokens, heads, dim], fp16 or fp32, contiguous dim
    const at::Tensor& heads(int i, const char* name) const {
        const at::Tensor& t = tensor(i, name);
        if (t.dim() != 3 || (t.scalar_type() != at::kHalf && t.scalar_type() != at::kFloat) || t.stride(2) != 1)
            refuse(name, "float16 or float32 [tokens, heads, dim] with contiguous dim", t);
        here(t, name);
        return t;
    }
    long long extent(int i, const char* name, int d) const {
        const at::Tensor& t = tensor(i, name);
        if (t.dim() <= d) refuse(name, "more dimensions", t);
        return t.size(d);
    }
    const ZtqKvCache* cache(int i, int tensor_at) const {
        here(tensor(tensor_at, "cache"), "cache");
        return reinterpret_cast<const ZtqKvCache*>(integer(i));
    }
    cudaStream_t stream(int i) const {
        return none(i) ? c10::cuda::getCurrentCUDAStream(device).stream() : reinterpret_cast<cudaStream_t>(integer(i));
    }
};

int as_int(long long v, const char* name) {
    if (v > 0x7fffffffll) throw Refused{std::string(name) + ": too large"};
    return (int)v;
}

PyObject* done(cudaError_t e, const char* name) {
    if (e != cudaSuccess) {
        PyErr_Format(PyExc_RuntimeError, "%s kernel failed (cuda error %d)", name, (int)e);
        return nullptr;
    }
    Py_RETURN_NONE;
}

template <typename F>
PyObject* guarded(F f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Refused& r) {
        PyErr_SetString(PyExc_ValueError, r.what.c_str());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

bool is_f32(const at::Tensor& t) { return t.scalar_type() == at::kFloat; }

// ctx_len, new_len, block_table, ring, ring_state, ring_state_out, next_len, kv_len, query_start, positions, slots, status, block_size, flags, stream
PyObject* kv_plan(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&] {
        const Call c(args, count, 15);
        const long long n = c.extent(0, "ctx_len", 0), width = c.extent(2, "block_table", 1), pool = c.extent(3, "ring", 0), rows = c.extent(10, "slots", 0);
        constexpr auto I = at::kInt;
        return done(ztq_kv_plan(c.flat<int>(0, "ctx_len", I, {n}), c.flat<int>(1, "new_len", I, {n}), c.flat<int>(2, "block_table", I, {n, width}), c.flat<int>(3, "ring", I, {pool}),
                                c.flat<int>(4, "ring_state", I, {2}), c.flat<int>(5, "ring_state_out", I, {2}), c.flat<int>(6, "next_len", I, {n}), c.flat<int>(7, "kv_len", I, {n}),
                                c.flat<int>(8, "query_start", I, {n + 1}), c.flat<int>(9, "positions", I, {rows}), c.flat<int>(10, "slots", I, {rows}), c.flat<int>(11, "status", I, {n}),
                                as_int(n, "ctx_len"), as_int(width, "block_table"), c.small(12, "block_size"), as_int(pool, "ring"), as_int(rows, "slots"), c.small(13, "flags"), c.stream(14)),
                    "ztq_kv_plan");
    });
}

// q, k, v, q_out, slots, cache address, cache codes, kv_heads, head_dim, table, positions, flags, stream
PyObject* rope_append_q8(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        const Call c(args, count, 13);
        const at::Tensor &k = c.heads(1, "k"), &v = c.heads(2, "v");
        const long long n = k.size(0), heads = c.integer(7), dim = c.integer(8);
        if (k.size(1) != heads || k.size(2) != dim) refuse("k", "the cache's heads and dim", k);
        if (v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type()) refuse("v", "the shape and type of k", v);
        int flags = c.small(11, "flags") | (is_f32(k) ? ZTQ_X_F32 : 0);
        const void* q = nullptr;
        void* qo = nullptr;
        long long qs[4] = {0, 0, 0, 0}, q_heads = 0;
        if (!c.none(0)) {
            const at::Tensor &a = c.heads(0, "q"), &b = c.heads(3, "q_out");
            if (a.size(0) != n || a.size(2) != dim || a.scalar_type() != k.scalar_type()) refuse("q", "the rows, dim and type of k", a);
            if (b.sizes() != a.sizes()) refuse("q_out", "the shape of q", b);
            q = a.data_ptr();
            qo = b.data_ptr();
            qs[0] = a.stride(0); qs[1] = a.stride(1); qs[2] = b.stride(0); qs[3] = b.stride(1);
            q_heads = a.size(1);
            if (is_f32(b)) flags |= ZTQ_Y_F32;
        }
        const float* table = nullptr;
        const int* positions = nullptr;
        long long rows = 0, half = 0;
        if (!c.none(9)) {
            rows = c.extent(9, "table", 0);
            half = c.extent(9, "table", 1);
            table = c.flat<float>(9, "table", at::kFloat, {rows, half, 2});
            positions = c.flat<int>(10, "positions", at::kInt, {n});
        }
        return done(ztq_rope_append_q8(q, k.data_ptr(), v.data_ptr(), qo, qs[0], qs[1], k.stride(0), k.stride(1), v.stride(0), v.stride(1), qs[2], qs[3], as_int(n, "k"), as_int(q_heads, "q"),
                                       table, as_int(rows, "table"), as_int(2 * half, "table"), positions, c.flat<int>(4, "slots", at::kInt, {n}), c.cache(5, 6), flags, c.stream(12)),
                    "ztq_rope_append_q8");
    });
}

// cache address, cache codes, kv_heads, head_dim, slots, k_out, v_out, flags, stream
PyObject* kv_read_q8(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        const Call c(args, count, 9);
        const int first = c.none(5) ? 6 : 5;
        if (c.none(first)) throw Refused{"k_out, v_out: at least one float16 or float32 tensor expected"};
        const at::ScalarType type = c.tensor(first, first == 5 ? "k_out" : "v_out").scalar_type();
        if (type != at::kHalf && type != at::kFloat) throw Refused{"k_out, v_out: at least one float16 or float32 tensor expected"};
        const long long n = c.extent(4, "slots", 0), heads = c.integer(2), dim = c.integer(3);
        void* k = c.flat<void>(5, "k_out", type, {n, heads, dim}, true);
        void* v = c.flat<void>(6, "v_out", type, {n, heads, dim}, true);
        return done(ztq_kv_read_q8(c.cache(0, 1), c.flat<int>(4, "slots", at::kInt, {n}), as_int(n, "slots"), k, v, c.small(7, "flags") | (type == at::kFloat ? ZTQ_Y_F32 : 0), c.stream(8)),
                    "ztq_kv_read_q8");
    });
}

// q, y, query_start, kv_len, block_table, cache address, cache codes, head_dim, workspace, max_new, scale, window, flags, stream
PyObject* attn_q8(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        const Call c(args, count, 14);
        const at::Tensor &q = c.heads(0, "q"), &y = c.heads(1, "y"), &w = c.tensor(8, "workspace");
        if (q.size(2) != c.integer(7)) refuse("q", "the cache's dim", q);
        if (y.sizes() != q.sizes()) refuse("y", "the shape of q", y);
        if (!w.is_contiguous()) refuse("workspace", "a contiguous tensor", w);
        c.here(w, "workspace");
        const long long seqs = c.extent(3, "kv_len", 0), width = c.extent(4, "block_table", 1);
        const double d = PyFloat_AsDouble(args[10]);
        if (d == -1.0 && PyErr_Occurred()) throw python_error();
        const float scale = (float)d;
        unsigned bits;
        std::memcpy(&bits, &scale, 4);
        return done(ztq_attn_q8(q.data_ptr(), y.data_ptr(), q.stride(0), q.stride(1), y.stride(0), y.stride(1), as_int(q.size(0), "q"), as_int(q.size(1), "q"),
                                c.flat<int>(2, "query_start", at::kInt, {seqs + 1}), c.flat<int>(3, "kv_len", at::kInt, {seqs}), c.flat<int>(4, "block_table", at::kInt, {seqs, width}),
                                as_int(seqs, "kv_len"), as_int(width, "block_table"), c.small(9, "max_new"), c.small(11, "window"), bits, c.cache(5, 6), w.data_ptr(), w.nbytes(),
                                c.small(12, "flags") | (is_f32(q) ? ZTQ_X_F32 : 0) | (is_f32(y) ? ZTQ_Y_F32 : 0), c.stream(13)),
                    "ztq_attn_q8");
    });
}

// logits, uniform, token, logprob, temperature, top_k, top_p, min_p, flags, stream
PyObject* sample(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded([&]() -> PyObject* {
        const Call c(args, count, 10);
        const at::Tensor& x = c.tensor(0, "logits");
        if (x.dim() != 2 || (x.scalar_type() != at::kHalf && x.scalar_type() != at::kFloat) || (x.size(1) > 1 && x.stride(1) != 1))
            refuse("logits", "float16 or float32 [rows, vocab] with contiguous rows", x);
        c.here(x, "logits");
        const long long n = x.size(0);
        constexpr auto F = at::kFloat, I = at::kInt;
        return done(ztq_sample(x.data_ptr(), n > 1 ? x.stride(0) : 0, as_int(n, "logits"), as_int(x.size(1), "logits"), c.flat<float>(4, "temperature", F, {n}, true),
                               c.flat<int>(5, "top_k", I, {n}, true), c.flat<float>(6, "top_p", F, {n}, true), c.flat<float>(7, "min_p", F, {n}, true), c.flat<float>(1, "uniform", F, {n}),
                               c.flat<int>(2, "token", I, {n}), c.flat<float>(3, "logprob", F, {n}, true), c.small(8, "flags") | (is_f32(x) ? ZTQ_X_F32 : 0), c.stream(9)),
                    "ztq_sample");
    });
}

#define ENTRY(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {ENTRY(kv_plan), ENTRY(rope_append_q8), ENTRY(kv_read_q8), ENTRY(attn_q8), ENTRY(sample), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_step", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__step() { return PyModule_Create(&kModule); }
