// Python binding of the 4-bit cache's and the block tables' calls: checks torch tensors, fills the C
// ABI's argument structs and launches on torch's current stream. These calls take a few microseconds on
// the GPU, less than a Python function needs to look at its tensors; here that takes about one.
//
// The functions are the bodies of `vllm_ttkv.ops`' functions of the same purpose, which document them.
// They raise TypeError for a wrong type, ValueError for a wrong shape, stride or device, and return the
// C ABI's code, which the caller turns into its exception.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>

#include "ttkv_b200.h"

namespace {

// An argument that is refused: the Python exception is set.
struct Refused {};

[[noreturn]] void refuse(PyObject* type, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    PyErr_FormatV(type, fmt, ap);
    va_end(ap);
    throw Refused{};
}

// A tensor argument on the call's device (set by the first one).
const at::Tensor& tensor(PyObject* o, const char* name, int& dev) {
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda())
        refuse(PyExc_ValueError, "expected a CUDA tensor, got %s on the CPU: the TT-KV ops run only on the GPU (no CPU path)", name);
    const int d = t.device().index();
    if (dev < 0) dev = d;
    else if (d != dev) refuse(PyExc_ValueError, "%s is on cuda:%d, the cache or block table on cuda:%d", name, d, dev);
    return t;
}

int32_t i32(int64_t v, const char* name) {
    if (v < INT32_MIN || v > INT32_MAX) refuse(PyExc_ValueError, "%s = %lld does not fit 32 bits", name, (long long)v);
    return int32_t(v);
}

int64_t integer(PyObject* o, const char* name) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        PyObject* n = PyNumber_Index(o);
        if (!n) throw Refused{};
        const int64_t w = PyLong_AsLongLong(n);
        Py_DECREF(n);
        if (w == -1 && PyErr_Occurred()) refuse(PyExc_ValueError, "%s is out of range", name);
        return w;
    }
    return v;
}

int dtype_code(const at::Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return TTKV_F32;
        case at::kHalf: return TTKV_F16;
        case at::kBFloat16: return TTKV_BF16;
        default: refuse(PyExc_TypeError, "%s must be float32, float16 or bfloat16, got %s", name, c10::toString(t.scalar_type()));
    }
}

// The address of a contiguous 1-D tensor of at least `least` entries.
void* vector(PyObject* o, at::ScalarType dt, int64_t least, const char* name, int& dev) {
    const at::Tensor& t = tensor(o, name, dev);
    if (t.scalar_type() != dt) refuse(PyExc_TypeError, "%s must be %s, got %s", name, c10::toString(dt), c10::toString(t.scalar_type()));
    if (t.dim() != 1 || t.size(0) < least || (least > 1 && t.stride(0) != 1))
        refuse(PyExc_ValueError, "%s must be contiguous with %lld entries at least", name, (long long)least);
    return t.data_ptr();
}

// The rows of a [n, heads, d] tensor whose [heads, d] rows are contiguous (a size-1 dimension may carry
// any stride); heads < 0: any. Returns the stride between rows.
int64_t rows(const at::Tensor& t, int64_t heads, int64_t d, const char* name) {
    if (t.dim() != 3 || (heads >= 0 && t.size(1) != heads) || t.size(2) != d)
        refuse(PyExc_ValueError, "%s must be [n, heads, %lld] with its heads, got %lld dimensions", name, (long long)d, (long long)t.dim());
    const int64_t H = t.size(1);
    if (t.stride(2) != 1 || (H > 1 && t.stride(1) != d))
        refuse(PyExc_ValueError, "%s must have contiguous [heads, d] rows", name);
    if (t.size(0) < 2) return H * d;
    if (t.stride(0) < H * d) refuse(PyExc_ValueError, "%s's rows overlap", name);
    return t.stride(0);
}

int32_t* status_word(PyObject* o, int& dev) { return static_cast<int32_t*>(vector(o, at::kInt, 1, "status", dev)); }

// lay is (H, d, group, panel bytes).
ttkv_q4_cache_t cache_of(PyObject* lay, PyObject* o, int flags, int& dev) {
    if (!PyTuple_Check(lay) || PyTuple_GET_SIZE(lay) != 4) refuse(PyExc_TypeError, "a layout is (H, d, group, panel bytes)");
    int64_t v[4];
    for (int i = 0; i < 4; ++i) v[i] = integer(PyTuple_GET_ITEM(lay, i), "layout");
    const at::Tensor& t = tensor(o, "cache", dev);
    if (t.scalar_type() != at::kByte || t.dim() != 4 || !t.is_contiguous())
        refuse(PyExc_ValueError, "expected a contiguous uint8 [blocks, H, block_size/16, bytes] cache");
    if (t.size(1) != v[0] || t.size(3) != v[3] || t.size(2) < 1)
        refuse(PyExc_ValueError, "a cache [%lld, %lld, %lld, %lld] does not hold H=%lld heads in panels of %lld bytes",
               (long long)t.size(0), (long long)t.size(1), (long long)t.size(2), (long long)t.size(3), (long long)v[0], (long long)v[3]);
    ttkv_q4_cache_t c{};
    c.base = static_cast<uint8_t*>(t.data_ptr());
    c.n_blocks = t.size(0);
    c.H = i32(v[0], "H");
    c.d = i32(v[1], "d");
    c.group = i32(v[2], "group");
    c.block_size = i32(16 * t.size(2), "block size");
    c.flags = flags;
    return c;
}

void table_of(PyObject* o, int& dev, int32_t*& p, int32_t& n, int32_t& cols, int64_t& stride) {
    const at::Tensor& t = tensor(o, "block_table", dev);
    if (t.scalar_type() != at::kInt || t.dim() != 2)
        refuse(PyExc_TypeError, "block_table must be int32 [n_reqs, max_blocks], got %s of %lld dimensions",
               c10::toString(t.scalar_type()), (long long)t.dim());
    n = i32(t.size(0), "block_table rows");
    cols = i32(t.size(1), "block_table columns");
    if (t.numel() && cols > 1 && t.stride(1) != 1) refuse(PyExc_ValueError, "block_table must have unit column stride");
    stride = n > 1 ? t.stride(0) : cols;
    p = static_cast<int32_t*>(t.data_ptr());
}

// Runs the call on `dev`, which need not be the current device, and its current stream.
template <typename A>
PyObject* launch(int (*fn)(const A*), A& args, int dev) {
    const c10::cuda::OptionalCUDAGuard guard(c10::Device(c10::kCUDA, c10::DeviceIndex(dev)));
    args.stream = c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(dev)).stream();
    return PyLong_FromLong(fn(&args));
}

void arity(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) refuse(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
}

template <typename F>
PyObject* guarded(F f) {
    try {
        return f();
    } catch (const Refused&) {
        return nullptr;
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
        return nullptr;
    }
}

// (write, layout, cache, slots, k, v, status, skip_pad)
PyObject* store(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        arity(n, 8);
        int dev = -1;
        ttkv_q4_store_args_t s{};
        s.cache = cache_of(a[1], a[2], a[7] == Py_True ? TTKV_CACHE_SKIP_PAD : 0, dev);
        s.slots = static_cast<const int64_t*>(vector(a[3], at::kLong, 0, "slot_mapping", dev));
        const at::Tensor &slots = THPVariable_Unpack(a[3]), &k = tensor(a[4], "k", dev), &v = tensor(a[5], "v", dev);
        if (!slots.is_contiguous()) refuse(PyExc_ValueError, "slot_mapping must be contiguous");
        s.n = i32(slots.size(0), "tokens");
        s.k_stride = rows(k, s.cache.H, s.cache.d, "k");
        s.v_stride = rows(v, s.cache.H, s.cache.d, "v");
        if (k.size(0) < s.n || v.size(0) < s.n)
            refuse(PyExc_ValueError, "k and v hold %lld and %lld tokens for %d slot ids", (long long)k.size(0), (long long)v.size(0), s.n);
        s.k = k.data_ptr();
        s.v = v.data_ptr();
        s.k_dtype = dtype_code(k, "k");
        s.v_dtype = dtype_code(v, "v");
        s.status = status_word(a[6], dev);
        return launch(a[0] == Py_True ? ttkv_q4_write : ttkv_q4_read, s, dev);
    });
}

// Decode: (layout, cache, block_table, seq_lens, q, scale, out, status); prefill: and (q_start, q_len,
// max_q_len, max_seq_len).
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const bool prefill = n == 12;
        if (!prefill) arity(n, 8);
        int dev = -1;
        ttkv_q4_attn_args_t s{};
        s.cache = cache_of(a[0], a[1], 0, dev);
        int32_t* table;
        table_of(a[2], dev, table, s.n_reqs, s.bt_cols, s.bt_stride);
        s.block_table = table;
        s.seq_lens = static_cast<const int32_t*>(vector(a[3], at::kInt, s.n_reqs, "seq_lens", dev));
        const at::Tensor &q = tensor(a[4], "q", dev), &out = tensor(a[6], "out", dev);
        if ((q.scalar_type() != at::kHalf && q.scalar_type() != at::kBFloat16) || out.scalar_type() != q.scalar_type())
            refuse(PyExc_TypeError, "queries and outputs are both float16 or both bfloat16, got %s and %s",
                   c10::toString(q.scalar_type()), c10::toString(out.scalar_type()));
        s.q_stride = rows(q, -1, s.cache.d, "q");
        s.HQ = i32(q.size(1), "HQ");
        if (s.HQ == 0 || s.HQ % s.cache.H)
            refuse(PyExc_ValueError, "q must be [n, HQ, %d] with HQ a multiple of H=%d, got HQ=%d", s.cache.d, s.cache.H, s.HQ);
        s.out_stride = rows(out, s.HQ, s.cache.d, "out");
        if (out.size(0) < q.size(0))
            refuse(PyExc_ValueError, "%lld queries, %lld outputs", (long long)q.size(0), (long long)out.size(0));
        s.n_rows = i32(q.size(0), "queries");
        s.q = q.data_ptr();
        s.out = out.data_ptr();
        s.dtype = q.scalar_type() == at::kHalf ? TTKV_F16 : TTKV_BF16;
        const double scale = PyFloat_AsDouble(a[5]);
        if (scale == -1.0 && PyErr_Occurred()) throw Refused{};
        s.scale = float(scale);
        if (!std::isfinite(s.scale)) refuse(PyExc_ValueError, "scale is not a finite number");
        s.status = status_word(a[7], dev);
        if (prefill) {
            s.q_start = static_cast<const int32_t*>(vector(a[8], at::kInt, s.n_reqs, "q_start", dev));
            s.q_len = static_cast<const int32_t*>(vector(a[9], at::kInt, s.n_reqs, "q_len", dev));
            s.max_q_len = i32(integer(a[10], "max_q_len"), "max_q_len");
            s.max_seq_len = i32(integer(a[11], "max_seq_len"), "max_seq_len");
            if (s.max_q_len < 0 || s.max_seq_len < 0)
                refuse(PyExc_ValueError, "max_q_len=%d and max_seq_len=%d must not be negative", s.max_q_len, s.max_seq_len);
        } else if (s.n_rows != s.n_reqs) {
            refuse(PyExc_ValueError, "%d queries, %d block-table rows", s.n_rows, s.n_reqs);
        }
        if (s.n_reqs == 0 || s.n_rows == 0) return PyLong_FromLong(TTKV_OK);
        // scratch of this call alone, from torch's allocator in the stream's order: calls on other streams,
        // and captured graphs, have their own
        const int G = s.HQ / s.cache.H;
        s.workspace_bytes = prefill ? ttkv_q4_prefill_workspace_bytes(s.cache.d, s.n_reqs, G, s.max_q_len)
                                    : ttkv_q4_decode_workspace_bytes(s.cache.d, s.n_reqs, G);
        const at::Tensor ws = at::empty({int64_t(s.workspace_bytes)}, q.options().dtype(at::kByte));
        s.workspace = ws.data_ptr();
        return launch(prefill ? ttkv_q4_prefill : ttkv_q4_decode, s, dev);
    });
}

// Release: (block_table, lens, free_blocks, free_count, free_count_out, block_size, status); plan: and
// (query_start_loc, slot_mapping, positions or None).
PyObject* plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        const bool step = n == 10;
        if (!step) arity(n, 7);
        int dev = -1;
        ttkv_plan_args_t s{};
        table_of(a[0], dev, s.block_table, s.n_reqs, s.bt_cols, s.bt_stride);
        if (s.n_reqs > 1 && s.bt_stride < s.bt_cols) refuse(PyExc_ValueError, "block_table's rows overlap");
        if (s.n_reqs > TTKV_PLAN_MAX_REQS)
            refuse(PyExc_ValueError, "%d requests in one call: at most %d", s.n_reqs, TTKV_PLAN_MAX_REQS);
        s.lens = static_cast<const int32_t*>(vector(a[1], at::kInt, s.n_reqs, step ? "seq_lens" : "lens", dev));
        const at::Tensor& free_blocks = tensor(a[2], "free_blocks", dev);
        s.capacity = i32(free_blocks.numel(), "free_blocks");
        s.free_blocks = static_cast<int32_t*>(vector(a[2], at::kInt, s.capacity, "free_blocks", dev));
        const at::Tensor &count = tensor(a[3], "free_count", dev), &count_out = tensor(a[4], "free_count_out", dev);
        if (count.scalar_type() != at::kInt || count_out.scalar_type() != at::kInt)
            refuse(PyExc_TypeError, "free_count and free_count_out must be int32");
        if (count.numel() != 1 || count_out.numel() != 1)
            refuse(PyExc_ValueError, "free_count and free_count_out hold one number each");
        s.free_count = static_cast<const int32_t*>(count.data_ptr());
        s.free_count_out = static_cast<int32_t*>(count_out.data_ptr());
        s.block_size = i32(integer(a[5], "block_size"), "block_size");
        s.status = status_word(a[6], dev);
        if (step) {
            s.query_start_loc = static_cast<const int32_t*>(vector(a[7], at::kInt, int64_t(s.n_reqs) + 1, "query_start_loc", dev));
            const at::Tensor& slots = tensor(a[8], "slot_mapping", dev);
            s.n_tokens = i32(slots.numel(), "tokens");
            s.slots = static_cast<int64_t*>(vector(a[8], at::kLong, s.n_tokens, "slot_mapping", dev));
            if (a[9] != Py_None) s.positions = static_cast<int64_t*>(vector(a[9], at::kLong, s.n_tokens, "positions", dev));
        }
        return launch(step ? ttkv_plan_step : ttkv_release_blocks, s, dev);
    });
}

PyMethodDef methods[] = {
    {"store", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(store)), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attend)), METH_FASTCALL, nullptr},
    {"plan", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(plan)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ttkv_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ttkv_torch() { return PyModule_Create(&module); }
