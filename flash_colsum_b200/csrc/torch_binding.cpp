// The operator's path from a Python call to the kernels' launches, natively: argument checks,
// the output and scratch tensors, the stream, the launch.  A call of a dozen microseconds of GPU
// work is bound by this path when calls are issued back to back; through torch's Python API and
// ctypes it took 17 us a call, here it takes about 5.
//
// Every entry returns None for arguments it does not take (wrong shapes, types, devices, a
// library that is not bound yet): the Python wrapper then finds out what is wrong and raises the
// documented error.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <dlfcn.h>

#include <cmath>
#include <exception>
#include <vector>

#include "../../include/flash_colsum_b200.h"
#include "host_api.h"

namespace {

FcsRunCallFn g_run_call = nullptr;
FcsRunHostCallFn g_run_host_call = nullptr;
FcsSelectTopkFn g_select_topk = nullptr;
FcsSelectThresholdFn g_select_threshold = nullptr;
FcsLastErrorFn g_last_error = nullptr;
FcsAppendPagedFn g_append_paged = nullptr;
FcsSelectPagesWorkspaceFn g_select_pages_workspace = nullptr;
FcsSelectPagesFn g_select_pages = nullptr;
FcsAttendPagesFn g_attend_pages = nullptr;

constexpr int MAX_DEVICES = 64;
int* g_status[MAX_DEVICES] = {nullptr};   // the device status words (owned by the Python package)

// The launches run without the interpreter lock: they may wait for room in the launch queue.
struct WithoutGil {
    PyThreadState* state;
    WithoutGil() : state(PyEval_SaveThread()) {}
    ~WithoutGil() { PyEval_RestoreThread(state); }
};

PyObject* raise_library_error(int rc) {
    PyErr_Format(PyExc_RuntimeError, "flash_colsum_b200: %s (code %d)", g_last_error ? g_last_error() : "", rc);
    return nullptr;
}

at::Tensor empty_f32(int64_t rows, int64_t cols, c10::Device dev) {
    const int64_t size[2] = {rows, cols};
    return at::detail::empty_cuda(c10::IntArrayRef(size, 2), at::kFloat, dev, std::nullopt);
}

at::Tensor empty_on(c10::IntArrayRef size, at::ScalarType type, c10::Device dev) {
    return at::detail::empty_cuda(size, type, dev, std::nullopt);
}

// Scratch of one call; freed when the call returns (the caching allocator hands it out again in
// stream order only).  What the allocator throws does not pass through the library, which has copies
// in flight to wait for: it is kept, and thrown again by `rethrow` once the library has returned.
struct Scratch {
    c10::Device dev;
    std::vector<at::Tensor> held;
    std::exception_ptr error;
    static void* alloc(void* ctx, size_t bytes) noexcept {
        Scratch* s = static_cast<Scratch*>(ctx);
        try {
            const int64_t size[1] = {static_cast<int64_t>(bytes)};
            s->held.push_back(at::detail::empty_cuda(c10::IntArrayRef(size, 1), at::kByte, s->dev, std::nullopt));
            return s->held.back().mutable_data_ptr();
        } catch (...) {
            s->error = std::current_exception();
            return nullptr;
        }
    }
    void rethrow() const {
        if (error) std::rethrow_exception(error);
    }
};

int dtype_code(at::ScalarType t) {
    return t == at::kHalf ? FCS_DTYPE_FP16 : t == at::kBFloat16 ? FCS_DTYPE_BF16 : t == at::kFloat ? FCS_DTYPE_FP32 : -1;
}

// Unit inner stride, positive outer strides in multiples of 16 bytes, 16-byte aligned base.  The
// stride of an axis of one entry says nothing; the contiguous one stands in for it.
void kernel_strides(const at::Tensor& t, int64_t (&st)[3]) {
    int64_t dense = t.size(3);
    for (int i = 2; i >= 0; --i) {
        st[i] = t.size(i) > 1 ? t.stride(i) : dense;
        dense *= t.size(i);
    }
}
bool kernel_ready(const at::Tensor& t) {
    int64_t st[3];
    kernel_strides(t, st);
    const int64_t granule = 16 / t.element_size();
    return t.stride(3) == 1 && st[0] > 0 && st[1] > 0 && st[2] > 0 && ((st[0] | st[1] | st[2]) & (granule - 1)) == 0 &&
           (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0;
}

bool usable(PyObject* o) { return THPVariable_Check(o); }

// One call on checked operands.  Returns a new reference, or NULL with an exception set.
PyObject* run(at::Tensor q, at::Tensor k, double scale, bool causal, int k_past, int cls_n, int h_norm) {
    const c10::Device dev = q.device();
    at::Tensor out;
    int rc;
    {
        WithoutGil nogil;
        const c10::DeviceGuard guard(dev);
        if (!kernel_ready(q)) q = q.contiguous();
        if (!kernel_ready(k)) k = k.contiguous();
        FcsCall c;
        c.B = (int)q.size(0);
        c.H = (int)q.size(1);
        c.Sq = (int)q.size(2);
        c.Sk = (int)k.size(2);
        c.D = (int)q.size(3);
        out = empty_f32(c.B, c.Sk, dev);
        c.q = q.const_data_ptr();
        c.k = k.const_data_ptr();
        c.out = static_cast<float*>(out.mutable_data_ptr());
        c.out_ld = c.Sk;
        c.dtype = dtype_code(q.scalar_type());
        kernel_strides(q, c.q_stride);
        kernel_strides(k, c.k_stride);
        c.scale = (float)scale;
        c.causal = causal ? 1 : 0;
        c.k_past = k_past;
        c.cls_n = cls_n;
        c.h_norm = h_norm;
        c.status = g_status[dev.index()];
        c.stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
        Scratch scratch{dev, {}, nullptr};
        c.alloc = &Scratch::alloc;
        c.alloc_ctx = &scratch;
        rc = g_run_call(&c);
        scratch.rethrow();
    }
    if (rc != FCS_OK) return raise_library_error(rc);
    return THPVariable_Wrap(std::move(out));
}

// Whether the kernels take this pair of operands: CUDA tensors of one device whose status word is
// known, 4-D, no empty axis, one supported type, matching batch, heads and head dimension.
bool operands_ok(const at::Tensor& q, const at::Tensor& k) {
    if (q.dim() != 4 || k.dim() != 4 || !q.is_cuda() || q.device() != k.device()) return false;
    const int idx = q.device().index();
    if (idx < 0 || idx >= MAX_DEVICES || !g_status[idx]) return false;
    if (q.scalar_type() != k.scalar_type() || dtype_code(q.scalar_type()) < 0) return false;
    const auto a = q.sizes(), b = k.sizes();
    if (a[0] != b[0] || a[1] != b[1] || a[3] != b[3] || a[3] < 8 || a[3] > 128 || a[3] % 8) return false;
    for (int i = 0; i < 4; ++i)
        if (a[i] <= 0 || b[i] <= 0 || a[i] > 0x7fffffffLL || b[i] > 0x7fffffffLL) return false;
    return g_run_call != nullptr;
}

double scale_or_default(PyObject* o, const at::Tensor& q) {
    return o == Py_None ? 1.0 / std::pow((double)q.size(3), 0.5) : PyFloat_AsDouble(o);
}

// colsum(query, key, scale, is_causal, cls_len): `flash_colsum`'s rules
PyObject* py_colsum(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5 || !usable(args[0]) || !usable(args[1])) Py_RETURN_NONE;
    const at::Tensor& q = THPVariable_Unpack(args[0]);
    const at::Tensor& k = THPVariable_Unpack(args[1]);
    if (!operands_ok(q, k)) Py_RETURN_NONE;
    const int causal = PyObject_IsTrue(args[3]);
    if (causal < 0) return nullptr;
    int cls_n = -1;
    if (args[4] != Py_None) {
        if (causal || !PyLong_CheckExact(args[4])) Py_RETURN_NONE;
        int overflow = 0;
        const long long v = PyLong_AsLongLongAndOverflow(args[4], &overflow);
        if (overflow || v <= 0 || v > 0x7fffffffLL) Py_RETURN_NONE;
        cls_n = (int)v;
    }
    if (causal ? q.size(0) != 1 : q.size(2) != k.size(2)) Py_RETURN_NONE;
    const double scale = scale_or_default(args[2], q);
    if (PyErr_Occurred()) return nullptr;
    return run(q, k, scale, causal != 0, -1, cls_n, 0);
    END_HANDLE_TH_ERRORS
}

// launch(query, key, scale, is_causal, k_past, cls_n, h_norm): checked arguments, -1 / 0 for defaults
PyObject* py_launch(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7 || !usable(args[0]) || !usable(args[1])) Py_RETURN_NONE;
    const at::Tensor& q = THPVariable_Unpack(args[0]);
    const at::Tensor& k = THPVariable_Unpack(args[1]);
    if (!operands_ok(q, k)) Py_RETURN_NONE;
    const double scale = scale_or_default(args[2], q);
    const int causal = PyObject_IsTrue(args[3]);
    const long k_past = PyLong_AsLong(args[4]), cls_n = PyLong_AsLong(args[5]), h_norm = PyLong_AsLong(args[6]);
    if (PyErr_Occurred()) return nullptr;
    if (!causal && q.size(2) != k.size(2)) Py_RETURN_NONE;
    const long most = 0x7fffffffL;
    return run(q, k, scale, causal != 0, (int)(k_past < most ? k_past : most), (int)(cls_n < most ? cls_n : most),
               (int)h_norm);
    END_HANDLE_TH_ERRORS
}

// host(query, key, scale, is_causal, cls_len, device index, batch_chunk or 0) -> host tensor
PyObject* py_host(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7 || !g_run_host_call || !usable(args[0]) || !usable(args[1])) Py_RETURN_NONE;
    const at::Tensor& q = THPVariable_Unpack(args[0]);
    const at::Tensor& k = THPVariable_Unpack(args[1]);
    const int causal = PyObject_IsTrue(args[3]);
    const long idx = PyLong_AsLong(args[5]), batch_chunk = PyLong_AsLong(args[6]);
    if (PyErr_Occurred()) return nullptr;
    if (idx < 0 || idx >= MAX_DEVICES || !g_status[idx] || batch_chunk < 0) Py_RETURN_NONE;
    if (q.dim() != 4 || k.dim() != 4 || !q.is_cpu() || !k.is_cpu() || !q.is_contiguous() || !k.is_contiguous()) Py_RETURN_NONE;
    if (q.scalar_type() != k.scalar_type() || dtype_code(q.scalar_type()) < 0) Py_RETURN_NONE;
    const auto a = q.sizes(), b = k.sizes();
    if (a[0] != b[0] || a[1] != b[1] || a[3] != b[3] || a[3] < 8 || a[3] > 128 || a[3] % 8) Py_RETURN_NONE;
    for (int i = 0; i < 4; ++i)
        if (a[i] <= 0 || b[i] <= 0 || a[i] > 0x7fffffffLL || b[i] > 0x7fffffffLL) Py_RETURN_NONE;
    if (causal ? a[0] != 1 : a[2] != b[2]) Py_RETURN_NONE;
    int cls_n = -1;
    if (args[4] != Py_None) {
        if (causal || !PyLong_CheckExact(args[4])) Py_RETURN_NONE;
        int overflow = 0;
        const long long v = PyLong_AsLongLongAndOverflow(args[4], &overflow);
        if (overflow || v <= 0 || v > 0x7fffffffLL) Py_RETURN_NONE;
        cls_n = (int)v;
    }
    const double scale = scale_or_default(args[2], q);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor host_out;
    int rc;
    {
        WithoutGil nogil;
        const c10::Device dev(c10::kCUDA, (c10::DeviceIndex)idx);
        const c10::DeviceGuard guard(dev);
        const at::Tensor dq = at::detail::empty_cuda(a, q.scalar_type(), dev, std::nullopt);
        const at::Tensor dk = at::detail::empty_cuda(b, k.scalar_type(), dev, std::nullopt);
        const at::Tensor out = empty_f32(a[0], b[2], dev);
        host_out = at::empty({a[0], b[2]}, at::TensorOptions().dtype(at::kFloat).device(at::kCPU));
        FcsHostCall hc;
        FcsCall& c = hc.call;
        c.B = (int)a[0];
        c.H = (int)a[1];
        c.Sq = (int)a[2];
        c.Sk = (int)b[2];
        c.D = (int)a[3];
        c.q = dq.const_data_ptr();
        c.k = dk.const_data_ptr();
        c.out = static_cast<float*>(out.mutable_data_ptr());
        c.out_ld = c.Sk;
        c.dtype = dtype_code(q.scalar_type());
        kernel_strides(dq, c.q_stride);
        kernel_strides(dk, c.k_stride);
        c.scale = (float)scale;
        c.causal = causal;
        c.k_past = -1;
        c.cls_n = cls_n;
        c.h_norm = 0;
        c.status = g_status[idx];
        c.stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)idx).stream();
        Scratch scratch{dev, {}, nullptr};
        c.alloc = &Scratch::alloc;
        c.alloc_ctx = &scratch;
        hc.host_q = q.const_data_ptr();
        hc.host_k = k.const_data_ptr();
        hc.host_out = static_cast<float*>(host_out.mutable_data_ptr());
        hc.batch_chunk = (int)(batch_chunk < 0x7fffffffL ? batch_chunk : 0x7fffffffL);
        rc = g_run_host_call(&hc);
        scratch.rethrow();
    }
    if (rc != FCS_OK) return raise_library_error(rc);
    return THPVariable_Wrap(std::move(host_out));
    END_HANDLE_TH_ERRORS
}

bool means_ok(const at::Tensor& t) {
    return t.dim() == 2 && t.scalar_type() == at::kFloat && t.is_cuda();
}

PyObject* pair(at::Tensor a, at::Tensor b) {
    PyObject* t = PyTuple_New(2);
    if (!t) return nullptr;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(a)));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(b)));
    return t;
}

// topk(colsum, k) -> (values, indices)
PyObject* py_topk(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 2 || !g_select_topk || !usable(args[0]) || !PyLong_Check(args[1])) Py_RETURN_NONE;
    at::Tensor x = THPVariable_Unpack(args[0]);
    if (!means_ok(x)) Py_RETURN_NONE;
    const long long k = PyLong_AsLongLong(args[1]);
    if (PyErr_Occurred() || k < 1 || k > x.size(1)) { PyErr_Clear(); Py_RETURN_NONE; }
    const c10::Device dev = x.device();
    at::Tensor idx, val;
    int rc;
    {
        WithoutGil nogil;
        const c10::DeviceGuard guard(dev);
        if (x.stride(1) != 1 || x.stride(0) < x.size(1)) x = x.contiguous();
        const int64_t size[2] = {x.size(0), (int64_t)k};
        idx = at::detail::empty_cuda(c10::IntArrayRef(size, 2), at::kInt, dev, std::nullopt);
        val = empty_f32(size[0], size[1], dev);
        rc = g_select_topk(static_cast<const float*>(x.const_data_ptr()), x.size(0) > 1 ? x.stride(0) : x.size(1),
                           (int)x.size(0), (int)x.size(1), (int)k, static_cast<int*>(idx.mutable_data_ptr()),
                           static_cast<float*>(val.mutable_data_ptr()),
                           c10::cuda::getCurrentCUDAStream(dev.index()).stream());
    }
    if (rc != FCS_OK) return raise_library_error(rc);
    return pair(std::move(val), std::move(idx));
    END_HANDLE_TH_ERRORS
}

// threshold(colsum, threshold, relative) -> (indices, counts)
PyObject* py_threshold(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 3 || !g_select_threshold || !usable(args[0])) Py_RETURN_NONE;
    at::Tensor x = THPVariable_Unpack(args[0]);
    if (!means_ok(x)) Py_RETURN_NONE;
    const double thr = PyFloat_AsDouble(args[1]);
    const int relative = PyObject_IsTrue(args[2]);
    if (PyErr_Occurred()) return nullptr;
    if (std::isnan(thr)) Py_RETURN_NONE;
    const c10::Device dev = x.device();
    at::Tensor idx, cnt;
    int rc;
    {
        WithoutGil nogil;
        const c10::DeviceGuard guard(dev);
        if (x.stride(1) != 1 || x.stride(0) < x.size(1)) x = x.contiguous();
        const int64_t size[2] = {x.size(0), x.size(1)};
        idx = at::detail::empty_cuda(c10::IntArrayRef(size, 2), at::kInt, dev, std::nullopt);
        cnt = at::detail::empty_cuda(c10::IntArrayRef(size, 1), at::kInt, dev, std::nullopt);
        rc = g_select_threshold(static_cast<const float*>(x.const_data_ptr()),
                                x.size(0) > 1 ? x.stride(0) : x.size(1), (int)x.size(0), (int)x.size(1), (float)thr,
                                relative, static_cast<int*>(idx.mutable_data_ptr()),
                                static_cast<int*>(cnt.mutable_data_ptr()),
                                c10::cuda::getCurrentCUDAStream(dev.index()).stream());
    }
    if (rc != FCS_OK) return raise_library_error(rc);
    return pair(std::move(idx), std::move(cnt));
    END_HANDLE_TH_ERRORS
}

// ---- the paged cache

// A tensor argument that may be None; `ok` falls where it is neither.
const at::Tensor* optional_tensor(PyObject* o, bool& ok) {
    if (o == Py_None) return nullptr;
    if (!usable(o)) {
        ok = false;
        return nullptr;
    }
    return &THPVariable_Unpack(o);
}

bool indices_ok(const at::Tensor& t, int64_t dims, c10::Device dev) {
    return t.dim() == dims && t.scalar_type() == at::kInt && t.device() == dev && t.numel() > 0;
}

// Rows of 16-bit elements that are read in pieces of 16 bytes: unit inner stride, the other strides multiples of 8.
template <int N>
bool rows_ready(const at::Tensor& t, int64_t (&st)[N]) {
    int64_t any = 0;
    for (int i = 0; i < N; ++i) {
        st[i] = t.size(i) > 1 ? t.stride(i) : 0;      // (the stride of an axis of one entry says nothing)
        if (st[i] < 0) return false;
        any |= st[i];
    }
    return (t.size(N) == 1 || t.stride(N) == 1) && any % 8 == 0 && (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0;
}

// A result of rows as the kernels write it.
bool result_ready(const at::Tensor& t, int64_t (&st)[2]) {
    const int64_t size[2] = {t.size(0), t.size(1)};
    return rows_ready<2>(t, st) && fcs_rows_apart(2, size, st, t.size(2));
}

// A pool as the kernels take it: strides that hold a row and, where it is written, keep the rows apart.
bool pool_ready(const at::Tensor& t, int64_t (&st)[3], bool write) {
    if (!rows_ready<3>(t, st) || (write && !fcs_rows_apart(3, t.sizes().data(), st, t.size(3)))) return false;
    for (int i = 0; i < 3; ++i)
        if (t.size(i) > 1 && st[i] < t.size(3)) return false;
    return true;
}

// Memory of the caller's that a call writes, asked for when nothing can refuse the call any more: a tensor that shares its memory until
// it is written gets its own, and the version counter tells autograd that a saved tensor has changed.  (Tensors of inference mode
// have none.)
void* written(const at::Tensor& t) {
    void* at = t.mutable_data_ptr();
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    return at;
}

// The batch and, unless they are not given, the pools of a call; whatever had to be laid out anew is held until it returns.
struct PagedArgs {
    FcsPagedCache c = {};
    at::Tensor table, lens, starts;
    c10::Device dev = c10::Device(c10::kCPU);
    int* status = nullptr;

    bool batch(const at::Tensor& rows, const at::Tensor& t, const at::Tensor& n, const at::Tensor* s) {
        dev = rows.device();
        const int idx = dev.index();
        if (!dev.is_cuda() || idx < 0 || idx >= MAX_DEVICES || !g_status[idx] || !g_append_paged) return false;
        if (rows.dim() != 3 || !indices_ok(t, 2, dev) || !indices_ok(n, 1, dev)) return false;
        const int64_t T = rows.size(0), B = n.size(0), D = rows.size(2);
        if (T < 1 || T > 0x7fffffffLL || B > 0x7fffffffLL || t.size(0) != B || t.size(1) > 0x7fffffffLL) return false;
        if (D % 8 || D < 8 || D > 128 || (rows.scalar_type() != at::kHalf && rows.scalar_type() != at::kBFloat16)) return false;
        if (s ? !indices_ok(*s, 1, dev) || s->size(0) != B + 1 : T != B) return false;
        status = g_status[idx];
        table = t.stride(1) == 1 || t.size(1) == 1 ? t : t.contiguous();
        if (B > 1 && table.stride(0) < t.size(1)) table = t.contiguous();
        lens = n.contiguous();
        if (s) starts = s->contiguous();
        c.page_table = static_cast<const int*>(table.const_data_ptr());
        c.table_stride = B > 1 ? table.stride(0) : t.size(1);
        c.lens = static_cast<const int*>(lens.const_data_ptr());
        c.starts = s ? static_cast<const int*>(starts.const_data_ptr()) : nullptr;
        c.dim = (int)D;
        c.dtype = dtype_code(rows.scalar_type());
        c.sequences = (int)B;
        c.table_width = (int)t.size(1);
        c.tokens = (int)T;
        return true;
    }
    bool pools(const at::Tensor& rows, const at::Tensor& k, const at::Tensor& v, bool write) {
        if (k.dim() != 4 || v.dim() != 4 || k.sizes() != v.sizes() || k.device() != dev || v.device() != dev) return false;
        if (k.scalar_type() != rows.scalar_type() || v.scalar_type() != rows.scalar_type()) return false;
        const auto n = k.sizes();
        if (n[0] < 1 || n[0] > 0x7fffffffLL || n[1] < 1 || n[1] > 65535 || n[3] != c.dim) return false;
        if (n[2] != 16 && n[2] != 32 && n[2] != 64 && n[2] != 128) return false;
        if (!pool_ready(k, c.key_stride, write) || !pool_ready(v, c.value_stride, write)) return false;
        c.key_pages = const_cast<void*>(k.const_data_ptr());      // (to be read; append_paged asks again)
        c.value_pages = const_cast<void*>(v.const_data_ptr());
        c.pages = (int)n[0];
        c.kv_heads = (int)n[1];
        c.page_size = (int)n[2];
        return true;
    }
    bool heads_ok(const at::Tensor& query) const {
        return query.size(1) > 0 && query.size(1) % c.kv_heads == 0 && query.size(1) <= 0x7ffffLL;
    }
    void* stream() const { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }
};

bool like_rows(const at::Tensor& t, const at::Tensor& rows) {
    return t.dim() == 3 && t.size(0) == rows.size(0) && t.size(2) == rows.size(2) && t.device() == rows.device() &&
           t.scalar_type() == rows.scalar_type();
}

int int_or(PyObject* o, bool& ok) {
    const long long v = PyLong_CheckExact(o) ? PyLong_AsLongLong(o) : -1;
    if (v < 0 || v > 0x7fffffffLL) {
        PyErr_Clear();
        ok = false;
    }
    return (int)v;
}

// append_paged(key, value, key_pages, value_pages, page_table, lens, starts, query, cos, sin, positions, interleaved,
// bounds, query_out) -> rotated query, or True without one
PyObject* py_append_paged(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 14) Py_RETURN_NONE;
    for (int i = 0; i < 6; ++i)
        if (!usable(args[i])) Py_RETURN_NONE;
    bool ok = true;
    const at::Tensor *starts = optional_tensor(args[6], ok), *query_in = optional_tensor(args[7], ok),
                     *cos = optional_tensor(args[8], ok), *sin = optional_tensor(args[9], ok),
                     *positions = optional_tensor(args[10], ok), *bounds = optional_tensor(args[12], ok),
                     *query_out = optional_tensor(args[13], ok);
    const int interleaved = PyObject_IsTrue(args[11]);
    if (interleaved < 0) return nullptr;
    if (!ok) Py_RETURN_NONE;
    at::Tensor key = THPVariable_Unpack(args[0]), value = THPVariable_Unpack(args[1]), query, out, where;
    PagedArgs a;
    FcsPagedRows r = {};
    int rc;
    {
        const c10::OptionalDeviceGuard guard(key.is_cuda() ? std::optional<c10::Device>(key.device()) : std::nullopt);
        if (!a.batch(key, THPVariable_Unpack(args[4]), THPVariable_Unpack(args[5]), starts)) Py_RETURN_NONE;
        if (!a.pools(key, THPVariable_Unpack(args[2]), THPVariable_Unpack(args[3]), true)) Py_RETURN_NONE;
        if (!like_rows(value, key) || key.size(1) != a.c.kv_heads || value.size(1) != a.c.kv_heads) Py_RETURN_NONE;
        if ((cos == nullptr) != (sin == nullptr) || (positions && !cos)) Py_RETURN_NONE;
        if (cos) {
            if (cos->dim() != 2 || cos->sizes() != sin->sizes() || cos->scalar_type() != at::kFloat ||
                sin->scalar_type() != at::kFloat || cos->device() != a.dev || sin->device() != a.dev || !cos->is_contiguous() ||
                !sin->is_contiguous() || cos->size(0) < 1 || cos->size(0) > 0x7fffffffLL || cos->size(1) < 8 ||
                cos->size(1) % 8 || 2 * cos->size(1) > a.c.dim ||
                ((reinterpret_cast<uintptr_t>(cos->const_data_ptr()) | reinterpret_cast<uintptr_t>(sin->const_data_ptr())) & 15))
                Py_RETURN_NONE;
            r.cos = static_cast<const float*>(cos->const_data_ptr());
            r.sin = static_cast<const float*>(sin->const_data_ptr());
            r.table_rows = (int)cos->size(0);
            r.rotary = 2 * (int)cos->size(1);
            r.interleaved = interleaved;
            if (positions) {
                if (!indices_ok(*positions, 1, a.dev) || positions->size(0) != key.size(0)) Py_RETURN_NONE;
                where = positions->contiguous();
                r.positions = static_cast<const int*>(where.const_data_ptr());
            }
        }
        if (bounds) {
            if (bounds->dim() != 4 || bounds->size(0) != a.c.pages || bounds->size(1) != a.c.kv_heads || bounds->size(2) != 2 ||
                bounds->size(3) != a.c.dim || bounds->scalar_type() != key.scalar_type() || bounds->device() != a.dev ||
                !bounds->is_contiguous() || (reinterpret_cast<uintptr_t>(bounds->const_data_ptr()) & 15))
                Py_RETURN_NONE;
        }
        if (query_out && !query_in) Py_RETURN_NONE;
        if (query_in) {
            if (!like_rows(*query_in, key) || !a.heads_ok(*query_in)) Py_RETURN_NONE;
            if (query_out && (!like_rows(*query_out, key) || query_out->size(1) != query_in->size(1) ||
                              !result_ready(*query_out, r.query_out_stride)))
                Py_RETURN_NONE;
            query = rows_ready<2>(*query_in, r.query_stride) ? *query_in : query_in->contiguous();
            rows_ready<2>(query, r.query_stride);
            r.fill_tail = query_out == nullptr;
            out = query_out ? *query_out : empty_on(query.sizes(), query.scalar_type(), a.dev);
            rows_ready<2>(out, r.query_out_stride);
            r.query_out = query_out ? written(out) : out.mutable_data_ptr();
            r.query = query.const_data_ptr();
            r.q_heads = (int)query.size(1);
        }
        if (!rows_ready<2>(key, r.key_stride)) key = key.contiguous();
        if (!rows_ready<2>(value, r.value_stride)) value = value.contiguous();
        rows_ready<2>(key, r.key_stride);
        rows_ready<2>(value, r.value_stride);
        r.key = key.const_data_ptr();
        r.value = value.const_data_ptr();
        a.c.key_pages = written(THPVariable_Unpack(args[2]));
        a.c.value_pages = written(THPVariable_Unpack(args[3]));
        if (bounds) r.bounds = written(*bounds);
        WithoutGil nogil;
        rc = g_append_paged(&a.c, &r, a.status, a.stream());
    }
    if (rc != FCS_OK) return raise_library_error(rc);
    if (!query_in) Py_RETURN_TRUE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// select_pages(query, bounds, page_table, lens, k, page_size, starts, first, last, out) -> (tokens, kv_heads, k)
PyObject* py_select_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10) Py_RETURN_NONE;
    for (int i = 0; i < 4; ++i)
        if (!usable(args[i])) Py_RETURN_NONE;
    bool ok = true;
    const int k = int_or(args[4], ok), page_size = int_or(args[5], ok), first = int_or(args[7], ok), last = int_or(args[8], ok);
    const at::Tensor *starts = optional_tensor(args[6], ok), *given = optional_tensor(args[9], ok);
    if (!ok || k < 1 || last < 1 || (int64_t)first + last > k) Py_RETURN_NONE;
    at::Tensor query = THPVariable_Unpack(args[0]), out;
    const at::Tensor& bounds = THPVariable_Unpack(args[1]);
    PagedArgs a;
    int rc;
    {
        const c10::OptionalDeviceGuard guard(query.is_cuda() ? std::optional<c10::Device>(query.device()) : std::nullopt);
        if (!a.batch(query, THPVariable_Unpack(args[2]), THPVariable_Unpack(args[3]), starts)) Py_RETURN_NONE;
        if (bounds.dim() != 4 || bounds.size(0) < 1 || bounds.size(0) > 0x7fffffffLL || bounds.size(1) < 1 ||
            bounds.size(1) > 65535 || bounds.size(2) != 2 || bounds.size(3) != a.c.dim ||
            bounds.scalar_type() != query.scalar_type() || bounds.device() != a.dev || !bounds.is_contiguous() ||
            (reinterpret_cast<uintptr_t>(bounds.const_data_ptr()) & 15))
            Py_RETURN_NONE;
        if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) Py_RETURN_NONE;
        a.c.pages = (int)bounds.size(0);
        a.c.kv_heads = (int)bounds.size(1);
        a.c.page_size = page_size;
        if (!a.heads_ok(query)) Py_RETURN_NONE;
        const int64_t size[3] = {query.size(0), bounds.size(1), k};
        if (given && (given->sizes() != c10::IntArrayRef(size, 3) || given->scalar_type() != at::kInt || given->device() != a.dev ||
                      !given->is_contiguous()))
            Py_RETURN_NONE;
        out = given ? *given : empty_on(c10::IntArrayRef(size, 3), at::kInt, a.dev);
        int64_t st[2];
        if (!rows_ready<2>(query, st)) query = query.contiguous();
        rows_ready<2>(query, st);
        const int64_t bytes[1] = {(int64_t)g_select_pages_workspace(&a.c)};
        const at::Tensor scratch = empty_on(c10::IntArrayRef(bytes, 1), at::kByte, a.dev);
        int* const chosen = static_cast<int*>(given ? written(out) : out.mutable_data_ptr());
        WithoutGil nogil;
        rc = g_select_pages(&a.c, query.const_data_ptr(), st, (int)query.size(1), bounds.const_data_ptr(), k, first, last,
                            chosen, given == nullptr, scratch.mutable_data_ptr(),
                            (size_t)bytes[0], a.status, a.stream());
    }
    if (rc != FCS_OK) return raise_library_error(rc);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// attend_pages(query, key_pages, value_pages, page_table, lens, pages, starts, scale, with_lse, out) -> out, or (out, lse)
PyObject* py_attend_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10) Py_RETURN_NONE;
    for (int i = 0; i < 6; ++i)
        if (!usable(args[i])) Py_RETURN_NONE;
    bool ok = true;
    const at::Tensor *starts = optional_tensor(args[6], ok), *given = optional_tensor(args[9], ok);
    const int with_lse = PyObject_IsTrue(args[8]);
    if (with_lse < 0) return nullptr;
    if (!ok) Py_RETURN_NONE;
    at::Tensor query = THPVariable_Unpack(args[0]), out, lse, pages;
    if (query.dim() != 3) Py_RETURN_NONE;
    const double scale = args[7] == Py_None ? 1.0 / std::sqrt((double)query.size(2)) : PyFloat_AsDouble(args[7]);
    if (PyErr_Occurred()) return nullptr;
    if (std::isnan(scale)) Py_RETURN_NONE;
    const at::Tensor& chosen = THPVariable_Unpack(args[5]);
    PagedArgs a;
    int rc;
    {
        const c10::OptionalDeviceGuard guard(query.is_cuda() ? std::optional<c10::Device>(query.device()) : std::nullopt);
        if (!a.batch(query, THPVariable_Unpack(args[3]), THPVariable_Unpack(args[4]), starts)) Py_RETURN_NONE;
        if (!a.pools(query, THPVariable_Unpack(args[1]), THPVariable_Unpack(args[2]), false) || !a.heads_ok(query)) Py_RETURN_NONE;
        if (!indices_ok(chosen, 3, a.dev) || chosen.size(0) != query.size(0) || chosen.size(1) != a.c.kv_heads ||
            chosen.size(2) > FCS_LIST_MAX)
            Py_RETURN_NONE;
        int64_t st[2], out_st[2];
        if (given && (!like_rows(*given, query) || given->size(1) != query.size(1) || !result_ready(*given, out_st))) Py_RETURN_NONE;
        if (!rows_ready<2>(query, st)) query = query.contiguous();
        rows_ready<2>(query, st);
        pages = chosen.contiguous();
        out = given ? *given : empty_on(query.sizes(), query.scalar_type(), a.dev);
        rows_ready<2>(out, out_st);
        if (with_lse) lse = empty_f32(query.size(0), query.size(1), a.dev);
        void* const result = given ? written(out) : out.mutable_data_ptr();
        WithoutGil nogil;
        rc = g_attend_pages(&a.c, query.const_data_ptr(), st, (int)query.size(1), static_cast<const int*>(pages.const_data_ptr()),
                            (int)pages.size(2), (float)scale, result, out_st,
                            with_lse ? static_cast<float*>(lse.mutable_data_ptr()) : nullptr, given ? 2 : 3, a.status, a.stream());
    }
    if (rc != FCS_OK) return raise_library_error(rc);
    if (!with_lse) return THPVariable_Wrap(std::move(out));
    return pair(std::move(out), std::move(lse));
    END_HANDLE_TH_ERRORS
}

// bind(handle): the entry points of the loaded CUDA library (a dlopen handle)
PyObject* py_bind(PyObject*, PyObject* arg) {
    void* h = PyLong_AsVoidPtr(arg);
    if (PyErr_Occurred()) return nullptr;
    auto sym = [&](const char* name) { return dlsym(h, name); };
    g_last_error = reinterpret_cast<FcsLastErrorFn>(sym("fcs_last_error"));
    g_select_topk = reinterpret_cast<FcsSelectTopkFn>(sym("fcs_select_topk"));
    g_select_threshold = reinterpret_cast<FcsSelectThresholdFn>(sym("fcs_select_threshold"));
    g_run_call = reinterpret_cast<FcsRunCallFn>(sym("fcs_run_call"));
    g_run_host_call = reinterpret_cast<FcsRunHostCallFn>(sym("fcs_run_host_call"));
    g_append_paged = reinterpret_cast<FcsAppendPagedFn>(sym("fcs_append_paged"));
    g_select_pages_workspace = reinterpret_cast<FcsSelectPagesWorkspaceFn>(sym("fcs_select_pages_workspace_bytes"));
    g_select_pages = reinterpret_cast<FcsSelectPagesFn>(sym("fcs_select_pages"));
    g_attend_pages = reinterpret_cast<FcsAttendPagesFn>(sym("fcs_attend_pages"));
    if (!g_last_error || !g_select_topk || !g_select_threshold || !g_run_call || !g_run_host_call || !g_append_paged ||
        !g_select_pages_workspace || !g_select_pages || !g_attend_pages) {
        PyErr_SetString(PyExc_RuntimeError, "flash_colsum_b200: the CUDA library lacks an entry point of this binding");
        return nullptr;
    }
    Py_RETURN_NONE;
}

// set_status(device_index, address): the status word that this device's calls report into
PyObject* py_set_status(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2) { PyErr_SetString(PyExc_TypeError, "set_status(device_index, address)"); return nullptr; }
    const long idx = PyLong_AsLong(args[0]);
    void* p = PyLong_AsVoidPtr(args[1]);
    if (PyErr_Occurred()) return nullptr;
    if (idx >= 0 && idx < MAX_DEVICES) g_status[idx] = static_cast<int*>(p);
    Py_RETURN_NONE;
}

template <typename F>
constexpr PyCFunction fast(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)); }

PyMethodDef g_methods[] = {
    {"colsum", fast(py_colsum), METH_FASTCALL, nullptr},
    {"launch", fast(py_launch), METH_FASTCALL, nullptr},
    {"host", fast(py_host), METH_FASTCALL, nullptr},
    {"topk", fast(py_topk), METH_FASTCALL, nullptr},
    {"threshold", fast(py_threshold), METH_FASTCALL, nullptr},
    {"append_paged", fast(py_append_paged), METH_FASTCALL, nullptr},
    {"select_pages", fast(py_select_pages), METH_FASTCALL, nullptr},
    {"attend_pages", fast(py_attend_pages), METH_FASTCALL, nullptr},
    {"bind", py_bind, METH_O, nullptr},
    {"set_status", fast(py_set_status), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_fcs_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fcs_torch(void) { return PyModule_Create(&g_module); }
