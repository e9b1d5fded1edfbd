// The Python layer's calls in native code: femto_native.
//
// A decode call of a few sequences keeps the GPU busy for 4-10 us, and in
// Python its checks, its strides and a ctypes call of 27 arguments cost the
// host 18 us, so every small call ran at the host's pace.  The functions here
// make the same checks on the tensors' C++ objects, allocate the output, look
// up the stream's workspace in the dict that the Python layer keeps, and call
// the library through the pointers that the Python layer passes to bind() (so
// both use one loaded library).
//
// None means "not handled here": a check failed, the call is empty, there is
// no workspace yet, an argument is not a plain tensor or int, or the tensor
// library threw.  Nothing has been launched then, and the caller takes its
// Python path, which allocates, raises or returns as it always did.  An error
// of the library itself raises RuntimeError with the library's message.
#include <Python.h>

#include <ATen/Functions.h>
#include <hip/hip_runtime_api.h>
#include <c10/hip/HIPStream.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>

#include "femto_attn.h"

namespace {

decltype(&femto_attn_last_error) g_last_error;
decltype(&femto_paged_attention_gemv) g_gemv;
decltype(&femto_paged_attention_gemv_workspace_size) g_gemv_ws;
decltype(&femto_paged_attention_gemm) g_gemm;
decltype(&femto_paged_attention_gemm_workspace_size) g_gemm_ws;
decltype(&femto_qk_norm_rope_cache_write) g_prologue;
decltype(&femto_flash_attention) g_flash;
decltype(&femto_rope_cache_write) g_rope;
decltype(&femto_paged_attention_gemv_shared_prefix) g_shared;
decltype(&femto_paged_attention_gemv_shared_prefix_workspace_size) g_shared_ws;
decltype(&femto_paged_attention_gemv_window) g_gemv_window;
decltype(&femto_paged_attention_gemv_window_workspace_size) g_gemv_window_ws;
decltype(&femto_paged_attention_gemm_window) g_gemm_window;
decltype(&femto_paged_attention_gemm_window_workspace_size) g_gemm_window_ws;
decltype(&femto_fp4_page_bytes) g_fp4_page;
decltype(&femto_kv_cache_write_fp4) g_write_fp4;
decltype(&femto_kv_cache_read_fp4) g_read_fp4;
decltype(&femto_rope_cache_write_fp4) g_rope_fp4;
decltype(&femto_paged_attention_gemv_fp4) g_gemv_fp4;
decltype(&femto_paged_attention_gemv_fp4_workspace_size) g_gemv_fp4_ws;
decltype(&femto_paged_attention_gemm_fp4) g_gemm_fp4;
decltype(&femto_paged_attention_gemm_fp4_workspace_size) g_gemm_fp4_ws;

// Thrown (and caught in `guarded`) where the Python path has to take over.
struct NotHere {};
inline void need(bool ok) {
    if (!ok) throw NotHere{};
}

// Exactly torch.Tensor or torch.nn.Parameter: subclasses may override what is read here.
const at::Tensor& tensor(PyObject* o) {
    need(THPVariable_CheckExact(o));
    return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o) {
    need(PyLong_CheckExact(o));
    int overflow = 0;
    const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
    need(!overflow);
    return v;
}

int int32(int64_t v) {
    need(v >= INT32_MIN && v <= INT32_MAX);
    return (int)v;
}

int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return FEMTO_F32;
        case at::kHalf: return FEMTO_F16;
        case at::kBFloat16: return FEMTO_BF16;
        default: throw NotHere{};
    }
}

void* stream_of(const at::Tensor& t) {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

// The calls below launch on the current device, and a call that is being
// captured into a graph gets a workspace of its own: both left to the Python
// path where they apply.
void need_current_device(const at::Tensor& t) {
    int dev = -1;
    need(hipGetDevice(&dev) == hipSuccess && dev == t.device().index());
}
void need_not_captured(void* stream) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    const bool known = hipStreamIsCapturing((hipStream_t)stream, &status) == hipSuccess;
    if (!known) (void)hipGetLastError();
    need(known && status == hipStreamCaptureStatusNone);
}

const int32_t* i32(const at::Tensor& t) { return static_cast<const int32_t*>(t.const_data_ptr()); }

// (pointer, bytes) of the (device, stream) entry of a workspace dict, 256-byte aligned as the Python
// layer aligns it; the entry has to hold nbytes + 256.
struct Workspace {
    void* ptr = nullptr;
    size_t bytes = 0;
    at::Tensor hold;  // another thread may replace the dict's entry during the call
};
Workspace workspace(PyObject* dict, const at::Tensor& on, void* stream, size_t nbytes) {
    Workspace w;
    if (nbytes == 0) return w;
    need(PyDict_CheckExact(dict));
    PyObject* key = Py_BuildValue("(iK)", (int)on.device().index(), (unsigned long long)(uintptr_t)stream);
    need(key != nullptr);
    PyObject* o = PyDict_GetItemWithError(dict, key);  // borrowed
    Py_DECREF(key);
    if (!o) PyErr_Clear();
    need(o != nullptr);
    const at::Tensor& t = tensor(o);
    need((size_t)t.numel() >= nbytes + 256);
    const uintptr_t p = (uintptr_t)t.data_ptr(), a = (p + 255) & ~(uintptr_t)255;
    w.ptr = (void*)a;
    w.bytes = (size_t)t.numel() - (a - p);
    w.hold = t;
    return w;
}

// The checks that the decode and the prefill call share (_check_paged in _C.py).
void check_paged(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& tables,
                 const at::Tensor& kv_lens, bool contiguous_q, int64_t unit_bytes, int64_t unit_elems) {
    need(q.is_cuda() && k.is_cuda() && v.is_cuda());
    need(!contiguous_q || q.is_contiguous());
    need(q.dim() == 3 && k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes());
    need(k.is_contiguous() && v.is_contiguous());
    const int64_t d = q.size(2);
    need(d == k.size(3) && q.stride(2) == 1);
    need(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type());
    need(tables.scalar_type() == at::kInt && kv_lens.scalar_type() == at::kInt);
    need(tables.dim() == 2 && (tables.size(1) <= 1 || tables.stride(1) == 1));
    need(kv_lens.dim() == 1 && kv_lens.is_contiguous());
    need(tables.device() == q.device() && kv_lens.device() == q.device());
    need(k.size(2) == 16 && d > 0 && d <= 128);
    need((d * q.element_size()) % unit_bytes == 0 && d % unit_elems == 0);
    need(k.size(1) > 0 && q.size(0) % k.size(1) == 0);
}

// The library call and its result.  The result's Python object is made first and whatever the library
// throws is an error: nothing can decline the call once the library has been entered (the Python path
// would make it a second time, on a q that the first may have overwritten).
// HOLD_GIL: for calls of more than one launch over the stream's workspace, which
// another thread's call on the stream must not come between.
template <bool HOLD_GIL = false, typename F>
PyObject* launch_for(PyObject* result, F call) {
    int rc;
    PyThreadState* gil = HOLD_GIL ? nullptr : PyEval_SaveThread();
    try {
        rc = call();
    } catch (...) {
        rc = -1;
    }
    if (!HOLD_GIL) PyEval_RestoreThread(gil);
    if (rc == 0) return result;
    Py_DECREF(result);
    PyErr_SetString(PyExc_RuntimeError, rc < 0 ? "femto_native: the library threw" : g_last_error());
    return nullptr;
}

template <bool HOLD_GIL = false, typename F>
PyObject* launch(const at::Tensor& out, F call) {
    PyObject* result = THPVariable_Wrap(out);
    need(result != nullptr);
    return launch_for<HOLD_GIL>(result, call);
}

template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F f) {
    try {
        need(n == want && g_gemv);
        return f();
    } catch (const NotHere&) {
    } catch (const std::exception&) {  // raised again, as Python sees it, by the Python path
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}

// gemv(q, k_pool, v_pool, tables, kv_lens, max_kv_len, contiguous_q, max_kv_len_limit, workspaces)
PyObject* gemv(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 9, [&]() -> PyObject* {
        const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]), &tab = tensor(a[3]), &len = tensor(a[4]);
        const int max_kv = int32(integer(a[5]));
        check_paged(q, k, v, tab, len, a[6] == Py_True, 16, 1);
        const int64_t H = q.size(0), B = q.size(1);
        need(B > 0 && B == tab.size(0) && B == len.size(0));
        need(a[7] == Py_None || max_kv <= integer(a[7]));
        const int dt = dtype_code(q);
        void* st = stream_of(q);
        const Workspace w = workspace(a[8], q, st, g_gemv_ws(int32(B), int32(H), max_kv));
        at::Tensor out = at::empty({H, B, q.size(2)}, q.options());
        const void *qp = q.const_data_ptr(), *kp = k.const_data_ptr(), *vp = v.const_data_ptr();
        const int32_t *tp = i32(tab), *lp = i32(len);
        void* op = out.data_ptr();
        return launch(out, [&] {
            return g_gemv(dt, qp, q.stride(0), q.stride(1), op, out.stride(0), out.stride(1), kp, vp, k.size(0), (int)k.size(1),
                          (int)k.size(2), (int)k.size(3), k.stride(0), k.stride(1), k.stride(2), tp, (int)tab.size(1),
                          tab.stride(0), lp, (int)B, (int)H, max_kv, w.ptr, w.bytes, st);
        });
    });
}

// Whether the pools, too, are on q's device, and that device is the current one.
void need_one_device(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
    need(k.device() == q.device() && v.device() == q.device());
    need_current_device(q);
}

// A window or sinks argument: those past int32 see as many keys as the largest int32.
int key_count(PyObject* o, int64_t lowest) {
    const int64_t n = integer(o);
    need(n >= lowest);
    return (int)std::min<int64_t>(n, INT32_MAX);
}

// gemv_window(q, k_pool, v_pool, tables, kv_lens, max_kv_len, window, sinks, workspaces)
PyObject* gemv_window(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 9, [&]() -> PyObject* {
        need(g_gemv_window);
        const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]), &tab = tensor(a[3]), &len = tensor(a[4]);
        const int max_kv = int32(integer(a[5])), window = key_count(a[6], 1), sinks = key_count(a[7], 0);
        check_paged(q, k, v, tab, len, false, 16, 1);
        need_one_device(q, k, v);
        const int64_t H = q.size(0), B = q.size(1);
        need(B > 0 && B == tab.size(0) && B == len.size(0));
        const int dt = dtype_code(q);
        void* st = stream_of(q);
        const size_t bytes = g_gemv_window_ws(dt, int32(B), int32(H), (int)k.size(1), max_kv, window, sinks);
        if (bytes) need_not_captured(st);
        const Workspace w = workspace(a[8], q, st, bytes);
        at::Tensor out = at::empty({H, B, q.size(2)}, q.options());
        const void *qp = q.const_data_ptr(), *kp = k.const_data_ptr(), *vp = v.const_data_ptr();
        const int32_t *tp = i32(tab), *lp = i32(len);
        void* op = out.data_ptr();
        return launch<true>(out, [&] {
            return g_gemv_window(dt, qp, q.stride(0), q.stride(1), op, out.stride(0), out.stride(1), kp, vp, k.size(0),
                                 (int)k.size(1), (int)k.size(2), (int)k.size(3), k.stride(0), k.stride(1), k.stride(2), tp,
                                 (int)tab.size(1), tab.stride(0), lp, (int)B, (int)H, max_kv, window, sinks, w.ptr, w.bytes, st);
        });
    });
}

// gemv_shared(q, k_pool, v_pool, prefix_pages, tables, kv_lens, max_kv_len, workspaces)
PyObject* gemv_shared(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&]() -> PyObject* {
        need(g_shared);
        const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]), &pre = tensor(a[3]);
        const at::Tensor &tab = tensor(a[4]), &len = tensor(a[5]);
        const int max_kv = int32(integer(a[6]));
        check_paged(q, k, v, tab, len, false, 1, 16);
        need_one_device(q, k, v);
        need(pre.scalar_type() == at::kInt && pre.dim() == 1 && pre.is_contiguous() && pre.device() == q.device());
        const int64_t H = q.size(0), B = q.size(1);
        need(B > 0 && B == tab.size(0) && B == len.size(0));
        need(q.scalar_type() != at::kFloat);
        const int dt = dtype_code(q), pages = int32(pre.size(0));
        void* st = stream_of(q);
        need_not_captured(st);
        const size_t bytes = g_shared_ws(int32(B), int32(H), (int)k.size(1), pages, max_kv);
        need(bytes > 0);
        const Workspace w = workspace(a[7], q, st, bytes);
        at::Tensor out = at::empty({H, B, q.size(2)}, q.options());
        const void *qp = q.const_data_ptr(), *kp = k.const_data_ptr(), *vp = v.const_data_ptr();
        const int32_t *pp = i32(pre), *tp = i32(tab), *lp = i32(len);
        void* op = out.data_ptr();
        return launch<true>(out, [&] {
            return g_shared(dt, qp, q.stride(0), q.stride(1), op, out.stride(0), out.stride(1), kp, vp, k.size(0), (int)k.size(1),
                            (int)k.size(2), (int)k.size(3), k.stride(0), k.stride(1), k.stride(2), pp, pages, tp,
                            (int)tab.size(1), tab.stride(0), lp, (int)B, (int)H, max_kv, w.ptr, w.bytes, st);
        });
    });
}

// gemm(q, k_pool, v_pool, cu_seqlens, max_q_len, tables, kv_lens, positions, contiguous_q, workspaces)
PyObject* gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 10, [&]() -> PyObject* {
        const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]), &cu = tensor(a[3]);
        const at::Tensor &tab = tensor(a[5]), &len = tensor(a[6]), &pos = tensor(a[7]);
        const int max_q = int32(integer(a[4]));
        check_paged(q, k, v, tab, len, a[8] == Py_True, 1, 16);
        need(cu.scalar_type() == at::kInt && cu.is_contiguous() && cu.device() == q.device());
        need(pos.scalar_type() == at::kInt && pos.is_contiguous() && pos.device() == q.device());
        const int64_t H = q.size(0), T = q.size(1), B = cu.numel() - 1;
        need(B > 0 && T > 0 && B == tab.size(0) && B == len.size(0) && T == pos.numel());
        need(q.scalar_type() != at::kFloat);
        const int dt = dtype_code(q);
        void* st = stream_of(q);
        const Workspace w = workspace(a[9], q, st, g_gemm_ws(int32(B), int32(T), max_q, int32(H), (int)k.size(1),
                                                             int32(tab.size(1))));
        at::Tensor out = at::empty({H, T, q.size(2)}, q.options());
        const void *qp = q.const_data_ptr(), *kp = k.const_data_ptr(), *vp = v.const_data_ptr();
        const int32_t *cp = i32(cu), *tp = i32(tab), *lp = i32(len), *pp = i32(pos);
        void* op = out.data_ptr();
        return launch(out, [&] {
            return g_gemm(dt, qp, q.stride(0), q.stride(1), op, out.stride(0), out.stride(1), kp, vp, k.size(0), (int)k.size(1),
                          (int)k.size(2), (int)k.size(3), k.stride(0), k.stride(1), k.stride(2), cp, (int)B, (int)T, max_q, (int)H,
                          tp, (int)tab.size(1), tab.stride(0), lp, pp, w.ptr, w.bytes, st);
        });
    });
}

// gemm_window(q, k_pool, v_pool, cu_seqlens, max_q_len, tables, kv_lens, positions, window, sinks, workspaces)
PyObject* gemm_window(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 11, [&]() -> PyObject* {
        need(g_gemm_window);
        const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]), &cu = tensor(a[3]);
        const at::Tensor &tab = tensor(a[5]), &len = tensor(a[6]), &pos = tensor(a[7]);
        const int max_q = int32(integer(a[4])), window = key_count(a[8], 1), sinks = key_count(a[9], 0);
        check_paged(q, k, v, tab, len, false, 1, 16);
        need_one_device(q, k, v);
        need(cu.scalar_type() == at::kInt && cu.is_contiguous() && cu.device() == q.device());
        need(pos.scalar_type() == at::kInt && pos.is_contiguous() && pos.device() == q.device());
        const int64_t H = q.size(0), T = q.size(1), B = cu.numel() - 1;
        need(B > 0 && T > 0 && B == tab.size(0) && B == len.size(0) && T == pos.numel());
        need(q.scalar_type() != at::kFloat);
        const int dt = dtype_code(q);
        void* st = stream_of(q);
        const size_t bytes = g_gemm_window_ws(int32(B), int32(T), max_q, int32(H), (int)k.size(1), int32(tab.size(1)), window,
                                              sinks);
        if (bytes) need_not_captured(st);
        const Workspace w = workspace(a[10], q, st, bytes);
        at::Tensor out = at::empty({H, T, q.size(2)}, q.options());
        const void *qp = q.const_data_ptr(), *kp = k.const_data_ptr(), *vp = v.const_data_ptr();
        const int32_t *cp = i32(cu), *tp = i32(tab), *lp = i32(len), *pp = i32(pos);
        void* op = out.data_ptr();
        return launch<true>(out, [&] {
            return g_gemm_window(dt, qp, q.stride(0), q.stride(1), op, out.stride(0), out.stride(1), kp, vp, k.size(0),
                                 (int)k.size(1), (int)k.size(2), (int)k.size(3), k.stride(0), k.stride(1), k.stride(2), cp, (int)B,
                                 (int)T, max_q, (int)H, tp, (int)tab.size(1), tab.stride(0), lp, pp, window, sinks, w.ptr, w.bytes,
                                 st);
        });
    });
}

// prologue(q, k, v, q_weight, k_weight, eps, cos, sin, positions, k_pool, v_pool, tables, cu_seqlens | None,
//          max_q_len, out | None)
PyObject* prologue(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 15, [&]() -> PyObject* {
        const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]), &wq = tensor(a[3]), &wk = tensor(a[4]);
        const at::Tensor &cos = tensor(a[6]), &sin = tensor(a[7]), &pos = tensor(a[8]);
        const at::Tensor &kp = tensor(a[9]), &vp = tensor(a[10]), &tab = tensor(a[11]);
        need(PyFloat_CheckExact(a[5]));
        const float eps = (float)PyFloat_AS_DOUBLE(a[5]);
        const int max_q = int32(integer(a[13]));
        need(q.is_cuda());
        for (const at::Tensor* t : {&k, &v, &wq, &wk, &cos, &sin, &kp, &vp, &pos, &tab}) need(t->device() == q.device());
        need(q.dim() == 3 && k.dim() == 3 && v.dim() == 3 && k.sizes() == v.sizes());
        need(q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.size(2) == 128);
        need(q.stride(2) == 1 && k.stride(2) == 1 && v.stride(2) == 1);
        need(wq.numel() == 128 && wk.numel() == 128 && wq.is_contiguous() && wk.is_contiguous());
        for (const at::Tensor* t : {&k, &v, &wq, &wk, &kp, &vp}) need(t->scalar_type() == q.scalar_type());
        need(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat);
        need(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.strides() == sin.strides() && cos.stride(1) == 1 &&
             cos.size(1) >= 128);
        need(kp.dim() == 4 && kp.sizes() == vp.sizes() && kp.is_contiguous() && vp.is_contiguous());
        need(k.size(1) == kp.size(1) && kp.size(3) == 128 && kp.size(2) == 16);
        need(k.size(1) > 0 && q.size(1) % k.size(1) == 0);
        need(pos.scalar_type() == at::kInt && pos.is_contiguous());
        need(tab.scalar_type() == at::kInt && tab.dim() == 2 && (tab.size(1) <= 1 || tab.stride(1) == 1));
        const int64_t T = q.size(0), B = tab.size(0);
        need(T > 0 && B > 0 && pos.numel() == T);
        const int32_t* cp = nullptr;
        if (a[12] == Py_None) {
            need(T == B);
        } else {
            const at::Tensor& cu = tensor(a[12]);
            need(cu.scalar_type() == at::kInt && cu.is_contiguous() && cu.device() == q.device() && cu.numel() - 1 == B);
            cp = i32(cu);
        }
        const int dt = dtype_code(q);
        at::Tensor out = a[14] == Py_None ? at::empty_like(q) : tensor(a[14]);
        need(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.stride(2) == 1 &&
             out.device() == q.device());
        void* st = stream_of(q);
        const void *qd = q.const_data_ptr(), *kd = k.const_data_ptr(), *vd = v.const_data_ptr();
        const void *wqd = wq.const_data_ptr(), *wkd = wk.const_data_ptr();
        const float* cd = static_cast<const float*>(cos.const_data_ptr());
        const float* sd = static_cast<const float*>(sin.const_data_ptr());
        void *od = out.data_ptr(), *kpd = kp.data_ptr(), *vpd = vp.data_ptr();
        const int32_t *pd = i32(pos), *td = i32(tab);
        const int H = int32(q.size(1)), rows = int32(cos.size(0)), tokens = int32(T), seqs = int32(B);
        return launch(out, [&] {
            return g_prologue(dt, qd, q.stride(0), q.stride(1), kd, k.stride(0), k.stride(1), vd, v.stride(0), v.stride(1), od,
                              out.stride(0), out.stride(1), wqd, wkd, eps, cd, sd, cos.stride(0), rows, kpd, vpd, kp.size(0), H,
                              (int)kp.size(1), (int)kp.size(2), (int)kp.size(3), kp.stride(0), kp.stride(1), kp.stride(2), cp, seqs,
                              tokens, max_q, pd, td, (int)tab.size(1), tab.stride(0), st);
        });
    });
}

// Whether two (tokens, heads, dim) tensors contiguous in dim plainly have no element in common: their spans do not
// meet, or they are columns of one array of token rows.  (The Python path looks at every row.)
bool plainly_apart(const at::Tensor& a, const at::Tensor& b) {
    const int64_t size = a.element_size();
    const int64_t row_a = (a.size(1) - 1) * a.stride(1) + a.size(2), row_b = (b.size(1) - 1) * b.stride(1) + b.size(2);
    const int64_t pa = (int64_t)(uintptr_t)a.const_data_ptr(), pb = (int64_t)(uintptr_t)b.const_data_ptr();
    if (pa + size * ((a.size(0) - 1) * a.stride(0) + row_a) <= pb || pb + size * ((b.size(0) - 1) * b.stride(0) + row_b) <= pa)
        return true;
    const int64_t step = a.stride(0);
    if (step <= 0 || step != b.stride(0) || (pb - pa) % size) return false;
    const int64_t at = ((pb - pa) / size % step + step) % step;  // b's first column
    return row_a <= at && at + row_b <= step;
}

// rope(q, k, v, cos, sin, positions, k_pool, v_pool, tables, cu_seqlens | None, max_q_len, interleaved, out | None)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 13, [&]() -> PyObject* {
        need(g_rope);
        const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]), &cos = tensor(a[3]), &sin = tensor(a[4]);
        const at::Tensor &pos = tensor(a[5]), &kp = tensor(a[6]), &vp = tensor(a[7]), &tab = tensor(a[8]);
        const int max_q = int32(integer(a[10]));
        need(PyBool_Check(a[11]));
        const int interleaved = a[11] == Py_True;
        need(q.is_cuda());
        for (const at::Tensor* t : {&k, &v, &cos, &sin, &kp, &vp, &pos, &tab}) need(t->device() == q.device());
        need_current_device(q);
        need(q.dim() == 3 && k.dim() == 3 && v.dim() == 3 && k.sizes() == v.sizes());
        need(q.size(0) == k.size(0) && q.size(2) == k.size(2));
        need(q.stride(2) == 1 && k.stride(2) == 1 && v.stride(2) == 1);
        for (const at::Tensor* t : {&k, &v, &kp, &vp}) need(t->scalar_type() == q.scalar_type());
        need(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat);
        need(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.strides() == sin.strides() && cos.stride(1) == 1);
        need(kp.dim() == 4 && kp.sizes() == vp.sizes() && kp.is_contiguous() && vp.is_contiguous());
        need(k.size(1) == kp.size(1) && kp.size(3) == q.size(2) && kp.size(2) == 16 && q.size(1) > 0 && k.size(1) > 0);
        need(pos.scalar_type() == at::kInt && pos.is_contiguous());
        need(tab.scalar_type() == at::kInt && tab.dim() == 2 && (tab.size(1) <= 1 || tab.stride(1) == 1));
        need(cos.stride(0) >= cos.size(1) && tab.stride(0) >= tab.size(1));
        const int64_t T = q.size(0), B = tab.size(0);
        need(T > 0 && B > 0 && pos.numel() == T);
        const int32_t* cp = nullptr;
        if (a[9] == Py_None) {
            need(T == B);
        } else {
            const at::Tensor& cu = tensor(a[9]);
            need(cu.scalar_type() == at::kInt && cu.is_contiguous() && cu.device() == q.device() && cu.numel() - 1 == B);
            cp = i32(cu);
        }
        const int dt = dtype_code(q);
        at::Tensor out = a[12] == Py_None ? at::empty_like(q) : tensor(a[12]);
        need(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.stride(2) == 1 && out.device() == q.device());
        if (a[12] != Py_None) {
            need(out.const_data_ptr() == q.const_data_ptr() && out.strides() == q.strides());
            need(plainly_apart(out, k) && plainly_apart(out, v));
            need(out.stride(1) >= out.size(2) || out.size(1) == 1);  // its rows, head by head and token by token
            need(out.stride(0) >= (out.size(1) - 1) * out.stride(1) + out.size(2) || out.size(0) == 1);
        }
        void* st = stream_of(q);
        const void *qd = q.const_data_ptr(), *kd = k.const_data_ptr(), *vd = v.const_data_ptr();
        const float* cd = static_cast<const float*>(cos.const_data_ptr());
        const float* sd = static_cast<const float*>(sin.const_data_ptr());
        void *od = out.data_ptr(), *kpd = kp.data_ptr(), *vpd = vp.data_ptr();
        const int32_t *pd = i32(pos), *td = i32(tab);
        const int H = int32(q.size(1)), rows = int32(cos.size(0)), R = int32(2 * cos.size(1)), tokens = int32(T), seqs = int32(B);
        return launch(out, [&] {
            return g_rope(dt, qd, q.stride(0), q.stride(1), kd, k.stride(0), k.stride(1), vd, v.stride(0), v.stride(1), od,
                          out.stride(0), out.stride(1), cd, sd, cos.stride(0), rows, R, interleaved, kpd, vpd, kp.size(0), H,
                          (int)kp.size(1), (int)kp.size(2), (int)kp.size(3), kp.stride(0), kp.stride(1), kp.stride(2), cp, seqs,
                          tokens, max_q, pd, td, (int)tab.size(1), tab.stride(0), st);
        });
    });
}

// ---- calls over a KV cache held in 4 bits (the checks of _C.py) ----

void check_fp4_pool(const at::Tensor& pool, int64_t dim, const at::Device& dev) {
    need(pool.is_cuda() && pool.device() == dev && pool.scalar_type() == at::kByte && pool.dim() == 3 && pool.is_contiguous());
    need(dim > 0 && dim <= 128 && dim % 16 == 0 && pool.size(1) > 0 && pool.size(2) == (int64_t)g_fp4_page((int)dim));
}

// Positions, tables and cu_seqlens (or None) of a cache write of T > 0 tokens.
struct Placement {
    const int32_t *cu = nullptr, *positions, *tables;
    int seqs, tokens, width;
    int64_t stride;
};
Placement placement(PyObject* pos_o, PyObject* tab_o, PyObject* cu_o, int64_t T, const at::Device& dev) {
    const at::Tensor &pos = tensor(pos_o), &tab = tensor(tab_o);
    need(pos.scalar_type() == at::kInt && pos.is_contiguous() && pos.device() == dev && pos.numel() == T);
    need(tab.scalar_type() == at::kInt && tab.dim() == 2 && tab.device() == dev && (tab.size(1) <= 1 || tab.stride(1) == 1));
    Placement p;
    p.seqs = int32(tab.size(0));
    p.tokens = int32(T);
    p.width = int32(tab.size(1));
    need(p.seqs > 0 && T > 0);
    p.stride = p.seqs > 1 ? tab.stride(0) : std::max(tab.stride(0), tab.size(1));
    if (cu_o == Py_None) {
        need(T == p.seqs);
    } else {
        const at::Tensor& cu = tensor(cu_o);
        need(cu.scalar_type() == at::kInt && cu.is_contiguous() && cu.device() == dev && cu.numel() - 1 == p.seqs);
        p.cu = i32(cu);
    }
    p.positions = i32(pos);
    p.tables = i32(tab);
    return p;
}

int check_kv_source(const at::Tensor& k, const at::Tensor& v, const at::Tensor& pool) {
    need(k.is_cuda() && v.device() == k.device() && k.dim() == 3 && v.dim() == 3 && k.sizes() == v.sizes());
    need(k.stride(2) == 1 && v.stride(2) == 1 && k.scalar_type() == v.scalar_type() && k.scalar_type() != at::kFloat);
    check_fp4_pool(pool, k.size(2), k.device());
    need(k.size(1) == pool.size(1));
    need_current_device(k);
    return dtype_code(k);
}

// write_fp4(k, v, kv_pool, positions, tables, cu_seqlens | None, max_q_len): True where it was made
PyObject* write_fp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 7, [&]() -> PyObject* {
        need(g_write_fp4 && g_fp4_page);
        const at::Tensor &k = tensor(a[0]), &v = tensor(a[1]), &pool = tensor(a[2]);
        const int max_q = int32(integer(a[6]));
        const int dt = check_kv_source(k, v, pool);
        const Placement p = placement(a[3], a[4], a[5], k.size(0), k.device());
        void *st = stream_of(k), *pp = pool.data_ptr();
        const void *kd = k.const_data_ptr(), *vd = v.const_data_ptr();
        Py_INCREF(Py_True);
        return launch_for(Py_True, [&] {
            return g_write_fp4(dt, kd, k.stride(0), k.stride(1), vd, v.stride(0), v.stride(1), pp, pool.size(0), (int)pool.size(1),
                               (int)k.size(2), p.cu, p.seqs, p.tokens, max_q, p.positions, p.tables, p.width, p.stride, st);
        });
    });
}

// read_fp4(kv_pool, head_dim, bf16, positions, tables, cu_seqlens | None, max_q_len): (k, v)
PyObject* read_fp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 7, [&]() -> PyObject* {
        need(g_read_fp4 && g_fp4_page);
        const at::Tensor& pool = tensor(a[0]);
        const int64_t dim = integer(a[1]), T = tensor(a[3]).numel();
        need(PyBool_Check(a[2]));
        const bool bf16 = a[2] == Py_True;
        const int max_q = int32(integer(a[6]));
        check_fp4_pool(pool, dim, pool.device());
        need_current_device(pool);
        const Placement p = placement(a[3], a[4], a[5], T, pool.device());
        const auto options = pool.options().dtype(bf16 ? at::kBFloat16 : at::kHalf);
        at::Tensor k = at::empty({T, pool.size(1), dim}, options), v = at::empty({T, pool.size(1), dim}, options);
        PyObject *ko = THPVariable_Wrap(k), *vo = ko ? THPVariable_Wrap(v) : nullptr;
        PyObject* both = vo ? PyTuple_Pack(2, ko, vo) : nullptr;
        Py_XDECREF(ko);
        Py_XDECREF(vo);
        need(both != nullptr);
        void *st = stream_of(pool), *kd = k.data_ptr(), *vd = v.data_ptr();
        const void* pp = pool.const_data_ptr();
        return launch_for(both, [&] {
            return g_read_fp4(bf16 ? FEMTO_BF16 : FEMTO_F16, pp, pool.size(0), (int)pool.size(1), (int)dim, kd, vd, p.cu, p.seqs,
                              p.tokens, max_q, p.positions, p.tables, p.width, p.stride, st);
        });
    });
}

// rope_fp4(q, k, v, cos, sin, positions, kv_pool, tables, cu_seqlens | None, max_q_len, interleaved, q_weight | None,
//          k_weight | None, eps, out | None)
PyObject* rope_fp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 15, [&]() -> PyObject* {
        need(g_rope_fp4 && g_fp4_page);
        const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]), &cos = tensor(a[3]), &sin = tensor(a[4]);
        const at::Tensor& pool = tensor(a[6]);
        const int max_q = int32(integer(a[9]));
        need(PyBool_Check(a[10]) && PyFloat_CheckExact(a[13]));
        const int interleaved = a[10] == Py_True;
        const double eps = PyFloat_AS_DOUBLE(a[13]);
        const int dt = check_kv_source(k, v, pool);
        for (const at::Tensor* t : {&q, &cos, &sin}) need(t->device() == k.device());
        need(q.dim() == 3 && q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.size(1) > 0 && q.stride(2) == 1);
        need(q.scalar_type() == k.scalar_type());
        need(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat);
        need(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.strides() == sin.strides() && cos.stride(1) == 1);
        need(cos.stride(0) >= cos.size(1));
        const void *wq = nullptr, *wk = nullptr;
        need((a[11] == Py_None) == (a[12] == Py_None));
        if (a[11] != Py_None) {
            const at::Tensor &x = tensor(a[11]), &y = tensor(a[12]);
            for (const at::Tensor* t : {&x, &y})
                need(t->device() == q.device() && t->scalar_type() == q.scalar_type() && t->dim() == 1 && t->is_contiguous() &&
                     t->size(0) == q.size(2));
            wq = x.const_data_ptr();
            wk = y.const_data_ptr();
        }
        const Placement p = placement(a[5], a[7], a[8], k.size(0), k.device());
        at::Tensor out = a[14] == Py_None ? at::empty_like(q) : tensor(a[14]);
        need(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.stride(2) == 1 && out.device() == q.device());
        if (a[14] != Py_None) {
            need(out.const_data_ptr() == q.const_data_ptr() && out.strides() == q.strides());
            need(plainly_apart(out, k) && plainly_apart(out, v));
            need(out.stride(1) >= out.size(2) || out.size(1) == 1);  // its rows, head by head and token by token
            need(out.stride(0) >= (out.size(1) - 1) * out.stride(1) + out.size(2) || out.size(0) == 1);
        }
        void *st = stream_of(q), *od = out.data_ptr(), *pp = pool.data_ptr();
        const void *qd = q.const_data_ptr(), *kd = k.const_data_ptr(), *vd = v.const_data_ptr();
        const float* cd = static_cast<const float*>(cos.const_data_ptr());
        const float* sd = static_cast<const float*>(sin.const_data_ptr());
        const int H = int32(q.size(1)), rows = int32(cos.size(0)), R = int32(2 * cos.size(1));
        return launch(out, [&] {
            return g_rope_fp4(dt, qd, q.stride(0), q.stride(1), kd, k.stride(0), k.stride(1), vd, v.stride(0), v.stride(1), od,
                              out.stride(0), out.stride(1), wq, wk, eps, cd, sd, cos.stride(0), rows, R, interleaved, pp,
                              pool.size(0), H, (int)pool.size(1), (int)q.size(2), p.cu, p.seqs, p.tokens, max_q, p.positions,
                              p.tables, p.width, p.stride, st);
        });
    });
}

int check_fp4_attention(const at::Tensor& q, const at::Tensor& pool, const at::Tensor& tab, const at::Tensor& len) {
    need(q.is_cuda() && q.dim() == 3 && q.stride(2) == 1 && q.scalar_type() != at::kFloat);
    check_fp4_pool(pool, q.size(2), q.device());
    need(q.size(0) > 0 && q.size(0) % pool.size(1) == 0);
    need(tab.scalar_type() == at::kInt && tab.dim() == 2 && tab.device() == q.device() && (tab.size(1) <= 1 || tab.stride(1) == 1));
    need(len.scalar_type() == at::kInt && len.dim() == 1 && len.is_contiguous() && len.device() == q.device());
    need_current_device(q);
    return dtype_code(q);
}

// gemv_fp4(q, kv_pool, tables, kv_lens, max_kv_len, workspaces)
PyObject* gemv_fp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 6, [&]() -> PyObject* {
        need(g_gemv_fp4 && g_gemv_fp4_ws && g_fp4_page);
        const at::Tensor &q = tensor(a[0]), &pool = tensor(a[1]), &tab = tensor(a[2]), &len = tensor(a[3]);
        const int max_kv = int32(integer(a[4]));
        const int dt = check_fp4_attention(q, pool, tab, len);
        const int64_t H = q.size(0), B = q.size(1);
        need(B > 0 && B == tab.size(0) && B == len.size(0));
        void* st = stream_of(q);
        const size_t bytes = g_gemv_fp4_ws(int32(B), int32(H), (int)pool.size(1), max_kv);
        if (bytes) need_not_captured(st);
        const Workspace w = workspace(a[5], q, st, bytes);
        at::Tensor out = at::empty({H, B, q.size(2)}, q.options());
        const void *qp = q.const_data_ptr(), *pp = pool.const_data_ptr();
        const int32_t *tp = i32(tab), *lp = i32(len);
        void* op = out.data_ptr();
        return launch<true>(out, [&] {
            return g_gemv_fp4(dt, qp, q.stride(0), q.stride(1), op, out.stride(0), out.stride(1), pp, pool.size(0),
                              (int)pool.size(1), (int)q.size(2), tp, (int)tab.size(1), tab.stride(0), lp, (int)B, (int)H, max_kv,
                              w.ptr, w.bytes, st);
        });
    });
}

// gemm_fp4(q, kv_pool, cu_seqlens, max_q_len, tables, kv_lens, positions, workspaces)
PyObject* gemm_fp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&]() -> PyObject* {
        need(g_gemm_fp4 && g_gemm_fp4_ws && g_fp4_page);
        const at::Tensor &q = tensor(a[0]), &pool = tensor(a[1]), &cu = tensor(a[2]), &tab = tensor(a[4]), &len = tensor(a[5]);
        const at::Tensor& pos = tensor(a[6]);
        const int max_q = int32(integer(a[3]));
        const int dt = check_fp4_attention(q, pool, tab, len);
        need(cu.scalar_type() == at::kInt && cu.is_contiguous() && cu.device() == q.device());
        need(pos.scalar_type() == at::kInt && pos.is_contiguous() && pos.device() == q.device());
        const int64_t H = q.size(0), T = q.size(1), B = cu.numel() - 1;
        need(B > 0 && T > 0 && B == tab.size(0) && B == len.size(0) && T == pos.numel());
        void* st = stream_of(q);
        need_not_captured(st);
        const Workspace w = workspace(a[7], q, st, g_gemm_fp4_ws(int32(B), int32(T), max_q, int32(H), (int)pool.size(1),
                                                                 int32(tab.size(1))));
        need(w.ptr != nullptr);
        at::Tensor out = at::empty({H, T, q.size(2)}, q.options());
        const void *qp = q.const_data_ptr(), *pp = pool.const_data_ptr();
        const int32_t *cp = i32(cu), *tp = i32(tab), *lp = i32(len), *sp = i32(pos);
        void* op = out.data_ptr();
        return launch<true>(out, [&] {
            return g_gemm_fp4(dt, qp, q.stride(0), q.stride(1), op, out.stride(0), out.stride(1), pp, pool.size(0),
                              (int)pool.size(1), (int)q.size(2), cp, (int)B, (int)T, max_q, (int)H, tp, (int)tab.size(1),
                              tab.stride(0), lp, sp, w.ptr, w.bytes, st);
        });
    });
}

// flash(q, k, v)
PyObject* flash(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 3, [&]() -> PyObject* {
        const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]);
        for (const at::Tensor* t : {&q, &k, &v})
            need(t->is_cuda() && t->dim() == 4 && t->is_contiguous() && (uintptr_t)t->const_data_ptr() % 16 == 0);
        need(k.sizes() == v.sizes() && q.size(0) == k.size(0) && q.size(3) == k.size(3) && q.size(3) == 128);
        need(k.size(1) > 0 && q.size(1) % k.size(1) == 0);
        need(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type() && q.scalar_type() != at::kFloat);
        const int dt = dtype_code(q);
        at::Tensor out = at::empty_like(q);
        void* st = stream_of(q);
        const void *qp = q.const_data_ptr(), *kp = k.const_data_ptr(), *vp = v.const_data_ptr();
        void* op = out.data_ptr();
        const int B = int32(q.size(0)), H = int32(q.size(1)), KVH = int32(k.size(1)), Tq = int32(q.size(2)),
                  Tk = int32(k.size(2));
        return launch(out, [&] {
            return g_flash(dt, qp, q.stride(0), q.stride(1), q.stride(2), kp, k.stride(0), k.stride(1), k.stride(2), vp,
                           v.stride(0), v.stride(1), v.stride(2), op, out.stride(0), out.stride(1), out.stride(2), B, H, KVH, Tq,
                           Tk, 128, st);
        });
    });
}

// bind({function name: address}): the library's entry points.
PyObject* bind(PyObject*, PyObject* names) {
    auto get = [&](const char* name, auto& fn) {
        PyObject* o = PyDict_Check(names) ? PyDict_GetItemString(names, name) : nullptr;
        void* p = o ? PyLong_AsVoidPtr(o) : nullptr;
        if (!p && !PyErr_Occurred()) PyErr_Format(PyExc_KeyError, "femto_native.bind: no address of %s", name);
        if (p) fn = reinterpret_cast<std::decay_t<decltype(fn)>>(p);
        return p != nullptr;
    };
    if (!get("femto_attn_last_error", g_last_error) || !get("femto_paged_attention_gemv_workspace_size", g_gemv_ws) ||
        !get("femto_paged_attention_gemm", g_gemm) || !get("femto_paged_attention_gemm_workspace_size", g_gemm_ws) ||
        !get("femto_qk_norm_rope_cache_write", g_prologue) || !get("femto_flash_attention", g_flash) ||
        !get("femto_paged_attention_gemv", g_gemv))
        return nullptr;
    // A call whose function is not bound is declined.
    auto optional = [&](const char* name, auto& fn) { return !PyDict_GetItemString(names, name) || get(name, fn); };
    if (!optional("femto_rope_cache_write", g_rope) || !optional("femto_paged_attention_gemv_shared_prefix", g_shared) ||
        !optional("femto_paged_attention_gemv_shared_prefix_workspace_size", g_shared_ws) || !optional("femto_paged_attention_gemv_window", g_gemv_window) ||
        !optional("femto_paged_attention_gemv_window_workspace_size", g_gemv_window_ws) ||
        !optional("femto_paged_attention_gemm_window", g_gemm_window) ||
        !optional("femto_paged_attention_gemm_window_workspace_size", g_gemm_window_ws) ||
        !optional("femto_fp4_page_bytes", g_fp4_page) || !optional("femto_kv_cache_write_fp4", g_write_fp4) ||
        !optional("femto_kv_cache_read_fp4", g_read_fp4) || !optional("femto_rope_cache_write_fp4", g_rope_fp4) ||
        !optional("femto_paged_attention_gemv_fp4", g_gemv_fp4) ||
        !optional("femto_paged_attention_gemv_fp4_workspace_size", g_gemv_fp4_ws) ||
        !optional("femto_paged_attention_gemm_fp4", g_gemm_fp4) ||
        !optional("femto_paged_attention_gemm_fp4_workspace_size", g_gemm_fp4_ws))
        return nullptr;
    Py_RETURN_NONE;
}

#define FEMTO_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {
    {"bind", bind, METH_O, nullptr},
    {"gemv", FEMTO_FAST(gemv)},
    {"gemm", FEMTO_FAST(gemm)},
    {"gemv_window", FEMTO_FAST(gemv_window)},
    {"gemm_window", FEMTO_FAST(gemm_window)},
    {"prologue", FEMTO_FAST(prologue)},
    {"gemv_shared", FEMTO_FAST(gemv_shared)},
    {"rope", FEMTO_FAST(rope)},
    {"write_fp4", FEMTO_FAST(write_fp4)},
    {"read_fp4", FEMTO_FAST(read_fp4)},
    {"rope_fp4", FEMTO_FAST(rope_fp4)},
    {"gemv_fp4", FEMTO_FAST(gemv_fp4)},
    {"gemm_fp4", FEMTO_FAST(gemm_fp4)},
    {"flash", FEMTO_FAST(flash)},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "femto_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_femto_native() { return PyModule_Create(&module); }
