// The host side of one call, from tensors to mmx_gemm_splitk, mmx_gemm_unpacked, mmx_matvec or the packing and quantising
// entry points, as CPython functions (module mm_amx_amd._host_call).
//
// What bounds a small product is the host: the same checks as Python statements, the descriptor as a ctypes structure, the query
// of the workspace and the call through ctypes took 9.7 us for 256 x 256 x 256, under 4 us of which are on the device; 4.7 now.
// (A norm of one row 16.7 -> 5.9, a linear layer in e4m3 of one token 15.8 -> 10.3; one decode row over 512 x 512 int4 weights 9.2 -> 4.2, a 64 x 512 x 512 layer with a bias 10.2 -> 5.2.)  The functions below
// take the calls that are regular in every respect - tensors of exactly torch's own type on one GPU, the current one, everything
// large enough - and leave all others to the Python form (they return None, and have done nothing), which accepts them or says
// what is wrong.  They keep nothing from one call for the next.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/mm_amx_amd.h"

namespace {

using gemm_fn = decltype(&mmx_gemm_splitk);
using need_fn = decltype(&mmx_gemm_workspace_bytes);
using unpacked_fn = decltype(&mmx_gemm_unpacked);
using unpacked_need_fn = decltype(&mmx_gemm_unpacked_workspace_bytes);
using matvec_fn = decltype(&mmx_matvec);
gemm_fn call_gemm = nullptr;  // of the library that the package has loaded, set once
need_fn call_need = nullptr;
unpacked_fn call_unpacked = nullptr;
unpacked_need_fn call_unpacked_need = nullptr;
matvec_fn call_matvec = nullptr;
decltype(&mmx_packed_b_bytes) call_packed_bytes = nullptr;
decltype(&mmx_repack_b) call_repack = nullptr;
decltype(&mmx_quantize_weights_scratch) call_quantize = nullptr;
decltype(&mmx_quantize_weights_scaled) call_quantize_scaled = nullptr;
decltype(&mmx_quantize_pack_int4) call_quantize_int4 = nullptr;
decltype(&mmx_quantize_pack_scaled) call_quantize_pack_scaled = nullptr;

struct Leave {};  // not a regular call

bool whole_number(PyObject* o, long long lo, long long hi, int& v) {
    if (!PyLong_CheckExact(o)) return false;
    int over = 0;
    const long long x = PyLong_AsLongLongAndOverflow(o, &over);
    if (over || x < lo || x > hi) return false;
    v = (int)x;
    return true;
}

int code_of(at::ScalarType t) {
    switch (t) {
    case at::kFloat: return MMX_F32;
    case at::kBFloat16: return MMX_BF16;
    case at::kChar: return MMX_I8;
    case at::kInt: return MMX_I32;
    case at::kByte: return MMX_U8;
    default: return -1;
    }
}

const at::Tensor& tensor_on(PyObject* o, int device) {
    if (!THPVariable_CheckExact(o)) throw Leave();
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.get_device() != device || t.layout() != at::kStrided) throw Leave();
    return t;
}

// a matrix whose elements of a row follow each other; of a single row or column torch leaves the other stride arbitrary
int64_t row_stride_bytes(const at::Tensor& t) {
    if (t.dim() != 2 || (t.stride(1) != 1 && t.size(1) != 1)) throw Leave();
    return (t.size(0) == 1 ? t.size(1) : t.stride(0)) * (int64_t)t.element_size();
}

const float* column_operand(PyObject* o, int device, int n1) {
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor_on(o, device);
    if (t.scalar_type() != at::kFloat || !t.is_contiguous() || t.numel() < n1) throw Leave();
    return static_cast<const float*>(t.mutable_data_ptr());
}

void* stream_of(PyObject* o) {
    void* const stream = PyLong_AsVoidPtr(o);
    if (!stream && PyErr_Occurred()) {
        PyErr_Clear();
        throw Leave();
    }
    return stream;
}

// a: C, steps, bias, deq, deq_per_oc, q, q_per_oc; C holds the M x n1 result (half the columns with SILU_GATE)
mmx_epilogue epilogue_of(PyObject* const* a, int device, int64_t M, int n1) {
    const at::Tensor& C = tensor_on(a[0], device);
    int steps;
    if (!whole_number(a[1], 0, INT32_MAX, steps) || !PyFloat_CheckExact(a[3]) || !PyFloat_CheckExact(a[5])) throw Leave();
    mmx_epilogue e = {};
    e.steps = (uint32_t)steps;
    e.out_dtype = code_of(C.scalar_type());
    e.ldc_bytes = row_stride_bytes(C);
    if (e.out_dtype < 0 || C.size(0) < M || C.size(1) < ((steps & MMX_PP_SILU_GATE) ? n1 / 2 : n1)) throw Leave();
    e.C = C.mutable_data_ptr();
    e.bias = column_operand(a[2], device, n1);
    e.deq_scale = (float)PyFloat_AS_DOUBLE(a[3]);
    e.deq_scale_per_oc = column_operand(a[4], device, n1);
    e.q_scale = (float)PyFloat_AS_DOUBLE(a[5]);
    e.q_scale_per_oc = column_operand(a[6], device, n1);
    return e;
}

// gemm(A, Bpacked, N, b_dtype, n0, n1, k_splits, ws, device, stream, C, steps, bias, deq, deq_per_oc, q, q_per_oc)
//   b_dtype: None = that of A; n1: None = N; ws: None = unsplit if the call has no use for one
PyObject* gemm(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 17 || !call_gemm) Py_RETURN_NONE;
    int rc;
    try {
        int N, n0, n1, ks, device, b_dt;
        if (!whole_number(a[8], 0, 1 << 20, device) || !whole_number(a[2], 1, INT32_MAX, N)) throw Leave();
        n1 = N;
        if (a[5] != Py_None && !whole_number(a[5], 1, N, n1)) throw Leave();
        if (!whole_number(a[4], 0, n1 - 1, n0) || !whole_number(a[6], 0, 1 << 20, ks)) throw Leave();
        const at::Tensor &A = tensor_on(a[0], device), &B = tensor_on(a[1], device);
        const int64_t lda = row_stride_bytes(A), M = A.size(0), K = A.size(1);
        const int a_dt = code_of(A.scalar_type());
        if (M < 1 || M > INT32_MAX || K < 1 || K > INT32_MAX || (a_dt != MMX_BF16 && a_dt != MMX_I8)) throw Leave();
        b_dt = a_dt;
        if (a[3] != Py_None && !whole_number(a[3], 0, 255, b_dt)) throw Leave();
        if (b_dt != MMX_BF16 && b_dt != MMX_I8 && b_dt != MMX_I4) throw Leave();
        // everything that the kernels take on trust: what is too small is an error, and the Python form says which
        const int64_t panels = ((int64_t)N + 31) / 32;
        const int64_t need = b_dt == MMX_I4 ? panels * ((K + 255) / 256 * 4) * 1024 : panels * 32 * ((K * (b_dt == MMX_BF16 ? 2 : 1) + 127) / 128 * 128);
        if (B.scalar_type() != at::kByte || !B.is_contiguous() || B.numel() < need) throw Leave();
        const mmx_epilogue e = epilogue_of(a + 10, device, M, n1);
        void* ws = nullptr;
        size_t ws_bytes = 0;
        if (a[7] != Py_None) {
            const at::Tensor& w = tensor_on(a[7], device);
            if (w.scalar_type() != at::kByte || !w.is_contiguous()) throw Leave();
            ws = w.mutable_data_ptr();
            ws_bytes = (size_t)w.numel();
        } else if (ks != 1) {
            // an explicit count of slices, or a first call that has a use for a workspace: it is made outside
            if (ks || call_need(a_dt, b_dt, (int)M, (int)K, N, n0, n1, e.steps, 0)) throw Leave();
            ks = 1;
        }
        void* const stream = stream_of(a[9]);
        const void *pa = A.mutable_data_ptr(), *pb = B.mutable_data_ptr();
        Py_BEGIN_ALLOW_THREADS
        rc = call_gemm(a_dt, b_dt, pa, lda, pb, (int)M, (int)K, N, n0, n1, &e, ks, ws, ws_bytes, stream);
        Py_END_ALLOW_THREADS
    } catch (...) {  // (tensors without memory of their own throw when asked for it)
        Py_RETURN_NONE;
    }
    return PyLong_FromLong(rc);
}

// gemm_unpacked(A, B, transpose, ws, device, stream, C, steps, bias, deq, deq_per_oc, q, q_per_oc): a B that is used once, where
// the library reads it in place
PyObject* gemm_unpacked(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 13 || !call_unpacked) Py_RETURN_NONE;
    int rc;
    try {
        int device;
        if (!whole_number(a[4], 0, 1 << 20, device) || !PyBool_Check(a[2])) throw Leave();
        const int transpose = a[2] == Py_True;
        const at::Tensor &A = tensor_on(a[0], device), &B = tensor_on(a[1], device);
        const int64_t lda = row_stride_bytes(A), ldb = row_stride_bytes(B), M = A.size(0), K = A.size(1), N = B.size(transpose ? 0 : 1);
        if (A.scalar_type() != at::kBFloat16 || B.scalar_type() != at::kBFloat16 || B.size(transpose ? 1 : 0) != K) throw Leave();
        if (M < 1 || M > INT32_MAX || K < 1 || K > INT32_MAX || N < 1 || N > INT32_MAX) throw Leave();
        const int64_t need = call_unpacked_need(MMX_BF16, (int)M, (int)K, (int)N, lda, ldb, transpose);
        if (need < 0) throw Leave();
        const mmx_epilogue e = epilogue_of(a + 6, device, M, (int)N);
        if (e.steps & MMX_PP_SILU_GATE) throw Leave();
        const char *pa = static_cast<const char*>(A.mutable_data_ptr()), *pb = static_cast<const char*>(B.mutable_data_ptr()), *pc = static_cast<const char*>(e.C);
        // (a result that is written over B is not computed from B in place)
        if (pc < pb + (B.size(0) - 1) * ldb + 2 * B.size(1) && pb < pc + (M - 1) * e.ldc_bytes + N * (e.out_dtype == MMX_BF16 ? 2 : (e.out_dtype == MMX_I8 ? 1 : 4))) throw Leave();
        void* ws = nullptr;
        size_t ws_bytes = 0;
        if (need) {
            const at::Tensor& w = tensor_on(a[3], device);
            if (w.numel() < need) throw Leave();  // (it is made outside)
            ws = w.mutable_data_ptr();
            ws_bytes = (size_t)w.numel();
        }
        void* const stream = stream_of(a[5]);
        Py_BEGIN_ALLOW_THREADS
        rc = call_unpacked(MMX_BF16, pa, lda, pb, ldb, transpose, (int)M, (int)K, (int)N, &e, ws, ws_bytes, stream);
        Py_END_ALLOW_THREADS
    } catch (...) {
        Py_RETURN_NONE;
    }
    return PyLong_FromLong(rc);
}

// matvec(A, b, out, device, stream)
PyObject* matvec(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 5 || !call_matvec) Py_RETURN_NONE;
    int rc;
    try {
        int device;
        if (!whole_number(a[3], 0, 1 << 20, device)) throw Leave();
        const at::Tensor &A = tensor_on(a[0], device), &b = tensor_on(a[1], device), &c = tensor_on(a[2], device);
        const int64_t lda = row_stride_bytes(A), M = A.size(0), K = A.size(1);
        const int dt = code_of(A.scalar_type());
        if (M < 1 || M > INT32_MAX || K < 1 || K > INT32_MAX || (dt != MMX_BF16 && dt != MMX_I8)) throw Leave();
        if (b.scalar_type() != A.scalar_type() || b.numel() != K || !b.is_contiguous()) throw Leave();
        if (c.scalar_type() != (dt == MMX_BF16 ? at::kFloat : at::kInt) || c.numel() < M || !c.is_contiguous()) throw Leave();
        const void *pa = A.mutable_data_ptr(), *pb = b.mutable_data_ptr();
        void *pc = c.mutable_data_ptr(), *stream = stream_of(a[4]);
        Py_BEGIN_ALLOW_THREADS
        rc = call_matvec(dt, pa, lda, pb, pc, (int)M, (int)K, stream);
        Py_END_ALLOW_THREADS
    } catch (...) {
        Py_RETURN_NONE;
    }
    return PyLong_FromLong(rc);
}

// ---- packing and quantising: results are made here; an error of the library comes back as its number -------------------
// f() with the interpreter's lock released, as torch's own calls and ctypes have it; what it throws (no memory
// left, say) is left to the Python form, which then says so
template <typename F>
bool unlocked(F&& f) {
    bool ok = true;
    PyThreadState* const state = PyEval_SaveThread();
    try {
        f();
    } catch (...) {
        ok = false;
    }
    PyEval_RestoreThread(state);
    return ok;
}

at::Tensor make(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
    return at::empty(sizes, at::TensorOptions().dtype(type).device(like.device()));
}

struct Matrix {
    const at::Tensor* t;
    int64_t ld;
    int rows, cols;
    const void* data;
};
Matrix matrix(PyObject* o, int device) {
    const at::Tensor& t = tensor_on(o, device);
    const int64_t ld = row_stride_bytes(t);
    if (t.size(0) < 1 || t.size(0) > INT32_MAX || t.size(1) < 1 || t.size(1) > INT32_MAX) throw Leave();
    return {&t, ld, (int)t.size(0), (int)t.size(1), t.mutable_data_ptr()};
}

// gemm_packing(A, B, transpose, ws, device, stream, C, steps, bias, deq, deq_per_oc, q, q_per_oc) -> packed: a B that is used once, where the
// library would have it packed first
PyObject* gemm_packing(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 13 || !call_unpacked_need || !call_repack || !call_gemm) Py_RETURN_NONE;
    try {
        int device, rc = 0;
        if (!whole_number(a[4], 0, 1 << 20, device) || !PyBool_Check(a[2])) throw Leave();
        const int transpose = a[2] == Py_True;
        const Matrix A = matrix(a[0], device), B = matrix(a[1], device);
        const int M = A.rows, K = A.cols, N = transpose ? B.rows : B.cols;
        if (A.t->scalar_type() != at::kBFloat16 || B.t->scalar_type() != at::kBFloat16 || (transpose ? B.cols : B.rows) != K) throw Leave();
        if (call_unpacked_need(MMX_BF16, M, K, N, A.ld, B.ld, transpose) >= 0) throw Leave();
        const mmx_epilogue e = epilogue_of(a + 6, device, M, N);
        if (e.steps & MMX_PP_SILU_GATE) throw Leave();
        void* ws = nullptr;
        size_t ws_bytes = 0;
        if (a[3] != Py_None) {
            const at::Tensor& w = tensor_on(a[3], device);
            if (w.scalar_type() != at::kByte || !w.is_contiguous()) throw Leave();
            ws = w.mutable_data_ptr();
            ws_bytes = (size_t)w.numel();
        } else if (call_need(MMX_BF16, MMX_BF16, M, K, N, 0, N, e.steps, 0)) {
            throw Leave();  // (it is made outside)
        }
        void* const stream = stream_of(a[5]);
        at::Tensor out;
        if (!unlocked([&] {
                out = make({(int64_t)call_packed_bytes(MMX_BF16, K, N)}, at::kByte, *B.t);
                rc = call_repack(MMX_BF16, B.data, B.ld, K, N, transpose, out.mutable_data_ptr(), stream);
                if (!rc) rc = call_gemm(MMX_BF16, MMX_BF16, A.data, A.ld, out.mutable_data_ptr(), M, K, N, 0, N, &e, ws ? 0 : 1, ws, ws_bytes, stream);
            })) throw Leave();
        return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    } catch (...) {
        Py_RETURN_NONE;
    }
}

// repack(B, transpose, device, stream) -> packed
PyObject* repack(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 4 || !call_repack) Py_RETURN_NONE;
    try {
        int device, rc = 0;
        if (!whole_number(a[2], 0, 1 << 20, device) || !PyBool_Check(a[1])) throw Leave();
        const Matrix B = matrix(a[0], device);
        const int dt = code_of(B.t->scalar_type()), transpose = a[1] == Py_True, K = transpose ? B.cols : B.rows, N = transpose ? B.rows : B.cols;
        if (dt != MMX_BF16 && dt != MMX_I8 && dt != MMX_U8) throw Leave();
        void* const stream = stream_of(a[3]);
        at::Tensor out;
        if (!unlocked([&] {
                out = make({(int64_t)call_packed_bytes(dt, K, N)}, at::kByte, *B.t);
                rc = call_repack(dt, B.data, B.ld, K, N, transpose, out.mutable_data_ptr(), stream);
            })) throw Leave();
        return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    } catch (...) {
        Py_RETURN_NONE;
    }
}

// quantize(W, device, stream) -> (Wq, scales)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 3 || !call_quantize) Py_RETURN_NONE;
    try {
        int device, rc = 0;
        if (!whole_number(a[1], 0, 1 << 20, device)) throw Leave();
        const Matrix W = matrix(a[0], device);
        if (W.t->scalar_type() != at::kBFloat16) throw Leave();
        void* const stream = stream_of(a[2]);
        at::Tensor Wq, scales, scratch;
        if (!unlocked([&] {
                Wq = make({W.rows, W.cols}, at::kChar, *W.t);
                scales = make({2}, at::kFloat, *W.t);
                scratch = make({MMX_QUANTIZE_SCRATCH_BYTES / 4}, at::kInt, *W.t);
                rc = call_quantize(W.data, W.ld, W.rows, W.cols, Wq.mutable_data_ptr(), W.cols, static_cast<float*>(scales.mutable_data_ptr()),
                                   static_cast<uint32_t*>(scratch.mutable_data_ptr()), MMX_QUANTIZE_SCRATCH_BYTES, stream);
            })) throw Leave();
        return rc ? PyLong_FromLong(rc) : Py_BuildValue("(NN)", THPVariable_Wrap(Wq), THPVariable_Wrap(scales));
    } catch (...) {
        Py_RETURN_NONE;
    }
}

// quantize_scaled(W, scale, device, stream) -> Wq
PyObject* quantize_scaled(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 4 || !call_quantize_scaled) Py_RETURN_NONE;
    try {
        int device, rc = 0;
        if (!whole_number(a[2], 0, 1 << 20, device) || !PyFloat_CheckExact(a[1])) throw Leave();
        const Matrix W = matrix(a[0], device);
        if (W.t->scalar_type() != at::kBFloat16) throw Leave();
        const float scale = (float)PyFloat_AS_DOUBLE(a[1]);
        void* const stream = stream_of(a[3]);
        at::Tensor Wq;
        if (!unlocked([&] {
                Wq = make({W.rows, W.cols}, at::kChar, *W.t);
                rc = call_quantize_scaled(W.data, W.ld, W.rows, W.cols, scale, Wq.mutable_data_ptr(), W.cols, stream);
            })) throw Leave();
        return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(Wq);
    } catch (...) {
        Py_RETURN_NONE;
    }
}

// quantize_pack_scaled(W, scale, device, stream) -> packed
PyObject* quantize_pack_scaled(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 4 || !call_quantize_pack_scaled) Py_RETURN_NONE;
    try {
        int device, rc = 0;
        if (!whole_number(a[2], 0, 1 << 20, device) || !PyFloat_CheckExact(a[1])) throw Leave();
        const Matrix W = matrix(a[0], device);
        if (W.t->scalar_type() != at::kBFloat16) throw Leave();
        const float scale = (float)PyFloat_AS_DOUBLE(a[1]);
        void* const stream = stream_of(a[3]);
        at::Tensor out;
        if (!unlocked([&] {
                out = make({(int64_t)call_packed_bytes(MMX_I8, W.rows, W.cols)}, at::kByte, *W.t);
                rc = call_quantize_pack_scaled(W.data, W.ld, W.rows, W.cols, scale, out.mutable_data_ptr(), stream);
            })) throw Leave();
        return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    } catch (...) {
        Py_RETURN_NONE;
    }
}

// quantize_pack_int4(W, transpose, device, stream) -> (packed, deq)
PyObject* quantize_pack_int4(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 4 || !call_quantize_int4) Py_RETURN_NONE;
    try {
        int device, rc = 0;
        if (!whole_number(a[2], 0, 1 << 20, device) || !PyBool_Check(a[1])) throw Leave();
        const Matrix W = matrix(a[0], device);
        if (W.t->scalar_type() != at::kBFloat16) throw Leave();
        const int transpose = a[1] == Py_True, K = transpose ? W.cols : W.rows, N = transpose ? W.rows : W.cols;
        void* const stream = stream_of(a[3]);
        at::Tensor packed, deq;
        if (!unlocked([&] {
                packed = make({(int64_t)call_packed_bytes(MMX_I4, K, N)}, at::kByte, *W.t);
                deq = make({N}, at::kFloat, *W.t);
                rc = call_quantize_int4(W.data, W.ld, K, N, transpose, packed.mutable_data_ptr(), static_cast<float*>(deq.mutable_data_ptr()), stream);
            })) throw Leave();
        return rc ? PyLong_FromLong(rc) : Py_BuildValue("(NN)", THPVariable_Wrap(packed), THPVariable_Wrap(deq));
    } catch (...) {
        Py_RETURN_NONE;
    }
}

// ---- the feed-forward block in 8-bit floating point ----------------------------------------------------------------------
decltype(&mmx_quantize_rows_fp8) call_quantize_rows = nullptr;
decltype(&mmx_gemm_fp8_scratch_bytes) call_gemm_fp8_need = nullptr;
decltype(&mmx_gemm_fp8) call_gemm_fp8 = nullptr;
decltype(&mmx_mlp_fp8_scratch_bytes) call_mlp_fp8_need = nullptr;
decltype(&mmx_mlp_fp8) call_mlp_fp8 = nullptr;
decltype(&mmx_moe_route) call_moe_route = nullptr;
decltype(&mmx_moe_experts_scratch_bytes) call_moe_need = nullptr;
decltype(&mmx_moe_experts) call_moe_experts = nullptr;
decltype(&mmx_block_norm) call_block_norm = nullptr;
decltype(&mmx_mxfp4_bytes) call_mxfp4_bytes = nullptr;
decltype(&mmx_quantize_mxfp4) call_quantize_mxfp4 = nullptr;
decltype(&mmx_dequantize_mxfp4) call_dequantize_mxfp4 = nullptr;
decltype(&mmx_gemm_mxfp4_scratch_bytes) call_gemm_mxfp4_need = nullptr;
decltype(&mmx_gemm_mxfp4) call_gemm_mxfp4 = nullptr;
decltype(&mmx_mlp_mxfp4_scratch_bytes) call_mlp_mxfp4_need = nullptr;
decltype(&mmx_mlp_mxfp4) call_mlp_mxfp4 = nullptr;
decltype(&mmx_sample_scratch_bytes) call_sample_need = nullptr;
decltype(&mmx_sample) call_sample = nullptr;

int64_t blocks(int64_t n) { return (n + 127) / 128; }

int float_code(const at::Tensor& t) {  // bf16 or fp32
    const int c = code_of(t.scalar_type());
    if (c != MMX_BF16 && c != MMX_F32) throw Leave();
    return c;
}

const float* floats(PyObject* o, int device, at::IntArrayRef sizes) {
    const at::Tensor& t = tensor_on(o, device);
    if (t.scalar_type() != at::kFloat || !t.is_contiguous() || t.sizes() != sizes) throw Leave();
    return static_cast<const float*>(t.mutable_data_ptr());
}

const void* packed_bytes(PyObject* o, int device, int64_t need) {
    const at::Tensor& t = tensor_on(o, device);
    void* const p = t.mutable_data_ptr();
    if (t.scalar_type() != at::kByte || t.dim() != 1 || !t.is_contiguous() || t.numel() < need || (reinterpret_cast<uintptr_t>(p) & 15)) throw Leave();
    return p;
}
int64_t packed_e4m3(int64_t K, int64_t N) { return (N + 31) / 32 * 32 * blocks(K) * 128; }

// Activations: (bf16 or fp32 rows, None, K), or the padded rows, the scales and K of quantised ones
struct Activations {
    const at::Tensor* t;
    int dtype, M, K;
    const void* data;
    int64_t ld, ld_scales;
    const float* scales;
};
Activations activations(PyObject* const* a, int device) {
    const Matrix x = matrix(a[0], device);
    Activations r = {x.t, 0, x.rows, 0, x.data, x.ld, 0, nullptr};
    if (!whole_number(a[2], 1, 1 << 30, r.K)) throw Leave();
    if (a[1] == Py_None) {
        r.dtype = float_code(*x.t);
        if (x.cols != r.K) throw Leave();
        return r;
    }
    r.dtype = MMX_F8;
    const at::Tensor& s = tensor_on(a[1], device);
    if (x.t->scalar_type() != at::kFloat8_e4m3fn || x.cols != blocks(r.K) * 128 || s.scalar_type() != at::kFloat || s.dim() != 2 || s.size(0) != blocks(r.K) ||
        s.size(1) != r.M || (s.stride(1) != 1 && r.M != 1)) throw Leave();
    r.scales = static_cast<const float*>(s.mutable_data_ptr());
    r.ld_scales = s.size(0) <= 1 ? r.M : s.stride(0);
    return r;
}

// the caller's result [M, N] in bf16 or fp32, if there is one (else it is made in bf16)
at::Tensor result(PyObject* o, int device, int64_t M, int64_t N) {
    if (o == Py_None) return at::Tensor();
    const at::Tensor& y = tensor_on(o, device);
    if (y.dim() != 2 || y.size(0) != M || y.size(1) != N) throw Leave();
    float_code(y);
    return y;
}

// quantize_fp8(x, device, stream) -> (padded rows, scales)
PyObject* quantize_fp8(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 3 || !call_quantize_rows) Py_RETURN_NONE;
    try {
        int device, rc = 0;
        if (!whole_number(a[1], 0, 1 << 20, device)) throw Leave();
        const Matrix x = matrix(a[0], device);
        const int dt = float_code(*x.t);
        void* const stream = stream_of(a[2]);
        at::Tensor q, s;
        if (!unlocked([&] {
                const int64_t n = blocks(x.cols) * 128;
                q = make({x.rows, n % 2048 ? n : n + 128}, at::kFloat8_e4m3fn, *x.t).narrow(1, 0, n);
                s = make({blocks(x.cols), x.rows}, at::kFloat, *x.t);
                rc = call_quantize_rows(dt, x.data, x.ld, x.rows, x.cols, q.mutable_data_ptr(), q.stride(0), static_cast<float*>(s.mutable_data_ptr()), x.rows, stream);
            })) throw Leave();
        return rc ? PyLong_FromLong(rc) : Py_BuildValue("(NN)", THPVariable_Wrap(q), THPVariable_Wrap(s));
    } catch (...) {
        Py_RETURN_NONE;
    }
}

// gemm_fp8(x, x_scales, K, packed, scales, N, device, stream, C, steps, bias, deq, deq_per_oc, q, q_per_oc)
PyObject* gemm_fp8(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 15 || !call_gemm_fp8) Py_RETURN_NONE;
    int rc = 0;
    try {
        int N, device;
        if (!whole_number(a[6], 0, 1 << 20, device) || !whole_number(a[5], 1, 1 << 30, N)) throw Leave();
        const Activations x = activations(a, device);
        const mmx_epilogue e = epilogue_of(a + 8, device, x.M, N);
        const bool pair = e.steps & MMX_PP_SILU_GATE;
        const at::Tensor& C = tensor_on(a[8], device);
        if (C.size(0) != x.M || C.size(1) != (pair ? N / 2 : N) || (a[10] != Py_None && tensor_on(a[10], device).numel() != N)) throw Leave();
        const void* const w = packed_bytes(a[3], device, packed_e4m3(x.K, N));
        const float* const s = floats(a[4], device, {pair ? 2 * blocks(N / 2) : blocks(N), blocks(x.K)});
        void* const stream = stream_of(a[7]);
        if (!unlocked([&] {
                const size_t need = call_gemm_fp8_need(x.dtype, x.M, x.K, N);
                at::Tensor scratch;
                if (need) scratch = make({(int64_t)need}, at::kByte, *x.t);
                rc = call_gemm_fp8(x.dtype, x.data, x.ld, x.scales, x.ld_scales, w, s, x.M, x.K, N, &e, need ? scratch.mutable_data_ptr() : nullptr, need, stream);
            })) throw Leave();
    } catch (...) {
        Py_RETURN_NONE;
    }
    return PyLong_FromLong(rc);
}

// mlp_fp8(x, x_scales, K, gate_up, gate_up_scales, down, down_scales, N, y, device, stream) -> y
PyObject* mlp_fp8(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 11 || !call_mlp_fp8) Py_RETURN_NONE;
    try {
        int N, device, rc = 0;
        if (!whole_number(a[9], 0, 1 << 20, device) || !whole_number(a[7], 1, 1 << 29, N) || N % 32) throw Leave();
        const Activations x = activations(a, device);
        const void* const gu = packed_bytes(a[3], device, packed_e4m3(x.K, 2 * (int64_t)N));
        const float* const gus = floats(a[4], device, {2 * blocks(N), blocks(x.K)});
        const void* const d = packed_bytes(a[5], device, packed_e4m3(N, x.K));
        const float* const ds = floats(a[6], device, {blocks(x.K), blocks(N)});
        void* const stream = stream_of(a[10]);
        at::Tensor y = result(a[8], device, x.M, x.K);
        if (!unlocked([&] {
                if (!y.defined()) y = make({x.M, x.K}, at::kBFloat16, *x.t);
                const size_t need = call_mlp_fp8_need(x.dtype, x.M, x.K, N);
                const at::Tensor scratch = make({(int64_t)need}, at::kByte, *x.t);
                rc = call_mlp_fp8(x.dtype, x.data, x.ld, x.scales, x.ld_scales, gu, gus, d, ds, code_of(y.scalar_type()), y.mutable_data_ptr(), row_stride_bytes(y), x.M, x.K, N,
                                  scratch.mutable_data_ptr(), need, stream);
            })) throw Leave();
        return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(y);
    } catch (...) {
        Py_RETURN_NONE;
    }
}

// moe(x, router, bias, top_k, flags, scale, gate_up, gate_up_scales, down, down_scales, I, y, device, stream) -> y: routing and experts
PyObject* moe(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 14 || !call_moe_route || !call_moe_experts) Py_RETURN_NONE;
    try {
        int k, flags, I, device, rc = 0;
        if (!whole_number(a[12], 0, 1 << 20, device) || !whole_number(a[3], 1, 16, k) || !whole_number(a[4], 0, 3, flags) || !PyFloat_CheckExact(a[5]) ||
            !whole_number(a[10], 32, 1 << 29, I) || I % 32) throw Leave();
        const Matrix x = matrix(a[0], device), router = matrix(a[1], device);
        const int T = x.rows, H = x.cols, E = router.rows;
        if (x.t->scalar_type() != at::kBFloat16 || router.t->scalar_type() != at::kBFloat16 || router.cols != H || E > 1024 || k > E) throw Leave();
        const float scale = (float)PyFloat_AS_DOUBLE(a[5]);
        const float* const bias = a[2] == Py_None ? nullptr : floats(a[2], device, {E});
        const bool f8 = a[7] != Py_None;
        const auto bytes = [&](int64_t K, int64_t N) { return f8 ? packed_e4m3(K, N) : (N + 31) / 32 * 32 * ((K * 2 + 127) / 128 * 128); };
        const void* const gu = packed_bytes(a[6], device, E * bytes(H, 2 * (int64_t)I));
        const void* const d = packed_bytes(a[8], device, E * bytes(I, H));
        const float* const gus = f8 ? floats(a[7], device, {E, 2 * blocks(I), blocks(H)}) : nullptr;
        const float* const ds = f8 ? floats(a[9], device, {E, blocks(H), blocks(I)}) : nullptr;
        if (!f8 && a[9] != Py_None) throw Leave();
        void* const stream = stream_of(a[13]);
        at::Tensor y = result(a[11], device, T, H);
        if (!unlocked([&] {
                if (!y.defined()) y = make({T, H}, at::kBFloat16, *x.t);
                const auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
                const size_t logits = up((size_t)T * E * 8), ids = up((size_t)T * k * 4), need = call_moe_need(T, H, I, k);
                const at::Tensor memory = make({(int64_t)(logits + 2 * ids + need)}, at::kByte, *x.t);
                char* const at = static_cast<char*>(memory.mutable_data_ptr());
                int32_t* const chosen = reinterpret_cast<int32_t*>(at + logits);
                float* const weights = reinterpret_cast<float*>(at + logits + ids);
                rc = call_moe_route(x.data, x.ld, router.data, router.ld, T, H, E, k, flags, scale, bias, reinterpret_cast<double*>(at), chosen, weights, stream);
                if (!rc)
                    rc = call_moe_experts(f8 ? MMX_F8 : MMX_BF16, x.data, x.ld, chosen, weights, T, H, I, E, k, gu, gus, d, ds, code_of(y.scalar_type()), y.mutable_data_ptr(),
                                          row_stride_bytes(y), at + logits + 2 * ids, need, stream);
            })) throw Leave();
        return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(y);
    } catch (...) {
        Py_RETURN_NONE;
    }
}

// ---- microscaled 4-bit floating point: rows of bf16 or fp32 with (None, None), or packed rows with their (M, K)
struct Rows4 {
    const at::Tensor* t;
    int dtype, M, K;
    const void* data;
    int64_t ld;
};
Rows4 rows4(PyObject* const* a, int device) {
    if (a[1] == Py_None) {
        const Matrix x = matrix(a[0], device);
        return {x.t, float_code(*x.t), x.rows, x.cols, x.data, x.ld};
    }
    Rows4 r = {&tensor_on(a[0], device), MMX_F4, 0, 0, nullptr, 0};
    if (!whole_number(a[1], 1, 1 << 30, r.M) || !whole_number(a[2], 1, 1 << 22, r.K)) throw Leave();
    r.data = packed_bytes(a[0], device, (int64_t)call_mxfp4_bytes(r.M, r.K));
    return r;
}

// quantize_mxfp4(x, device, stream) -> packed rows
PyObject* quantize_mxfp4(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 3 || !call_quantize_mxfp4) Py_RETURN_NONE;
    try {
        int device, rc = 0;
        if (!whole_number(a[1], 0, 1 << 20, device)) throw Leave();
        const Matrix x = matrix(a[0], device);
        const int dt = float_code(*x.t);
        void* const stream = stream_of(a[2]);
        at::Tensor packed;
        if (!unlocked([&] {
                packed = make({(int64_t)call_mxfp4_bytes(x.rows, x.cols)}, at::kByte, *x.t);
                rc = call_quantize_mxfp4(dt, x.data, x.ld, x.rows, x.cols, 0, packed.mutable_data_ptr(), stream);
            })) throw Leave();
        return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(packed);
    } catch (...) {
        Py_RETURN_NONE;
    }
}

// dequantize_mxfp4(packed rows, M, K, whether fp32, device, stream) -> their values
PyObject* dequantize_mxfp4(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 6 || !call_dequantize_mxfp4) Py_RETURN_NONE;
    try {
        int device, rc = 0;
        if (!whole_number(a[4], 0, 1 << 20, device) || a[1] == Py_None || !PyBool_Check(a[3])) throw Leave();
        const Rows4 x = rows4(a, device);
        const bool wide = a[3] == Py_True;
        void* const stream = stream_of(a[5]);
        at::Tensor y;
        if (!unlocked([&] {
                y = make({x.M, x.K}, wide ? at::kFloat : at::kBFloat16, *x.t);
                rc = call_dequantize_mxfp4(x.data, x.M, x.K, wide ? MMX_F32 : MMX_BF16, y.mutable_data_ptr(), (int64_t)x.K * (wide ? 4 : 2), stream);
            })) throw Leave();
        return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(y);
    } catch (...) {
        Py_RETURN_NONE;
    }
}

// gemm_mxfp4(x, M, K, packed, N, device, stream, C, steps, bias, deq, deq_per_oc, q, q_per_oc)
PyObject* gemm_mxfp4(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 14 || !call_gemm_mxfp4) Py_RETURN_NONE;
    int rc = 0;
    try {
        int N, device;
        if (!whole_number(a[5], 0, 1 << 20, device) || !whole_number(a[4], 1, 1 << 30, N)) throw Leave();
        const Rows4 x = rows4(a, device);
        const mmx_epilogue e = epilogue_of(a + 7, device, x.M, N);
        const at::Tensor& C = tensor_on(a[7], device);
        if (C.size(0) != x.M || C.size(1) != (e.steps & MMX_PP_SILU_GATE ? N / 2 : N) || (a[9] != Py_None && tensor_on(a[9], device).numel() != N)) throw Leave();
        const void* const w = packed_bytes(a[3], device, (int64_t)call_mxfp4_bytes(N, x.K));
        void* const stream = stream_of(a[6]);
        if (!unlocked([&] {
                const size_t need = call_gemm_mxfp4_need(x.dtype, x.M, x.K, N);
                at::Tensor scratch;
                if (need) scratch = make({(int64_t)need}, at::kByte, *x.t);
                rc = call_gemm_mxfp4(x.dtype, x.data, x.ld, w, x.M, x.K, N, &e, need ? scratch.mutable_data_ptr() : nullptr, need, stream);
            })) throw Leave();
    } catch (...) {
        Py_RETURN_NONE;
    }
    return PyLong_FromLong(rc);
}

// mlp_mxfp4(x, M, K, gate_up, down, N, y, device, stream) -> y
PyObject* mlp_mxfp4(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 9 || !call_mlp_mxfp4) Py_RETURN_NONE;
    try {
        int N, device, rc = 0;
        if (!whole_number(a[7], 0, 1 << 20, device) || !whole_number(a[5], 1, 1 << 29, N) || N % 32) throw Leave();
        const Rows4 x = rows4(a, device);
        const void* const gu = packed_bytes(a[3], device, (int64_t)call_mxfp4_bytes(2 * (int64_t)N, x.K));
        const void* const d = packed_bytes(a[4], device, (int64_t)call_mxfp4_bytes(x.K, N));
        void* const stream = stream_of(a[8]);
        at::Tensor y = result(a[6], device, x.M, x.K);
        if (!unlocked([&] {
                if (!y.defined()) y = make({x.M, x.K}, at::kBFloat16, *x.t);
                const size_t need = call_mlp_mxfp4_need(x.dtype, x.M, x.K, N);
                const at::Tensor scratch = make({(int64_t)need}, at::kByte, *x.t);
                rc = call_mlp_mxfp4(x.dtype, x.data, x.ld, gu, d, code_of(y.scalar_type()), y.mutable_data_ptr(), row_stride_bytes(y), x.M, x.K, N, scratch.mutable_data_ptr(), need,
                                    stream);
            })) throw Leave();
        return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(y);
    } catch (...) {
        Py_RETURN_NONE;
    }
}

// block_norm(f, residual, post, post_weight, gate, scale, pre, pre_weight, eps, offset, quantize, r, device, stream) -> (r, z), (r, padded rows of z, scales) or (r, packed z)
//   quantize: False, True (e4m3) or 2 (packed e2m1); r: where to put it, None: made here, False: not wanted
PyObject* block_norm(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 14 || !call_block_norm) Py_RETURN_NONE;
    try {
        int device, rc = 0;
        if (!whole_number(a[12], 0, 1 << 20, device) || !PyBool_Check(a[2]) || !PyBool_Check(a[6]) || !PyFloat_CheckExact(a[5]) ||
            !PyFloat_CheckExact(a[8]) || !PyFloat_CheckExact(a[9])) throw Leave();
        const Matrix f = matrix(a[0], device);
        const int64_t M = f.rows, H = f.cols;
        if (f.t->scalar_type() != at::kBFloat16) throw Leave();
        mmx_block_norm_args n = {};
        n.f = f.data;
        n.ldf_bytes = f.ld;
        n.residual_dtype = MMX_BF16;
        const auto same = [&](PyObject* o) {
            const Matrix m = matrix(o, device);
            if (m.rows != M || m.cols != H) throw Leave();
            return m;
        };
        if (a[1] != Py_None) {
            const Matrix m = same(a[1]);
            n.residual_dtype = float_code(*m.t);
            n.residual = m.data;
            n.ld_residual_bytes = m.ld;
        }
        const auto vector = [&](PyObject* o) -> const void* {
            if (o == Py_None) return nullptr;
            const at::Tensor& t = tensor_on(o, device);
            if (t.scalar_type() != at::kBFloat16 || t.dim() != 1 || t.numel() != H || !t.is_contiguous()) throw Leave();
            return t.mutable_data_ptr();
        };
        n.post = a[2] == Py_True;
        n.post_weight = vector(a[3]);
        n.pre = a[6] == Py_True;
        n.pre_weight = vector(a[7]);
        if ((n.post_weight && !n.post) || (n.pre_weight && !n.pre)) throw Leave();
        if (a[4] != Py_None && tensor_on(a[4], device).dim() == 2) {
            const Matrix m = same(a[4]);
            if (m.t->scalar_type() != at::kBFloat16) throw Leave();
            n.gate = m.data;
            n.ld_gate_bytes = M == 1 ? 0 : m.ld;
        } else {
            n.gate = vector(a[4]);
        }
        n.scale = (float)PyFloat_AS_DOUBLE(a[5]);
        n.eps = (float)PyFloat_AS_DOUBLE(a[8]);
        n.weight_offset = (float)PyFloat_AS_DOUBLE(a[9]);
        int two = 0;
        if (!PyBool_Check(a[10]) && !whole_number(a[10], 2, 2, two)) throw Leave();
        const bool quantize = a[10] == Py_True, packed = two == 2;
        const at::ScalarType stream_type = n.residual_dtype == MMX_F32 ? at::kFloat : at::kBFloat16;
        const bool keep = a[11] != Py_False;
        if (keep && a[11] != Py_None && same(a[11]).t->scalar_type() != stream_type) throw Leave();
        void* const stream = stream_of(a[13]);
        at::Tensor r, z, s;
        if (keep && a[11] != Py_None) r = THPVariable_Unpack(a[11]);
        if (!unlocked([&] {
                if (keep) {
                    if (!r.defined()) r = make({M, H}, stream_type, *f.t);
                    n.r = r.mutable_data_ptr();
                    n.ldr_bytes = row_stride_bytes(r);
                }
                if (packed) {
                    z = make({(int64_t)call_mxfp4_bytes(M, (int)H)}, at::kByte, *f.t);
                    n.z_dtype = MMX_F4;
                } else if (quantize) {
                    const int64_t p = blocks(H) * 128;
                    z = make({M, p % 2048 ? p : p + 128}, at::kFloat8_e4m3fn, *f.t).narrow(1, 0, p);
                    s = make({blocks(H), M}, at::kFloat, *f.t);
                    n.z_scales = static_cast<float*>(s.mutable_data_ptr());
                    n.ld_z_scales = M;
                    n.z_dtype = MMX_F8;
                    n.ldz_bytes = z.stride(0);
                } else {
                    z = make({M, H}, at::kBFloat16, *f.t);
                    n.z_dtype = MMX_BF16;
                    n.ldz_bytes = 2 * H;
                }
                n.z = z.mutable_data_ptr();
                rc = call_block_norm(&n, (int)M, (int)H, stream);
            })) throw Leave();
        if (rc) return PyLong_FromLong(rc);
        PyObject* const kept = keep ? THPVariable_Wrap(r) : (Py_INCREF(Py_None), Py_None);
        return quantize ? Py_BuildValue("(NNN)", kept, THPVariable_Wrap(z), THPVariable_Wrap(s)) : Py_BuildValue("(NN)", kept, THPVariable_Wrap(z));
    } catch (...) {
        Py_RETURN_NONE;
    }
}

// sample(logits, u, temperature, top_k, top_p, min_p, device, stream) -> ids; each of the four a number or a tensor with one for each row
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 8 || !call_sample) Py_RETURN_NONE;
    try {
        int device, rc = 0;
        if (!whole_number(a[6], 0, 1 << 20, device)) throw Leave();
        const Matrix l = matrix(a[0], device);
        mmx_sample_args s = {};
        s.logits = l.data;
        s.ld_bytes = l.ld;
        s.dtype = float_code(*l.t);
        s.u = floats(a[1], device, {l.rows});
        const auto asked = [&](PyObject* o, const float*& of, double& all) {
            if (PyFloat_CheckExact(o)) {
                all = PyFloat_AS_DOUBLE(o);
            } else if (PyLong_CheckExact(o)) {  // (0 and 1 are written so; not a truth value, which is a number of its own type)
                int n;
                if (!whole_number(o, 0, INT32_MAX, n)) throw Leave();
                all = n;
            } else {
                of = floats(o, device, {l.rows});
            }
        };
        asked(a[2], s.temperature_of, s.temperature);
        asked(a[4], s.top_p_of, s.top_p);
        asked(a[5], s.min_p_of, s.min_p);
        if (!whole_number(a[3], 0, INT32_MAX, s.top_k)) {
            const at::Tensor& k = tensor_on(a[3], device);
            if (k.scalar_type() != at::kInt || k.dim() != 1 || k.size(0) != l.rows || !k.is_contiguous()) throw Leave();
            s.top_k_of = static_cast<const int32_t*>(k.mutable_data_ptr());
        }
        void* const stream = stream_of(a[7]);
        at::Tensor ids;
        if (!unlocked([&] {
                ids = make({l.rows}, at::kInt, *l.t);
                s.ids = static_cast<int32_t*>(ids.mutable_data_ptr());
                const size_t need = call_sample_need(l.rows, l.cols);
                at::Tensor scratch;
                if (need) scratch = make({(int64_t)need}, at::kByte, *l.t);
                rc = call_sample(&s, l.rows, l.cols, need ? scratch.mutable_data_ptr() : nullptr, need, stream);
            })) throw Leave();
        return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(ids);
    } catch (...) {
        Py_RETURN_NONE;
    }
}

// bind(addresses of the entry points, in the order below)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t count) {
    constexpr int ENTRIES = 29;
    if (count != ENTRIES) {
        PyErr_SetString(PyExc_TypeError, "bind takes an address for each entry point");
        return nullptr;
    }
    void* at[ENTRIES];
    for (int i = 0; i < ENTRIES; i++) at[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
    int i = 0;
    auto set = [&](auto& f) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(at[i++]); };
    set(call_gemm);
    set(call_need);
    set(call_unpacked);
    set(call_unpacked_need);
    set(call_matvec);
    set(call_packed_bytes);
    set(call_repack);
    set(call_quantize);
    set(call_quantize_scaled);
    set(call_quantize_int4);
    set(call_quantize_pack_scaled);
    set(call_quantize_rows);
    set(call_gemm_fp8_need);
    set(call_gemm_fp8);
    set(call_mlp_fp8_need);
    set(call_mlp_fp8);
    set(call_moe_route);
    set(call_moe_need);
    set(call_moe_experts);
    set(call_block_norm);
    set(call_mxfp4_bytes);
    set(call_quantize_mxfp4);
    set(call_dequantize_mxfp4);
    set(call_gemm_mxfp4_need);
    set(call_gemm_mxfp4);
    set(call_mlp_mxfp4_need);
    set(call_mlp_mxfp4);
    set(call_sample_need);
    set(call_sample);
    Py_RETURN_NONE;
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(gemm), METHOD(gemm_unpacked), METHOD(gemm_packing), METHOD(matvec), METHOD(repack), METHOD(quantize), METHOD(quantize_scaled),
                         METHOD(quantize_pack_int4), METHOD(quantize_pack_scaled), METHOD(quantize_fp8),
                         METHOD(gemm_fp8), METHOD(mlp_fp8), METHOD(moe), METHOD(block_norm),
                         METHOD(quantize_mxfp4), METHOD(dequantize_mxfp4), METHOD(gemm_mxfp4), METHOD(mlp_mxfp4), METHOD(sample), METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version: of the torch that this was compiled against, whose classes may be laid out differently in another
PyMODINIT_FUNC PyInit__host_call(void) {
    PyObject* const m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", MMX_TORCH_VERSION) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
