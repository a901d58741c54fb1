// torch_kv8.cpp -- the torch side of the 8-bit key/value cache (Python module _b200torch): checks of
// the tensors, outputs and workspaces from torch's allocator, and the calls of the C ABI on torch's
// current stream.
//
// These calls are made once a layer and token, with thirty arguments each; in Python with ctypes
// their host time (17 us an attention, 10 us an append) was several times what the GPU takes for a
// short batch.  b200lab.py documents the arguments.
#include <Python.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/b200lab.h"

namespace {

using at::Tensor;

const Tensor& tensor(PyObject* o, const char* name) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
    return THPVariable_Unpack(o);
}

int integer(PyObject* o, const char* name) {
    const Py_ssize_t v = PyNumber_AsSsize_t(o, nullptr);  // clipped where it does not fit
    if (v == -1 && PyErr_Occurred()) throw python_error();
    TORCH_CHECK_VALUE(v >= -0x7fffffffLL && v <= 0x7fffffffLL, name, " does not fit 32 bits");
    return (int)v;
}

int size32(int64_t v, const char* name) {
    TORCH_CHECK_VALUE(v <= 0x7fffffffLL, name, " does not fit 32 bits");
    return (int)v;
}

int dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kHalf: return B200LAB_F16;
        case at::kBFloat16: return B200LAB_BF16;
        case at::kFloat: return B200LAB_F32;
        default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t.scalar_type());
    }
}

// The cache's five tensors, checked against one another.
struct Cache {
    const Tensor &k, &v, &ks, &vs, &table;
    c10::Device device;
    int n_blocks, Hkv, block_size, D, B, max_blocks;

    explicit Cache(PyObject* const* o)
        : k(tensor(o[0], "k_cache")), v(tensor(o[1], "v_cache")), ks(tensor(o[2], "k_scale")),
          vs(tensor(o[3], "v_scale")), table(tensor(o[4], "block_table")), device(k.device()) {
        TORCH_CHECK_VALUE(device.is_cuda(), "k_cache must be a CUDA tensor (no CPU path)");
        TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes(),
                          "k_cache and v_cache must be [n_blocks, Hkv, block_size, D], alike");
        TORCH_CHECK_TYPE(k.scalar_type() == at::kFloat8_e4m3fn && v.scalar_type() == at::kFloat8_e4m3fn,
                         "k_cache and v_cache must be float8_e4m3fn");
        for (const Tensor* s : {&ks, &vs}) {
            TORCH_CHECK_VALUE(s->dim() == 2 && s->size(0) == k.size(0) && s->size(1) == k.size(1),
                              "k_scale and v_scale must be [n_blocks, Hkv]");
            TORCH_CHECK_TYPE(s->scalar_type() == at::kFloat, "k_scale and v_scale must be float32");
        }
        TORCH_CHECK_VALUE(table.dim() == 2 && table.scalar_type() == at::kInt, "block_table must be int32 [B, max_blocks]");
        for (const Tensor* t : {&k, &v, &ks, &vs, &table})
            TORCH_CHECK_VALUE(t->is_contiguous() && t->device() == device,
                              "the cache, its scales and the block table must be contiguous, on one device");
        n_blocks = size32(k.size(0), "n_blocks"), Hkv = size32(k.size(1), "Hkv");
        block_size = size32(k.size(2), "block_size"), D = size32(k.size(3), "D");
        B = size32(table.size(0), "B"), max_blocks = size32(table.size(1), "max_blocks");
    }

    // int32 [n] on the cache's device; None gives null
    const int* ints(PyObject* o, int64_t n, const char* name, bool optional) const {
        if (optional && o == Py_None) return nullptr;
        const Tensor& t = tensor(o, name);
        TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 1 && t.numel() == n && t.is_contiguous() &&
                              t.device() == device,
                          name, " must be contiguous int32 [", n, "] on the cache's device");
        return static_cast<const int*>(t.data_ptr());
    }
    // token-major [total, H, D] with contiguous channels
    const void* rows(const Tensor& t, int64_t total, int64_t H, const char* name) const {
        TORCH_CHECK_VALUE(t.dim() == 3 && t.size(0) == total && t.size(1) == H && t.size(2) == D, name, " must be [", total,
                          ", ", H, ", ", D, "]");
        TORCH_CHECK_VALUE(t.device() == device, name, " must be on the cache's device");
        TORCH_CHECK_VALUE(t.stride(2) == 1, name, " must have contiguous channels");
        return t.data_ptr();
    }
};

// The stride of a dimension; 0 where it has one entry and is never stepped over, when torch lets it be any number.
int64_t stride(const Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }

Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, c10::Device device) {
    return at::empty(sizes, at::TensorOptions().dtype(dtype).device(device));
}

void* current_stream(c10::Device device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

PyObject* status(int st) { return PyLong_FromLong(st); }

// append(k, v, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_seqlens, max_seqlen) -> status
PyObject* append(PyObject*, PyObject* const* o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 10, "append takes 10 arguments");
    const Tensor &k = tensor(o[0], "k"), &v = tensor(o[1], "v");
    const Cache c(o + 2);
    TORCH_CHECK_VALUE(k.dim() == 3, "k must be [total, Hkv, D]");
    const int total = size32(k.size(0), "tokens");
    TORCH_CHECK_TYPE(v.scalar_type() == k.scalar_type(), "k and v must share a dtype");
    const void *kp = c.rows(k, total, c.Hkv, "k"), *vp = c.rows(v, total, c.Hkv, "v");
    const int* lens = c.ints(o[7], c.B, "seq_lens", false);
    const int* cu = c.ints(o[8], (int64_t)c.B + 1, "cu_seqlens", true);
    const int code = dtype_code(k), most = integer(o[9], "max_seqlen");
    if (total == 0 && (cu || c.B == 0)) return status(B200LAB_OK);
    const c10::cuda::CUDAGuard guard(c.device);
    return status(kv8_append_sm100(kp, stride(k, 0), stride(k, 1), vp, stride(v, 0), stride(v, 1), c.k.data_ptr(),
                                   c.v.data_ptr(), static_cast<float*>(c.ks.data_ptr()),
                                   static_cast<float*>(c.vs.data_ptr()), static_cast<const int*>(c.table.data_ptr()), lens,
                                   cu, most, total, c.B, c.max_blocks, c.n_blocks, c.block_size, c.Hkv, c.D, code,
                                   current_stream(c.device)));
    END_HANDLE_TH_ERRORS
}

// read(k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens, max_seqlen, total, out_dtype, k_out, v_out)
// -> (k, v), or a status that is not OK
PyObject* read(PyObject*, PyObject* const* o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 11, "read takes 11 arguments");
    const Cache c(o);
    const int* cu = c.ints(o[5], (int64_t)c.B + 1, "cu_seqlens", false);
    const int most = integer(o[6], "max_seqlen"), total = integer(o[7], "total_tokens");
    TORCH_CHECK_VALUE(total >= 0, "total_tokens must not be negative");
    at::ScalarType dtype = at::kBFloat16;
    if (o[8] != Py_None) {
        TORCH_CHECK_TYPE(THPDtype_Check(o[8]), "out_dtype must be a dtype");
        dtype = reinterpret_cast<THPDtype*>(o[8])->scalar_type;
    }
    const c10::cuda::CUDAGuard guard(c.device);
    Tensor k, v;
    if (o[9] == Py_None && o[10] == Py_None) {
        k = empty({total, c.Hkv, c.D}, dtype, c.device);
        v = empty({total, c.Hkv, c.D}, dtype, c.device);
    } else {
        TORCH_CHECK_VALUE(o[9] != Py_None && o[10] != Py_None, "k_out and v_out go together");
        k = tensor(o[9], "k_out"), v = tensor(o[10], "v_out");
        if (o[8] == Py_None) dtype = k.scalar_type();
        for (const Tensor* t : {&k, &v})
            TORCH_CHECK_VALUE(t->dim() == 3 && t->size(0) == total && t->size(1) == c.Hkv && t->size(2) == c.D &&
                                  t->device() == c.device && t->is_contiguous() && t->scalar_type() == dtype,
                              "k_out and v_out must be contiguous [total_tokens, Hkv, D] of out_dtype on the cache's device");
    }
    const int code = dtype_code(k);
    if (total > 0) {
        const int st = kv8_read_sm100(c.k.data_ptr(), c.v.data_ptr(), static_cast<const float*>(c.ks.data_ptr()),
                                      static_cast<const float*>(c.vs.data_ptr()),
                                      static_cast<const int*>(c.table.data_ptr()), cu, most, total, k.data_ptr(),
                                      v.data_ptr(), c.B, c.max_blocks, c.n_blocks, c.block_size, c.Hkv, c.D, code,
                                      current_stream(c.device));
        if (st != B200LAB_OK) return status(st);
    }
    PyObject* pair = PyTuple_New(2);
    if (!pair) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(k));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(v));
    return pair;
    END_HANDLE_TH_ERRORS
}

// attend(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_seqlens_q, max_seqlen_q, gate, scale,
//        causal, out, workspace) -> out, or a status that is not OK
PyObject* attend(PyObject*, PyObject* const* o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 14, "attend takes 14 arguments");
    const Tensor& q = tensor(o[0], "q");
    const Cache c(o + 1);
    TORCH_CHECK_VALUE(q.dim() == 3, "q must be [total_q, Hq, D]");
    const int total = size32(q.size(0), "tokens"), Hq = size32(q.size(1), "Hq");
    const void* qp = c.rows(q, total, Hq, "q");
    const int* lens = c.ints(o[6], c.B, "seq_lens", false);
    const int* cu = c.ints(o[7], (int64_t)c.B + 1, "cu_seqlens_q", true);
    const int most = integer(o[8], "max_seqlen_q"), code = dtype_code(q);
    const void* gp = nullptr;
    int64_t gt = 0, gh = 0;
    if (o[9] != Py_None) {
        const Tensor& g = tensor(o[9], "gate");
        TORCH_CHECK_TYPE(g.scalar_type() == q.scalar_type(), "gate must have q's dtype");
        gp = c.rows(g, total, Hq, "gate");
        gt = stride(g, 0), gh = stride(g, 1);
    }
    double scale = 1.0 / std::sqrt((double)c.D);
    if (o[10] != Py_None) {
        scale = PyFloat_AsDouble(o[10]);
        if (scale == -1.0 && PyErr_Occurred()) throw python_error();
    }
    const int causal = PyObject_IsTrue(o[11]);
    if (causal < 0) throw python_error();
    const c10::cuda::CUDAGuard guard(c.device);
    Tensor out, ws;
    if (o[12] == Py_None) {
        out = empty({total, Hq, c.D}, q.scalar_type(), c.device);
    } else {
        out = tensor(o[12], "out");
        TORCH_CHECK_VALUE(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.is_contiguous() &&
                              out.device() == c.device,
                          "out must be contiguous, like q, on the cache's device");
    }
    if (total == 0 && (cu || c.B == 0)) return THPVariable_Wrap(out);
    if (o[13] == Py_None) {
        // at least a byte, so that wrong sizes reach the library's own checks
        const size_t need = attn_fwd_sm100_kv8_workspace(Hq, c.Hkv, most, c.D);
        ws = empty({(int64_t)(need ? need : 1)}, at::kByte, c.device);
    } else {
        ws = tensor(o[13], "workspace");
        TORCH_CHECK_VALUE(ws.is_contiguous() && ws.device() == c.device,
                          "workspace must be contiguous, on the cache's device");
    }
    const int st = attn_fwd_sm100_kv8(
        qp, stride(q, 0), stride(q, 1), gp, gt, gh, c.k.data_ptr(), c.v.data_ptr(),
        static_cast<const float*>(c.ks.data_ptr()), static_cast<const float*>(c.vs.data_ptr()),
        static_cast<const int*>(c.table.data_ptr()), lens, cu, most, total, out.data_ptr(), c.B, c.max_blocks, c.n_blocks,
        c.block_size, Hq, c.Hkv, c.D, (float)scale, causal, code, ws.data_ptr(), (size_t)ws.numel() * ws.element_size(),
        current_stream(c.device));
    return st == B200LAB_OK ? THPVariable_Wrap(out) : status(st);
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
    {"read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(read)), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_b200torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__b200torch() { return PyModule_Create(&module); }
