// Native front of the Python entry points: argument checks, output allocation and the call into the
// C ABI in one CPython call.
//
// A small GEMM runs for 3 to 8 us on the device; the Python wrapper in front of it took the host 8 us
// (quantizer) and 10 us (GEMM), most of it attribute reads of tensors and the conversion of some twenty
// ctypes arguments, so a chain of eager calls ran at the host's pace (128 x 256 x 512 with its
// quantizer: 26 us of host time, 7.4 us of kernels).  Here the same checks read the tensors' fields.
//
// A function below handles the ordinary call: plain CUDA tensors, flags that are real bools, every check
// passed and the C ABI's return code 0.  For anything else it returns None without having
// done anything, and the Python wrapper goes through its own checks, which own all error texts (a call
// that the C ABI refused launches nothing, so it can be made again for its message).

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "../../include/halops_b200.h"

namespace {

constexpr int kErrLen = 512;

// The signatures are the header's, so a changed one does not compile here until its call is changed too.
using QuantFn = decltype(&hq_group_wise_quant);
using RmsFn = decltype(&hq_rms_norm_quant);
using DenseFn = decltype(&hq_dense_gemm);
using SituFn = decltype(&hq_dense_gemm_situ_quant);
using DescribeGroupFn = decltype(&hq_describe_group_tile);
using MaskedFn = decltype(&hq_group_masked_gemm);
using ContiguousFn = decltype(&hq_group_contiguous_gemm);

// the entry points of the shared library that the Python package has loaded
struct {
    QuantFn quant;
    RmsFn rms;
    DenseFn dense;
    SituFn situ;
    DescribeGroupFn describe_group;
    MaskedFn masked;
    ContiguousFn contiguous;
    decltype(&hq_hold_switches) hold_switches;
    decltype(&hq_block_quant) block_quant;
    decltype(&hq_swiglu_block_quant) swiglu;
    decltype(&hq_block_gemm) block_gemm;
    decltype(&hq_group_block_gemm) group_block_gemm;
    decltype(&hq_moe_sort) moe_sort;
    decltype(&hq_moe_permute) moe_permute;
    decltype(&hq_moe_permute_block_quant) moe_permute_quant;
    decltype(&hq_moe_unpermute) moe_unpermute;
    decltype(&hq_moe_unpermute_backward) moe_unpermute_backward;
} g_fn;

// the package's mode names
int mode_id(PyObject* o) {
    if (!PyUnicode_CheckExact(o)) return -1;
    const char* s = PyUnicode_AsUTF8(o);
    if (s == nullptr) {
        PyErr_Clear();
        return -1;
    }
    if (std::strcmp(s, "w8a8-mxfp8") == 0) return HQ_MODE_W8A8_MXFP8;
    if (std::strcmp(s, "w4a4-mxfp4") == 0) return HQ_MODE_W4A4_MXFP4;
    if (std::strcmp(s, "w4a4-nvfp4") == 0) return HQ_MODE_W4A4_NVFP4;
    if (std::strcmp(s, "w4a8-mxfp4") == 0) return HQ_MODE_W4A8_MXFP4;
    return -1;
}

// A plain strided CUDA tensor (no subclass, no wrapper of a transform) or null.
const at::Tensor* plain_tensor(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage()) return nullptr;
    if (t.unsafeGetTensorImpl()->is_python_dispatch()) return nullptr;
    return &t;
}

bool flag(PyObject* o, int* out) {
    if (o == Py_True || o == Py_False) {
        *out = o == Py_True ? 1 : 0;
        return true;
    }
    return false;
}

bool small_int(PyObject* o, int* out) {  // an int or an IntEnum member
    if (!PyLong_Check(o)) return false;
    int overflow = 0;
    const long v = PyLong_AsLongAndOverflow(o, &overflow);
    if (overflow != 0 || v < INT32_MIN || v > INT32_MAX) return false;
    *out = int(v);
    return true;
}

bool real(PyObject* o, float* out) {
    if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred() != nullptr) {
        PyErr_Clear();
        return false;
    }
    *out = float(v);
    return true;
}

bool bytes(const at::Tensor& t) { return t.itemsize() == 1; }
bool u8(const at::Tensor& t) { return t.scalar_type() == at::kByte; }

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// Gives the interpreter lock away for its lifetime.
class Unlocked {
    PyThreadState* const state_ = PyEval_SaveThread();

public:
    Unlocked() = default;
    Unlocked(const Unlocked&) = delete;
    ~Unlocked() { PyEval_RestoreThread(state_); }
};

// Runs without the interpreter lock, as torch.empty and a ctypes call do: the C ABI call, and the allocation of the
// outputs, which may wait for the device when the allocator has to free memory for it.
template <typename F>
int unlocked(F&& f) {
    char err[kErrLen];
    const Unlocked scope;
    return f(err);
}

// The same for the GEMMs, whose C ABI reads environment switches: they are read before the lock is given away, since an
// assignment to os.environ in another thread moves the array that they are in.
template <typename F>
int unlocked_gemm(F&& f) {
    const struct Held {
        Held() { g_fn.hold_switches(1); }
        Held(const Held&) = delete;
        ~Held() { g_fn.hold_switches(0); }
    } held;
    return unlocked(f);
}

PyObject* pair_of(const at::Tensor& a, const at::Tensor& b) {
    PyObject* const x = THPVariable_Wrap(a);
    PyObject* const y = x != nullptr ? THPVariable_Wrap(b) : nullptr;
    PyObject* const t = y != nullptr ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return t;
}

// rows of 16-bit elements as the quantizers read them
bool quant_input(const at::Tensor& x) {
    return x.dim() == 2 && x.stride(1) == 1 && (x.stride(0) * 2) % 16 == 0 &&
           reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
}

// group_wise_quant(input, mode, use_swizzle, use_pdl, output_quant, output_sf)
PyObject* group_wise_quant(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    int swizzle, pdl;
    if (nargs != 6 || g_fn.quant == nullptr || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor* const x = plain_tensor(a[0]);
    const int mode = mode_id(a[1]);
    if (x == nullptr || mode < 0 || mode == HQ_MODE_W4A8_MXFP4 || !flag(a[2], &swizzle) || !flag(a[3], &pdl)) Py_RETURN_NONE;
    const bool bf16 = x->scalar_type() == at::kBFloat16;
    if ((!bf16 && x->scalar_type() != at::kHalf) || !quant_input(*x)) Py_RETURN_NONE;
    const int64_t m = x->size(0), k = x->size(1), group = mode == HQ_MODE_W4A4_NVFP4 ? 16 : 32, kb = k / group;
    if (m == 0 || k == 0 || k % group != 0 || (swizzle != 0 && kb % 4 != 0)) Py_RETURN_NONE;
    const int64_t m_sf = swizzle != 0 ? (m + 127) / 128 * 128 : m;
    const int64_t qk = mode == HQ_MODE_W8A8_MXFP8 ? k : k / 2;
    const auto qt = mode == HQ_MODE_W8A8_MXFP8 ? at::kFloat8_e4m3fn : at::kByte;
    at::Tensor q, sf;
    if (a[4] != Py_None) {
        const at::Tensor* const t = plain_tensor(a[4]);
        if (t == nullptr || !t->is_contiguous() || t->scalar_type() != qt || t->numel() != m * qk || t->device() != x->device()) {
            Py_RETURN_NONE;
        }
        q = *t;
    }
    if (a[5] != Py_None) {
        const at::Tensor* const t = plain_tensor(a[5]);
        if (t == nullptr || !t->is_contiguous() || !u8(*t) || t->numel() != m_sf * kb || t->device() != x->device()) {
            Py_RETURN_NONE;
        }
        sf = *t;
    }
    const void* const px = x->data_ptr();
    const int64_t ld = x->stride(0);
    const int dev = x->get_device();
    void* const st = stream_of(*x);
    const auto on_device = at::TensorOptions().device(x->device());
    if (unlocked([&](char* err) {
            if (!q.defined()) q = at::empty({m, qk}, on_device.dtype(qt));
            if (!sf.defined()) sf = at::empty({m_sf, kb}, on_device.dtype(at::kByte));
            return g_fn.quant(px, ld, bf16 ? HQ_DTYPE_BF16 : HQ_DTYPE_FP16, m, k, mode, swizzle, pdl, q.data_ptr(), sf.data_ptr(), dev, st, err, kErrLen);
        }) != 0) {
        Py_RETURN_NONE;
    }
    if (a[4] != Py_None && a[5] != Py_None) return PyTuple_Pack(2, a[4], a[5]);
    return pair_of(q, sf);
    END_HANDLE_TH_ERRORS
}

// rms_norm_quant(input, weight, eps, use_swizzle, use_pdl)
PyObject* rms_norm_quant(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    int swizzle, pdl;
    float eps;
    if (nargs != 5 || g_fn.rms == nullptr || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor* const x = plain_tensor(a[0]);
    const at::Tensor* const w = plain_tensor(a[1]);
    if (x == nullptr || w == nullptr || !real(a[2], &eps) || !flag(a[3], &swizzle) || !flag(a[4], &pdl)) Py_RETURN_NONE;
    if (x->scalar_type() != at::kBFloat16 || !quant_input(*x) || x->size(0) == 0) Py_RETURN_NONE;
    const int64_t m = x->size(0), k = x->size(1);
    if (k % 128 != 0 || k <= 0 || k > 8192 || w->dim() != 1 || w->size(0) != k || w->scalar_type() != at::kBFloat16 ||
        !w->is_contiguous() || w->device() != x->device()) {
        Py_RETURN_NONE;
    }
    const int64_t m_sf = swizzle != 0 ? (m + 127) / 128 * 128 : m;
    const void* const px = x->data_ptr();
    const int64_t ld = x->stride(0);
    const void* const pw = w->data_ptr();
    const int dev = x->get_device();
    void* const st = stream_of(*x);
    const auto on_device = at::TensorOptions().device(x->device());
    at::Tensor q, sf;
    if (unlocked([&](char* err) {
            q = at::empty({m, k}, on_device.dtype(at::kFloat8_e4m3fn));
            sf = at::empty({m_sf, k / 32}, on_device.dtype(at::kByte));
            return g_fn.rms(px, ld, pw, eps, m, k, swizzle, pdl, q.data_ptr(), sf.data_ptr(), dev, st, err, kErrLen);
        }) != 0) {
        Py_RETURN_NONE;
    }
    return pair_of(q, sf);
    END_HANDLE_TH_ERRORS
}

// ---- FP8 with a scale per block of 128, tokens in expert order

int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

int in_dtype(const at::Tensor& t) {
    return t.scalar_type() == at::kBFloat16 ? HQ_DTYPE_BF16 : t.scalar_type() == at::kHalf ? HQ_DTYPE_FP16 : -1;
}
int any_dtype(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? HQ_DTYPE_FP32 : in_dtype(t); }

// rows of 16-bit elements as the kernels read them
bool rows16(const at::Tensor& x) {
    if (x.stride(-1) != 1 || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0) return false;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) {
        if (x.size(i) > 1 && x.stride(i) % 8 != 0) return false;
    }
    return true;
}
// elements between rows (of a single row: of no consequence, whatever its stride)
int64_t pitch(const at::Tensor& x, int64_t dim) { return x.size(dim) > 1 ? x.stride(dim) : (x.size(-1) + 7) / 8 * 8; }

// An output that the caller may have given: false if it is not what it should be.
bool given(PyObject* o, c10::IntArrayRef shape, at::ScalarType type, const at::Tensor& like, at::Tensor* out) {
    if (o == Py_None) return true;
    const at::Tensor* const t = plain_tensor(o);
    if (t == nullptr || !t->is_contiguous() || t->scalar_type() != type || t->sizes() != shape || t->device() != like.device()) return false;
    *out = *t;
    return true;
}

// A new tensor without the dispatcher: at::empty takes the host 1.2 us, and a small call makes up to four.
at::Tensor fresh(c10::IntArrayRef shape, at::ScalarType type, c10::Device device) {
    return at::Tensor(at::detail::empty_cuda(shape, type, device, c10::nullopt));
}

// Several tensors of one allocation (256-byte aligned), which lives as long as the last of them: for a sort, whose four are of one use (one
// allocation instead of four saves the host 1.4 of 6.0 us).  Codes and scales have a storage each: in a common one the scales would
// keep 33 times their bytes, be saved together with the codes, and be gone with them when a caller frees the codes' storage.
class Together {
    int64_t bytes_ = 0;
    struct Part {
        at::Tensor* to;
        c10::IntArrayRef shape;
        at::ScalarType type;
        int64_t at;
    } parts_[4];
    int n_ = 0;

public:
    void add(at::Tensor* to, c10::IntArrayRef shape, at::ScalarType type) {
        int64_t size = int64_t(c10::elementSize(type));
        for (const int64_t d : shape) size *= d;
        parts_[n_++] = {to, shape, type, bytes_};
        bytes_ += (size + 255) / 256 * 256;
    }
    void make(c10::Device device) {
        const at::Tensor whole = fresh({bytes_}, at::kByte, device);
        for (int i = 0; i < n_; ++i) {
            const Part& p = parts_[i];
            at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), c10::scalarTypeToTypeMeta(p.type));
            t.unsafeGetTensorImpl()->set_sizes_contiguous(p.shape);
            t.unsafeGetTensorImpl()->set_storage_offset(p.at / int64_t(c10::elementSize(p.type)));
            *p.to = std::move(t);
        }
    }
};

PyObject* pair_or_given(PyObject* a, const at::Tensor& x, PyObject* b, const at::Tensor& y) {
    PyObject* const p = a != Py_None ? Py_NewRef(a) : THPVariable_Wrap(x);
    PyObject* const q = p == nullptr ? nullptr : b != Py_None ? Py_NewRef(b) : THPVariable_Wrap(y);
    PyObject* const t = q != nullptr ? PyTuple_Pack(2, p, q) : nullptr;
    Py_XDECREF(p);
    Py_XDECREF(q);
    return t;
}

// block_quant(input, block, transpose, use_pdl, output_quant, output_sf)
PyObject* block_quant(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    int transpose, pdl, rows, cols;
    if (nargs != 6 || g_fn.block_quant == nullptr || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor* const x = plain_tensor(a[0]);
    if (x == nullptr || !PyTuple_CheckExact(a[1]) || PyTuple_GET_SIZE(a[1]) != 2 || !small_int(PyTuple_GET_ITEM(a[1], 0), &rows) ||
        !small_int(PyTuple_GET_ITEM(a[1], 1), &cols) || !flag(a[2], &transpose) || !flag(a[3], &pdl)) {
        Py_RETURN_NONE;
    }
    if (cols != 128 || (rows != 1 && rows != 128) || !(x->dim() == 2 || (rows == 128 && x->dim() == 3))) Py_RETURN_NONE;
    const int type = in_dtype(*x);
    const int64_t m = x->size(-2), k = x->size(-1), e = x->dim() == 3 ? x->size(0) : 1;
    if (type < 0 || k % 16 != 0 || !rows16(*x)) Py_RETURN_NONE;
    const int64_t m16 = (m + 15) / 16 * 16, r = transpose ? k : m, c = transpose ? m : k;
    const int64_t q_shape[3] = {e, r, transpose ? m16 : k}, s_shape[3] = {e, rows == 128 ? blocks_of(r) : r, blocks_of(c)};
    const size_t skip = x->dim() == 3 ? 0 : 1;
    const c10::IntArrayRef qs(q_shape + skip, 3 - skip), ss(s_shape + skip, 3 - skip);
    at::Tensor q, sf;
    if (!given(a[4], qs, at::kFloat8_e4m3fn, *x, &q) || !given(a[5], ss, at::kFloat, *x, &sf)) Py_RETURN_NONE;
    const void* const px = x->data_ptr();
    const int64_t ld = pitch(*x, -2), batch = x->dim() == 3 ? pitch(*x, 0) : 0;
    const int dev = x->get_device();
    void* const st = stream_of(*x);
    const c10::Device device = x->device();
    if (unlocked([&](char* err) {
            if (!q.defined()) q = fresh(qs, at::kFloat8_e4m3fn, device);
            if (!sf.defined()) sf = fresh(ss, at::kFloat, device);
            return g_fn.block_quant(px, ld, batch, type, e, m, k, rows, transpose, pdl, q.data_ptr(), sf.data_ptr(), dev, st, err, kErrLen);
        }) != 0) {
        Py_RETURN_NONE;
    }
    return pair_or_given(a[4], q, a[5], sf);
    END_HANDLE_TH_ERRORS
}

// swiglu_block_quant(input, offsets, use_pdl, output_quant, output_sf)
PyObject* swiglu_block_quant(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    int pdl;
    if (nargs != 5 || g_fn.swiglu == nullptr || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor* const x = plain_tensor(a[0]);
    if (x == nullptr || x->dim() != 2 || !flag(a[2], &pdl)) Py_RETURN_NONE;
    const int type = in_dtype(*x);
    const int64_t m = x->size(0), k = x->size(1) / 2;
    if (type < 0 || x->size(1) % 32 != 0 || !rows16(*x)) Py_RETURN_NONE;
    const int32_t* limit = nullptr;
    if (a[1] != Py_None) {
        const at::Tensor* const o = plain_tensor(a[1]);
        if (o == nullptr || o->dim() != 1 || o->size(0) < 1 || o->scalar_type() != at::kInt || !o->is_contiguous() || o->device() != x->device()) {
            Py_RETURN_NONE;
        }
        limit = static_cast<const int32_t*>(o->data_ptr()) + (o->size(0) - 1);
    }
    const int64_t qs[2] = {m, k}, ss[2] = {m, blocks_of(k)};
    at::Tensor q, sf;
    if (!given(a[3], qs, at::kFloat8_e4m3fn, *x, &q) || !given(a[4], ss, at::kFloat, *x, &sf)) Py_RETURN_NONE;
    const void* const px = x->data_ptr();
    const int64_t ld = pitch(*x, 0);
    const int dev = x->get_device();
    void* const st = stream_of(*x);
    const c10::Device device = x->device();
    if (unlocked([&](char* err) {
            if (!q.defined()) q = fresh(qs, at::kFloat8_e4m3fn, device);
            if (!sf.defined()) sf = fresh(ss, at::kFloat, device);
            return g_fn.swiglu(px, ld, type, m, k, limit, pdl, q.data_ptr(), sf.data_ptr(), dev, st, err, kErrLen);
        }) != 0) {
        Py_RETURN_NONE;
    }
    return pair_or_given(a[3], q, a[4], sf);
    END_HANDLE_TH_ERRORS
}

// block_gemm(input, weight, sfa, sfb, offsets or None, output, sm_count, use_pdl) -> True
PyObject* block_gemm(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    int pdl, sm_count;
    if (nargs != 8 || g_fn.block_gemm == nullptr || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor* const x = plain_tensor(a[0]);
    const at::Tensor* const w = plain_tensor(a[1]);
    const at::Tensor* const sfa = plain_tensor(a[2]);
    const at::Tensor* const sfb = plain_tensor(a[3]);
    const bool grouped = a[4] != Py_None;
    const at::Tensor* const offsets = grouped ? plain_tensor(a[4]) : nullptr;
    const at::Tensor* const out = plain_tensor(a[5]);
    if (x == nullptr || w == nullptr || sfa == nullptr || sfb == nullptr || out == nullptr || (grouped && offsets == nullptr) ||
        !small_int(a[6], &sm_count) || !flag(a[7], &pdl)) {
        Py_RETURN_NONE;
    }
    if (x->dim() != 2 || w->dim() != (grouped ? 3 : 2) || sfa->dim() != 2 || sfb->dim() != w->dim() || out->dim() != 2) Py_RETURN_NONE;
    const int64_t m = x->size(0), k = x->size(1), n = w->size(-2), e = grouped ? w->size(0) : 1, kb = blocks_of(k);
    const int type = any_dtype(*out);
    if (m == 0 || n == 0 || e == 0 || k < 16 || k % 16 != 0 || w->size(-1) != k || type < 0) Py_RETURN_NONE;
    if (x->scalar_type() != at::kFloat8_e4m3fn || w->scalar_type() != at::kFloat8_e4m3fn || sfa->scalar_type() != at::kFloat ||
        sfb->scalar_type() != at::kFloat) {
        Py_RETURN_NONE;
    }
    const auto dev = x->device();
    if (w->device() != dev || sfa->device() != dev || sfb->device() != dev || out->device() != dev) Py_RETURN_NONE;
    if (!x->is_contiguous() || !w->is_contiguous() || !sfa->is_contiguous() || !sfb->is_contiguous()) Py_RETURN_NONE;
    if (sfa->size(0) != m || sfa->size(1) != kb || sfb->size(-1) != kb) Py_RETURN_NONE;
    const bool square = sfb->size(-2) == blocks_of(n);
    if (grouped ? (!square || sfb->size(0) != e) : (!square && sfb->size(0) != n)) Py_RETURN_NONE;
    if (out->size(0) != m || out->size(1) != n || (out->stride(1) != 1 && n > 1) || (out->stride(0) < n && m > 1)) Py_RETURN_NONE;
    if (grouped && (offsets->dim() != 1 || offsets->scalar_type() != at::kInt || offsets->size(0) != e + 1 || !offsets->is_contiguous() ||
                    offsets->device() != dev)) {
        Py_RETURN_NONE;
    }
    const void *const px = x->data_ptr(), *const pw = w->data_ptr();
    if (reinterpret_cast<uintptr_t>(px) % 16 != 0 || reinterpret_cast<uintptr_t>(pw) % 16 != 0) Py_RETURN_NONE;
    const float *const pa = static_cast<const float*>(sfa->data_ptr()), *const pb = static_cast<const float*>(sfb->data_ptr());
    const int32_t* const po = grouped ? static_cast<const int32_t*>(offsets->data_ptr()) : nullptr;
    void* const y = out->data_ptr();
    const int64_t ldo = std::max(out->stride(0), n);
    const int d = x->get_device();
    void* const st = stream_of(*x);
    const int rc = unlocked([&](char* err) {
        return grouped ? g_fn.group_block_gemm(px, pw, pa, pb, po, y, type, e, m, n, k, ldo, sm_count, pdl, d, st, err, kErrLen)
                       : g_fn.block_gemm(px, pw, pa, pb, y, type, m, n, k, square ? 0 : 1, ldo, sm_count, pdl, d, st, err, kErrLen);
    });
    if (rc != 0) Py_RETURN_NONE;
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// moe_sort(topk_ids, num_experts, align, use_pdl) -> (rows, pairs, offsets, expert_ids)
PyObject* moe_sort(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    int experts, align, pdl;
    if (nargs != 4 || g_fn.moe_sort == nullptr || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor* const ids = plain_tensor(a[0]);
    if (ids == nullptr || ids->dim() != 2 || !ids->is_contiguous() || !small_int(a[1], &experts) || !small_int(a[2], &align) || !flag(a[3], &pdl)) {
        Py_RETURN_NONE;
    }
    if ((ids->scalar_type() != at::kInt && ids->scalar_type() != at::kLong) || experts < 1 || experts > 1024 || align < 1 || align > 4096) {
        Py_RETURN_NONE;
    }
    const int64_t n = ids->numel(), n_rows = (n + std::min<int64_t>(experts, n) * (align - 1)) / align * align;
    if (n > (int64_t(1) << 31) - 8192 || n_rows > INT32_MAX) Py_RETURN_NONE;
    const void* const p = ids->data_ptr();
    const int dev = ids->get_device();
    void* const st = stream_of(*ids);
    const c10::Device device = ids->device();
    const int64_t rows_shape[1] = {n_rows}, offsets_shape[1] = {experts + 1};
    at::Tensor out[4];
    if (unlocked([&](char* err) {
            Together outputs;
            outputs.add(&out[0], ids->sizes(), at::kInt);
            outputs.add(&out[1], rows_shape, at::kInt);
            outputs.add(&out[2], offsets_shape, at::kInt);
            outputs.add(&out[3], rows_shape, at::kInt);
            outputs.make(device);
            int32_t* at[4];
            for (int i = 0; i < 4; ++i) at[i] = static_cast<int32_t*>(out[i].data_ptr());
            return g_fn.moe_sort(p, int(ids->element_size()), ids->size(0), ids->size(1), experts, align, n_rows, pdl, at[0], at[1], at[2], at[3],
                                 dev, st, err, kErrLen);
        }) != 0) {
        Py_RETURN_NONE;
    }
    PyObject* const t = PyTuple_New(4);
    for (int i = 0; t != nullptr && i < 4; ++i) {
        PyObject* const v = THPVariable_Wrap(out[i]);
        if (v == nullptr) {
            Py_DECREF(t);
            return nullptr;
        }
        PyTuple_SET_ITEM(t, i, v);
    }
    return t;
    END_HANDLE_TH_ERRORS
}

// the fields of a MoeSort
struct Order {
    const int32_t *rows, *pairs, *offsets;
    int64_t tokens, topk, n_rows, experts;
    int padded;

    bool read(PyObject* o, c10::Device device) {
        if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 5) return false;
        const at::Tensor* t[3];
        for (int i = 0; i < 3; ++i) {
            t[i] = plain_tensor(PyTuple_GET_ITEM(o, i));
            if (t[i] == nullptr || t[i]->dim() != (i == 0 ? 2 : 1) || t[i]->scalar_type() != at::kInt || !t[i]->is_contiguous() ||
                t[i]->device() != device) {
                return false;
            }
        }
        int align;
        if (!small_int(PyTuple_GET_ITEM(o, 4), &align) || t[2]->size(0) < 1) return false;
        rows = static_cast<const int32_t*>(t[0]->data_ptr());
        pairs = static_cast<const int32_t*>(t[1]->data_ptr());
        offsets = static_cast<const int32_t*>(t[2]->data_ptr());
        tokens = t[0]->size(0), topk = t[0]->size(1), n_rows = t[1]->size(0), experts = t[2]->size(0) - 1;
        padded = align > 1 ? 1 : 0;
        return true;
    }
};

// moe_permute(input, sort, output, use_pdl)
PyObject* moe_permute(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    int pdl;
    Order order;
    if (nargs != 4 || g_fn.moe_permute == nullptr || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor* const x = plain_tensor(a[0]);
    if (x == nullptr || x->dim() != 2 || (x->stride(1) != 1 && x->size(1) > 1) || !order.read(a[1], x->device()) || !flag(a[3], &pdl)) Py_RETURN_NONE;
    const int64_t size = x->element_size(), h = x->size(1);
    if ((size != 1 && size != 2 && size != 4) || x->size(0) != order.tokens) Py_RETURN_NONE;
    const int64_t shape[2] = {order.n_rows, h};
    at::Tensor out;
    if (!given(a[2], shape, x->scalar_type(), *x, &out)) Py_RETURN_NONE;
    const void* const px = x->data_ptr();
    const int64_t ld = x->stride(0) * size;
    const int dev = x->get_device();
    void* const st = stream_of(*x);
    if (unlocked([&](char* err) {
            if (!out.defined()) out = fresh(shape, x->scalar_type(), x->device());
            return g_fn.moe_permute(px, ld, order.tokens, h * size, order.topk, order.rows, order.pairs, order.offsets, order.experts, order.n_rows,
                                    order.padded, pdl, out.data_ptr(), dev, st, err, kErrLen);
        }) != 0) {
        Py_RETURN_NONE;
    }
    return a[2] != Py_None ? Py_NewRef(a[2]) : THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// moe_permute_block_quant(input, sort, use_pdl, output_quant, output_sf)
PyObject* moe_permute_block_quant(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    int pdl;
    Order order;
    if (nargs != 5 || g_fn.moe_permute_quant == nullptr || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor* const x = plain_tensor(a[0]);
    if (x == nullptr || x->dim() != 2 || !order.read(a[1], x->device()) || !flag(a[2], &pdl)) Py_RETURN_NONE;
    const int type = in_dtype(*x);
    const int64_t h = x->size(1);
    if (type < 0 || h % 16 != 0 || !rows16(*x) || x->size(0) != order.tokens) Py_RETURN_NONE;
    const int64_t qs[2] = {order.n_rows, h}, ss[2] = {order.n_rows, blocks_of(h)};
    at::Tensor q, sf;
    if (!given(a[3], qs, at::kFloat8_e4m3fn, *x, &q) || !given(a[4], ss, at::kFloat, *x, &sf)) Py_RETURN_NONE;
    const void* const px = x->data_ptr();
    const int64_t ld = pitch(*x, 0);
    const int dev = x->get_device();
    void* const st = stream_of(*x);
    const c10::Device device = x->device();
    if (unlocked([&](char* err) {
            if (!q.defined()) q = fresh(qs, at::kFloat8_e4m3fn, device);
            if (!sf.defined()) sf = fresh(ss, at::kFloat, device);
            return g_fn.moe_permute_quant(px, ld, type, order.tokens, h, order.topk, order.rows, order.pairs, order.offsets, order.experts,
                                          order.n_rows, order.padded, pdl, q.data_ptr(), sf.data_ptr(), dev, st, err, kErrLen);
        }) != 0) {
        Py_RETURN_NONE;
    }
    return pair_or_given(a[3], q, a[4], sf);
    END_HANDLE_TH_ERRORS
}

// the weights of the pairs, or none
bool pair_weights(PyObject* o, const Order& order, c10::Device device, const float** weights) {
    *weights = nullptr;
    if (o == Py_None) return true;
    const at::Tensor* const t = plain_tensor(o);
    if (t == nullptr || t->scalar_type() != at::kFloat || t->dim() != 2 || t->size(0) != order.tokens || t->size(1) != order.topk ||
        !t->is_contiguous() || t->device() != device) {
        return false;
    }
    *weights = static_cast<const float*>(t->data_ptr());
    return true;
}

// moe_unpermute(input, sort, weights, use_pdl)
PyObject* moe_unpermute(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    int pdl;
    Order order;
    const float* weights;
    if (nargs != 4 || g_fn.moe_unpermute == nullptr || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor* const z = plain_tensor(a[0]);
    if (z == nullptr || z->dim() != 2 || (z->stride(1) != 1 && z->size(1) > 1) || !order.read(a[1], z->device()) ||
        !pair_weights(a[2], order, z->device(), &weights) || !flag(a[3], &pdl)) {
        Py_RETURN_NONE;
    }
    const int type = any_dtype(*z);
    const int64_t h = z->size(1);
    if (type < 0 || z->size(0) != order.n_rows) Py_RETURN_NONE;
    const void* const pz = z->data_ptr();
    const int64_t ld = z->stride(0);
    const int dev = z->get_device();
    void* const st = stream_of(*z);
    at::Tensor out;
    if (unlocked([&](char* err) {
            out = fresh({order.tokens, h}, z->scalar_type(), z->device());
            return g_fn.moe_unpermute(pz, ld, type, order.n_rows, h, order.tokens, order.topk, order.rows, weights, pdl, out.data_ptr(), dev, st, err,
                                      kErrLen);
        }) != 0) {
        Py_RETURN_NONE;
    }
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// moe_unpermute_backward(grad_output, input, sort, weights, use_pdl, grad_input)
PyObject* moe_unpermute_backward(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    int pdl;
    Order order;
    const float* weights;
    if (nargs != 6 || g_fn.moe_unpermute_backward == nullptr || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor* const g = plain_tensor(a[0]);
    const at::Tensor* const z = plain_tensor(a[1]);
    if (g == nullptr || z == nullptr || g->dim() != 2 || z->dim() != 2 || (z->stride(1) != 1 && z->size(1) > 1) ||
        (g->stride(1) != 1 && g->size(1) > 1) || !order.read(a[2], z->device()) || !pair_weights(a[3], order, z->device(), &weights) ||
        !flag(a[4], &pdl)) {
        Py_RETURN_NONE;
    }
    const int type = any_dtype(*z);
    const int64_t h = z->size(1);
    if (type < 0 || g->scalar_type() != z->scalar_type() || g->device() != z->device() || z->size(0) != order.n_rows || g->size(0) != order.tokens ||
        g->size(1) != h) {
        Py_RETURN_NONE;
    }
    const int64_t shape[2] = {order.n_rows, h};
    at::Tensor gz, gw;
    if (!given(a[5], shape, z->scalar_type(), *z, &gz)) Py_RETURN_NONE;
    const void *const pg = g->data_ptr(), *const pz = z->data_ptr();
    const int64_t ld_g = g->stride(0), ld_z = z->stride(0);
    const int dev = z->get_device();
    void* const st = stream_of(*z);
    if (unlocked([&](char* err) {
            if (!gz.defined()) gz = fresh(shape, z->scalar_type(), z->device());
            if (a[3] != Py_None) gw = fresh({order.tokens, order.topk}, at::kFloat, z->device());
            return g_fn.moe_unpermute_backward(pg, ld_g, pz, ld_z, type, order.n_rows, h, order.tokens, order.topk, order.rows, order.pairs,
                                               order.offsets, order.experts, order.padded, weights, pdl, gz.data_ptr(),
                                               gw.defined() ? static_cast<float*>(gw.data_ptr()) : nullptr, dev, st, err, kErrLen);
        }) != 0) {
        Py_RETURN_NONE;
    }
    PyObject* const p = a[5] != Py_None ? Py_NewRef(a[5]) : THPVariable_Wrap(gz);
    PyObject* const q = p == nullptr ? nullptr : gw.defined() ? THPVariable_Wrap(gw) : Py_NewRef(Py_None);
    PyObject* const t = q != nullptr ? PyTuple_Pack(2, p, q) : nullptr;
    Py_XDECREF(p);
    Py_XDECREF(q);
    return t;
    END_HANDLE_TH_ERRORS
}

// ---- GEMMs with block scales of the MX kinds: they read environment switches

// dense_gemm(input, weight, sfa, sfb, output, bias, alpha, sm_count, mode, use_pdl, epilogue, output_sf,
//            situ_beta, situ_linear_beta) -> True, or None when the call is not an ordinary one
PyObject* dense_gemm(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    constexpr int kIdentity = HQ_EPILOGUE_IDENTITY, kSigmoid = HQ_EPILOGUE_SIGMOID, kSitu = HQ_EPILOGUE_SITU_QUANT;
    int sm_count, pdl, epilogue;
    if (nargs != 14 || g_fn.dense == nullptr || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor* const x = plain_tensor(a[0]);
    const at::Tensor* const w = plain_tensor(a[1]);
    const at::Tensor* const sfa = plain_tensor(a[2]);
    const at::Tensor* const sfb = plain_tensor(a[3]);
    const at::Tensor* const out = plain_tensor(a[4]);
    const int mode = mode_id(a[8]);
    if (x == nullptr || w == nullptr || sfa == nullptr || sfb == nullptr || out == nullptr || mode < 0 ||
        mode == HQ_MODE_W4A8_MXFP4 || !small_int(a[7], &sm_count) || !small_int(a[9], &pdl) || pdl < 0 || pdl > 2 || !small_int(a[10], &epilogue)) {
        Py_RETURN_NONE;
    }
    const bool fp8 = mode == HQ_MODE_W8A8_MXFP8, nvfp4 = mode == HQ_MODE_W4A4_NVFP4, situ = epilogue == kSitu;
    if (epilogue != kIdentity && epilogue != kSigmoid && !(situ && fp8)) Py_RETURN_NONE;
    if (x->dim() != 2 || w->dim() != 2 || out->dim() != 2 || sfa->dim() < 1 || sfb->dim() < 1) Py_RETURN_NONE;
    if (!bytes(*x) || !bytes(*w) || !u8(*sfa) || !u8(*sfb)) Py_RETURN_NONE;
    const auto dev = x->device();
    if (w->device() != dev || sfa->device() != dev || sfb->device() != dev || out->device() != dev) Py_RETURN_NONE;
    if (!x->is_contiguous() || !w->is_contiguous() || !sfa->is_contiguous() || !sfb->is_contiguous()) Py_RETURN_NONE;
    const int64_t m = x->size(0), n = w->size(0), k = fp8 ? w->size(1) : w->size(1) * 2;
    if (m == 0 || n == 0 || x->size(1) != w->size(1)) Py_RETURN_NONE;
    if (out->size(0) != m || out->size(1) != (situ ? n / 2 : n)) Py_RETURN_NONE;
    const int64_t sf_k = k / (nvfp4 ? 16 : 32), m_sf = (m + 127) / 128 * 128;
    if (sfa->numel() < m_sf * sf_k) Py_RETURN_NONE;
    if (!fp8 && (sfa->size(-1) != sf_k || sfb->size(-1) != sf_k)) Py_RETURN_NONE;
    const void* bias = nullptr;
    if (a[5] != Py_None) {
        const at::Tensor* const b = plain_tensor(a[5]);
        if (!fp8 || (!situ && m % 256 != 0) || b == nullptr || b->scalar_type() != at::kBFloat16 || b->dim() != 1 ||
            b->numel() != n || !b->is_contiguous() || b->device() != dev) {
            Py_RETURN_NONE;
        }
        bias = b->data_ptr();
    }
    const float* alpha = nullptr;
    if (a[6] != Py_None) {
        const at::Tensor* const t = plain_tensor(a[6]);
        if (!nvfp4 || t == nullptr || t->scalar_type() != at::kFloat || t->numel() < 1 || t->device() != dev) Py_RETURN_NONE;
        alpha = static_cast<const float*>(t->data_ptr());
    } else if (nvfp4) {
        Py_RETURN_NONE;
    }
    const void* const px = x->data_ptr();
    const void* const pw = w->data_ptr();
    const void* const psa = sfa->data_ptr();
    const void* const psb = sfb->data_ptr();
    void* const po = out->data_ptr();
    const int64_t na = sfa->numel(), nb = sfb->numel(), ldo = out->stride(0);
    const int d = x->get_device();
    void* const st = stream_of(*x);
    int rc;
    if (situ) {
        float beta, lin = 0.0f;
        const at::Tensor* const osf = plain_tensor(a[11]);
        if (osf == nullptr || !u8(*osf) || !osf->is_contiguous() || osf->device() != dev || !out->is_contiguous() ||
            out->scalar_type() != at::kFloat8_e4m3fn || !real(a[12], &beta) || (a[13] != Py_None && !real(a[13], &lin))) {
            Py_RETURN_NONE;
        }
        void* const pos = osf->data_ptr();
        const int64_t no = osf->numel();
        rc = unlocked_gemm([&](char* err) {
            return g_fn.situ(px, pw, psa, psb, po, pos, bias, m, n, k, na, nb, no, beta, lin, sm_count, pdl != 0 ? 1 : 0, d, st,
                             err, kErrLen);
        });
    } else {
        if (out->scalar_type() != at::kBFloat16 || out->stride(1) != 1) Py_RETURN_NONE;
        rc = unlocked_gemm([&](char* err) {
            return g_fn.dense(px, pw, psa, psb, po, bias, alpha, m, n, k, na, nb, ldo, mode, epilogue, sm_count, pdl, d, st, err,
                              kErrLen);
        });
    }
    if (rc != 0) Py_RETURN_NONE;
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// grouped_gemm(kind, input, weight, sfa, sfb, table, output, bias, alpha, max_m_per_expert, sm_count, mode): kind 2 masked,
// 3 contiguous (whose max_m_per_expert is ignored)
PyObject* grouped_gemm(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    int kind, max_m, sm_count;
    if (nargs != 12 || g_fn.masked == nullptr || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
    const at::Tensor* const x = plain_tensor(a[1]);
    const at::Tensor* const w = plain_tensor(a[2]);
    const at::Tensor* const sfa = plain_tensor(a[3]);
    const at::Tensor* const sfb = plain_tensor(a[4]);
    const at::Tensor* const table = plain_tensor(a[5]);
    const at::Tensor* const out = plain_tensor(a[6]);
    const int mode = mode_id(a[11]);
    if (x == nullptr || w == nullptr || sfa == nullptr || sfb == nullptr || table == nullptr || out == nullptr || mode < 0 ||
        !small_int(a[0], &kind) || !small_int(a[9], &max_m) || !small_int(a[10], &sm_count)) {
        Py_RETURN_NONE;
    }
    const bool masked = kind == 2, fp8 = mode == HQ_MODE_W8A8_MXFP8, nvfp4 = mode == HQ_MODE_W4A4_NVFP4,
               w4a8 = mode == HQ_MODE_W4A8_MXFP4;
    if (x->dim() != 2 || w->dim() != 3 || table->dim() != 1 || out->dim() != 2 || sfa->dim() < 1 || sfb->dim() < 1) {
        Py_RETURN_NONE;
    }
    if (!bytes(*x) || !bytes(*w) || !u8(*sfa) || !u8(*sfb) || table->scalar_type() != at::kInt) Py_RETURN_NONE;
    const auto dev = x->device();
    if (w->device() != dev || sfa->device() != dev || sfb->device() != dev || out->device() != dev || table->device() != dev) {
        Py_RETURN_NONE;
    }
    const int64_t m = x->size(0), e = w->size(0), n = w->size(1), k = fp8 ? w->size(2) : w->size(2) * 2;
    if (m == 0 || n == 0 || e == 0 || x->size(1) != (w4a8 ? k : w->size(2))) Py_RETURN_NONE;
    if (masked ? (max_m <= 0 || m != e * int64_t(max_m) || table->size(0) != e) : table->size(0) != m) Py_RETURN_NONE;
    if (out->size(0) != m || out->size(1) != n || out->scalar_type() != at::kBFloat16 || out->stride(1) != 1) Py_RETURN_NONE;
    if (!x->is_contiguous() || !w->is_contiguous() || !sfa->is_contiguous() || !sfb->is_contiguous() ||
        !table->is_contiguous()) {
        Py_RETURN_NONE;
    }
    const int64_t sf_k = k / (nvfp4 ? 16 : 32);
    if (!fp8 && (sfa->size(-1) != sf_k || sfb->size(-1) != sf_k)) Py_RETURN_NONE;
    const void* bias = nullptr;
    if (a[7] != Py_None) {
        const at::Tensor* const b = plain_tensor(a[7]);
        if (!fp8 || b == nullptr || b->scalar_type() != at::kBFloat16 || b->numel() != e * n || !b->is_contiguous() ||
            b->device() != dev) {
            Py_RETURN_NONE;
        }
        bias = b->data_ptr();
    }
    const float* alpha = nullptr;
    if (a[8] != Py_None) {
        const at::Tensor* const t = plain_tensor(a[8]);
        if (!nvfp4 || t == nullptr || t->scalar_type() != at::kFloat || t->numel() != e || !t->is_contiguous() ||
            t->device() != dev) {
            Py_RETURN_NONE;
        }
        alpha = static_cast<const float*>(t->data_ptr());
    } else if (nvfp4) {
        Py_RETURN_NONE;
    }
    const void* const px = x->data_ptr();
    const void* const pw = w->data_ptr();
    const void* const psa = sfa->data_ptr();
    const void* const psb = sfb->data_ptr();
    const int32_t* const pt = static_cast<const int32_t*>(table->data_ptr());
    void* const po = out->data_ptr();
    const int64_t na = sfa->numel(), nb = sfb->numel(), ldo = out->stride(0);
    const int d = x->get_device();
    void* const st = stream_of(*x);
    const int rc = unlocked_gemm([&](char* err) {
        // the shape rules that the wrapper asks for first
        if (g_fn.describe_group(kind, e, masked ? max_m : m / e, m, n, k, mode, 148, -1, err, kErrLen) != 0) return 1;
        return (masked ? g_fn.masked : g_fn.contiguous)(px, pw, psa, psb, pt, po, bias, alpha, e, masked ? max_m : m, n, k, na,
                                                        nb, ldo, mode, sm_count, 1, d, st, err, kErrLen);
    });
    if (rc != 0) Py_RETURN_NONE;
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// bind_block(block_quant, swiglu, block_gemm, group_block_gemm, moe_sort, moe_permute, moe_permute_quant, moe_unpermute,
// moe_unpermute_backward): addresses, as for bind
PyObject* bind_block(PyObject*, PyObject* args) {
    unsigned long long p[9];
    if (!PyArg_ParseTuple(args, "KKKKKKKKK", &p[0], &p[1], &p[2], &p[3], &p[4], &p[5], &p[6], &p[7], &p[8])) return nullptr;
    const auto set = [&](auto& fn, int i) { fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(p[i]); };
    set(g_fn.block_quant, 0);
    set(g_fn.swiglu, 1);
    set(g_fn.block_gemm, 2);
    set(g_fn.group_block_gemm, 3);
    set(g_fn.moe_sort, 4);
    set(g_fn.moe_permute, 5);
    set(g_fn.moe_permute_quant, 6);
    set(g_fn.moe_unpermute, 7);
    set(g_fn.moe_unpermute_backward, 8);
    Py_RETURN_NONE;
}

// bind(quant, rms, dense, situ, describe_group, masked, contiguous, hold_switches): addresses of the C ABI's entry points
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long p[8];
    if (!PyArg_ParseTuple(args, "KKKKKKKK", &p[0], &p[1], &p[2], &p[3], &p[4], &p[5], &p[6], &p[7])) return nullptr;
    g_fn.quant = reinterpret_cast<QuantFn>(p[0]);
    g_fn.rms = reinterpret_cast<RmsFn>(p[1]);
    g_fn.dense = reinterpret_cast<DenseFn>(p[2]);
    g_fn.situ = reinterpret_cast<SituFn>(p[3]);
    g_fn.describe_group = reinterpret_cast<DescribeGroupFn>(p[4]);
    g_fn.masked = reinterpret_cast<MaskedFn>(p[5]);
    g_fn.contiguous = reinterpret_cast<ContiguousFn>(p[6]);
    g_fn.hold_switches = reinterpret_cast<decltype(&hq_hold_switches)>(p[7]);
    Py_RETURN_NONE;
}

template <typename F>
PyCFunction method(F f) {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {{"group_wise_quant", method(group_wise_quant), METH_FASTCALL, nullptr},
                         {"rms_norm_quant", method(rms_norm_quant), METH_FASTCALL, nullptr},
                         {"dense_gemm", method(dense_gemm), METH_FASTCALL, nullptr},
                         {"grouped_gemm", method(grouped_gemm), METH_FASTCALL, nullptr},
                         {"block_quant", method(block_quant), METH_FASTCALL, nullptr},
                         {"swiglu_block_quant", method(swiglu_block_quant), METH_FASTCALL, nullptr},
                         {"block_gemm", method(block_gemm), METH_FASTCALL, nullptr},
                         {"moe_sort", method(moe_sort), METH_FASTCALL, nullptr},
                         {"moe_permute", method(moe_permute), METH_FASTCALL, nullptr},
                         {"moe_permute_block_quant", method(moe_permute_block_quant), METH_FASTCALL, nullptr},
                         {"moe_unpermute", method(moe_unpermute), METH_FASTCALL, nullptr},
                         {"moe_unpermute_backward", method(moe_unpermute_backward), METH_FASTCALL, nullptr},
                         {"bind", bind, METH_VARARGS, nullptr},
                         {"bind_block", bind_block, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "halops_b200_fast_path", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_halops_b200_fast_path() { return PyModule_Create(&module); }
