// The host side of one call, natively: checks, output allocation, stream and scratch lookup, launch.
//
// At decode sizes a kernel of this library takes 3 to 10 us while the same steps in Python (tensor attribute reads, a
// device context manager, a stream object, two or three ctypes calls) take about 15 us, so an eager program is bound by
// them; here they take about 4 us.  Every function answers None for whatever is not the plain case -- CPU tensors,
// wrong types or shapes, tensors that need a copy first, an active dispatch mode, another current device, scratch that does not exist yet, a
// call that failed -- and the Python function that called it then takes its general path, which checks, copies,
// allocates and reports errors.  So this file decides nothing: it only makes the plain case short.
//
// The library's entry points are given as addresses by bind() (the ctypes binding looks them up), so that one loaded
// copy of the library serves both paths.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <type_traits>
#include <unordered_map>
#include <utility>

#include "../../include/hidet_b200q.h"

namespace {

struct Library {
    decltype(&b200q_symmetric_quantize) quantize = nullptr;
    decltype(&b200q_symmetric_dequantize) dequantize = nullptr;
    decltype(&b200q_embedding_dequantize) take = nullptr;
    decltype(&b200q_qlinear_workspace_bytes) workspace_bytes = nullptr;
    decltype(&b200q_qlinear_f16_i8) linear = nullptr;
    decltype(&b200q_qlinear_f16_i8_fused) linear_fused = nullptr;
    decltype(&b200q_qlinear_f16_u4_workspace_bytes) w4_workspace_bytes = nullptr;
    decltype(&b200q_qlinear_f16_u4) w4 = nullptr;
    decltype(&b200q_rotary_embedding) rotary = nullptr;
    decltype(&b200q_quantized_cache_append) append = nullptr;
    decltype(&b200q_quantized_cache_read) read = nullptr;
    decltype(&b200q_quantized_cache_attention_workspace_bytes) attention_workspace_bytes = nullptr;
    decltype(&b200q_quantized_cache_attention) attention = nullptr;
    decltype(&b200q_token_log_probs) log_probs = nullptr;
} lib;

// Scratch buffers that the Python side owns and has told us about, by stream and device.
struct Scratch {
    void *ptr;
    size_t bytes;
};
struct KeyHash {
    size_t operator()(const std::pair<uintptr_t, int> &k) const { return std::hash<uintptr_t>()(k.first) * 31 + (size_t)k.second; }
};
std::unordered_map<std::pair<uintptr_t, int>, Scratch, KeyHash> scratch;  // guarded by the GIL

#define PLAIN_OR_NONE(cond) \
    do {                    \
        if (!(cond)) Py_RETURN_NONE; \
    } while (0)

// A dispatch mode (fake tensors, tracing, counting) wants to see the operators the Python path runs.
inline bool watched() { return c10::impl::TorchDispatchModeTLS::any_modes_set(); }
// A strided CUDA tensor with memory of its own (a vmap or grad wrapper has none) and no Python-level overrides,
// contiguous: what a kernel can be given.
inline bool plain(const at::Tensor &t) {
    return t.is_cuda() && t.layout() == at::kStrided && t.has_storage() && !t.unsafeGetTensorImpl()->is_python_dispatch() &&
           t.is_contiguous() && !t.is_neg();
}
inline const at::Tensor *plain_tensor(PyObject *o) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    return plain(t) ? &t : nullptr;
}

struct Where {
    int device;
    cudaStream_t stream;
};
// The current stream of the tensor's device, if that device is the current one.
inline bool where_is(const at::Tensor &t, Where &w) {
    w.device = t.get_device();
    if (c10::cuda::current_device() != w.device) return false;
    w.stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)w.device).stream();
    return true;
}
inline bool find_scratch(const Where &w, size_t need, void *&ptr, size_t &bytes) {
    ptr = nullptr;
    bytes = 0;
    if (need == 0) return true;
    const auto it = scratch.find({reinterpret_cast<uintptr_t>(w.stream), w.device});
    if (it == scratch.end() || it->second.bytes < need) return false;
    ptr = it->second.ptr;
    bytes = it->second.bytes;
    return true;
}
inline at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, int device) {
    return at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, (c10::DeviceIndex)device), c10::nullopt);
}
inline int float_code(at::ScalarType t) { return t == at::kHalf ? B200Q_F16 : t == at::kBFloat16 ? B200Q_BF16 : t == at::kFloat ? B200Q_F32 : -1; }
inline int quant_code(at::ScalarType t) { return t == at::kChar ? B200Q_I8 : t == at::kShort ? B200Q_I16 : -1; }
inline bool is_text(PyObject *o, const char *text) { return PyUnicode_Check(o) && PyUnicode_CompareWithASCIIString(o, text) == 0; }

// dims of a 2-D tensor -> reduce_dim, or -1
inline int reduce_dim_of(PyObject *o) {
    if (!PyLong_CheckExact(o)) return -1;
    const long d = PyLong_AsLong(o);
    return d == 0 || d == -2 ? 0 : d == 1 || d == -1 ? 1 : -1;
}

#define WITHOUT_GIL(status, call) \
    do {                          \
        Py_BEGIN_ALLOW_THREADS status = (call); \
        Py_END_ALLOW_THREADS      \
    } while (0)

// linear(a, weight, scale, weight_layout, out, bias, residual, activation)
PyObject *linear(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    PLAIN_OR_NONE(n_args == 8 && lib.linear != nullptr && !watched());
    const at::Tensor *a = plain_tensor(args[0]), *weight = plain_tensor(args[1]), *scale = plain_tensor(args[2]);
    PLAIN_OR_NONE(a && weight && scale);
    const bool nk = is_text(args[3], "NK");
    PLAIN_OR_NONE(nk || is_text(args[3], "KN"));
    PLAIN_OR_NONE(a->dim() >= 2 && weight->dim() == 2 && scale->dim() == 1);
    PLAIN_OR_NONE(a->scalar_type() == at::kHalf && weight->scalar_type() == at::kChar && scale->scalar_type() == at::kHalf);
    const int64_t k = a->size(-1), m = [&] {
        int64_t p = 1;
        for (int64_t d = 0; d + 1 < a->dim(); ++d) p *= a->size(d);
        return p;
    }();
    const int64_t n = weight->size(nk ? 0 : 1);
    PLAIN_OR_NONE(k == weight->size(nk ? 1 : 0) && n == scale->size(0) && k % 2 == 0 && weight->size(1) % 2 == 0 && m > 0 && n > 0 && k > 0);
    const bool pairs = is_text(args[7], "silu_mul");
    PLAIN_OR_NONE(pairs || args[7] == Py_None);
    const bool fused = pairs || args[5] != Py_None || args[6] != Py_None;
    PLAIN_OR_NONE(!(fused && nk));
    Where w;
    PLAIN_OR_NONE(where_is(*a, w) && weight->get_device() == w.device && scale->get_device() == w.device);
    const int64_t n_out = pairs ? n / 2 : n;
    auto of_result_shape = [&](const at::Tensor *t) {
        if (!t || t->scalar_type() != at::kHalf || t->get_device() != w.device || t->dim() != a->dim() || t->size(-1) != n_out) return false;
        for (int64_t d = 0; d + 1 < a->dim(); ++d)
            if (t->size(d) != a->size(d)) return false;
        return true;
    };
    b200q_epilogue ep = {};
    if (args[5] != Py_None) {
        const at::Tensor *bias = plain_tensor(args[5]);
        PLAIN_OR_NONE(bias && bias->scalar_type() == at::kHalf && bias->get_device() == w.device && bias->dim() == 1 && bias->size(0) == n);
        ep.bias = bias->const_data_ptr();
    }
    if (args[6] != Py_None) {
        const at::Tensor *residual = plain_tensor(args[6]);
        PLAIN_OR_NONE(of_result_shape(residual));
        ep.residual = residual->const_data_ptr();
    }
    ep.ldr = n_out;
    ep.activation = pairs ? B200Q_ACT_SILU_MUL : B200Q_ACT_NONE;
    const int layout = nk ? B200Q_LAYOUT_NK : B200Q_LAYOUT_KN;
    void *ws;
    size_t ws_bytes;
    PLAIN_OR_NONE(find_scratch(w, lib.workspace_bytes(m, n, k, layout), ws, ws_bytes));
    at::Tensor made;
    void *c;
    if (args[4] != Py_None) {
        const at::Tensor *out = plain_tensor(args[4]);
        PLAIN_OR_NONE(of_result_shape(out));
        c = out->data_ptr();
    } else {
        at::DimVector shape(a->sizes());
        shape.back() = n_out;
        made = empty(shape, at::kHalf, w.device);
        c = made.data_ptr();
    }
    int status;
    const void *ap = a->const_data_ptr(), *wp = weight->const_data_ptr(), *sp = scale->const_data_ptr();
    WITHOUT_GIL(status, fused ? lib.linear_fused(ap, wp, sp, c, m, n, k, layout, &ep, ws, ws_bytes, w.stream)
                              : lib.linear(ap, wp, sp, c, m, n, k, layout, ws, ws_bytes, w.stream));
    PLAIN_OR_NONE(status == B200Q_OK);
    if (!made.defined()) return Py_NewRef(args[4]);
    return THPVariable_Wrap(std::move(made));
    END_HANDLE_TH_ERRORS
}

// quantize(w, quant_type, dims) -> (wq, scale)
PyObject *quantize(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    PLAIN_OR_NONE(n_args == 3 && lib.quantize != nullptr && !watched());
    const at::Tensor *x = plain_tensor(args[0]);
    PLAIN_OR_NONE(x && x->dim() == 2 && float_code(x->scalar_type()) >= 0);
    at::ScalarType q;
    if (is_text(args[1], "int8")) q = at::kChar;
    else if (is_text(args[1], "int16")) q = at::kShort;
    else if (THPDtype_Check(args[1])) q = reinterpret_cast<THPDtype *>(args[1])->scalar_type;
    else Py_RETURN_NONE;
    const int reduce = reduce_dim_of(args[2]);
    Where w;
    PLAIN_OR_NONE(quant_code(q) >= 0 && reduce >= 0 && x->numel() > 0 && where_is(*x, w));
    at::Tensor wq = empty(x->sizes(), q, w.device), scale = empty({x->size(reduce == 0 ? 1 : 0)}, x->scalar_type(), w.device);
    int status;
    const void *src = x->const_data_ptr();
    void *codes = wq.data_ptr(), *scales = scale.data_ptr();
    WITHOUT_GIL(status, lib.quantize(src, codes, scales, x->size(0), x->size(1), float_code(x->scalar_type()), quant_code(q), reduce, w.stream));
    PLAIN_OR_NONE(status == B200Q_OK);
    PyObject *first = THPVariable_Wrap(std::move(wq));
    PyObject *second = first ? THPVariable_Wrap(std::move(scale)) : nullptr;
    PyObject *pair = second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return pair;
    END_HANDLE_TH_ERRORS
}

// dequantize(wq, scale, dims)
PyObject *dequantize(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    PLAIN_OR_NONE(n_args == 3 && lib.dequantize != nullptr && !watched());
    const at::Tensor *q = plain_tensor(args[0]), *scale = plain_tensor(args[1]);
    PLAIN_OR_NONE(q && scale && q->dim() == 2 && scale->dim() == 1 && q->numel() > 0);
    const int reduce = reduce_dim_of(args[2]);
    const int fc = float_code(scale->scalar_type()), qc = quant_code(q->scalar_type());
    Where w;
    PLAIN_OR_NONE(reduce >= 0 && fc >= 0 && qc >= 0 && scale->size(0) == q->size(reduce == 0 ? 1 : 0) && where_is(*q, w) && scale->get_device() == w.device);
    at::Tensor out = empty(q->sizes(), scale->scalar_type(), w.device);
    int status;
    const void *codes = q->const_data_ptr(), *scales = scale->const_data_ptr();
    void *dst = out.data_ptr();
    WITHOUT_GIL(status, lib.dequantize(codes, scales, dst, q->size(0), q->size(1), fc, qc, reduce, w.stream));
    PLAIN_OR_NONE(status == B200Q_OK);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// take(wq, scale, indices)
PyObject *take(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    PLAIN_OR_NONE(n_args == 3 && lib.take != nullptr && !watched());
    const at::Tensor *q = plain_tensor(args[0]), *scale = plain_tensor(args[1]), *idx = plain_tensor(args[2]);
    PLAIN_OR_NONE(q && scale && idx && q->dim() == 2 && scale->dim() == 1 && scale->size(0) == q->size(0));
    const int fc = float_code(scale->scalar_type()), qc = quant_code(q->scalar_type());
    const bool wide = idx->scalar_type() == at::kLong;
    Where w;
    PLAIN_OR_NONE(fc >= 0 && qc >= 0 && (wide || idx->scalar_type() == at::kInt) && q->numel() > 0 && idx->numel() > 0 && where_is(*q, w) &&
                  scale->get_device() == w.device && idx->get_device() == w.device);
    at::DimVector shape(idx->sizes());
    shape.push_back(q->size(1));
    at::Tensor out = empty(shape, scale->scalar_type(), w.device);
    int status;
    const void *table = q->const_data_ptr(), *scales = scale->const_data_ptr(), *which = idx->const_data_ptr();
    void *dst = out.data_ptr();
    WITHOUT_GIL(status, lib.take(table, scales, which, dst, q->size(0), q->size(1), idx->numel(), fc, qc, wide ? 8 : 4, w.stream));
    PLAIN_OR_NONE(status == B200Q_OK);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// w4(a, codes, scale, zeros or None, k, n, group_size)
PyObject *w4(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    PLAIN_OR_NONE(n_args == 7 && lib.w4 != nullptr && !watched());
    const at::Tensor *a = plain_tensor(args[0]), *q = plain_tensor(args[1]), *scale = plain_tensor(args[2]);
    PLAIN_OR_NONE(a && q && scale && PyLong_CheckExact(args[4]) && PyLong_CheckExact(args[5]) && PyLong_CheckExact(args[6]));
    const int64_t k = PyLong_AsLongLong(args[4]), n = PyLong_AsLongLong(args[5]), group = PyLong_AsLongLong(args[6]);
    PLAIN_OR_NONE(k > 0 && n > 0 && group > 0);
    PLAIN_OR_NONE(a->dim() == 2 && a->scalar_type() == at::kHalf && a->size(1) == k && a->size(0) > 0);
    PLAIN_OR_NONE(q->dim() == 2 && q->size(0) == k && q->size(1) * (int64_t)q->element_size() * 2 == n);
    auto grouped = [&](const at::Tensor *t) { return t && t->scalar_type() == at::kHalf && t->dim() == 2 && t->size(0) == k / group && t->size(1) == n; };
    Where w;
    PLAIN_OR_NONE(grouped(scale) && where_is(*a, w) && q->get_device() == w.device && scale->get_device() == w.device);
    const void *zp = nullptr;
    if (args[3] != Py_None) {
        const at::Tensor *zeros = plain_tensor(args[3]);
        PLAIN_OR_NONE(grouped(zeros) && zeros->get_device() == w.device);
        zp = zeros->const_data_ptr();
    }
    const int64_t m = a->size(0);
    PLAIN_OR_NONE(group % 16 != 0 || (reinterpret_cast<uintptr_t>(a->const_data_ptr()) & 15u) == 0);  // else the general path aligns it
    void *ws;
    size_t ws_bytes;
    PLAIN_OR_NONE(find_scratch(w, lib.w4_workspace_bytes(m, n, k, group), ws, ws_bytes));
    at::Tensor out = empty({m, n}, at::kHalf, w.device);
    int status;
    const void *ap = a->const_data_ptr(), *codes = q->const_data_ptr(), *sp = scale->const_data_ptr();
    void *dst = out.data_ptr();
    WITHOUT_GIL(status, lib.w4(ap, codes, sp, zp, dst, m, n, k, group, ws, ws_bytes, w.stream));
    PLAIN_OR_NONE(status == B200Q_OK);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// Like plain_tensor for the heads of tokens, [tokens, heads, dim]: strides between tokens and heads are the kernels' to follow.
inline const at::Tensor *heads_tensor(PyObject *o) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    return t.is_cuda() && t.layout() == at::kStrided && t.has_storage() && !t.unsafeGetTensorImpl()->is_python_dispatch() && !t.is_neg() && t.dim() == 3 &&
                   t.stride(2) == 1 && t.numel() > 0
               ? &t
               : nullptr;
}
inline b200q_heads heads_of(const at::Tensor &t) { return {const_cast<void *>(t.const_data_ptr()), t.stride(0), t.stride(1)}; }
inline int layout_code(PyObject *o) { return is_text(o, "half") ? B200Q_ROTARY_HALF : is_text(o, "interleaved") ? B200Q_ROTARY_INTERLEAVED : -1; }
inline bool is_index(const at::Tensor *t) { return t && (t->scalar_type() == at::kLong || t->scalar_type() == at::kInt); }
inline bool is_table(const at::Tensor *t, int64_t dim) { return t && t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(1) % 2 == 0 && t->size(1) >= 2 && t->size(1) <= dim; }
// head_dim of a cache, or 0
inline int64_t cache_dim(const at::Tensor *t) {
    if (!t || t->scalar_type() != at::kByte || t->dim() != 4 || t->numel() == 0) return 0;
    const int64_t d = (t->size(3) - 128) / 32;
    return t->size(3) == 32 * d + 128 && (d == 64 || d == 96 || d == 128 || d == 192 || d == 256) ? d : 0;
}
// The new references of `first` and `second` as a pair, or what went wrong.
inline PyObject *pair_of(PyObject *first, PyObject *second) {
    PyObject *pair = first && second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return pair;
}

// rotary(q, k or None, positions, table, layout) -> (q', k')
PyObject *rotary(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    PLAIN_OR_NONE(n_args == 5 && lib.rotary != nullptr && !watched());
    const at::Tensor *q = heads_tensor(args[0]), *k = args[1] != Py_None ? heads_tensor(args[1]) : nullptr;
    const at::Tensor *positions = plain_tensor(args[2]), *table = plain_tensor(args[3]);
    PLAIN_OR_NONE(q && (k || args[1] == Py_None) && is_index(positions) && layout_code(args[4]) >= 0);
    const int64_t tokens = q->size(0), heads = q->size(1), dim = q->size(2), kv_heads = k ? k->size(1) : 0;
    const int type = float_code(q->scalar_type());
    Where w;
    PLAIN_OR_NONE(type >= 0 && is_table(table, dim) && positions->dim() == 1 && positions->size(0) == tokens && where_is(*q, w) && positions->get_device() == w.device &&
                  table->get_device() == w.device);
    PLAIN_OR_NONE(!k || (k->size(0) == tokens && k->size(2) == dim && k->scalar_type() == q->scalar_type() && k->get_device() == w.device));
    at::Tensor q_out = empty(q->sizes(), q->scalar_type(), w.device), k_out;
    if (k) k_out = empty(k->sizes(), q->scalar_type(), w.device);
    const b200q_heads qs = heads_of(*q), qo = heads_of(q_out), ks = k ? heads_of(*k) : b200q_heads{}, ko = k ? heads_of(k_out) : b200q_heads{};
    const void *at = positions->const_data_ptr();
    const float *angles = static_cast<const float *>(table->const_data_ptr());
    int status;
    WITHOUT_GIL(status, lib.rotary(&qs, k ? &ks : nullptr, &qo, k ? &ko : nullptr, at, angles, tokens, heads, kv_heads, dim, table->size(1), table->size(0), layout_code(args[4]), type,
                                   (int)positions->element_size(), w.stream));
    PLAIN_OR_NONE(status == B200Q_OK);
    PyObject *first = THPVariable_Wrap(std::move(q_out));
    return pair_of(first, k ? THPVariable_Wrap(std::move(k_out)) : Py_NewRef(Py_None));
    END_HANDLE_TH_ERRORS
}

// append(cache, k, v, slots, q or None, positions or None, table or None, layout) -> q', or True without q
PyObject *append(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    PLAIN_OR_NONE(n_args == 8 && lib.append != nullptr && !watched());
    const at::Tensor *cache = plain_tensor(args[0]), *k = heads_tensor(args[1]), *v = heads_tensor(args[2]), *slots = plain_tensor(args[3]);
    const int64_t dim = cache_dim(cache);
    PLAIN_OR_NONE(dim > 0 && k && v && is_index(slots) && layout_code(args[7]) >= 0);
    const int64_t tokens = k->size(0), kv_heads = cache->size(1);
    const int type = float_code(k->scalar_type());
    Where w;
    PLAIN_OR_NONE(type >= 0 && v->scalar_type() == k->scalar_type() && k->size(1) == kv_heads && k->size(2) == dim && v->sizes() == k->sizes() && slots->dim() == 1 &&
                  slots->size(0) == tokens && where_is(*k, w) && v->get_device() == w.device && cache->get_device() == w.device && slots->get_device() == w.device);
    const at::Tensor *q = nullptr, *positions = nullptr, *table = nullptr;
    PLAIN_OR_NONE((args[5] == Py_None) == (args[6] == Py_None) && (args[4] == Py_None || args[5] != Py_None));
    if (args[5] != Py_None) {
        positions = plain_tensor(args[5]);
        table = plain_tensor(args[6]);
        PLAIN_OR_NONE(is_index(positions) && is_table(table, dim) && table->size(1) % 16 == 0 && positions->dim() == 1 && positions->size(0) == tokens &&
                      positions->get_device() == w.device && table->get_device() == w.device);
    }
    at::Tensor q_out;
    b200q_heads qs = {}, qo = {};
    if (args[4] != Py_None) {
        q = heads_tensor(args[4]);
        PLAIN_OR_NONE(q && q->scalar_type() == k->scalar_type() && q->size(0) == tokens && q->size(2) == dim && q->get_device() == w.device);
        q_out = empty(q->sizes(), q->scalar_type(), w.device);
        qs = heads_of(*q);
        qo = heads_of(q_out);
    }
    const b200q_heads ks = heads_of(*k), vs = heads_of(*v);
    void *bytes = cache->data_ptr();
    const void *where = slots->const_data_ptr(), *at = positions ? positions->const_data_ptr() : nullptr;
    const float *angles = table ? static_cast<const float *>(table->const_data_ptr()) : nullptr;
    int status;
    WITHOUT_GIL(status, lib.append(bytes, cache->size(0), cache->size(2) * 16, &ks, &vs, q ? &qs : nullptr, q ? &qo : nullptr, where, at, angles, tokens, q ? q->size(1) : 0, kv_heads, dim,
                                   table ? table->size(1) : 0, table ? table->size(0) : 0, layout_code(args[7]), type, (int)slots->element_size(),
                                   positions ? (int)positions->element_size() : 0, w.stream));
    PLAIN_OR_NONE(status == B200Q_OK);
    if (!q) Py_RETURN_TRUE;
    return THPVariable_Wrap(std::move(q_out));
    END_HANDLE_TH_ERRORS
}

// read(cache, slots, dtype) -> (k, v)
PyObject *read(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    PLAIN_OR_NONE(n_args == 3 && lib.read != nullptr && !watched() && THPDtype_Check(args[2]));
    const at::Tensor *cache = plain_tensor(args[0]), *slots = plain_tensor(args[1]);
    const at::ScalarType dtype = reinterpret_cast<THPDtype *>(args[2])->scalar_type;
    const int64_t dim = cache_dim(cache);
    Where w;
    PLAIN_OR_NONE(dim > 0 && is_index(slots) && slots->numel() > 0 && float_code(dtype) >= 0 && where_is(*cache, w) && slots->get_device() == w.device);
    at::DimVector shape(slots->sizes());
    shape.push_back(cache->size(1));
    shape.push_back(dim);
    at::Tensor k = empty(shape, dtype, w.device), v = empty(shape, dtype, w.device);
    const void *bytes = cache->const_data_ptr(), *where = slots->const_data_ptr();
    void *kp = k.data_ptr(), *vp = v.data_ptr();
    int status;
    WITHOUT_GIL(status, lib.read(bytes, cache->size(0), cache->size(2) * 16, where, kp, vp, slots->numel(), cache->size(1), dim, float_code(dtype), (int)slots->element_size(), w.stream));
    PLAIN_OR_NONE(status == B200Q_OK);
    PyObject *first = THPVariable_Wrap(std::move(k));
    return pair_of(first, THPVariable_Wrap(std::move(v)));
    END_HANDLE_TH_ERRORS
}

// attention(q, cache, page_table, lengths, starts or None, mask or None, scale or None, return_lse) -> out or (out, lse)
PyObject *attention(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    PLAIN_OR_NONE(n_args == 8 && lib.attention != nullptr && !watched());
    const at::Tensor *q = plain_tensor(args[0]), *cache = plain_tensor(args[1]), *pages = plain_tensor(args[2]), *lengths = plain_tensor(args[3]);
    const int64_t dim = cache_dim(cache);
    PLAIN_OR_NONE(q && dim > 0 && pages && lengths && (q->dim() == 3 || q->dim() == 4) && q->numel() > 0 && q->size(-1) == dim);
    PLAIN_OR_NONE(q->scalar_type() == at::kHalf || q->scalar_type() == at::kBFloat16);
    PLAIN_OR_NONE(lengths->scalar_type() == at::kInt && lengths->dim() == 1 && pages->scalar_type() == at::kInt && pages->dim() == 2);
    const int64_t batch = lengths->size(0), heads = q->size(-2), kv_heads = cache->size(1), tokens = q->dim() == 3 ? q->size(0) : q->size(0) * q->size(1);
    Where w;
    PLAIN_OR_NONE(batch > 0 && pages->size(0) == batch && pages->size(1) > 0 && heads % kv_heads == 0 && where_is(*q, w) && cache->get_device() == w.device &&
                  pages->get_device() == w.device && lengths->get_device() == w.device && (reinterpret_cast<uintptr_t>(q->const_data_ptr()) & 15u) == 0);
    const at::Tensor *starts = nullptr, *mask = nullptr;
    if (args[4] != Py_None) {
        starts = plain_tensor(args[4]);
        PLAIN_OR_NONE(starts && q->dim() == 3 && starts->scalar_type() == at::kInt && starts->dim() == 1 && starts->size(0) == batch + 1 && starts->get_device() == w.device);
    } else {
        PLAIN_OR_NONE(q->size(0) == batch);
    }
    if (args[5] != Py_None) {
        mask = plain_tensor(args[5]);
        PLAIN_OR_NONE(mask && (mask->scalar_type() == at::kBool || mask->scalar_type() == at::kByte) && mask->dim() == 2 && mask->size(0) == tokens && mask->get_device() == w.device &&
                      (starts || mask->size(1) >= tokens / batch));
    }
    double scale = 1.0 / std::sqrt((double)dim);
    if (args[6] != Py_None) {
        PLAIN_OR_NONE(PyFloat_CheckExact(args[6]));
        scale = PyFloat_AS_DOUBLE(args[6]);
    }
    PLAIN_OR_NONE(PyBool_Check(args[7]));
    const bool with_lse = args[7] == Py_True;
    void *ws;
    size_t ws_bytes;
    PLAIN_OR_NONE(find_scratch(w, lib.attention_workspace_bytes(batch, tokens, heads, kv_heads, dim), ws, ws_bytes));
    at::Tensor out = empty(q->sizes(), q->scalar_type(), w.device), lse;
    if (with_lse) lse = empty(q->sizes().slice(0, q->dim() - 1), at::kFloat, w.device);
    const b200q_heads rows = {const_cast<void *>(q->const_data_ptr()), heads * dim, dim};
    void *dst = out.data_ptr();
    float *lse_dst = with_lse ? static_cast<float *>(lse.data_ptr()) : nullptr;
    const void *bytes = cache->const_data_ptr(), *seen = mask ? mask->const_data_ptr() : nullptr;
    const int32_t *table = static_cast<const int32_t *>(pages->const_data_ptr()), *n = static_cast<const int32_t *>(lengths->const_data_ptr());
    const int32_t *first_rows = starts ? static_cast<const int32_t *>(starts->const_data_ptr()) : nullptr;
    int status;
    WITHOUT_GIL(status, lib.attention(&rows, dst, lse_dst, bytes, cache->size(0), cache->size(2) * 16, table, pages->size(1), pages->size(1), n, first_rows, seen, mask ? mask->size(1) : 0,
                                      mask ? mask->size(1) : 0, batch, tokens, heads, kv_heads, dim, (float)scale, float_code(q->scalar_type()), ws, ws_bytes, w.stream));
    PLAIN_OR_NONE(status == B200Q_OK);
    PyObject *first = THPVariable_Wrap(std::move(out));
    if (!with_lse) return first;
    return pair_of(first, THPVariable_Wrap(std::move(lse)));
    END_HANDLE_TH_ERRORS
}

// log_probs(logits, tokens, top) -> (log_probs, entropy, top_log_probs, top_indices)
PyObject *log_probs(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    PLAIN_OR_NONE(n_args == 3 && lib.log_probs != nullptr && !watched() && PyLong_CheckExact(args[2]));
    const at::Tensor *logits = plain_tensor(args[0]), *tokens = plain_tensor(args[1]);
    PLAIN_OR_NONE(logits && is_index(tokens) && logits->dim() >= 1 && logits->numel() > 0 && tokens->numel() > 0);
    const int64_t lead = logits->dim() - 1, vocab = logits->size(-1), top = PyLong_AsLongLong(args[2]);
    PLAIN_OR_NONE(float_code(logits->scalar_type()) >= 0 && top >= 0 && top <= 32 && top <= vocab && (tokens->dim() == lead || tokens->dim() == lead + 1));
    for (int64_t d = 0; d < lead; ++d) PLAIN_OR_NONE(tokens->size(d) == logits->size(d));
    const int64_t rows = logits->numel() / vocab, given = tokens->dim() > lead ? tokens->size(-1) : 1;
    Where w;
    PLAIN_OR_NONE(where_is(*logits, w) && tokens->get_device() == w.device);
    const at::IntArrayRef shape = logits->sizes().slice(0, lead);
    at::DimVector top_shape(shape);
    top_shape.push_back(top);
    at::Tensor result[4] = {empty(tokens->sizes(), at::kFloat, w.device), empty(shape, at::kFloat, w.device), empty(top_shape, at::kFloat, w.device),
                            empty(top_shape, at::kLong, w.device)};
    float *lp = static_cast<float *>(result[0].data_ptr()), *entropy = static_cast<float *>(result[1].data_ptr()), *values = static_cast<float *>(result[2].data_ptr());
    int64_t *indices = static_cast<int64_t *>(result[3].data_ptr());
    const void *x = logits->const_data_ptr(), *which = tokens->const_data_ptr();
    int status;
    WITHOUT_GIL(status, lib.log_probs(x, vocab, which, lp, entropy, values, indices, rows, vocab, given, top, float_code(logits->scalar_type()), (int)tokens->element_size(), w.stream));
    PLAIN_OR_NONE(status == B200Q_OK);
    PyObject *all = PyTuple_New(4);
    for (int i = 0; all && i < 4; ++i) {
        PyObject *one = THPVariable_Wrap(std::move(result[i]));
        if (!one) {
            Py_CLEAR(all);
            break;
        }
        PyTuple_SET_ITEM(all, i, one);
    }
    return all;
    END_HANDLE_TH_ERRORS
}

// bind(an address for each member of Library, in their order)
PyObject *bind(PyObject *, PyObject *args) {
    static_assert(sizeof(Library) % sizeof(void *) == 0, "");
    constexpr Py_ssize_t N = sizeof(Library) / sizeof(void *);
    if (PyTuple_GET_SIZE(args) != N) return PyErr_Format(PyExc_TypeError, "bind takes %zd addresses", N);
    unsigned long long p[N];
    for (Py_ssize_t i = 0; i < N; ++i) {
        p[i] = PyLong_AsUnsignedLongLong(PyTuple_GET_ITEM(args, i));
        if (PyErr_Occurred()) return nullptr;
    }
    int i = 0;
    auto set = [&](auto &member) { member = reinterpret_cast<std::remove_reference_t<decltype(member)>>(p[i++]); };
    set(lib.quantize), set(lib.dequantize), set(lib.take), set(lib.workspace_bytes), set(lib.linear), set(lib.linear_fused), set(lib.w4_workspace_bytes), set(lib.w4);
    set(lib.rotary), set(lib.append), set(lib.read), set(lib.attention_workspace_bytes), set(lib.attention), set(lib.log_probs);
    Py_RETURN_NONE;
}

// set_scratch(device, stream, address, bytes): the buffer of that stream from now on; 0 bytes: it has none
PyObject *set_scratch(PyObject *, PyObject *args) {
    HANDLE_TH_ERRORS
    int device;
    unsigned long long stream, ptr, bytes;
    if (!PyArg_ParseTuple(args, "iKKK", &device, &stream, &ptr, &bytes)) return nullptr;
    const std::pair<uintptr_t, int> key((uintptr_t)stream, device);
    if (bytes == 0) scratch.erase(key);
    else scratch[key] = {reinterpret_cast<void *>((uintptr_t)ptr), (size_t)bytes};
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyObject *clear_scratch(PyObject *, PyObject *) {
    scratch.clear();
    Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(linear),
                         FAST(quantize),
                         FAST(dequantize),
                         FAST(take),
                         FAST(w4),
                         FAST(rotary),
                         FAST(append),
                         FAST(read),
                         FAST(attention),
                         FAST(log_probs),
                         {"bind", bind, METH_VARARGS, nullptr},
                         {"set_scratch", set_scratch, METH_VARARGS, nullptr},
                         {"clear_scratch", clear_scratch, METH_NOARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "hidet_b200_host", "the host side of one call, natively", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_hidet_b200_host() { return PyModule_Create(&module); }
