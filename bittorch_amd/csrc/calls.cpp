// Host side of the calls whose kernels take a few microseconds: what the functions of _C.py do for an ordinary call (plain GPU
// tensors as the library reads them, on the current device), in one native call.  In Python the checks, the allocations, the
// workspace query and some twenty argument conversions were most of such a call's time: one fp16 row through 4096 x 4096 took
// 13.6 us a call around a kernel of 4.6.
//
// Every function returns None for a call that is not ordinary: another dtype, device, stride or alignment, a subclass, a mode, a
// transform or a trace being active, or an argument that the Python function refuses.  _C.py then goes on as if it had not asked,
// with its copies, its conversions and its messages.  Nothing is kept from one call for the next.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/autocast_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <string>
#include <type_traits>

#include "../../include/bittorch_hip.h"

namespace {

// The library as _lib.py has loaded it: bind() gives the addresses.
#define BT_FUNCTIONS(X)                                                                                                       \
    X(bt_last_error) X(bt_tiled_weights_bytes) X(bt_tiled_forward_workspace_bytes) X(bt_packed_forward_workspace_bytes)        \
    X(bt_packed_forward_fused_workspace_bytes) X(bt_tensor_core_workspace_bytes) X(bt_linear_grad_weight_workspace_bytes)      \
    X(bt_linear_grad_weight_16_workspace_bytes) X(bt_ternary_linear_tiled_forward) X(bt_ternary_linear_packed_forward)         \
    X(bt_ternary_linear_tensor_core_forward) X(bt_quantize_pack) X(bt_ternary_linear_grad_input) X(bt_linear_grad_weight)      \
    X(bt_linear_grad_weight_16) X(bt_unpack_dequant) X(bt_swiglu) X(bt_rmsnorm) X(bt_ternary_gemm_i8_tiled) \
    X(bt_ternary_swiglu_i8_tiled) X(bt_act_quant_i8_layout) X(bt_add_rmsnorm) X(bt_add_rmsnorm_backward)                       \
    X(bt_add_rmsnorm_backward_workspace_bytes) X(bt_gated_quantize) X(bt_gated_quantize_workspace_bytes) X(bt_gated_split)     \
    X(bt_gated_split_bytes) X(bt_gated_grad_input) X(bt_gated_grad_input_workspace_bytes)                                      \
    X(bt_ternary_gated_forward) X(bt_gated_grad) X(bt_gated_grad_masters) X(bt_gated_grad_workspace_bytes)                     \
    X(bt_gated_masters_serves) X(bt_gated_masters_forward) X(bt_rotary) X(bt_cache_head_dim) X(bt_cache_append)                  \
    X(bt_cached_attention_workspace_bytes) X(bt_cached_attention)
struct Library {
#define X(name) decltype(&::name) name = nullptr;
    BT_FUNCTIONS(X)
#undef X
} lib;
bool bound = false;

int tag(at::ScalarType t) {
    return t == at::kFloat ? BT_F32 : t == at::kHalf ? BT_F16 : t == at::kBFloat16 ? BT_BF16 : -1;
}

// No mode, transform or trace that would see, or stand in for, the tensor operations of the Python function.
bool undisturbed() {
    using c10::DispatchKey;
    return bound && at::impl::PythonTorchFunctionTLS::stack_len() == 0 && !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
           !c10::impl::tls_is_dispatch_key_included(DispatchKey::FuncTorchDynamicLayerFrontMode) &&
           !c10::impl::tls_is_dispatch_key_included(DispatchKey::Tracer) &&
           !c10::impl::tls_is_dispatch_key_included(DispatchKey::Functionalize) &&
           !c10::impl::tls_is_dispatch_key_included(DispatchKey::PythonDispatcher);
}

// A tensor of this very class with values of its own on the current device, or null; plain: in contiguous memory.
const at::Tensor* on_device(PyObject* o, int device) {
    using c10::DispatchKey;
    static const c10::DispatchKeySet special({DispatchKey::Python, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
                                              DispatchKey::Batched, DispatchKey::Functionalize, DispatchKey::Conjugate,
                                              DispatchKey::Negative, DispatchKey::ZeroTensor});
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has_any(special) && t.get_device() == device && t.numel() > 0
               ? &t : nullptr;
}
const at::Tensor* plain(PyObject* o, int device) {
    const at::Tensor* t = on_device(o, device);
    return t && t->is_contiguous() ? t : nullptr;
}
bool aligned(const at::Tensor& t, uintptr_t to) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % to == 0; }

// A scale or bias vector of n entries (or one), fp32 or 16-bit.
const at::Tensor* vec(PyObject* o, int64_t n, bool one_entry, int device) {
    const at::Tensor* t = plain(o, device);
    return t && t->dim() == 1 && (t->size(0) == n || (one_entry && t->size(0) == 1)) && tag(t->scalar_type()) >= 0 ? t : nullptr;
}

at::Tensor output(at::IntArrayRef shape, at::ScalarType dtype, const at::Tensor& like) {
    return at::empty(shape, at::TensorOptions().dtype(dtype).device(like.device()));
}
struct Scratch {  // of one call
    at::Tensor t;
    Scratch(size_t bytes, const at::Tensor& like) {
        if (bytes) t = output({(int64_t)bytes}, at::kByte, like);
    }
    void* ptr() const { return t.defined() ? t.data_ptr() : nullptr; }
    size_t size() const { return t.defined() ? (size_t)t.numel() : 0; }
};
void* stream_of(int device) { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }

struct Unlocked {  // the interpreter, until the end of the block however it is left
    PyThreadState* const state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};
// The library's call without the interpreter lock, as through ctypes.  Its arguments are values: what they are read from (tensors, whose
// accessors may throw and which other threads may point elsewhere) is asked under the lock.
void check_status(int rc) {
    if (rc != 0) {
        const char* text = lib.bt_last_error();
        TORCH_CHECK_WITH(Error, false, text && text[0] ? std::string(text) : "libbittorch_hip call failed (" + std::to_string(rc) + ")");
    }
}
template <typename... P>
void call(int (*f)(P...), std::common_type_t<P>... args) {
    int rc;
    {
        const Unlocked unlocked;
        rc = f(args...);
    }
    check_status(rc);
}

bool as_int(PyObject* o, int64_t* v) {
    if (!PyLong_CheckExact(o)) return false;
    *v = PyLong_AsLongLong(o);
    if (*v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
bool as_float(PyObject* o, double* v) {
    if (PyFloat_CheckExact(o)) *v = PyFloat_AS_DOUBLE(o);
    else {
        int64_t i;
        if (!as_int(o, &i)) return false;
        *v = (double)i;
    }
    return true;
}
bool as_bool(PyObject* o, bool* v) {
    *v = o == Py_True;
    return o == Py_True || o == Py_False;
}

// The current device, if the first argument is a GPU tensor and nothing stands in between.
bool here(PyObject* o, int* device) {
    if (!undisturbed() || !THPVariable_CheckExact(o) || !THPVariable_Unpack(o).is_cuda()) return false;
    *device = (int)c10::hip::current_device();
    return true;
}
// X as the first argument: rows of values of a float type.
const at::Tensor* rows_of(PyObject* o, int* device) {
    if (!here(o, device)) return nullptr;
    const at::Tensor* x = plain(o, *device);
    return x && x->dim() >= 1 && tag(x->scalar_type()) >= 0 ? x : nullptr;
}
// A residual of the output's shape and dtype.
const at::Tensor* residual_of(PyObject* o, const at::Tensor& x, int64_t n, int device) {
    const at::Tensor* r = plain(o, device);
    if (!r || r->scalar_type() != x.scalar_type() || r->dim() != x.dim() || r->size(-1) != n || !aligned(*r, 16)) return nullptr;
    for (int64_t d = 0; d + 1 < x.dim(); d++)
        if (r->size(d) != x.size(d)) return nullptr;
    return r;
}
at::DimVector with_last(const at::Tensor& x, int64_t n) {
    at::DimVector shape(x.sizes());
    shape.back() = n;
    return shape;
}
#define ORDINARY(cond) \
    if (!(cond)) Py_RETURN_NONE

// tiled_forward(X, W_tiled, scale, bias, in_features, out_features, residual, norm, swiglu_up, swiglu_pairs, natural_from_pairs)
PyObject* tiled_forward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    int64_t K, N;
    bool pairs, natural;
    ORDINARY(n_args == 11);
    const at::Tensor* x = rows_of(a[0], &device);
    ORDINARY(x && as_int(a[4], &K) && as_int(a[5], &N) && as_bool(a[9], &pairs) && as_bool(a[10], &natural));
    ORDINARY(K > 0 && N > 0 && x->size(-1) == K && !(pairs && natural) && (!(pairs || natural) || N % 32 == 0));
    const at::Tensor *w = plain(a[1], device), *scale = vec(a[2], N, true, device);
    ORDINARY(w && scale && w->scalar_type() == at::kByte && w->dim() == 1 && (size_t)w->numel() == lib.bt_tiled_weights_bytes(N, K));
    const at::Tensor *bias = nullptr, *res = nullptr, *pro = nullptr;
    if (a[3] != Py_None) ORDINARY((bias = vec(a[3], N, false, device)));
    if (a[6] != Py_None) ORDINARY(!pairs && (res = residual_of(a[6], *x, N, device)));
    int op = 0;
    double eps = 0.0;
    if (a[7] != Py_None) {
        ORDINARY(a[8] == Py_None && PyTuple_CheckExact(a[7]) && PyTuple_GET_SIZE(a[7]) == 2 && as_float(PyTuple_GET_ITEM(a[7], 1), &eps));
        PyObject* weight = PyTuple_GET_ITEM(a[7], 0);
        op = 1;
        if (weight != Py_None) {
            pro = plain(weight, device);
            ORDINARY(pro && pro->dim() == 1 && pro->size(0) == K && pro->scalar_type() == x->scalar_type());
        }
    } else if (a[8] != Py_None) {
        pro = plain(a[8], device);
        ORDINARY(!pairs && pro && pro->sizes() == x->sizes() && pro->scalar_type() == x->scalar_type());
        op = 2;
    }
    const int dt = tag(x->scalar_type()), epi = pairs ? 1 : natural ? 2 : 0;
    const int64_t B = x->numel() / K, Ny = pairs ? N / 2 : N;
    at::Tensor y = output(with_last(*x, Ny), x->scalar_type(), *x);
    const Scratch ws(op == 0 && !pairs ? lib.bt_tiled_forward_workspace_bytes(B, N, K, dt) : lib.bt_packed_forward_fused_workspace_bytes(B, N, K, dt), *x);
    void* st = stream_of(device);
    call(lib.bt_ternary_linear_tiled_forward, x->const_data_ptr(), K, dt, op, pro ? pro->const_data_ptr() : nullptr,
        op == 2 ? K : 0, (float)eps, (const uint8_t*)w->const_data_ptr(), scale->const_data_ptr(), tag(scale->scalar_type()),
        scale->numel(), bias ? bias->const_data_ptr() : nullptr, bias ? tag(bias->scalar_type()) : 0,
        res ? res->const_data_ptr() : nullptr, epi, y.data_ptr(), B, N, K, ws.ptr(), ws.size(), st);
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// W_T [ceil(K / 4), N]
const at::Tensor* packed_weights(PyObject* o, int64_t K, int device) {
    const at::Tensor* w = plain(o, device);
    return w && w->scalar_type() == at::kByte && w->dim() == 2 && w->size(0) == (K + 3) / 4 ? w : nullptr;
}

// packed_forward(X, W_T, scale, bias, in_features)
PyObject* packed_forward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    int64_t K;
    ORDINARY(n_args == 5);
    const at::Tensor* x = rows_of(a[0], &device);
    ORDINARY(x && as_int(a[4], &K) && K > 0 && x->size(-1) == K);
    const at::Tensor* w = packed_weights(a[1], K, device);
    ORDINARY(w);
    const int64_t N = w->size(1), B = x->numel() / K;
    const at::Tensor *scale = vec(a[2], N, true, device), *bias = nullptr;
    ORDINARY(scale);
    if (a[3] != Py_None) ORDINARY((bias = vec(a[3], N, false, device)));
    const int dt = tag(x->scalar_type());
    at::Tensor y = output(with_last(*x, N), x->scalar_type(), *x);
    const Scratch ws(lib.bt_packed_forward_workspace_bytes(B, N, K, dt), *x);
    void* st = stream_of(device);
    call(lib.bt_ternary_linear_packed_forward, x->const_data_ptr(), dt, (const uint8_t*)w->const_data_ptr(),
        scale->const_data_ptr(), tag(scale->scalar_type()), scale->numel(), bias ? bias->const_data_ptr() : nullptr,
        bias ? tag(bias->scalar_type()) : 0, y.data_ptr(), B, N, K, ws.ptr(), ws.size(), st);
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// tensor_core_forward(X, W_T, scale, bias, in_features): version 2
PyObject* tensor_core_forward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    int64_t K;
    ORDINARY(n_args == 5);
    const at::Tensor* x = rows_of(a[0], &device);
    ORDINARY(x && x->dim() == 2 && as_int(a[4], &K) && K > 0 && x->size(1) == K);
    const at::Tensor* w = packed_weights(a[1], K, device);
    ORDINARY(w);
    const int64_t N = w->size(1), B = x->size(0);
    const at::Tensor *scale = vec(a[2], N, true, device), *bias = nullptr;
    ORDINARY(scale);
    if (a[3] != Py_None) ORDINARY((bias = vec(a[3], N, false, device)));
    at::Tensor y = output({B, N}, x->scalar_type(), *x);
    const Scratch ws(lib.bt_tensor_core_workspace_bytes(B, N, K), *x);
    void* st = stream_of(device);
    call(lib.bt_ternary_linear_tensor_core_forward, x->const_data_ptr(), tag(x->scalar_type()), (const uint8_t*)w->const_data_ptr(),
        scale->const_data_ptr(), tag(scale->scalar_type()), scale->numel(), bias ? bias->const_data_ptr() : nullptr,
        bias ? tag(bias->scalar_type()) : 0, y.data_ptr(), B, N, K, ws.ptr(), ws.size(), st);
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// quantize_pack(weight, threshold_factor, per_channel, as_half) -> (packed, scale, None)
PyObject* quantize_pack(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    double threshold;
    bool per_channel, as_half;
    ORDINARY(n_args == 4);
    const at::Tensor* w = rows_of(a[0], &device);
    ORDINARY(w && w->dim() == 2 && as_float(a[1], &threshold) && as_bool(a[2], &per_channel) && as_bool(a[3], &as_half));
    ORDINARY(!as_half || w->scalar_type() == at::kFloat);
    const int64_t N = w->size(0), K = w->size(1);
    at::Tensor packed = output({(K + 3) / 4, N}, at::kByte, *w), scale = output({per_channel ? N : 1}, at::kFloat, *w);
    void* st = stream_of(device);
    constexpr int kF32AsF16 = 4;
    call(lib.bt_quantize_pack, w->const_data_ptr(), as_half ? kF32AsF16 : tag(w->scalar_type()), N, K, threshold,
        per_channel ? 1 : 0, (uint8_t*)packed.data_ptr(), (float*)scale.data_ptr(), nullptr, st);
    const at::ScalarType dtype = as_half ? at::kHalf : w->scalar_type();
    if (dtype != at::kFloat) scale = scale.to(dtype);
    if (!per_channel) scale = scale.squeeze(0);
    PyObject* out = PyTuple_New(3);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(packed)));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(scale)));
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(out, 2, Py_None);
    return out;
    END_HANDLE_TH_ERRORS
}

// grad_input(dY, W_T, scale, in_features): fp32
PyObject* grad_input(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    int64_t K;
    ORDINARY(n_args == 4);
    const at::Tensor* dy = rows_of(a[0], &device);
    ORDINARY(dy && dy->dim() == 2 && dy->scalar_type() == at::kFloat && as_int(a[3], &K) && K > 0);
    const at::Tensor *w = packed_weights(a[1], K, device), *scale = plain(a[2], device);
    const int64_t M = dy->size(0), N = dy->size(1);
    ORDINARY(w && w->size(1) == N && scale && scale->scalar_type() == at::kFloat && (scale->numel() == N || scale->numel() == 1));
    at::Tensor out = output({M, K}, at::kFloat, *dy);
    void* st = stream_of(device);
    call(lib.bt_ternary_linear_grad_input, (const float*)dy->const_data_ptr(), (const uint8_t*)w->const_data_ptr(),
        (const float*)scale->const_data_ptr(), scale->numel(), (float*)out.data_ptr(), M, N, K, st);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// grad_weight(dY, X, scale, want_bias) -> (dW, dBias or None): fp32
PyObject* grad_weight(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    bool want_bias;
    ORDINARY(n_args == 4);
    const at::Tensor* dy = rows_of(a[0], &device);
    ORDINARY(dy && dy->dim() == 2 && dy->scalar_type() == at::kFloat && as_bool(a[3], &want_bias));
    const at::Tensor *x = plain(a[1], device), *scale = plain(a[2], device);
    ORDINARY(x && x->dim() == 2 && x->scalar_type() == at::kFloat && x->size(0) == dy->size(0) && scale && scale->scalar_type() == at::kFloat);
    const int64_t M = dy->size(0), N = dy->size(1), K = x->size(1);
    ORDINARY(scale->numel() == N || scale->numel() == 1);
    at::Tensor dw = output({N, K}, at::kFloat, *dy), db;
    if (want_bias) db = output({N}, at::kFloat, *dy);
    const Scratch ws(lib.bt_linear_grad_weight_workspace_bytes(M, N, K), *dy);
    void* st = stream_of(device);
    call(lib.bt_linear_grad_weight, (const float*)dy->const_data_ptr(), (const float*)x->const_data_ptr(),
        (const float*)scale->const_data_ptr(), scale->numel(), (float*)dw.data_ptr(), want_bias ? (float*)db.data_ptr() : nullptr,
        M, N, K, ws.ptr(), ws.size(), st);
    PyObject* out = PyTuple_New(2);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(dw)));
    if (want_bias) {
        PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(db)));
    } else {
        Py_INCREF(Py_None);
        PyTuple_SET_ITEM(out, 1, Py_None);
    }
    return out;
    END_HANDLE_TH_ERRORS
}

// int8 rows quantized by row_op, times a tiled copy:
// gemm_i8_tiled(Q [B, K], s_x, W_tiled, scale, bias, in_features, out_features, like (its dtype), residual [B, N], q_operand_order)
PyObject* gemm_i8_tiled(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    int64_t K, N;
    bool oo;
    ORDINARY(n_args == 10 && here(a[0], &device) && as_int(a[5], &K) && as_int(a[6], &N) && as_bool(a[9], &oo) && K > 0 && N > 0);
    const at::Tensor *q = plain(a[0], device), *sx = plain(a[1], device), *w = plain(a[2], device), *scale = vec(a[3], N, true, device);
    ORDINARY(q && q->scalar_type() == at::kChar && q->dim() == 2 && q->size(1) == K && sx && sx->scalar_type() == at::kFloat &&
             sx->numel() == q->size(0) && scale);
    ORDINARY(w && w->scalar_type() == at::kByte && w->dim() == 1 && (size_t)w->numel() == lib.bt_tiled_weights_bytes(N, K));
    ORDINARY(THPDtype_Check(a[7]));
    const at::ScalarType dtype = reinterpret_cast<THPDtype*>(a[7])->scalar_type;
    ORDINARY(tag(dtype) >= 0);
    const int64_t B = q->size(0);
    const at::Tensor *bias = nullptr, *res = nullptr;
    if (a[4] != Py_None) ORDINARY((bias = vec(a[4], N, false, device)));
    if (a[8] != Py_None) {
        res = plain(a[8], device);
        ORDINARY(res && res->scalar_type() == dtype && res->dim() == 2 && res->size(0) == B && res->size(1) == N && aligned(*res, 16));
    }
    at::Tensor y = output({B, N}, dtype, *q);
    void* st = stream_of(device);
    call(lib.bt_ternary_gemm_i8_tiled, (const int8_t*)q->const_data_ptr(), oo ? 1 : 0, (const float*)sx->const_data_ptr(),
        (const uint8_t*)w->const_data_ptr(), scale->const_data_ptr(), tag(scale->scalar_type()), scale->numel(),
        bias ? bias->const_data_ptr() : nullptr, bias ? tag(bias->scalar_type()) : 0, res ? res->const_data_ptr() : nullptr,
        y.data_ptr(), tag(dtype), nullptr, B, N, K, st);
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// swiglu_i8_tiled(Q [B, K] in operand order, s_x, W_tiled, scale, bias, in_features, out_features, dtype) -> [B, N / 2]
PyObject* swiglu_i8_tiled(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    int64_t K, N;
    ORDINARY(n_args == 8 && here(a[0], &device) && as_int(a[5], &K) && as_int(a[6], &N) && K > 0 && N > 0 && N % 32 == 0);
    const at::Tensor *q = plain(a[0], device), *sx = plain(a[1], device), *w = plain(a[2], device), *scale = vec(a[3], N, true, device);
    ORDINARY(q && q->scalar_type() == at::kChar && q->dim() == 2 && q->size(1) == K && sx && sx->scalar_type() == at::kFloat &&
             sx->numel() == q->size(0) && scale);
    ORDINARY(w && w->scalar_type() == at::kByte && w->dim() == 1 && (size_t)w->numel() == lib.bt_tiled_weights_bytes(N, K));
    ORDINARY(THPDtype_Check(a[7]));
    const at::ScalarType dtype = reinterpret_cast<THPDtype*>(a[7])->scalar_type;
    ORDINARY(dtype == at::kHalf || dtype == at::kBFloat16);
    const int64_t B = q->size(0);
    const at::Tensor* bias = nullptr;
    if (a[4] != Py_None) ORDINARY((bias = vec(a[4], N, false, device)));
    at::Tensor h = output({B, N / 2}, dtype, *q);
    void* st = stream_of(device);
    call(lib.bt_ternary_swiglu_i8_tiled, (const int8_t*)q->const_data_ptr(), (const float*)sx->const_data_ptr(),
        (const uint8_t*)w->const_data_ptr(), scale->const_data_ptr(), tag(scale->scalar_type()), scale->numel(),
        bias ? bias->const_data_ptr() : nullptr, bias ? tag(bias->scalar_type()) : 0, h.data_ptr(), tag(dtype), B, N, K, st);
    return THPVariable_Wrap(std::move(h));
    END_HANDLE_TH_ERRORS
}

// grad_weight_16(dY, X, scale, out_dtype)
PyObject* grad_weight_16(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    ORDINARY(n_args == 4);
    const at::Tensor* dy = rows_of(a[0], &device);
    ORDINARY(dy && dy->dim() == 2 && dy->scalar_type() != at::kFloat && THPDtype_Check(a[3]));
    const at::ScalarType dtype = reinterpret_cast<THPDtype*>(a[3])->scalar_type;
    const at::Tensor *x = plain(a[1], device), *scale = plain(a[2], device);
    ORDINARY(x && x->dim() == 2 && x->scalar_type() == dy->scalar_type() && x->size(0) == dy->size(0) && scale && tag(scale->scalar_type()) >= 0);
    const int64_t M = dy->size(0), N = dy->size(1), K = x->size(1);
    ORDINARY((dtype == dy->scalar_type() || dtype == at::kFloat) && (scale->numel() == N || scale->numel() == 1));
    at::Tensor out = output({N, K}, dtype, *dy);
    const Scratch ws(lib.bt_linear_grad_weight_16_workspace_bytes(M, N, K), *dy);
    void* st = stream_of(device);
    call(lib.bt_linear_grad_weight_16, dy->const_data_ptr(), x->const_data_ptr(), tag(dy->scalar_type()), scale->const_data_ptr(),
        tag(scale->scalar_type()), scale->numel(), out.data_ptr(), tag(dtype), M, N, K, ws.ptr(), ws.size(), st);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// A matrix whose rows lie any distance apart, their elements side by side.
const at::Tensor* strided_rows(PyObject* o, int device) {
    const at::Tensor* t = on_device(o, device);
    return t && t->dim() == 2 && t->stride(1) == 1 && t->stride(0) >= t->size(1) ? t : nullptr;
}
PyObject* int8_rows(at::Tensor q, at::Tensor s) {
    PyObject* out = PyTuple_New(2);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(q)));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(s)));
    return out;
}

// act_quant_int8(x [B, K], operand_order) -> (Q, s_x)
PyObject* act_quant_int8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    bool oo;
    ORDINARY(n_args == 2);
    const at::Tensor* x = rows_of(a[0], &device);
    ORDINARY(x && x->dim() == 2 && as_bool(a[1], &oo));
    const int64_t B = x->size(0), K = x->size(1);
    at::Tensor q = output({B, K}, at::kChar, *x), s = output({B}, at::kFloat, *x);
    void* st = stream_of(device);
    call(lib.bt_act_quant_i8_layout, x->const_data_ptr(), tag(x->scalar_type()), B, K, (int8_t*)q.data_ptr(), (float*)s.data_ptr(),
        oo ? 1 : 0, st);
    return int8_rows(std::move(q), std::move(s));
    END_HANDLE_TH_ERRORS
}

// rmsnorm_int8(x [B, K], weight, eps, operand_order) -> (Q, s_x)
PyObject* rmsnorm_int8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    double eps;
    bool oo;
    ORDINARY(n_args == 4);
    const at::Tensor* x = rows_of(a[0], &device);
    ORDINARY(x && x->dim() == 2 && as_float(a[2], &eps) && as_bool(a[3], &oo));
    const int64_t B = x->size(0), K = x->size(1);
    const at::Tensor* w = nullptr;
    if (a[1] != Py_None) {
        w = plain(a[1], device);
        ORDINARY(w && w->dim() == 1 && w->size(0) == K && w->scalar_type() == x->scalar_type());
    }
    at::Tensor q = output({B, K}, at::kChar, *x), s = output({B}, at::kFloat, *x);
    void* st = stream_of(device);
    call(lib.bt_rmsnorm, x->const_data_ptr(), K, w ? w->const_data_ptr() : nullptr, (float)eps, tag(x->scalar_type()), B, K,
        nullptr, (int8_t*)q.data_ptr(), (float*)s.data_ptr(), oo ? 1 : 0, st);
    return int8_rows(std::move(q), std::move(s));
    END_HANDLE_TH_ERRORS
}

// swiglu_int8(gate [B, K], up [B, K], operand_order) -> (Q, s_x)
PyObject* swiglu_int8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    bool oo;
    ORDINARY(n_args == 3 && here(a[0], &device) && as_bool(a[2], &oo));
    const at::Tensor *g = strided_rows(a[0], device), *u = strided_rows(a[1], device);
    ORDINARY(g && u && tag(g->scalar_type()) >= 0 && u->scalar_type() == g->scalar_type() && u->sizes() == g->sizes());
    const int64_t B = g->size(0), K = g->size(1);
    at::Tensor q = output({B, K}, at::kChar, *g), s = output({B}, at::kFloat, *g);
    void* st = stream_of(device);
    call(lib.bt_swiglu, g->const_data_ptr(), g->stride(0), u->const_data_ptr(), u->stride(0), tag(g->scalar_type()), B, K, nullptr,
        (int8_t*)q.data_ptr(), (float*)s.data_ptr(), oo ? 1 : 0, st);
    return int8_rows(std::move(q), std::move(s));
    END_HANDLE_TH_ERRORS
}

// unpack_dequant(W_T, in_features, scale, out_dtype): dense [N, K] of a float type
PyObject* unpack_dequant(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    int64_t K;
    ORDINARY(n_args == 4 && here(a[0], &device) && as_int(a[1], &K) && K > 0 && THPDtype_Check(a[3]));
    const at::ScalarType dtype = reinterpret_cast<THPDtype*>(a[3])->scalar_type;
    const at::Tensor *w = packed_weights(a[0], K, device), *scale = plain(a[2], device);
    ORDINARY(tag(dtype) >= 0 && w && scale && tag(scale->scalar_type()) >= 0 && (scale->numel() == w->size(1) || scale->numel() == 1));
    const at::Tensor scale_f = scale->scalar_type() == at::kFloat ? *scale : scale->detach().to(at::kFloat);
    at::Tensor out = output({w->size(1), K}, dtype, *w);
    void* st = stream_of(device);
    call(lib.bt_unpack_dequant, (const uint8_t*)w->const_data_ptr(), (const float*)scale_f.const_data_ptr(), scale_f.numel(),
        out.data_ptr(), tag(dtype), w->size(1), K, st);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---- calls that are differentiated: the autograd functions of ops/fused.py and ops/gated.py -----------------------------------
// A training call of a small layer spends more time in those two Python functions than on the GPU (the norm of 777 x 1001 and its gradient:
// 146 us a step, of kernels that take 15).  Backward passes run on autograd's own threads, which do not hold the interpreter lock.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<at::Tensor>;

const void* data_of(const MaybeTensor& t) { return t ? t->const_data_ptr() : nullptr; }
int tag_of(const MaybeTensor& t) { return t ? tag(t->scalar_type()) : 0; }
MaybeTensor maybe(const at::Tensor* t) { return t ? MaybeTensor(*t) : std::nullopt; }

// A gradient for each argument of a forward, and whether it is wanted: autograd asks by the number of a tensor argument that there was.
struct Wanted {
    variable_list grads;
    std::vector<bool> want;
    Wanted(AutogradContext* ctx, size_t args, std::initializer_list<bool> there) : grads(args), want(there.size()) {
        size_t edge = 0, i = 0;
        for (bool t : there) want[i++] = t && ctx->needs_input_grad(edge++);
    }
};
// What the gradients are where a graph of the backward pass is kept (`graph`): values whose own gradient is an error.
variable_list once(const char* name, bool graph, variable_list grads, const variable_list& incoming) {
    bool depends = false;
    for (const at::Tensor& t : incoming) depends = depends || (t.defined() && t.requires_grad());
    if (!graph || !depends) return grads;
    const at::AutoGradMode on(true);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string("trying to differentiate twice a function that was marked with @once_differentiable (") + name + ")", (int64_t)grads.size());
    variable_list out(grads.size()), some;
    std::vector<size_t> at;
    for (size_t i = 0; i < grads.size(); i++)
        if (grads[i].defined()) {
            some.push_back(grads[i].detach().requires_grad_());
            at.push_back(i);
        }
    some = (*error)(std::move(some));
    for (size_t i = 0; i < at.size(); i++) out[at[i]] = some[i];
    return out;
}

struct NormFlags {
    double eps;
    bool store, quantize, operand_order, rowsum;
};
struct NormOut {
    at::Tensor s, y, q, s_x, rowsum, rstd;
};
NormOut add_norm_run(const at::Tensor& x, const MaybeTensor& residual, const MaybeTensor& weight, const NormFlags& f, bool want_rstd) {
    const int64_t K = x.size(-1), B = x.numel() / K;
    const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
    NormOut o;
    if (residual) o.s = output(x.sizes(), residual->scalar_type(), x);
    if (f.store) o.y = output(x.sizes(), x.scalar_type(), x);
    if (f.quantize) {
        o.q = output(x.sizes(), at::kChar, x);
        o.s_x = output(lead, at::kFloat, x);
    }
    if (f.rowsum) o.rowsum = output(lead, at::kInt, x);
    if (want_rstd) o.rstd = output({B}, at::kFloat, x);
    auto ptr = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    void* st = stream_of(x.get_device());
    call(lib.bt_add_rmsnorm, x.const_data_ptr(), K, tag(x.scalar_type()), data_of(residual), residual ? K : 0, tag_of(residual), data_of(weight),
         tag_of(weight), (float)f.eps, B, K, ptr(o.s), ptr(o.y), (float*)ptr(o.rstd), (int8_t*)ptr(o.q), (float*)ptr(o.s_x), (int32_t*)ptr(o.rowsum),
         f.operand_order ? 1 : 0, st);
    return o;
}

struct AddRMSNorm : torch::autograd::Function<AddRMSNorm> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const MaybeTensor& residual, const MaybeTensor& weight, double eps,
                                 bool store, bool quantize, bool operand_order, bool rowsum) {
        NormOut o = add_norm_run(x, residual, weight, {eps, store, quantize, operand_order, rowsum}, true);
        ctx->set_materialize_grads(false);
        variable_list out, none;
        for (at::Tensor* t : {&o.s, &o.y, &o.q, &o.s_x, &o.rowsum})
            if (t->defined()) {
                out.push_back(*t);
                if (t != &o.s && t != &o.y) none.push_back(*t);
            }
        ctx->mark_non_differentiable(none);
        ctx->save_for_backward({residual ? o.s : x, o.rstd, weight ? *weight : at::Tensor()});
        ctx->saved_data["residual"] = residual.has_value();
        ctx->saved_data["store"] = store;
        ctx->saved_data["dtype"] = x.scalar_type();
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list incoming) {
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &s = saved[0], &rstd = saved[1], &weight = saved[2];
        const bool has_residual = ctx->saved_data["residual"].toBool(), stored = ctx->saved_data["store"].toBool();
        const at::ScalarType x_dtype = ctx->saved_data["dtype"].toScalarType();
        Wanted w(ctx, 8, {true, has_residual, weight.defined()});
        const bool want_x = w.want[0], want_r = w.want[1], want_w = w.want[2];
        const at::Tensor d_sum = has_residual ? incoming[0] : at::Tensor(), d_norm = stored ? incoming[has_residual ? 1 : 0] : at::Tensor();
        const bool graph = at::GradMode::is_enabled();
        const at::NoGradGuard no_grad;
        const c10::DeviceGuard guard(s.device());
        if (!d_norm.defined()) {  // the norm was not used
            if (d_sum.defined()) {
                if (want_x) w.grads[0] = d_sum.to(x_dtype);
                if (want_r) w.grads[1] = d_sum;
            }
            if (want_w) w.grads[2] = at::zeros_like(weight);
        } else {
            const int64_t K = s.size(-1), B = s.numel() / K;
            const at::Tensor dy = d_norm.contiguous(), ds = d_sum.defined() ? d_sum.contiguous() : d_sum;
            const bool one = x_dtype == s.scalar_type();
            at::Tensor dx, dr, dw;
            if (want_r || (one && want_x)) dr = output(s.sizes(), s.scalar_type(), s);
            if (want_x && !one) dx = output(s.sizes(), x_dtype, s);
            if (want_w) dw = output({K}, weight.scalar_type(), s);
            const Scratch ws(want_w ? lib.bt_add_rmsnorm_backward_workspace_bytes(B, K) : 0, s);
            auto ptr = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
            check_status(lib.bt_add_rmsnorm_backward(
                s.const_data_ptr(), tag(s.scalar_type()), (const float*)rstd.const_data_ptr(), weight.defined() ? weight.const_data_ptr() : nullptr,
                weight.defined() ? tag(weight.scalar_type()) : 0, dy.const_data_ptr(), tag(x_dtype), ds.defined() ? ds.const_data_ptr() : nullptr, B, K,
                ptr(dx), ptr(dr), ptr(dw), ws.ptr(), ws.size(), stream_of(s.get_device())));
            if (want_x) w.grads[0] = one ? dr : dx;
            if (want_r) w.grads[1] = dr;
            if (want_w) w.grads[2] = dw;
        }
        return once("add_rmsnorm", graph, std::move(w.grads), incoming);
    }
};

// (a tangent, made for forward-mode derivatives, is left to Python, whose functions refuse it)
bool has_tangent(std::initializer_list<const at::Tensor*> ts) {
    for (const at::Tensor* t : ts)
        if (t && t->_fw_grad(0).defined()) return true;
    return false;
}
bool differentiated(std::initializer_list<const at::Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const at::Tensor* t : ts)
        if (t && t->requires_grad()) return true;
    return false;
}
PyObject* tuple_of(const variable_list& list, PyObject* first) {
    PyObject* out = PyTuple_New((Py_ssize_t)list.size() + (first ? 1 : 0));
    if (!out) return nullptr;
    Py_ssize_t i = 0;
    if (first) {
        Py_INCREF(first);
        PyTuple_SET_ITEM(out, i++, first);
    }
    for (const at::Tensor& t : list) PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(t));
    return out;
}

// add_rmsnorm(x, residual, weight, eps, store, quantize, operand_order, return_rowsum) -> (s, [y], [q, s_x], [rowsum])
PyObject* add_rmsnorm(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    NormFlags f;
    ORDINARY(n_args == 8);
    const at::Tensor* x = rows_of(a[0], &device);
    ORDINARY(x && as_float(a[3], &f.eps) && as_bool(a[4], &f.store) && as_bool(a[5], &f.quantize) && as_bool(a[6], &f.operand_order) &&
             as_bool(a[7], &f.rowsum));
    const int64_t K = x->size(-1);
    ORDINARY((f.store || f.quantize) && (f.quantize || !f.rowsum));
    const at::Tensor *residual = nullptr, *weight = nullptr;
    if (a[1] != Py_None) {
        residual = plain(a[1], device);
        ORDINARY(residual && residual->sizes() == x->sizes() && (residual->scalar_type() == x->scalar_type() || residual->scalar_type() == at::kFloat));
    }
    if (a[2] != Py_None) {
        weight = plain(a[2], device);
        ORDINARY(weight && weight->dim() == 1 && weight->size(0) == K && (weight->scalar_type() == x->scalar_type() || weight->scalar_type() == at::kFloat));
    }
    ORDINARY(!has_tangent({x, residual, weight}));
    if (differentiated({x, residual, weight}))
        return tuple_of(AddRMSNorm::apply(*x, maybe(residual), maybe(weight), f.eps, f.store, f.quantize, f.operand_order, f.rowsum),
                        residual ? nullptr : a[0]);
    NormOut o = add_norm_run(*x, maybe(residual), maybe(weight), f, false);
    variable_list out;
    for (at::Tensor* t : {&o.s, &o.y, &o.q, &o.s_x, &o.rowsum})
        if (t->defined()) out.push_back(std::move(*t));
    return tuple_of(out, residual ? nullptr : a[0]);
    END_HANDLE_TH_ERRORS
}

struct GatedOut {
    at::Tensor h, rows, pre, w_back, scale;  // rows: x, or the copy of it that the kernels read; scale: for the gradient of fp16 rows its parts
};
// fp32 rows: K >= 4.  All tensors contiguous.
GatedOut gated_run(const at::Tensor& x, const at::Tensor& gate, const at::Tensor& up, const MaybeTensor& gate_bias, const MaybeTensor& up_bias,
                   double threshold, bool per_channel, bool keep, bool want_back) {
    const int64_t F = gate.size(0), K = gate.size(1), Fp = (F + 15) / 16 * 16, B = x.numel() / K;
    const bool fp32 = x.scalar_type() == at::kFloat;
    const int dt = tag(x.scalar_type());
    void* st = stream_of(x.get_device());
    GatedOut o;
    o.rows = x;
    if (!keep && lib.bt_gated_masters_serves(B, K, tag(gate.scalar_type()), per_channel ? 1 : 0)) {
        o.h = output(with_last(x, F), x.scalar_type(), x);
        call(lib.bt_gated_masters_forward, x.const_data_ptr(), dt, gate.const_data_ptr(), up.const_data_ptr(), tag(gate.scalar_type()), threshold,
             data_of(gate_bias), data_of(up_bias), gate_bias ? tag_of(gate_bias) : tag_of(up_bias), o.h.data_ptr(), F, K, st);
        return o;
    }
    const at::Tensor w = output({(int64_t)lib.bt_tiled_weights_bytes(2 * Fp, K)}, at::kByte, x);
    if (want_back) o.w_back = output({(int64_t)lib.bt_tiled_weights_bytes(K, 2 * Fp)}, at::kByte, x);
    o.scale = output({2 * Fp + 1}, at::kFloat, x);
    at::Tensor bias;
    if (gate_bias || up_bias) bias = output({2 * Fp}, at::kFloat, x);
    float* const scale_at = (float*)o.scale.data_ptr();
    float* const bias_at = bias.defined() ? (float*)bias.data_ptr() : nullptr;
    {
        const Scratch ws(lib.bt_gated_quantize_workspace_bytes(F, K, per_channel ? 1 : 0), x);
        call(lib.bt_gated_quantize, gate.const_data_ptr(), up.const_data_ptr(), tag(gate.scalar_type()), F, K, threshold, per_channel ? 1 : 0,
             data_of(gate_bias), data_of(up_bias), gate_bias ? tag_of(gate_bias) : tag_of(up_bias), (uint8_t*)w.data_ptr(),
             want_back ? (uint8_t*)o.w_back.data_ptr() : nullptr, scale_at, bias_at, ws.ptr(), ws.size(), st);
    }
    o.h = output(with_last(x, F), x.scalar_type(), x);
    if (fp32) o.pre = output({B, 2 * Fp}, at::kFloat, x);
    else if (keep) o.pre = output({B, Fp / 2 * 3}, at::kInt, x);
    if (!fp32) {
        void* padded = nullptr;
        if (K % 8 != 0 || !aligned(x, 16)) {
            o.rows = output({B, (K + 7) / 8 * 8}, x.scalar_type(), x);
            padded = o.rows.data_ptr();
        }
        call(lib.bt_ternary_gated_forward, x.const_data_ptr(), dt, padded, (const uint8_t*)w.const_data_ptr(), scale_at, bias_at, o.h.data_ptr(),
             keep ? o.pre.data_ptr() : nullptr, B, F, K, st);
        if (keep && x.scalar_type() == at::kHalf) {
            const at::Tensor split = output({(int64_t)lib.bt_gated_split_bytes(F) / 4}, at::kFloat, x);
            call(lib.bt_gated_split, scale_at, F, (float*)split.data_ptr(), st);
            o.scale = split;  // (the scales are the stream's until the kernels that read them have ended)
        }
        return o;
    }
    const Scratch ws(lib.bt_tiled_forward_workspace_bytes(B, 2 * Fp, K, dt), x);
    call(lib.bt_ternary_linear_tiled_forward, x.const_data_ptr(), K, dt, 0, nullptr, 0, 0.0f, (const uint8_t*)w.const_data_ptr(), scale_at, BT_F32, 2 * Fp,
         bias_at, BT_F32, nullptr, BT_EPI_NATURAL_FROM_PAIRS, o.pre.data_ptr(), B, 2 * Fp, K, ws.ptr(), ws.size(), st);
    call(lib.bt_swiglu, o.pre.const_data_ptr(), 2 * Fp, (const float*)o.pre.const_data_ptr() + Fp, 2 * Fp, BT_F32, B, F, o.h.data_ptr(), nullptr, nullptr, 0, st);
    return o;
}

struct GatedLinear : torch::autograd::Function<GatedLinear> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& gate, const at::Tensor& up, const MaybeTensor& gate_bias,
                              const MaybeTensor& up_bias, double threshold, bool per_channel) {
        GatedOut o = gated_run(x, gate, up, gate_bias, up_bias, threshold, per_channel, true, x.requires_grad());
        ctx->save_for_backward({o.rows, o.pre, o.w_back, o.scale});
        ctx->saved_data["shape"] = std::vector<int64_t>{gate.size(0), gate.size(1)};
        ctx->saved_data["dtype"] = gate.scalar_type();
        ctx->saved_data["biases"] = (int64_t)((gate_bias ? 1 : 0) | (up_bias ? 2 : 0));
        ctx->saved_data["bias_dtype"] = gate_bias ? gate_bias->scalar_type() : up_bias ? up_bias->scalar_type() : at::kFloat;
        return o.h;
    }
    static variable_list backward(AutogradContext* ctx, variable_list incoming) {
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &pre = saved[1], &w_back = saved[2], &scale = saved[3];
        const int64_t biases = ctx->saved_data["biases"].toInt();
        Wanted w(ctx, 7, {true, true, true, (biases & 1) != 0, (biases & 2) != 0});
        if (!incoming[0].defined()) return w.grads;
        const auto shape = ctx->saved_data["shape"].toIntVector();
        const at::ScalarType w_dtype = ctx->saved_data["dtype"].toScalarType(), b_dtype = ctx->saved_data["bias_dtype"].toScalarType();
        const bool graph = at::GradMode::is_enabled();
        const at::NoGradGuard no_grad;
        const c10::DeviceGuard guard(x.device());
        const int64_t F = shape[0], K = shape[1], Kr = x.size(-1), B = x.numel() / Kr;  // (a padded copy has longer rows)
        const bool fp32 = x.scalar_type() == at::kFloat, split = x.scalar_type() == at::kHalf;  // (split: scale is bt_gated_split's)
        const int64_t Fp = (F + 15) / 16 * 16;
        const int dt = tag(x.scalar_type());
        const bool want_w = w.want[1] || w.want[2], want_b = w.want[3] || w.want[4];
        void* st = stream_of(x.get_device());
        const at::Tensor dh = incoming[0].contiguous(), g = output({B, 2 * Fp}, x.scalar_type(), x);
        const float *scale_at = (const float*)scale.const_data_ptr(), *one = scale_at + 2 * Fp;
        at::Tensor db;
        if (want_b) db = output({2 * F}, b_dtype, x);
        {
            const Scratch ws(want_b ? lib.bt_gated_grad_workspace_bytes(B, F) : 0, x);
            check_status(lib.bt_gated_grad(dh.const_data_ptr(), dt, pre.const_data_ptr(), scale_at, g.data_ptr(), want_b ? db.data_ptr() : nullptr,
                                           want_b ? tag(b_dtype) : 0, B, F, ws.ptr(), ws.size(), st));
        }
        if (w.want[0] && split) {
            w.grads[0] = output(with_last(incoming[0], K), x.scalar_type(), x);
            const Scratch ws(lib.bt_gated_grad_input_workspace_bytes(B, F, K), x);
            check_status(lib.bt_gated_grad_input(g.const_data_ptr(), (const uint8_t*)w_back.const_data_ptr(), scale_at, w.grads[0].data_ptr(), B, F, K,
                                                 ws.ptr(), ws.size(), st));
        } else if (w.want[0]) {
            w.grads[0] = output(with_last(incoming[0], K), x.scalar_type(), x);
            const Scratch ws(lib.bt_tiled_forward_workspace_bytes(B, K, 2 * Fp, dt), x);
            check_status(lib.bt_ternary_linear_tiled_forward(g.const_data_ptr(), 2 * Fp, dt, 0, nullptr, 0, 0.0f, (const uint8_t*)w_back.const_data_ptr(), one,
                                                             BT_F32, 1, nullptr, 0, nullptr, 0, w.grads[0].data_ptr(), B, K, 2 * Fp, ws.ptr(), ws.size(), st));
        }
        if (want_w) {
            const at::ScalarType dtype = w_dtype == x.scalar_type() ? w_dtype : at::kFloat;
            const int64_t rows = fp32 ? Fp : F;  // of a half
            at::Tensor dw = output({2 * rows, K}, dtype, x);
            if (fp32) {
                const Scratch ws(lib.bt_linear_grad_weight_workspace_bytes(B, 2 * Fp, K), x);
                check_status(lib.bt_linear_grad_weight((const float*)g.const_data_ptr(), (const float*)x.const_data_ptr(), one, 1, (float*)dw.data_ptr(),
                                                       nullptr, B, 2 * Fp, K, ws.ptr(), ws.size(), st));
            } else {
                const Scratch ws(lib.bt_linear_grad_weight_16_workspace_bytes(B, 2 * Fp, Kr), x);
                check_status(lib.bt_gated_grad_masters(g.const_data_ptr(), x.const_data_ptr(), dt, split ? scale_at + 2 * Fp + 16 : one, split ? 2 * Fp : 1,
                                                       dw.data_ptr(), tag(dtype), B, F, K, ws.ptr(), ws.size(), st));
            }
            for (int i = 0; i < 2; i++)
                if (w.want[1 + i]) w.grads[1 + i] = dw.narrow(0, i * rows, F).to(w_dtype);
        }
        for (int i = 0; i < 2; i++)
            if (w.want[3 + i]) w.grads[3 + i] = db.narrow(0, i * F, F);
        return once("ternary_gated_linear", graph, std::move(w.grads), incoming);
    }
};

// gated_linear(x, gate, up, gate_bias, up_bias, threshold_factor, per_channel) -> h, where no autocast asks for another dtype
PyObject* gated_linear(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    double threshold;
    bool per_channel;
    ORDINARY(n_args == 7);
    const at::Tensor* x = rows_of(a[0], &device);
    ORDINARY(x && as_float(a[5], &threshold) && as_bool(a[6], &per_channel) && !at::autocast::is_autocast_enabled(at::kCUDA));
    const at::Tensor *gate = plain(a[1], device), *up = plain(a[2], device), *gate_bias = nullptr, *up_bias = nullptr;
    ORDINARY(gate && up && gate->dim() == 2 && gate->sizes() == up->sizes() && gate->scalar_type() == up->scalar_type() && tag(gate->scalar_type()) >= 0);
    const int64_t F = gate->size(0), K = gate->size(1);
    ORDINARY(x->size(-1) == K && (x->scalar_type() != at::kFloat || K >= 4));
    if (a[3] != Py_None) ORDINARY((gate_bias = vec(a[3], F, false, device)));
    if (a[4] != Py_None) ORDINARY((up_bias = vec(a[4], F, false, device)) && (!gate_bias || gate_bias->scalar_type() == up_bias->scalar_type()));
    ORDINARY(!has_tangent({x, gate, up, gate_bias, up_bias}));
    if (differentiated({x, gate, up, gate_bias, up_bias}))
        return THPVariable_Wrap(GatedLinear::apply(*x, *gate, *up, maybe(gate_bias), maybe(up_bias), threshold, per_channel));
    return THPVariable_Wrap(gated_run(*x, *gate, *up, maybe(gate_bias), maybe(up_bias), threshold, per_channel, false, false).h);
    END_HANDLE_TH_ERRORS
}

// ---- positions, the paged cache and the attention over it ------------------------------------------------------------------

// [tokens][heads][dim] with a stride for each of the first two.  A dimension of one entry may have any stride, in contiguous memory too.
struct HeadRows {
    const void* data = nullptr;
    int64_t tokens = 0, heads = 0, dim = 0, token = 0, head = 0;
};
bool head_rows(const at::Tensor& t, HeadRows* r) {
    const int64_t d = t.dim();
    if (d < 2 || tag(t.scalar_type()) < 0 || (t.stride(-1) != 1 && t.size(-1) != 1)) return false;
    *r = {t.const_data_ptr(), 1, t.size(-2), t.size(-1), 0, t.stride(-2)};
    for (int64_t i = d - 3; i >= 0; i--) {
        if (t.size(i) == 1) continue;
        if (r->tokens == 1) r->token = t.stride(i);
        else if (t.stride(i) != r->token * r->tokens) return false;
        r->tokens *= t.size(i);
    }
    return true;
}
const at::Tensor* head_rows_of(PyObject* o, int device, HeadRows* r) {
    const at::Tensor* t = on_device(o, device);
    return t && head_rows(*t, r) ? t : nullptr;
}
// Frequencies as the library reads them
const at::Tensor* frequencies(PyObject* o, int64_t dim, int device) {
    const at::Tensor* f = plain(o, device);
    return f && f->dim() == 1 && (f->scalar_type() == at::kFloat || f->scalar_type() == at::kDouble) && 2 * f->size(0) <= dim && !f->requires_grad() ? f : nullptr;
}

struct Turned {
    at::Tensor q, k;
};
// LOCKED: the calling thread holds the interpreter lock, and lets go of it around the call
template <bool LOCKED>
Turned rotary_run(const at::Tensor& q, const HeadRows& qr, const at::Tensor* k, const HeadRows& kr, const at::Tensor& positions, const at::Tensor& freq,
                  bool interleaved, double amplitude, bool backward) {
    Turned o;
    o.q = output(q.sizes(), q.scalar_type(), q);
    if (k) o.k = output(k->sizes(), k->scalar_type(), *k);
    void* st = stream_of(q.get_device());
    const int dt = tag(q.scalar_type()), wide = positions.scalar_type() == at::kLong, f64 = freq.scalar_type() == at::kDouble;
    const void *pos = positions.const_data_ptr(), *f = freq.const_data_ptr();
    void *q_out = o.q.data_ptr(), *k_out = k ? o.k.data_ptr() : nullptr;
    const int64_t rot = 2 * freq.size(0);
    if constexpr (LOCKED)
        call(lib.bt_rotary, qr.data, qr.token, qr.head, kr.data, kr.token, kr.head, dt, pos, wide, f, f64, interleaved ? 1 : 0, (float)amplitude, backward ? 1 : 0,
             qr.tokens, qr.heads, kr.heads, qr.dim, rot, q_out, k_out, st);
    else
        check_status(lib.bt_rotary(qr.data, qr.token, qr.head, kr.data, kr.token, kr.head, dt, pos, wide, f, f64, interleaved ? 1 : 0, (float)amplitude,
                                   backward ? 1 : 0, qr.tokens, qr.heads, kr.heads, qr.dim, rot, q_out, k_out, st));
    return o;
}

struct Rotary : torch::autograd::Function<Rotary> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const MaybeTensor& k, const at::Tensor& positions, const at::Tensor& freq,
                                 bool interleaved, double amplitude) {
        HeadRows qr, kr;
        head_rows(q, &qr);
        if (k) head_rows(*k, &kr);
        Turned o = rotary_run<true>(q, qr, k ? &*k : nullptr, kr, positions, freq, interleaved, amplitude, false);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({positions, freq});
        ctx->saved_data["k"] = k.has_value();
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["amplitude"] = amplitude;
        variable_list out{o.q};
        if (k) out.push_back(o.k);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list incoming) {
        const variable_list saved = ctx->get_saved_variables();
        const bool has_k = ctx->saved_data["k"].toBool(), interleaved = ctx->saved_data["interleaved"].toBool();
        const double amplitude = ctx->saved_data["amplitude"].toDouble();
        Wanted w(ctx, 6, {true, has_k});
        const bool graph = at::GradMode::is_enabled();
        const at::NoGradGuard no_grad;
        at::Tensor d[2];
        for (int i = 0; i < (has_k ? 2 : 1); i++)
            if (w.want[i] && incoming[i].defined()) d[i] = incoming[i];
        const int first = d[0].defined() ? 0 : 1;
        if (d[first].defined()) {
            const c10::DeviceGuard guard(d[first].device());
            HeadRows r[2];
            for (int i = first; i < 2; i++)
                if (d[i].defined() && !head_rows(d[i], &r[i])) {
                    d[i] = d[i].contiguous();
                    TORCH_CHECK(head_rows(d[i], &r[i]), "rotary: a gradient of ", d[i].sizes(), " is not rows of heads");
                }
            const bool both = first == 0 && d[1].defined();
            Turned o = rotary_run<false>(d[first], r[first], both ? &d[1] : nullptr, both ? r[1] : HeadRows(), saved[0], saved[1], interleaved, amplitude, true);
            w.grads[first] = o.q;
            if (both) w.grads[1] = o.k;
        }
        return once("rotary", graph, std::move(w.grads), incoming);
    }
};

// rotary(q, k, positions, inv_freq, interleaved, amplitude) -> (q, k), or q without k
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    bool interleaved;
    double amplitude;
    HeadRows qr, kr;
    ORDINARY(n_args == 6 && here(a[0], &device) && as_bool(a[4], &interleaved) && as_float(a[5], &amplitude));
    const at::Tensor *q = head_rows_of(a[0], device, &qr), *k = nullptr;
    ORDINARY(q);
    if (a[1] != Py_None) {
        k = head_rows_of(a[1], device, &kr);
        ORDINARY(k && k->dim() == q->dim() && k->scalar_type() == q->scalar_type() && kr.dim == qr.dim &&
                 k->sizes().slice(0, k->dim() - 2) == q->sizes().slice(0, q->dim() - 2));
    }
    const at::Tensor *positions = plain(a[2], device), *freq = frequencies(a[3], qr.dim, device);
    ORDINARY(positions && freq && (positions->scalar_type() == at::kLong || positions->scalar_type() == at::kInt) &&
             positions->sizes() == q->sizes().slice(0, q->dim() - 2));
    ORDINARY(!has_tangent({q, k}));
    variable_list out;
    if (differentiated({q, k})) out = Rotary::apply(*q, maybe(k), *positions, *freq, interleaved, amplitude);
    else {
        Turned o = rotary_run<true>(*q, qr, k, kr, *positions, *freq, interleaved, amplitude, false);
        out = {std::move(o.q), std::move(o.k)};
    }
    if (!k) return THPVariable_Wrap(std::move(out[0]));
    return tuple_of(out, nullptr);
    END_HANDLE_TH_ERRORS
}

// What both calls on the cache share, as the library reads it
struct CacheArgs {
    const at::Tensor *k = nullptr, *v = nullptr, *table = nullptr, *lengths = nullptr, *starts = nullptr;
    int64_t pages, kv_heads, page, width, sequences;
};
const at::Tensor* int32_of(PyObject* o, int64_t dim, int device) {
    const at::Tensor* t = plain(o, device);
    return t && t->dim() == dim && t->scalar_type() == at::kInt ? t : nullptr;
}
// a: k_cache, v_cache, block_table, lengths, q_starts; like: the rows
bool cache_of(PyObject* const* a, const at::Tensor& like, const HeadRows& rows, int device, CacheArgs* c) {
    c->k = plain(a[0], device), c->v = plain(a[1], device);
    if (!c->k || !c->v || c->k->dim() != 4 || c->k->sizes() != c->v->sizes() || c->k->scalar_type() != like.scalar_type() ||
        c->v->scalar_type() != like.scalar_type() || like.dim() != 3 || !aligned(*c->k, 16) || !aligned(*c->v, 16))
        return false;
    c->pages = c->k->size(0), c->kv_heads = c->k->size(1), c->page = c->k->size(2);
    if (c->page < 32 || (c->page & (c->page - 1)) || c->k->size(3) != lib.bt_cache_head_dim(tag(like.scalar_type()), rows.dim)) return false;
    c->table = int32_of(a[2], 2, device), c->lengths = int32_of(a[3], 1, device);
    if (!c->table || !c->lengths || c->table->size(0) != c->lengths->size(0)) return false;
    c->width = c->table->size(1), c->sequences = c->lengths->size(0);
    if (a[4] == Py_None) return c->sequences == rows.tokens;
    c->starts = int32_of(a[4], 1, device);
    return c->starts && c->starts->size(0) == c->sequences + 1;
}

// cache_append(k, v, k_cache, v_cache, block_table, lengths, q_starts, q, inv_freq, interleaved, amplitude, first_position) -> q turned
// (for a call without q Python's None is the answer and also says that the call was not ordinary: those are left to Python)
PyObject* cache_append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    bool interleaved;
    double amplitude;
    int64_t first;
    HeadRows kr, vr, qr;
    CacheArgs c;
    ORDINARY(n_args == 12 && here(a[0], &device) && as_bool(a[9], &interleaved) && as_float(a[10], &amplitude) && as_int(a[11], &first));
    const at::Tensor *k = head_rows_of(a[0], device, &kr), *v = head_rows_of(a[1], device, &vr), *q = head_rows_of(a[7], device, &qr);
    ORDINARY(k && v && q && cache_of(a + 2, *k, kr, device, &c) && v->sizes() == k->sizes() && v->scalar_type() == k->scalar_type() && q->dim() == 3 &&
             qr.tokens == kr.tokens && qr.dim == kr.dim && q->scalar_type() == k->scalar_type() && c.kv_heads == kr.heads);
    const at::Tensor* freq = frequencies(a[8], kr.dim, device);
    ORDINARY(freq && !differentiated({k, v, q, c.k, c.v}) && !has_tangent({k, v, q, c.k, c.v}));
    const char *kc = (const char*)c.k->data_ptr(), *vc = (const char*)c.v->data_ptr();
    ORDINARY(kc + c.k->nbytes() <= vc || vc + c.v->nbytes() <= kc);
    at::Tensor out = output(q->sizes(), q->scalar_type(), *q);
    for (const at::Tensor* t : {c.k, c.v})
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    void* st = stream_of(device);
    call(lib.bt_cache_append, kr.data, kr.token, kr.head, vr.data, vr.token, vr.head, qr.data, qr.token, qr.head, tag(k->scalar_type()), freq->const_data_ptr(),
         freq->scalar_type() == at::kDouble ? 1 : 0, interleaved ? 1 : 0, (float)amplitude, first, kr.tokens, qr.heads, kr.heads, kr.dim, 2 * freq->size(0),
         c.k->data_ptr(), c.v->data_ptr(), c.pages, c.page, (const int32_t*)c.table->const_data_ptr(), c.width, (const int32_t*)c.lengths->const_data_ptr(),
         c.starts ? (const int32_t*)c.starts->const_data_ptr() : nullptr, c.sequences, out.data_ptr(), st);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// cached_attention(q, k_cache, v_cache, block_table, lengths, q_starts, scale, prefix_table, prefix_length, return_lse, max_length) -> out or (out, lse)
PyObject* cached_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    int device;
    bool want_lse;
    int64_t prefix, longest;
    HeadRows qr;
    CacheArgs c;
    ORDINARY(n_args == 11 && here(a[0], &device) && as_int(a[8], &prefix) && as_bool(a[9], &want_lse) && prefix >= 0);
    const at::Tensor *q = head_rows_of(a[0], device, &qr), *shared = nullptr;
    ORDINARY(q && cache_of(a + 1, *q, qr, device, &c) && qr.heads % c.kv_heads == 0 && !differentiated({q, c.k, c.v}) && !has_tangent({q, c.k, c.v}));
    double scale = 1.0 / std::sqrt((double)qr.dim);
    if (a[6] != Py_None) ORDINARY(as_float(a[6], &scale));
    ORDINARY(scale > 0.0 && scale < 3.0e38);
    const int64_t most = c.width * c.page;
    longest = most;
    if (a[10] != Py_None) ORDINARY(as_int(a[10], &longest) && longest >= 0 && longest <= most);
    if (prefix) {
        shared = int32_of(a[7], 1, device);
        ORDINARY(shared && prefix <= shared->size(0) * c.page);
    }
    const int64_t T = qr.tokens;
    at::Tensor out = output(q->sizes(), q->scalar_type(), *q), lse;
    if (want_lse) lse = output({T, qr.heads}, at::kFloat, *q);
    const int64_t per = 16 / (int64_t)q->element_size();
    const int in_place = qr.dim % per == 0 && qr.token % per == 0 && qr.head % per == 0 && aligned(*q, 16) ? 1 : 0;
    const Scratch ws(lib.bt_cached_attention_workspace_bytes(tag(q->scalar_type()), in_place, T, qr.heads, c.kv_heads, qr.dim, c.page, c.width, longest, c.starts ? 1 : 0, c.sequences, prefix), *q);
    void* st = stream_of(device);
    call(lib.bt_cached_attention, qr.data, qr.token, qr.head, tag(q->scalar_type()), c.k->const_data_ptr(), c.v->const_data_ptr(), c.pages, c.page,
         (const int32_t*)c.table->const_data_ptr(), c.width, longest, (const int32_t*)c.lengths->const_data_ptr(),
         c.starts ? (const int32_t*)c.starts->const_data_ptr() : nullptr, c.sequences, shared ? (const int32_t*)shared->const_data_ptr() : nullptr, prefix,
         (float)scale, T, qr.heads, c.kv_heads, qr.dim, out.data_ptr(), want_lse ? (float*)lse.data_ptr() : nullptr, ws.ptr(), ws.size(), st);
    if (!want_lse) return THPVariable_Wrap(std::move(out));
    return tuple_of({std::move(out), std::move(lse)}, nullptr);
    END_HANDLE_TH_ERRORS
}

// generic_kernel_asked(): whether BITTORCH_KERNEL=generic, read now
PyObject* generic_kernel_asked(PyObject*, PyObject* const*, Py_ssize_t) {
    const char* env = std::getenv("BITTORCH_KERNEL");
    return PyBool_FromLong(env && !std::strcmp(env, "generic"));
}

// stamp(): what this file was compiled against.  Its accessors are inlined from torch's headers and its calls typed by
// bittorch_hip.h, so _lib.py binds it to that build of torch and that ABI alone.
#define BT_TEXT(x) #x
#define BT_TEXT_OF(x) BT_TEXT(x)
PyObject* stamp(PyObject*, PyObject* const*, Py_ssize_t) { return PyUnicode_FromString("abi " BT_TEXT_OF(BT_ABI_VERSION) ", " BT_CALLS_BUILD); }

// bind({name: address}): the library's functions
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (n_args != 1 || !PyDict_Check(a[0])) {
        PyErr_SetString(PyExc_TypeError, "bind takes a dict of addresses");
        return nullptr;
    }
#define X(name)                                                                   \
    {                                                                             \
        PyObject* at = PyDict_GetItemString(a[0], #name);                         \
        void* p = at ? PyLong_AsVoidPtr(at) : nullptr;                            \
        if (!p) {                                                                 \
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_KeyError, #name);        \
            return nullptr;                                                       \
        }                                                                         \
        lib.name = reinterpret_cast<decltype(lib.name)>(p);                       \
    }
    BT_FUNCTIONS(X)
#undef X
    bound = true;
    Py_RETURN_NONE;
}
PyObject* names(PyObject*, PyObject* const*, Py_ssize_t) {
    static const char* const all[] = {
#define X(name) #name,
        BT_FUNCTIONS(X)
#undef X
    };
    PyObject* out = PyList_New(0);
    for (const char* n : all) {
        PyObject* s = PyUnicode_FromString(n);
        if (!out || !s || PyList_Append(out, s) != 0) return nullptr;
        Py_DECREF(s);
    }
    return out;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(names), METHOD(stamp), METHOD(tiled_forward), METHOD(packed_forward), METHOD(tensor_core_forward),
                         METHOD(quantize_pack), METHOD(grad_input), METHOD(grad_weight),
                         METHOD(grad_weight_16), METHOD(unpack_dequant), METHOD(rmsnorm_int8), METHOD(swiglu_int8), METHOD(gemm_i8_tiled), METHOD(swiglu_i8_tiled), METHOD(act_quant_int8), METHOD(add_rmsnorm), METHOD(gated_linear),
                         METHOD(rotary), METHOD(cache_append), METHOD(cached_attention),
                         METHOD(generic_kernel_asked), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "Native host side of small calls (csrc/calls.cpp)", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
