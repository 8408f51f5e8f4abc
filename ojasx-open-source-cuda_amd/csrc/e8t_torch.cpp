// e8t_torch.cpp -- the eager calls of ojasx_amd on plain GPU tensors, without the Python-level
// op dispatch (a CPython extension over the C ABI and torch's C++ tensors).
//
// A call of a torch.library custom op from Python costs 15-20 us of host time before its
// kernel is enqueued (op dispatch through Python kernels, argument checks, allocation, the
// ctypes call), more than most decode and small-batch kernels run.  These functions make
// the same checks, allocations and library calls in C++.  Each returns None, having done
// nothing, for every call that is not plain eager work on tensors it knows: the caller then
// takes the registered op, which handles (or refuses) it as before.  Plain means: exact
// Tensor or Parameter objects on one ROCm device; no autograd to record (grad mode off, or
// nothing requires grad; token_logprobs_recorded and rotary_recorded bring nodes of their own); no
// tangents; and no
// dispatch or function mode, functorch transform or tracer active.
//
// Measured, us per call among others: one bf16 token through a 4096 x 4096 layer 26.2 -> 6.2
// (host time 5.9, kernel 5.2), 77 rows in 2 bits through 3072 x 4100 32.0 -> 21.2, a training
// step of 16 fp32 tokens with an adapter 239 -> 106.

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/record_function.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <string>

#include "../../include/ojasx_e8t.h"

namespace {

using at::Tensor;

// Tensors and thread states that only the dispatcher treats correctly.
const c10::DispatchKeySet kSpecialTensor({
    c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::Conjugate,
    c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor, c10::DispatchKey::Functionalize,
    c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
    c10::DispatchKey::BatchedNestedTensor, c10::DispatchKey::Batched,
});
const c10::DispatchKeySet kSpecialState({
    c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::PythonDispatcher,
    c10::DispatchKey::PreDispatch, c10::DispatchKey::Functionalize, c10::DispatchKey::Tracer,
    c10::DispatchKey::FuncTorchDynamicLayerFrontMode, c10::DispatchKey::FuncTorchDynamicLayerBackMode,
    c10::DispatchKey::FuncTorchVmapMode, c10::DispatchKey::VmapMode,
});

bool plain_state() {
    return c10::impl::TorchDispatchModeTLS::stack_len() == 0 &&
           at::impl::PythonTorchFunctionTLS::stack_len() == 0 &&
           !c10::impl::tls_local_dispatch_key_set().included_.has_any(kSpecialState);
}

bool plain(const Tensor& t) {
    return t.defined() && t.layout() == at::kStrided && t.is_cuda() &&
           !t.key_set().has_any(kSpecialTensor) && !t._fw_grad(0).defined();
}
bool plain(PyObject* o) { return THPVariable_CheckExact(o) && plain(THPVariable_Unpack(o)); }

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return OJX_F32;
        case at::kHalf: return OJX_F16;
        case at::kBFloat16: return OJX_BF16;
        default: return -1;
    }
}

// Code bytes of `padded` weights; the unit a group size must be a multiple of.
int64_t code_bytes(int fmt, int64_t padded) {
    return fmt == OJX_FMT_TERNARY ? padded * 3 / 16 : fmt == OJX_FMT_E8 ? padded / 4 : padded / 8;
}
int64_t gs_unit(int fmt) { return fmt == OJX_FMT_TERNARY ? 16 : fmt == OJX_FMT_E8 ? 4 : 8; }
int64_t padded_to(int64_t n, int64_t gs) { return n + (gs - n % gs) % gs; }

// A layer's buffers as the ops accept them without a copy.
bool layer_ok(const Tensor& packed, const Tensor& scales, int fmt, int64_t N, int64_t K,
              int64_t gs) {
    if (fmt < 0 || fmt > 2 || gs <= 0 || gs % gs_unit(fmt) != 0 || N < 1 || K < 1) return false;
    const int64_t padded = padded_to(N * K, gs);
    return packed.scalar_type() == at::kByte && scales.scalar_type() == at::kHalf &&
           packed.is_contiguous() && scales.is_contiguous() &&
           packed.numel() >= code_bytes(fmt, padded) && scales.numel() >= padded / gs;
}

// The interpreter lock is given up while memory is allocated and kernels are launched, as the
// registered ops do: both can wait (a full queue, a new segment), and other threads go on.
class Unlocked {
  public:
    Unlocked() : state_(PyEval_SaveThread()) {}
    ~Unlocked() { lock(); }
    void lock() {
        if (state_) PyEval_RestoreThread(state_);
        state_ = nullptr;
    }

  private:
    PyThreadState* state_;
};

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void* current_stream(const c10::Device& d) {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(d.index()).stream();
}

void check(int status, const char* what) {
    if (status != OJX_OK)
        throw std::runtime_error(std::string("ojasx_e8t ") + what + " failed (status " +
                                 std::to_string(status) + "): " + ojx_e8t_last_error());
}

Tensor workspace(size_t bytes, const Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

struct Args {
    PyObject* const* a;
    Py_ssize_t n;
    int64_t i64(int i) const {
        const int64_t v = PyLong_AsLongLong(a[i]);
        if (v == -1 && PyErr_Occurred()) throw python_error();
        return v;
    }
    double f64(int i) const {
        const double v = PyFloat_AsDouble(a[i]);
        if (v == -1.0 && PyErr_Occurred()) throw python_error();
        return v;
    }
    bool flag(int i) const { return a[i] == Py_True; }
    bool truth(int i) const {
        const int v = PyObject_IsTrue(a[i]);
        if (v < 0) throw python_error();
        return v != 0;
    }
    const Tensor& t(int i) const { return THPVariable_Unpack(a[i]); }
};

void expect(Py_ssize_t n, Py_ssize_t want, const char* what) {
    if (n != want)
        throw std::runtime_error(std::string(what) + " takes " + std::to_string(want) +
                                 " arguments (got " + std::to_string(n) + ")");
}

typedef int (*FwdFn)(const void*, const uint8_t*, const uint16_t*, const void*, void*, int64_t,
                     int64_t, int64_t, int64_t, int, void*, size_t, void*);
typedef int (*LoraFn)(const void*, const uint8_t*, const uint16_t*, const void*, const void*,
                      const void*, int64_t, float, float*, void*, int64_t, int64_t, int64_t,
                      int64_t, int, void*, size_t, void*);
typedef int (*BwdFn)(const void*, const uint8_t*, const uint16_t*, void*, int64_t, int64_t, int64_t,
                     int64_t, int, void*, size_t, void*);
const FwdFn kFwd[] = {ojx_e8t_gemm_fwd, ojx_e8_gemm_fwd, ojx_e8r_gemm_fwd};
const LoraFn kFwdLora[] = {ojx_e8t_gemm_fwd_lora, ojx_e8_gemm_fwd_lora, ojx_e8r_gemm_fwd_lora};
const BwdFn kBwd[] = {ojx_e8t_gemm_bwd_dx, ojx_e8_gemm_bwd_dx, ojx_e8r_gemm_bwd_dx};

bool records(const Tensor& t) { return t.defined() && t.requires_grad(); }

std::vector<int64_t> with_last(const Tensor& x, int64_t last) {
    std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
    s.back() = last;
    return s;
}

// linear(x, packed, scales, bias | None, N, K, gs, fmt): y, the forward of one layer
PyObject* linear(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 8, "linear");
    const Args a{argv, n};
    if (!plain_state() || !plain(argv[0]) || !plain(argv[1]) || !plain(argv[2]) ||
        (argv[3] != Py_None && !plain(argv[3])))
        Py_RETURN_NONE;
    const Tensor &x = a.t(0), &packed = a.t(1), &scales = a.t(2);
    const Tensor bias = argv[3] == Py_None ? Tensor() : a.t(3);
    const int64_t N = a.i64(4), K = a.i64(5), gs = a.i64(6);
    const int fmt = (int)a.i64(7), dt = dtype_code(x.scalar_type());
    if (dt < 0 || x.dim() < 1 || x.size(-1) != K || !layer_ok(packed, scales, fmt, N, K, gs) ||
        packed.device() != x.device() || scales.device() != x.device())
        Py_RETURN_NONE;
    if (bias.defined() && (bias.numel() != N || bias.scalar_type() != x.scalar_type() ||
                           !bias.is_contiguous() || bias.device() != x.device()))
        Py_RETURN_NONE;
    if (c10::GradMode::is_enabled() && (records(x) || records(bias))) Py_RETURN_NONE;
    RECORD_FUNCTION("ojasx_e8t::linear", std::vector<c10::IValue>());
    Unlocked unlocked;
    const c10::DeviceGuard on_device(x.device());
    const Tensor xc = x.contiguous();
    const int64_t M = xc.numel() / K;
    Tensor y = at::empty(with_last(x, N), x.options());
    size_t bytes = 0;
    check(ojx_gemm_workspace_bytes(fmt, 0, M, N, K, gs, dt, &bytes), "gemm_workspace_bytes");
    const Tensor ws = workspace(bytes, x);
    check(kFwd[fmt](data(xc), (const uint8_t*)data(packed), (const uint16_t*)data(scales),
                    data(bias), data(y), M, N, K, gs, dt, data(ws), bytes,
                    current_stream(x.device())),
          "gemm_fwd");
    unlocked.lock();
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// linear_bwd(gy, packed, scales, N, K, gs, fmt): gx
PyObject* linear_bwd(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 7, "linear_bwd");
    const Args a{argv, n};
    if (!plain_state() || !plain(argv[0]) || !plain(argv[1]) || !plain(argv[2])) Py_RETURN_NONE;
    const Tensor &gy = a.t(0), &packed = a.t(1), &scales = a.t(2);
    const int64_t N = a.i64(3), K = a.i64(4), gs = a.i64(5);
    const int fmt = (int)a.i64(6), dt = dtype_code(gy.scalar_type());
    if (dt < 0 || gy.dim() < 1 || gy.size(-1) != N || !layer_ok(packed, scales, fmt, N, K, gs) ||
        packed.device() != gy.device() || scales.device() != gy.device() ||
        (c10::GradMode::is_enabled() && records(gy)))
        Py_RETURN_NONE;
    RECORD_FUNCTION("ojasx_e8t::linear_bwd", std::vector<c10::IValue>());
    Unlocked unlocked;
    const c10::DeviceGuard on_device(gy.device());
    const Tensor gc = gy.contiguous();
    const int64_t M = gc.numel() / N;
    Tensor gx = at::empty(with_last(gy, K), gy.options());
    size_t bytes = 0;
    check(ojx_gemm_workspace_bytes(fmt, 1, M, N, K, gs, dt, &bytes), "gemm_workspace_bytes");
    const Tensor ws = workspace(bytes, gy);
    check(kBwd[fmt](data(gc), (const uint8_t*)data(packed), (const uint16_t*)data(scales), data(gx),
                    M, N, K, gs, dt, data(ws), bytes, current_stream(gy.device())),
          "gemm_bwd_dx");
    unlocked.lock();
    return THPVariable_Wrap(std::move(gx));
    END_HANDLE_TH_ERRORS
}

// The adapter's factors as the kernels read them.
bool factors_ok(const Tensor& x, const Tensor& la, const Tensor& lb, int64_t N, int64_t K) {
    return la.dim() == 2 && lb.dim() == 2 && la.size(0) == K && lb.size(1) == N &&
           la.size(1) == lb.size(0) && la.size(1) >= 1 && la.size(1) <= 64 &&
           la.scalar_type() == x.scalar_type() && lb.scalar_type() == x.scalar_type() &&
           la.is_contiguous() && lb.is_contiguous() && la.device() == x.device() &&
           lb.device() == x.device();
}

// linear_lora(x, packed, scales, bias | None, lora_a, lora_b, scaling, fmt, N, K, gs): y
PyObject* linear_lora(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 11, "linear_lora");
    const Args a{argv, n};
    if (!plain_state() || !plain(argv[0]) || !plain(argv[1]) || !plain(argv[2]) ||
        (argv[3] != Py_None && !plain(argv[3])) || !plain(argv[4]) || !plain(argv[5]))
        Py_RETURN_NONE;
    const Tensor &x = a.t(0), &packed = a.t(1), &scales = a.t(2), &la = a.t(4), &lb = a.t(5);
    const Tensor bias = argv[3] == Py_None ? Tensor() : a.t(3);
    const float scaling = (float)a.f64(6);
    const int fmt = (int)a.i64(7), dt = dtype_code(x.scalar_type());
    const int64_t N = a.i64(8), K = a.i64(9), gs = a.i64(10);
    if (dt < 0 || x.dim() < 1 || x.size(-1) != K || !layer_ok(packed, scales, fmt, N, K, gs) ||
        packed.device() != x.device() || scales.device() != x.device() ||
        !factors_ok(x, la, lb, N, K))
        Py_RETURN_NONE;
    if (bias.defined() && (bias.numel() != N || bias.scalar_type() != x.scalar_type() ||
                           !bias.is_contiguous() || bias.device() != x.device()))
        Py_RETURN_NONE;
    if (c10::GradMode::is_enabled() && (records(x) || records(bias) || records(la) || records(lb)))
        Py_RETURN_NONE;
    RECORD_FUNCTION("ojasx_e8t::linear_lora", std::vector<c10::IValue>());
    Unlocked unlocked;
    const c10::DeviceGuard on_device(x.device());
    const Tensor xc = x.contiguous();
    const int64_t M = xc.numel() / K, r = la.size(1);
    Tensor y = at::empty(with_last(x, N), x.options());
    const Tensor u = at::empty({M, r}, x.options().dtype(at::kFloat));
    size_t bytes = 0;
    check(ojx_gemm_workspace_bytes(fmt, 0, M, N, K, gs, dt, &bytes), "gemm_workspace_bytes");
    const Tensor ws = workspace(bytes, x);
    check(kFwdLora[fmt](data(xc), (const uint8_t*)data(packed), (const uint16_t*)data(scales),
                        data(bias), data(la), data(lb), r, scaling, (float*)data(u), data(y), M, N,
                        K, gs, dt, data(ws), bytes, current_stream(x.device())),
          "gemm_fwd_lora");
    unlocked.lock();
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// linear_lora_bwd(x, gy, packed, scales, lora_a, lora_b, scaling, fmt, N, K, gs, need_x, need_a,
// need_b): (gx | None, ga | None, gb | None)
PyObject* linear_lora_bwd(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 14, "linear_lora_bwd");
    const Args a{argv, n};
    if (!plain_state()) Py_RETURN_NONE;
    for (int i = 0; i < 6; ++i)
        if (!plain(argv[i])) Py_RETURN_NONE;
    const Tensor &x = a.t(0), &gy = a.t(1), &packed = a.t(2), &scales = a.t(3), &la = a.t(4),
                 &lb = a.t(5);
    const float scaling = (float)a.f64(6);
    const int fmt = (int)a.i64(7), dt = dtype_code(x.scalar_type());
    const int64_t N = a.i64(8), K = a.i64(9), gs = a.i64(10);
    const bool need_x = a.flag(11), need_a = a.flag(12), need_b = a.flag(13);
    if (dt < 0 || gy.scalar_type() != x.scalar_type() || x.dim() < 1 || x.size(-1) != K ||
        gy.dim() < 1 || gy.size(-1) != N || !layer_ok(packed, scales, fmt, N, K, gs) ||
        packed.device() != x.device() || scales.device() != x.device() ||
        gy.device() != x.device() || !factors_ok(x, la, lb, N, K) || x.numel() == 0 ||
        x.numel() / K != gy.numel() / N || c10::GradMode::is_enabled())
        Py_RETURN_NONE;
    RECORD_FUNCTION("ojasx_e8t::linear_lora_bwd", std::vector<c10::IValue>());
    Unlocked unlocked;
    const c10::DeviceGuard on_device(x.device());
    const Tensor xc = x.contiguous(), gc = gy.contiguous();
    const int64_t M = xc.numel() / K, r = la.size(1);
    Tensor gx = need_x ? at::empty(x.sizes(), gy.options()) : Tensor();
    Tensor ga = need_a ? at::empty({K, r}, gy.options()) : Tensor();
    Tensor gb = need_b ? at::empty({r, N}, gy.options()) : Tensor();
    const Tensor uv = at::empty({2, M, r}, x.options().dtype(at::kFloat));
    size_t bytes = 0;
    check(ojx_gemm_bwd_lora_workspace_bytes(fmt, M, N, K, gs, r, need_x, need_a, need_b, dt, &bytes),
          "gemm_bwd_lora_workspace_bytes");
    const Tensor ws = workspace(bytes, x);
    check(ojx_gemm_bwd_lora(fmt, data(xc), data(gc), (const uint8_t*)data(packed),
                            (const uint16_t*)data(scales), data(la), data(lb), r, scaling,
                            (float*)data(uv), data(gx), data(ga), data(gb), M, N, K, gs, dt,
                            data(ws), bytes, current_stream(x.device())),
          "gemm_bwd_lora");
    unlocked.lock();
    PyObject* out = PyTuple_New(3);
    if (!out) throw python_error();
    Tensor* ts[] = {&gx, &ga, &gb};
    for (int i = 0; i < 3; ++i) {
        if (ts[i]->defined()) {
            PyTuple_SET_ITEM(out, i, THPVariable_Wrap(std::move(*ts[i])));
        } else {
            Py_INCREF(Py_None);
            PyTuple_SET_ITEM(out, i, Py_None);
        }
    }
    return out;
    END_HANDLE_TH_ERRORS
}

typedef int (*EncodeFn)(const void*, int, int64_t, int64_t, uint8_t*, uint16_t*, void*);
typedef int (*DecodeFn)(const uint8_t*, const uint16_t*, int64_t, int64_t, int, void*, void*);
const EncodeFn kEncode[] = {ojx_e8t_encode, ojx_e8_encode, ojx_e8r_encode};
const DecodeFn kDecode[] = {ojx_e8t_decode, ojx_e8_decode, ojx_e8r_decode};
int64_t pack_unit(int fmt) { return fmt == OJX_FMT_TERNARY ? 16 : 8; }

// encode(w, gs, fmt): (packed, scales)
PyObject* encode(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 3, "encode");
    const Args a{argv, n};
    if (!plain_state() || !plain(argv[0])) Py_RETURN_NONE;
    const Tensor& w = a.t(0);
    const int64_t gs = a.i64(1);
    const int fmt = (int)a.i64(2), dt = dtype_code(w.scalar_type());
    if (dt < 0 || fmt < 0 || fmt > 2 || gs <= 0 || gs % pack_unit(fmt) != 0 ||
        (c10::GradMode::is_enabled() && records(w)))
        Py_RETURN_NONE;
    RECORD_FUNCTION("ojasx_e8t::encode", std::vector<c10::IValue>());
    Unlocked unlocked;
    const c10::DeviceGuard on_device(w.device());
    const Tensor wc = w.contiguous();
    const int64_t padded = padded_to(wc.numel(), gs);
    Tensor packed = at::empty({code_bytes(fmt, padded)}, w.options().dtype(at::kByte));
    Tensor scales = at::empty({padded / gs}, w.options().dtype(at::kHalf));
    check(kEncode[fmt](data(wc), dt, wc.numel(), gs, (uint8_t*)data(packed),
                       (uint16_t*)data(scales), current_stream(w.device())),
          "encode");
    unlocked.lock();
    PyObject* out = PyTuple_New(2);
    if (!out) throw python_error();
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(packed)));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(scales)));
    return out;
    END_HANDLE_TH_ERRORS
}

// decode(packed, scales, numel, gs, dtype, fmt): flat weights, dtype a code of the C ABI
PyObject* decode(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 6, "decode");
    const Args a{argv, n};
    if (!plain_state() || !plain(argv[0]) || !plain(argv[1])) Py_RETURN_NONE;
    const Tensor &packed = a.t(0), &scales = a.t(1);
    const int64_t numel = a.i64(2), gs = a.i64(3);
    const int dt = (int)a.i64(4), fmt = (int)a.i64(5);
    if (dt < 0 || dt > 2 || fmt < 0 || fmt > 2 || gs <= 0 || gs % pack_unit(fmt) != 0 ||
        numel < 0 || packed.scalar_type() != at::kByte || scales.scalar_type() != at::kHalf ||
        !packed.is_contiguous() || !scales.is_contiguous() ||
        packed.device() != scales.device() ||
        packed.numel() < code_bytes(fmt, padded_to(numel, gs)) ||
        scales.numel() < padded_to(numel, gs) / gs ||
        (c10::GradMode::is_enabled() && records(scales)))
        Py_RETURN_NONE;
    RECORD_FUNCTION("ojasx_e8t::decode", std::vector<c10::IValue>());
    Unlocked unlocked;
    const c10::DeviceGuard on_device(packed.device());
    const at::ScalarType types[] = {at::kFloat, at::kHalf, at::kBFloat16};
    Tensor out = at::empty({numel}, packed.options().dtype(types[dt]));
    check(kDecode[fmt]((const uint8_t*)data(packed), (const uint16_t*)data(scales), numel, gs, dt,
                       data(out), current_stream(packed.device())),
          "decode");
    unlocked.lock();
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- cache, log probabilities

bool kv_block(int64_t b) { return b == 16 || b == 32 || b == 64 || b == 128 || b == 256; }

bool ints(const Tensor& t, at::ScalarType type, int64_t n) {
    return t.scalar_type() == type && t.dim() == 1 && t.numel() == n && t.is_contiguous();
}

// A cache's tensors as the ops take them, for heads of size d.
bool cache_ok(const Tensor& k, const Tensor& v, const Tensor& scales, int64_t d) {
    return k.scalar_type() == at::kChar && v.scalar_type() == at::kChar &&
           scales.scalar_type() == at::kFloat && k.dim() == 4 && k.sizes() == v.sizes() &&
           scales.dim() == 3 && scales.size(0) == k.size(0) && scales.size(1) == k.size(1) &&
           scales.size(2) == 2 && k.is_contiguous() && v.is_contiguous() &&
           scales.is_contiguous() && kv_block(k.size(2)) && d >= 1 && d <= 256 &&
           k.size(3) == (d + 63) / 64 * 64 && v.device() == k.device() &&
           scales.device() == k.device();
}

PyObject* tuple_of(Tensor* ts, int n) {
    PyObject* out = PyTuple_New(n);
    if (!out) throw python_error();
    for (int i = 0; i < n; ++i) PyTuple_SET_ITEM(out, i, THPVariable_Wrap(std::move(ts[i])));
    return out;
}

// Results of one call, side by side in an allocation: the allocator costs 0.7 us a tensor, as much as
// a seventh of the kernel of a small call.  A result that is kept keeps its neighbours, so those of
// over kTogether bytes are in two allocations, each of results of about the same size (with one for
// each result a plan of some thousand tokens took 9.4 us, 7.2 in one or two).
class Results {
  public:
    static constexpr int64_t kTogether = 64 * 1024;

    // Bytes of a result of n elements; all begin at multiples of 16.
    static int64_t room(int64_t n, int64_t element) { return (n * element + 15) / 16 * 16; }

    Results(int64_t first, int64_t second, const Tensor& like)
        : options_(like.options().dtype(at::kByte)),
          second_(first + second > kTogether ? second : 0),
          all_(at::empty({second_ ? first : first + second}, options_)) {}

    // The second part's results follow.
    void second() {
        if (!second_) return;
        all_ = at::empty({second_}, options_);
        used_ = 0;
    }

    Tensor next(at::IntArrayRef shape, at::ScalarType type) {
        const int64_t element = (int64_t)c10::elementSize(type);
        Tensor t = at::detail::make_tensor<c10::TensorImpl>(
            c10::Storage(all_.storage()), all_.key_set(), c10::scalarTypeToTypeMeta(type));
        t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
        t.unsafeGetTensorImpl()->set_storage_offset(used_ / element);
        used_ += room(t.numel(), element);
        TORCH_INTERNAL_ASSERT(used_ <= all_.numel());
        return t;
    }

  private:
    at::TensorOptions options_;
    int64_t second_;
    Tensor all_;
    int64_t used_ = 0;
};

bool all_plain(PyObject* const* argv, int n) {
    if (!plain_state()) return false;
    for (int i = 0; i < n; ++i)
        if (!plain(argv[i])) return false;
    return true;
}

// kv8_plan(seq_lens, new_lens, tables, free, num_free, block_size, tokens): the op's results
PyObject* kv8_plan(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 7, "kv8_plan");
    const Args a{argv, n};
    if (!all_plain(argv, 5)) Py_RETURN_NONE;
    const Tensor &seq = a.t(0), &fresh = a.t(1), &tables = a.t(2), &free = a.t(3), &left = a.t(4);
    const int64_t block = a.i64(5), tokens = a.i64(6), r = seq.numel();
    if (!ints(seq, at::kInt, r) || !ints(fresh, at::kInt, r) ||
        !ints(free, at::kInt, free.numel()) || !ints(left, at::kInt, 1) ||
        tables.scalar_type() != at::kInt || tables.dim() != 2 || tables.size(0) != r ||
        (tables.numel() > 0 && tables.stride(1) != 1) || !kv_block(block) || tokens < 0 ||
        fresh.device() != seq.device() || tables.device() != seq.device() ||
        free.device() != seq.device() || left.device() != seq.device())
        Py_RETURN_NONE;
    RECORD_FUNCTION("ojasx_e8t::kv8_plan", std::vector<c10::IValue>());
    Unlocked unlocked;
    const c10::DeviceGuard on_device(seq.device());
    Results all(Results::room(tokens, 8) + 2 * Results::room(tokens, 4),
                Results::room(r + 1, 4) + Results::room(r, 4) + Results::room(1, 4), seq);
    Tensor out[6];
    out[0] = all.next({tokens}, at::kLong);
    for (int i = 1; i < 3; ++i) out[i] = all.next({tokens}, at::kInt);
    all.second();
    out[3] = all.next({r + 1}, at::kInt);
    out[4] = all.next({r}, at::kInt);
    out[5] = all.next({1}, at::kInt);
    check(ojx_kv8_plan((const int32_t*)data(seq), (const int32_t*)data(fresh), r,
                       (int32_t*)data(tables), tables.stride(0), tables.size(1),
                       (const int32_t*)data(free), free.numel(), (const int32_t*)data(left), block,
                       tokens, (int64_t*)data(out[0]), (int32_t*)data(out[1]),
                       (int32_t*)data(out[2]), (int32_t*)data(out[3]), (int32_t*)data(out[4]),
                       (int32_t*)data(out[5]), current_stream(seq.device())),
          "kv8_plan");
    torch::autograd::impl::bump_version(tables);
    unlocked.lock();
    return tuple_of(out, 6);
    END_HANDLE_TH_ERRORS
}

// kv8_reorder(parents, seq_lens, tables, free, num_free, block_size, num_blocks): the op's results
PyObject* kv8_reorder(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 7, "kv8_reorder");
    const Args a{argv, n};
    if (!all_plain(argv, 5)) Py_RETURN_NONE;
    const Tensor &parents = a.t(0), &seq = a.t(1), &tables = a.t(2), &free = a.t(3), &left = a.t(4);
    const int64_t block = a.i64(5), blocks = a.i64(6), r = seq.numel(), c = parents.numel();
    if (!ints(parents, at::kLong, c) || !ints(seq, at::kInt, r) ||
        !ints(free, at::kInt, free.numel()) || !ints(left, at::kInt, 1) ||
        tables.scalar_type() != at::kInt || tables.dim() != 2 || tables.size(0) != r ||
        (tables.numel() > 0 && tables.stride(1) != 1) || !kv_block(block) || blocks < 0 ||
        parents.device() != seq.device() || tables.device() != seq.device() ||
        free.device() != seq.device() || left.device() != seq.device())
        Py_RETURN_NONE;
    RECORD_FUNCTION("ojasx_e8t::kv8_reorder", std::vector<c10::IValue>());
    Unlocked unlocked;
    const c10::DeviceGuard on_device(seq.device());
    const int64_t w = tables.size(1);
    Results all(Results::room(c * w, 4) + 3 * Results::room(c, 4),
                Results::room(blocks, 4) + Results::room(1, 4), seq);
    Tensor out[6];
    out[0] = all.next({c, w}, at::kInt);
    for (int i : {1, 4, 5}) out[i] = all.next({c}, at::kInt);
    all.second();
    out[2] = all.next({blocks}, at::kInt);
    out[3] = all.next({1}, at::kInt);
    size_t bytes = 0;
    check(ojx_kv8_reorder_workspace_bytes(r, c, w, block, blocks, &bytes),
          "kv8_reorder_workspace_bytes");
    const Tensor ws = workspace(bytes, seq);
    check(ojx_kv8_reorder((const int64_t*)data(parents), c, (const int32_t*)data(seq), r,
                          (const int32_t*)data(tables), tables.stride(0), w,
                          (const int32_t*)data(free), free.numel(), (const int32_t*)data(left), block,
                          blocks, (int32_t*)data(out[0]), (int32_t*)data(out[1]),
                          (int32_t*)data(out[2]), (int32_t*)data(out[3]), (int32_t*)data(out[4]),
                          (int32_t*)data(out[5]), data(ws), bytes, current_stream(seq.device())),
          "kv8_reorder");
    unlocked.lock();
    return tuple_of(out, 6);
    END_HANDLE_TH_ERRORS
}

// kv8_copy_blocks(caches, sources, targets): True; caches a list or tuple of triples of tensors or of
// objects that have them as k_codes, v_codes and scales
PyObject* kv8_copy_blocks(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 3, "kv8_copy_blocks");
    const Args a{argv, n};
    if (!(PyList_Check(argv[0]) || PyTuple_Check(argv[0])) || !all_plain(argv + 1, 2)) Py_RETURN_NONE;
    const Tensor sources = a.t(1), targets = a.t(2);
    const int64_t m = sources.numel(), layers = PySequence_Fast_GET_SIZE(argv[0]);
    if (layers == 0 || !ints(sources, at::kInt, m) || !ints(targets, at::kInt, m) ||
        sources.device() != targets.device())
        Py_RETURN_NONE;
    static PyObject* const names[] = {PyUnicode_InternFromString("k_codes"),
                                      PyUnicode_InternFromString("v_codes"),
                                      PyUnicode_InternFromString("scales")};
    std::vector<Tensor> parts;
    std::vector<ojx_kv8_storage> caches;
    parts.reserve(3 * layers);
    caches.reserve(layers);
    for (int64_t i = 0; i < layers; ++i) {
        PyObject* c = PySequence_Fast_GET_ITEM(argv[0], i);
        const bool triple = PyTuple_CheckExact(c);
        if (triple && PyTuple_GET_SIZE(c) != 3) Py_RETURN_NONE;
        for (int j = 0; j < 3; ++j) {
            PyObject* t = triple ? PyTuple_GET_ITEM(c, j) : PyObject_GetAttr(c, names[j]);
            if (!t) {
                PyErr_Clear();
                Py_RETURN_NONE;
            }
            const bool known = plain(t);
            if (known) parts.push_back(THPVariable_Unpack(t));
            if (!triple) Py_DECREF(t);
            if (!known) Py_RETURN_NONE;
        }
        const Tensor *t = &parts[3 * i], &k = t[0];
        if (k.dim() != 4 || !cache_ok(k, t[1], t[2], k.size(3)) || k.sizes() != parts[0].sizes() ||
            k.device() != sources.device())
            Py_RETURN_NONE;
        caches.push_back({(int8_t*)data(k), (int8_t*)data(t[1]), (float*)data(t[2])});
    }
    const Tensor& first = parts[0];
    RECORD_FUNCTION("ojasx_e8t::kv8_copy_blocks", std::vector<c10::IValue>());
    Unlocked unlocked;
    const c10::DeviceGuard on_device(first.device());
    check(ojx_kv8_copy_blocks(caches.data(), layers, first.size(0), first.size(1), first.size(2),
                              first.size(3), (const int32_t*)data(sources),
                              (const int32_t*)data(targets), m, current_stream(first.device())),
          "kv8_copy_blocks");
    for (const Tensor& t : parts) torch::autograd::impl::bump_version(t);
    unlocked.lock();
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// kv8_append(k, v, slots, k_codes, v_codes, scales): True
PyObject* kv8_append(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 6, "kv8_append");
    const Args a{argv, n};
    if (!all_plain(argv, 6)) Py_RETURN_NONE;
    const Tensor &k = a.t(0), &v = a.t(1), &slots = a.t(2), &kc = a.t(3), &vc = a.t(4),
                 &scales = a.t(5);
    const int dt = dtype_code(k.scalar_type());
    if (dt < 0 || v.scalar_type() != k.scalar_type() || k.dim() != 3 || k.sizes() != v.sizes() ||
        k.stride(2) != 1 || v.stride(2) != 1 || !cache_ok(kc, vc, scales, k.size(2)) ||
        k.size(1) != kc.size(1) || !ints(slots, at::kLong, k.size(0)) ||
        k.device() != kc.device() || v.device() != kc.device() || slots.device() != kc.device())
        Py_RETURN_NONE;
    RECORD_FUNCTION("ojasx_e8t::kv8_append", std::vector<c10::IValue>());
    Unlocked unlocked;
    const c10::DeviceGuard on_device(kc.device());
    check(ojx_kv8_append((int8_t*)data(kc), (int8_t*)data(vc), (float*)data(scales), kc.size(0),
                         kc.size(1), kc.size(2), k.size(2), data(k), k.stride(0), k.stride(1),
                         data(v), v.stride(0), v.stride(1), dt, (const int64_t*)data(slots),
                         k.size(0), current_stream(kc.device())),
          "kv8_append");
    for (const Tensor* t : {&kc, &vc, &scales}) torch::autograd::impl::bump_version(*t);
    unlocked.lock();
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// kv8_read(k_codes, v_codes, scales, blocks, head_dim, dtype): (k, v, scales), dtype a code of
// the C ABI
PyObject* kv8_read(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 6, "kv8_read");
    const Args a{argv, n};
    if (!all_plain(argv, 4)) Py_RETURN_NONE;
    const Tensor &kc = a.t(0), &vc = a.t(1), &scales = a.t(2), &blocks = a.t(3);
    const int64_t d = a.i64(4), m = blocks.numel();
    const int dt = (int)a.i64(5);
    if (dt < 0 || dt > 2 || !cache_ok(kc, vc, scales, d) || !ints(blocks, at::kInt, m) ||
        blocks.device() != kc.device())
        Py_RETURN_NONE;
    RECORD_FUNCTION("ojasx_e8t::kv8_read", std::vector<c10::IValue>());
    Unlocked unlocked;
    const c10::DeviceGuard on_device(kc.device());
    const at::ScalarType types[] = {at::kFloat, at::kHalf, at::kBFloat16};
    const auto opt = kc.options().dtype(types[dt]);
    Tensor out[] = {at::empty({m, kc.size(2), kc.size(1), d}, opt),
                    at::empty({m, kc.size(2), kc.size(1), d}, opt),
                    at::empty({m, kc.size(1), 2}, scales.options())};
    check(ojx_kv8_read((const int8_t*)data(kc), (const int8_t*)data(vc),
                       (const float*)data(scales), kc.size(0), kc.size(1), kc.size(2), d,
                       (const int32_t*)data(blocks), m, dt, data(out[0]), data(out[1]),
                       (float*)data(out[2]), current_stream(kc.device())),
          "kv8_read");
    unlocked.lock();
    return tuple_of(out, 3);
    END_HANDLE_TH_ERRORS
}

// kv8_attention(q, k_codes, v_codes, scales, tables, seq_lens, query_starts | None, scale, window,
// max_query_len, max_seq_len, return_lse): (out, lse | None)
PyObject* kv8_attention(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 12, "kv8_attention");
    const Args a{argv, n};
    if (!all_plain(argv, 6) || (argv[6] != Py_None && !plain(argv[6]))) Py_RETURN_NONE;
    const Tensor &q = a.t(0), &kc = a.t(1), &vc = a.t(2), &scales = a.t(3), &tables = a.t(4),
                 &lens = a.t(5);
    const Tensor starts = argv[6] == Py_None ? Tensor() : a.t(6);
    const int dt = dtype_code(q.scalar_type());
    const int64_t r = lens.numel(), window = a.i64(8), most = a.i64(9), longest = a.i64(10);
    const double scale = a.f64(7);
    if (dt < 0 || q.dim() != 3 || q.stride(2) != 1 || !cache_ok(kc, vc, scales, q.size(2)) ||
        !ints(lens, at::kInt, r) || (starts.defined() && !ints(starts, at::kInt, r + 1)) ||
        tables.scalar_type() != at::kInt || tables.dim() != 2 || tables.size(0) != r ||
        (tables.numel() > 0 && tables.stride(1) != 1) || q.device() != kc.device() ||
        tables.device() != kc.device() || lens.device() != kc.device() ||
        (starts.defined() && starts.device() != kc.device()) ||
        (c10::GradMode::is_enabled() && records(q)))
        Py_RETURN_NONE;
    RECORD_FUNCTION("ojasx_e8t::kv8_attention", std::vector<c10::IValue>());
    Unlocked unlocked;
    const c10::DeviceGuard on_device(kc.device());
    const int64_t t = q.size(0), heads = q.size(1), d = q.size(2);
    const bool with_lse = a.flag(11);
    Tensor out[] = {at::empty({t, heads, d}, q.options()),
                    with_lse ? at::empty({t, heads}, scales.options()) : Tensor()};
    size_t bytes = 0;
    check(ojx_kv8_attention_workspace_bytes(t, r, heads, kc.size(1), d, window, most, longest, dt,
                                            &bytes),
          "kv8_attention_workspace_bytes");
    const Tensor ws = workspace(bytes, q);
    check(ojx_kv8_attention(data(q), q.stride(0), q.stride(1), t, heads, dt,
                            (const int8_t*)data(kc), (const int8_t*)data(vc),
                            (const float*)data(scales), kc.size(0), kc.size(1), kc.size(2), d,
                            (const int32_t*)data(tables), tables.stride(0), tables.size(1),
                            (const int32_t*)data(lens), (const int32_t*)data(starts), r, most,
                            longest, (float)scale, window, data(out[0]),
                            with_lse ? (float*)data(out[1]) : nullptr, data(ws), bytes,
                            current_stream(kc.device())),
          "kv8_attention");
    unlocked.lock();
    return tuple_of(out, 2);
    END_HANDLE_TH_ERRORS
}

// Logits [..., V] as rows with neighbouring logits, without a copy; ids as they lie.
bool logits_ok(const Tensor& x, const Tensor& ids) {
    if (x.dim() < 1 || x.size(-1) < 1 || ids.scalar_type() != at::kLong || !ids.is_contiguous() ||
        ids.device() != x.device() || ids.dim() != x.dim() - 1)
        return false;
    for (int64_t i = 0; i < ids.dim(); ++i)
        if (ids.size(i) != x.size(i)) return false;
    return x.is_contiguous() || (x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= x.size(1));
}
int64_t row_stride(const Tensor& x) { return x.is_contiguous() ? x.size(-1) : x.stride(0); }

struct Logprobs {
    Tensor out[6];  // the op's results

    Logprobs(const Tensor& x, const Tensor& ids, int64_t top) {
        const c10::DeviceGuard on_device(x.device());
        const int dt = dtype_code(x.scalar_type());
        const int64_t v = x.size(-1), rows = ids.numel();
        std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end()), tops = shape,
                             two = shape;
        tops.push_back(top);
        two.push_back(2);
        Results all(3 * Results::room(rows, 4) + Results::room(2 * rows, 4),
                    Results::room(rows * top, 4) + Results::room(rows * top, 8), x);
        for (int i = 0; i < 3; ++i) out[i] = all.next(shape, at::kFloat);
        out[5] = all.next(two, at::kFloat);
        all.second();
        out[3] = all.next(tops, at::kFloat);
        out[4] = all.next(tops, at::kLong);
        size_t bytes = 0;
        check(ojx_token_logprobs_workspace_bytes(rows, v, top, dt, &bytes),
              "token_logprobs_workspace_bytes");
        const Tensor ws = workspace(bytes, x);
        check(ojx_token_logprobs(data(x), row_stride(x), rows, v, dt, (const int64_t*)data(ids),
                                 top, (float*)data(out[0]), (float*)data(out[1]),
                                 (float*)data(out[2]), (float*)data(out[5]), (float*)data(out[3]),
                                 (int64_t*)data(out[4]), data(ws), bytes,
                                 current_stream(x.device())),
              "token_logprobs");
    }
};

Tensor logprobs_gradient(const Tensor& x, const Tensor& ids, const Tensor& entropy,
                         const Tensor& stats, const Tensor& top_ids, const Tensor* g) {
    const c10::DeviceGuard on_device(x.device());
    Tensor gx = at::empty(x.sizes(), x.options());
    check(ojx_token_logprobs_bwd(data(x), row_stride(x), ids.numel(), x.size(-1),
                                 dtype_code(x.scalar_type()), (const int64_t*)data(ids),
                                 (const float*)data(entropy), (const float*)data(stats),
                                 top_ids.size(-1), (const int64_t*)data(top_ids),
                                 (const float*)data(g[0]), (const float*)data(g[1]),
                                 (const float*)data(g[2]), (const float*)data(g[3]), data(gx),
                                 current_stream(x.device())),
          "token_logprobs_bwd");
    return gx;
}

// The registered op's autograd formula as a node of the C++ engine: a Python one costs a call
// of some rows 30 us more than its kernels run.
struct RecordedLogprobs : torch::autograd::Function<RecordedLogprobs> {
    using Context = torch::autograd::AutogradContext;
    using List = torch::autograd::variable_list;

    static List forward(Context* ctx, const Tensor& x, const Tensor& ids, int64_t top) {
        Logprobs r(x, ids, top);
        ctx->save_for_backward({x, ids, r.out[1], r.out[5], r.out[4]});
        ctx->mark_non_differentiable({r.out[4]});
        ctx->set_materialize_grads(false);
        return {r.out[0], r.out[1], r.out[2], r.out[3], r.out[4]};
    }

    static List backward(Context* ctx, List grads) {
        const List saved = ctx->get_saved_variables();
        const Tensor& x = saved[0];
        Tensor g[4];
        bool any = false, known = plain_state() && plain(x), again = x.requires_grad();
        for (int i = 0; i < 4; ++i) {
            if (!grads[i].defined()) continue;
            any = true;
            again |= grads[i].requires_grad();
            known &= plain(grads[i]) && grads[i].device() == x.device() &&
                     grads[i].scalar_type() == at::kFloat;
            g[i] = grads[i];
        }
        if (!any) return {Tensor(), Tensor(), Tensor()};
        again &= c10::GradMode::is_enabled();
        const at::AutoGradMode off(false);
        Tensor gx;
        if (known) {
            for (Tensor& t : g)
                if (t.defined()) t = t.contiguous();
            RECORD_FUNCTION("ojasx_e8t::token_logprobs_bwd", std::vector<c10::IValue>());
            gx = logprobs_gradient(x, saved[1], saved[2], saved[3], saved[4], g);
        } else {
            static const auto op =
                c10::Dispatcher::singleton().findSchemaOrThrow("ojasx_e8t::token_logprobs_bwd", "");
            std::vector<c10::IValue> stack(saved.begin(), saved.end());
            for (const Tensor& t : g) stack.push_back(t.defined() ? c10::IValue(t) : c10::IValue());
            op.callBoxed(stack);
            gx = stack[0].toTensor();
        }
        if (again) {  // a graph of this gradient was asked for, which it has none of
            const at::AutoGradMode on(true);
            gx = gx.detach();
            gx.set_requires_grad(true);
            const auto refuse = std::make_shared<torch::autograd::DelayedError>(
                "the gradient of token_logprobs cannot be differentiated", 1);
            gx = (*refuse)({gx})[0];
        }
        return {gx, Tensor(), Tensor()};
    }
};

// Whether token_logprobs(logits, ids, top_k) is a call on tensors as the kernels take them
bool logprobs_ok(PyObject* const* argv, const Args& a) {
    if (!all_plain(argv, 2)) return false;
    const int64_t top = a.i64(2);
    return dtype_code(a.t(0).scalar_type()) >= 0 && logits_ok(a.t(0), a.t(1)) && top >= 0 &&
           top <= 64 && top <= a.t(0).size(-1);
}

// token_logprobs(logits, ids, top_k): the op's results
PyObject* token_logprobs(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 3, "token_logprobs");
    const Args a{argv, n};
    if (!logprobs_ok(argv, a) || (c10::GradMode::is_enabled() && records(a.t(0)))) Py_RETURN_NONE;
    const int64_t top = a.i64(2);
    RECORD_FUNCTION("ojasx_e8t::token_logprobs", std::vector<c10::IValue>());
    Unlocked unlocked;
    Logprobs r(a.t(0), a.t(1), top);
    unlocked.lock();
    return tuple_of(r.out, 6);
    END_HANDLE_TH_ERRORS
}

// token_logprobs_recorded(logits, ids, top_k): the op's results but the last, for autograd
PyObject* token_logprobs_recorded(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 3, "token_logprobs_recorded");
    const Args a{argv, n};
    if (!logprobs_ok(argv, a)) Py_RETURN_NONE;
    const int64_t top = a.i64(2);
    RECORD_FUNCTION("ojasx_e8t::token_logprobs", std::vector<c10::IValue>());
    Unlocked unlocked;
    auto out = RecordedLogprobs::apply(a.t(0), a.t(1), top);
    unlocked.lock();
    return tuple_of(out.data(), 5);
    END_HANDLE_TH_ERRORS
}

// Heads [tokens, heads, d] or [batch, tokens, heads, d] as the kernels take them, of q's sizes.
bool heads_ok(const Tensor& x, const Tensor& q) {
    const int64_t n = q.dim();
    return x.dim() == n && x.scalar_type() == q.scalar_type() && x.device() == q.device() &&
           x.size(0) == q.size(0) && (n == 3 || x.size(1) == q.size(1)) &&
           x.size(n - 1) == q.size(n - 1) && x.stride(n - 1) == 1;
}

bool rotation_ok(const Tensor& positions, const Tensor& rates, const Tensor& q) {
    const int64_t n = q.dim(), tokens = q.size(n - 3);
    return (positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong) &&
           positions.device() == q.device() && rates.device() == q.device() &&
           ((positions.dim() == 1 && positions.size(0) == tokens) ||
            (positions.dim() == 2 && n == 4 && positions.size(0) == q.size(0) &&
             positions.size(1) == tokens)) &&
           rates.scalar_type() == at::kLong && rates.dim() == 1 && rates.is_contiguous() &&
           rates.numel() >= 1 && 2 * rates.numel() <= q.size(n - 1);
}

ojx_rotation rotation_of(const Tensor& positions, const Tensor& rates, double gain, bool interleaved,
                         bool inverse) {
    ojx_rotation r;
    r.rates = (const int64_t*)data(rates);
    r.pairs = rates.numel();
    r.positions = data(positions);
    r.positions64 = positions.scalar_type() == at::kLong;
    r.interleaved = interleaved;
    r.gain = (float)gain;
    r.inverse = inverse;
    return r;
}

// As x lies, where that leaves a head's elements neighbours (not of heads that overlap in x).
Tensor heads_like(const Tensor& x) {
    Tensor y = at::empty_like(x);
    return y.stride(-1) == 1 ? y : at::empty_like(x, at::MemoryFormat::Contiguous);
}

// q and k (undefined: none) rotated; what heads_ok and rotation_ok took.
void rotate_into(const Tensor& q, const Tensor& k, const Tensor& positions, const ojx_rotation& r,
                 Tensor* out) {
    const c10::DeviceGuard on_device(q.device());
    const int64_t n = q.dim();
    ojx_rotary_rows rows[2];
    for (int i = 0; i < 2; ++i) {
        const Tensor& x = i ? k : q;
        if (!x.defined()) continue;
        const Tensor y = out[i] = heads_like(x);
        rows[i] = {data(x), data(y), n == 4 ? x.stride(0) : 0, x.stride(n - 3), x.stride(n - 2),
                   n == 4 ? y.stride(0) : 0, y.stride(n - 3), y.stride(n - 2), x.size(n - 2)};
    }
    check(ojx_rotary(&rows[0], k.defined() ? &rows[1] : nullptr, n == 4 ? q.size(0) : 1, q.size(n - 3),
                     q.size(n - 1), dtype_code(q.scalar_type()), &r,
                     positions.dim() == 2 ? positions.stride(0) : 0,
                     positions.stride(positions.dim() - 1), current_stream(q.device())),
          "rotary");
}

// The registered op's autograd formula as a node of the C++ engine (see RecordedLogprobs).
struct RecordedRotary : torch::autograd::Function<RecordedRotary> {
    using Context = torch::autograd::AutogradContext;
    using List = torch::autograd::variable_list;

    static List forward(Context* ctx, const Tensor& q, const std::optional<Tensor>& keys,
                        const Tensor& positions, const Tensor& rates, double gain, bool interleaved, bool inverse) {
        ctx->save_for_backward({positions, rates});
        ctx->saved_data["gain"] = gain;
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["inverse"] = inverse;
        ctx->set_materialize_grads(false);
        const Tensor k = keys ? *keys : Tensor();
        Tensor out[2];
        rotate_into(q, k, positions, rotation_of(positions, rates, gain, interleaved, inverse), out);
        if (!k.defined()) return {out[0]};
        return {out[0], out[1]};
    }

    static List backward(Context* ctx, List grads) {
        const List saved = ctx->get_saved_variables();
        const Tensor &positions = saved[0], &rates = saved[1];
        const double gain = ctx->saved_data["gain"].toDouble();
        const bool interleaved = ctx->saved_data["interleaved"].toBool();
        const bool inverse = !ctx->saved_data["inverse"].toBool();
        // those that came for what needs one, in order: queries, keys
        Tensor g[2];
        int n = 0, from[2] = {0, 0};
        for (int i = 0; i < (int)grads.size() && i < 2; ++i)
            if (grads[i].defined() && ctx->needs_input_grad(i)) {
                from[n] = i;
                g[n++] = grads[i];
            }
        List result(7);
        if (n == 0) return result;
        bool known = plain_state() && plain(positions) && plain(rates), again = false;
        for (int i = 0; i < n; ++i) {
            known &= plain(g[i]);
            again |= g[i].requires_grad();
        }
        Tensor out[2];
        if (known && !(again && c10::GradMode::is_enabled())) {
            const at::AutoGradMode off(false);
            for (int i = 0; i < n; ++i)
                if (g[i].stride(-1) != 1) g[i] = g[i].contiguous();
            known = rotation_ok(positions, rates, g[0]) && (n == 1 || heads_ok(g[1], g[0]));
            if (known) {
                RECORD_FUNCTION("ojasx_e8t::rotary", std::vector<c10::IValue>());
                rotate_into(g[0], g[1], positions,
                            rotation_of(positions, rates, gain, interleaved, inverse), out);
            }
        } else {
            known = false;
        }
        if (!known) {  // the registered op, which records a gradient of this one where asked
            static const auto op =
                c10::Dispatcher::singleton().findSchemaOrThrow("ojasx_e8t::rotary", "");
            std::vector<c10::IValue> stack{g[0], n > 1 ? c10::IValue(g[1]) : c10::IValue(), positions,
                                           rates, gain, interleaved, inverse};
            op.callBoxed(stack);
            for (int i = 0; i < n; ++i) out[i] = stack[i].toTensor();
        }
        for (int i = 0; i < n; ++i) result[from[i]] = out[i];
        return result;
    }
};

// kv8_rotate_append(q, k, v, positions, slots, rates, gain, interleaved, k_codes, v_codes, scales):
// q rotated
PyObject* kv8_rotate_append(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 11, "kv8_rotate_append");
    const Args a{argv, n};
    if (!all_plain(argv, 6) || !plain(argv[8]) || !plain(argv[9]) || !plain(argv[10])) Py_RETURN_NONE;
    const Tensor &q = a.t(0), &k = a.t(1), &v = a.t(2), &positions = a.t(3), &slots = a.t(4),
                 &rates = a.t(5), &kc = a.t(8), &vc = a.t(9), &scales = a.t(10);
    const int dt = dtype_code(k.scalar_type());
    if (dt < 0 || v.scalar_type() != k.scalar_type() || k.dim() != 3 || k.sizes() != v.sizes() ||
        k.stride(2) != 1 || v.stride(2) != 1 || !cache_ok(kc, vc, scales, k.size(2)) ||
        k.size(1) != kc.size(1) || !ints(slots, at::kLong, k.size(0)) ||
        k.device() != kc.device() || v.device() != kc.device() || slots.device() != kc.device() ||
        !heads_ok(q, k) || !rotation_ok(positions, rates, q) ||
        !positions.is_contiguous() || (c10::GradMode::is_enabled() && records(q)))
        Py_RETURN_NONE;
    const ojx_rotation r = rotation_of(positions, rates, a.f64(6), a.truth(7), false);
    RECORD_FUNCTION("ojasx_e8t::kv8_rotate_append", std::vector<c10::IValue>());
    Unlocked unlocked;
    const c10::DeviceGuard on_device(kc.device());
    Tensor out = heads_like(q);
    const ojx_rotary_rows rows = {data(q), data(out), 0, q.stride(0), q.stride(1),
                                  0, out.stride(0), out.stride(1), q.size(1)};
    check(ojx_kv8_rotate_append((int8_t*)data(kc), (int8_t*)data(vc), (float*)data(scales), kc.size(0),
                                kc.size(1), kc.size(2), k.size(2), data(k), k.stride(0), k.stride(1),
                                data(v), v.stride(0), v.stride(1), dt, (const int64_t*)data(slots),
                                k.size(0), &rows, &r, current_stream(kc.device())),
          "kv8_rotate_append");
    for (const Tensor* t : {&kc, &vc, &scales}) torch::autograd::impl::bump_version(*t);
    unlocked.lock();
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// Whether rotary(q, k | None, positions, rates, gain, interleaved, inverse) is a call on tensors as
// the kernels take them
bool rotary_ok(PyObject* const* argv, const Args& a) {
    if (!plain_state() || !plain(argv[0]) || (argv[1] != Py_None && !plain(argv[1])) ||
        !plain(argv[2]) || !plain(argv[3]))
        return false;
    const Tensor& q = a.t(0);
    return dtype_code(q.scalar_type()) >= 0 && (q.dim() == 3 || q.dim() == 4) && heads_ok(q, q) &&
           rotation_ok(a.t(2), a.t(3), q) && (argv[1] == Py_None || heads_ok(a.t(1), q));
}

// rotary(...): (q, k | None)
PyObject* rotary(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 7, "rotary");
    const Args a{argv, n};
    if (!rotary_ok(argv, a)) Py_RETURN_NONE;
    const Tensor q = a.t(0), k = argv[1] == Py_None ? Tensor() : a.t(1);
    if (c10::GradMode::is_enabled() && (records(q) || records(k))) Py_RETURN_NONE;
    const ojx_rotation r = rotation_of(a.t(2), a.t(3), a.f64(4), a.truth(5), a.truth(6));
    RECORD_FUNCTION("ojasx_e8t::rotary", std::vector<c10::IValue>());
    Unlocked unlocked;
    Tensor out[2];
    rotate_into(q, k, a.t(2), r, out);
    unlocked.lock();
    return tuple_of(out, 2);
    END_HANDLE_TH_ERRORS
}

// rotary_recorded(...): the same for autograd
PyObject* rotary_recorded(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 7, "rotary_recorded");
    const Args a{argv, n};
    if (!rotary_ok(argv, a)) Py_RETURN_NONE;
    const Tensor q = a.t(0), k = argv[1] == Py_None ? Tensor() : a.t(1);
    const double gain = a.f64(4);
    const bool interleaved = a.truth(5), inverse = a.truth(6);
    RECORD_FUNCTION("ojasx_e8t::rotary", std::vector<c10::IValue>());
    Unlocked unlocked;
    const std::optional<Tensor> keys = k.defined() ? std::optional<Tensor>(k) : std::nullopt;
    auto got = RecordedRotary::apply(q, keys, a.t(2), a.t(3), gain, interleaved, inverse);
    unlocked.lock();
    Tensor out[2] = {got[0], k.defined() ? got[1] : Tensor()};
    return tuple_of(out, 2);
    END_HANDLE_TH_ERRORS
}

// beam_select(logits, scores, num, finished | None, pad_id): the op's results
PyObject* beam_select(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 5, "beam_select");
    const Args a{argv, n};
    if (!all_plain(argv, 2) || (argv[3] != Py_None && !plain(argv[3]))) Py_RETURN_NONE;
    const Tensor &x = a.t(0), &scores = a.t(1);
    const Tensor done = argv[3] == Py_None ? Tensor() : a.t(3);
    const int64_t num = a.i64(2), pad = a.i64(4);
    const int dt = dtype_code(x.scalar_type());
    if (dt < 0 || x.dim() != 3 || x.size(2) < 1 || x.size(1) < 1 || x.size(1) > 64 || num < 1 || num > 64 ||
        num > x.size(1) * x.size(2) || x.stride(2) != 1 || x.stride(1) < x.size(2) ||
        (x.size(0) > 1 && x.stride(0) != x.size(1) * x.stride(1)) ||
        scores.scalar_type() != at::kFloat || scores.dim() != 2 || scores.size(0) != x.size(0) ||
        scores.size(1) != x.size(1) || !scores.is_contiguous() || scores.device() != x.device() ||
        (done.defined() && (done.scalar_type() != at::kBool || done.sizes() != scores.sizes() ||
                            !done.is_contiguous() || done.device() != x.device() || pad < 0 ||
                            pad >= x.size(2))) ||
        (c10::GradMode::is_enabled() && (records(x) || records(scores))))
        Py_RETURN_NONE;
    RECORD_FUNCTION("ojasx_e8t::beam_select", std::vector<c10::IValue>());
    Unlocked unlocked;
    const c10::DeviceGuard on_device(x.device());
    const int64_t g = x.size(0), k = x.size(1), v = x.size(2);
    // 20 bytes a result: side by side whatever their number
    Results all(Results::room(g * num, 4) + 2 * Results::room(g * num, 8), 0, x);
    Tensor out[] = {all.next({g, num}, at::kFloat), all.next({g, num}, at::kLong),
                    all.next({g, num}, at::kLong)};
    size_t bytes = 0;
    check(ojx_beam_select_workspace_bytes(g, k, v, num, dt, &bytes), "beam_select_workspace_bytes");
    const Tensor ws = workspace(bytes, x);
    check(ojx_beam_select(data(x), x.stride(1), g, k, v, dt, (const float*)data(scores),
                          (const uint8_t*)data(done), pad, num, (float*)data(out[0]),
                          (int64_t*)data(out[1]), (int64_t*)data(out[2]), data(ws), bytes,
                          current_stream(x.device())),
          "beam_select");
    unlocked.lock();
    return tuple_of(out, 3);
    END_HANDLE_TH_ERRORS
}

// plain(tensor, ...): whether a Function over these tensors is plain eager work (grad aside)
PyObject* is_plain(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!plain_state()) Py_RETURN_FALSE;
    for (Py_ssize_t i = 0; i < n; ++i)
        if (argv[i] != Py_None && !plain(argv[i])) Py_RETURN_FALSE;
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"linear", (PyCFunction)(void*)linear, METH_FASTCALL, nullptr},
    {"linear_bwd", (PyCFunction)(void*)linear_bwd, METH_FASTCALL, nullptr},
    {"linear_lora", (PyCFunction)(void*)linear_lora, METH_FASTCALL, nullptr},
    {"linear_lora_bwd", (PyCFunction)(void*)linear_lora_bwd, METH_FASTCALL, nullptr},
    {"encode", (PyCFunction)(void*)encode, METH_FASTCALL, nullptr},
    {"decode", (PyCFunction)(void*)decode, METH_FASTCALL, nullptr},
    {"kv8_plan", (PyCFunction)(void*)kv8_plan, METH_FASTCALL, nullptr},
    {"kv8_reorder", (PyCFunction)(void*)kv8_reorder, METH_FASTCALL, nullptr},
    {"kv8_copy_blocks", (PyCFunction)(void*)kv8_copy_blocks, METH_FASTCALL, nullptr},
    {"kv8_append", (PyCFunction)(void*)kv8_append, METH_FASTCALL, nullptr},
    {"kv8_read", (PyCFunction)(void*)kv8_read, METH_FASTCALL, nullptr},
    {"kv8_attention", (PyCFunction)(void*)kv8_attention, METH_FASTCALL, nullptr},
    {"token_logprobs", (PyCFunction)(void*)token_logprobs, METH_FASTCALL, nullptr},
    {"token_logprobs_recorded", (PyCFunction)(void*)token_logprobs_recorded, METH_FASTCALL,
     nullptr},
    {"kv8_rotate_append", (PyCFunction)(void*)kv8_rotate_append, METH_FASTCALL, nullptr},
    {"rotary", (PyCFunction)(void*)rotary, METH_FASTCALL, nullptr},
    {"rotary_recorded", (PyCFunction)(void*)rotary_recorded, METH_FASTCALL, nullptr},
    {"beam_select", (PyCFunction)(void*)beam_select, METH_FASTCALL, nullptr},
    {"is_plain", (PyCFunction)(void*)is_plain, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_ojasx_eager", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ojasx_eager(void) { return PyModule_Create(&kModule); }
