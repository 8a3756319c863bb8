// Native call path of the ordinary calls of the Python API.
//
// Every function here takes a call whose tensors the kernels can use as they
// are, allocates the results, launches through the C ABI
// (include/smooth_attn_amd.h) on torch's current stream and returns; for any
// other call (a wrong or unusual argument, a tensor that must be copied or
// padded first, a tensor subclass, a functorch transform, tracing, a dispatch
// or function mode, forward-mode gradients) it returns None and launches
// nothing, and the Python path of smooth_attn/kernels.py handles or refuses
// that call as it always did.
//
// Why: small calls are bound by the host.  Per pass, Python path -> this one,
// same kernels: causal normalisation forward [2,8,512,512] 9.2 -> 4.4 us,
// prefill [1,32/8,512,128] 18.0 -> 11.4, a decode step (append + attention) of
// 8 sequences 44 -> 22, training steps [2,16,1023,1023] normalisation 95 -> 48
// and [4,12,1024,64] attention 154 -> 89, each now bound by its kernels.  The
// autograd nodes are C++, so the backward needs no interpreter on the autograd
// thread.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/version.h>

#include <array>
#include <cmath>
#include <cstring>
#include <memory>
#include <optional>
#include <stdexcept>
#include <string>
#include <unordered_set>
#include <vector>

#include "smooth_attn_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---------------------------------------------------------------------------
// The C ABI, bound once to the addresses of the loaded library.
// ---------------------------------------------------------------------------
struct Abi {
    decltype(&sa_status_string) status_string = nullptr;
    decltype(&sa_norm_fwd) norm_fwd = nullptr;
    decltype(&sa_norm_bwd) norm_bwd = nullptr;
    decltype(&sa_flash_fwd) flash_fwd = nullptr;
    decltype(&sa_flash_bwd_ws) flash_bwd_ws = nullptr;
    decltype(&sa_flash_bwd_workspace_size) flash_bwd_workspace_size = nullptr;
    decltype(&sa_paged_decode) paged_decode = nullptr;
    decltype(&sa_paged_decode_workspace_size) paged_decode_workspace_size = nullptr;
    decltype(&sa_paged_kv_append_lens) paged_kv_append_lens = nullptr;
    decltype(&sa_qk_norm_rope_fwd) qk_norm_rope_fwd = nullptr;
    decltype(&sa_qk_norm_rope_bwd) qk_norm_rope_bwd = nullptr;
    decltype(&sa_qk_norm_rope_bwd_workspace_size) qk_norm_rope_bwd_workspace_size = nullptr;
    decltype(&sa_paged_qk_norm_rope_append) paged_qk_norm_rope_append = nullptr;
    decltype(&sa_paged_reserve) paged_reserve = nullptr;
    decltype(&sa_paged_release) paged_release = nullptr;
    decltype(&sa_paged_key_bounds) paged_key_bounds = nullptr;
    decltype(&sa_paged_select_pages) paged_select_pages = nullptr;
    decltype(&sa_paged_select_workspace_size) paged_select_workspace_size = nullptr;
    decltype(&sa_paged_sparse_decode) paged_sparse_decode = nullptr;
    decltype(&sa_paged_sparse_workspace_size) paged_sparse_workspace_size = nullptr;
} abi;

template <typename F>
bool bind_one(PyObject* table, const char* name, F& fn) {
    PyObject* v = PyDict_GetItemString(table, name);
    if (v == nullptr) {
        PyErr_Format(PyExc_KeyError, "no address for %s", name);
        return false;
    }
    fn = reinterpret_cast<F>(PyLong_AsVoidPtr(v));
    return !PyErr_Occurred();
}

// bind({name: address}): call once, before anything else.
PyObject* py_bind(PyObject*, PyObject* table) {
    if (!PyDict_Check(table)) {
        PyErr_SetString(PyExc_TypeError, "bind() takes a dict of addresses");
        return nullptr;
    }
    if (!bind_one(table, "sa_status_string", abi.status_string) || !bind_one(table, "sa_norm_fwd", abi.norm_fwd) ||
        !bind_one(table, "sa_norm_bwd", abi.norm_bwd) || !bind_one(table, "sa_flash_fwd", abi.flash_fwd) ||
        !bind_one(table, "sa_flash_bwd_ws", abi.flash_bwd_ws) ||
        !bind_one(table, "sa_flash_bwd_workspace_size", abi.flash_bwd_workspace_size) ||
        !bind_one(table, "sa_paged_decode", abi.paged_decode) ||
        !bind_one(table, "sa_paged_decode_workspace_size", abi.paged_decode_workspace_size) ||
        !bind_one(table, "sa_paged_kv_append_lens", abi.paged_kv_append_lens) ||
        !bind_one(table, "sa_qk_norm_rope_fwd", abi.qk_norm_rope_fwd) ||
        !bind_one(table, "sa_qk_norm_rope_bwd", abi.qk_norm_rope_bwd) ||
        !bind_one(table, "sa_qk_norm_rope_bwd_workspace_size", abi.qk_norm_rope_bwd_workspace_size) ||
        !bind_one(table, "sa_paged_qk_norm_rope_append", abi.paged_qk_norm_rope_append) ||
        !bind_one(table, "sa_paged_reserve", abi.paged_reserve) ||
        !bind_one(table, "sa_paged_release", abi.paged_release) ||
        !bind_one(table, "sa_paged_key_bounds", abi.paged_key_bounds) ||
        !bind_one(table, "sa_paged_select_pages", abi.paged_select_pages) ||
        !bind_one(table, "sa_paged_select_workspace_size", abi.paged_select_workspace_size) ||
        !bind_one(table, "sa_paged_sparse_decode", abi.paged_sparse_decode) ||
        !bind_one(table, "sa_paged_sparse_workspace_size", abi.paged_sparse_workspace_size))
        return nullptr;
    Py_RETURN_NONE;
}

void check(int status, const char* what) {
    if (status != 0)
        throw std::runtime_error(std::string(what) + " failed (status " + std::to_string(status) +
                                 "): " + abi.status_string(status));
}

// Lets other Python threads run while a call allocates and launches, which may
// wait: for a full queue, a first load of the kernel's code, an allocation that
// frees cached memory first.  Gives the interpreter back before an exception
// leaves its scope.
struct NoGil {
    PyThreadState* state = PyEval_SaveThread();
    NoGil() = default;
    NoGil(const NoGil&) = delete;
    NoGil& operator=(const NoGil&) = delete;
    ~NoGil() { PyEval_RestoreThread(state); }
};

// ---------------------------------------------------------------------------
// Which calls are ordinary.
// ---------------------------------------------------------------------------
// No interposer of any kind between this call and the device.
bool plain_mode() {
    return !torch::jit::tracer::isTracing() && !at::impl::torch_function_mode_enabled() &&
           !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
           !c10::impl::tls_local_dispatch_key_set().included_.has(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

// A dense tensor on a GPU, of exactly torch.Tensor or torch.nn.Parameter, and
// no wrapper or lazily conjugated / negated view.
const Tensor* plain(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    static const c10::DispatchKeySet wrappers(
        {c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Batched,
         c10::DispatchKey::Functionalize, c10::DispatchKey::Python, c10::DispatchKey::Fake,
         c10::DispatchKey::ZeroTensor, c10::DispatchKey::Conjugate, c10::DispatchKey::Negative,
         c10::DispatchKey::Quantized});
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() ||
        t.key_set().has_any(wrappers) || t._fw_grad(0).defined())
        return nullptr;
    return &t;
}

int code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return SA_F32;
        case at::kHalf: return SA_F16;
        case at::kBFloat16: return SA_BF16;
        case at::kFloat8_e4m3fn: return SA_FP8_E4M3FN;
        default: return -1;
    }
}
bool float_code(int c) { return c == SA_F32 || c == SA_F16 || c == SA_BF16; }

bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// kernels.py's _flash_operand: (b, h, t) strides that are multiples of 16
// bytes, unit stride along D, a 16-byte aligned base, rows at most 16 MiB
// apart.
bool operand_ok(const Tensor& t) {
    const int64_t es = t.element_size(), a = 16 / es;
    const auto s = t.strides();
    if (s.back() != 1 || !aligned16(t) || s[s.size() - 2] * es > (int64_t(1) << 24)) return false;
    for (size_t i = 0; i + 1 < s.size(); ++i)
        if (s[i] % a != 0) return false;
    return true;
}

sa_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
const int64_t* strides(const Tensor& t) { return t.strides().data(); }

bool as_double(PyObject* o, double& v) {
    v = PyFloat_Check(o) ? PyFloat_AS_DOUBLE(o) : PyLong_CheckExact(o) ? PyLong_AsDouble(o) : NAN;
    if (PyErr_Occurred()) PyErr_Clear();
    return std::isfinite(v);
}
// A non-negative int (not a bool or an int-like object) below 2^31.
bool as_int(PyObject* o, int& v) {
    if (!PyLong_CheckExact(o)) return false;
    int over = 0;
    const long x = PyLong_AsLongAndOverflow(o, &over);
    if (over != 0 || x < 0 || x > INT32_MAX) return false;
    v = static_cast<int>(x);
    return true;
}

// ---------------------------------------------------------------------------
// Normalisation.
// ---------------------------------------------------------------------------
constexpr int64_t kMaxCols = 8192;  // kernels.py MAX_ROW_COLS

struct Family {
    double alpha, theta;
    int power;
    bool parse(PyObject* a, PyObject* t, PyObject* p) {
        return as_double(a, alpha) && as_double(t, theta) && as_int(p, power) && power >= 1 && power <= 3;
    }
};

// Rows of contiguous x into contiguous y.
void norm_fwd(const Tensor& x, const Tensor& y, bool causal, const Family& f) {
    const int64_t cols = x.size(-1);
    const c10::DeviceGuard guard(x.device());
    check(abi.norm_fwd(x.data_ptr(), y.data_ptr(), x.numel() / cols, cols, cols, cols, code_of(x.scalar_type()), causal,
                       static_cast<float>(f.alpha), static_cast<float>(f.theta), f.power, stream_of(x)),
          "sa_norm_fwd");
}

bool norm_input_ok(const Tensor& x, bool causal) {
    return float_code(code_of(x.scalar_type())) && (causal ? x.dim() >= 2 : x.dim() == 2) && x.numel() > 0 &&
           x.is_contiguous() && x.size(-1) <= kMaxCols && (!causal || x.size(-1) == x.size(-2));
}

// norm_out(out, x, causal, alpha, theta, power) -> bool: whether it ran.
PyObject* py_norm_out(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Family f;
    const Tensor *out, *x;
    if (n != 6 || !plain_mode() || !(out = plain(a[0])) || !(x = plain(a[1])) || !f.parse(a[3], a[4], a[5]))
        Py_RETURN_FALSE;
    const bool causal = a[2] == Py_True;
    if (!norm_input_ok(*x, causal) || out->scalar_type() != x->scalar_type() || out->device() != x->device() ||
        out->sizes() != x->sizes() || !out->is_contiguous())
        Py_RETURN_FALSE;
    {
        const NoGil released;
        norm_fwd(*x, *out, causal, f);
    }
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

struct CausalNorm : public torch::autograd::Function<CausalNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, double alpha, double theta, int64_t power) {
        const Family f{alpha, theta, static_cast<int>(power)};
        Tensor y = at::empty_like(x);
        norm_fwd(x, y, true, f);
        ctx->save_for_backward({x});
        ctx->saved_data["alpha"] = alpha;
        ctx->saved_data["theta"] = theta;
        ctx->saved_data["power"] = power;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (!ctx->needs_input_grad(0)) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const Tensor saved = ctx->get_saved_variables()[0];
        Tensor g = grads[0];
        TORCH_CHECK_VALUE(g.is_cuda() && g.device() == saved.device(),
                          "grad_output must live on the same CUDA device as x");
        TORCH_CHECK_VALUE(float_code(code_of(saved.scalar_type())) && saved.sizes() == g.sizes(),
                          "the saved x must have grad_output's shape and a dtype of the fused kernels");
        const int64_t cols = saved.size(-1);
        // (unpack hooks may hand back another layout or type than forward saved)
        const bool as_saved = saved.is_contiguous();
        Tensor x = as_saved ? saved : saved.reshape({-1, cols});
        if (!as_saved && (x.stride(1) != 1 || x.stride(0) < cols)) x = x.contiguous();
        if (g.scalar_type() != at::kFloat && g.scalar_type() != x.scalar_type()) g = g.to(at::kFloat);
        g = g.contiguous();
        Tensor dx = at::empty_like(x);
        const c10::DeviceGuard guard(x.device());
        check(abi.norm_bwd(x.data_ptr(), g.data_ptr(), dx.data_ptr(), x.numel() / cols, cols, x.stride(-2), cols,
                           dx.stride(-2),
                           code_of(x.scalar_type()), code_of(g.scalar_type()), 1,
                           static_cast<float>(ctx->saved_data["alpha"].toDouble()),
                           static_cast<float>(ctx->saved_data["theta"].toDouble()),
                           static_cast<int>(ctx->saved_data["power"].toInt()), stream_of(x)),
              "sa_norm_bwd");
        return {as_saved ? dx : dx.view(saved.sizes()), Tensor(), Tensor(), Tensor()};
    }
};

// causal_norm(x, alpha, theta, power) -> y or None.
PyObject* py_causal_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Family f;
    const Tensor* x;
    if (n != 4 || !plain_mode() || !(x = plain(a[0])) || !f.parse(a[1], a[2], a[3]) || !norm_input_ok(*x, true))
        Py_RETURN_NONE;
    Tensor y;
    {
        const NoGil released;
        if (at::GradMode::is_enabled() && x->requires_grad()) {
            y = CausalNorm::apply(*x, f.alpha, f.theta, static_cast<int64_t>(f.power));
        } else {
            y = at::empty_like(*x);
            norm_fwd(*x, y, true, f);
        }
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------
// Fused attention.
// ---------------------------------------------------------------------------
struct FlashCall {
    double scale;
    int window;
    bool exact;
};

// Whether the kernels take q, k and v as they are (kernels.py's checks).
bool flash_ok(const Tensor& q, const Tensor& k, const Tensor& v) {
    if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || q.numel() == 0 || k.numel() == 0) return false;
    const int code = code_of(q.scalar_type());
    if (!float_code(code) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) return false;
    if (k.device() != q.device() || v.device() != q.device()) return false;
    const int64_t D = q.size(3), Hkv = k.size(1);
    if (k.size(0) != q.size(0) || k.size(2) != q.size(2) || k.size(3) != D || v.sizes() != k.sizes() ||
        q.size(1) % Hkv != 0)
        return false;
    if (D > 512 || D % (code == SA_F32 ? 4 : 8) != 0 || q.size(0) > INT32_MAX || q.size(1) > INT32_MAX ||
        q.size(2) > INT32_MAX)
        return false;
    return operand_ok(q) && operand_ok(k) && operand_ok(v);
}

int dim(const Tensor& t, int i) { return static_cast<int>(t.size(i)); }

void flash_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const FlashCall& c, Tensor& o, Tensor& row_sums) {
    o = at::empty_like(q);
    if (o.stride(-1) != 1) o = at::empty(q.sizes(), q.options());
    row_sums = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    const c10::DeviceGuard guard(q.device());
    check(abi.flash_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), row_sums.data_ptr<float>(), dim(q, 0),
                        dim(q, 1), dim(k, 1), dim(q, 2), dim(q, 3), strides(q), strides(k), strides(v), strides(o),
                        static_cast<float>(c.scale), c.window, c.exact, code_of(q.scalar_type()), stream_of(q)),
          "sa_flash_fwd");
}

// What backward reads: q, k, v, o and the row sums as forward saved them, or
// as unpack hooks hand them back.
void check_saved(const variable_list& saved, const Tensor& grad) {
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &o = saved[3], &row_sums = saved[4];
    for (const Tensor* t : {&q, &k, &v, &o, &row_sums, &grad})
        TORCH_CHECK_VALUE(t->is_cuda() && t->device() == q.device(),
                          "attention tensors must live on the same CUDA device as q");
    TORCH_CHECK_VALUE(float_code(code_of(q.scalar_type())) && k.scalar_type() == q.scalar_type() &&
                          v.scalar_type() == q.scalar_type(),
                      "fused attention expects bf16, fp16 or fp32 q/k/v of one dtype, got ", q.scalar_type(), "/",
                      k.scalar_type(), "/", v.scalar_type());
    TORCH_CHECK_VALUE(o.scalar_type() == q.scalar_type() && row_sums.scalar_type() == at::kFloat,
                      "the saved output must have q's dtype and the saved row sums fp32");
    TORCH_CHECK_VALUE(q.sizes() == grad.sizes() && o.sizes() == grad.sizes() && k.dim() == 4 && v.sizes() == k.sizes() &&
                          k.size(0) == q.size(0) && k.size(1) > 0 && q.size(1) % k.size(1) == 0 &&
                          k.size(2) == q.size(2) && k.size(3) == q.size(3) &&
                          row_sums.sizes() == q.sizes().slice(0, 3),
                      "the saved attention tensors must have the shapes that forward saved");
}

struct Flash : public torch::autograd::Function<Flash> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, double scale,
                          int64_t window, bool exact) {
        Tensor o, row_sums;
        flash_fwd(q, k, v, FlashCall{scale, static_cast<int>(window), exact}, o, row_sums);
        ctx->save_for_backward({q, k, v, o, row_sums});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["window"] = window;
        ctx->saved_data["exact"] = exact;
        return o;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        check_saved(saved, grads[0]);
        // (unpack hooks may hand back tensors of another layout, or of a type that takes fewer head dims)
        const int64_t D0 = saved[0].size(3), step = saved[0].scalar_type() == at::kFloat ? 4 : 8;
        const int64_t pad = (step - D0 % step) % step;
        const auto fix = [pad](const Tensor& t) {
            if (pad != 0) return at::constant_pad_nd(t, {0, pad});
            return operand_ok(t) ? t : t.clone(at::MemoryFormat::Contiguous);
        };
        const Tensor q = fix(saved[0]), k = fix(saved[1]), v = fix(saved[2]), o = fix(saved[3]);
        const Tensor row_sums = saved[4].contiguous();
        const Tensor g = fix(grads[0].to(q.scalar_type()));
        const double scale = ctx->saved_data["scale"].toDouble();
        const int window = static_cast<int>(ctx->saved_data["window"].toInt());
        const bool exact = ctx->saved_data["exact"].toBool();
        const int B = dim(q, 0), Hq = dim(q, 1), Hkv = dim(k, 1), T = dim(q, 2), D = dim(q, 3);
        const int code = code_of(q.scalar_type());
        Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
        Tensor delta = at::empty({B, Hq, T}, q.options().dtype(at::kFloat));
        // fp32 partials of the dK/dV blocks split over their query tiles, when the library splits them
        const int64_t ws_bytes = std::max<int64_t>(abi.flash_bwd_workspace_size(B, Hq, Hkv, T, D, window, code), 0);
        Tensor ws;
        if (ws_bytes > 0) ws = at::empty({ws_bytes / 4}, delta.options());
        const c10::DeviceGuard guard(q.device());
        check(abi.flash_bwd_ws(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), g.data_ptr(),
                               row_sums.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                               delta.data_ptr<float>(), B, Hq, Hkv, T, D, strides(q), strides(k), strides(v),
                               strides(o), strides(g), strides(dq), strides(dk), strides(dv),
                               static_cast<float>(scale), window, exact, code,
                               ws.defined() ? ws.data_ptr() : nullptr, ws_bytes, stream_of(q)),
              "sa_flash_bwd_ws");
        for (Tensor* t : {&dq, &dk, &dv})
            if (pad != 0) *t = t->narrow(3, 0, D0).contiguous();
        return {dq, dk, dv, Tensor(), Tensor(), Tensor()};
    }
};

// flash(q, k, v, scale or None, window, exact) -> o or None.
PyObject* py_flash(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *q, *k, *v;
    FlashCall c;
    if (n != 6 || !plain_mode() || !(q = plain(a[0])) || !(k = plain(a[1])) || !(v = plain(a[2])) ||
        !flash_ok(*q, *k, *v) || !as_int(a[4], c.window) || !PyBool_Check(a[5]))
        Py_RETURN_NONE;
    if (a[3] == Py_None)
        c.scale = 1.0 / std::sqrt(static_cast<double>(q->size(3)));
    else if (!as_double(a[3], c.scale))
        Py_RETURN_NONE;
    c.exact = a[5] == Py_True;
    Tensor o;
    {
        const NoGil released;
        if (at::GradMode::is_enabled() && (q->requires_grad() || k->requires_grad() || v->requires_grad())) {
            o = Flash::apply(*q, *k, *v, c.scale, static_cast<int64_t>(c.window), c.exact);
        } else {
            Tensor row_sums;
            flash_fwd(*q, *k, *v, c, o, row_sums);
        }
    }
    return THPVariable_Wrap(o);
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------
// Paged decode and append.
// ---------------------------------------------------------------------------
// Caches [n_pages, Hkv, block_size, D], an int32 table and int32 lengths of
// at least B sequences, all on q's device and in the layout the kernels take.
bool paging_ok(const Tensor& like, int64_t B, int64_t Hkv, int64_t D, int block_size, const Tensor& k, const Tensor& v,
               const Tensor& table, const Tensor& lens) {
    for (const Tensor* t : {&k, &v, &table, &lens})
        if (t->device() != like.device()) return false;
    return k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && k.numel() > 0 &&
           k.size(1) == Hkv && k.size(2) == block_size && k.size(3) == D && block_size > 0 &&
           (block_size & (block_size - 1)) == 0 && k.size(0) <= INT32_MAX && operand_ok(k) && operand_ok(v) &&
           table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) >= B && table.stride(1) == 1 &&
           table.size(1) <= INT32_MAX && lens.scalar_type() == at::kInt && lens.is_contiguous() && lens.numel() >= B;
}

// paged(q, k_cache, v_cache, block_table, context_lens, scale or None, block_size) -> out or None.
PyObject* py_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *q, *k, *v, *table, *lens;
    int block_size;
    if (n != 7 || !plain_mode() || !(q = plain(a[0])) || !(k = plain(a[1])) || !(v = plain(a[2])) ||
        !(table = plain(a[3])) || !(lens = plain(a[4])) || !as_int(a[6], block_size))
        Py_RETURN_NONE;
    if (q->dim() != 4 || q->size(2) != 1 || q->numel() == 0 || k->dim() != 4) Py_RETURN_NONE;
    const int64_t B = q->size(0), Hq = q->size(1), D = q->size(3), Hkv = k->size(1);
    const int qc = code_of(q->scalar_type()), kc = code_of(k->scalar_type());
    // one type for all, or bf16 q over e4m3fn caches (other pairs convert q first)
    const bool mixed = qc == SA_BF16 && kc == SA_FP8_E4M3FN;
    if (!(mixed || (qc == kc && float_code(qc))) || Hkv == 0 || Hq % Hkv != 0 || D % (mixed ? 16 : 8) != 0 || D > 512 ||
        B > INT32_MAX || Hq > INT32_MAX || !operand_ok(*q) ||
        !paging_ok(*q, B, Hkv, D, block_size, *k, *v, *table, *lens))
        Py_RETURN_NONE;
    double scale;
    if (a[5] == Py_None)
        scale = 1.0 / std::sqrt(static_cast<double>(D));
    else if (!as_double(a[5], scale))
        Py_RETURN_NONE;
    Tensor out;
    {
        const NoGil released;
        out = at::empty({B, Hq, D}, q->options().dtype(at::kBFloat16).requires_grad(false));
        const int b = static_cast<int>(B), hq = static_cast<int>(Hq), d = static_cast<int>(D);
        const int max_pages = static_cast<int>(table->size(1));
        const int64_t ws_bytes = abi.paged_decode_workspace_size(b, hq, d, max_pages, block_size);
        Tensor ws = at::empty({std::max<int64_t>(1, (ws_bytes + 3) / 4)}, out.options().dtype(at::kFloat));
        const c10::DeviceGuard guard(q->device());
        check(abi.paged_decode(q->data_ptr(), k->data_ptr(), v->data_ptr(), out.data_ptr(), table->data_ptr<int32_t>(),
                               lens->data_ptr<int32_t>(), b, hq, static_cast<int>(Hkv), d, block_size, max_pages,
                               static_cast<int>(k->size(0)), strides(*q), strides(*k), strides(*v), strides(out),
                               table->stride(0), static_cast<float>(scale), mixed ? SA_PAGED_DTYPES(qc, kc) : qc,
                               ws.data_ptr<float>(), ws.numel() * 4, stream_of(*q)),
              "sa_paged_decode");
    }
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// paged_append(k_cache, v_cache, k_new, v_new, block_table, context_lens, block_size) -> new lengths or None.
PyObject* py_paged_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *k, *v, *kn, *vn, *table, *lens;
    int block_size;
    if (n != 7 || !plain_mode() || !(k = plain(a[0])) || !(v = plain(a[1])) || !(kn = plain(a[2])) ||
        !(vn = plain(a[3])) || !(table = plain(a[4])) || !(lens = plain(a[5])) || !as_int(a[6], block_size))
        Py_RETURN_NONE;
    const int code = code_of(k->scalar_type());
    if (code < 0 || kn->dim() != 4 || kn->numel() == 0 || vn->sizes() != kn->sizes() ||
        kn->scalar_type() != k->scalar_type() || vn->scalar_type() != k->scalar_type() ||
        kn->device() != k->device() || vn->device() != k->device())
        Py_RETURN_NONE;
    const int64_t B = kn->size(0), Hkv = kn->size(1), n_new = kn->size(2), D = kn->size(3);
    if (!paging_ok(*k, B, Hkv, D, block_size, *k, *v, *table, *lens) || D % (16 / k->element_size()) != 0 ||
        !operand_ok(*kn) || !operand_ok(*vn) || kn->strides() != vn->strides() || B > INT32_MAX || n_new > INT32_MAX)
        Py_RETURN_NONE;
    Tensor out;
    {
        const NoGil released;
        const c10::DeviceGuard guard(k->device());
        out = at::empty(lens->sizes(), lens->options());
        check(abi.paged_kv_append_lens(kn->data_ptr(), vn->data_ptr(), k->data_ptr(), v->data_ptr(),
                                       table->data_ptr<int32_t>(), lens->data_ptr<int32_t>(), out.data_ptr<int32_t>(),
                                       lens->numel(), static_cast<int>(B), static_cast<int>(Hkv),
                                       static_cast<int>(n_new), static_cast<int>(D), block_size,
                                       static_cast<int>(table->size(1)), static_cast<int>(k->size(0)), strides(*kn),
                                       strides(*k), strides(*v), table->stride(0), code, stream_of(*k)),
              "sa_paged_kv_append_lens");
    }
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------
// RMS norm + RoPE of queries and keys.
// ---------------------------------------------------------------------------
// A tensor argument that may be None: false where it is neither None nor plain.
bool plain_or_none(PyObject* o, const Tensor*& t) {
    t = nullptr;
    return o == Py_None || (t = plain(o)) != nullptr;
}

const void* ptr(const Tensor* t) { return t ? t->data_ptr() : nullptr; }

// Weights [D] of x's type or fp32, of one type.
bool norm_weight_ok(const Tensor* w, const Tensor& x) {
    return w == nullptr || (w->dim() == 1 && w->size(0) == x.size(-1) && w->is_contiguous() && aligned16(*w) &&
                            w->device() == x.device() &&
                            (w->scalar_type() == x.scalar_type() || w->scalar_type() == at::kFloat));
}
int norm_weight_code(const Tensor* qw, const Tensor* kw, const Tensor& x) {
    const Tensor* w = qw ? qw : kw;
    return code_of(w ? w->scalar_type() : x.scalar_type());
}

bool norm_common_ok(const Tensor& q, const Tensor* qw, const Tensor* kw, const Tensor& cos, const Tensor& sin) {
    const int64_t D = q.size(-1);
    if (!float_code(code_of(q.scalar_type())) || D % 16 != 0 || D < 16 || D > 512 || !norm_weight_ok(qw, q) ||
        !norm_weight_ok(kw, q) || (qw && kw && qw->scalar_type() != kw->scalar_type()))
        return false;
    for (const Tensor* t : {&cos, &sin})
        if (t->dim() != 2 || t->size(1) != D / 2 || t->size(0) != cos.size(0) || t->size(0) == 0 ||
            t->size(0) > INT32_MAX || t->scalar_type() != at::kFloat || !t->is_contiguous() || !aligned16(*t) ||
            t->device() != q.device() || t->requires_grad())
            return false;
    return true;
}

bool qk_norm_ok(const Tensor& q, const Tensor& k, const Tensor* qw, const Tensor* kw, const Tensor& cos,
                const Tensor& sin, const Tensor* pos) {
    if (q.dim() != 4 || k.dim() != 4 || q.numel() == 0 || k.numel() == 0 || k.size(0) != q.size(0) ||
        k.size(2) != q.size(2) || k.size(3) != q.size(3) || k.scalar_type() != q.scalar_type() ||
        k.device() != q.device() || !norm_common_ok(q, qw, kw, cos, sin) || !operand_ok(q) || !operand_ok(k))
        return false;
    const int64_t B = q.size(0), T = q.size(2);
    if (B > (1 << 24) || T > (1 << 24) || B * T > (1 << 24) || q.size(1) > 16383 || k.size(1) > 16383) return false;
    if (pos == nullptr) return cos.size(0) >= T;
    return pos->scalar_type() == at::kInt && pos->is_contiguous() && pos->device() == q.device() &&
           ((pos->dim() == 1 && pos->size(0) == T) || (pos->dim() == 2 && pos->size(0) == B && pos->size(1) == T));
}

// A dense tensor in x's order of dims, if that keeps D innermost (kernels.py's rule).
Tensor output_like(const Tensor& x) {
    Tensor y = at::empty_like(x);
    return y.stride(-1) == 1 ? y : at::empty(x.sizes(), x.options());
}

const int32_t* positions_ptr(const Tensor* pos) { return pos ? pos->data_ptr<int32_t>() : nullptr; }
int64_t positions_stride(const Tensor* pos) { return pos && pos->dim() == 2 ? pos->size(1) : 0; }

void qk_norm_fwd(const Tensor& q, const Tensor& k, const Tensor* qw, const Tensor* kw, const Tensor& cos,
                 const Tensor& sin, const Tensor* pos, double eps, Tensor& yq, Tensor& yk) {
    yq = output_like(q);
    yk = output_like(k);
    const c10::DeviceGuard guard(q.device());
    check(abi.qk_norm_rope_fwd(q.data_ptr(), k.data_ptr(), yq.data_ptr(), yk.data_ptr(), ptr(qw), ptr(kw),
                               cos.data_ptr<float>(), sin.data_ptr<float>(), positions_ptr(pos), positions_stride(pos),
                               dim(q, 0), dim(q, 1), dim(k, 1), dim(q, 2), dim(q, 3), dim(cos, 0), strides(q),
                               strides(k), strides(yq), strides(yk), static_cast<float>(eps),
                               code_of(q.scalar_type()), norm_weight_code(qw, kw, q), stream_of(q)),
          "sa_qk_norm_rope_fwd");
}

// A backward that is being captured, and reaches a leaf whose gradient
// accumulator lives on the default stream, because a graph or a hook made outside
// of any other stream still holds it (a leaf has one as long as anything does): the
// engine makes the accumulator's stream and the backward's wait for each other,
// which the default stream cannot do for a capture, and the process ends.  Raised
// here instead, before that; called from a node's backward.  Any other stream joins
// the capture with the first wait and is waited for with the second.
void refuse_default_stream_leaves(c10::Device device) {
    {
        const c10::DeviceGuard guard(device);
        if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    }
    const std::shared_ptr<torch::autograd::Node> node = torch::autograd::get_current_node();
    if (!node) return;
    std::vector<torch::autograd::Node*> todo{node.get()};
    std::unordered_set<torch::autograd::Node*> seen{node.get()};
    while (!todo.empty()) {
        torch::autograd::Node* n = todo.back();
        todo.pop_back();
        if (n->num_outputs() == 0) {  // a leaf's
            const auto stream = n->stream();
            TORCH_CHECK(!stream || stream->id() != c10::hip::getDefaultHIPStream(stream->device_index()).id(),
                        "sp2norm_qk_norm_rope: this backward is being captured into a graph while an autograd graph or "
                        "a hook of the same leaves lives on the default stream; drop that first, or make it on another "
                        "stream");
        }
        for (uint32_t i = 0; i < n->num_outputs(); ++i)
            if (n->task_should_compute_output(i) && seen.insert(n->next_edge(i).function.get()).second)
                todo.push_back(n->next_edge(i).function.get());
    }
}

// check_capture(x): raises as the native backward does; for the backward of a node of Python's.
PyObject* py_check_capture(PyObject*, PyObject* x) {
    HANDLE_TH_ERRORS
    if (THPVariable_Check(x) && THPVariable_Unpack(x).is_cuda()) refuse_default_stream_leaves(THPVariable_Unpack(x).device());
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

struct QKNorm : public torch::autograd::Function<QKNorm> {
    using MaybeTensor = std::optional<Tensor>;
    static const Tensor* get(const MaybeTensor& t) { return t.has_value() ? &*t : nullptr; }
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const MaybeTensor& qw,
                                 const MaybeTensor& kw, const Tensor& cos, const Tensor& sin, const MaybeTensor& pos,
                                 double eps) {
        Tensor yq, yk;
        qk_norm_fwd(q, k, get(qw), get(kw), cos, sin, get(pos), eps, yq, yk);
        variable_list save{q, k, cos, sin};
        for (const MaybeTensor* t : {&qw, &kw, &pos})
            if (t->has_value()) save.push_back(**t);
        ctx->save_for_backward(std::move(save));
        ctx->saved_data["given"] = int64_t(qw.has_value()) | int64_t(kw.has_value()) << 1 | int64_t(pos.has_value()) << 2;
        ctx->saved_data["eps"] = eps;
        return {yq, yk};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const bool again = at::GradMode::is_enabled() && (grads[0].requires_grad() || grads[1].requires_grad());
        const at::AutoGradMode off(false);
        const variable_list saved = ctx->get_saved_variables();
        const int64_t given = ctx->saved_data["given"].toInt();
        const Tensor* opt[3] = {nullptr, nullptr, nullptr};  // q_weight, k_weight, positions
        int at_saved = 4;
        for (int i = 0; i < 3; ++i)
            if (given >> i & 1) opt[i] = &saved[at_saved++];
        const auto fix = [](const Tensor& t) { return operand_ok(t) ? t : t.clone(at::MemoryFormat::Contiguous); };
        // (unpack hooks may hand back other layouts, and other types or sizes, which are refused)
        TORCH_CHECK_VALUE(saved[0].is_cuda() && saved[0].dim() == 4 && saved[1].dim() == 4 &&
                              float_code(code_of(saved[0].scalar_type())),
                          "the saved tensors of the norm must have the shapes and dtype that forward saved");
        for (const Tensor* t : std::initializer_list<const Tensor*>{&saved[1], &saved[2], &saved[3], opt[0], opt[1],
                                                                   opt[2], &grads[0], &grads[1]})
            TORCH_CHECK_VALUE(t == nullptr || (t->is_cuda() && t->device() == saved[0].device()),
                              "the norm's tensors must live on the same CUDA device as q");
        // (only the tensors given have an edge)
        const bool need_w[2] = {opt[0] && ctx->needs_input_grad(2), opt[1] && ctx->needs_input_grad(opt[0] ? 3 : 2)};
        refuse_default_stream_leaves(saved[0].device());
        const Tensor q = fix(saved[0]), k = fix(saved[1]);
        const auto plain_table = [](const Tensor& t) {
            return t.is_contiguous() && aligned16(t) ? t : t.clone(at::MemoryFormat::Contiguous);
        };
        const Tensor cos = plain_table(saved[2]), sin = plain_table(saved[3]);
        Tensor w[2], pos;
        for (int i = 0; i < 2; ++i)
            if (opt[i]) w[i] = plain_table(*opt[i]);
        if (opt[2]) pos = opt[2]->contiguous();
        const Tensor *qw = opt[0] ? &w[0] : nullptr, *kw = opt[1] ? &w[1] : nullptr, *ps = opt[2] ? &pos : nullptr;
        TORCH_CHECK_VALUE(q.sizes() == grads[0].sizes() && k.sizes() == grads[1].sizes() &&
                              qk_norm_ok(q, k, qw, kw, cos, sin, ps),
                          "the saved tensors of the norm must have the shapes and dtype that forward saved");
        const Tensor gq = fix(grads[0].to(q.scalar_type())), gk = fix(grads[1].to(q.scalar_type()));
        const int B = dim(q, 0), Hq = dim(q, 1), Hkv = dim(k, 1), T = dim(q, 2), D = dim(q, 3);
        Tensor dq = output_like(q), dk = output_like(k), dw[2], ws;
        if (need_w[0]) dw[0] = at::empty_like(*qw);
        if (need_w[1]) dw[1] = at::empty_like(*kw);
        const bool any = dw[0].defined() || dw[1].defined();
        const int64_t ws_bytes = any ? abi.qk_norm_rope_bwd_workspace_size(B, Hq, Hkv, T, D) : 0;
        if (any) ws = at::empty({ws_bytes / 4}, q.options().dtype(at::kFloat));
        const auto out = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
        {
            const c10::DeviceGuard guard(q.device());
            check(abi.qk_norm_rope_bwd(
                      q.data_ptr(), k.data_ptr(), gq.data_ptr(), gk.data_ptr(), dq.data_ptr(), dk.data_ptr(), out(dw[0]),
                      out(dw[1]), ptr(qw), ptr(kw), cos.data_ptr<float>(), sin.data_ptr<float>(), positions_ptr(ps),
                      positions_stride(ps), B, Hq, Hkv, T, D, dim(cos, 0), strides(q), strides(k), strides(gq),
                      strides(gk), strides(dq), strides(dk), static_cast<float>(ctx->saved_data["eps"].toDouble()),
                      code_of(q.scalar_type()), norm_weight_code(qw, kw, q),
                      any ? ws.data_ptr<float>() : nullptr, ws_bytes, stream_of(q)),
                  "sa_qk_norm_rope_bwd");
        }
        variable_list result{dq, dk, dw[0], dw[1]};
        if (again) {  // differentiated twice: the second time raises
            const at::AutoGradMode on(true);
            for (Tensor& t : result)
                if (t.defined()) t.set_requires_grad(true);
            auto error = std::make_shared<torch::autograd::DelayedError>(
                "trying to differentiate twice a function that has one derivative (sp2norm_qk_norm_rope)",
                static_cast<int64_t>(result.size()));
            result = (*error)(std::move(result));
        }
        return {result[0], result[1], result[2], result[3], Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps) -> (q', k') or None.
PyObject* py_qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *q, *k, *qw, *kw, *cos, *sin, *pos;
    double eps;
    if (n != 8 || !plain_mode() || !(q = plain(a[0])) || !(k = plain(a[1])) || !plain_or_none(a[2], qw) ||
        !plain_or_none(a[3], kw) || !(cos = plain(a[4])) || !(sin = plain(a[5])) || !plain_or_none(a[6], pos) ||
        !as_double(a[7], eps) || !qk_norm_ok(*q, *k, qw, kw, *cos, *sin, pos))
        Py_RETURN_NONE;
    Tensor yq, yk;
    {
        const NoGil released;
        const auto wants = [](const Tensor* t) { return t && t->requires_grad(); };
        if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(qw) || wants(kw))) {
            const auto maybe = [](const Tensor* t) { return t ? std::optional<Tensor>(*t) : std::nullopt; };
            variable_list y = QKNorm::apply(*q, *k, maybe(qw), maybe(kw), *cos, *sin, maybe(pos), eps);
            yq = y[0];
            yk = y[1];
        } else {
            qk_norm_fwd(*q, *k, qw, kw, *cos, *sin, pos, eps, yq, yk);
        }
    }
    PyObject* pair = PyTuple_New(2);
    if (pair == nullptr) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(yq));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(yk));
    return pair;
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------
// Serving operators.
// ---------------------------------------------------------------------------
// A block table [>= B, max_pages] of rows that do not overlap.
bool table_ok(const Tensor& t, int64_t B, const Tensor& like) {
    return t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) >= B && t.size(1) > 0 && t.size(1) <= INT32_MAX &&
           t.stride(1) == 1 && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) && t.device() == like.device();
}
int64_t table_stride(const Tensor& t) { return std::max(t.stride(0), t.size(1)); }

// A contiguous int32 vector of at least n entries.
bool ints_ok(const Tensor& t, int64_t n, const Tensor& like) {
    return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) >= n && t.is_contiguous() &&
           t.device() == like.device();
}

// Caches [n_pages, Hkv, block_size, D] in the layout that the kernels take.
bool cache_ok(const Tensor& c, int64_t Hkv, int block_size, int64_t D, const Tensor& like) {
    return c.dim() == 4 && c.numel() > 0 && c.size(1) == Hkv && c.size(2) == block_size && c.size(3) == D &&
           code_of(c.scalar_type()) >= 0 && c.size(0) <= INT32_MAX / block_size && D % (16 / c.element_size()) == 0 &&
           c.device() == like.device() && operand_ok(c);
}
bool power_of_two(int x) { return x > 0 && (x & (x - 1)) == 0; }

// paged_norm_append(q, k, v, q_weight, k_weight, cos, sin, positions, slots, k_cache, v_cache, eps,
// block_size) -> q' or None.
PyObject* py_paged_norm_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *q, *k, *v, *qw, *kw, *cos, *sin, *pos, *slots, *kc, *vc;
    double eps;
    int block_size;
    if (n != 13 || !plain_mode() || !(q = plain(a[0])) || !(k = plain(a[1])) || !(v = plain(a[2])) ||
        !plain_or_none(a[3], qw) || !plain_or_none(a[4], kw) || !(cos = plain(a[5])) || !(sin = plain(a[6])) ||
        !(pos = plain(a[7])) || !(slots = plain(a[8])) || !(kc = plain(a[9])) || !(vc = plain(a[10])) ||
        !as_double(a[11], eps) || !as_int(a[12], block_size) || block_size == 0)
        Py_RETURN_NONE;
    if (q->dim() != 3 || k->dim() != 3 || q->numel() == 0 || k->numel() == 0 || v->sizes() != k->sizes() ||
        k->size(0) != q->size(0) || k->size(2) != q->size(2) || q->size(0) > (1 << 24) || q->size(1) > 16383 ||
        k->size(1) > 16383 || !norm_common_ok(*q, qw, kw, *cos, *sin))
        Py_RETURN_NONE;
    for (const Tensor* t : {k, v})
        if (t->scalar_type() != q->scalar_type() || t->device() != q->device()) Py_RETURN_NONE;
    const int64_t N = q->size(0), Hkv = k->size(1), D = q->size(2);
    if (!operand_ok(*q) || !operand_ok(*k) || !operand_ok(*v) || !ints_ok(*pos, N, *q) || !ints_ok(*slots, N, *q) ||
        pos->size(0) != N || slots->size(0) != N || !cache_ok(*kc, Hkv, block_size, D, *q) ||
        !cache_ok(*vc, Hkv, block_size, D, *q) || vc->sizes() != kc->sizes() || vc->scalar_type() != kc->scalar_type())
        Py_RETURN_NONE;
    Tensor out;
    {
        const NoGil released;
        const at::AutoGradMode off(false);
        out = output_like(*q);
        const c10::DeviceGuard guard(q->device());
        check(abi.paged_qk_norm_rope_append(
                  q->data_ptr(), k->data_ptr(), v->data_ptr(), out.data_ptr(), kc->data_ptr(), vc->data_ptr(), ptr(qw),
                  ptr(kw), cos->data_ptr<float>(), sin->data_ptr<float>(), pos->data_ptr<int32_t>(),
                  slots->data_ptr<int32_t>(), static_cast<int>(N), dim(*q, 1), static_cast<int>(Hkv),
                  static_cast<int>(D), dim(*cos, 0), block_size, dim(*kc, 0), strides(*q), strides(*k), strides(*v),
                  strides(out), strides(*kc), strides(*vc), static_cast<float>(eps), code_of(q->scalar_type()),
                  norm_weight_code(qw, kw, *q), code_of(kc->scalar_type()), stream_of(*q)),
              "sa_paged_qk_norm_rope_append");
    }
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// int32 vectors of the given sizes in one allocation, each from a multiple of
// 256 bytes on: an allocation costs about as much host time as half a launch.
template <size_t N>
std::array<Tensor, N> int_vectors(const int64_t (&sizes)[N], const Tensor& like) {
    constexpr int64_t step = 64;
    int64_t total = 0;
    for (int64_t n : sizes) total += (n + step - 1) / step * step;
    const Tensor all = at::empty({total}, like.options().requires_grad(false));
    std::array<Tensor, N> out;
    int64_t at_element = 0;
    for (size_t i = 0; i < N; ++i) {
        out[i] = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
        out[i].unsafeGetTensorImpl()->set_storage_offset(at_element);
        out[i].unsafeGetTensorImpl()->set_sizes_contiguous({sizes[i]});
        at_element += (sizes[i] + step - 1) / step * step;
    }
    return out;
}

// What reserve and release take as they are: a table of B rows, lengths [B],
// the stack and its count.
bool maps_ok(const Tensor& table, const Tensor& lens, const Tensor& free_pages, const Tensor& n_free, int block_size) {
    if (table.dim() != 2 || table.numel() == 0 || block_size == 0) return false;
    const int64_t B = table.size(0);
    return B <= 4096 && table_ok(table, B, table) && ints_ok(lens, B, table) && lens.size(0) == B &&
           ints_ok(free_pages, 1, table) && n_free.scalar_type() == at::kInt && n_free.numel() == 1 &&
           n_free.device() == table.device() && std::max(free_pages.size(0), table.size(1)) <= INT32_MAX / block_size;
}

// paged_reserve(block_table, context_lens, new_lens, free_pages, n_free, n_tokens, block_size) -> (slots,
// positions, sequences, starts, context_lens, n_free) or None.
PyObject* py_paged_reserve(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *table, *lens, *fresh, *free_pages, *n_free;
    int n_tokens, block_size;
    if (n != 7 || !plain_mode() || !(table = plain(a[0])) || !(lens = plain(a[1])) || !(fresh = plain(a[2])) ||
        !(free_pages = plain(a[3])) || !(n_free = plain(a[4])) || !as_int(a[5], n_tokens) || !as_int(a[6], block_size) ||
        !maps_ok(*table, *lens, *free_pages, *n_free, block_size) || !ints_ok(*fresh, table->size(0), *table) ||
        fresh->size(0) != table->size(0))
        Py_RETURN_NONE;
    std::array<Tensor, 6> out;
    {
        const NoGil released;
        const int64_t B = table->size(0);
        // (what a program keeps from step to step holds nothing of the tokens' maps)
        const auto maps = int_vectors({n_tokens, n_tokens, n_tokens}, *table);
        const auto lengths = int_vectors({B + 1, B, 1}, *table);
        out = {maps[0], maps[1], maps[2], lengths[0], lengths[1], lengths[2]};
        const c10::DeviceGuard guard(table->device());
        const auto p = [](const Tensor& t) { return t.data_ptr<int32_t>(); };
        check(abi.paged_reserve(p(*table), p(*lens), p(*fresh), p(*free_pages), p(*n_free), p(out[0]), p(out[1]),
                                p(out[2]), p(out[3]), p(out[4]), p(out[5]), static_cast<int>(B), dim(*table, 1),
                                block_size, dim(*free_pages, 0), n_tokens, table_stride(*table), stream_of(*table)),
              "sa_paged_reserve");
    }
    PyObject* all = PyTuple_New(6);
    if (all == nullptr) return nullptr;
    for (int i = 0; i < 6; ++i) PyTuple_SET_ITEM(all, i, THPVariable_Wrap(out[i]));
    return all;
    END_HANDLE_TH_ERRORS
}

// paged_release(block_table, context_lens, finished, free_pages, n_free, block_size) -> (context_lens, n_free) or None.
PyObject* py_paged_release(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *table, *lens, *finished, *free_pages, *n_free;
    int block_size;
    if (n != 6 || !plain_mode() || !(table = plain(a[0])) || !(lens = plain(a[1])) || !(finished = plain(a[2])) ||
        !(free_pages = plain(a[3])) || !(n_free = plain(a[4])) || !as_int(a[5], block_size) ||
        !maps_ok(*table, *lens, *free_pages, *n_free, block_size) || finished->scalar_type() != at::kBool ||
        finished->dim() != 1 || finished->size(0) != table->size(0) || !finished->is_contiguous() ||
        finished->device() != table->device())
        Py_RETURN_NONE;
    Tensor out, left, counts;
    {
        const NoGil released;
        const int64_t B = table->size(0);
        const auto made = int_vectors({B, 1, B}, *table);
        out = made[0];
        left = made[1];
        counts = made[2];
        const c10::DeviceGuard guard(table->device());
        const auto p = [](const Tensor& t) { return t.data_ptr<int32_t>(); };
        check(abi.paged_release(p(*table), p(*lens), static_cast<const uint8_t*>(finished->data_ptr()), p(*free_pages),
                                p(*n_free), p(out), p(left), p(counts), static_cast<int>(B), dim(*table, 1), block_size,
                                dim(*free_pages, 0), table_stride(*table), stream_of(*table)),
              "sa_paged_release");
    }
    PyObject* pair = PyTuple_New(2);
    if (pair == nullptr) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(out));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(left));
    return pair;
    END_HANDLE_TH_ERRORS
}

// Bounds of a cache [n_pages, Hkv, block_size, D], contiguous [n_pages, Hkv, 2, D].
bool bounds_ok(const Tensor& b, const Tensor& like) {
    return b.dim() == 4 && b.numel() > 0 && b.size(2) == 2 && b.size(0) <= INT32_MAX && b.is_contiguous() &&
           aligned16(b) && b.device() == like.device() && code_of(b.scalar_type()) >= 0 && b.size(3) <= 1024 &&
           b.size(3) % 8 == 0 && (b.element_size() != 1 || b.size(3) % 16 == 0);
}

// paged_key_bounds(k_cache, block_table, from_lens, to_lens, bounds, block_size) -> bool: whether it ran.
PyObject* py_paged_key_bounds(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *kc, *table, *from, *to, *bounds;
    int block_size;
    if (n != 6 || !plain_mode() || !(kc = plain(a[0])) || !(table = plain(a[1])) || !(from = plain(a[2])) ||
        !(to = plain(a[3])) || !(bounds = plain(a[4])) || !as_int(a[5], block_size) || !power_of_two(block_size) ||
        kc->dim() != 4 || table->dim() != 2)
        Py_RETURN_FALSE;
    const int64_t B = table->size(0), Hkv = kc->size(1), D = kc->size(3);
    if (B == 0 || B > INT32_MAX || !cache_ok(*kc, Hkv, block_size, D, *kc) || !table_ok(*table, B, *kc) ||
        !ints_ok(*from, B, *kc) || !ints_ok(*to, B, *kc) || !bounds_ok(*bounds, *kc) ||
        bounds->scalar_type() != kc->scalar_type() || bounds->size(0) != kc->size(0) || bounds->size(1) != Hkv ||
        bounds->size(3) != D)
        Py_RETURN_FALSE;
    {
        const NoGil released;
        const c10::DeviceGuard guard(kc->device());
        check(abi.paged_key_bounds(kc->data_ptr(), bounds->data_ptr(), table->data_ptr<int32_t>(),
                                   from->data_ptr<int32_t>(), to->data_ptr<int32_t>(), static_cast<int>(B),
                                   static_cast<int>(Hkv), static_cast<int>(D), block_size, dim(*table, 1), dim(*kc, 0),
                                   strides(*kc), table_stride(*table), code_of(kc->scalar_type()), stream_of(*kc)),
              "sa_paged_key_bounds");
    }
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// One query token of each sequence, [B, Hq, 1, D].
bool decode_q_ok(const Tensor& q, int64_t Hkv) {
    return q.dim() == 4 && q.size(2) == 1 && q.numel() > 0 && q.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX &&
           Hkv > 0 && q.size(1) % Hkv == 0 && operand_ok(q);
}

// paged_select_pages(q, bounds, block_table, context_lens, top_k, n_first, n_last, block_size) -> pages or None.
PyObject* py_paged_select_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *q, *bounds, *table, *lens;
    int top_k, n_first, n_last, block_size;
    if (n != 8 || !plain_mode() || !(q = plain(a[0])) || !(bounds = plain(a[1])) || !(table = plain(a[2])) ||
        !(lens = plain(a[3])) || !as_int(a[4], top_k) || !as_int(a[5], n_first) || !as_int(a[6], n_last) ||
        !as_int(a[7], block_size) || !power_of_two(block_size) || top_k < 1 || top_k >= (1 << 24) ||
        static_cast<int64_t>(n_first) + n_last > top_k)
        Py_RETURN_NONE;
    if (!bounds_ok(*bounds, *bounds) || !decode_q_ok(*q, bounds->size(1)) || !float_code(code_of(q->scalar_type())) ||
        q->size(3) != bounds->size(3) || q->device() != bounds->device() || !table_ok(*table, q->size(0), *q) ||
        !ints_ok(*lens, q->size(0), *q) || bounds->size(0) > INT32_MAX / block_size)
        Py_RETURN_NONE;
    Tensor pages;
    {
        const NoGil released;
        const int B = dim(*q, 0), Hkv = dim(*bounds, 1), W = dim(*table, 1);
        pages = at::empty({B, Hkv, top_k}, table->options());
        const int64_t ws_bytes = top_k < W ? abi.paged_select_workspace_size(B, Hkv, W) : 0;
        Tensor ws;
        if (ws_bytes > 0) ws = at::empty({(ws_bytes + 7) / 8}, table->options().dtype(at::kDouble));
        const c10::DeviceGuard guard(q->device());
        check(abi.paged_select_pages(q->data_ptr(), bounds->data_ptr(), table->data_ptr<int32_t>(),
                                     lens->data_ptr<int32_t>(), pages.data_ptr<int32_t>(), B, dim(*q, 1), Hkv,
                                     dim(*q, 3), block_size, W, dim(*bounds, 0), top_k, n_first, n_last, strides(*q),
                                     table_stride(*table), code_of(q->scalar_type()), code_of(bounds->scalar_type()),
                                     ws.defined() ? ws.data_ptr() : nullptr, ws_bytes, stream_of(*q)),
              "sa_paged_select_pages");
    }
    return THPVariable_Wrap(pages);
    END_HANDLE_TH_ERRORS
}

// paged_sparse(q, k_cache, v_cache, block_table, context_lens, pages, scale or None, block_size) -> out or None.
PyObject* py_paged_sparse(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *q, *k, *v, *table, *lens, *pages;
    int block_size;
    if (n != 8 || !plain_mode() || !(q = plain(a[0])) || !(k = plain(a[1])) || !(v = plain(a[2])) ||
        !(table = plain(a[3])) || !(lens = plain(a[4])) || !(pages = plain(a[5])) || !as_int(a[7], block_size) ||
        !power_of_two(block_size) || k->dim() != 4 || !decode_q_ok(*q, k->size(1)))
        Py_RETURN_NONE;
    const int64_t B = q->size(0), Hq = q->size(1), D = q->size(3), Hkv = k->size(1);
    const int qc = code_of(q->scalar_type()), kc = code_of(k->scalar_type());
    const bool mixed = qc == SA_BF16 && kc == SA_FP8_E4M3FN;  // (other pairs convert q first)
    if (!(mixed || (qc == kc && float_code(qc))) || Hq / Hkv > 32 || D % (mixed ? 16 : 8) != 0 || D > 512 ||
        !paging_ok(*q, B, Hkv, D, block_size, *k, *v, *table, *lens) || !table_ok(*table, B, *q) ||
        !ints_ok(*lens, B, *q) || k->size(0) > INT32_MAX / block_size || pages->dim() != 3 || pages->size(0) != B ||
        pages->size(1) != Hkv || pages->size(2) > INT32_MAX || pages->scalar_type() != at::kInt ||
        !pages->is_contiguous() || pages->device() != q->device())
        Py_RETURN_NONE;
    double scale;
    if (a[6] == Py_None)
        scale = 1.0 / std::sqrt(static_cast<double>(D));
    else if (!as_double(a[6], scale))
        Py_RETURN_NONE;
    Tensor out;
    {
        const NoGil released;
        out = at::empty({B, Hq, D}, q->options().dtype(at::kBFloat16).requires_grad(false));
        const int b = static_cast<int>(B), hq = static_cast<int>(Hq), d = static_cast<int>(D);
        const int hkv = static_cast<int>(Hkv), listed = dim(*pages, 2);
        const int64_t ws_bytes =
            std::max<int64_t>(16, abi.paged_sparse_workspace_size(b, hq, hkv, d, listed, block_size));
        Tensor ws = at::empty({(ws_bytes + 3) / 4}, out.options().dtype(at::kFloat));
        const c10::DeviceGuard guard(q->device());
        check(abi.paged_sparse_decode(q->data_ptr(), k->data_ptr(), v->data_ptr(), out.data_ptr(),
                                      table->data_ptr<int32_t>(), lens->data_ptr<int32_t>(), pages->data_ptr<int32_t>(),
                                      b, hq, hkv, d, block_size, dim(*table, 1), dim(*k, 0), listed, strides(*q),
                                      strides(*k), strides(*v), strides(out), table_stride(*table),
                                      static_cast<float>(scale), mixed ? SA_PAGED_DTYPES(qc, kc) : qc,
                                      ws.data_ptr<float>(), ws.numel() * 4, stream_of(*q)),
              "sa_paged_sparse_decode");
    }
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

template <typename F>
PyCFunction fast(F f) {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_O, "bind({name: address of a C ABI function})"},
    {"norm_out", fast(py_norm_out), METH_FASTCALL, "norm_out(out, x, causal, alpha, theta, power) -> bool"},
    {"causal_norm", fast(py_causal_norm), METH_FASTCALL, "causal_norm(x, alpha, theta, power) -> y or None"},
    {"flash", fast(py_flash), METH_FASTCALL, "flash(q, k, v, scale, window, exact) -> o or None"},
    {"paged", fast(py_paged), METH_FASTCALL,
     "paged(q, k_cache, v_cache, block_table, context_lens, scale, block_size) -> out or None"},
    {"paged_append", fast(py_paged_append), METH_FASTCALL,
     "paged_append(k_cache, v_cache, k_new, v_new, block_table, context_lens, block_size) -> lens or None"},
    {"qk_norm_rope", fast(py_qk_norm_rope), METH_FASTCALL,
     "qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps) -> (q', k') or None"},
    {"check_capture", py_check_capture, METH_O, "check_capture(x): in a backward on x's device"},
    {"paged_norm_append", fast(py_paged_norm_append), METH_FASTCALL,
     "paged_norm_append(q, k, v, q_weight, k_weight, cos, sin, positions, slots, k_cache, v_cache, eps, block_size) "
     "-> q' or None"},
    {"paged_reserve", fast(py_paged_reserve), METH_FASTCALL,
     "paged_reserve(block_table, context_lens, new_lens, free_pages, n_free, n_tokens, block_size) -> 6 tensors or "
     "None"},
    {"paged_release", fast(py_paged_release), METH_FASTCALL,
     "paged_release(block_table, context_lens, finished, free_pages, n_free, block_size) -> 2 tensors or None"},
    {"paged_key_bounds", fast(py_paged_key_bounds), METH_FASTCALL,
     "paged_key_bounds(k_cache, block_table, from_lens, to_lens, bounds, block_size) -> bool"},
    {"paged_select_pages", fast(py_paged_select_pages), METH_FASTCALL,
     "paged_select_pages(q, bounds, block_table, context_lens, top_k, n_first, n_last, block_size) -> pages or None"},
    {"paged_sparse", fast(py_paged_sparse), METH_FASTCALL,
     "paged_sparse(q, k_cache, v_cache, block_table, context_lens, pages, scale, block_size) -> out or None"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Native call path (see csrc/host/host.cpp).", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
    PyObject* m = PyModule_Create(&module);
    // (the tensors' layout in memory is that torch's)
    if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) Py_CLEAR(m);
    return m;
}
