// Host path of the Python package: argument checks, output and scratch allocation, the C ABI calls and
// the autograd nodes of the ops, in one native call per op.
//
// What bounds the small calls is the host: a dense forward at one sample is three launches of 5-12 us,
// and the same call made through ctypes and torch.autograd.Function spent 15-25 us of interpreter time
// per op and as much again per backward node (784-800-800-10 at B=256: 348 us per training step for
// 215 us of kernels).  Here an op costs its launches plus 3-4 us.
//
// The library is reached through function pointers looked up in the very file _lib.py has loaded.
// Scratch comes from PyTorch's caching allocator per call: it is stream-ordered, belongs to the graph's
// pool while a stream is captured, and is safe with several threads and streams without a pool of ours.
// The GIL is released while an op runs.
//
// The nodes below know reverse mode over ordinary tensors.  Everything else PyTorch can hand an op -- forward-mode
// tangents, functorch's wrappers, tensors of Python modes, a tracer that has to see the call -- goes to the
// torch.autograd.Function of the same op in ops.py, which refuses or records it as any such function does (`plain`).
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <dlfcn.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/autograd.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <array>
#include <optional>
#include <string>
#include <vector>

#include "../../include/snntc.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// ---- the library ---------------------------------------------------------------------------------------------------

#define SNNTC_BOUND(F)                                                                                             \
    F(snntc_last_error) F(snntc_fc_forward) F(snntc_fc_forward_workspace_bytes) F(snntc_fc_backward)               \
    F(snntc_fc_backward_workspace_bytes) F(snntc_cv_output_dims) F(snntc_cv_forward)                               \
    F(snntc_cv_forward_chained) F(snntc_cv_forward_workspace_bytes) F(snntc_cv_backward_cropped)                   \
    F(snntc_cv_backward_workspace_bytes) F(snntc_softmax_time_loss) F(snntc_sgd_update)                            \
    F(snntc_min_pool_forward) F(snntc_min_pool_forward_chained) F(snntc_min_pool_backward)                         \
    F(snntc_pad_time_forward) F(snntc_pad_time_backward) F(snntc_encode_time) F(snntc_label_loss)                  \
    F(snntc_weight_cost_workspace_bytes) F(snntc_weight_cost_sums) F(snntc_weight_cost_grad) F(snntc_recipe_total)    \
    F(snntc_embed_forward) F(snntc_embed_backward) F(snntc_embed_backward_workspace_bytes)                         \
    F(snntc_gated_scan_forward) F(snntc_gated_scan_backward) F(snntc_gated_scan_workspace_bytes)                   \
    F(snntc_gated_step) F(snntc_choice_workspace_bytes) F(snntc_preference_workspace_bytes) F(snntc_time_logp)     \
    F(snntc_time_logp_backward)                                                                                    \
    F(snntc_policy_loss) F(snntc_preference_loss) F(snntc_loss_total) F(snntc_rule_times)                          \
    F(snntc_rule_times_backward) F(snntc_choose_workspace_bytes) F(snntc_choose) F(snntc_grad_norm_workspace_bytes) \
    F(snntc_grad_norm) F(snntc_adamw_update) F(snntc_adamw_moments)

struct Library {
#define SNNTC_FIELD(f) decltype(&::f) f = nullptr;
    SNNTC_BOUND(SNNTC_FIELD)
#undef SNNTC_FIELD
} lib;

PyObject* g_library_error = nullptr;   // snntc_amd._lib.SnntcLibraryError
PyObject* g_error = nullptr;           // snntc_amd._lib.SnntcError
PyObject* g_params = nullptr;          // snntc_amd._lib.params_array: any sequence -> contiguous float32 vector
PyObject* g_general = nullptr;         // snntc_amd.ops.GENERAL: name of a differentiable op -> its torch.autograd.Function

// Raises a Python exception of class `cls` from code that may run without the GIL (an autograd thread).
[[noreturn]] void raise_class(PyObject* cls, PyObject* (*args)(int, const std::string&), int status, const std::string& msg) {
    PyGILState_STATE gil = PyGILState_Ensure();
    PyObject* a = args(status, msg);
    if (a) PyErr_SetObject(cls, a);
    Py_XDECREF(a);
    python_error err;
    err.persist();
    PyGILState_Release(gil);
    throw std::move(err);
}

PyObject* message_args(int, const std::string& m) { return Py_BuildValue("(s)", m.c_str()); }
PyObject* status_args(int s, const std::string& m) { return Py_BuildValue("(is)", s, m.c_str()); }

// Maps a status code to the exception the reference's Python caller would see.
void check(int status) {
    if (status == SNNTC_OK) return;
    const std::string msg = lib.snntc_last_error();
    if (status == SNNTC_ERR_DIM_MISMATCH || status == SNNTC_ERR_TOO_LARGE || status == SNNTC_ERR_BAD_ARGUMENT)
        TORCH_CHECK_VALUE(false, msg);
    raise_class(g_error, status_args, status, msg);
}

// ---- tensors -------------------------------------------------------------------------------------------------------

std::string shape_text(const Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + (t.dim() == 1 ? ",)" : ")");
}

Tensor dev_f32(const Tensor& t, const char* name, int64_t ndim) {
    if (!t.is_cuda())
        raise_class(g_library_error, message_args, 0, std::string(name) + " lives on " + t.device().str() +
                    ": the SNN-TC ops run on a ROCm GPU only (no CPU fallback)");
    TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, name, " must be float32, got ", t.scalar_type());
    TORCH_CHECK_VALUE(t.dim() == ndim, name, " must have ", ndim, " dimensions, got shape ", shape_text(t));
    return t.contiguous();
}

// A device tensor of float32 or a 16-bit float type.
Tensor dev_float(const Tensor& t, const char* name) {
    if (!t.is_cuda())
        raise_class(g_library_error, message_args, 0, std::string(name) + " lives on " + t.device().str() +
                    ": the SNN-TC ops run on a ROCm GPU only (no CPU fallback)");
    const at::ScalarType s = t.scalar_type();
    TORCH_CHECK_TYPE(s == at::kFloat || s == at::kBFloat16 || s == at::kHalf, name, " must be float32, bfloat16 or float16, got ", s);
    return t.contiguous();
}

int float_type(const Tensor& t) {
    return t.scalar_type() == at::kFloat ? SNNTC_F32 : t.scalar_type() == at::kBFloat16 ? SNNTC_BF16 : SNNTC_F16;
}

void same_device(const Tensor& t, const Tensor& with, const char* name) {
    if (!t.is_cuda())
        raise_class(g_library_error, message_args, 0, std::string(name) + " lives on " + t.device().str() +
                    ": the SNN-TC ops run on a ROCm GPU only (no CPU fallback)");
    TORCH_CHECK_VALUE(t.device() == with.device(), name, " lives on ", t.device().str(), ", not on ", with.device().str());
}

// A float32 tensor of the given shape on the device of `with`; undefined stays undefined.
Tensor f32_like(const Tensor& t, const Tensor& with, at::IntArrayRef sizes, const char* name) {
    if (!t.defined()) return t;
    same_device(t, with, name);
    TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, name, " must be float32, got ", t.scalar_type());
    TORCH_CHECK_VALUE(t.sizes() == sizes, name, " must have shape ", sizes, ", got ", shape_text(t));
    return t.contiguous();
}

Tensor index_like(const Tensor& t, const Tensor& with, const char* name, bool narrow) {
    same_device(t, with, name);
    TORCH_CHECK_TYPE(t.scalar_type() == at::kLong || (narrow && t.scalar_type() == at::kInt), name, " must be ",
                     narrow ? "int64 or int32" : "int64", ", got ", t.scalar_type());
    return t.contiguous();
}

int64_t* i64(const Tensor& t) { return t.defined() ? static_cast<int64_t*>(t.data_ptr()) : nullptr; }
void* raw(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
size_t bytes_of(const Tensor& t) { return t.defined() ? (size_t)t.numel() : 0; }

void no_gradient(std::initializer_list<std::pair<const Tensor*, const char*>> tensors, const char* who) {
    for (const auto& t : tensors)
        TORCH_CHECK_VALUE(!t.first->defined() || !t.first->requires_grad(), who, ": ", t.second, " must not require a gradient");
}

float* f32(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

Tensor scratch(const Tensor& like, size_t bytes) {
    return at::empty({(int64_t)std::max<size_t>(bytes, 256)}, like.options().dtype(at::kByte));
}

Tensor empty(const Tensor& like, at::IntArrayRef sizes) { return at::empty(sizes, like.options()); }

// The first half of an op's [2B,...] output: the spike times.  It shares storage and version counter
// with the whole, so an in-place change of it is seen by the saved whole.
Tensor first_half(const Tensor& y, int64_t B) {
    at::AutoDispatchBelowADInplaceOrView guard;
    Tensor half = y.narrow(0, 0, B);
    torch::autograd::impl::set_version_counter(half, torch::autograd::impl::version_counter(y));
    return half;
}

bool wants_grad(const Tensor& a) { return at::GradMode::is_enabled() && a.requires_grad(); }
bool wants_grad(const Tensor& a, const Tensor& b) { return at::GradMode::is_enabled() && (a.requires_grad() || b.requires_grad()); }

// Whether the native nodes may stand for PyTorch's own machinery: no tangent to carry on, no wrapper without memory of
// its own, no mode, transform or tracer that has to see the operation.
bool plain(std::initializer_list<std::reference_wrapper<const Tensor>> tensors) {
    static const c10::DispatchKeySet special{
        c10::DispatchKey::Python, c10::DispatchKey::Functionalize, c10::DispatchKey::Conjugate, c10::DispatchKey::Negative,
        c10::DispatchKey::ZeroTensor, c10::DispatchKey::Batched, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper};
    if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::any_modes_set() ||
        c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode))
        return false;
    for (const Tensor& t : tensors)
        if (t.defined() && (t.key_set().has_any(special) || t._fw_grad(0).defined())) return false;
    return true;
}

// ---- the ops -------------------------------------------------------------------------------------------------------

using FcParams = std::array<float, 6>;
using CvParams = std::array<float, 12>;

Tensor fc_forward(const Tensor& x, const Tensor& w, const FcParams& p) {
    const int64_t B = x.size(0), I = x.size(1), rows = w.size(0), J = w.size(1);
    const c10::DeviceGuard guard(x.device());
    size_t need = 0;
    check(lib.snntc_fc_forward_workspace_bytes(B, I, J, &need));
    const Tensor ws = scratch(x, need), out = empty(x, {2 * B, J});
    check(lib.snntc_fc_forward(f32(x), f32(w), p.data(), f32(out), B, I, J, rows, ws.data_ptr(), ws.numel(), stream_of(x)));
    return out;
}

struct Grads { Tensor dx, dw, dp; };

Grads fc_backward(const Tensor& grad, const Tensor& x, const Tensor& w, const FcParams& p, const Tensor& y, bool want_dx,
                  bool want_dw, bool want_dp, bool first_half_grad) {
    const int64_t B = x.size(0), I = x.size(1), rows = w.size(0), J = w.size(1);
    TORCH_CHECK_VALUE(y.size(0) == 2 * B && y.size(1) == J && grad.size(1) == J, "Grad/Oldout batch should be 2 * batch: Y ",
                      shape_text(y), ", grad ", shape_text(grad), ", X ", shape_text(x), ", W ", shape_text(w));
    const c10::DeviceGuard guard(x.device());
    size_t need = 0;
    check(lib.snntc_fc_backward_workspace_bytes(B, I, J, &need));
    const Tensor ws = scratch(x, need);
    Grads g;
    if (want_dx) g.dx = empty(x, x.sizes());
    if (want_dw) g.dw = empty(w, w.sizes());
    if (want_dp) g.dp = empty(x, {6});
    // the op only ever reads rows [0,B) of grad, so a caller that holds just those rows passes them as is
    const int64_t grad_rows = first_half_grad && grad.size(0) == B ? 2 * B : grad.size(0);
    check(lib.snntc_fc_backward(f32(grad), f32(x), f32(w), p.data(), f32(y), f32(g.dx), f32(g.dw), f32(g.dp), B, I, J, rows,
                                grad_rows, ws.data_ptr(), ws.numel(), stream_of(x)));
    return g;
}

// Where an op also writes its spike times: pixel (nh + top, nw + left) of the next layer's padded input.
struct Feed { Tensor dst; int64_t top = 0, left = 0; };

Tensor feed_target(const Feed& feed, int64_t B, int64_t C, const char* what) {
    Tensor nx = dev_f32(feed.dst, "next_xpad", 4);
    TORCH_CHECK_VALUE(nx.size(0) == B && nx.size(3) == C, "next_xpad ", shape_text(nx), " does not match batch ", B, " / channels ", C);
    TORCH_CHECK_VALUE(nx.is_same(feed.dst), what, ": next_xpad must be contiguous");
    return nx;
}

// A kernel has written into `t` through its raw pointer: its version counter is advanced, so that autograd
// refuses a backward pass whose saved input has been overwritten by a later forward pass.
void written_behind_autograd(const Tensor& t) { t.unsafeGetTensorImpl()->bump_version(); }

Tensor cv_forward(const Tensor& x, const Tensor& w, const CvParams& p, const Feed& feed) {
    const int64_t B = x.size(0), H = x.size(1), W = x.size(2), C = x.size(3), rows = w.size(0), Kc = w.size(1);
    const c10::DeviceGuard guard(x.device());
    int64_t nh = 0, nw = 0;
    size_t need = 0;
    check(lib.snntc_cv_output_dims(H, W, p.data(), &nh, &nw));
    check(lib.snntc_cv_forward_workspace_bytes(B, H, W, C, Kc, p.data(), &need));
    const Tensor ws = scratch(x, need), out = empty(x, {2 * B, nh, nw, Kc});
    if (!feed.dst.defined()) {
        check(lib.snntc_cv_forward(f32(x), f32(w), p.data(), f32(out), B, H, W, C, Kc, rows, ws.data_ptr(), ws.numel(), stream_of(x)));
        return out;
    }
    const Tensor nx = feed_target(feed, B, Kc, "snncv");
    check(lib.snntc_cv_forward_chained(f32(x), f32(w), p.data(), f32(out), f32(nx), nx.size(1), nx.size(2), feed.top, feed.left,
                                       B, H, W, C, Kc, rows, ws.data_ptr(), ws.numel(), stream_of(x)));
    written_behind_autograd(nx);
    return out;
}

struct Window { int64_t h = 0, w = 0, top = 0, left = 0; };

Grads cv_backward(const Tensor& grad, const Tensor& x, const Tensor& w, const CvParams& p, const Tensor& y, bool want_dx,
                  bool want_dw, bool want_dp, bool first_half_grad, const Window* crop) {
    const int64_t B = x.size(0), H = x.size(1), W = x.size(2), C = x.size(3), rows = w.size(0), Kc = w.size(1);
    TORCH_CHECK_VALUE(y.size(0) == 2 * B && grad.sizes().slice(1) == y.sizes().slice(1) && y.size(3) == Kc,
                      "Grad/Oldout batch should be 2 * batch: Y ", shape_text(y), ", grad ", shape_text(grad), ", X ",
                      shape_text(x), ", W ", shape_text(w));
    const c10::DeviceGuard guard(x.device());
    size_t need = 0;
    check(lib.snntc_cv_backward_workspace_bytes(B, H, W, C, Kc, p.data(), &need));
    const Tensor ws = scratch(x, need);
    const Window win = crop ? *crop : Window{H, W, 0, 0};
    Grads g;
    if (want_dx) g.dx = empty(x, {B, win.h, win.w, C});
    if (want_dw) g.dw = empty(w, w.sizes());
    if (want_dp) g.dp = empty(x, {12});
    const int64_t grad_rows = first_half_grad && grad.size(0) == B ? 2 * B : grad.size(0);
    check(lib.snntc_cv_backward_cropped(f32(grad), f32(x), f32(w), p.data(), f32(y), f32(g.dx), win.h, win.w, win.top, win.left,
                                        f32(g.dw), f32(g.dp), B, H, W, C, Kc, rows, grad_rows, ws.data_ptr(), ws.numel(),
                                        stream_of(x)));
    return g;
}

struct Pads { int64_t top = 0, bottom = 0, left = 0, right = 0; };

Tensor pad_time(const Tensor& x, const Pads& pad, float value) {
    const int64_t B = x.size(0), H = x.size(1), W = x.size(2), C = x.size(3);
    const int64_t Hp = pad.top + H + pad.bottom, Wp = pad.left + W + pad.right;
    const c10::DeviceGuard guard(x.device());
    const Tensor out = empty(x, {B, Hp, Wp, C});
    check(lib.snntc_pad_time_forward(f32(x), f32(out), B, H, W, C, pad.top, pad.left, Hp, Wp, value, stream_of(x)));
    return out;
}

struct PoolShape { int64_t kh, kw, sh, sw, top, left, nh, nw; float pad_value; };

struct Pooled { Tensor y, arg; };

Pooled min_pool(const Tensor& x, const PoolShape& s, bool want_arg, const Feed& feed) {
    const int64_t B = x.size(0), H = x.size(1), W = x.size(2), C = x.size(3);
    const c10::DeviceGuard guard(x.device());
    Pooled r;
    r.y = empty(x, {B, s.nh, s.nw, C});
    if (want_arg) r.arg = at::empty({B, s.nh, s.nw, C}, x.options().dtype(at::kInt));
    int32_t* arg = want_arg ? static_cast<int32_t*>(r.arg.data_ptr()) : nullptr;
    if (!feed.dst.defined()) {
        check(lib.snntc_min_pool_forward(f32(x), f32(r.y), arg, B, H, W, C, s.kh, s.kw, s.sh, s.sw, s.top, s.left, s.nh, s.nw,
                                         s.pad_value, stream_of(x)));
        return r;
    }
    const Tensor nx = feed_target(feed, B, C, "min_pool");
    check(lib.snntc_min_pool_forward_chained(f32(x), f32(r.y), arg, f32(nx), nx.size(1), nx.size(2), feed.top, feed.left, B, H, W,
                                             C, s.kh, s.kw, s.sh, s.sw, s.top, s.left, s.nh, s.nw, s.pad_value, stream_of(x)));
    written_behind_autograd(nx);
    return r;
}

struct LossOut { Tensor loss, grad; };

LossOut time_loss(const Tensor& times, const Tensor& label, bool want_loss, bool want_grad) {
    TORCH_CHECK_VALUE(times.sizes() == label.sizes(), "loss: times ", shape_text(times), " and label ", shape_text(label),
                      " differ in shape");
    const c10::DeviceGuard guard(times.device());
    LossOut r;
    if (want_loss) r.loss = empty(times, {times.size(0)});
    if (want_grad) r.grad = empty(times, times.sizes());
    check(lib.snntc_softmax_time_loss(f32(times), f32(label), f32(r.loss), f32(r.grad), times.size(0), times.size(1),
                                      stream_of(times)));
    return r;
}

// ---- sequences of tokens and choices ---------------------------------------------------------------------------------

struct EmbedArgs { Tensor tokens, table; float scale; bool encode; };

EmbedArgs embed_args(const Tensor& tokens, const Tensor& table, float scale, bool encode) {
    EmbedArgs a{Tensor(), dev_float(table, "table"), scale, encode};
    TORCH_CHECK_VALUE(table.dim() == 2, "table must have 2 dimensions, got shape ", shape_text(table));
    a.tokens = index_like(tokens, a.table, "tokens", true);
    return a;
}

Tensor embed_tokens(const EmbedArgs& a) {
    const c10::DeviceGuard guard(a.table.device());
    std::vector<int64_t> sizes = a.tokens.sizes().vec();
    sizes.push_back(a.table.size(1));
    const Tensor z = at::empty(sizes, a.table.options().dtype(at::kFloat));
    check(lib.snntc_embed_forward(raw(a.tokens), (int)a.tokens.element_size(), raw(a.table), float_type(a.table), f32(z), a.tokens.numel(),
                                  a.table.size(0), a.table.size(1), a.scale, a.encode, stream_of(a.table)));
    return z;
}

Tensor embed_tokens_grad(const Tensor& grad_in, const EmbedArgs& a) {
    std::vector<int64_t> sizes = a.tokens.sizes().vec();
    sizes.push_back(a.table.size(1));
    const Tensor grad = f32_like(grad_in, a.table, sizes, "grad");
    const c10::DeviceGuard guard(a.table.device());
    const int64_t N = a.tokens.numel(), V = a.table.size(0), D = a.table.size(1);
    size_t need = 0;
    check(lib.snntc_embed_backward_workspace_bytes(N, V, D, &need));
    const Tensor ws = need ? scratch(a.table, need) : Tensor(), d = empty(a.table, a.table.sizes());
    check(lib.snntc_embed_backward(f32(grad), raw(a.tokens), (int)a.tokens.element_size(), raw(a.table), float_type(a.table), raw(d), N, V,
                                   D, a.scale, a.encode, raw(ws), bytes_of(ws), stream_of(a.table)));
    return d;
}

struct GatedArgs { Tensor x, gate, state, lengths; };

GatedArgs gated_args(const Tensor& x_in, const Tensor& gate_in, const Tensor& state, const Tensor& lengths) {
    GatedArgs a;
    a.x = dev_f32(x_in, "x", 3);
    TORCH_CHECK_VALUE(gate_in.sizes() == a.x.sizes(), "gate ", shape_text(gate_in), " does not match x ", shape_text(a.x));
    a.gate = dev_float(gate_in, "gate");
    same_device(a.gate, a.x, "gate");
    a.state = f32_like(state, a.x, {a.x.size(0), a.x.size(2)}, "state");
    if (lengths.defined()) {
        a.lengths = index_like(lengths, a.x, "lengths", false);
        TORCH_CHECK_VALUE(a.lengths.dim() == 1 && a.lengths.size(0) == a.x.size(0), "lengths must have one entry per sequence, got shape ",
                          shape_text(a.lengths), " for x ", shape_text(a.x));
    }
    return a;
}

struct Scanned { Tensor y, final; };

// (Undefined where the sequences need none.)
Tensor gated_scratch(const GatedArgs& a) {
    size_t need = 0;
    check(lib.snntc_gated_scan_workspace_bytes(a.x.size(0), a.x.size(1), a.x.size(2), &need));
    return need ? scratch(a.x, need) : Tensor();
}

Scanned gated_scan(const GatedArgs& a) {
    const c10::DeviceGuard guard(a.x.device());
    const int64_t B = a.x.size(0), T = a.x.size(1), D = a.x.size(2);
    const Tensor ws = gated_scratch(a);
    Scanned r{empty(a.x, a.x.sizes()), empty(a.x, {B, D})};
    check(lib.snntc_gated_scan_forward(f32(a.x), raw(a.gate), float_type(a.gate), f32(a.state), i64(a.lengths), f32(r.y), f32(r.final), B,
                                       T, D, raw(ws), bytes_of(ws), stream_of(a.x)));
    return r;
}

struct ScanGrads { Tensor dx, dgate, dstate; };

ScanGrads gated_scan_grad(const Tensor& dy_in, const Tensor& dfinal_in, const GatedArgs& a, const Tensor& y_in, bool want_dx, bool want_dgate,
                          bool want_dstate) {
    const c10::DeviceGuard guard(a.x.device());
    const int64_t B = a.x.size(0), T = a.x.size(1), D = a.x.size(2);
    TORCH_CHECK_VALUE(y_in.defined(), "y, the forward output, is required");
    const Tensor y = f32_like(y_in, a.x, a.x.sizes(), "y"), dy = f32_like(dy_in, a.x, a.x.sizes(), "grad_y"),
                 dfinal = f32_like(dfinal_in, a.x, {B, D}, "grad_final");
    const Tensor ws = gated_scratch(a);
    ScanGrads g;
    if (want_dx) g.dx = empty(a.x, a.x.sizes());
    if (want_dgate) g.dgate = empty(a.gate, a.x.sizes());
    if (want_dstate) g.dstate = empty(a.x, {B, D});
    check(lib.snntc_gated_scan_backward(f32(dy), f32(dfinal), f32(a.x), raw(a.gate), float_type(a.gate), f32(y), f32(a.state),
                                        i64(a.lengths), f32(g.dx), raw(g.dgate), f32(g.dstate), B, T, D, raw(ws), bytes_of(ws), stream_of(a.x)));
    return g;
}

Tensor gated_step(const Tensor& x_in, const Tensor& gate_in, const Tensor& state_in, const Tensor& out_in) {
    const Tensor x = dev_f32(x_in, "x", x_in.dim());
    TORCH_CHECK_VALUE(gate_in.sizes() == x.sizes(), "gate ", shape_text(gate_in), " does not match x ", shape_text(x));
    const Tensor gate = dev_float(gate_in, "gate");
    same_device(gate, x, "gate");
    const Tensor state = f32_like(state_in, x, x.sizes(), "state");
    const c10::DeviceGuard guard(x.device());
    Tensor out = f32_like(out_in, x, x.sizes(), "out");
    if (!out.defined()) out = empty(x, x.sizes());
    else TORCH_CHECK_VALUE(out.is_same(out_in), "out must be contiguous");
    check(lib.snntc_gated_step(f32(x), raw(gate), float_type(gate), f32(state), f32(out), x.numel(), stream_of(x)));
    if (out_in.defined()) written_behind_autograd(out);
    return out;
}

// times[..., J] with one token per row.
struct ChoiceArgs { Tensor times, tokens, weight; int64_t rows = 0, J = 0; };

ChoiceArgs choice_args(const Tensor& times, const Tensor& tokens, const Tensor& weight, const char* name) {
    ChoiceArgs a;
    a.times = dev_float(times, "times");
    TORCH_CHECK_VALUE(times.dim() >= 2, "times must have at least 2 dimensions, got shape ", shape_text(times));
    const at::IntArrayRef rows = times.sizes().slice(0, times.dim() - 1);
    a.tokens = index_like(tokens, a.times, name, false);
    TORCH_CHECK_VALUE(tokens.sizes() == rows, name, " must have shape ", rows, ", got ", shape_text(tokens));
    a.weight = f32_like(weight, a.times, rows, "weight");
    a.rows = tokens.numel();
    a.J = times.size(-1);
    return a;
}

Tensor row_floats(const ChoiceArgs& a, at::IntArrayRef sizes) { return at::empty(sizes, a.times.options().dtype(at::kFloat)); }

// (Undefined where the rows need none.)
Tensor choice_scratch(const ChoiceArgs& a) {
    size_t need = 0;
    check(lib.snntc_choice_workspace_bytes(a.rows, a.J, &need));
    return need ? scratch(a.times, need) : Tensor();
}

Tensor time_logp(const ChoiceArgs& a) {
    const c10::DeviceGuard guard(a.times.device());
    const Tensor ws = choice_scratch(a), logp = row_floats(a, a.tokens.sizes());
    check(lib.snntc_time_logp(raw(a.times), float_type(a.times), i64(a.tokens), f32(a.weight), f32(logp), nullptr, a.rows, a.J,
                              raw(ws), bytes_of(ws), stream_of(a.times)));
    return logp;
}

// Loss per row or pair, log-probabilities and, as asked for, the gradient of the objective or what its backward pass needs.
struct ChoiceOut { Tensor loss, logp, dtimes, stats, coef; };

struct PolicyIn { Tensor old_logp, advantage, ref_logp; float low, high, kl; };

ChoiceOut policy_loss(const ChoiceArgs& a, const PolicyIn& p, bool want_grad, bool save) {
    const c10::DeviceGuard guard(a.times.device());
    const at::IntArrayRef rows = a.tokens.sizes();
    TORCH_CHECK_VALUE(p.old_logp.defined() && p.advantage.defined(), "old_logp and advantage are required");
    const Tensor old_logp = f32_like(p.old_logp, a.times, rows, "old_logp"), advantage = f32_like(p.advantage, a.times, rows, "advantage"),
                 ref = f32_like(p.ref_logp, a.times, rows, "ref_logp");
    const Tensor ws = choice_scratch(a);
    ChoiceOut r{row_floats(a, rows), row_floats(a, rows), Tensor(), Tensor(), Tensor()};
    if (want_grad) r.dtimes = empty(a.times, a.times.sizes());
    if (save) { r.stats = row_floats(a, {a.rows, 2}); r.coef = row_floats(a, {a.rows}); }
    check(lib.snntc_policy_loss(raw(a.times), float_type(a.times), i64(a.tokens), f32(old_logp), f32(advantage), f32(ref), f32(a.weight),
                                p.low, p.high, p.kl, f32(r.loss), f32(r.logp), f32(r.stats), f32(r.coef), raw(r.dtimes), a.rows, a.J,
                                raw(ws), bytes_of(ws), stream_of(a.times)));
    return r;
}

ChoiceOut preference_loss(const ChoiceArgs& a, const Tensor& ref_in, float beta, float smoothing, bool want_grad, bool save) {
    const c10::DeviceGuard guard(a.times.device());
    TORCH_CHECK_VALUE(a.tokens.dim() == 2 && a.tokens.size(0) % 2 == 0, "tokens must be [2 pairs, steps], got shape ", shape_text(a.tokens));
    TORCH_CHECK_VALUE(ref_in.defined(), "ref_logp is required");
    const int64_t P = a.tokens.size(0) / 2, T = a.tokens.size(1);
    const Tensor ref = f32_like(ref_in, a.times, {2 * P}, "ref_logp");
    size_t need = 0;
    check(lib.snntc_preference_workspace_bytes(P, T, a.J, &need));
    const Tensor ws = scratch(a.times, need);
    ChoiceOut r{row_floats(a, {P}), row_floats(a, {2 * P}), Tensor(), Tensor(), Tensor()};
    if (want_grad) r.dtimes = empty(a.times, a.times.sizes());
    if (save) { r.stats = row_floats(a, {a.rows, 2}); r.coef = row_floats(a, {a.rows}); }
    check(lib.snntc_preference_loss(raw(a.times), float_type(a.times), i64(a.tokens), f32(ref), f32(a.weight), beta, smoothing, f32(r.loss),
                                    f32(r.logp), f32(r.stats), f32(r.coef), raw(r.dtimes), P, T, a.J, ws.data_ptr(), ws.numel(),
                                    stream_of(a.times)));
    return r;
}

Tensor loss_total(const Tensor& loss, const Tensor& weight) {
    const Tensor total = empty(loss, {});
    check(lib.snntc_loss_total(f32(loss), f32(weight), f32(total), loss.numel(), stream_of(loss)));
    return total;
}

// An objective, and what its gradient is made from if that is wanted (`save`).
struct Objective { Tensor total, stats, coef; };

Objective policy_objective(const ChoiceArgs& a, const PolicyIn& p, bool save) {
    const ChoiceOut r = policy_loss(a, p, false, save);
    const c10::DeviceGuard guard(a.times.device());
    return {loss_total(r.loss, a.weight), r.stats, r.coef};
}

Objective preference_objective(const ChoiceArgs& a, const Tensor& ref, float beta, float smoothing, bool save) {
    const ChoiceOut r = preference_loss(a, ref, beta, smoothing, false, save);
    const c10::DeviceGuard guard(a.times.device());
    return {loss_total(r.loss, Tensor()), r.stats, r.coef};
}

// The gradient of an objective by the times, from the row statistics and the derivative by each row's log-probability that it has left.
Tensor objective_grad(const ChoiceArgs& a, const Tensor& stats_in, const Tensor& coef_in, const Tensor& upstream) {
    const Tensor stats = f32_like(stats_in, a.times, {a.rows, 2}, "stats"), coef = f32_like(coef_in, a.times, {a.rows}, "coef"),
                 up = f32_like(upstream, a.times, {}, "upstream");
    const c10::DeviceGuard guard(a.times.device());
    const Tensor d = empty(a.times, a.times.sizes());
    check(lib.snntc_time_logp_backward(raw(a.times), float_type(a.times), i64(a.tokens), f32(stats), f32(coef), f32(up), raw(d), a.rows, a.J,
                                       stream_of(a.times)));
    return d;
}

// ---- choices by rules --------------------------------------------------------------------------------------------------

// A number for all sequences, or a tensor with one for each.
struct PerRow { Tensor each; float all; };

struct RuleIn { Tensor history, lengths, prompts; PerRow repetition, presence, frequency; Tensor delay, allowed; };

// times[..., J] and what rules it; `c` points into the tensors.
struct RuleSet {
    Tensor times, history, lengths, prompts, repetition, presence, frequency, delay, allowed;
    int64_t rows = 0, J = 0;
    snntc_rules c{};
};

RuleSet rule_set(const Tensor& times, const RuleIn& in) {
    RuleSet r;
    r.times = dev_float(times, "times");
    TORCH_CHECK_VALUE(times.dim() >= 2, "times must have at least 2 dimensions, got shape ", shape_text(times));
    const at::IntArrayRef lead = times.sizes().slice(0, times.dim() - 1);
    r.J = times.size(-1);
    r.rows = 1;
    for (const int64_t n : lead) r.rows *= n;
    int64_t sequences = 0;
    if (in.history.defined()) {
        r.history = index_like(in.history, r.times, "history", false);
        TORCH_CHECK_VALUE(r.history.dim() == 2, "history must be [sequences, tokens], got shape ", shape_text(r.history));
        sequences = r.history.size(0);
        TORCH_CHECK_VALUE(sequences ? r.rows % sequences == 0 : r.rows == 0, "times ", shape_text(times), " do not divide into the ", sequences,
                          " sequences of history");
        if (in.lengths.defined()) {
            r.lengths = index_like(in.lengths, r.times, "lengths", false);
            TORCH_CHECK_VALUE(r.lengths.sizes() == lead, "lengths must have one entry per row of times, got shape ", shape_text(r.lengths),
                              " for times ", shape_text(times));
        }
        if (in.prompts.defined()) {
            r.prompts = index_like(in.prompts, r.times, "prompts", false);
            TORCH_CHECK_VALUE(r.prompts.dim() == 1 && r.prompts.size(0) == sequences, "prompts must have one entry per sequence of history, got shape ",
                              shape_text(r.prompts));
        }
    } else {
        TORCH_CHECK_VALUE(!in.lengths.defined() && !in.prompts.defined() && !in.repetition.each.defined() && !in.presence.each.defined() &&
                              !in.frequency.each.defined(), "lengths, prompts and penalties per sequence need a history");
    }
    r.repetition = f32_like(in.repetition.each, r.times, {sequences}, "repetition");
    r.presence = f32_like(in.presence.each, r.times, {sequences}, "presence");
    r.frequency = f32_like(in.frequency.each, r.times, {sequences}, "frequency");
    // one row for all, or one for each row of times
    const auto one_row = [&](const Tensor& t) { return t.dim() == 1; };
    std::vector<int64_t> sizes = lead.vec();
    if (in.delay.defined()) {
        sizes.push_back(r.J);
        r.delay = f32_like(in.delay, r.times, one_row(in.delay) ? at::IntArrayRef(r.J) : at::IntArrayRef(sizes), "delay");
        sizes.pop_back();
    }
    if (in.allowed.defined()) {
        const int64_t words = (r.J + 31) / 32;
        sizes.push_back(words);
        same_device(in.allowed, r.times, "allowed");
        TORCH_CHECK_TYPE(in.allowed.scalar_type() == at::kInt, "allowed must be int32, 32 outputs a word, got ", in.allowed.scalar_type());
        TORCH_CHECK_VALUE(one_row(in.allowed) ? in.allowed.size(0) == words : in.allowed.sizes() == at::IntArrayRef(sizes), "allowed must have ", words,
                          " words, or so many per row of times, got shape ", shape_text(in.allowed), " for times ", shape_text(times));
        r.allowed = in.allowed.contiguous();
    }
    snntc_rules& c = r.c;
    c.history = i64(r.history);
    c.history_rows = sequences;
    c.history_len = r.history.defined() ? r.history.size(1) : 0;
    c.lengths = i64(r.lengths); c.prompts = i64(r.prompts);
    c.repetition = f32(r.repetition); c.presence = f32(r.presence); c.frequency = f32(r.frequency);
    c.repetition_all = in.repetition.all; c.presence_all = in.presence.all; c.frequency_all = in.frequency.all;
    c.delay = f32(r.delay);
    c.delay_rows = r.delay.defined() && r.delay.dim() > 1 ? r.rows : 1;
    c.allowed = static_cast<const int32_t*>(raw(r.allowed));
    c.allowed_rows = r.allowed.defined() && r.allowed.dim() > 1 ? r.rows : 1;
    return r;
}

Tensor rule_times(const RuleSet& r) {
    const c10::DeviceGuard guard(r.times.device());
    const Tensor out = empty(r.times, r.times.sizes());
    check(lib.snntc_rule_times(raw(r.times), float_type(r.times), &r.c, raw(out), r.rows, r.J, stream_of(r.times)));
    return out;
}

Tensor rule_times_grad(const Tensor& grad_in, const RuleSet& r) {
    same_device(grad_in, r.times, "grad");
    TORCH_CHECK_TYPE(grad_in.scalar_type() == r.times.scalar_type(), "grad must be ", r.times.scalar_type(), " as times are, got ",
                     grad_in.scalar_type());
    TORCH_CHECK_VALUE(grad_in.sizes() == r.times.sizes(), "grad ", shape_text(grad_in), " does not match times ", shape_text(r.times));
    const c10::DeviceGuard guard(r.times.device());
    const Tensor grad = grad_in.contiguous(), d = empty(r.times, r.times.sizes());
    check(lib.snntc_rule_times_backward(raw(grad), raw(r.times), float_type(r.times), &r.c, raw(d), r.rows, r.J, stream_of(r.times)));
    return d;
}

struct Choice { Tensor tokens, logp; };

Choice choose_tokens(const RuleSet& r, const Tensor& uniform_in, const PerRow& temperature) {
    const at::IntArrayRef lead = r.times.sizes().slice(0, r.times.dim() - 1);
    const Tensor uniform = f32_like(uniform_in, r.times, lead, "uniform"), heat = f32_like(temperature.each, r.times, lead, "temperature");
    TORCH_CHECK_VALUE(uniform.defined() || (!heat.defined() && temperature.all == 0.0f), "uniform is required unless temperature is 0");
    const c10::DeviceGuard guard(r.times.device());
    size_t need = 0;
    check(lib.snntc_choose_workspace_bytes(r.rows, r.J, &need));
    const Tensor ws = need ? scratch(r.times, need) : Tensor();
    Choice out{at::empty(lead, r.times.options().dtype(at::kLong)), at::empty(lead, r.times.options().dtype(at::kFloat))};
    check(lib.snntc_choose(raw(r.times), float_type(r.times), f32(uniform), f32(heat), temperature.all, &r.c, i64(out.tokens), f32(out.logp), r.rows,
                           r.J, raw(ws), bytes_of(ws), stream_of(r.times)));
    return out;
}

// ---- the update over many tensors --------------------------------------------------------------------------------------

// Device tensors of one type each on one device, by their addresses.
struct TensorList {
    std::vector<Tensor> keep;
    std::vector<void*> at;
    std::vector<int> types;
    std::vector<int64_t> n;
    void reserve(size_t tensors) { keep.reserve(tensors); at.reserve(tensors); types.reserve(tensors); n.reserve(tensors); }
};

void add_tensor(TensorList& list, const Tensor& t) {
    list.at.push_back(t.numel() ? t.data_ptr() : nullptr);
    list.n.push_back(t.numel());
    list.keep.push_back(t);
}

void on_device(const Tensor& t, const Tensor& with, const char* who, const char* what, size_t i) {
    if (!t.is_cuda())
        raise_class(g_library_error, message_args, 0, std::string(who) + ": " + what + " " + std::to_string(i) + " lives on " + t.device().str() +
                    ": the SNN-TC ops run on a ROCm GPU only (no CPU fallback)");
    TORCH_CHECK_VALUE(t.device() == with.device(), who, ": ", what, " ", i, " lives on ", t.device().str(), ", not on ", with.device().str());
}

bool is_float(const Tensor& t) {
    return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf;
}

TensorList gradients(const std::vector<Tensor>& gs, const char* who) {
    TensorList list;
    list.reserve(gs.size());
    for (size_t i = 0; i < gs.size(); ++i) {
        on_device(gs[i], gs[0], who, "gradient", i);
        TORCH_CHECK_TYPE(is_float(gs[i]), who, ": gradient ", i, " must be float32, bfloat16 or float16, got ", gs[i].scalar_type());
        add_tensor(list, gs[i].contiguous());
        list.types.push_back(float_type(gs[i]));
    }
    return list;
}

Tensor grad_norm(const std::vector<Tensor>& gs) {
    TORCH_CHECK_VALUE(!gs.empty(), "grad_norm: no gradients");
    on_device(gs[0], gs[0], "grad_norm", "gradient", 0);
    const c10::DeviceGuard guard(gs[0].device());
    const TensorList g = gradients(gs, "grad_norm");
    size_t need = 0;
    check(lib.snntc_grad_norm_workspace_bytes(g.n.data(), (int64_t)g.n.size(), &need));
    const Tensor ws = scratch(gs[0], need), norm = at::empty({}, gs[0].options().dtype(at::kFloat));
    check(lib.snntc_grad_norm(g.at.data(), g.types.data(), g.n.data(), (int64_t)g.n.size(), f32(norm), ws.data_ptr(), ws.numel(), stream_of(gs[0])));
    return norm;
}

// A tensor that the update writes: contiguous, of the given type and size.
void add_written(TensorList& list, const Tensor& t, const Tensor& with, at::ScalarType type, int64_t n, const char* what, size_t i) {
    on_device(t, with, "adamw", what, i);
    TORCH_CHECK_TYPE(t.scalar_type() == type, "adamw: ", what, " ", i, " must be ", type, ", got ", t.scalar_type());
    TORCH_CHECK_VALUE(t.is_contiguous() && t.numel() == n, "adamw: ", what, " ", i, " must be contiguous with ", n, " elements, got shape ", shape_text(t));
    add_tensor(list, t);
}

int64_t state_blocks(int64_t n) { return (n + SNNTC_STATE_BLOCK - 1) / SNNTC_STATE_BLOCK; }

// No two written tensors may overlap, nor a written one with one that is read.
struct Span { const char* from; const char* to; bool written; };
void no_overlap(std::vector<Span>& spans) {
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
    const char *written = nullptr, *any = nullptr;
    for (const Span& s : spans) {
        TORCH_CHECK_VALUE(!(s.from < written || (s.written && s.from < any)), "adamw: two of the tensors overlap, of which one is updated");
        if (s.written) written = std::max(written, s.to);
        any = std::max(any, s.to);
    }
}
void add_span(std::vector<Span>& spans, const Tensor& t, bool written) {
    if (t.defined() && t.numel()) spans.push_back({static_cast<const char*>(t.data_ptr()), static_cast<const char*>(t.data_ptr()) + t.nbytes(), written});
}
void add_spans(std::vector<Span>& spans, const TensorList& list, bool written) {
    for (const Tensor& t : list.keep) add_span(spans, t, written);
}

struct Moments { std::vector<Tensor> first, second, first_scale, second_scale; bool coded; };

void moment_lists(const Moments& m, const std::vector<Tensor>& sizes, TensorList (&out)[4]) {
    const size_t n = sizes.size();
    TORCH_CHECK_VALUE(m.first.size() == n && m.second.size() == n && (!m.coded || (m.first_scale.size() == n && m.second_scale.size() == n)),
                      "adamw: as many states and scales are needed as there are tensors (", n, ")");
    for (TensorList& list : out) list.reserve(n);
    for (size_t i = 0; i < n; ++i) {
        const int64_t k = sizes[i].numel();
        add_written(out[0], m.first[i], sizes[0], m.coded ? at::kByte : at::kFloat, k, "first", i);
        add_written(out[1], m.second[i], sizes[0], m.coded ? at::kByte : at::kFloat, k, "second", i);
        if (!m.coded) continue;
        add_written(out[2], m.first_scale[i], sizes[0], at::kFloat, state_blocks(k), "first_scale", i);
        add_written(out[3], m.second_scale[i], sizes[0], at::kFloat, state_blocks(k), "second_scale", i);
    }
}

void adamw_update(const std::vector<Tensor>& ws, const std::vector<Tensor>& gs, const Moments& moments, const Tensor& steps, const Tensor& norm,
                  snntc_adamw how) {
    TORCH_CHECK_VALUE(ws.size() == gs.size(), "adamw: ", ws.size(), " weight tensors but ", gs.size(), " gradients");
    const Tensor& with = ws.empty() ? steps : ws[0];            // (no tensors: a step's number on the device still counts)
    if (!with.defined()) return;
    on_device(with, with, "adamw", ws.empty() ? "step" : "weight", 0);
    const c10::DeviceGuard guard(with.device());
    TensorList w, state[4];
    const TensorList g = gradients(gs, "adamw");
    w.reserve(ws.size());
    for (size_t i = 0; i < ws.size(); ++i) {
        TORCH_CHECK_TYPE(is_float(ws[i]), "adamw: weight ", i, " must be float32, bfloat16 or float16, got ", ws[i].scalar_type());
        TORCH_CHECK_VALUE(gs[i].sizes() == ws[i].sizes() && gs[i].scalar_type() == ws[i].scalar_type() && gs[i].device() == ws[i].device(),
                          "adamw: gradient ", i, " does not match its weight tensor");
        add_written(w, ws[i], ws[0], ws[i].scalar_type(), ws[i].numel(), "weight", i);
    }
    moment_lists(moments, ws, state);
    Tensor scratch_ws;
    if (steps.defined()) {
        on_device(steps, with, "adamw", "step", 0);
        TORCH_CHECK_TYPE(steps.scalar_type() == at::kLong && steps.numel() == 1, "adamw: a step on the device is one int64");
        how.steps = i64(steps);
        scratch_ws = scratch(with, SNNTC_ADAMW_WORKSPACE_BYTES);
    }
    if (norm.defined()) {
        on_device(norm, with, "adamw", "norm", 0);
        TORCH_CHECK_TYPE(norm.scalar_type() == at::kFloat && norm.numel() == 1, "adamw: norm is one float32");
        how.norm = f32(norm);
    }
    std::vector<Span> spans;
    spans.reserve(6 * ws.size() + 2);
    add_spans(spans, w, true); add_spans(spans, g, false);
    for (const TensorList& s : state) add_spans(spans, s, true);
    add_span(spans, steps, true); add_span(spans, norm, false);
    no_overlap(spans);
    const auto floats = [](TensorList& l) { return reinterpret_cast<float* const*>(l.at.data()); };
    check(lib.snntc_adamw_update(w.at.data(), g.at.data(), state[0].at.data(), state[1].at.data(), moments.coded ? floats(state[2]) : nullptr,
                                 moments.coded ? floats(state[3]) : nullptr, g.types.data(), w.n.data(), (int64_t)w.n.size(), &how, raw(scratch_ws),
                                 bytes_of(scratch_ws), stream_of(with)));
    const auto changed = [](const Tensor& t) { if (!t.is_inference()) written_behind_autograd(t); };
    for (const Tensor& t : ws) changed(t);
    for (const TensorList& s : state)
        for (const Tensor& t : s.keep) changed(t);
    if (steps.defined()) changed(steps);
}

// A contiguous tensor of its own on a part of another's memory.
Tensor part_of(const Tensor& all, int64_t offset, at::IntArrayRef sizes) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
    impl->set_storage_offset(offset);
    impl->set_sizes_contiguous(sizes);
    return Tensor(std::move(impl));
}

struct MomentsOut { std::vector<Tensor> first, second; };

MomentsOut adamw_moments(const Moments& m) {
    MomentsOut out;
    if (m.first.empty() && m.second.empty()) return out;
    TORCH_CHECK_VALUE(!m.first.empty(), "adamw: as many states and scales are needed as there are tensors (0)");
    on_device(m.first[0], m.first[0], "adamw", "first", 0);
    const c10::DeviceGuard guard(m.first[0].device());
    TensorList state[4], to[2];
    moment_lists(m, m.first, state);
    // parts of one allocation: by themselves the tensors of a small network took as long as all the rest of the call (16 tensors 38 us)
    int64_t total = 0;
    for (const Tensor& t : m.first) total += (t.numel() + 63) / 64 * 128;
    const Tensor all = at::empty({total}, m.first[0].options().dtype(at::kFloat));
    int64_t used = 0;
    for (TensorList& list : to) list.reserve(m.first.size());
    for (const Tensor& t : m.first)
        for (int k = 0; k < 2; ++k) {
            add_tensor(to[k], part_of(all, used, t.sizes()));
            used += (t.numel() + 63) / 64 * 64;
        }
    const auto codes = [](TensorList& l) { return reinterpret_cast<const uint8_t* const*>(l.at.data()); };
    const auto floats = [](TensorList& l) { return reinterpret_cast<float* const*>(l.at.data()); };
    check(lib.snntc_adamw_moments(codes(state[0]), codes(state[1]), floats(state[2]), floats(state[3]), floats(to[0]), floats(to[1]),
                                  state[0].n.data(), (int64_t)state[0].n.size(), stream_of(m.first[0])));
    out.first = std::move(to[0].keep);
    out.second = std::move(to[1].keep);
    return out;
}

// ---- autograd nodes ------------------------------------------------------------------------------------------------

template <typename N>
Tensor with_history(Tensor out, const std::shared_ptr<N>& node) {
    torch::autograd::set_history(out, node);
    return out;
}

template <typename N>
std::shared_ptr<N> make_node(std::initializer_list<std::reference_wrapper<const Tensor>> inputs) {
    std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
    torch::autograd::edge_list edges;
    for (const Tensor& t : inputs) edges.push_back(torch::autograd::impl::gradient_edge(t));
    node->set_next_edges(std::move(edges));
    return node;
}

struct LayerNode : public Node {
    SavedVariable x, w, y;
    void save(const Tensor& x_, const Tensor& w_, const Tensor& y_) {
        x = SavedVariable(x_, false); w = SavedVariable(w_, false); y = SavedVariable(y_, false);
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data(); w.reset_data(); y.reset_data();
    }
};

struct FcNode : public LayerNode {
    FcParams params;
    bool first_half;                    // the upstream gradient has the rows of the spike times only
    std::string name() const override { return "SnnFcBackward"; }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(2);
        if (!grads[0].defined()) return out;
        const Tensor X = x.unpack(), Wt = w.unpack(), Y = y.unpack();
        at::AutoGradMode no_grad(false);
        Grads g = fc_backward(dev_f32(grads[0], "grad", 2), X, Wt, params, Y, task_should_compute_output(0),
                              task_should_compute_output(1), false, first_half);
        out[0] = g.dx; out[1] = g.dw;
        return out;
    }
};

struct CvNode : public LayerNode {
    CvParams params;
    bool first_half;
    std::optional<Window> crop;
    std::string name() const override { return "SnnCvBackward"; }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(2);
        if (!grads[0].defined()) return out;
        const Tensor X = x.unpack(), Wt = w.unpack(), Y = y.unpack();
        at::AutoGradMode no_grad(false);
        Grads g = cv_backward(dev_f32(grads[0], "grad", 4), X, Wt, params, Y, task_should_compute_output(0),
                              task_should_compute_output(1), false, first_half, crop ? &*crop : nullptr);
        out[0] = g.dx; out[1] = g.dw;
        return out;
    }
};

struct PoolNode : public Node {
    SavedVariable arg;
    PoolShape shape;
    std::array<int64_t, 4> in;
    std::string name() const override { return "SnnMinPoolBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        arg.reset_data();
    }
    variable_list apply(variable_list&& grads) override;
};

struct PadNode : public Node {
    std::array<int64_t, 4> in;
    int64_t top, left;
    std::string name() const override { return "SnnPadTimeBackward"; }
    variable_list apply(variable_list&& grads) override;
};

struct LossNode : public Node {
    SavedVariable grad;
    std::string name() const override { return "SoftmaxTimeLossBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        grad.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return variable_list(1);
        return {grad.unpack() * grads[0]};                  // (differentiable in the upstream factor)
    }
};

Tensor min_pool_grad(const Tensor& gy, const Tensor& arg, const std::array<int64_t, 4>& in, const PoolShape& s) {
    TORCH_CHECK_VALUE(arg.sizes() == gy.sizes() && arg.scalar_type() == at::kInt && arg.is_contiguous(),
                      "arg must be the contiguous int32 tensor min_pool returned");
    const c10::DeviceGuard guard(gy.device());
    const Tensor dx = empty(gy, {in[0], in[1], in[2], in[3]});
    check(lib.snntc_min_pool_backward(f32(gy), static_cast<int32_t*>(arg.data_ptr()), f32(dx), in[0], in[1], in[2], in[3], s.kh, s.kw,
                                      s.sh, s.sw, s.top, s.left, gy.size(1), gy.size(2), stream_of(gy)));
    return dx;
}

Tensor pad_time_grad(const Tensor& dxpad, const std::array<int64_t, 4>& in, int64_t top, int64_t left) {
    const c10::DeviceGuard guard(dxpad.device());
    const Tensor dx = empty(dxpad, {in[0], in[1], in[2], in[3]});
    check(lib.snntc_pad_time_backward(f32(dxpad), f32(dx), in[0], in[1], in[2], in[3], top, left, dxpad.size(1), dxpad.size(2),
                                      stream_of(dxpad)));
    return dx;
}

variable_list PoolNode::apply(variable_list&& grads) {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined() || !task_should_compute_output(0)) return variable_list(1);
    const Tensor a = arg.unpack();
    at::AutoGradMode no_grad(false);
    return {min_pool_grad(dev_f32(grads[0], "grad_y", 4), a, in, shape)};
}

variable_list PadNode::apply(variable_list&& grads) {
    if (!grads[0].defined() || !task_should_compute_output(0)) return variable_list(1);
    at::AutoGradMode no_grad(false);
    return {pad_time_grad(dev_f32(grads[0], "dxpad", 4), in, top, left)};
}

// `times`: hand out the spike times Y[:B] rather than the whole [2B,...] output.
Tensor fc_layer(const Tensor& x_in, const Tensor& w_in, const FcParams& p, bool times) {
    const Tensor x = dev_f32(x_in, "X", 2), w = dev_f32(w_in, "W", 2);
    Tensor y;
    {
        at::AutoGradMode no_grad(false);
        y = fc_forward(x, w, p);
    }
    Tensor out = times ? first_half(y, x.size(0)) : y;
    if (!wants_grad(x, w)) return out;
    auto node = make_node<FcNode>({x, w});
    node->params = p; node->first_half = times;
    // the whole output is handed out as it is: it is saved as a detached alias, or it would keep itself alive
    node->save(x, w, times ? y : y.detach());
    return with_history(out, node);
}

Tensor cv_layer(const Tensor& x_grad, const Tensor& x, const Tensor& w, const CvParams& p, bool times,
                const std::optional<Window>& crop, const Feed& feed) {
    Tensor y;
    {
        at::AutoGradMode no_grad(false);
        y = cv_forward(x, w, p, feed);
    }
    Tensor out = times ? first_half(y, x.size(0)) : y;
    if (!wants_grad(x_grad, w)) return out;
    auto node = make_node<CvNode>({x_grad, w});
    node->params = p; node->first_half = times; node->crop = crop;
    node->save(x, w, times ? y : y.detach());
    return with_history(out, node);
}

// SNN_conv with SAME padding on the un-padded image x: `xpad`, if given, is the layer's padded input buffer and
// already holds x.
Tensor cv_same(const Tensor& x_in, const Tensor& w_in, const CvParams& p, const Pads& pad, const Tensor& xpad_in, const Feed& feed) {
    const Tensor x = dev_f32(x_in, "X", 4), w = dev_f32(w_in, "W", 2);
    const int64_t B = x.size(0), H = x.size(1), W = x.size(2), C = x.size(3);
    Tensor xpad = xpad_in;
    if (!xpad.defined()) {
        at::AutoGradMode no_grad(false);
        xpad = pad.top || pad.bottom || pad.left || pad.right ? pad_time(x, pad, p[0]) : x;
    } else {
        TORCH_CHECK_VALUE((xpad.sizes() == at::IntArrayRef{B, pad.top + H + pad.bottom, pad.left + W + pad.right, C}),
                          "padded buffer ", shape_text(xpad), " does not match input ", shape_text(x), " and its pads");
        xpad = dev_f32(xpad, "X", 4);
    }
    return cv_layer(x, xpad, w, p, true, Window{H, W, pad.top, pad.left}, feed);
}

Tensor pool_layer(const Tensor& x_in, const PoolShape& s, const Feed& feed) {
    const Tensor x = dev_f32(x_in, "x", 4);
    const bool grad = wants_grad(x);
    Pooled r;
    {
        at::AutoGradMode no_grad(false);
        r = min_pool(x, s, grad, feed);
    }
    if (!grad) return r.y;
    auto node = make_node<PoolNode>({x});
    node->shape = s;
    node->in = {x.size(0), x.size(1), x.size(2), x.size(3)};
    node->arg = SavedVariable(r.arg, false);
    return with_history(r.y, node);
}

Tensor pad_layer(const Tensor& x_in, const Pads& pad, float value) {
    const Tensor x = dev_f32(x_in, "x", 4);
    Tensor out;
    {
        at::AutoGradMode no_grad(false);
        out = pad_time(x, pad, value);
    }
    if (!wants_grad(x)) return out;
    auto node = make_node<PadNode>({x});
    node->in = {x.size(0), x.size(1), x.size(2), x.size(3)};
    node->top = pad.top; node->left = pad.left;
    return with_history(out, node);
}

Tensor loss_layer(const Tensor& times_in, const Tensor& label_in) {
    const Tensor times = dev_f32(times_in, "times", 2), label = dev_f32(label_in, "label", 2);
    const bool grad = wants_grad(times);
    LossOut r;
    Tensor mean;
    {
        at::AutoGradMode no_grad(false);
        r = time_loss(times, label, true, grad);
        mean = r.loss.mean();
    }
    if (!grad) return mean;
    auto node = make_node<LossNode>({times});
    node->grad = SavedVariable(r.grad, false);
    return with_history(mean, node);
}

void sgd_update(const std::vector<Tensor>& ws, const std::vector<Tensor>& gs, float lr) {
    std::vector<float*> wp;
    std::vector<const float*> gp;
    std::vector<int64_t> n;
    std::vector<Tensor> keep;
    at::AutoGradMode no_grad(false);
    for (size_t i = 0; i < ws.size(); ++i) {
        const Tensor& w = ws[i];
        if (!(w.is_cuda() && w.scalar_type() == at::kFloat && w.is_contiguous()))
            raise_class(g_library_error, message_args, 0, "sgd_update: weight " + std::to_string(i) +
                        " must be a contiguous float32 tensor on a ROCm GPU");
        TORCH_CHECK_VALUE(gs[i].sizes() == w.sizes() && gs[i].scalar_type() == at::kFloat && gs[i].device() == w.device(),
                          "sgd_update: gradient ", i, " does not match its weight tensor");
        keep.push_back(gs[i].contiguous());
        wp.push_back(f32(w));
        gp.push_back(f32(keep.back()));
        n.push_back(w.numel());
    }
    const c10::DeviceGuard guard(ws[0].device());
    check(lib.snntc_sgd_update(wp.data(), gp.data(), n.data(), (int64_t)n.size(), lr, stream_of(ws[0])));
}

// ---- layers and losses over sequences ---------------------------------------------------------------------------------

// Gradients of a node that can be differentiated once: where a graph of them is built, a pass through it raises.  The node that does leads
// on to all that the gradients depend on, the node's own inputs and the upstream gradients: a pass that is only to reach some of
// these runs nothing else, and would leave these terms out.
variable_list once(variable_list grads, const Node& node, const variable_list& upstream, const char* who) {
    if (!at::GradMode::is_enabled()) return grads;
    torch::autograd::edge_list edges = node.next_edges();
    for (const Tensor& up : upstream)
        if (up.defined()) edges.push_back(torch::autograd::impl::gradient_edge(up));
    const std::shared_ptr<Node> error(new torch::autograd::Error(std::string(who) + " can be differentiated once only", std::move(edges)),
                                      torch::autograd::deleteNode);
    for (Tensor& g : grads) {
        if (!g.defined()) continue;
        g = g.detach();
        torch::autograd::set_history(g, error);
    }
    return grads;
}

struct EmbedNode : public Node {
    SavedVariable tokens, table;
    Tensor shape;                                            // not encoded: in table's place, whose values the gradient does not need
    float scale;
    bool encode;
    std::string name() const override { return "SnnEmbedBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        tokens.reset_data(); table.reset_data(); shape.reset();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined() || !task_should_compute_output(0)) return variable_list(1);
        const Tensor tok = tokens.unpack(), tab = encode ? table.unpack() : shape;
        variable_list out(1);
        {
            at::AutoGradMode no_grad(false);
            out[0] = embed_tokens_grad(grads[0], embed_args(tok, tab, scale, encode));
        }
        return once(std::move(out), *this, grads, "embed_tokens");
    }
};

Tensor embed_layer(const Tensor& tokens, const Tensor& table, float scale, bool encode) {
    const EmbedArgs a = embed_args(tokens, table, scale, encode);
    Tensor z;
    {
        at::AutoGradMode no_grad(false);
        z = embed_tokens(a);
    }
    if (!wants_grad(a.table)) return z;
    auto node = make_node<EmbedNode>({a.table});
    node->scale = scale; node->encode = encode;
    node->tokens = SavedVariable(a.tokens, false);
    if (encode) node->table = SavedVariable(a.table, false);
    else node->shape = a.table.detach();
    return with_history(z, node);
}

struct GatedNode : public Node {
    SavedVariable x, gate, state, lengths, y;
    bool has_state, has_lengths;
    std::string name() const override { return "SnnGatedScanBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data(); gate.reset_data(); state.reset_data(); lengths.reset_data(); y.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(3);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        const Tensor X = x.unpack(), G = gate.unpack(), S = has_state ? state.unpack() : Tensor(),
                     L = has_lengths ? lengths.unpack() : Tensor(), Y = y.unpack();
        {
            at::AutoGradMode no_grad(false);
            ScanGrads g = gated_scan_grad(grads[0], grads[1], GatedArgs{X, G, S, L}, Y, task_should_compute_output(0),
                                          task_should_compute_output(1), has_state && task_should_compute_output(2));
            out[0] = g.dx; out[1] = g.dgate; out[2] = g.dstate;
        }
        return once(std::move(out), *this, grads, "gated_scan");
    }
};

Scanned gated_layer(const Tensor& x, const Tensor& gate, const Tensor& state, const Tensor& lengths) {
    const GatedArgs a = gated_args(x, gate, state, lengths);
    Scanned r;
    {
        at::AutoGradMode no_grad(false);
        r = gated_scan(a);
    }
    if (!wants_grad(a.x, a.gate) && !(a.state.defined() && wants_grad(a.state))) return r;
    std::shared_ptr<GatedNode> node(new GatedNode(), torch::autograd::deleteNode);
    torch::autograd::edge_list edges{torch::autograd::impl::gradient_edge(a.x), torch::autograd::impl::gradient_edge(a.gate),
                                     a.state.defined() ? torch::autograd::impl::gradient_edge(a.state) : torch::autograd::Edge()};
    node->set_next_edges(std::move(edges));
    node->has_state = a.state.defined(); node->has_lengths = a.lengths.defined();
    node->x = SavedVariable(a.x, false); node->gate = SavedVariable(a.gate, false);
    if (node->has_state) node->state = SavedVariable(a.state, false);
    if (node->has_lengths) node->lengths = SavedVariable(a.lengths, false);
    node->y = SavedVariable(r.y.detach(), false);            // a detached alias, or the output would keep itself alive
    torch::autograd::set_history(r.y, node);
    torch::autograd::set_history(r.final, node);
    return r;
}

// The objective of a loss over choices: its gradient by the times is made in the backward pass, from the row statistics and the
// derivative by each row's log-probability that the forward pass has left.
struct ChoiceNode : public Node {
    SavedVariable times, tokens, stats, coef;
    std::string name() const override { return "ChoiceLossBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        times.reset_data(); tokens.reset_data(); stats.reset_data(); coef.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined() || !task_should_compute_output(0)) return variable_list(1);
        const Tensor t = times.unpack(), k = tokens.unpack(), s = stats.unpack(), c = coef.unpack();
        variable_list out(1);
        {
            at::AutoGradMode no_grad(false);
            out[0] = objective_grad(choice_args(t, k, Tensor(), "tokens"), s, c, grads[0]);
        }
        return once(std::move(out), *this, grads, "a loss over choices");
    }
};

Tensor choice_history(const ChoiceArgs& a, const Objective& r) {
    auto node = make_node<ChoiceNode>({a.times});
    node->times = SavedVariable(a.times, false); node->tokens = SavedVariable(a.tokens, false);
    node->stats = SavedVariable(r.stats, false); node->coef = SavedVariable(r.coef, false);
    return with_history(r.total, node);
}

Tensor policy_layer(const ChoiceArgs& a, const PolicyIn& p) {
    no_gradient({{&p.old_logp, "old_logp"}, {&p.advantage, "advantage"}, {&p.ref_logp, "ref_logp"}, {&a.weight, "weight"}}, "policy loss");
    const bool grad = wants_grad(a.times);
    Objective r;
    {
        at::AutoGradMode no_grad(false);
        r = policy_objective(a, p, grad);
    }
    return grad ? choice_history(a, r) : r.total;
}

Tensor preference_layer(const ChoiceArgs& a, const Tensor& ref, float beta, float smoothing) {
    no_gradient({{&ref, "ref_logp"}, {&a.weight, "weight"}}, "preference loss");
    const bool grad = wants_grad(a.times);
    Objective r;
    {
        at::AutoGradMode no_grad(false);
        r = preference_objective(a, ref, beta, smoothing, grad);
    }
    return grad ? choice_history(a, r) : r.total;
}

// Ruled times; the gradient reads the times themselves only where a repetition changed them.
struct RuleNode : public Node {
    SavedVariable times, history, lengths, repetition, allowed;
    bool has_history, has_lengths, has_repetition, has_allowed;
    float repetition_all;
    std::string name() const override { return "TimeRulesBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        times.reset_data(); history.reset_data(); lengths.reset_data(); repetition.reset_data(); allowed.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined() || !task_should_compute_output(0)) return variable_list(1);
        RuleIn in{};
        in.repetition.all = 1.0f;
        if (has_history) {
            in.history = history.unpack();
            in.repetition.all = repetition_all;
            if (has_lengths) in.lengths = lengths.unpack();
            if (has_repetition) in.repetition.each = repetition.unpack();
        }
        if (has_allowed) in.allowed = allowed.unpack();
        variable_list out(1);
        {
            at::AutoGradMode no_grad(false);
            // without penalties the gradient reads no times: a tensor of their shape and type stands for them, and none of them is held
            const Tensor g = grads[0].contiguous();
            out[0] = rule_times_grad(g, rule_set(has_history ? times.unpack() : g, in));
        }
        return once(std::move(out), *this, grads, "rule_times");
    }
};

Tensor rule_layer(const RuleSet& r, const RuleIn& in) {
    no_gradient({{&in.repetition.each, "repetition"}, {&in.presence.each, "presence"}, {&in.frequency.each, "frequency"}, {&in.delay, "delay"}},
                "rule_times");
    Tensor out;
    {
        at::AutoGradMode no_grad(false);
        out = rule_times(r);
    }
    if (!wants_grad(r.times)) return out;
    auto node = make_node<RuleNode>({r.times});
    node->has_history = r.history.defined() && (r.repetition.defined() || in.repetition.all != 1.0f);
    node->has_lengths = node->has_history && r.lengths.defined();
    node->has_repetition = node->has_history && r.repetition.defined();
    node->has_allowed = r.allowed.defined();
    node->repetition_all = in.repetition.all;
    if (node->has_history) {
        node->times = SavedVariable(r.times, false);
        node->history = SavedVariable(r.history, false);
    }
    if (node->has_lengths) node->lengths = SavedVariable(r.lengths, false);
    if (node->has_repetition) node->repetition = SavedVariable(r.repetition, false);
    if (node->has_allowed) node->allowed = SavedVariable(r.allowed, false);
    return with_history(out, node);
}

// ---- the example training recipe -------------------------------------------------------------------------------------

Tensor encode_time(const Tensor& image) {
    const Tensor x = image.contiguous();
    const c10::DeviceGuard guard(x.device());
    const Tensor z = empty(x, x.sizes());
    check(lib.snntc_encode_time(f32(x), f32(z), x.numel(), stream_of(x)));
    return z;
}

// Host arrays of the weight tensors the constraint cost runs over, and its device scratch.
struct CostArgs {
    std::vector<const float*> w;
    std::vector<int64_t> rows, cols;
    Tensor ws;
    explicit CostArgs(const std::vector<Tensor>& weights) {
        for (const Tensor& t : weights) {
            w.push_back(f32(t));
            rows.push_back(t.size(0));
            cols.push_back(t.size(1));
        }
    }
    int64_t count() const { return (int64_t)w.size(); }
    void sums(const Tensor& like, void* stream) {
        size_t need = 0;
        check(lib.snntc_weight_cost_workspace_bytes(rows.data(), cols.data(), count(), &need));
        ws = scratch(like, need);
        check(lib.snntc_weight_cost_sums(w.data(), rows.data(), cols.data(), count(), ws.data_ptr(), ws.numel(), stream));
    }
    void grad(float* const* g, float k, float k2, const float* upstream, bool accumulate, void* stream) {
        check(lib.snntc_weight_cost_grad(w.data(), g, rows.data(), cols.data(), count(), k, k2, upstream, accumulate, ws.data_ptr(),
                                         ws.numel(), stream));
    }
};

struct CostNode : public Node {
    std::vector<SavedVariable> weights;
    Tensor ws;
    float k, k2;
    std::string name() const override { return "ConstraintCostBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable& w : weights) w.reset_data();
        ws.reset();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(weights.size());
        if (!grads[0].defined()) return out;
        std::vector<Tensor> w;
        for (SavedVariable& s : weights) w.push_back(s.unpack());
        if (at::GradMode::is_enabled() || !plain({grads[0]})) {        // a graph of the gradient is wanted: differentiable ops
            for (size_t i = 0; i < w.size(); ++i) {
                if (!task_should_compute_output(i)) continue;
                const Tensor low = (1.0 - w[i].detach().sum(0)).ge(0).to(at::kFloat);
                out[i] = grads[0] * (low * (-k / (float)w[i].size(1)) + w[i] * (2.0f * k2 / (float)w[i].numel()));
            }
            return out;
        }
        const Tensor up = grads[0].contiguous();
        const c10::DeviceGuard guard(up.device());
        CostArgs args(w);
        args.ws = ws;
        std::vector<float*> g;
        for (size_t i = 0; i < w.size(); ++i) {
            if (task_should_compute_output(i)) out[i] = empty(w[i], w[i].sizes());
            g.push_back(f32(out[i]));
        }
        args.grad(g.data(), k, k2, f32(up), false, stream_of(up));
        return out;
    }
};

// The weight-constraint cost of contiguous float32 weight matrices on one device, differentiable.
Tensor constraint_cost(const std::vector<Tensor>& weights, float k, float k2) {
    const c10::DeviceGuard guard(weights[0].device());
    void* stream = stream_of(weights[0]);
    CostArgs args(weights);
    Tensor total;
    bool grad = false;
    {
        at::AutoGradMode no_grad(false);
        args.sums(weights[0], stream);
        total = empty(weights[0], {});
        check(lib.snntc_recipe_total(args.rows.data(), args.cols.data(), args.count(), k, k2, nullptr, nullptr, 0, f32(total), nullptr,
                                     args.ws.data_ptr(), args.ws.numel(), stream));
    }
    for (const Tensor& w : weights) grad = grad || wants_grad(w);
    if (!grad) return total;
    std::shared_ptr<CostNode> node(new CostNode(), torch::autograd::deleteNode);
    torch::autograd::edge_list edges;
    for (const Tensor& w : weights) {
        edges.push_back(torch::autograd::impl::gradient_edge(w));
        node->weights.emplace_back(w, false);
    }
    node->set_next_edges(std::move(edges));
    node->ws = args.ws; node->k = k; node->k2 = k2;
    return with_history(total, node);
}

// Loss, cost, count of correct samples and -- with `train` -- every gradient of one step: the data gradients
// through the engine from the loss kernel's dtimes, then the cost's added into each weight's .grad.
LossOut recipe_step(const Tensor& pred_in, const Tensor& labels_in, const std::vector<Tensor>& weights, float k, float k2, bool train) {
    const Tensor pred = dev_f32(pred_in, "predictions", 2);
    const int64_t B = pred.size(0), J = pred.size(1);
    const c10::DeviceGuard guard(pred.device());
    void* stream = stream_of(pred);
    Tensor sample_loss, dtimes, correct, total, n_correct;
    CostArgs args(weights);
    {
        at::AutoGradMode no_grad(false);
        const Tensor labels = labels_in.contiguous();
        sample_loss = empty(pred, {B});
        correct = at::empty({B}, pred.options().dtype(at::kInt));
        if (train) dtimes = empty(pred, pred.sizes());
        check(lib.snntc_label_loss(f32(pred), static_cast<int64_t*>(labels.data_ptr()), f32(sample_loss), f32(dtimes),
                                   static_cast<int32_t*>(correct.data_ptr()), B, J, stream));
    }
    if (train) torch::autograd::backward({pred}, {dtimes});
    at::AutoGradMode no_grad(false);
    args.sums(pred, stream);
    total = empty(pred, {});
    n_correct = at::empty({}, pred.options().dtype(at::kLong));
    check(lib.snntc_recipe_total(args.rows.data(), args.cols.data(), args.count(), k, k2, f32(sample_loss),
                                 static_cast<int32_t*>(correct.data_ptr()), B, f32(total), static_cast<int64_t*>(n_correct.data_ptr()),
                                 args.ws.data_ptr(), args.ws.numel(), stream));
    if (train) {
        std::vector<float*> g;
        std::vector<Tensor> keep;
        for (const Tensor& w : weights) {
            Tensor& wg = w.mutable_grad();
            if (!w.requires_grad()) { g.push_back(nullptr); continue; }
            if (!wg.defined()) {
                wg = at::zeros_like(w);
            } else if (!(wg.is_cuda() && wg.scalar_type() == at::kFloat && wg.is_contiguous() && wg.sizes() == w.sizes())) {
                wg = wg.to(w.options()).contiguous();
            }
            written_behind_autograd(wg);
            g.push_back(f32(wg));
        }
        args.grad(g.data(), k, k2, nullptr, true, stream);
    }
    return LossOut{total, n_correct};
}

// ---- Python arguments ----------------------------------------------------------------------------------------------

const Tensor& tensor_arg(PyObject* o, const char* name) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a torch.Tensor");
    return THPVariable_Unpack(o);
}

Tensor optional_tensor(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor_arg(o, name); }

int64_t int_arg(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}

float float_arg(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return (float)v;
}

bool bool_arg(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}

// A Params vector: read straight out of a float32 vector's buffer (what the layers keep), anything else is
// converted first.
template <size_t N>
std::array<float, N> params_arg(PyObject* o) {
    std::array<float, N> p;
    auto read = [&](PyObject* v) {
        Py_buffer b;
        if (PyObject_GetBuffer(v, &b, PyBUF_C_CONTIGUOUS | PyBUF_FORMAT) != 0) { PyErr_Clear(); return false; }
        const bool plain = b.format && b.format[0] == 'f' && b.format[1] == 0 && b.len == (Py_ssize_t)(N * sizeof(float));
        if (plain) memcpy(p.data(), b.buf, N * sizeof(float));
        PyBuffer_Release(&b);
        return plain;
    };
    if (read(o)) return p;
    PyObject* conv = PyObject_CallFunction(g_params, "On", o, (Py_ssize_t)N);     // raises ValueError on a wrong length
    if (!conv) throw python_error();
    const bool ok = read(conv);
    Py_DECREF(conv);
    TORCH_CHECK_VALUE(ok, "Params must hold ", N, " float32 values");
    return p;
}

struct NoGil {
    PyThreadState* state;
    NoGil() : state(PyEval_SaveThread()) {}
    ~NoGil() { PyEval_RestoreThread(state); }
};

void arity(Py_ssize_t got, Py_ssize_t want, const char* who) {
    TORCH_CHECK_TYPE(got == want, who, " takes ", want, " arguments, got ", got);
}

PyObject* wrap(const Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}

PyObject* wrap3(const Tensor& a, const Tensor& b, const Tensor& c) {
    PyObject *pa = wrap(a), *pb = wrap(b), *pc = wrap(c);
    PyObject* t = pa && pb && pc ? PyTuple_Pack(3, pa, pb, pc) : nullptr;
    Py_XDECREF(pa); Py_XDECREF(pb); Py_XDECREF(pc);
    return t;
}

PyObject* wrap2(const Tensor& a, const Tensor& b) {
    PyObject *pa = wrap(a), *pb = wrap(b);
    PyObject* t = pa && pb ? PyTuple_Pack(2, pa, pb) : nullptr;
    Py_XDECREF(pa); Py_XDECREF(pb);
    return t;
}

Feed feed_arg(PyObject* dst, PyObject* top, PyObject* left) {
    return Feed{optional_tensor(dst, "next_xpad"), int_arg(top), int_arg(left)};
}

PyObject* general(const char* name, PyObject* const* a, Py_ssize_t n) {
    PyObject* f = PyDict_GetItemString(g_general, name);
    TORCH_CHECK(f, "no general path for ", name);
    return PyObject_Vectorcall(f, a, n, nullptr);
}

#define SNNTC_METHOD(name) PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t n)

// fc_forward(X, W, params) -> Y[2B,J]
SNNTC_METHOD(py_fc_forward) {
    HANDLE_TH_ERRORS
    arity(n, 3, "fc_forward");
    const Tensor x = tensor_arg(a[0], "X"), w = tensor_arg(a[1], "W");
    const auto p = params_arg<6>(a[2]);
    Tensor out;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        out = fc_forward(dev_f32(x, "X", 2), dev_f32(w, "W", 2), p);
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// fc_layer(X, W, params, times) -> Y[:B] or Y, differentiable
SNNTC_METHOD(py_fc_layer) {
    HANDLE_TH_ERRORS
    arity(n, 4, "fc_layer");
    const Tensor x = tensor_arg(a[0], "X"), w = tensor_arg(a[1], "W");
    if (!plain({x, w})) return general("fc_layer", a, n);
    const auto p = params_arg<6>(a[2]);
    const bool times = bool_arg(a[3]);
    Tensor out;
    {
        NoGil nogil;
        out = fc_layer(x, w, p, times);
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// fc_backward(grad, X, W, params, Y, want_dx, want_dw, want_dp, first_half_grad) -> (dX, dW, dP)
SNNTC_METHOD(py_fc_backward) {
    HANDLE_TH_ERRORS
    arity(n, 9, "fc_backward");
    const Tensor g = tensor_arg(a[0], "grad"), x = tensor_arg(a[1], "X"), w = tensor_arg(a[2], "W"), y = tensor_arg(a[4], "Y");
    const auto p = params_arg<6>(a[3]);
    const bool want_dx = bool_arg(a[5]), want_dw = bool_arg(a[6]), want_dp = bool_arg(a[7]), half = bool_arg(a[8]);
    Grads r;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        r = fc_backward(dev_f32(g, "grad", 2), dev_f32(x, "X", 2), dev_f32(w, "W", 2), p, dev_f32(y, "Y", 2), want_dx, want_dw,
                        want_dp, half);
    }
    return wrap3(r.dx, r.dw, r.dp);
    END_HANDLE_TH_ERRORS
}

// cv_forward(X, W, params, next_xpad, top, left) -> Y[2B,Nh,Nw,Kc]
SNNTC_METHOD(py_cv_forward) {
    HANDLE_TH_ERRORS
    arity(n, 6, "cv_forward");
    const Tensor x = tensor_arg(a[0], "X"), w = tensor_arg(a[1], "W");
    const auto p = params_arg<12>(a[2]);
    const Feed feed = feed_arg(a[3], a[4], a[5]);
    Tensor out;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        out = cv_forward(dev_f32(x, "X", 4), dev_f32(w, "W", 2), p, feed);
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// cv_layer(X, W, params, times) -> Y[:B] or Y, differentiable
SNNTC_METHOD(py_cv_layer) {
    HANDLE_TH_ERRORS
    arity(n, 4, "cv_layer");
    const Tensor x = tensor_arg(a[0], "X"), w = tensor_arg(a[1], "W");
    if (!plain({x, w})) return general("cv_layer", a, n);
    const auto p = params_arg<12>(a[2]);
    const bool times = bool_arg(a[3]);
    Tensor out;
    {
        NoGil nogil;
        const Tensor xc = dev_f32(x, "X", 4);
        out = cv_layer(xc, xc, dev_f32(w, "W", 2), p, times, std::nullopt, Feed{});
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// cv_same(x, W, params, top, bottom, left, right, xpad, next_xpad, next_top, next_left) -> spike times, differentiable
SNNTC_METHOD(py_cv_same) {
    HANDLE_TH_ERRORS
    arity(n, 11, "cv_same");
    const Tensor x = tensor_arg(a[0], "X"), w = tensor_arg(a[1], "W");
    const auto p = params_arg<12>(a[2]);
    const Pads pad{int_arg(a[3]), int_arg(a[4]), int_arg(a[5]), int_arg(a[6])};
    const Tensor xpad = optional_tensor(a[7], "xpad");
    const Feed feed = feed_arg(a[8], a[9], a[10]);
    if (!plain({x, w, xpad, feed.dst})) return general("cv_same", a, n);
    Tensor out;
    {
        NoGil nogil;
        out = cv_same(x, w, p, pad, xpad, feed);
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// cv_backward(grad, X, W, params, Y, want_dx, want_dw, want_dp, first_half_grad, crop) -> (dX, dW, dP)
SNNTC_METHOD(py_cv_backward) {
    HANDLE_TH_ERRORS
    arity(n, 10, "cv_backward");
    const Tensor g = tensor_arg(a[0], "grad"), x = tensor_arg(a[1], "X"), w = tensor_arg(a[2], "W"), y = tensor_arg(a[4], "Y");
    const auto p = params_arg<12>(a[3]);
    const bool want_dx = bool_arg(a[5]), want_dw = bool_arg(a[6]), want_dp = bool_arg(a[7]), half = bool_arg(a[8]);
    Window win;
    const bool cropped = a[9] != Py_None;
    if (cropped) {
        long long h, w2, t, l;
        if (!PyTuple_Check(a[9]) || !PyArg_ParseTuple(a[9], "LLLL", &h, &w2, &t, &l)) throw python_error();
        win = Window{h, w2, t, l};
    }
    Grads r;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        r = cv_backward(dev_f32(g, "grad", 4), dev_f32(x, "X", 4), dev_f32(w, "W", 2), p, dev_f32(y, "Y", 4), want_dx, want_dw,
                        want_dp, half, cropped ? &win : nullptr);
    }
    return wrap3(r.dx, r.dw, r.dp);
    END_HANDLE_TH_ERRORS
}

PoolShape pool_arg(PyObject* const* a) {
    return PoolShape{int_arg(a[0]), int_arg(a[1]), int_arg(a[2]), int_arg(a[3]), int_arg(a[4]), int_arg(a[5]), int_arg(a[6]),
                     int_arg(a[7]), float_arg(a[8])};
}

// min_pool(x, kh, kw, sh, sw, top, left, nh, nw, pad_value, want_arg, next_xpad, next_top, next_left) -> (y, arg)
SNNTC_METHOD(py_min_pool) {
    HANDLE_TH_ERRORS
    arity(n, 14, "min_pool");
    const Tensor x = tensor_arg(a[0], "x");
    const PoolShape s = pool_arg(a + 1);
    const bool want_arg = bool_arg(a[10]);
    const Feed feed = feed_arg(a[11], a[12], a[13]);
    Pooled r;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        r = min_pool(dev_f32(x, "x", 4), s, want_arg, feed);
    }
    return wrap2(r.y, r.arg);
    END_HANDLE_TH_ERRORS
}

// min_pool_layer(x, kh, kw, sh, sw, top, left, nh, nw, pad_value, next_xpad, next_top, next_left) -> y, differentiable
SNNTC_METHOD(py_min_pool_layer) {
    HANDLE_TH_ERRORS
    arity(n, 13, "min_pool_layer");
    const Tensor x = tensor_arg(a[0], "x");
    const PoolShape s = pool_arg(a + 1);
    const Feed feed = feed_arg(a[10], a[11], a[12]);
    if (!plain({x, feed.dst})) return general("min_pool_layer", a, n);
    Tensor out;
    {
        NoGil nogil;
        out = pool_layer(x, s, feed);
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// pad_layer(x, top, bottom, left, right, value) -> padded, differentiable
SNNTC_METHOD(py_pad_layer) {
    HANDLE_TH_ERRORS
    arity(n, 6, "pad_layer");
    const Tensor x = tensor_arg(a[0], "x");
    if (!plain({x})) return general("pad_layer", a, n);
    const Pads pad{int_arg(a[1]), int_arg(a[2]), int_arg(a[3]), int_arg(a[4])};
    const float value = float_arg(a[5]);
    Tensor out;
    {
        NoGil nogil;
        out = pad_layer(x, pad, value);
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// time_loss(times, label, want_loss, want_grad) -> (loss[B], dtimes)
SNNTC_METHOD(py_time_loss) {
    HANDLE_TH_ERRORS
    arity(n, 4, "time_loss");
    const Tensor t = tensor_arg(a[0], "times"), l = tensor_arg(a[1], "label");
    const bool want_loss = bool_arg(a[2]), want_grad = bool_arg(a[3]);
    LossOut r;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        r = time_loss(dev_f32(t, "times", 2), dev_f32(l, "label", 2), want_loss, want_grad);
    }
    return wrap2(r.loss, r.grad);
    END_HANDLE_TH_ERRORS
}

// loss_layer(times, label) -> mean loss, differentiable in times
SNNTC_METHOD(py_loss_layer) {
    HANDLE_TH_ERRORS
    arity(n, 2, "loss_layer");
    const Tensor t = tensor_arg(a[0], "times"), l = tensor_arg(a[1], "label");
    if (!plain({t, l})) return general("loss_layer", a, n);
    Tensor out;
    {
        NoGil nogil;
        out = loss_layer(t, l);
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// sgd_update(list of weights, list of gradients, lr)
SNNTC_METHOD(py_sgd_update) {
    HANDLE_TH_ERRORS
    arity(n, 3, "sgd_update");
    TORCH_CHECK_TYPE(PyList_Check(a[0]) && PyList_Check(a[1]), "sgd_update takes lists");
    std::vector<Tensor> ws, gs;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a[0]); ++i) {
        PyObject* w = PyList_GET_ITEM(a[0], i);
        if (!THPVariable_Check(w))
            raise_class(g_library_error, message_args, 0, "sgd_update: weight " + std::to_string(i) +
                        " must be a contiguous float32 tensor on a ROCm GPU");
        ws.push_back(THPVariable_Unpack(w));
        gs.push_back(tensor_arg(PyList_GET_ITEM(a[1], i), "gradient"));
    }
    const float lr = float_arg(a[2]);
    {
        NoGil nogil;
        sgd_update(ws, gs, lr);
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

std::vector<Tensor> tensor_list(PyObject* o, const char* name) {
    TORCH_CHECK_TYPE(PyList_Check(o), name, " must be a list");
    std::vector<Tensor> v;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(o); ++i) v.push_back(tensor_arg(PyList_GET_ITEM(o, i), name));
    return v;
}

// plain(tensors...): whether the native entry points that have no general path may take them
SNNTC_METHOD(py_plain) {
    HANDLE_TH_ERRORS
    bool ok = plain({});
    for (Py_ssize_t i = 0; ok && i < n; ++i) ok = plain({tensor_arg(a[i], "argument")});
    return PyBool_FromLong(ok);
    END_HANDLE_TH_ERRORS
}

// encode_time(image) -> exp(1 - image) for a float32 device tensor
SNNTC_METHOD(py_encode_time) {
    HANDLE_TH_ERRORS
    arity(n, 1, "encode_time");
    const Tensor x = tensor_arg(a[0], "image");
    Tensor z;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        z = encode_time(x);
    }
    return wrap(z);
    END_HANDLE_TH_ERRORS
}

// constraint_cost(weights, k, k2) -> scalar, differentiable
SNNTC_METHOD(py_constraint_cost) {
    HANDLE_TH_ERRORS
    arity(n, 3, "constraint_cost");
    const std::vector<Tensor> w = tensor_list(a[0], "weights");
    const float k = float_arg(a[1]), k2 = float_arg(a[2]);
    Tensor out;
    {
        NoGil nogil;
        out = constraint_cost(w, k, k2);
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// recipe_step(predictions, labels, weights, k, k2, train) -> (loss, number of correct samples)
SNNTC_METHOD(py_recipe_step) {
    HANDLE_TH_ERRORS
    arity(n, 6, "recipe_step");
    const Tensor p = tensor_arg(a[0], "predictions"), l = tensor_arg(a[1], "labels");
    const std::vector<Tensor> w = tensor_list(a[2], "weights");
    const float k = float_arg(a[3]), k2 = float_arg(a[4]);
    const bool train = bool_arg(a[5]);
    LossOut r;
    {
        NoGil nogil;
        r = recipe_step(p, l, w, k, k2, train);
    }
    return wrap2(r.loss, r.grad);
    END_HANDLE_TH_ERRORS
}

// embed_tokens(tokens, table, scale, encode) -> z[..., D]
SNNTC_METHOD(py_embed_tokens) {
    HANDLE_TH_ERRORS
    arity(n, 4, "embed_tokens");
    const Tensor tok = tensor_arg(a[0], "tokens"), tab = tensor_arg(a[1], "table");
    const float scale = float_arg(a[2]);
    const bool encode = bool_arg(a[3]);
    Tensor z;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        z = embed_tokens(embed_args(tok, tab, scale, encode));
    }
    return wrap(z);
    END_HANDLE_TH_ERRORS
}

// embed_tokens_grad(grad, tokens, table, scale, encode) -> gradient of the table
SNNTC_METHOD(py_embed_tokens_grad) {
    HANDLE_TH_ERRORS
    arity(n, 5, "embed_tokens_grad");
    const Tensor g = tensor_arg(a[0], "grad"), tok = tensor_arg(a[1], "tokens"), tab = tensor_arg(a[2], "table");
    const float scale = float_arg(a[3]);
    const bool encode = bool_arg(a[4]);
    Tensor d;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        d = embed_tokens_grad(g, embed_args(tok, tab, scale, encode));
    }
    return wrap(d);
    END_HANDLE_TH_ERRORS
}

// embed_layer(tokens, table, scale, encode) -> z, differentiable in the table
SNNTC_METHOD(py_embed_layer) {
    HANDLE_TH_ERRORS
    arity(n, 4, "embed_layer");
    const Tensor tok = tensor_arg(a[0], "tokens"), tab = tensor_arg(a[1], "table");
    if (!plain({tok, tab})) return general("embed_layer", a, n);
    const float scale = float_arg(a[2]);
    const bool encode = bool_arg(a[3]);
    Tensor z;
    {
        NoGil nogil;
        z = embed_layer(tok, tab, scale, encode);
    }
    return wrap(z);
    END_HANDLE_TH_ERRORS
}

// gated_scan(x, gate, state, lengths) -> (y, final)
SNNTC_METHOD(py_gated_scan) {
    HANDLE_TH_ERRORS
    arity(n, 4, "gated_scan");
    const Tensor x = tensor_arg(a[0], "x"), g = tensor_arg(a[1], "gate"), s = optional_tensor(a[2], "state"),
                 l = optional_tensor(a[3], "lengths");
    Scanned r;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        r = gated_scan(gated_args(x, g, s, l));
    }
    return wrap2(r.y, r.final);
    END_HANDLE_TH_ERRORS
}

// gated_scan_grad(grad_y, grad_final, x, gate, y, state, lengths, want_dx, want_dgate, want_dstate) -> (dx, dgate, dstate)
SNNTC_METHOD(py_gated_scan_grad) {
    HANDLE_TH_ERRORS
    arity(n, 10, "gated_scan_grad");
    const Tensor dy = optional_tensor(a[0], "grad_y"), df = optional_tensor(a[1], "grad_final"), x = tensor_arg(a[2], "x"),
                 g = tensor_arg(a[3], "gate"), y = tensor_arg(a[4], "y"), s = optional_tensor(a[5], "state"),
                 l = optional_tensor(a[6], "lengths");
    const bool want_dx = bool_arg(a[7]), want_dgate = bool_arg(a[8]), want_dstate = bool_arg(a[9]);
    ScanGrads r;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        r = gated_scan_grad(dy, df, gated_args(x, g, s, l), y, want_dx, want_dgate, want_dstate);
    }
    return wrap3(r.dx, r.dgate, r.dstate);
    END_HANDLE_TH_ERRORS
}

// gated_layer(x, gate, state, lengths) -> (y, final), differentiable in x, gate and state
SNNTC_METHOD(py_gated_layer) {
    HANDLE_TH_ERRORS
    arity(n, 4, "gated_layer");
    const Tensor x = tensor_arg(a[0], "x"), g = tensor_arg(a[1], "gate"), s = optional_tensor(a[2], "state"),
                 l = optional_tensor(a[3], "lengths");
    if (!plain({x, g, s, l})) return general("gated_layer", a, n);
    Scanned r;
    {
        NoGil nogil;
        r = gated_layer(x, g, s, l);
    }
    return wrap2(r.y, r.final);
    END_HANDLE_TH_ERRORS
}

// gated_step(x, gate, state, out) -> the new state
SNNTC_METHOD(py_gated_step) {
    HANDLE_TH_ERRORS
    arity(n, 4, "gated_step");
    const Tensor x = tensor_arg(a[0], "x"), g = tensor_arg(a[1], "gate"), s = optional_tensor(a[2], "state"),
                 o = optional_tensor(a[3], "out");
    Tensor out;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        out = gated_step(x, g, s, o);
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// time_logp(times, tokens, weight) -> logp
SNNTC_METHOD(py_time_logp) {
    HANDLE_TH_ERRORS
    arity(n, 3, "time_logp");
    const Tensor t = tensor_arg(a[0], "times"), k = tensor_arg(a[1], "tokens"), w = optional_tensor(a[2], "weight");
    Tensor logp;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        logp = time_logp(choice_args(t, k, w, "tokens"));
    }
    return wrap(logp);
    END_HANDLE_TH_ERRORS
}

PolicyIn policy_in(PyObject* const* a) {
    return PolicyIn{tensor_arg(a[0], "old_logp"), tensor_arg(a[1], "advantage"), optional_tensor(a[2], "ref_logp"), float_arg(a[4]),
                    float_arg(a[5]), float_arg(a[6])};
}

// policy_loss(times, actions, old_logp, advantage, ref_logp, weight, clip_low, clip_high, kl_coef, want_grad) -> (row_loss, logp, dtimes)
SNNTC_METHOD(py_policy_loss) {
    HANDLE_TH_ERRORS
    arity(n, 10, "policy_loss");
    const Tensor t = tensor_arg(a[0], "times"), k = tensor_arg(a[1], "actions"), w = optional_tensor(a[5], "weight");
    const PolicyIn p = policy_in(a + 2);
    const bool want_grad = bool_arg(a[9]);
    ChoiceOut r;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        r = policy_loss(choice_args(t, k, w, "actions"), p, want_grad, false);
    }
    return wrap3(r.loss, r.logp, r.dtimes);
    END_HANDLE_TH_ERRORS
}

// policy_layer(times, actions, old_logp, advantage, ref_logp, weight, clip_low, clip_high, kl_coef) -> objective, differentiable
SNNTC_METHOD(py_policy_layer) {
    HANDLE_TH_ERRORS
    arity(n, 9, "policy_layer");
    const Tensor t = tensor_arg(a[0], "times"), k = tensor_arg(a[1], "actions"), w = optional_tensor(a[5], "weight");
    const PolicyIn p = policy_in(a + 2);
    if (!plain({t, k, w, p.old_logp, p.advantage, p.ref_logp})) return general("policy_layer", a, n);
    Tensor total;
    {
        NoGil nogil;
        total = policy_layer(choice_args(t, k, w, "actions"), p);
    }
    return wrap(total);
    END_HANDLE_TH_ERRORS
}

// preference_loss(times, tokens, ref_logp, weight, beta, smoothing, want_grad) -> (pair_loss, seq_logp, dtimes)
SNNTC_METHOD(py_preference_loss) {
    HANDLE_TH_ERRORS
    arity(n, 7, "preference_loss");
    const Tensor t = tensor_arg(a[0], "times"), k = tensor_arg(a[1], "tokens"), ref = tensor_arg(a[2], "ref_logp"),
                 w = optional_tensor(a[3], "weight");
    const float beta = float_arg(a[4]), smoothing = float_arg(a[5]);
    const bool want_grad = bool_arg(a[6]);
    ChoiceOut r;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        r = preference_loss(choice_args(t, k, w, "tokens"), ref, beta, smoothing, want_grad, false);
    }
    return wrap3(r.loss, r.logp, r.dtimes);
    END_HANDLE_TH_ERRORS
}

// preference_layer(times, tokens, ref_logp, weight, beta, smoothing) -> objective, differentiable
SNNTC_METHOD(py_preference_layer) {
    HANDLE_TH_ERRORS
    arity(n, 6, "preference_layer");
    const Tensor t = tensor_arg(a[0], "times"), k = tensor_arg(a[1], "tokens"), ref = tensor_arg(a[2], "ref_logp"),
                 w = optional_tensor(a[3], "weight");
    const float beta = float_arg(a[4]), smoothing = float_arg(a[5]);
    if (!plain({t, k, ref, w})) return general("preference_layer", a, n);
    Tensor total;
    {
        NoGil nogil;
        total = preference_layer(choice_args(t, k, w, "tokens"), ref, beta, smoothing);
    }
    return wrap(total);
    END_HANDLE_TH_ERRORS
}

// policy_objective(times, actions, old_logp, advantage, ref_logp, weight, clip_low, clip_high, kl_coef, save) -> (objective, stats, coef)
SNNTC_METHOD(py_policy_objective) {
    HANDLE_TH_ERRORS
    arity(n, 10, "policy_objective");
    const Tensor t = tensor_arg(a[0], "times"), k = tensor_arg(a[1], "actions"), w = optional_tensor(a[5], "weight");
    const PolicyIn p = policy_in(a + 2);
    const bool save = bool_arg(a[9]);
    Objective r;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        r = policy_objective(choice_args(t, k, w, "actions"), p, save);
    }
    return wrap3(r.total, r.stats, r.coef);
    END_HANDLE_TH_ERRORS
}

// preference_objective(times, tokens, ref_logp, weight, beta, smoothing, save) -> (objective, stats, coef)
SNNTC_METHOD(py_preference_objective) {
    HANDLE_TH_ERRORS
    arity(n, 7, "preference_objective");
    const Tensor t = tensor_arg(a[0], "times"), k = tensor_arg(a[1], "tokens"), ref = tensor_arg(a[2], "ref_logp"),
                 w = optional_tensor(a[3], "weight");
    const float beta = float_arg(a[4]), smoothing = float_arg(a[5]);
    const bool save = bool_arg(a[6]);
    Objective r;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        r = preference_objective(choice_args(t, k, w, "tokens"), ref, beta, smoothing, save);
    }
    return wrap3(r.total, r.stats, r.coef);
    END_HANDLE_TH_ERRORS
}

// objective_grad(times, tokens, stats, coef, upstream) -> dtimes
SNNTC_METHOD(py_objective_grad) {
    HANDLE_TH_ERRORS
    arity(n, 5, "objective_grad");
    const Tensor t = tensor_arg(a[0], "times"), k = tensor_arg(a[1], "tokens"), s = tensor_arg(a[2], "stats"), c = tensor_arg(a[3], "coef"),
                 up = tensor_arg(a[4], "upstream");
    Tensor d;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        d = objective_grad(choice_args(t, k, Tensor(), "tokens"), s, c, up);
    }
    return wrap(d);
    END_HANDLE_TH_ERRORS
}

double double_arg(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}

// A number, or a tensor with one for each row or sequence.
PerRow per_row_arg(PyObject* o) {
    if (THPVariable_Check(o)) return PerRow{THPVariable_Unpack(o), 1.0f};
    return PerRow{Tensor(), float_arg(o)};
}

// history, lengths, prompts, repetition, presence, frequency, delay, allowed
RuleIn rule_in(PyObject* const* a) {
    RuleIn in{optional_tensor(a[0], "history"), optional_tensor(a[1], "lengths"), optional_tensor(a[2], "prompts"), per_row_arg(a[3]),
              per_row_arg(a[4]), per_row_arg(a[5]), optional_tensor(a[6], "delay"), optional_tensor(a[7], "allowed")};
    return in;
}

// rule_layer(times, history, lengths, prompts, repetition, presence, frequency, delay, allowed) -> ruled times, differentiable in times
SNNTC_METHOD(py_rule_layer) {
    HANDLE_TH_ERRORS
    arity(n, 9, "rule_times");
    const Tensor t = tensor_arg(a[0], "times");
    const RuleIn in = rule_in(a + 1);
    if (!plain({t, in.history, in.lengths, in.prompts, in.repetition.each, in.presence.each, in.frequency.each, in.delay, in.allowed}))
        return general("rule_layer", a, n);
    Tensor out;
    {
        NoGil nogil;
        out = rule_layer(rule_set(t, in), in);
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// rule_times(the same) -> ruled times, without a graph
SNNTC_METHOD(py_rule_times) {
    HANDLE_TH_ERRORS
    arity(n, 9, "rule_times");
    const Tensor t = tensor_arg(a[0], "times");
    const RuleIn in = rule_in(a + 1);
    Tensor out;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        out = rule_times(rule_set(t, in));
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// rule_times_grad(grad, times, history, lengths, repetition, allowed) -> gradient by the times
SNNTC_METHOD(py_rule_times_grad) {
    HANDLE_TH_ERRORS
    arity(n, 6, "rule_times_grad");
    const Tensor g = tensor_arg(a[0], "grad"), t = tensor_arg(a[1], "times");
    RuleIn in{};
    in.history = optional_tensor(a[2], "history"); in.lengths = optional_tensor(a[3], "lengths");
    in.repetition = per_row_arg(a[4]); in.allowed = optional_tensor(a[5], "allowed");
    Tensor d;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        d = rule_times_grad(g, rule_set(t, in));
    }
    return wrap(d);
    END_HANDLE_TH_ERRORS
}

// choose_tokens(times, uniform, temperature, history, lengths, prompts, repetition, presence, frequency, delay, allowed) -> (tokens, logp)
SNNTC_METHOD(py_choose_tokens) {
    HANDLE_TH_ERRORS
    arity(n, 11, "choose_tokens");
    const Tensor t = tensor_arg(a[0], "times"), u = optional_tensor(a[1], "uniform");
    const PerRow heat = per_row_arg(a[2]);
    const RuleIn in = rule_in(a + 3);
    Choice c;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        c = choose_tokens(rule_set(t, in), u, heat);
    }
    return wrap2(c.tokens, c.logp);
    END_HANDLE_TH_ERRORS
}

// grad_norm(list of gradients) -> norm
SNNTC_METHOD(py_grad_norm) {
    HANDLE_TH_ERRORS
    arity(n, 1, "grad_norm");
    const std::vector<Tensor> gs = tensor_list(a[0], "gradients");
    Tensor norm;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        norm = grad_norm(gs);
    }
    return wrap(norm);
    END_HANDLE_TH_ERRORS
}

Moments moments_in(PyObject* const* a) {
    Moments m{tensor_list(a[0], "first"), tensor_list(a[1], "second"), {}, {}, a[2] != Py_None};
    TORCH_CHECK_VALUE((a[2] == Py_None) == (a[3] == Py_None), "adamw: first_scale and second_scale go together");
    if (m.coded) {
        m.first_scale = tensor_list(a[2], "first_scale");
        m.second_scale = tensor_list(a[3], "second_scale");
    }
    return m;
}

// adamw_update(weights, gradients, first, second, first_scale, second_scale, step, lr, beta1, beta2, eps, weight_decay, norm, max_norm, seed, paired)
SNNTC_METHOD(py_adamw_update) {
    HANDLE_TH_ERRORS
    arity(n, 16, "adamw_update");
    const std::vector<Tensor> ws = tensor_list(a[0], "params"), gs = tensor_list(a[1], "grads");
    const Moments m = moments_in(a + 2);
    snntc_adamw how{};
    const Tensor steps = THPVariable_Check(a[6]) ? THPVariable_Unpack(a[6]) : Tensor();
    if (!steps.defined()) how.step = int_arg(a[6]);
    how.lr = double_arg(a[7]); how.beta1 = double_arg(a[8]); how.beta2 = double_arg(a[9]); how.eps = double_arg(a[10]);
    how.weight_decay = double_arg(a[11]);
    const Tensor norm = optional_tensor(a[12], "norm");
    how.max_norm = double_arg(a[13]);
    how.seed = PyLong_AsUnsignedLongLongMask(a[14]);
    if (PyErr_Occurred()) throw python_error();
    how.paired = PyObject_IsTrue(a[15]);
    if (how.paired < 0) throw python_error();
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        adamw_update(ws, gs, m, steps, norm, how);
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyObject* wrap_list(const std::vector<Tensor>& v) {
    PyObject* list = PyList_New((Py_ssize_t)v.size());
    for (size_t i = 0; list && i < v.size(); ++i) {
        PyObject* t = wrap(v[i]);
        if (!t) { Py_DECREF(list); return nullptr; }
        PyList_SET_ITEM(list, (Py_ssize_t)i, t);
    }
    return list;
}

// adamw_moments(first, second, first_scale, second_scale) -> (list of first moments, list of second moments), float32
SNNTC_METHOD(py_adamw_moments) {
    HANDLE_TH_ERRORS
    arity(n, 4, "adamw_moments");
    const Moments m = moments_in(a);
    TORCH_CHECK_VALUE(m.coded, "adamw: moments are read back from codes and scales");
    MomentsOut out;
    {
        NoGil nogil;
        at::AutoGradMode no_grad(false);
        out = adamw_moments(m);
    }
    PyObject *first = wrap_list(out.first), *second = wrap_list(out.second);
    PyObject* both = first && second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first); Py_XDECREF(second);
    return both;
    END_HANDLE_TH_ERRORS
}

// bind(path, SnntcLibraryError, SnntcError, params_array, general paths): looks the C ABI up in the library loaded from `path`
SNNTC_METHOD(py_bind) {
    HANDLE_TH_ERRORS
    arity(n, 5, "bind");
    const char* path = PyUnicode_AsUTF8(a[0]);
    if (!path) throw python_error();
    TORCH_CHECK_TYPE(PyDict_Check(a[4]), "bind takes a dict of general paths");
    for (int i = 1; i < 5; ++i) Py_INCREF(a[i]);
    Py_XDECREF(g_library_error); Py_XDECREF(g_error); Py_XDECREF(g_params); Py_XDECREF(g_general);
    g_library_error = a[1]; g_error = a[2]; g_params = a[3]; g_general = a[4];
    void* handle = dlopen(path, RTLD_NOW | RTLD_LOCAL);
    if (!handle) raise_class(g_library_error, message_args, 0, std::string("cannot load ") + path + ": " + dlerror());
    Library l;
#define SNNTC_LOOKUP(f)                                                                                            \
    l.f = reinterpret_cast<decltype(l.f)>(dlsym(handle, #f));                                                      \
    if (!l.f) raise_class(g_library_error, message_args, 0, std::string(path) + " lacks symbol " #f);
    SNNTC_BOUND(SNNTC_LOOKUP)
#undef SNNTC_LOOKUP
    lib = l;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

#define SNNTC_ENTRY(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {SNNTC_ENTRY(bind), SNNTC_ENTRY(fc_forward), SNNTC_ENTRY(fc_layer), SNNTC_ENTRY(fc_backward),
                           SNNTC_ENTRY(cv_forward), SNNTC_ENTRY(cv_layer), SNNTC_ENTRY(cv_same), SNNTC_ENTRY(cv_backward),
                           SNNTC_ENTRY(min_pool), SNNTC_ENTRY(min_pool_layer), SNNTC_ENTRY(pad_layer), SNNTC_ENTRY(time_loss),
                           SNNTC_ENTRY(loss_layer), SNNTC_ENTRY(sgd_update), SNNTC_ENTRY(plain), SNNTC_ENTRY(encode_time),
                           SNNTC_ENTRY(constraint_cost), SNNTC_ENTRY(recipe_step), SNNTC_ENTRY(embed_tokens),
                           SNNTC_ENTRY(embed_tokens_grad), SNNTC_ENTRY(embed_layer), SNNTC_ENTRY(gated_scan),
                           SNNTC_ENTRY(gated_scan_grad), SNNTC_ENTRY(gated_layer), SNNTC_ENTRY(gated_step), SNNTC_ENTRY(time_logp),
                           SNNTC_ENTRY(policy_loss), SNNTC_ENTRY(policy_layer), SNNTC_ENTRY(preference_loss),
                           SNNTC_ENTRY(preference_layer), SNNTC_ENTRY(policy_objective),
                           SNNTC_ENTRY(preference_objective), SNNTC_ENTRY(objective_grad), SNNTC_ENTRY(rule_layer),
                           SNNTC_ENTRY(rule_times), SNNTC_ENTRY(rule_times_grad), SNNTC_ENTRY(choose_tokens), SNNTC_ENTRY(grad_norm),
                           SNNTC_ENTRY(adamw_update), SNNTC_ENTRY(adamw_moments), {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_binding", "Native host path of the SNN-TC ops.", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&g_module); }
