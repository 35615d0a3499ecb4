// The operators around the recurrences, from torch tensors to the C ABI (include/t2fw_hip.h): checks, allocations, launches, and
// their gradients as nodes of torch's graph.  The nodes are C++ ones: they cost a call a few microseconds where a Python
// autograd function costs 44 to 91 (host.cpp).  A backward runs on the stream of its forward, as torch runs every node.
#include "host.hpp"

#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/custom_function.h>

#include <algorithm>

namespace t2fw_host {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

double real(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
Tensor optional_tensor(PyObject *o) { return o == Py_None ? Tensor() : tensor(o); }
// A node's arguments that may be missing go to it as optional ones, which torch does not look into where there is none
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : std::nullopt; }
Tensor of(const Maybe &t) { return t.has_value() ? *t : Tensor(); }
bool truth(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}
void *data(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

int32_t dtype_code(const Tensor &t, const char *name) {
    switch (t.scalar_type()) {
        case at::kFloat: return T2FW_F32;
        case at::kHalf: return T2FW_F16;
        case at::kBFloat16: return T2FW_BF16;
        case at::kDouble: return T2FW_F64;
        default: TORCH_CHECK(false, "t2fw: unsupported dtype ", t.scalar_type(), " of ", name);
    }
}
at::ScalarType accumulators_type(const Tensor &t) { return t.scalar_type() == at::kDouble ? at::kDouble : at::kFloat; }

void check_on(const Tensor &t, const Tensor &like, const char *name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.layout() == at::kStrided, name, " must be a dense tensor");
    // (its memory holds the other sign)
    TORCH_CHECK(!t.is_neg(), name, " is a negated view: call resolve_neg()");
    TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", not on ", like.device());
}
void check_contiguous(const Tensor &t, const Tensor &like, const char *name) {
    check_on(t, like, name);
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}
void check_sizes(const Tensor &t, at::IntArrayRef sizes, const char *name) {
    TORCH_CHECK(t.sizes() == sizes, "t2fw: ", name, " is ", t.sizes(), ", expected ", sizes);
}
void check_type(const Tensor &t, at::ScalarType type, const char *name) {
    TORCH_CHECK(t.scalar_type() == type, "t2fw: ", name, " is ", t.scalar_type(), ", expected ", type);
}
bool wants_grad(std::initializer_list<Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor &t : ts)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}
// Forward-mode derivatives: there are none, and a result without its tangent would pass for one whose tangent is zero
void no_tangents(std::initializer_list<Tensor> ts, const char *what) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor &t : ts) TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "t2fw: ", what, " has no forward-mode derivatives");
}
// The gradients are results of kernels that torch knows nothing of
void once(const char *what) { TORCH_CHECK(!at::GradMode::is_enabled(), "t2fw: ", what, " can be differentiated once only (create_graph)"); }

// What a node has saved, dense and of the type and number of elements that its kernels take: hooks on saved tensors may bring it back in
// another order of memory
Tensor restored(const Tensor &t, const Tensor &like, at::ScalarType type, int64_t numel) {
    check_on(t, like, "a saved tensor");
    check_type(t, type, "a saved tensor");
    TORCH_CHECK(t.numel() == numel, "t2fw: a saved tensor has ", t.numel(), " elements, expected ", numel);
    return t.contiguous();
}

// An address in a node's saved data
int64_t as_integer(void *p) { return (int64_t)(uintptr_t)p; }
void *as_address(const c10::IValue &v) { return reinterpret_cast<void *>((uintptr_t)v.toInt()); }

// ---- gated_scan ---------------------------------------------------------------------------------------------------
// (a gradient may be a view that torch negates when it reads it)
// x, f [B, T, D] with dense channels; anything else is copied (gradients that are expanded scalars, say)
Tensor dense_channels(const Tensor &t) {
    return t.size(2) <= 1 || t.stride(2) == 1 ? t.resolve_neg() : t.contiguous().resolve_neg();
}

struct ScanResult {
    Tensor out, last, ckpt;
};
ScanResult scan_forward(const Tensor &x, const Tensor &f, const Tensor &state, const Tensor &lengths, int32_t flags, bool need_grad, void *stream) {
    const int64_t B = x.size(0), T = x.size(1), D = x.size(2);
    const int32_t dtype = dtype_code(x, "x");
    ScanResult r;
    r.out = at::empty({B, T, D}, x.options());
    r.last = at::empty({B, D}, x.options().dtype(accumulators_type(x)));
    if (need_grad) r.ckpt = bytes_like(x, (int64_t)t2fw_gated_scan_checkpoint_bytes(B, T, D, dtype));
    const size_t bytes = t2fw_gated_scan_workspace_bytes(B, T, D, dtype);
    Tensor ws;
    if (bytes > 0) ws = bytes_like(x, (int64_t)bytes);
    const int64_t strides[4] = {x.stride(0), x.stride(1), f.stride(0), f.stride(1)};
    done(t2fw_gated_scan_forward(x.data_ptr(), f.data_ptr(), data(state), data(lengths), r.out.data_ptr(), r.last.data_ptr(), data(r.ckpt), B, T, D,
                                 strides, dtype, flags, data(ws), bytes, stream));
    return r;
}

struct GatedScan : torch::autograd::Function<GatedScan> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &f, const Maybe &state_, const Maybe &lengths_, int64_t flags,
                                 int64_t stream) {
        const Tensor state = of(state_), lengths = of(lengths_);
        const ScanResult r = scan_forward(x, f, state, lengths, (int32_t)flags, true, reinterpret_cast<void *>((uintptr_t)stream));
        ctx->save_for_backward({x, f, lengths, r.ckpt});
        ctx->saved_data["flags"] = flags;
        ctx->saved_data["stream"] = stream;
        ctx->saved_data["state"] = state.defined();
        ctx->set_materialize_grads(false);
        return {r.out, r.last};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        once("gated_scan");
        const variable_list saved = ctx->get_saved_variables();
        check_on(saved[0], saved[0], "a saved tensor");
        check_on(saved[1], saved[0], "a saved tensor");
        TORCH_CHECK(saved[0].dim() == 3, "t2fw: a saved tensor has ", saved[0].dim(), " axes, expected 3");
        check_type(saved[1], saved[0].scalar_type(), "a saved tensor");
        check_sizes(saved[1], saved[0].sizes(), "a saved tensor");
        const c10::DeviceGuard guard(saved[0].device());
        const Tensor x = dense_channels(saved[0]), f = dense_channels(saved[1]);
        const int64_t B = x.size(0), T = x.size(1), D = x.size(2);
        const int32_t dtype = dtype_code(x, "x");
        const Tensor ckpt = restored(saved[3], x, at::kByte, (int64_t)t2fw_gated_scan_checkpoint_bytes(B, T, D, dtype));
        const bool wide = (ctx->saved_data["flags"].toInt() & T2FW_SCAN_LENGTHS64) != 0;
        const Tensor lengths = saved[2].defined() ? restored(saved[2], x, wide ? at::kLong : at::kInt, B) : Tensor();
        // a result that nothing depends on has no gradient
        const Tensor go = grads[0].defined() ? dense_channels(grads[0]) : at::zeros({1}, x.options()).expand({B, T, D}).contiguous();
        const Tensor gs = grads[1].defined() ? grads[1].contiguous().resolve_neg() : Tensor();
        check_type(go, x.scalar_type(), "the gradient");
        check_sizes(go, x.sizes(), "the gradient");
        if (gs.defined()) {
            check_type(gs, accumulators_type(x), "the state's gradient");
            check_sizes(gs, {B, D}, "the state's gradient");
        }
        const Tensor dx = at::empty({B, T, D}, x.options()), df = at::empty({B, T, D}, f.options());
        Tensor ds, ws;
        if (ctx->saved_data["state"].toBool()) ds = at::empty({B, D}, x.options().dtype(accumulators_type(x)));
        const size_t bytes = t2fw_gated_scan_workspace_bytes(B, T, D, dtype);
        if (bytes > 0) ws = bytes_like(x, (int64_t)bytes);
        const int64_t strides[6] = {x.stride(0), x.stride(1), f.stride(0), f.stride(1), go.stride(0), go.stride(1)};
        done(t2fw_gated_scan_backward(go.data_ptr(), data(gs), x.data_ptr(), f.data_ptr(), data(lengths), ckpt.data_ptr(), dx.data_ptr(),
                                      df.data_ptr(), data(ds), B, T, D, strides, dtype, (int32_t)ctx->saved_data["flags"].toInt(), data(ws), bytes,
                                      as_address(ctx->saved_data["stream"])));
        return {dx, df, ds, Tensor(), Tensor(), Tensor()};
    }
};

void check_lengths(const Tensor &lengths, const Tensor &x) {
    if (!lengths.defined()) return;
    check_contiguous(lengths, x, "lengths");
    TORCH_CHECK(lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong, "t2fw: lengths are ", lengths.scalar_type(),
                ", expected int32 or int64");
    check_sizes(lengths, {x.size(0)}, "lengths");
}

// gated_scan(x, f, state or None, lengths or None, logits, stream) -> (h, last state)
PyObject *gated_scan(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 6);
    const Tensor x = tensor(a[0]), f = tensor(a[1]), state = optional_tensor(a[2]), lengths = optional_tensor(a[3]);
    check_on(x, x, "x");
    no_tangents({x, f, state}, "gated_scan");
    check_on(f, x, "f");
    TORCH_CHECK(x.dim() == 3 && x.size(2) >= 1, "t2fw: expected x, f [B, T, D] with at least one channel, x is ", x.sizes());
    check_sizes(f, x.sizes(), "f");
    dtype_code(x, "x");
    check_type(f, x.scalar_type(), "f");
    TORCH_CHECK(x.size(2) == 1 || (x.stride(2) == 1 && f.stride(2) == 1), "x and f must be contiguous along their channels");
    if (state.defined()) {
        check_contiguous(state, x, "state");
        check_sizes(state, {x.size(0), x.size(2)}, "state");
        check_type(state, accumulators_type(x), "state");
    }
    check_lengths(lengths, x);
    const int64_t flags = (truth(a[4]) ? T2FW_SCAN_LOGITS : 0) |
                          (lengths.defined() && lengths.scalar_type() == at::kLong ? T2FW_SCAN_LENGTHS64 : 0);
    void *const stream = address(a[5]);
    const c10::DeviceGuard guard(x.device());
    pybind11::gil_scoped_release release;
    if (!wants_grad({x, f, state})) {
        const ScanResult r = scan_forward(x, f, state, lengths, (int32_t)flags, false, stream);
        pybind11::gil_scoped_acquire acquire;
        return wrapped({r.out, r.last});
    }
    const variable_list r = GatedScan::apply(x, f, maybe(state), maybe(lengths), flags, as_integer(stream));
    pybind11::gil_scoped_acquire acquire;
    return wrapped({r[0], r[1]});
    END_HANDLE_TH_ERRORS
}

// gated_scan_step(x, f, state, out or None, logits, inplace, stream) -> (h, state)
PyObject *gated_scan_step(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 7);
    const Tensor &x = tensor(a[0]), &f = tensor(a[1]), &state = tensor(a[2]);
    check_contiguous(x, x, "x");
    check_contiguous(f, x, "f");
    check_contiguous(state, x, "state");
    TORCH_CHECK(x.dim() == 2 && x.size(1) >= 1, "t2fw: expected x, f [B, D] with at least one channel, x is ", x.sizes());
    check_sizes(f, x.sizes(), "f");
    check_sizes(state, x.sizes(), "state");
    const int32_t dtype = dtype_code(x, "x");
    check_type(f, x.scalar_type(), "f");
    check_type(state, accumulators_type(x), "state");
    TORCH_CHECK(!wants_grad({x, f, state}), "t2fw: gated_scan_step has no gradients: call gated_scan, or this under torch.no_grad()");
    Tensor out = optional_tensor(a[3]);
    no_tangents({x, f, state, out}, "gated_scan_step");
    if (out.defined()) {
        check_contiguous(out, x, "out");
        check_sizes(out, x.sizes(), "out");
        check_type(out, x.scalar_type(), "out");
    }
    const c10::DeviceGuard guard(x.device());
    if (!out.defined()) out = at::empty(x.sizes(), x.options());
    const bool inplace = truth(a[5]);
    const Tensor next = inplace ? state : at::empty(state.sizes(), state.options());
    const int32_t flags = truth(a[4]) ? T2FW_SCAN_LOGITS : 0;
    void *const stream = address(a[6]);
    done(unlocked([&] {
        return t2fw_gated_scan_step(x.data_ptr(), f.data_ptr(), state.data_ptr(), out.data_ptr(), next.data_ptr(), x.size(0), x.size(1), dtype,
                                    flags, stream);
    }));
    // written behind torch's back
    if (inplace && !state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
    if (a[3] != Py_None && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
    return wrapped({out, next});
    END_HANDLE_TH_ERRORS
}

// ---- residual_rms_norm --------------------------------------------------------------------------------------------
struct NormCall {
    int64_t N, D;
    int32_t dtype, flags;
};
NormCall check_norm(const Tensor &x, const Tensor &res, const Tensor &w) {
    NormCall c;
    check_contiguous(x, x, "x");
    check_contiguous(w, x, "weight");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "t2fw: expected x [..., D] with at least one column, x is ", x.sizes());
    c.D = x.size(-1);
    c.N = x.numel() / c.D;
    c.dtype = dtype_code(x, "x");
    c.flags = 0;
    const bool narrow = c.dtype == T2FW_F16 || c.dtype == T2FW_BF16;
    check_sizes(w, {c.D}, "weight");
    if (narrow && w.scalar_type() == at::kFloat) c.flags |= T2FW_NORM_WEIGHT_F32;
    else check_type(w, x.scalar_type(), "weight");
    if (res.defined()) {
        check_contiguous(res, x, "residual");
        check_sizes(res, x.sizes(), "residual");
        if (narrow && res.scalar_type() == at::kFloat) c.flags |= T2FW_NORM_STREAM_F32;
        else check_type(res, x.scalar_type(), "residual");
    }
    return c;
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Maybe &res_, const Tensor &w, double eps, int64_t N, int64_t D,
                                 int64_t dtype, int64_t flags, int64_t stream) {
        const Tensor res = of(res_);
        const Tensor y = at::empty(x.sizes(), x.options());
        const Tensor stored = res.defined() ? at::empty(res.sizes(), res.options()) : Tensor();
        done(t2fw_rms_norm_forward(x.data_ptr(), data(res), w.data_ptr(), y.data_ptr(), data(stored), N, D, eps, (int32_t)dtype, (int32_t)flags,
                                   reinterpret_cast<void *>((uintptr_t)stream)));
        // without a residual the stream is x itself
        ctx->save_for_backward({res.defined() ? stored : x, w});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["N"] = N;
        ctx->saved_data["D"] = D;
        ctx->saved_data["dtype"] = dtype;
        ctx->saved_data["flags"] = flags;
        ctx->saved_data["stream"] = stream;
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        ctx->saved_data["residual"] = res.defined();
        ctx->set_materialize_grads(false);
        return res.defined() ? variable_list{y, stored} : variable_list{y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        once("residual_rms_norm");
        const variable_list saved = ctx->get_saved_variables();
        const c10::DeviceGuard guard(saved[0].device());
        const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
        const int64_t N = ctx->saved_data["N"].toInt(), D = ctx->saved_data["D"].toInt();
        const int32_t dtype = (int32_t)ctx->saved_data["dtype"].toInt(), flags = (int32_t)ctx->saved_data["flags"].toInt();
        const bool residual = ctx->saved_data["residual"].toBool(), wide = (flags & T2FW_NORM_STREAM_F32) != 0;
        const Tensor stored = restored(saved[0], saved[0], wide ? at::kFloat : type, N * D);
        const Tensor w = restored(saved[1], stored, (flags & T2FW_NORM_WEIGHT_F32) != 0 ? at::kFloat : type, D);
        const auto options = stored.options().dtype(type);
        const Tensor gy = grads[0].defined() ? grads[0].contiguous().resolve_neg() : at::zeros(stored.sizes(), options);
        const Tensor gres = residual && grads[1].defined() ? grads[1].contiguous().resolve_neg() : Tensor();
        const Tensor dx = at::empty(stored.sizes(), options), dw = at::empty(w.sizes(), w.options());
        const Tensor dres = wide ? at::empty(stored.sizes(), stored.options()) : Tensor();
        const size_t bytes = t2fw_rms_norm_backward_workspace_bytes(N, D, dtype);
        Tensor ws;
        if (bytes > 0) ws = bytes_like(stored, (int64_t)bytes);
        done(t2fw_rms_norm_backward(gy.data_ptr(), data(gres), stored.data_ptr(), w.data_ptr(), dx.data_ptr(), data(dres), dw.data_ptr(), N, D,
                                    ctx->saved_data["eps"].toDouble(), dtype, flags, data(ws), bytes, as_address(ctx->saved_data["stream"])));
        // one array serves both sides of the addition where their types are one
        const Tensor for_res = !residual ? Tensor() : wide ? dres : dx;
        return {dx, for_res, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// residual_rms_norm(x, residual or None, weight, eps, stream) -> (y, stream after the addition, or None)
PyObject *residual_rms_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 5);
    const Tensor x = tensor(a[0]), res = optional_tensor(a[1]), w = tensor(a[2]);
    const NormCall c = check_norm(x, res, w);
    no_tangents({x, res, w}, "residual_rms_norm");
    const double eps = real(a[3]);
    void *const stream = address(a[4]);
    const c10::DeviceGuard guard(x.device());
    pybind11::gil_scoped_release release;
    if (!wants_grad({x, res, w})) {
        const Tensor y = at::empty(x.sizes(), x.options());
        const Tensor stored = res.defined() ? at::empty(res.sizes(), res.options()) : Tensor();
        done(t2fw_rms_norm_forward(x.data_ptr(), data(res), w.data_ptr(), y.data_ptr(), data(stored), c.N, c.D, eps, c.dtype, c.flags, stream));
        pybind11::gil_scoped_acquire acquire;
        return wrapped({y, stored});
    }
    const variable_list r = ResidualNorm::apply(x, maybe(res), w, eps, c.N, c.D, (int64_t)c.dtype, (int64_t)c.flags, as_integer(stream));
    pybind11::gil_scoped_acquire acquire;
    return wrapped({r[0], r.size() > 1 ? r[1] : Tensor()});
    END_HANDLE_TH_ERRORS
}

// residual_rms_norm_fp8(x, residual or None, weight, eps, group, stream) -> (q, scales, stream after the addition, or None)
PyObject *residual_rms_norm_fp8(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 6);
    const Tensor &x = tensor(a[0]), res = optional_tensor(a[1]), &w = tensor(a[2]);
    const NormCall c = check_norm(x, res, w);
    TORCH_CHECK(!wants_grad({x, res, w}), "t2fw: residual_rms_norm_fp8 has no gradients: call it under torch.no_grad()");
    no_tangents({x, res, w}, "residual_rms_norm_fp8");
    const double eps = real(a[3]);
    const int64_t group = integer(a[4]);
    void *const stream = address(a[5]);
    const c10::DeviceGuard guard(x.device());
    const Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
    std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end());
    sizes.back() = group > 0 ? (c.D + group - 1) / group : 1;
    const Tensor scales = at::empty(sizes, x.options().dtype(at::kFloat));
    const Tensor stored = res.defined() ? at::empty(res.sizes(), res.options()) : Tensor();
    done(unlocked([&] {
        return t2fw_rms_norm_forward_fp8(x.data_ptr(), data(res), w.data_ptr(), q.data_ptr(), (float *)scales.data_ptr(), data(stored), c.N, c.D,
                                         group, eps, c.dtype, c.flags, stream);
    }));
    return wrapped({q, scales, stored});
    END_HANDLE_TH_ERRORS
}

// ---- policy_loss --------------------------------------------------------------------------------------------------
struct LossCall {
    double low, high, kl, scale;
};
struct LossResult {
    Tensor loss, logp, tops, coef;
};
LossResult loss_forward(const Tensor &logits, const Tensor &targets, const Tensor &old_logp, const Tensor &ref_logp, const Tensor &adv,
                        const Tensor &mask, const Tensor &d_logits, const LossCall &c, void *stream) {
    const int64_t V = logits.size(-1), N = targets.numel();
    const auto options = logits.options().dtype(at::kFloat);
    LossResult r;
    r.loss = at::empty({}, options);
    r.logp = at::empty(targets.sizes(), options);
    // the largest logits and sums, the coefficients of the rows, and the call's scratch
    const size_t bytes = t2fw_policy_loss_workspace_bytes(N);
    const Tensor all = at::empty({3, N}, options), ws = bytes_like(logits, (int64_t)bytes);
    r.tops = all.narrow(0, 0, 2);
    r.coef = all.select(0, 2);
    done(t2fw_policy_loss_forward(logits.data_ptr(), (const int64_t *)targets.data_ptr(), (const float *)old_logp.data_ptr(),
                                  (const float *)ref_logp.data_ptr(), (const float *)adv.data_ptr(), data(mask), (float *)r.loss.data_ptr(),
                                  (float *)r.logp.data_ptr(), (float *)r.tops.data_ptr(), (float *)r.coef.data_ptr(), data(d_logits), N, V,
                                  (float)c.low, (float)c.high, (float)c.kl, (float)c.scale, dtype_code(logits, "logits"), ws.data_ptr(), bytes,
                                  stream));
    return r;
}

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &targets, const Tensor &old_logp, const Tensor &ref_logp,
                                 const Tensor &adv, const Maybe &mask_, double low, double high, double kl, double scale, int64_t stream) {
        const Tensor mask = of(mask_);
        // float16 losses are scaled before their gradients are taken, by a factor that is not known here: their gradient is made in the
        // backward.  The other types' is made now, for a gradient of the loss of one, while the row is at hand.
        Tensor made;
        if (logits.scalar_type() != at::kHalf) made = at::empty(logits.sizes(), logits.options());
        const LossResult r = loss_forward(logits, targets, old_logp, ref_logp, adv, mask, made, {low, high, kl, scale},
                                          reinterpret_cast<void *>((uintptr_t)stream));
        ctx->save_for_backward({logits, targets, r.tops, r.coef});
        if (made.defined()) ctx->saved_data["made"] = made;
        ctx->saved_data["N"] = targets.numel();
        ctx->saved_data["V"] = logits.size(-1);
        ctx->saved_data["type"] = (int64_t)logits.scalar_type();
        ctx->saved_data["stream"] = stream;
        ctx->mark_non_differentiable({r.logp});
        return {r.loss, r.logp};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        once("policy_loss");
        const variable_list saved = ctx->get_saved_variables();
        const c10::DeviceGuard guard(saved[0].device());
        const int64_t N = ctx->saved_data["N"].toInt(), V = ctx->saved_data["V"].toInt();
        const Tensor logits = restored(saved[0], saved[0], (at::ScalarType)ctx->saved_data["type"].toInt(), N * V);
        const Tensor targets = restored(saved[1], logits, at::kLong, N), tops = restored(saved[2], logits, at::kFloat, 2 * N);
        const Tensor coef = restored(saved[3], logits, at::kFloat, N);
        const Tensor g = grads[0].contiguous().resolve_neg();
        Tensor d;
        int32_t flags = 0;
        const auto made = ctx->saved_data.find("made");
        if (made != ctx->saved_data.end()) {             // handed over once: what becomes of it then is its owner's
            d = made->second.toTensor();
            ctx->saved_data.erase(made);
            flags = T2FW_LOSS_UNLESS_ONE;
        } else {
            d = at::empty(logits.sizes(), logits.options());
        }
        done(t2fw_policy_loss_backward(logits.data_ptr(), (const int64_t *)targets.data_ptr(), (const float *)tops.data_ptr(),
                                       (const float *)coef.data_ptr(), (const float *)g.data_ptr(), d.data_ptr(), N, V,
                                       dtype_code(logits, "logits"), flags, as_address(ctx->saved_data["stream"])));
        return {d, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// policy_loss(logits, targets, old_logp, ref_logp, advantages, mask or None, low, high, kl, scale, stream) -> (loss, logp)
PyObject *policy_loss(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 11);
    const Tensor logits = tensor(a[0]), targets = tensor(a[1]), mask = optional_tensor(a[5]);
    const Tensor per[3] = {tensor(a[2]), tensor(a[3]), tensor(a[4])};
    check_contiguous(logits, logits, "logits");
    no_tangents({logits, per[0], per[1], per[2]}, "policy_loss");
    TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1, "t2fw: expected logits [..., V] with V of at least one, they are ", logits.sizes());
    TORCH_CHECK(dtype_code(logits, "logits") != T2FW_F64, "t2fw: unsupported dtype ", logits.scalar_type(), " of logits");
    const at::IntArrayRef tokens = logits.sizes().slice(0, logits.dim() - 1);
    check_contiguous(targets, logits, "targets");
    check_sizes(targets, tokens, "targets");
    check_type(targets, at::kLong, "targets");
    const char *const names[3] = {"old_logp", "ref_logp", "advantages"};
    for (int i = 0; i < 3; ++i) {
        check_contiguous(per[i], logits, names[i]);
        check_sizes(per[i], tokens, names[i]);
        check_type(per[i], at::kFloat, names[i]);
        TORCH_CHECK(!per[i].requires_grad() || !at::GradMode::is_enabled(), "t2fw: policy_loss has no gradient for ", names[i], ": detach() it");
    }
    if (mask.defined()) {
        check_contiguous(mask, logits, "mask");
        check_sizes(mask, tokens, "mask");
        check_type(mask, at::kBool, "mask");
    }
    const LossCall c{real(a[6]), real(a[7]), real(a[8]), real(a[9])};
    void *const stream = address(a[10]);
    const c10::DeviceGuard guard(logits.device());
    pybind11::gil_scoped_release release;
    if (!wants_grad({logits})) {
        const LossResult r = loss_forward(logits, targets, per[0], per[1], per[2], mask, Tensor(), c, stream);
        pybind11::gil_scoped_acquire acquire;
        return wrapped({r.loss, r.logp});
    }
    const variable_list r = PolicyLoss::apply(logits, targets, per[0], per[1], per[2], maybe(mask), c.low, c.high, c.kl, c.scale, as_integer(stream));
    pybind11::gil_scoped_acquire acquire;
    return wrapped({r[0], r[1]});
    END_HANDLE_TH_ERRORS
}

// ---- clip_grad_norm -----------------------------------------------------------------------------------------------
// An array that may be gone through element by element in the order of its memory
void check_dense(const Tensor &t, const Tensor &like, const char *name) {
    check_on(t, like, name);
    TORCH_CHECK(t.is_non_overlapping_and_dense(), name, " must be dense");
}

// Many workgroups write the results at once: none may share memory with another, nor with a gradient, but its own in place.
void check_apart(const std::vector<t2fw_clip_desc> &d, const std::vector<int64_t> &sizes) {
    struct Span {
        uintptr_t begin, end;
        bool operator<(const Span &o) const { return begin < o.begin; }
    };
    std::vector<Span> to;
    to.reserve(d.size());
    const auto span = [](const void *p, int64_t bytes) { return Span{reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + (uintptr_t)bytes}; };
    for (size_t i = 0; i < d.size(); ++i)
        if (d[i].dst != nullptr && d[i].n > 0) to.push_back(span(d[i].dst, d[i].n * sizes[2 * i + 1]));
    if (!std::is_sorted(to.begin(), to.end())) std::sort(to.begin(), to.end());
    for (size_t i = 1; i < to.size(); ++i) TORCH_CHECK(to[i - 1].end <= to[i].begin, "t2fw: two results of clip_grad_norm share memory");
    for (size_t i = 0; i < d.size(); ++i) {
        if (to.empty() || d[i].n == 0 || (d[i].src == d[i].dst && d[i].src_dtype == d[i].dst_dtype)) continue;
        const Span s = span(d[i].src, d[i].n * sizes[2 * i]);
        // the first result that begins at the gradient's end or later; the one before it is the last that could reach into the gradient
        const auto next = std::lower_bound(to.begin(), to.end(), Span{s.end, s.end});
        TORCH_CHECK(next == to.begin() || (next - 1)->end <= s.begin, "t2fw: a result of clip_grad_norm shares memory with a gradient");
    }
}

// clip_grad_norm(sequence of tensors, largest norm, sequence of results, None for in place, False for the norm alone, stream) -> norm
PyObject *clip_grad_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 4);
    const pybind11::object grads = pybind11::reinterpret_steal<pybind11::object>(PySequence_Fast(a[0], "t2fw: expected a sequence of tensors"));
    if (!grads) throw python_error();
    const bool inplace = a[2] == Py_None, alone = a[2] == Py_False;
    pybind11::object outs;
    const Py_ssize_t count = PySequence_Fast_GET_SIZE(grads.ptr());
    TORCH_CHECK(count > 0, "t2fw: no gradients");
    if (!inplace && !alone) {
        outs = pybind11::reinterpret_steal<pybind11::object>(PySequence_Fast(a[2], "t2fw: expected a sequence of tensors"));
        if (!outs) throw python_error();
        TORCH_CHECK(PySequence_Fast_GET_SIZE(outs.ptr()) == count, "t2fw: ", count, " gradients and ", PySequence_Fast_GET_SIZE(outs.ptr()), " results");
    }
    const Tensor first = tensor(PySequence_Fast_GET_ITEM(grads.ptr(), 0));
    check_on(first, first, "gradients");
    std::vector<t2fw_clip_desc> d((size_t)count);
    std::vector<int64_t> sizes((size_t)count * 2);       // of an element of each gradient and of its result
    for (Py_ssize_t i = 0; i < count; ++i) {
        const Tensor &g = tensor(PySequence_Fast_GET_ITEM(grads.ptr(), i));
        check_dense(g, first, "every gradient");
        no_tangents({g}, "clip_grad_norm");
        d[i].src = g.data_ptr();
        d[i].dst = inplace ? g.data_ptr() : nullptr;
        d[i].n = g.numel();
        d[i].src_dtype = d[i].dst_dtype = dtype_code(g, "a gradient");
        sizes[2 * i] = sizes[2 * i + 1] = g.element_size();
        if (!outs) continue;
        const Tensor &o = tensor(PySequence_Fast_GET_ITEM(outs.ptr(), i));
        check_dense(o, first, "every result");
        no_tangents({o}, "clip_grad_norm");
        check_sizes(o, g.sizes(), "a result");
        TORCH_CHECK(o.strides() == g.strides() || (o.is_contiguous() && g.is_contiguous()), "t2fw: a result is laid out otherwise than its gradient");
        d[i].dst = o.data_ptr();
        d[i].dst_dtype = dtype_code(o, "a result");
        sizes[2 * i + 1] = o.element_size();
    }
    check_apart(d, sizes);
    const double most = real(a[1]);
    void *const stream = address(a[3]);
    const c10::DeviceGuard guard(first.device());
    const size_t bytes = t2fw_clip_workspace_bytes(d.data(), count);
    const Tensor norm = at::empty({}, first.options().dtype(at::kFloat)), ws = bytes_like(first, (int64_t)bytes);
    done(unlocked([&] {
        return t2fw_clip_grad_norm_f64(d.data(), count, most, (float *)norm.data_ptr(), ws.data_ptr(), bytes, stream);
    }));
    if (!alone)
        for (Py_ssize_t i = 0; i < count; ++i) {
            const Tensor &t = tensor(PySequence_Fast_GET_ITEM(inplace ? grads.ptr() : outs.ptr(), i));
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
        }
    return wrapped({norm});
    END_HANDLE_TH_ERRORS
}

}  // namespace

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef operator_methods[] = {METHOD(gated_scan), METHOD(gated_scan_step), METHOD(residual_rms_norm), METHOD(residual_rms_norm_fp8),
                                  METHOD(policy_loss), METHOD(clip_grad_norm), {nullptr, nullptr, 0, nullptr}};

}  // namespace t2fw_host
