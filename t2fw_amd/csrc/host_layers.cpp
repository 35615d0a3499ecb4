// The selective state space layer and beam search, from torch tensors to the C ABI (include/t2fw_hip.h): as host_ops.cpp.
#include "host_checks.hpp"

#include <algorithm>

namespace t2fw_host {
namespace {

// float32, float16, bfloat16
int32_t lowp_code(const Tensor &t, const char *name) {
    const int32_t code = dtype_code(t, name);
    TORCH_CHECK(code != T2FW_F64, "t2fw: unsupported dtype ", t.scalar_type(), " of ", name);
    return code;
}
// [B, D] with dense channels
void check_rows(const Tensor &t, const Tensor &like, const char *name) {
    check_on(t, like, name);
    TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, name, " must be contiguous along its channels");
}
void bump(const Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// The same memory for two of a step's arrays, one of which is written: no kernel may do that
bool overlap(const Tensor &a, const Tensor &b) {
    if (a.numel() == 0 || b.numel() == 0) return false;
    const auto extent = [](const Tensor &t) {
        int64_t n = 1;
        for (int64_t i = 0; i < t.dim(); ++i) n += (t.size(i) - 1) * t.stride(i);
        return n * (int64_t)t.element_size();
    };
    const auto x = reinterpret_cast<uintptr_t>(a.data_ptr()), y = reinterpret_cast<uintptr_t>(b.data_ptr());
    return x < y + (uintptr_t)extent(b) && y < x + (uintptr_t)extent(a);
}
void check_apart(const Tensor &written, std::initializer_list<Tensor> read, const char *what) {
    for (const Tensor &t : read) TORCH_CHECK(!t.defined() || !overlap(written, t), "t2fw: ", what, " shares memory with another tensor of the call");
}

// ---- short_conv ---------------------------------------------------------------------------------------------------
struct ConvResult {
    Tensor y, last;
};
ConvResult conv_forward(const Tensor &x, const Tensor &w, const Tensor &bias, const Tensor &state, const Tensor &lengths, int32_t flags, void *stream) {
    const int64_t B = x.size(0), T = x.size(1), D = x.size(2), taps = w.size(1);
    ConvResult r;
    r.y = at::empty({B, T, D}, x.options());
    r.last = at::empty({B, taps - 1, D}, x.options());
    const int64_t strides[2] = {x.stride(0), x.stride(1)};
    done(t2fw_short_conv_forward(x.data_ptr(), w.data_ptr(), data(bias), data(state), data(lengths), r.y.data_ptr(), r.last.data_ptr(), B, T, D, taps,
                                 strides, dtype_code(x, "x"), flags, stream));
    return r;
}

struct ShortConv : torch::autograd::Function<ShortConv> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const Maybe &bias_, const Maybe &state_, const Maybe &lengths_,
                                 int64_t flags, int64_t stream) {
        const Tensor bias = of(bias_), state = of(state_), lengths = of(lengths_);
        const ConvResult r = conv_forward(x, w, bias, state, lengths, (int32_t)flags, reinterpret_cast<void *>((uintptr_t)stream));
        ctx->save_for_backward({x, w, bias, state, lengths});
        ctx->saved_data["flags"] = flags;
        ctx->saved_data["stream"] = stream;
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        ctx->saved_data["taps"] = w.size(1);
        ctx->set_materialize_grads(false);
        return {r.y, r.last};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        once("short_conv");
        const variable_list saved = ctx->get_saved_variables();
        check_on(saved[0], saved[0], "a saved tensor");
        TORCH_CHECK(saved[0].dim() == 3, "t2fw: a saved tensor has ", saved[0].dim(), " axes, expected 3");
        check_type(saved[0], (at::ScalarType)ctx->saved_data["type"].toInt(), "a saved tensor");
        const c10::DeviceGuard guard(saved[0].device());
        const Tensor x = dense_channels(saved[0]);
        const int64_t B = x.size(0), T = x.size(1), D = x.size(2), taps = ctx->saved_data["taps"].toInt();
        const int32_t dtype = lowp_code(x, "x"), flags = (int32_t)ctx->saved_data["flags"].toInt();
        const auto wide = flags & T2FW_CONV_WEIGHT_F32 ? at::kFloat : x.scalar_type();
        const Tensor w = restored(saved[1], x, wide, D * taps), bias = saved[2].defined() ? restored(saved[2], x, wide, D) : Tensor();
        const Tensor state = saved[3].defined() ? restored(saved[3], x, x.scalar_type(), B * (taps - 1) * D) : Tensor();
        const Tensor lengths = saved[4].defined() ? restored(saved[4], x, flags & T2FW_CONV_LENGTHS64 ? at::kLong : at::kInt, B) : Tensor();
        // a result that nothing depends on has no gradient
        const Tensor gy = grads[0].defined() ? dense_channels(grads[0]) : at::zeros({1}, x.options()).expand({B, T, D}).contiguous();
        const Tensor gs = grads[1].defined() ? grads[1].contiguous().resolve_neg() : Tensor();
        check_type(gy, x.scalar_type(), "the gradient");
        check_sizes(gy, x.sizes(), "the gradient");
        if (gs.defined()) {
            check_type(gs, x.scalar_type(), "the state's gradient");
            check_sizes(gs, {B, taps - 1, D}, "the state's gradient");
        }
        const Tensor dx = at::empty({B, T, D}, x.options()), dw = at::empty({D, taps}, w.options());
        const Tensor db = bias.defined() ? at::empty({D}, bias.options()) : Tensor(), ds = state.defined() ? at::empty({B, taps - 1, D}, x.options()) : Tensor();
        const size_t bytes = t2fw_short_conv_backward_workspace_bytes(B, T, D, taps, dtype);
        Tensor ws;
        if (bytes > 0) ws = bytes_like(x, (int64_t)bytes);
        const int64_t strides[4] = {x.stride(0), x.stride(1), gy.stride(0), gy.stride(1)};
        done(t2fw_short_conv_backward(gy.data_ptr(), data(gs), x.data_ptr(), w.data_ptr(), data(bias), data(state), data(lengths), dx.data_ptr(),
                                      dw.data_ptr(), data(db), data(ds), B, T, D, taps, strides, dtype, flags, data(ws), bytes,
                                      as_address(ctx->saved_data["stream"])));
        return {dx, dw, db, ds, Tensor(), Tensor(), Tensor()};
    }
};

// x [.., D], weight [D, taps], bias [D] or none; -> flags
int32_t check_conv(const Tensor &x, const Tensor &w, const Tensor &bias) {
    lowp_code(x, "x");
    check_contiguous(w, x, "weight");
    TORCH_CHECK(w.dim() == 2 && w.size(0) == x.size(-1), "t2fw: expected weight [D, taps], it is ", w.sizes(), " for ", x.size(-1), " channels");
    int32_t flags = 0;
    if (x.scalar_type() != at::kFloat && w.scalar_type() == at::kFloat) flags |= T2FW_CONV_WEIGHT_F32;
    else check_type(w, x.scalar_type(), "weight");
    if (bias.defined()) {
        check_contiguous(bias, x, "bias");
        check_sizes(bias, {w.size(0)}, "bias");
        check_type(bias, w.scalar_type(), "bias");
    }
    return flags;
}

// short_conv(x, weight, bias or None, state or None, lengths or None, silu, stream) -> (y, last inputs)
PyObject *short_conv(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 7);
    const Tensor x = tensor(a[0]), w = tensor(a[1]), bias = optional_tensor(a[2]), state = optional_tensor(a[3]), lengths = optional_tensor(a[4]);
    check_on(x, x, "x");
    no_tangents({x, w, bias, state}, "short_conv");
    TORCH_CHECK(x.dim() == 3 && x.size(2) >= 1, "t2fw: expected x [B, T, D] with at least one channel, it is ", x.sizes());
    check_rows(x, x, "x");
    int64_t flags = check_conv(x, w, bias);
    if (state.defined()) {
        check_contiguous(state, x, "state");
        check_sizes(state, {x.size(0), w.size(1) - 1, x.size(2)}, "state");
        check_type(state, x.scalar_type(), "state");
    }
    check_lengths(lengths, x);
    if (truth(a[5])) flags |= T2FW_CONV_SILU;
    if (lengths.defined() && lengths.scalar_type() == at::kLong) flags |= T2FW_CONV_LENGTHS64;
    void *const stream = address(a[6]);
    TORCH_CHECK(w.size(1) >= 2 && w.size(1) <= 8, "t2fw: 2 to 8 taps, not ", w.size(1));
    const c10::DeviceGuard guard(x.device());
    pybind11::gil_scoped_release release;
    if (!wants_grad({x, w, bias, state})) {
        const ConvResult r = conv_forward(x, w, bias, state, lengths, (int32_t)flags, stream);
        pybind11::gil_scoped_acquire acquire;
        return wrapped({r.y, r.last});
    }
    const variable_list r = ShortConv::apply(x, w, maybe(bias), maybe(state), maybe(lengths), flags, as_integer(stream));
    pybind11::gil_scoped_acquire acquire;
    return wrapped({r[0], r[1]});
    END_HANDLE_TH_ERRORS
}

// short_conv_step(x, weight, state, bias or None, silu, out or None, inplace, stream) -> (y, state)
PyObject *short_conv_step(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 8);
    const Tensor x = tensor(a[0]), w = tensor(a[1]), state = tensor(a[2]), bias = optional_tensor(a[3]);
    Tensor out = optional_tensor(a[5]);
    check_on(x, x, "x");
    no_tangents({x, w, state, bias, out}, "short_conv_step");
    TORCH_CHECK(x.dim() == 2 && x.size(1) >= 1, "t2fw: expected x [B, D] with at least one channel, it is ", x.sizes());
    check_rows(x, x, "x");
    int32_t flags = check_conv(x, w, bias);
    TORCH_CHECK(w.size(1) >= 2 && w.size(1) <= 8, "t2fw: 2 to 8 taps, not ", w.size(1));
    check_contiguous(state, x, "state");
    check_sizes(state, {x.size(0), w.size(1) - 1, x.size(1)}, "state");
    check_type(state, x.scalar_type(), "state");
    TORCH_CHECK(!wants_grad({x, w, state, bias}), "t2fw: short_conv_step has no gradients: call short_conv, or this under torch.no_grad()");
    const bool inplace = truth(a[6]);
    if (inplace) check_apart(state, {x, w, bias, out}, "state");
    if (out.defined()) {
        check_contiguous(out, x, "out");
        check_sizes(out, x.sizes(), "out");
        check_type(out, x.scalar_type(), "out");
        TORCH_CHECK(!wants_grad({out}), "t2fw: short_conv_step has no gradients: out requires one");
        check_apart(out, {w, bias, state}, "out");
        TORCH_CHECK(!overlap(out, x) || (out.data_ptr() == x.data_ptr() && x.is_contiguous()), "t2fw: out shares memory with x");
    }
    const c10::DeviceGuard guard(x.device());
    if (!out.defined()) out = at::empty(x.sizes(), x.options());
    const Tensor next = inplace ? state : at::empty(state.sizes(), state.options());
    if (truth(a[4])) flags |= T2FW_CONV_SILU;
    void *const stream = address(a[7]);
    done(unlocked([&] {
        return t2fw_short_conv_step(x.data_ptr(), w.data_ptr(), data(bias), state.data_ptr(), out.data_ptr(), next.data_ptr(), x.size(0), x.size(1),
                                    w.size(1), x.stride(0), dtype_code(x, "x"), flags, stream);
    }));
    // written behind torch's back
    if (inplace) bump(state);
    if (a[5] != Py_None) bump(out);
    return wrapped({out, next});
    END_HANDLE_TH_ERRORS
}

// ---- selective_scan -----------------------------------------------------------------------------------------------
// x, dt, a, b, c, state, skip, gate, dt_bias, lengths, as the entry points have them; those that may be missing are undefined then
struct SelectInputs {
    Tensor x, dt, a, b, c, state, skip, gate, dt_bias, lengths;
};
struct SelectResult {
    Tensor y, last, ckpt;
};
// Steps further apart than the kernels address are brought together
Tensor near_steps(const Tensor &t) {
    return t.defined() && t.size(1) > 1 && t.stride(1) > (int64_t)(0xffffffffu / (16 * t.element_size())) ? t.contiguous() : t;
}
SelectResult select_forward(const SelectInputs &in, int32_t flags, bool need_grad, void *stream) {
    const SelectInputs i{near_steps(in.x), near_steps(in.dt), in.a, near_steps(in.b), near_steps(in.c), in.state, in.skip, near_steps(in.gate), in.dt_bias,
                         in.lengths};
    const int64_t B = i.x.size(0), T = i.x.size(1), D = i.x.size(2), N = i.a.size(1);
    SelectResult r;
    r.y = at::empty({B, T, D}, i.x.options());
    r.last = at::empty({B, D, N}, i.a.options());
    if (need_grad) r.ckpt = bytes_like(i.x, (int64_t)t2fw_selective_scan_checkpoint_bytes(B, T, D, N));
    const size_t bytes = t2fw_selective_scan_workspace_bytes(B, T, D, N);
    Tensor ws;
    if (bytes > 0) ws = bytes_like(i.x, (int64_t)bytes);
    const bool gated = i.gate.defined();
    const int64_t strides[10] = {i.x.stride(0), i.x.stride(1), i.dt.stride(0), i.dt.stride(1), i.b.stride(0), i.b.stride(1), i.c.stride(0), i.c.stride(1),
                                 gated ? i.gate.stride(0) : 0, gated ? i.gate.stride(1) : 0};
    done(t2fw_selective_scan_forward(i.x.data_ptr(), i.dt.data_ptr(), (const float *)i.a.data_ptr(), i.b.data_ptr(), i.c.data_ptr(),
                                     (const float *)data(i.skip), data(i.gate), (const float *)data(i.dt_bias), (const float *)data(i.state),
                                     data(i.lengths), r.y.data_ptr(), (float *)r.last.data_ptr(), r.ckpt.defined() && r.ckpt.numel() > 0 ? r.ckpt.data_ptr() : nullptr,
                                     B, T, D, N, strides, dtype_code(i.x, "x"), flags, data(ws), bytes, stream));
    return r;
}

struct SelectiveScan : torch::autograd::Function<SelectiveScan> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &dt, const Tensor &a, const Tensor &b, const Tensor &c,
                                 const Maybe &state, const Maybe &skip, const Maybe &gate, const Maybe &dt_bias, const Maybe &lengths, int64_t flags,
                                 int64_t stream) {
        const SelectInputs i{x, dt, a, b, c, of(state), of(skip), of(gate), of(dt_bias), of(lengths)};
        const SelectResult r = select_forward(i, (int32_t)flags, true, reinterpret_cast<void *>((uintptr_t)stream));
        ctx->save_for_backward({x, dt, a, b, c, i.skip, i.gate, i.dt_bias, i.lengths, r.ckpt});
        ctx->saved_data["flags"] = flags;
        ctx->saved_data["stream"] = stream;
        ctx->saved_data["state"] = i.state.defined();
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        ctx->saved_data["sizes"] = std::vector<int64_t>{x.size(0), x.size(1), x.size(2), a.size(1)};
        ctx->set_materialize_grads(false);
        return {r.y, r.last};
    }
    // a saved tensor of steps, as its sizes have to be
    static Tensor steps(const Tensor &t, const Tensor &like, at::ScalarType type, at::IntArrayRef sizes) {
        check_on(t, like, "a saved tensor");
        check_type(t, type, "a saved tensor");
        check_sizes(t, sizes, "a saved tensor");
        return near_steps(dense_channels(t));
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        once("selective_scan");
        const variable_list saved = ctx->get_saved_variables();
        const std::vector<int64_t> n = ctx->saved_data["sizes"].toIntVector();
        const int64_t B = n[0], T = n[1], D = n[2], N = n[3];
        const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
        const c10::DeviceGuard guard(saved[0].device());
        const Tensor x = steps(saved[0], saved[0], type, {B, T, D}), dt = steps(saved[1], x, type, {B, T, D});
        const Tensor a = restored(saved[2], x, at::kFloat, D * N), b = steps(saved[3], x, type, {B, T, N}), c = steps(saved[4], x, type, {B, T, N});
        const Tensor skip = saved[5].defined() ? restored(saved[5], x, at::kFloat, D) : Tensor();
        const Tensor gate = saved[6].defined() ? steps(saved[6], x, type, {B, T, D}) : Tensor();
        const Tensor bias = saved[7].defined() ? restored(saved[7], x, at::kFloat, D) : Tensor();
        const int32_t flags = (int32_t)ctx->saved_data["flags"].toInt(), dtype = lowp_code(x, "x");
        const Tensor lengths = saved[8].defined() ? restored(saved[8], x, flags & T2FW_SELECT_LENGTHS64 ? at::kLong : at::kInt, B) : Tensor();
        const Tensor ckpt = restored(saved[9], x, at::kByte, (int64_t)t2fw_selective_scan_checkpoint_bytes(B, T, D, N));
        // a result that nothing depends on has no gradient
        const Tensor gy = grads[0].defined() ? near_steps(dense_channels(grads[0])) : at::zeros({1}, x.options()).expand({B, T, D}).contiguous();
        const Tensor gs = grads[1].defined() ? grads[1].contiguous().resolve_neg() : Tensor();
        check_type(gy, type, "the gradient");
        check_sizes(gy, {B, T, D}, "the gradient");
        if (gs.defined()) {
            check_type(gs, at::kFloat, "the state's gradient");
            check_sizes(gs, {B, D, N}, "the state's gradient");
        }
        const auto wide = x.options().dtype(at::kFloat);
        const Tensor dx = at::empty({B, T, D}, x.options()), ddt = at::empty({B, T, D}, x.options()), da = at::empty({D, N}, wide);
        const Tensor db = at::empty({B, T, N}, x.options()), dc = at::empty({B, T, N}, x.options());
        const Tensor dskip = skip.defined() ? at::empty({D}, wide) : Tensor(), dgate = gate.defined() ? at::empty({B, T, D}, x.options()) : Tensor();
        const Tensor dbias = bias.defined() ? at::empty({D}, wide) : Tensor(), ds = ctx->saved_data["state"].toBool() ? at::empty({B, D, N}, wide) : Tensor();
        const size_t bytes = t2fw_selective_scan_backward_workspace_bytes(B, T, D, N);
        Tensor ws;
        if (bytes > 0) ws = bytes_like(x, (int64_t)bytes);
        const bool gated = gate.defined();
        const int64_t strides[12] = {x.stride(0), x.stride(1), dt.stride(0), dt.stride(1), b.stride(0), b.stride(1), c.stride(0), c.stride(1),
                                     gated ? gate.stride(0) : 0, gated ? gate.stride(1) : 0, gy.stride(0), gy.stride(1)};
        done(t2fw_selective_scan_backward(gy.data_ptr(), (const float *)data(gs), x.data_ptr(), dt.data_ptr(), (const float *)a.data_ptr(), b.data_ptr(),
                                          c.data_ptr(), (const float *)data(skip), data(gate), (const float *)data(bias), data(lengths),
                                          ckpt.numel() > 0 ? ckpt.data_ptr() : nullptr, dx.data_ptr(), ddt.data_ptr(), (float *)da.data_ptr(),
                                          db.data_ptr(), dc.data_ptr(), (float *)data(dskip), data(dgate), (float *)data(dbias), (float *)data(ds), B, T, D,
                                          N, strides, dtype, flags, data(ws), bytes, as_address(ctx->saved_data["stream"])));
        return {dx, ddt, da, db, dc, ds, dskip, dgate, dbias, Tensor(), Tensor(), Tensor()};
    }
};

// Tensors of one call, of whole sequences (`axes` 3) or of a token (2)
void check_select(const SelectInputs &i, int64_t axes) {
    const char *const shape = axes == 3 ? "[B, T, D]" : "[B, D]";
    check_on(i.x, i.x, "x");
    TORCH_CHECK(i.x.dim() == axes && i.x.size(-1) >= 1, "t2fw: expected x ", shape, " with at least one channel, it is ", i.x.sizes());
    lowp_code(i.x, "x");
    check_rows(i.x, i.x, "x");
    const auto like_x = [&](const Tensor &t, const char *name) {
        check_on(t, i.x, name);
        check_sizes(t, i.x.sizes(), name);
        check_rows(t, i.x, name);
        check_type(t, i.x.scalar_type(), name);
    };
    like_x(i.dt, "dt");
    if (i.gate.defined()) like_x(i.gate, "gate");
    const int64_t B = i.x.size(0), D = i.x.size(-1);
    check_contiguous(i.a, i.x, "a");
    check_type(i.a, at::kFloat, "a");
    TORCH_CHECK(i.a.dim() == 2 && i.a.size(0) == D && i.a.size(1) >= 1 && i.a.size(1) <= 64, "t2fw: expected a [D, N] of ", D, " channels and 1 to 64 states, it is ", i.a.sizes());
    const int64_t N = i.a.size(1);
    std::vector<int64_t> per_step(i.x.sizes().begin(), i.x.sizes().end());
    per_step.back() = N;
    const Tensor *const rows[2] = {&i.b, &i.c};
    const char *const names[2] = {"b", "c"};
    for (int k = 0; k < 2; ++k) {
        check_on(*rows[k], i.x, names[k]);
        check_sizes(*rows[k], per_step, names[k]);
        check_rows(*rows[k], i.x, names[k]);
        check_type(*rows[k], i.x.scalar_type(), names[k]);
    }
    const auto per_channel = [&](const Tensor &t, at::IntArrayRef sizes, const char *name) {
        if (!t.defined()) return;
        check_contiguous(t, i.x, name);
        check_sizes(t, sizes, name);
        check_type(t, at::kFloat, name);
    };
    per_channel(i.state, {B, D, N}, "state");
    per_channel(i.skip, {D}, "skip");
    per_channel(i.dt_bias, {D}, "dt_bias");
}

// selective_scan(x, dt, a, b, c, state, skip, gate, dt_bias, lengths (five: or None), softplus, stream) -> (y, last state)
PyObject *selective_scan(PyObject *, PyObject *const *p, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 12);
    const SelectInputs i{tensor(p[0]), tensor(p[1]), tensor(p[2]), tensor(p[3]), tensor(p[4]), optional_tensor(p[5]), optional_tensor(p[6]),
                         optional_tensor(p[7]), optional_tensor(p[8]), optional_tensor(p[9])};
    check_select(i, 3);
    check_lengths(i.lengths, i.x);
    no_tangents({i.x, i.dt, i.a, i.b, i.c, i.state, i.skip, i.gate, i.dt_bias}, "selective_scan");
    const int64_t flags = (truth(p[10]) ? T2FW_SELECT_SOFTPLUS : 0) |
                          (i.lengths.defined() && i.lengths.scalar_type() == at::kLong ? T2FW_SELECT_LENGTHS64 : 0);
    void *const stream = address(p[11]);
    const c10::DeviceGuard guard(i.x.device());
    pybind11::gil_scoped_release release;
    if (!wants_grad({i.x, i.dt, i.a, i.b, i.c, i.state, i.skip, i.gate, i.dt_bias})) {
        const SelectResult r = select_forward(i, (int32_t)flags, false, stream);
        pybind11::gil_scoped_acquire acquire;
        return wrapped({r.y, r.last});
    }
    const variable_list r = SelectiveScan::apply(i.x, i.dt, i.a, i.b, i.c, maybe(i.state), maybe(i.skip), maybe(i.gate), maybe(i.dt_bias), maybe(i.lengths),
                                                 flags, as_integer(stream));
    pybind11::gil_scoped_acquire acquire;
    return wrapped({r[0], r[1]});
    END_HANDLE_TH_ERRORS
}

// selective_scan_step(x, dt, a, b, c, state, skip, gate, dt_bias (three: or None), softplus, out or None, inplace, stream) -> (y, state)
PyObject *selective_scan_step(PyObject *, PyObject *const *p, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 13);
    const SelectInputs i{tensor(p[0]), tensor(p[1]), tensor(p[2]), tensor(p[3]), tensor(p[4]), tensor(p[5]), optional_tensor(p[6]), optional_tensor(p[7]),
                         optional_tensor(p[8]), Tensor()};
    Tensor out = optional_tensor(p[10]);
    check_select(i, 2);
    no_tangents({i.x, i.dt, i.a, i.b, i.c, i.state, i.skip, i.gate, i.dt_bias, out}, "selective_scan_step");
    TORCH_CHECK(!wants_grad({i.x, i.dt, i.a, i.b, i.c, i.state, i.skip, i.gate, i.dt_bias, out}),
                "t2fw: selective_scan_step has no gradients: call selective_scan, or this under torch.no_grad()");
    const bool inplace = truth(p[11]);
    if (inplace) check_apart(i.state, {i.x, i.dt, i.a, i.b, i.c, i.skip, i.gate, i.dt_bias, out}, "state");
    if (out.defined()) {
        check_contiguous(out, i.x, "out");
        check_sizes(out, i.x.sizes(), "out");
        check_type(out, i.x.scalar_type(), "out");
        check_apart(out, {i.x, i.dt, i.a, i.b, i.c, i.state, i.skip, i.gate, i.dt_bias}, "out");
    }
    const c10::DeviceGuard guard(i.x.device());
    if (!out.defined()) out = at::empty(i.x.sizes(), i.x.options());
    const Tensor next = inplace ? i.state : at::empty(i.state.sizes(), i.state.options());
    const int32_t flags = truth(p[9]) ? T2FW_SELECT_SOFTPLUS : 0;
    void *const stream = address(p[12]);
    const int64_t strides[5] = {i.x.stride(0), i.dt.stride(0), i.b.stride(0), i.c.stride(0), i.gate.defined() ? i.gate.stride(0) : 0};
    done(unlocked([&] {
        return t2fw_selective_scan_step(i.x.data_ptr(), i.dt.data_ptr(), (const float *)i.a.data_ptr(), i.b.data_ptr(), i.c.data_ptr(),
                                        (const float *)data(i.skip), data(i.gate), (const float *)data(i.dt_bias), (const float *)i.state.data_ptr(),
                                        out.data_ptr(), (float *)next.data_ptr(), i.x.size(0), i.x.size(1), i.a.size(1), strides, dtype_code(i.x, "x"),
                                        flags, stream);
    }));
    // written behind torch's back
    if (inplace) bump(i.state);
    if (p[10] != Py_None) bump(out);
    return wrapped({out, next});
    END_HANDLE_TH_ERRORS
}

// ---- beam search --------------------------------------------------------------------------------------------------
// beam_select(logits, scores, count or None, finished or None, pad, stream) -> (scores, beams, tokens)
PyObject *beam_select(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 6);
    const Tensor logits = tensor(a[0]), scores = tensor(a[1]), finished = optional_tensor(a[3]);
    check_contiguous(logits, logits, "logits");
    no_tangents({logits, scores}, "beam_select");
    TORCH_CHECK(logits.dim() == 3, "t2fw: expected logits [B, beams, V], they are ", logits.sizes());
    const int32_t dtype = lowp_code(logits, "logits");
    const int64_t B = logits.size(0), K = logits.size(1), V = logits.size(2);
    check_contiguous(scores, logits, "scores");
    check_sizes(scores, {B, K}, "scores");
    check_type(scores, at::kFloat, "scores");
    if (finished.defined()) {
        check_contiguous(finished, logits, "finished");
        check_sizes(finished, {B, K}, "finished");
        check_type(finished, at::kBool, "finished");
    }
    TORCH_CHECK(!wants_grad({logits, scores}), "t2fw: beam_select has no gradients: call it under torch.no_grad()");
    const int64_t count = a[2] == Py_None ? K : integer(a[2]), pad = integer(a[4]);
    void *const stream = address(a[5]);
    TORCH_CHECK(count >= 1 && count <= 128 && count <= K * V, "t2fw: ", count, " candidates of ", K, " x ", V, ": 1 to 128, and no more than there are");
    TORCH_CHECK(K >= 1 && K <= 256 && V >= 1, "t2fw: 1 to 256 beams and at least one logit each, logits are ", logits.sizes());
    const c10::DeviceGuard guard(logits.device());
    const Tensor best = at::empty({B, count}, scores.options()), beams = at::empty({B, count}, scores.options().dtype(at::kLong));
    const Tensor tokens = at::empty({B, count}, beams.options());
    const size_t bytes = t2fw_beam_select_workspace_bytes(B, K, V, count, dtype);
    Tensor ws;
    if (bytes > 0) ws = bytes_like(logits, (int64_t)bytes);
    done(unlocked([&] {
        return t2fw_beam_select(logits.data_ptr(), (const float *)scores.data_ptr(), data(finished), (float *)best.data_ptr(), (int64_t *)beams.data_ptr(),
                                (int64_t *)tokens.data_ptr(), B, K, V, count, pad, dtype, data(ws), bytes, stream);
    }));
    return wrapped({best, beams, tokens});
    END_HANDLE_TH_ERRORS
}

// reorder_beams(sequence of tensors, beams, sequence of results or None for in place, stream)
PyObject *reorder_beams(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 4);
    const pybind11::object arrays = pybind11::reinterpret_steal<pybind11::object>(PySequence_Fast(a[0], "t2fw: expected a sequence of tensors"));
    if (!arrays) throw python_error();
    const Tensor beams = tensor(a[1]);
    const bool inplace = a[2] == Py_None;
    const Py_ssize_t count = PySequence_Fast_GET_SIZE(arrays.ptr());
    pybind11::object outs;
    if (!inplace) {
        outs = pybind11::reinterpret_steal<pybind11::object>(PySequence_Fast(a[2], "t2fw: expected a sequence of tensors"));
        if (!outs) throw python_error();
        TORCH_CHECK(PySequence_Fast_GET_SIZE(outs.ptr()) == count, "t2fw: ", count, " tensors and ", PySequence_Fast_GET_SIZE(outs.ptr()), " results");
    }
    check_contiguous(beams, beams, "beams");
    check_type(beams, at::kLong, "beams");
    TORCH_CHECK(beams.dim() == 2 && beams.size(1) >= 1 && beams.size(1) <= 64, "t2fw: expected beams [B, K] with 1 to 64 beams, they are ", beams.sizes());
    const int64_t B = beams.size(0), K = beams.size(1);
    std::vector<t2fw_reorder_desc> d((size_t)count);
    struct Range {
        uintptr_t begin, end;
        bool operator<(const Range &o) const { return begin < o.begin; }
    };
    std::vector<Range> written, read;
    const auto range = [](const Tensor &t) {
        const auto p = reinterpret_cast<uintptr_t>(t.data_ptr());
        return Range{p, p + (uintptr_t)t.nbytes()};
    };
    if (beams.numel() > 0) read.push_back(range(beams));
    for (Py_ssize_t i = 0; i < count; ++i) {
        const Tensor &t = tensor(PySequence_Fast_GET_ITEM(arrays.ptr(), i));
        check_contiguous(t, beams, "every tensor");
        TORCH_CHECK(!t.is_conj(), "every tensor is as it lies in memory: call resolve_conj()");
        no_tangents({t}, "reorder_beams");
        TORCH_CHECK(!wants_grad({t}), "t2fw: reorder_beams has no gradients: call it under torch.no_grad()");
        TORCH_CHECK(t.dim() >= 1 && (B == 0 ? t.size(0) == 0 : t.size(0) % (B * K) == 0), "t2fw: a tensor of ", t.sizes(), " for ", B, " x ", K, " beams");
        const Tensor &o = inplace ? t : tensor(PySequence_Fast_GET_ITEM(outs.ptr(), i));
        if (!inplace) {
            check_contiguous(o, beams, "every result");
            TORCH_CHECK(!o.is_conj(), "every result is as it lies in memory: call resolve_conj()");
            no_tangents({o}, "reorder_beams");
            TORCH_CHECK(!wants_grad({o}), "t2fw: reorder_beams has no gradients: call it under torch.no_grad()");
            check_sizes(o, t.sizes(), "a result");
            check_type(o, t.scalar_type(), "a result");
        }
        d[i].src = t.data_ptr();
        d[i].dst = o.data_ptr();
        d[i].row_bytes = B == 0 ? 0 : (int64_t)t.nbytes() / (B * K);
        if (t.nbytes() == 0) continue;
        written.push_back(range(o));
        if (!inplace) read.push_back(range(t));
    }
    // Many workgroups write the results at once: none may share memory with another, nor with what is read
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); ++i) TORCH_CHECK(written[i - 1].end <= written[i].begin, "t2fw: two results of reorder_beams share memory");
    for (const Range &r : read) {
        const auto next = std::lower_bound(written.begin(), written.end(), Range{r.end, r.end});
        TORCH_CHECK(next == written.begin() || (next - 1)->end <= r.begin, "t2fw: a result of reorder_beams shares memory with what it is made from");
    }
    void *const stream = address(a[3]);
    const c10::DeviceGuard guard(beams.device());
    done(unlocked([&] { return t2fw_beam_reorder(d.data(), count, (const int64_t *)beams.data_ptr(), B, K, stream); }));
    for (Py_ssize_t i = 0; i < count; ++i) bump(tensor(PySequence_Fast_GET_ITEM(inplace ? arrays.ptr() : outs.ptr(), i)));
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

}  // namespace

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef layer_methods[] = {METHOD(short_conv), METHOD(short_conv_step), METHOD(selective_scan), METHOD(selective_scan_step), METHOD(beam_select), METHOD(reorder_beams), {nullptr, nullptr, 0, nullptr}};

}  // namespace t2fw_host
