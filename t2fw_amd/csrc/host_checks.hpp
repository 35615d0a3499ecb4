// What the operators' host sides share (host_ops.cpp, host_layers.cpp): arguments, checks of tensors, what autograd nodes save.
#pragma once
#include "host.hpp"

#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/custom_function.h>

namespace t2fw_host {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline double real(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
inline Tensor optional_tensor(PyObject *o) { return o == Py_None ? Tensor() : tensor(o); }
// A node's arguments that may be missing go to it as optional ones, which torch does not look into where there is none
using Maybe = std::optional<Tensor>;
inline Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : std::nullopt; }
inline Tensor of(const Maybe &t) { return t.has_value() ? *t : Tensor(); }
inline bool truth(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}
inline void *data(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

inline int32_t dtype_code(const Tensor &t, const char *name) {
    switch (t.scalar_type()) {
        case at::kFloat: return T2FW_F32;
        case at::kHalf: return T2FW_F16;
        case at::kBFloat16: return T2FW_BF16;
        case at::kDouble: return T2FW_F64;
        default: TORCH_CHECK(false, "t2fw: unsupported dtype ", t.scalar_type(), " of ", name);
    }
}
inline at::ScalarType accumulators_type(const Tensor &t) { return t.scalar_type() == at::kDouble ? at::kDouble : at::kFloat; }

inline void check_on(const Tensor &t, const Tensor &like, const char *name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.layout() == at::kStrided, name, " must be a dense tensor");
    // (its memory holds the other sign)
    TORCH_CHECK(!t.is_neg(), name, " is a negated view: call resolve_neg()");
    TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", not on ", like.device());
}
inline void check_contiguous(const Tensor &t, const Tensor &like, const char *name) {
    check_on(t, like, name);
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}
inline void check_sizes(const Tensor &t, at::IntArrayRef sizes, const char *name) {
    TORCH_CHECK(t.sizes() == sizes, "t2fw: ", name, " is ", t.sizes(), ", expected ", sizes);
}
inline void check_type(const Tensor &t, at::ScalarType type, const char *name) {
    TORCH_CHECK(t.scalar_type() == type, "t2fw: ", name, " is ", t.scalar_type(), ", expected ", type);
}
inline bool wants_grad(std::initializer_list<Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor &t : ts)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}
// Forward-mode derivatives: there are none, and a result without its tangent would pass for one whose tangent is zero
inline void no_tangents(std::initializer_list<Tensor> ts, const char *what) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor &t : ts) TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "t2fw: ", what, " has no forward-mode derivatives");
}
// The gradients are results of kernels that torch knows nothing of
inline void once(const char *what) { TORCH_CHECK(!at::GradMode::is_enabled(), "t2fw: ", what, " can be differentiated once only (create_graph)"); }

// What a node has saved, dense and of the type and number of elements that its kernels take: hooks on saved tensors may bring it back in
// another order of memory
inline Tensor restored(const Tensor &t, const Tensor &like, at::ScalarType type, int64_t numel) {
    check_on(t, like, "a saved tensor");
    check_type(t, type, "a saved tensor");
    TORCH_CHECK(t.numel() == numel, "t2fw: a saved tensor has ", t.numel(), " elements, expected ", numel);
    return t.contiguous();
}

// An address in a node's saved data
inline int64_t as_integer(void *p) { return (int64_t)(uintptr_t)p; }
inline void *as_address(const c10::IValue &v) { return reinterpret_cast<void *>((uintptr_t)v.toInt()); }

// (a gradient may be a view that torch negates when it reads it)
// x, f [B, T, D] with dense channels; anything else is copied (gradients that are expanded scalars, say)
inline Tensor dense_channels(const Tensor &t) {
    return t.size(2) <= 1 || t.stride(2) == 1 ? t.resolve_neg() : t.contiguous().resolve_neg();
}

inline void check_lengths(const Tensor &lengths, const Tensor &x) {
    if (!lengths.defined()) return;
    check_contiguous(lengths, x, "lengths");
    TORCH_CHECK(lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong, "t2fw: lengths are ", lengths.scalar_type(),
                ", expected int32 or int64");
    check_sizes(lengths, {x.size(0)}, "lengths");
}

}  // namespace t2fw_host
