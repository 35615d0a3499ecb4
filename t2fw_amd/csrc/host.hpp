// What the sources of the extension module share (host.cpp, host_ops.cpp): arguments in, results out.
#pragma once
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>

#include <vector>

#include "../../include/t2fw_hip.h"

namespace t2fw_host {

using at::Tensor;

inline const Tensor &tensor(PyObject *o) {
    TORCH_CHECK(THPVariable_Check(o), "t2fw: expected a tensor");
    return THPVariable_Unpack(o);
}
inline int64_t integer(PyObject *o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
inline void *address(PyObject *o) {
    void *v = PyLong_AsVoidPtr(o);
    if (v == nullptr && PyErr_Occurred()) throw python_error();
    return v;
}
inline void arguments(Py_ssize_t n, Py_ssize_t want) { TORCH_CHECK(n == want, "t2fw: ", n, " arguments, expected ", want); }
inline void done(int rc) {
    TORCH_CHECK_WITH(Error, rc == 0, "t2fw error ", rc, ": ", t2fw_last_error());
}
inline PyObject *wrapped(std::initializer_list<Tensor> ts) {
    PyObject *t = PyTuple_New((Py_ssize_t)ts.size());
    if (t == nullptr) throw python_error();
    Py_ssize_t i = 0;
    for (const Tensor &v : ts) {
        PyObject *o = v.defined() ? THPVariable_Wrap(v) : Py_NewRef(Py_None);
        if (o == nullptr) {
            Py_DECREF(t);
            throw python_error();
        }
        PyTuple_SET_ITEM(t, i++, o);
    }
    return t;
}
// The launches run without the interpreter's lock: they wait where the device's queue is full.
template <typename F> int unlocked(F &&launch) {
    pybind11::gil_scoped_release release;
    return launch();
}
inline Tensor bytes_like(const Tensor &t, int64_t n) { return at::empty({n}, t.options().dtype(at::kByte)); }

// the operators around the recurrences (host_ops.cpp)
extern PyMethodDef operator_methods[];
// the selective state space layer and beam search (host_layers.cpp)
extern PyMethodDef layer_methods[];

}  // namespace t2fw_host
