// ops_torch.h -- what the Python module's operators (ops_torch.cpp,
// ops_train_torch.cpp) share: arguments, checks of tensors, errors.
#pragma once

#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <stdexcept>
#include <string>
#include <vector>

#include "ssla_hip.h"

namespace ssla_torch {

extern PyObject* g_error;        // ssla_hip.lib.SslaHipError

[[noreturn]] inline void refuse(const char* fn, const std::string& what) {
    throw std::invalid_argument(std::string(fn) + ": " + what);
}

struct LibraryError : std::runtime_error {
    using std::runtime_error::runtime_error;
};

inline void check(int rc, const char* entry) {
    if (rc < 0)
        throw LibraryError(std::string(entry) + " failed (" + std::to_string(rc) + "): " + ssla_hip_last_error());
}

// The arguments of a call, which ops.py passes by position.
struct Args {
    const char* fn;
    PyObject* const* v;

    const at::Tensor& tensor(int i, const char* name) const {
        if (!THPVariable_Check(v[i])) refuse(fn, std::string(name) + " must be a tensor");
        return THPVariable_Unpack(v[i]);
    }
    const at::Tensor* optional(int i, const char* name) const {
        return v[i] == Py_None ? nullptr : &tensor(i, name);
    }
    long long integer(int i, const char* name) const {
        const long long x = PyLong_AsLongLong(v[i]);
        if (x == -1 && PyErr_Occurred()) {
            PyErr_Clear();
            refuse(fn, std::string(name) + " must be an integer");
        }
        return x;
    }
    int count(int i, const char* name) const {
        const long long x = integer(i, name);
        if (x < 0 || x > 0x7fffffff) refuse(fn, std::string(name) + " must be 0 .. 2^31 - 1");
        return (int)x;
    }
    double real(int i, const char* name) const {
        const double x = PyFloat_AsDouble(v[i]);
        if (x == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            refuse(fn, std::string(name) + " must be a number");
        }
        return x;
    }
};

inline int dtype_of(const char* fn, const char* name, const at::Tensor& t) {
    if (!t.is_cuda()) refuse(fn, std::string(name) + " must be on a GPU");
    switch (t.scalar_type()) {
        case at::kFloat: return SSLA_F32;
        case at::kBFloat16: return SSLA_BF16;
        case at::kHalf: return SSLA_F16;
        default: refuse(fn, std::string(name) + " must be float32, bfloat16 or float16");
    }
}

// Type and device of a tensor of the call; there are no gradients, forward ones
// nowhere and backward ones only where `backward` says so.
inline void alike(const char* fn, const char* name, const at::Tensor& t, at::ScalarType type, at::Device dev,
                  bool backward = false) {
    if (t.scalar_type() != type || t.device() != dev || t.layout() != at::kStrided)
        refuse(fn, std::string(name) + " must be a " + c10::toString(type) + " tensor on " + dev.str());
    if (t.is_neg()) refuse(fn, std::string(name) + " is a negated view: call resolve_neg()");
    if (!backward && t.requires_grad() && at::GradMode::is_enabled())
        refuse(fn, std::string(name) + " requires a gradient, which there is none of: call under torch.no_grad()");
    if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
        refuse(fn, std::string(name) + " carries a forward gradient, which there is none of: call with its primal");
}

// A call has written to t: autograd notices, should it have kept t.  Inference
// tensors have no version.
inline void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

inline void shaped(const char* fn, const char* name, const at::Tensor& t, at::IntArrayRef shape) {
    if (t.sizes() != shape)
        refuse(fn, std::string(name) + " must have the shape " + c10::str(shape) + ", not " + c10::str(t.sizes()));
}

inline const int* index(const char* fn, const char* name, const at::Tensor& t, at::Device dev, int64_t n) {
    alike(fn, name, t, at::kInt, dev);
    if (t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1))
        refuse(fn, std::string(name) + " must be " + std::to_string(n) + " contiguous int32 values");
    return t.const_data_ptr<int>();
}

inline void* stream_of(at::Device dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }

inline at::Tensor workspace(at::Device dev, size_t bytes) {
    return bytes ? at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(dev)) : at::Tensor();
}

// C++ exceptions end here, as Python ones.
inline PyObject* to_python(const at::Tensor& t) { return THPVariable_Wrap(t); }
inline PyObject* to_python(const std::vector<at::Tensor>& ts) {
    PyObject* tuple = PyTuple_New((Py_ssize_t)ts.size());
    if (!tuple) return nullptr;
    for (size_t i = 0; i < ts.size(); ++i) PyTuple_SET_ITEM(tuple, (Py_ssize_t)i, THPVariable_Wrap(ts[i]));
    return tuple;
}
template <auto F>
PyObject* call(const char* fn, int want, PyObject* const* v, Py_ssize_t n) {
    try {
        if (n != want) refuse(fn, "wrong number of arguments");
        return to_python(F(Args{fn, v}));
    } catch (const std::invalid_argument& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const LibraryError& e) {
        PyErr_SetString(g_error, e.what());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

// ops_train_torch.cpp
PyObject* py_linear_recurrence(PyObject*, PyObject* const* v, Py_ssize_t n);
PyObject* py_linear_recurrence_step(PyObject*, PyObject* const* v, Py_ssize_t n);
PyObject* py_layer_norm(PyObject*, PyObject* const* v, Py_ssize_t n);

}  // namespace ssla_torch
