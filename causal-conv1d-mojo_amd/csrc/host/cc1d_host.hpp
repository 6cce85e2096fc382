// cc1d_host.hpp -- what the native host path's units share: when a call is the
// ordinary case, and how tensors become the C ABI's pointers and strides.
#pragma once

#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/record_function.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <optional>

#include "cc1d.h"

namespace cc1d_host {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::variable_list;

// No dispatch or torch-function mode, transform or tracer in force on this
// thread: what the dispatcher would send straight to the backend.
inline bool plain_thread() {
    if (c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled()) return false;
    const auto tls = c10::impl::tls_local_dispatch_key_set();
    return (tls.included_ - c10::default_included_set - c10::autocast_dispatch_keyset).empty();
}

// A strided GPU tensor without a subclass, lazy bit, wrapper or tangent.
inline bool plain(const Tensor& t) {
    static const auto allowed = c10::DispatchKeySet(c10::DispatchKey::CUDA) |
                                c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) |
                                c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView) |
                                c10::DispatchKeySet(c10::DispatchKey::AutocastCUDA);
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided &&
           (t.key_set().raw_repr() & ~allowed.raw_repr()) == 0 && !t._fw_grad(0).defined();
}

inline bool plain(PyObject* o) { return THPVariable_CheckExact(o) && plain(THPVariable_Unpack(o)); }
inline bool plain_or_none(PyObject* o) { return o == Py_None || plain(o); }
inline Tensor tensor_or_none(PyObject* o) { return o == Py_None ? Tensor() : THPVariable_Unpack(o); }

inline int dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
    case at::kHalf: return CC1D_DTYPE_FP16;
    case at::kBFloat16: return CC1D_DTYPE_BF16;
    case at::kFloat: return CC1D_DTYPE_FP32;
    default: return -1;
    }
}

// 0: no activation, 1: SiLU, -1: not one of the accepted values
inline int activation_code(PyObject* o) {
    if (o == Py_None) return 0;
    if (!PyUnicode_CheckExact(o)) return -1;
    return PyUnicode_CompareWithASCIIString(o, "silu") == 0 || PyUnicode_CompareWithASCIIString(o, "swish") == 0 ? 1 : -1;
}

inline bool same(const Tensor& t, const Tensor& like) {
    return t.scalar_type() == like.scalar_type() && t.device() == like.device();
}
inline bool shaped(const Tensor& t, at::IntArrayRef s) { return t.sizes() == s; }

inline const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
inline void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

template <int N> void strides(int64_t (&dst)[N], const Tensor& t) {
    for (int i = 0; i < N; ++i) dst[i] = t.defined() ? t.stride(i) : 0;
}

void check(int status);  // throws the library's message
inline void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// dout in x's layout: a copy only where the time strides differ (or any, in a layout without unit time stride)
inline Tensor match_layout(const Tensor& t, const Tensor& like) {
    if (t.strides() == like.strides()) return t;
    if (like.stride(-1) == 1) return t.stride(-1) == 1 ? t : t.contiguous();
    return at::empty_like(like).copy_(t);
}

inline PyObject* not_implemented() { Py_RETURN_NOTIMPLEMENTED; }

extern PyMethodDef ssm_methods[];  // cc1d_host_ssm.cpp

#define CC1D_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL

}  // namespace cc1d_host
