// Checks of arguments that the host fast paths (fast_cache.cpp, fast_layer.cpp) share.
#pragma once
#include <torch/extension.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cstdint>

namespace {

const at::Tensor* tensor(py::handle h) { return THPVariable_Check(h.ptr()) ? &THPVariable_Unpack(h.ptr()) : nullptr; }

// An int of exactly that type in [low, high].
bool integer(py::handle h, int64_t low, int64_t high, int64_t& value) {
    if (!PyLong_CheckExact(h.ptr())) return false;
    int overflow = 0;
    value = PyLong_AsLongLongAndOverflow(h.ptr(), &overflow);
    return overflow == 0 && value >= low && value <= high;
}

bool flag(py::handle h, bool& value) {
    if (!PyBool_Check(h.ptr())) return false;
    value = h.ptr() == Py_True;
    return true;
}

bool vector(const at::Tensor* t, at::ScalarType type, c10::Device dev, int64_t size) {
    return t && t->dim() == 1 && (size < 0 || t->size(0) == size) && t->scalar_type() == type && t->device() == dev &&
           t->is_contiguous();
}

bool aligned(const void* p, unsigned to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Autograd is told of a tensor that a call writes in place.
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Whether it carries a forward-mode derivative, or is one of a function transform's stand-ins (they hold no memory).
bool differentiated(const at::Tensor& t) { return t._fw_grad(0).defined() || !t.has_storage(); }

bool dims(const at::Tensor& t, std::initializer_list<int64_t> want) {
    return t.sizes() == at::IntArrayRef(want.begin(), want.size());
}

}  // namespace
