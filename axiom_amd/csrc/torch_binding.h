// What the torch bindings share: argument checks, outputs and workspaces, errors.
//
// Errors: bad arguments raise ValueError, tensors that are not on the GPU and HIP
// failures RuntimeError, as in the package's other calls.
#pragma once

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/python.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <optional>
#include <sstream>
#include <string>
#include <tuple>

#include "tree_mi355x.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

template <class... A>
[[noreturn]] void refuse(const char* what, const A&... parts) {
  std::ostringstream s;
  s << what << ": ";
  (s << ... << parts);
  throw py::value_error(s.str());
}

void checked(int rc, const char* what) {
  if (rc == KDA_OK) return;
  std::ostringstream s;
  s << what << ": " << kda_last_error() << " (status " << rc << ")";
  if (rc == KDA_ERR_HIP) throw std::runtime_error(s.str());
  throw py::value_error(s.str());
}

int code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return KDA_DTYPE_F32;
    case at::kBFloat16: return KDA_DTYPE_BF16;
    case at::kHalf: return KDA_DTYPE_F16;
    default: return -1;
  }
}

void contiguous(const char* name, const Tensor& t) {
  if (!t.is_contiguous()) throw py::value_error(std::string(name) + " must be contiguous");
}

void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

// the one GPU all tensors are on
template <class... T>
at::Device one_gpu(const char* what, const Tensor& first, const T&... rest) {
  const at::Device d = first.device();
  auto same = [&](const auto& t) {
    if constexpr (std::is_same_v<std::decay_t<decltype(t)>, OptTensor>) return !t || t->device() == d;
    else return t.device() == d;
  };
  if (!(same(rest) && ...)) refuse(what, "all tensors must be on one device");
  if (!d.is_cuda())
    throw std::runtime_error(std::string(what) + ": the kernels run only on the GPU (HIP, gfx950); got tensors on " + d.str() +
                             ". There is no CPU fallback.");
  return d;
}

// A call launches on the device that is current, and the default stream's handle
// names none: every entry point makes the tensors' device current while it runs.
hipStream_t stream_of(at::Device d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }

Tensor output(const char* what, const char* name, const OptTensor& t, at::IntArrayRef shape, at::ScalarType dt, at::Device d) {
  if (!t) return at::empty(shape, at::TensorOptions().dtype(dt).device(d));
  if (t->sizes() != shape || t->scalar_type() != dt || t->device() != d)
    refuse(what, name, " must be ", dt, " ", shape, " on ", d.str());
  contiguous(name, *t);
  return *t;
}

// a caller's workspace of at least `bytes`, or a new one
Tensor work(const OptTensor& t, size_t bytes, at::Device d) {
  if (bytes == 0) return Tensor();
  if (t && t->nbytes() >= bytes && t->device() == d && t->is_contiguous()) return *t;
  return at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(d));
}
void* work_ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// a caller's tensor has been written: autograd notices where it is needed as it was
void written(const OptTensor& t) {
  if (t && !t->is_inference()) torch::autograd::impl::bump_version(*t);
}

}  // namespace
