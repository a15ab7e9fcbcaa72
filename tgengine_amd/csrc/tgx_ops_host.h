// What the host glue of the model-side operators shares (tgx_ops.cpp, tgx_ops_block.cpp):
// argument checks, streams, workspaces.
#pragma once

#include <torch/extension.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <stdexcept>
#include <string>
#include <vector>

#include "tgx.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

[[noreturn]] inline void bad(const std::string& msg) { throw std::invalid_argument(msg); }

inline void check(int rc, const char* what) {
  if (rc != TGX_OK) throw std::runtime_error(std::string(what) + " failed: " + tgx_last_error());
}

inline void* stream_of(const Tensor& t) {
  return static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

inline int32_t dtype_of(const Tensor& t, const char* what) {
  if (t.scalar_type() == at::kFloat) return TGX_F32;
  if (t.scalar_type() == at::kBFloat16) return TGX_BF16;
  bad(std::string(what) + " must be float32 or bfloat16");
}

inline void on_gpu(const Tensor& t, const char* what) {
  if (!t.is_cuda()) throw std::runtime_error(std::string(what) + " must be on the GPU (libtgx has no CPU path)");
}

inline void same_device(const Tensor& t, const Tensor& like, const char* what) {
  if (t.device() != like.device()) bad(std::string(what) + " must be on the device of the first argument");
}

inline bool keeps_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// forward-mode derivatives would be taken for zeros, and a trace would record the outputs' bare
// memory
inline void reverse_mode_only(const char* what, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined())
      throw std::runtime_error(std::string(what) + " has no forward-mode derivative");
  if (torch::jit::tracer::isTracing()) throw std::runtime_error(std::string(what) + " cannot be traced");
}

// a backward pass that is asked for a graph of its own
inline void only_once(const char* what) {
  if (at::GradMode::is_enabled())
    throw std::runtime_error(std::string(what) + " can be differentiated once only (create_graph is not supported)");
}

inline Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes == 0 ? Tensor() : at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

inline void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// the values in memory: torch may hold them with their signs turned (the imaginary part of a
// conjugate)
inline Tensor stored(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// and one after the other
inline Tensor dense(const Tensor& t) { return stored(t.contiguous()); }

// rows of the last dimension as (rows, row stride): in place where the tensor is contiguous or
// of two dimensions with dense rows, and otherwise a contiguous copy, also where more dimensions
// have rows one even step apart (a half of a projection of (batch, tokens, 2 dim))
inline Tensor as_rows(const Tensor& in, int64_t& rows, int64_t& stride) {
  const Tensor t = stored(in);
  const int64_t dim = t.size(-1);
  rows = dim > 0 ? t.numel() / dim : 0;
  stride = dim;
  if (t.is_contiguous()) return t;
  if (t.dim() == 2 && (t.stride(1) == 1 || dim == 1)) {
    stride = t.stride(0);
    return t;
  }
  return t.contiguous();
}

// the tensor itself where its last dimension is one value after the other
inline Tensor dense_last(const Tensor& t) { return stored(t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous()); }

}  // namespace
