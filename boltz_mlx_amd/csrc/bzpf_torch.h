// What the files of the torch binding (boltz_mlx_amd/_train.so) share: the entry points, their errors, types and checks.
#pragma once

#include <torch/extension.h>

#include <c10/hip/HIPStream.h>

#include <stdexcept>
#include <string>
#include <tuple>

#include "bzpf.h"

namespace bzpf_torch {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef const std::optional<Tensor>& Opt;  // None: an undefined tensor
inline Tensor get(Opt o) { return o.value_or(Tensor()); }

inline int type_code(at::ScalarType t) {
  TORCH_CHECK_TYPE(t == at::kFloat || t == at::kHalf || t == at::kBFloat16, "unsupported dtype ", t);
  return t == at::kFloat ? BZPF_F32 : t == at::kHalf ? BZPF_F16 : BZPF_BF16;
}
inline int type_code(const Tensor& t) { return type_code(t.scalar_type()); }

// The calling thread's device is t's for the scope, and so the current stream one of t's device.
struct OnDevice {
  c10::OptionalDeviceGuard guard;
  void* stream;
  explicit OnDevice(const Tensor& t) : guard(t.device()) {
    stream = c10::hip::getCurrentHIPStream(t.device().index()).stream();
  }
};

// The entry points, in the library that boltz_mlx_amd._lib has loaded: this module links none, so that a process holds one
// copy, whichever it is. Set when the module is imported, before any call.
#define BZPF_ENTRIES(X)                                                                                                \
  X(last_error) X(layernorm) X(layernorm_bwd_ws) X(layernorm_bwd) X(dropout) X(dropout_add_ln) X(dropout_add_ln_bwd) \
  X(rel_bias) X(rel_bias_bwd_ws) X(rel_bias_bwd) X(qk_norm_rope) X(qk_norm_rope_bwd_ws) X(qk_norm_rope_bwd)            \
  X(attention_ws) X(attention) X(attention_bwd_ws) X(attention_bwd)
struct Entries {
#define X(f) decltype(&::bzpf_##f) f;
  BZPF_ENTRIES(X)
#undef X
};
extern Entries lib;

// An entry point's refusal or failure: boltz_mlx_amd._lib.BzpfError in Python, as from every other call of the package.
struct Failure : std::runtime_error {
  using std::runtime_error::runtime_error;
};
inline void check(int rc, const char* name) {
  if (rc != BZPF_OK) throw Failure(c10::str(name, " failed (", rc, "): ", lib.last_error()));
}

// A count as the entry points take it, in 32 bits: one that they do not hold is refused here, as they would see another.
inline void count_fits(const char* name, const char* what, int64_t n) {
  TORCH_CHECK_VALUE(n <= INT32_MAX, name, ": too many ", what, " (", n, ")");
}

template <typename... Ts>
void on_gpu(const char* name, const Ts&... ts) {
  TORCH_CHECK_VALUE((... && (!ts.defined() || ts.is_cuda())), name, ": need ROCm device tensors");
}

inline const float* f32(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
inline float* f32_out(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
inline const void* in(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
inline void* out(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Backward passes are not differentiable: a call that asks for their graph is refused rather than given none.
inline void once(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name, ": gradients of gradients are not provided (create_graph)");
}
inline int64_t type_of(const Tensor& t) { return static_cast<int64_t>(t.defined() ? t.scalar_type() : at::kFloat); }
// A parameter's gradient in its type.
inline Tensor as(const Tensor& g, int64_t type) {
  return g.defined() && type_of(g) != type ? g.to(static_cast<at::ScalarType>(type)) : g;
}
// A parameter as the kernels read it (itself where it is so already: a call's host time counts beside kernels of a few us).
inline Tensor param(const Tensor& w) {
  return !w.defined() || (w.scalar_type() == at::kFloat && w.is_contiguous()) ? w : w.detach().to(at::kFloat).contiguous();
}

// Adds the functions of the sequence attention's training form to the module (bzpf_torch_attn.cpp).
void bind_attention(pybind11::module_& m);

}  // namespace bzpf_torch
