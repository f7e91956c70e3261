// torch_common.h - what the torch operators share (torch_ops.cpp, torch_block_ops.cpp): checks of tensors, tensors as matrices, and
// the parts of autograd that every operator has.
#ifndef GF_TORCH_COMMON_H_
#define GF_TORCH_COMMON_H_

#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "../../include/gaussfield.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

void check_rc(int rc, const char* what) { TORCH_CHECK(rc == GF_OK, what, ": ", gf_last_error(), " (code ", rc, ")"); }

const char* type_name(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    default: return c10::toString(t);
  }
}

int dtype_of(const Tensor& x) {
  return x.scalar_type() == at::kFloat ? GF_DTYPE_F32 : x.scalar_type() == at::kBFloat16 ? GF_DTYPE_BF16 : GF_DTYPE_F16;
}

void check_first(const Tensor& x) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  const auto t = x.scalar_type();
  TORCH_CHECK(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, "x must be float32, bfloat16 or float16 (got ", type_name(t), ")");
}

void check_like(const Tensor& t, const char* name, const Tensor& x) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), name, " must be ", type_name(x.scalar_type()), " like x (got ", type_name(t.scalar_type()), ")");
  TORCH_CHECK(t.device() == x.device(), "all tensors must be on the same device (got ", x.device(), " and ", t.device(), ")");
}

bool present(const MaybeTensor& t) { return t.has_value() && t->defined(); }

// A tensor as a matrix of its last dimension's rows with unit column stride: itself wherever it can be read so.
struct Rows {
  Tensor t;
  int64_t rows, cols, ld;
  explicit Rows(const Tensor& x) : t(x), rows(0), cols(x.size(-1)), ld(cols) {
    if (!t.is_contiguous()) {
      if (t.dim() != 2) t = t.reshape({-1, cols});
      if ((t.stride(1) != 1 && cols > 1) || (t.stride(0) < cols && t.size(0) > 1)) t = t.contiguous();
      if (t.size(0) > 1) ld = t.stride(0);
    }
    rows = cols ? t.numel() / cols : 0;
  }
  const void* data() const { return t.data_ptr(); }
};

void* stream_of(const Tensor& x) { return c10::hip::getCurrentHIPStream(x.device().index()).stream(); }

// Gradients of a first backward that refuse a second one.
variable_list once(variable_list grads, const char* name, bool again) {
  if (!at::GradMode::is_enabled() || !again) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  const auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " is differentiable once only", grads.size());
  return (*error)(std::move(grads));
}

bool wants(const Tensor& t) { return t.requires_grad(); }
bool wants(const MaybeTensor& t) { return present(t) && t->requires_grad(); }

// There is no forward-mode derivative: a tangent must not get lost, whether or not gradients are wanted too.
template <typename... M>
void check_no_tangent(const char* name, const Tensor& x, const M&... others) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  const bool tangent = x._fw_grad(0).defined() || (... || (present(others) && others->_fw_grad(0).defined()));
  TORCH_CHECK_NOT_IMPLEMENTED(!tangent, name, " has no forward-mode derivative");
}

MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }

}  // namespace

#endif  // GF_TORCH_COMMON_H_
