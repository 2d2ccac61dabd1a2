// Group norm and dropout as differentiable calls.  The nodes are C++: a
// Python function's backward would take the interpreter's lock from the
// engine's thread, some 20 us that small activations feel.

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cmath>

#include "group_norm.h"

using at::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

std::vector<Tensor> group_norm_forward(const Tensor& x, int64_t groups,
                                       const Tensor& weight,
                                       const Tensor& bias, double eps,
                                       int64_t act, double p,
                                       const Tensor& rng, int64_t seed,
                                       int64_t offset, bool keep);
std::vector<Tensor> group_norm_backward(const Tensor& gy, const Tensor& x,
                                        int64_t groups, const Tensor& weight,
                                        const Tensor& bias,
                                        const Tensor& kept, int64_t act,
                                        double p, const Tensor& rng,
                                        int64_t seed, int64_t offset,
                                        bool need_x, bool need_weight,
                                        bool need_bias);
Tensor dropout_forward(const Tensor& x, int64_t act, double p,
                       const Tensor& rng, int64_t seed, int64_t offset);
Tensor dropout_backward(const Tensor& gy, const Tensor& x, int64_t act,
                        double p, const Tensor& rng, int64_t seed,
                        int64_t offset);

namespace {

// Gradients of gradients are not provided: where a graph of the gradients is
// being built, they carry a node that says so when it is reached.
variable_list once(variable_list grads, std::initializer_list<Tensor> from) {
  if (!at::GradMode::is_enabled()) return grads;
  bool any = false;
  for (const Tensor& t : from) any = any || (t.defined() && t.requires_grad());
  if (!any) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "deepof_amd: this gradient cannot be differentiated again",
      (int64_t)grads.size());
  return (*error)(std::move(grads));
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x,
                        const OptTensor& weight, const OptTensor& bias,
                        int64_t groups, double eps, int64_t act, double p,
                        const OptTensor& rng, int64_t seed, int64_t offset) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor r = rng.value_or(Tensor());
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    auto out = group_norm_forward(x, groups, w, b, eps, act, p, r, seed, offset,
                                  true);
    ctx->save_for_backward({x, w, b, out[1], r});
    ctx->saved_data["g"] = groups;
    ctx->saved_data["a"] = act;
    ctx->saved_data["p"] = p;
    ctx->saved_data["s"] = seed;
    ctx->saved_data["o"] = offset;
    return out[0];
  }

  static variable_list backward(AutogradContext* ctx, variable_list gy) {
    const auto s = ctx->get_saved_variables();
    variable_list g;
    // edges are those of the tensors that were there
    const bool has_w = s[1].defined(), has_b = s[2].defined();
    {
      at::AutoDispatchBelowADInplaceOrView below;
      g = group_norm_backward(
          gy[0].contiguous(at::MemoryFormat::ChannelsLast), s[0],
          ctx->saved_data["g"].toInt(), s[1], s[2], s[3],
          ctx->saved_data["a"].toInt(), ctx->saved_data["p"].toDouble(), s[4],
          ctx->saved_data["s"].toInt(), ctx->saved_data["o"].toInt(),
          ctx->needs_input_grad(0), has_w && ctx->needs_input_grad(1),
          has_b && ctx->needs_input_grad(has_w ? 2 : 1));
    }
    g = once(std::move(g), {gy[0], s[0], s[1], s[2]});
    g.resize(10);
    return g;
  }
};

at::MemoryFormat dense_format(const Tensor& x) {
  return x.dim() == 4 && !x.is_contiguous() &&
                 x.is_contiguous(at::MemoryFormat::ChannelsLast)
             ? at::MemoryFormat::ChannelsLast
             : at::MemoryFormat::Contiguous;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, int64_t act,
                        double p, const OptTensor& rng, int64_t seed,
                        int64_t offset) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor r = rng.value_or(Tensor());
    ctx->save_for_backward({act ? x : Tensor(), r});
    ctx->saved_data["a"] = act;
    ctx->saved_data["p"] = p;
    ctx->saved_data["s"] = seed;
    ctx->saved_data["o"] = offset;
    ctx->saved_data["f"] = (int64_t)dense_format(x);
    return dropout_forward(x, act, p, r, seed, offset);
  }

  static variable_list backward(AutogradContext* ctx, variable_list gy) {
    const auto s = ctx->get_saved_variables();
    const auto format = (at::MemoryFormat)ctx->saved_data["f"].toInt();
    Tensor g;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      g = dropout_backward(gy[0].contiguous(format), s[0],
                           ctx->saved_data["a"].toInt(),
                           ctx->saved_data["p"].toDouble(), s[1],
                           ctx->saved_data["s"].toInt(),
                           ctx->saved_data["o"].toInt());
    }
    variable_list out = once({g}, {gy[0], s[0]});
    out.resize(6);
    return out;
  }
};

void check_values(const Tensor& x, const char* name) {
  TORCH_CHECK_TYPE(x.scalar_type() == at::kFloat ||
                       x.scalar_type() == at::kHalf ||
                       x.scalar_type() == at::kBFloat16,
                   name, ": float32, float16 or bfloat16 expected, got ",
                   x.scalar_type());
}

// A tangent would be lost: kernels read a dual tensor's value alone.
void no_tangent(const Tensor& t, const char* name) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), name,
                              ": no forward-mode derivatives on the GPU");
}

// A tracer would record the result's allocation and not the kernels.
void not_traced(const char* name) {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  TORCH_CHECK_NOT_IMPLEMENTED(
      !torch::jit::tracer::isTracing() &&
          !TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY),
      name, ": cannot be traced on the GPU");
}

// A parameter as the kernels read it: fp32, contiguous.  A cast is part of the
// graph.
OptTensor param(const OptTensor& t, const Tensor& x, const char* name) {
  if (!t.has_value() || !t->defined()) return c10::nullopt;
  check_values(*t, name);
  no_tangent(*t, name);
  TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == x.size(1) &&
                        t->device() == x.device(),
                    name, " must be [", x.size(1), "] on ", x.device(),
                    ", got ", t->sizes(), " on ", t->device());
  if (t->scalar_type() == at::kFloat && t->is_contiguous()) return t;
  return t->to(at::kFloat).contiguous();
}

}  // namespace

Tensor group_norm(const Tensor& input, int64_t groups, const OptTensor& weight,
                  const OptTensor& bias, double eps, int64_t act, double p,
                  const OptTensor& rng, int64_t seed, int64_t offset) {
  not_traced("group_norm");
  check_values(input, "group_norm");
  no_tangent(input, "group_norm");
  TORCH_CHECK_VALUE(input.dim() == 4, "group_norm: [B, C, H, W] expected, got ",
                    input.sizes());
  const int64_t c = input.size(1);
  TORCH_CHECK_VALUE(groups >= 1 && groups <= MAX_GROUPS && c > 0 &&
                        c % groups == 0,
                    "group_norm: ", c, " channels in ", groups,
                    " groups (at most ", MAX_GROUPS, ")");
  TORCH_CHECK_VALUE((float)eps > 0.0f && std::isfinite(eps),
                    "group_norm: eps must be positive, got ", eps);
  const OptTensor w = param(weight, input, "group_norm: weight");
  const OptTensor b = param(bias, input, "group_norm: bias");
  const Tensor x = input.contiguous(at::MemoryFormat::ChannelsLast);
  const auto wanted = [](const OptTensor& t) {
    return t.has_value() && t->requires_grad();
  };
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || wanted(w) || wanted(b)))
    return GroupNorm::apply(x, w, b, groups, eps, act, p, rng, seed, offset);
  return group_norm_forward(x, groups, w.value_or(Tensor()),
                            b.value_or(Tensor()), eps, act, p,
                            rng.value_or(Tensor()), seed, offset, false)[0];
}

Tensor dropout(const Tensor& input, int64_t act, double p, const OptTensor& rng,
               int64_t seed, int64_t offset) {
  not_traced("dropout");
  check_values(input, "dropout");
  no_tangent(input, "dropout");
  const Tensor x = input.contiguous(dense_format(input));
  if (at::GradMode::is_enabled() && x.requires_grad())
    return Dropout::apply(x, act, p, rng, seed, offset);
  return dropout_forward(x, act, p, rng.value_or(Tensor()), seed, offset);
}
