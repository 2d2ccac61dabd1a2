// Group norm: checks, allocations and the choice of type.  The mathematics and
// the kernels are in group_norm.hip.h.

#include "group_norm.h"

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>

#include <algorithm>

namespace {

GroupNormShape shape_of(const at::Tensor& x, int64_t groups) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 4 &&
                  x.is_contiguous(at::MemoryFormat::ChannelsLast),
              "group_norm: x must be a 4-D channels-last GPU tensor");
  TORCH_CHECK(groups >= 1 && groups <= MAX_GROUPS && x.size(1) >= 1 &&
                  x.size(1) % groups == 0,
              "group_norm: the channels must divide into 1 to ", MAX_GROUPS,
              " groups");
  TORCH_CHECK(x.size(0) < (1ll << 24) && x.size(1) < (1ll << 20) &&
                  x.size(2) * x.size(3) < (1ll << 30),
              "group_norm: tensor too large");
  GroupNormShape s;
  s.hw = x.size(2) * x.size(3);
  s.b = (int)x.size(0);
  s.c = (int)x.size(1);
  s.g = (int)groups;
  s.cg = s.c / s.g;
  return s;
}

// The parameter, checked, where vectors of 4 can be read from it.
at::Tensor param(const at::Tensor& t, const at::Tensor& x, const char* name) {
  if (!t.defined()) return t;
  TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous() &&
                  t.dim() == 1 && t.size(0) == x.size(1) &&
                  t.device() == x.device(),
              "group_norm: ", name, " must be C floats on the input's device");
  return (uintptr_t)t.data_ptr() % 16 ? t.clone() : t;
}

const float* pointer(const at::Tensor& t) {
  return t.defined() ? t.data_ptr<float>() : nullptr;
}

#define GN_TYPE(t, call, args)                                              \
  switch (t) {                                                              \
    case at::kFloat: call##f32 args; break;                                 \
    case at::kHalf: call##f16 args; break;                                  \
    case at::kBFloat16: call##bf16 args; break;                             \
    default:                                                                \
      TORCH_CHECK(false,                                                    \
                  "group_norm: float32, float16 or bfloat16 expected");     \
  }

}  // namespace

// What a forward call keeps for its backward: floats, [2][b][g] mean and rstd,
// and behind them as many counters as a backward launch may need (a sample's,
// or a span of channels').
int64_t stat_floats(const GroupNormShape& s) {
  return 2 * (int64_t)s.b * s.g;
}

int counters(const GroupNormShape& s) { return std::max(s.b, s.c); }

// -> y, and what the backward needs where asked for
std::vector<at::Tensor> group_norm_forward(
    const at::Tensor& x, int64_t groups, const at::Tensor& weight,
    const at::Tensor& bias, double eps, int64_t act, double p,
    const at::Tensor& rng, int64_t seed, int64_t offset, bool keep) {
  const GroupNormShape s = shape_of(x, groups);
  TORCH_CHECK(eps > 0.0, "group_norm: eps must be positive");
  c10::DeviceGuard guard(x.device());
  const DropoutArgs d = dropout_args(p, rng, seed, offset, x);
  const at::Tensor wt = param(weight, x, "weight"), bt = param(bias, x, "bias");
  const float *w = pointer(wt), *b = pointer(bt);
  auto y = at::empty_like(x, x.options(), at::MemoryFormat::ChannelsLast);
  at::Tensor kept;
  float* stat = nullptr;
  uint32_t* counts = nullptr;
  if (keep) {
    kept = at::empty({stat_floats(s) + counters(s)},
                     x.options().dtype(at::kFloat));
    stat = kept.data_ptr<float>();
    counts = (uint32_t*)(stat + stat_floats(s));
  }
  if (x.numel() > 0)
    GN_TYPE(x.scalar_type(), gn_forward_,
            (x, y, w, b, stat, counts, counters(s), s, (float)eps, (int)act,
             d));
  return {y, kept};
}

// -> dx, dweight, dbias; an undefined tensor where none is wanted.  The
// counters in `kept` are used, and left as they were: calls with the same one
// follow each other on a stream, as the engine has them.  Replays of a graph
// follow nothing, so a call that is being recorded has counters of its own,
// cleared by a launch of some 2 us in the graph.
std::vector<at::Tensor> group_norm_backward(
    const at::Tensor& gy, const at::Tensor& x, int64_t groups,
    const at::Tensor& weight, const at::Tensor& bias, const at::Tensor& kept,
    int64_t act, double p, const at::Tensor& rng, int64_t seed, int64_t offset,
    bool need_x, bool need_weight, bool need_bias) {
  const GroupNormShape s = shape_of(x, groups);
  TORCH_CHECK(kept.scalar_type() == at::kFloat && kept.is_contiguous() &&
                  kept.numel() == stat_floats(s) + counters(s) &&
                  kept.device() == x.device(),
              "group_norm: not what the forward call kept");
  TORCH_CHECK(gy.sizes() == x.sizes() && gy.scalar_type() == x.scalar_type() &&
                  gy.device() == x.device() &&
                  gy.is_contiguous(at::MemoryFormat::ChannelsLast),
              "group_norm: gy must be like x");
  c10::DeviceGuard guard(x.device());
  const DropoutArgs d = dropout_args(p, rng, seed, offset, x);
  const at::Tensor wt = param(weight, x, "weight"), bt = param(bias, x, "bias");
  const float *w = pointer(wt), *b = pointer(bt);
  at::Tensor dx, dw, db;
  const auto opts = x.options().dtype(at::kFloat);
  if (need_x)
    dx = at::empty_like(x, x.options(), at::MemoryFormat::ChannelsLast);
  if (need_weight) dw = at::empty({x.size(1)}, opts);
  if (need_bias) db = at::empty({x.size(1)}, opts);
  if (x.numel() == 0) {
    if (need_weight) dw.zero_();
    if (need_bias) db.zero_();
    return {dx, dw, db};
  }
  if (!need_x && !need_weight && !need_bias) return {dx, dw, db};
  float* stat = kept.data_ptr<float>();
  uint32_t* counts = (uint32_t*)(stat + stat_floats(s));
  at::Tensor own;
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() !=
      c10::hip::CaptureStatus::None) {
    own = at::empty({counters(s)}, x.options().dtype(at::kInt)).zero_();
    counts = (uint32_t*)own.data_ptr<int>();
  }
  GN_TYPE(x.scalar_type(), gn_backward_,
          (x, gy, dx, w, b, stat, counts,
           need_bias ? db.data_ptr<float>() : nullptr,
           need_weight ? dw.data_ptr<float>() : nullptr, s, (int)act, d));
  return {dx, dw, db};
}
