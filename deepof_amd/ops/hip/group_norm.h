// Group norm's launches, per type of values.
#pragma once

#include <torch/extension.h>

#include "dropout_args.h"

constexpr int MAX_GROUPS = 4096;  // their sums live in LDS

struct GroupNormShape {
  int64_t hw;
  int b, c, g, cg;  // cg = c / g
};

// stat: [2][b][g], mean and rstd, and counts, for the way back; both written
// going forwards unless null.  Going backwards counts are 0 before and after.
// dx undefined, dw or db null: not wanted.
#define GN_DECLARE(NAME)                                                      \
  void gn_forward_##NAME(const at::Tensor& x, at::Tensor& y, const float* w,  \
                         const float* bias, float* stat, uint32_t* counts,    \
                         int n_counts, const GroupNormShape& s, float eps,    \
                         int act, const DropoutArgs& d);                      \
  void gn_backward_##NAME(const at::Tensor& x, const at::Tensor& gy,          \
                          at::Tensor& dx, const float* w, const float* bias,  \
                          const float* stat, uint32_t* counts, float* db,     \
                          float* dw, const GroupNormShape& s, int act,        \
                          const DropoutArgs& d);
GN_DECLARE(f32)
GN_DECLARE(f16)
GN_DECLARE(bf16)
