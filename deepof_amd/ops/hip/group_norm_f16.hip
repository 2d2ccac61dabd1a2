#include "group_norm.hip.h"

void gn_forward_f16(const at::Tensor& x, at::Tensor& y, const float* w,
                   const float* bias, float* stat, uint32_t* counts,
                   int n_counts, const GroupNormShape& s, float eps, int act,
                   const DropoutArgs& d) {
  gn_forward<fp16_t>(x, y, w, bias, stat, counts, n_counts, s, eps, act, d);
}

void gn_backward_f16(const at::Tensor& x, const at::Tensor& gy, at::Tensor& dx,
                    const float* w, const float* bias, const float* stat,
                    uint32_t* counts, float* db, float* dw,
                    const GroupNormShape& s, int act, const DropoutArgs& d) {
  gn_backward<fp16_t>(x, gy, dx, w, bias, stat, counts, db, dw, s, act, d);
}
