// Host side of a dropout call: its arguments, checked.
#pragma once

#include <torch/extension.h>

#include <cmath>

#include "philox.hip.h"

// p in [0, 1]; rng: int64 [seed, offset] on like's device, or none, in which
// case the mask is that of (seed, offset).
inline DropoutArgs dropout_args(double p, const c10::optional<at::Tensor>& rng,
                                int64_t seed, int64_t offset,
                                const at::Tensor& like) {
  TORCH_CHECK(p >= 0.0 && p <= 1.0, "dropout: p must lie in [0, 1]");
  DropoutArgs d{};
  d.on = p > 0.0;
  if (rng.has_value()) {
    TORCH_CHECK(rng->scalar_type() == at::kLong && rng->numel() == 2 &&
                    rng->is_contiguous() && rng->device() == like.device(),
                "dropout: rng must be 2 int64 on the input's device");
    d.rng = rng->data_ptr<int64_t>();
  }
  d.seed = (uint64_t)seed;
  d.offset = (uint64_t)offset;
  const uint64_t thr = (uint64_t)std::floor(p * 4294967296.0 + 0.5);
  d.thr_hi = (uint32_t)(thr >> 16);
  d.thr_lo = (uint32_t)(thr & 0xffff);
  // nothing is kept at p = 1: the scale is never used
  d.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
  return d;
}
