// A dropout call's arguments, as the kernels take them.
#pragma once

#include <torch/extension.h>

#include <cmath>

// Element i = 8 j + s has a 32-bit number u(i).  Its upper half is the s-th
// 16 bits of Philox(key = seed, counter = (j, offset)); its lower half is the
// same of the counter with bit 63 of j set.  The element is dropped iff
// u(i) < threshold.  The upper half alone decides unless it equals the
// threshold's, for one element in 65536, so that 8 elements cost one Philox
// and yet p is held to 2^-32; where the threshold's lower half is 0 (p = 0.5,
// 0.25, ...) nothing is ever undecided.
struct DropoutArgs {
  const int64_t* rng;   // device [seed, offset], or null: the two below
  uint64_t seed;
  uint64_t offset;
  uint32_t thr_hi;      // threshold's halves; thr_hi = 65536 drops all
  uint32_t thr_lo;
  float scale;          // 1 / (1 - p)
  bool on;
};

// p in [0, 1]; rng: int64 [seed, offset] on like's device, or undefined, in
// which case the mask is that of (seed, offset).
inline DropoutArgs dropout_args(double p, const at::Tensor& rng,
                                int64_t seed, int64_t offset,
                                const at::Tensor& like) {
  TORCH_CHECK(p >= 0.0 && p <= 1.0, "dropout: p must lie in [0, 1]");
  DropoutArgs d{};
  d.on = p > 0.0;
  if (rng.defined()) {
    TORCH_CHECK(rng.scalar_type() == at::kLong && rng.numel() == 2 &&
                    rng.is_contiguous() && rng.device() == like.device(),
                "dropout: rng must be 2 int64 on the input's device");
    d.rng = rng.data_ptr<int64_t>();
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
