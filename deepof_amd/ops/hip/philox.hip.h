// Counter-based random bits for dropout masks on gfx950.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", SC 2011): ten rounds of two 32x32 -> 64 bit products
// turn a 128-bit counter and a 64-bit key into 128 random bits.  A mask is a
// function of (seed, offset, element), so backward passes compute it again
// and nothing is stored.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dropout_args.h"

struct DropoutState {
  uint32_t k0, k1, o0, o1;
};

__device__ __forceinline__ DropoutState dropout_state(const DropoutArgs& d) {
  uint64_t seed = d.seed, offset = d.offset;
  if (d.on && d.rng) {
    seed = (uint64_t)d.rng[0];
    offset = (uint64_t)d.rng[1];
  }
  return {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)offset,
          (uint32_t)(offset >> 32)};
}

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);  // one instruction
}

__device__ __forceinline__ void philox4x32(uint32_t c[4], uint32_t k0,
                                           uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c[0] * 0xD2511F53u;
    const uint64_t b = (uint64_t)c[2] * 0xCD9E8D57u;
    const uint32_t n0 = xor3((uint32_t)(b >> 32), c[1], k0);
    const uint32_t n2 = xor3((uint32_t)(a >> 32), c[3], k1);
    c[0] = n0;
    c[1] = (uint32_t)b;
    c[2] = n2;
    c[3] = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// The 8 elements of block j: h[s] >= thr_hi iff element 8 j + s is kept.
__device__ __forceinline__ void dropout_numbers(const DropoutArgs& d,
                                                const DropoutState& st,
                                                uint64_t j, int h[8]) {
  uint32_t c[4] = {(uint32_t)j, (uint32_t)(j >> 32), st.o0, st.o1};
  philox4x32(c, st.k0, st.k1);
#pragma unroll
  for (int s = 0; s < 8; ++s)
    h[s] = (int)((c[s >> 1] >> ((s & 1) * 16)) & 0xffffu);
  if (d.thr_lo != 0) {
    bool open = false;
#pragma unroll
    for (int s = 0; s < 8; ++s) open |= h[s] == (int)d.thr_hi;
    if (open) {
      uint32_t l[4] = {(uint32_t)j, (uint32_t)(j >> 32) | 0x80000000u, st.o0,
                       st.o1};
      philox4x32(l, st.k0, st.k1);
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const uint32_t low = (l[s >> 1] >> ((s & 1) * 16)) & 0xffffu;
        if (h[s] == (int)d.thr_hi && low < d.thr_lo) h[s] = -1;
      }
    }
  }
}

// v[k], k < V, belong to elements at .. at + V - 1: v = kept ? v * scale : 0.
// Dropped values are selected away, not multiplied by 0, so that infinities
// and NaN in dropped places leave no trace.  `at` is a multiple of V, and V
// divides 8, so that one block of 8 holds all of them.
template <int V>
__device__ __forceinline__ void dropout_apply(const DropoutArgs& d,
                                              const DropoutState& st,
                                              uint64_t at, float (&v)[V]) {
  static_assert(8 % V == 0, "a vector lies in one block of 8 elements");
  int h[8];
  dropout_numbers(d, st, at >> 3, h);
  const int s0 = (int)(at & 7);
#pragma unroll
  for (int k = 0; k < V; ++k) {
    int n = h[k];
    if (V < 8) {
      n = h[0];
#pragma unroll
      for (int s = 1; s < 8; ++s) n = (s == s0 + k) ? h[s] : n;
    }
    v[k] = n >= (int)d.thr_hi ? v[k] * d.scale : 0.0f;
  }
}
