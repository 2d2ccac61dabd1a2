// Typed vectors of activations, and activation functions in fp32.
#pragma once

#include <hip/hip_runtime.h>

using bf16_t = __bf16;
using fp16_t = _Float16;

// V values of T, moved in as few instructions as their size allows.
template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V>& p, float (&f)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) f[k] = (float)p.v[k];
}

// Rounds to nearest, once, on the way out.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> pack(const float (&f)[V]) {
  Pack<T, V> p;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    // two at a time: one instruction converts a pair to bf16
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef T t16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int k = 0; k < V; k += 2) {
      const f32x2 pair = {f[k], f[k + 1]};
      *reinterpret_cast<t16x2*>(&p.v[k]) =
          __builtin_convertvector(pair, t16x2);
    }
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) p.v[k] = (T)f[k];
  }
  return p;
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* at) {
  return *reinterpret_cast<const Pack<T, V>*>(at);
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* at, const Pack<T, V>& p) {
  *reinterpret_cast<Pack<T, V>*>(at) = p;
}

// The same past the caches, where `stream` (uniform) says that what is moved
// is larger than they are.  403 MB are copied in 134 us so, in 148 us else;
// what fits is better kept for who reads it next.
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* at, bool stream) {
  if constexpr (sizeof(Pack<T, V>) % 16 == 0) {
    if (stream) {
      Pack<T, V> p;
#pragma unroll
      for (int i = 0; i < (int)sizeof(p) / 16; ++i)
        reinterpret_cast<u32x4_t*>(&p)[i] = __builtin_nontemporal_load(
            reinterpret_cast<const u32x4_t*>(at) + i);
      return p;
    }
  }
  return load_pack<T, V>(at);
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* at, const Pack<T, V>& p,
                                           bool stream) {
  if constexpr (sizeof(Pack<T, V>) % 16 == 0) {
    if (stream) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(p) / 16; ++i)
        __builtin_nontemporal_store(reinterpret_cast<const u32x4_t*>(&p)[i],
                                    reinterpret_cast<u32x4_t*>(at) + i);
      return;
    }
  }
  store_pack<T, V>(at, p);
}

// Bytes of a tensor above which it is streamed: the L2s' 32 MB.
constexpr int64_t STREAM_BYTES = 32ll << 20;

// ACT_ANY: not known at compile time, passed in.
enum Act { ACT_ANY = -1, ACT_NONE = 0, ACT_ELU = 1, ACT_LEAKY = 2, ACT_RELU = 3,
           ACT_SILU = 4 };

// e^z through the hardware's 2^t.  t = z log2(e) is carried in two floats,
// or its rounding would cost |z| 2^-24 of the result.
__device__ __forceinline__ float exp_f32(float z) {
  const float hi = 1.44269502162933349609375f;    // log2(e) in fp32
  const float lo = 1.92596299112661746887e-8f;    // log2(e) - hi
  const float t = z * hi;
  const float e = __builtin_amdgcn_exp2f(t);
  const float r = fmaf(z, hi, -t) + z * lo;
  // beyond fp32's range e is 0 or infinite, and r may be no number
  return e == 0.0f || e == __builtin_inff()
             ? e : fmaf(e * 0.693147180559945f, r, e);
}

// The same for what ends in T.  In front of 16 bits, and of sums over many
// values, t in one float will do: up to |z| = 16 it is 2^-20 off.
template <typename T>
__device__ __forceinline__ float exp_for(float z) {
  if (sizeof(T) == 4) return exp_f32(z);
  return __builtin_amdgcn_exp2f(z * 1.44269502162933349609375f);
}

// e^z - 1 for z <= 0.  Near 0 the subtraction would cancel: a Taylor sum
// takes over where what it leaves out is below half a step of what is stored
// (z^7 / 40320 < 2^-25 for fp32 results, z^3 / 24 < 2^-17 for 16 bits).
template <typename T>
__device__ __forceinline__ float expm1_neg(float z) {
  const float far = exp_for<T>(z) - 1.0f;
  if (sizeof(T) == 4) {
    float s = 1.0f / 5040.0f;
    s = fmaf(s, z, 1.0f / 720.0f);
    s = fmaf(s, z, 1.0f / 120.0f);
    s = fmaf(s, z, 1.0f / 24.0f);
    s = fmaf(s, z, 1.0f / 6.0f);
    s = fmaf(s, z, 0.5f);
    s = fmaf(s * z, z, z);
    return z > -0.35f ? s : far;
  }
  float s = fmaf(1.0f / 6.0f, z, 0.5f);
  s = fmaf(s * z, z, z);
  return z > -0.03125f ? s : far;
}

// v = act(v).  Comparisons are written so that NaN stays NaN.
template <typename T, int ACT, int V>
__device__ __forceinline__ void act_apply(int act, float (&v)[V]) {
  switch (ACT == ACT_ANY ? act : ACT) {
    case ACT_ELU:
#pragma unroll
      for (int k = 0; k < V; ++k)
        v[k] = v[k] <= 0.0f ? expm1_neg<T>(v[k]) : v[k];
      break;
    case ACT_LEAKY:
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = v[k] <= 0.0f ? 0.1f * v[k] : v[k];
      break;
    case ACT_RELU:
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = v[k] <= 0.0f ? 0.0f : v[k];
      break;
    case ACT_SILU:
#pragma unroll
      for (int k = 0; k < V; ++k)
        v[k] = v[k] * __builtin_amdgcn_rcpf(1.0f + exp_for<T>(-v[k]));
      break;
    default:
      break;
  }
}

// g *= act'(z)
template <typename T, int ACT, int V>
__device__ __forceinline__ void act_backward(int act, const float (&z)[V],
                                             float (&g)[V]) {
  switch (ACT == ACT_ANY ? act : ACT) {
    case ACT_ELU:
#pragma unroll
      for (int k = 0; k < V; ++k) g[k] *= exp_for<T>(fminf(z[k], 0.0f));
      break;
    case ACT_LEAKY:
#pragma unroll
      for (int k = 0; k < V; ++k) g[k] = z[k] <= 0.0f ? 0.1f * g[k] : g[k];
      break;
    case ACT_RELU:
#pragma unroll
      for (int k = 0; k < V; ++k) g[k] = z[k] <= 0.0f ? 0.0f : g[k];
      break;
    case ACT_SILU:
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float t = __builtin_amdgcn_rcpf(1.0f + exp_for<T>(-z[k]));
        g[k] *= t * fmaf(z[k], 1.0f - t, 1.0f);
      }
      break;
    default:
      break;
  }
}
