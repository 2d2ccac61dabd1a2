// Activation + dropout with a mask that is never stored, for gfx950.
//
//   forward   y  = kept(i) ? act(x_i) / (1 - p) : 0
//   backward  dx = kept(i) ? gy_i / (1 - p) * act'(x_i) : 0
//
// kept(i) is computed from (seed, offset, i) in both directions
// (philox.hip.h), so neither a mask is written nor read back.
//
// Memory bounds it: 64x64x192x256 bf16, 403 MB read and 403 MB written, takes
// 131 us each way (6.2 TB/s; a plain copy here takes 134 to 148).  The
// generator costs some 20 quarter-rate products and 100 other instructions per
// 8 elements, about 90 us of the vector units, which hide behind other waves'
// loads as long as those are many: at 180 registers a thread, with four vectors
// in flight, it took 289 us, at 44 with two 193, and 131 once what is larger
// than the L2s went past the caches.  One short pass per block, blocks in
// memory's order.

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include "dropout_args.h"
#include "philox.hip.h"
#include "vec.hip.h"

namespace {

constexpr int BLOCK = 256;
constexpr int UNROLL = 2;  // vectors of 8 in flight per thread

template <typename T, bool WIDE>
__device__ __forceinline__ Pack<T, 8> load8(const T* at, int count,
                                            bool stream) {
  if (WIDE && count == 8) return load_pack<T, 8>(at, stream);
  Pack<T, 8> p;
#pragma unroll
  for (int k = 0; k < 8; ++k) p.v[k] = k < count ? at[k] : (T)0.0f;
  return p;
}

// WIDE: every pointer is aligned to 16 bytes.  Forwards reads x alone;
// backwards gy, and x where the activation has a slope.
template <typename T, bool WIDE, bool BACK, int ACT>
__global__ __launch_bounds__(BLOCK) void dropout_kernel(
    const T* __restrict__ x, const T* __restrict__ gy, T* __restrict__ out,
    int64_t n, int act, bool stream, DropoutArgs d) {
  const bool need_x = !BACK || (ACT == ACT_ANY ? act : ACT) != ACT_NONE;
  const DropoutState st = dropout_state(d);
  const int64_t first = (int64_t)blockIdx.x * (BLOCK * UNROLL) + threadIdx.x;
  Pack<T, 8> rx[UNROLL], rg[UNROLL];
#pragma unroll
  for (int i = 0; i < UNROLL; ++i) {
    const int64_t at = (first + i * BLOCK) * 8;
    const int count = (int)min((int64_t)8, n - at);
    if (count <= 0) continue;
    if (need_x) rx[i] = load8<T, WIDE>(x + at, count, stream);
    if (BACK) rg[i] = load8<T, WIDE>(gy + at, count, stream);
  }
#pragma unroll
  for (int i = 0; i < UNROLL; ++i) {
    const int64_t at = (first + i * BLOCK) * 8;
    const int count = (int)min((int64_t)8, n - at);
    if (count <= 0) continue;
    float v[8];
    if (BACK) {
      unpack<T, 8>(rg[i], v);
      if (need_x) {
        float z[8];
        unpack<T, 8>(rx[i], z);
        act_backward<T, ACT, 8>(act, z, v);
      }
    } else {
      unpack<T, 8>(rx[i], v);
      act_apply<T, ACT, 8>(act, v);
    }
    if (d.on) dropout_apply<8>(d, st, (uint64_t)at, v);
    const Pack<T, 8> o = pack<T, 8>(v);
    if (WIDE && count == 8) {
      store_pack<T, 8>(out + at, o, stream);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < count) out[at + k] = o.v[k];
    }
  }
}

bool wide(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, bool BACK>
void launch(const void* x, const void* gy, void* out, int64_t n, int act,
            const DropoutArgs& d) {
  const int64_t per_block = (int64_t)BLOCK * UNROLL * 8;
  const int64_t blocks = (n + per_block - 1) / per_block;
  // a launch's threads are counted in 32 bits
  TORCH_CHECK(blocks * BLOCK < (1ll << 32), "dropout: tensor too large");
  const hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
  auto kernel = dropout_kernel<T, false, BACK, ACT_ANY>;
  if (wide(x) && wide(gy) && wide(out)) {
    switch (act) {
      case ACT_ELU: kernel = dropout_kernel<T, true, BACK, ACT_ELU>; break;
      case ACT_LEAKY: kernel = dropout_kernel<T, true, BACK, ACT_LEAKY>; break;
      case ACT_RELU: kernel = dropout_kernel<T, true, BACK, ACT_RELU>; break;
      case ACT_SILU: kernel = dropout_kernel<T, true, BACK, ACT_SILU>; break;
      default: kernel = dropout_kernel<T, true, BACK, ACT_NONE>; break;
    }
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(BLOCK), 0, stream,
                     (const T*)x, (const T*)gy, (T*)out, n, act, n *
                     (int64_t)sizeof(T) > STREAM_BYTES, d);
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

template <typename T>
void launch_any(const void* x, const void* gy, void* out, int64_t n, int act,
                const DropoutArgs& d) {
  if (gy)
    launch<T, true>(x, gy, out, n, act, d);
  else
    launch<T, false>(x, nullptr, out, n, act, d);
}

at::Tensor dropout_any(const at::Tensor& like, const void* x, const void* gy,
                       long act, const DropoutArgs& d) {
  auto out = at::empty_like(like);  // dense input: the same strides
  const int64_t n = like.numel();
  if (n == 0) return out;
  switch (like.scalar_type()) {
    case at::kFloat:
      launch_any<float>(x, gy, out.data_ptr(), n, (int)act, d);
      break;
    case at::kHalf:
      launch_any<fp16_t>(x, gy, out.data_ptr(), n, (int)act, d);
      break;
    case at::kBFloat16:
      launch_any<bf16_t>(x, gy, out.data_ptr(), n, (int)act, d);
      break;
    default:
      TORCH_CHECK(false, "dropout: float32, float16 or bfloat16 expected");
  }
  return out;
}

void check_dense(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "dropout: ", name, " must be on the GPU");
  TORCH_CHECK(t.is_contiguous() ||
                  t.is_contiguous(at::MemoryFormat::ChannelsLast),
              "dropout: ", name, " must be contiguous or channels last");
}

}  // namespace

at::Tensor dropout_forward(const at::Tensor& x, int64_t act, double p,
                           const at::Tensor& rng, int64_t seed,
                           int64_t offset) {
  check_dense(x, "x");
  c10::DeviceGuard guard(x.device());
  return dropout_any(x, x.data_ptr(), nullptr, act,
                     dropout_args(p, rng, seed, offset, x));
}

// x is read where the activation has a slope, and may be undefined elsewhere.
at::Tensor dropout_backward(const at::Tensor& gy, const at::Tensor& x,
                            int64_t act, double p, const at::Tensor& rng,
                            int64_t seed, int64_t offset) {
  check_dense(gy, "gy");
  c10::DeviceGuard guard(gy.device());
  const void* xp = nullptr;
  if (act != ACT_NONE) {
    const auto cl = at::MemoryFormat::ChannelsLast;
    TORCH_CHECK(x.defined() && x.sizes() == gy.sizes() &&
                    ((x.is_contiguous() && gy.is_contiguous()) ||
                     (x.is_contiguous(cl) && gy.is_contiguous(cl))) &&
                    x.scalar_type() == gy.scalar_type() &&
                    x.device() == gy.device(),
                "dropout: x must be like gy");
    xp = x.data_ptr();
  }
  return dropout_any(gy, xp, gy.data_ptr(), act,
                     dropout_args(p, rng, seed, offset, gy));
}
