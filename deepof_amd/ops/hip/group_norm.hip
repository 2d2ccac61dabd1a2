// Group normalisation + affine + activation (+ dropout), channels last, for
// gfx950.
//
// A group is the N = H W (C / G) values of one sample's C / G neighbouring
// channels.  With mean and var of the group, rstd = 1 / sqrt(var + eps),
// xhat = (x - mean) rstd and z = xhat w_c + b_c:
//
//   y    = act(z), with dropout behind it where asked for
//   gz   = gy (through dropout) act'(z)
//   db_c = sum gz,   dw_c = sum gz xhat       (over samples and pixels)
//   s1   = sum w gz, s2   = sum w gz xhat     (over the group)
//   dx   = rstd (w gz - (s1 + xhat s2) / N)
//
// z is computed again from x going backwards; mean and rstd, 2 B G floats,
// are all that is kept.  Everything between loading x and storing y or dx is
// fp32, and a result is rounded once.
//
// Memory bounds all of it.  Two routes:
//  - resident: a block holds a whole bundle of groups in registers, so x (and
//    gy) are read once, in one launch;
//  - split: pixels are split over blocks, which leave partial statistics; a
//    second launch joins them (every block for itself, in the same order) and
//    reads x again.
// Sums have a fixed order everywhere: no atomics, equal results every time.

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <algorithm>

#include "dropout_args.h"
#include "philox.hip.h"
#include "vec.hip.h"

namespace {

constexpr int WAVE = 64;
constexpr int BLOCK = 256;       // threads of the split route's blocks
constexpr int UNROLL = 2;        // vectors in flight per thread and tensor
constexpr int MAX_GROUPS = 4096; // their statistics live in LDS

struct Shape {
  int64_t hw;
  int b, c, g, cg;  // cg = c / g
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = WAVE / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE);
  return v;
}

// Pixels cut into n pieces, the first `more` of them one longer than `size`.
struct Cut {
  int n, size, more;
  __device__ __forceinline__ int first(int i) const {
    return i * size + min(i, more);
  }
  __device__ __forceinline__ int pixels(int i) const {
    return size + (i < more ? 1 : 0);
  }
};

// Joins the (n, mean, M2) of entries into lane-uniform totals, each lane
// bringing one entry at a time through `get(i, n, mean, m2)`.  Two passes:
// the mean first, taken relative to entry 0's, then squares about it.
template <typename Get>
__device__ __forceinline__ void join(int count, int lane, Get get, float& n,
                                     float& mean, float& m2) {
  float n0, ref, q0;
  get(0, n0, ref, q0);
  float sn = 0.0f, sm = 0.0f;
  for (int i = lane; i < count; i += WAVE) {
    float ni, mi, qi;
    get(i, ni, mi, qi);
    sn += ni;
    sm += ni * (mi - ref);
  }
  sn = wave_sum(sn);
  sm = wave_sum(sm);
  n = sn;
  mean = ref + sm / sn;
  float sq = 0.0f;
  for (int i = lane; i < count; i += WAVE) {
    float ni, mi, qi;
    get(i, ni, mi, qi);
    const float d = mi - mean;
    sq += qi + ni * d * d;
  }
  m2 = wave_sum(sq);
}

__device__ __forceinline__ float rstd_of(float m2, float n, float eps) {
  return 1.0f / sqrtf(fmaxf(m2, 0.0f) / n + eps);
}

// ---------------------------------------------------------------------------
// split route
// ---------------------------------------------------------------------------
// Block (split, sample): thread t owns the V channels of column t % cols of a
// chunk of columns and walks down its pixels.  A thread sums x - K and
// (x - K)^2 with K = its first value, so that a mean far from 0 costs no
// digits, and threads are joined by (n, mean, M2).  ONE: all V channels are
// in the same group, and share a sum.
//
// part: [b][g][splits] of (mean, M2); every split has the same kind of
// entry, so n follows from its bounds.
template <typename T, int V, bool ONE>
__global__ __launch_bounds__(BLOCK) void gn_stats(const T* __restrict__ x,
                                                  float2* __restrict__ part,
                                                  Shape s, Cut cut) {
  constexpr int A = ONE ? 1 : V;
  __shared__ float2 red[BLOCK * A];
  extern __shared__ float joined[];  // [3][g]: n, mean, M2 so far
  const int split = blockIdx.x % cut.n, b = blockIdx.x / cut.n;
  const int pixels = cut.pixels(split);
  const T* base = x + ((int64_t)b * s.hw + cut.first(split)) * s.c;
  const int nv = s.c / V;                // columns of V channels
  const int unit = V / A;                // channels per entry
  const int upg = s.cg / unit;           // entries per group and row
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;

  for (int c0 = 0; c0 < nv; c0 += BLOCK) {
    const int cols = min(BLOCK, nv - c0);
    const int rows = BLOCK / cols;
    const int row = threadIdx.x / cols, col = threadIdx.x % cols;
    const T* at = base + (int64_t)(c0 + col) * V;
    float k[A], s1[A], s2[A];
#pragma unroll
    for (int a = 0; a < A; ++a) k[a] = s1[a] = s2[a] = 0.0f;
    if (row < rows && row < pixels) {
      float v[V];
      unpack<T, V>(load_pack<T, V>(at + (int64_t)row * s.c), v);
#pragma unroll
      for (int a = 0; a < A; ++a) k[a] = v[a];
      int p = row;
      for (; p + (UNROLL - 1) * rows < pixels; p += UNROLL * rows) {
        Pack<T, V> raw[UNROLL];
#pragma unroll
        for (int i = 0; i < UNROLL; ++i)
          raw[i] = load_pack<T, V>(at + (int64_t)(p + i * rows) * s.c);
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
          unpack<T, V>(raw[i], v);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int a = ONE ? 0 : j;
            const float d = v[j] - k[a];
            s1[a] += d;
            s2[a] = fmaf(d, d, s2[a]);
          }
        }
      }
      for (; p < pixels; p += rows) {
        unpack<T, V>(load_pack<T, V>(at + (int64_t)p * s.c), v);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int a = ONE ? 0 : j;
          const float d = v[j] - k[a];
          s1[a] += d;
          s2[a] = fmaf(d, d, s2[a]);
        }
      }
    }
    const int filled = min(rows, pixels);  // rows that hold anything
    if (row < filled) {
      const float n = (float)(((pixels - row + rows - 1) / rows) * unit);
#pragma unroll
      for (int a = 0; a < A; ++a) {
        const float m = s1[a] / n;
        red[(row * cols + col) * A + a] =
            make_float2(k[a] + m, fmaxf(s2[a] - s1[a] * m, 0.0f));
      }
    }
    __syncthreads();
    // a wave per group that has entries in this chunk
    const int u0 = c0 * A, u1 = u0 + cols * A;
    for (int g = u0 / upg + wave; g * upg < u1; g += BLOCK / WAVE) {
      const int lo = max(g * upg, u0) - u0;
      const int here = min((g + 1) * upg, u1) - u0 - lo;
      float n, mean, m2;
      join(filled * here, lane,
           [&](int i, float& ni, float& mi, float& qi) {
             const int r = i / here;
             const float2 e = red[r * cols * A + lo + i % here];
             ni = (float)(((pixels - r + rows - 1) / rows) * unit);
             mi = e.x;
             qi = e.y;
           },
           n, mean, m2);
      if (lane == 0) {
        if (g * upg < u0) {  // begun in an earlier chunk
          const float na = joined[g], ma = joined[s.g + g];
          const float d = mean - ma, sum = na + n;
          m2 += joined[2 * s.g + g] + d * d * (na * n / sum);
          mean = ma + d * (n / sum);
          n = sum;
        }
        joined[g] = n;
        joined[s.g + g] = mean;
        joined[2 * s.g + g] = m2;
      }
    }
    __syncthreads();
  }
  for (int g = threadIdx.x; g < s.g; g += BLOCK)
    part[((int64_t)b * s.g + g) * cut.n + split] =
        make_float2(joined[s.g + g], joined[2 * s.g + g]);
}

// Block (chunk, sample): joins the sample's partial statistics, then reads x
// and writes y.  The first block of a sample leaves its mean and rstd.
template <typename T, int V, int ACT>
__global__ __launch_bounds__(BLOCK) void gn_apply(
    const T* __restrict__ x, T* __restrict__ y, const float* __restrict__ w,
    const float* __restrict__ bias, const float2* __restrict__ part,
    float* __restrict__ mean_out, float* __restrict__ rstd_out, Shape s,
    Cut cut, Cut chunks, float eps, int act, DropoutArgs d) {
  extern __shared__ float stat[];  // [2][g]: mean, rstd
  const int chunk = blockIdx.x % chunks.n, b = blockIdx.x / chunks.n;
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const DropoutState st = dropout_state(d);
  for (int g = wave; g < s.g; g += BLOCK / WAVE) {
    const float2* e = part + ((int64_t)b * s.g + g) * cut.n;
    float n, mean, m2;
    join(cut.n, lane,
         [&](int i, float& ni, float& mi, float& qi) {
           ni = (float)cut.pixels(i) * (float)s.cg;
           mi = e[i].x;
           qi = e[i].y;
         },
         n, mean, m2);
    if (lane == 0) {
      const float rstd = rstd_of(m2, n, eps);
      stat[g] = mean;
      stat[s.g + g] = rstd;
      if (chunk == 0) {
        mean_out[(int64_t)b * s.g + g] = mean;
        rstd_out[(int64_t)b * s.g + g] = rstd;
      }
    }
  }
  __syncthreads();
  const int pixels = chunks.pixels(chunk);
  const int64_t from = ((int64_t)b * s.hw + chunks.first(chunk)) * s.c;
  const int nv = s.c / V;
  for (int c0 = 0; c0 < nv; c0 += BLOCK) {
    const int cols = min(BLOCK, nv - c0);
    const int rows = BLOCK / cols;
    const int row = threadIdx.x / cols, col = threadIdx.x % cols;
    if (row >= rows) continue;
    const int ch = (c0 + col) * V;
    float m[V], a[V], o[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int g = (ch + j) / s.cg;
      m[j] = stat[g];
      a[j] = stat[s.g + g] * (w ? w[ch + j] : 1.0f);
      o[j] = bias ? bias[ch + j] : 0.0f;
    }
    auto emit = [&](int p, const Pack<T, V>& raw) {
      float v[V];
      unpack<T, V>(raw, v);
      const int64_t at = from + (int64_t)p * s.c + ch;
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = fmaf(v[j] - m[j], a[j], o[j]);
      act_apply<T, ACT, V>(act, v);
      if (d.on) dropout_apply<V>(d, st, (uint64_t)at, v);
      store_pack<T, V>(y + at, pack<T, V>(v));
    };
    const T* at = x + from + ch;
    int p = row;
    for (; p + (UNROLL - 1) * rows < pixels; p += UNROLL * rows) {
      Pack<T, V> raw[UNROLL];
#pragma unroll
      for (int i = 0; i < UNROLL; ++i)
        raw[i] = load_pack<T, V>(at + (int64_t)(p + i * rows) * s.c);
#pragma unroll
      for (int i = 0; i < UNROLL; ++i) emit(p + i * rows, raw[i]);
    }
    for (; p < pixels; p += rows)
      emit(p, load_pack<T, V>(at + (int64_t)p * s.c));
  }
}

// What a thread needs of its V channels going backwards.
template <int V>
struct Channel {
  float mean[V], rstd[V], w[V], b[V];
};

template <int V>
__device__ __forceinline__ void load_channel(Channel<V>& k, int ch, int cg,
                                             const float* mean,
                                             const float* rstd, const float* w,
                                             const float* bias) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int g = (ch + j) / cg;
    k.mean[j] = mean[g];
    k.rstd[j] = rstd[g];
    k.w[j] = w ? w[ch + j] : 1.0f;
    k.b[j] = bias ? bias[ch + j] : 0.0f;
  }
}

// (x, gy) -> (xhat, gz)
template <int ACT, int V>
__device__ __forceinline__ void through(const Channel<V>& k, int act,
                                        const DropoutArgs& d,
                                        const DropoutState& st, uint64_t at,
                                        float (&x)[V], float (&g)[V]) {
  if (d.on) dropout_apply<V>(d, st, at, g);
  float z[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    x[j] = (x[j] - k.mean[j]) * k.rstd[j];
    z[j] = fmaf(x[j], k.w[j], k.b[j]);
  }
  act_backward<ACT, V>(act, z, g);
}

// Block (split, sample): sums of gz and gz xhat of every channel over the
// split's pixels.  part_c: [2][b * splits][c]; part_g: [b][g][splits] of the
// same sums weighted by w and joined over the group.
template <typename T, int V, int ACT>
__global__ __launch_bounds__(BLOCK) void gn_bwd_sums(
    const T* __restrict__ x, const T* __restrict__ gy,
    const float* __restrict__ w, const float* __restrict__ bias,
    const float* __restrict__ mean, const float* __restrict__ rstd,
    float* __restrict__ part_c, float2* __restrict__ part_g, Shape s,
    Cut cut, int act, DropoutArgs d) {
  __shared__ float red[2][BLOCK * V];
  extern __shared__ float joined[];  // [2][g]
  const int split = blockIdx.x % cut.n, b = blockIdx.x / cut.n;
  const DropoutState st = dropout_state(d);
  const int pixels = cut.pixels(split);
  const int64_t from = ((int64_t)b * s.hw + cut.first(split)) * s.c;
  const int nv = s.c / V;
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  float* out1 = part_c + ((int64_t)b * cut.n + split) * s.c;
  float* out2 = out1 + (int64_t)s.b * cut.n * s.c;
  mean += (int64_t)b * s.g;
  rstd += (int64_t)b * s.g;

  for (int c0 = 0; c0 < nv; c0 += BLOCK) {
    const int cols = min(BLOCK, nv - c0);
    const int rows = BLOCK / cols;
    const int row = threadIdx.x / cols, col = threadIdx.x % cols;
    const int ch = (c0 + col) * V;
    float s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0f;
    if (row < rows) {
      Channel<V> k;
      load_channel<V>(k, ch, s.cg, mean, rstd, w, bias);
      auto add = [&](int p, const Pack<T, V>& rx, const Pack<T, V>& rg) {
        float h[V], g[V];
        unpack<T, V>(rx, h);
        unpack<T, V>(rg, g);
        through<ACT, V>(k, act, d, st, (uint64_t)(from + (int64_t)p * s.c + ch), h,
                   g);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          s1[j] += g[j];
          s2[j] = fmaf(g[j], h[j], s2[j]);
        }
      };
      const T* ax = x + from + ch;
      const T* ag = gy + from + ch;
      int p = row;
      for (; p + (UNROLL - 1) * rows < pixels; p += UNROLL * rows) {
        Pack<T, V> rx[UNROLL], rg[UNROLL];
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
          rx[i] = load_pack<T, V>(ax + (int64_t)(p + i * rows) * s.c);
          rg[i] = load_pack<T, V>(ag + (int64_t)(p + i * rows) * s.c);
        }
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) add(p + i * rows, rx[i], rg[i]);
      }
      for (; p < pixels; p += rows)
        add(p, load_pack<T, V>(ax + (int64_t)p * s.c),
            load_pack<T, V>(ag + (int64_t)p * s.c));
#pragma unroll
      for (int j = 0; j < V; ++j) {
        red[0][(row * cols + col) * V + j] = s1[j];
        red[1][(row * cols + col) * V + j] = s2[j];
      }
    }
    __syncthreads();
    // over the rows, channel by channel; totals land in row 0
    const int width = cols * V;
    for (int i = threadIdx.x; i < 2 * width; i += BLOCK) {
      const int which = i >= width, c = i - which * width;
      float sum = 0.0f;
      for (int r = 0; r < rows; ++r) sum += red[which][r * width + c];
      red[which][c] = sum;
      (which ? out2 : out1)[c0 * V + c] = sum;
    }
    __syncthreads();
    const int first = c0 * V, last = first + width;
    for (int g = first / s.cg + wave; g * s.cg < last; g += BLOCK / WAVE) {
      const int lo = max(g * s.cg, first), hi = min((g + 1) * s.cg, last);
      float t1 = 0.0f, t2 = 0.0f;
      for (int c = lo + lane; c < hi; c += WAVE) {
        const float wc = w ? w[c] : 1.0f;
        t1 = fmaf(wc, red[0][c - first], t1);
        t2 = fmaf(wc, red[1][c - first], t2);
      }
      t1 = wave_sum(t1);
      t2 = wave_sum(t2);
      if (lane == 0) {
        const bool begun = g * s.cg < first;
        joined[g] = t1 + (begun ? joined[g] : 0.0f);
        joined[s.g + g] = t2 + (begun ? joined[s.g + g] : 0.0f);
      }
    }
    __syncthreads();
  }
  for (int g = threadIdx.x; g < s.g; g += BLOCK)
    part_g[((int64_t)b * s.g + g) * cut.n + split] =
        make_float2(joined[g], joined[s.g + g]);
}

// Channels [8 block, 8 block + 8): sums of `rows` rows of part ([2][rows][c])
// into db and dw (either may be null).
__device__ __forceinline__ void param_sums(const float* __restrict__ part,
                                           int64_t rows, int c, int block,
                                           float* __restrict__ db,
                                           float* __restrict__ dw,
                                           float* red /* [BLOCK] */) {
  const int ch = block * 8 + (threadIdx.x & 7);
  const int r0 = threadIdx.x >> 3;
  for (int which = 0; which < 2; ++which) {
    float* out = which ? dw : db;
    if (!out) continue;
    const float* at = part + (int64_t)which * rows * c + ch;
    float sum = 0.0f;
    if (ch < c) {
#pragma unroll 8
      for (int64_t r = r0; r < rows; r += BLOCK / 8) sum += at[r * c];
    }
    red[threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.x < 8 && ch < c) {
      float total = 0.0f;
      for (int i = 0; i < BLOCK / 8; ++i) total += red[i * 8 + threadIdx.x];
      out[ch] = total;
    }
    __syncthreads();
  }
}

__global__ __launch_bounds__(BLOCK) void gn_param_grad(
    const float* __restrict__ part, int64_t rows, int c,
    float* __restrict__ db, float* __restrict__ dw) {
  __shared__ float red[BLOCK];
  param_sums(part, rows, c, blockIdx.x, db, dw, red);
}

// The first `param_blocks` blocks sum the parameters' gradients while the
// others, (chunk, sample), write dx.
template <typename T, int V, int ACT>
__global__ __launch_bounds__(BLOCK) void gn_bwd_dx(
    const T* __restrict__ x, const T* __restrict__ gy, T* __restrict__ dx,
    const float* __restrict__ w, const float* __restrict__ bias,
    const float* __restrict__ mean, const float* __restrict__ rstd,
    const float* __restrict__ part_c, const float2* __restrict__ part_g,
    float* __restrict__ db, float* __restrict__ dw, Shape s, Cut cut,
    Cut chunks, int param_blocks, int act, DropoutArgs d) {
  extern __shared__ float sums[];  // [2][g], at least BLOCK
  if ((int)blockIdx.x < param_blocks) {
    param_sums(part_c, (int64_t)s.b * cut.n, s.c, blockIdx.x, db, dw, sums);
    return;
  }
  const int at_block = blockIdx.x - param_blocks;
  const int chunk = at_block % chunks.n, b = at_block / chunks.n;
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const DropoutState st = dropout_state(d);
  const float inv_n = 1.0f / ((float)s.hw * (float)s.cg);
  for (int g = wave; g < s.g; g += BLOCK / WAVE) {
    const float2* e = part_g + ((int64_t)b * s.g + g) * cut.n;
    float t1 = 0.0f, t2 = 0.0f;
    for (int i = lane; i < cut.n; i += WAVE) {
      t1 += e[i].x;
      t2 += e[i].y;
    }
    t1 = wave_sum(t1);
    t2 = wave_sum(t2);
    if (lane == 0) {
      sums[g] = t1 * inv_n;
      sums[s.g + g] = t2 * inv_n;
    }
  }
  __syncthreads();
  mean += (int64_t)b * s.g;
  rstd += (int64_t)b * s.g;
  const int pixels = chunks.pixels(chunk);
  const int64_t from = ((int64_t)b * s.hw + chunks.first(chunk)) * s.c;
  const int nv = s.c / V;
  for (int c0 = 0; c0 < nv; c0 += BLOCK) {
    const int cols = min(BLOCK, nv - c0);
    const int rows = BLOCK / cols;
    const int row = threadIdx.x / cols, col = threadIdx.x % cols;
    if (row >= rows) continue;
    const int ch = (c0 + col) * V;
    Channel<V> k;
    load_channel<V>(k, ch, s.cg, mean, rstd, w, bias);
    float t1[V], t2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      t1[j] = sums[(ch + j) / s.cg];
      t2[j] = sums[s.g + (ch + j) / s.cg];
    }
    auto emit = [&](int p, const Pack<T, V>& rx, const Pack<T, V>& rg) {
      float h[V], g[V];
      unpack<T, V>(rx, h);
      unpack<T, V>(rg, g);
      const int64_t at = from + (int64_t)p * s.c + ch;
      through<ACT, V>(k, act, d, st, (uint64_t)at, h, g);
#pragma unroll
      for (int j = 0; j < V; ++j)
        g[j] = k.rstd[j] * (fmaf(k.w[j], g[j], -t1[j]) - h[j] * t2[j]);
      store_pack<T, V>(dx + at, pack<T, V>(g));
    };
    const T* ax = x + from + ch;
    const T* ag = gy + from + ch;
    int p = row;
    for (; p + (UNROLL - 1) * rows < pixels; p += UNROLL * rows) {
      Pack<T, V> rx[UNROLL], rg[UNROLL];
#pragma unroll
      for (int i = 0; i < UNROLL; ++i) {
        rx[i] = load_pack<T, V>(ax + (int64_t)(p + i * rows) * s.c);
        rg[i] = load_pack<T, V>(ag + (int64_t)(p + i * rows) * s.c);
      }
#pragma unroll
      for (int i = 0; i < UNROLL; ++i) emit(p + i * rows, rx[i], rg[i]);
    }
    for (; p < pixels; p += rows)
      emit(p, load_pack<T, V>(ax + (int64_t)p * s.c),
           load_pack<T, V>(ag + (int64_t)p * s.c));
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
Shape shape_of(const at::Tensor& x, int64_t groups) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 4 &&
                  x.is_contiguous(at::MemoryFormat::ChannelsLast),
              "group_norm: x must be a 4-D channels-last GPU tensor");
  TORCH_CHECK(groups >= 1 && groups <= MAX_GROUPS && x.size(1) >= 1 &&
                  x.size(1) % groups == 0,
              "group_norm: the channels must divide into 1 to ", MAX_GROUPS,
              " groups");
  TORCH_CHECK(x.size(0) < (1ll << 24) && x.size(1) < (1ll << 24) &&
                  x.size(2) * x.size(3) < (1ll << 31),
              "group_norm: tensor too large");
  Shape s;
  s.hw = x.size(2) * x.size(3);
  s.b = (int)x.size(0);
  s.c = (int)x.size(1);
  s.g = (int)groups;
  s.cg = s.c / s.g;
  return s;
}

const float* param(const c10::optional<at::Tensor>& t, const at::Tensor& x,
                   const char* name) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() &&
                  t->dim() == 1 && t->size(0) == x.size(1) &&
                  t->device() == x.device(),
              "group_norm: ", name, " must be C floats on the input's device");
  return t->data_ptr<float>();
}

bool aligned(const void* p, size_t to) {
  return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0;
}

// Channels a thread moves at once: the most of 8, 4 and 1 that divide C and
// whose vectors are aligned.
template <typename T>
int vector_of(const Shape& s, std::initializer_list<const void*> ptrs) {
  for (int v : {8, 4}) {
    const size_t to = std::min<size_t>(16, v * sizeof(T));
    bool ok = s.c % v == 0;
    for (const void* p : ptrs) ok = ok && aligned(p, to);
    if (ok) return v;
  }
  return 1;
}

// Blocks per sample: about `total` blocks over the batch, each with `least`
// values or more, and at most `most` (each costs the second launch a read).
Cut cut_pixels(const Shape& s, int total, int64_t least, int most) {
  int64_t n = (total + s.b - 1) / s.b;
  n = std::min<int64_t>(n, std::max<int64_t>(1, s.hw * s.c / least));
  n = std::min<int64_t>(n, s.hw);
  n = std::max<int64_t>(1, std::min<int64_t>(n, most));
  return {(int)n, (int)(s.hw / n), (int)(s.hw % n)};
}

// Activations are compiled in for whole vectors; narrower ones, which odd
// channel counts take, choose as they go.
#define GN_VARIANT(V_, ACT_, ...)                                    \
  do {                                                               \
    if (V_ == 8) {                                                   \
      constexpr int V = 8;                                           \
      switch (ACT_) {                                                \
        case ACT_ELU: { constexpr int ACT = ACT_ELU; __VA_ARGS__; break; }     \
        case ACT_LEAKY: { constexpr int ACT = ACT_LEAKY; __VA_ARGS__; break; } \
        case ACT_RELU: { constexpr int ACT = ACT_RELU; __VA_ARGS__; break; }   \
        case ACT_SILU: { constexpr int ACT = ACT_SILU; __VA_ARGS__; break; }   \
        default: { constexpr int ACT = ACT_NONE; __VA_ARGS__; break; }         \
      }                                                              \
    } else if (V_ == 4) {                                            \
      constexpr int V = 4, ACT = ACT_ANY;                            \
      __VA_ARGS__;                                                   \
    } else {                                                         \
      constexpr int V = 1, ACT = ACT_ANY;                            \
      __VA_ARGS__;                                                   \
    }                                                                \
  } while (0)

template <typename T, int V>
void launch_stats(const T* x, float2* part, const Shape& s, const Cut& cut,
                  hipStream_t stream) {
  auto kernel = s.cg % V == 0 ? gn_stats<T, V, true> : gn_stats<T, V, false>;
  kernel<<<s.b * cut.n, BLOCK, 3 * s.g * 4, stream>>>(x, part, s, cut);
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

template <typename T>
void forward(const at::Tensor& x, at::Tensor& y, const float* w,
             const float* bias, at::Tensor& mean, at::Tensor& rstd,
             const Shape& s, float eps, int act, const DropoutArgs& d) {
  const hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
  const T* px = (const T*)x.data_ptr();
  T* py = (T*)y.data_ptr();
  const int v = vector_of<T>(s, {px, py});
  const Cut cut = cut_pixels(s, 2048, 16384, 256);
  const Cut chunks = cut_pixels(s, 2048, 16384, 1 << 20);
  TORCH_CHECK((int64_t)s.b * std::max(cut.n, chunks.n) < (1ll << 31),
              "group_norm: tensor too large");
  auto part = at::empty({(int64_t)s.b * s.g * cut.n * 2}, mean.options());
  float2* pp = (float2*)part.data_ptr();
  if (v == 8)
    launch_stats<T, 8>(px, pp, s, cut, stream);
  else if (v == 4)
    launch_stats<T, 4>(px, pp, s, cut, stream);
  else
    launch_stats<T, 1>(px, pp, s, cut, stream);
  GN_VARIANT(v, act, {
    gn_apply<T, V, ACT><<<s.b * chunks.n, BLOCK, 2 * s.g * 4, stream>>>(
        px, py, w, bias, pp, mean.data_ptr<float>(), rstd.data_ptr<float>(), s,
        cut, chunks, eps, act, d);
    C10_HIP_KERNEL_LAUNCH_CHECK();
  });
}

template <typename T>
void backward(const at::Tensor& x, const at::Tensor& gy, T* dx, const float* w,
              const float* bias, const float* mean, const float* rstd,
              float* db, float* dw, const Shape& s, int act,
              const DropoutArgs& d) {
  const hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
  const T* px = (const T*)x.data_ptr();
  const T* pg = (const T*)gy.data_ptr();
  const int v = vector_of<T>(s, {px, pg, dx});
  const Cut cut = cut_pixels(s, 2048, 16384, 256);
  const Cut chunks = cut_pixels(s, 2048, 16384, 1 << 20);
  const int param_blocks = db || dw ? (s.c + 7) / 8 : 0;
  TORCH_CHECK((int64_t)s.b * std::max(cut.n, chunks.n) + param_blocks <
                  (1ll << 31),
              "group_norm: tensor too large");
  const auto opts = x.options().dtype(at::kFloat);
  auto part_c = at::empty({2 * (int64_t)s.b * cut.n * s.c}, opts);
  auto part_g = at::empty({(int64_t)s.b * s.g * cut.n * 2}, opts);
  float* pc = part_c.data_ptr<float>();
  float2* pp = (float2*)part_g.data_ptr();
  GN_VARIANT(v, act, {
    gn_bwd_sums<T, V, ACT><<<s.b * cut.n, BLOCK, 2 * s.g * 4, stream>>>(
        px, pg, w, bias, mean, rstd, pc, pp, s, cut, act, d);
    C10_HIP_KERNEL_LAUNCH_CHECK();
    if (dx) {
      gn_bwd_dx<T, V, ACT><<<s.b * chunks.n + param_blocks, BLOCK,
                             std::max(2 * s.g, BLOCK) * 4, stream>>>(
          px, pg, dx, w, bias, mean, rstd, pc, pp, db, dw, s, cut, chunks,
          param_blocks, act, d);
    } else {
      gn_param_grad<<<param_blocks, BLOCK, 0, stream>>>(
          pc, (int64_t)s.b * cut.n, s.c, db, dw);
    }
    C10_HIP_KERNEL_LAUNCH_CHECK();
  });
}

#define GN_TYPE(t, ...)                                                      \
  switch (t) {                                                               \
    case at::kFloat: { using T = float; __VA_ARGS__; break; }                \
    case at::kHalf: { using T = fp16_t; __VA_ARGS__; break; }                \
    case at::kBFloat16: { using T = bf16_t; __VA_ARGS__; break; }            \
    default:                                                                 \
      TORCH_CHECK(false, "group_norm: float32, float16 or bfloat16 expected"); \
  }

}  // namespace

// -> y, mean [B, G], rstd [B, G]
std::vector<at::Tensor> group_norm_forward(
    at::Tensor x, int64_t groups, c10::optional<at::Tensor> weight,
    c10::optional<at::Tensor> bias, double eps, int64_t act, double p,
    c10::optional<at::Tensor> rng, int64_t seed, int64_t offset) {
  const Shape s = shape_of(x, groups);
  TORCH_CHECK(eps > 0.0, "group_norm: eps must be positive");
  c10::DeviceGuard guard(x.device());
  const DropoutArgs d = dropout_args(p, rng, seed, offset, x);
  const float* w = param(weight, x, "weight");
  const float* b = param(bias, x, "bias");
  auto y = at::empty_like(x, x.options(), at::MemoryFormat::ChannelsLast);
  auto mean = at::empty({x.size(0), groups}, x.options().dtype(at::kFloat));
  auto rstd = at::empty_like(mean);
  if (x.numel() == 0) {
    mean.zero_();
    rstd.zero_();
    return {y, mean, rstd};
  }
  GN_TYPE(x.scalar_type(),
          forward<T>(x, y, w, b, mean, rstd, s, (float)eps, (int)act, d));
  return {y, mean, rstd};
}

// -> dx, dweight, dbias; an undefined tensor where none is wanted
std::vector<at::Tensor> group_norm_backward(
    at::Tensor gy, at::Tensor x, c10::optional<at::Tensor> weight,
    c10::optional<at::Tensor> bias, at::Tensor mean, at::Tensor rstd,
    int64_t act, double p, c10::optional<at::Tensor> rng, int64_t seed,
    int64_t offset, bool need_x, bool need_weight, bool need_bias) {
  const Shape s = shape_of(x, mean.size(1));
  TORCH_CHECK(gy.sizes() == x.sizes() && gy.scalar_type() == x.scalar_type() &&
                  gy.device() == x.device() &&
                  gy.is_contiguous(at::MemoryFormat::ChannelsLast),
              "group_norm: gy must be like x");
  for (const auto& t : {mean, rstd})
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous() &&
                    t.dim() == 2 && t.size(0) == x.size(0) &&
                    t.size(1) == mean.size(1) && t.device() == x.device(),
                "group_norm: mean and rstd must be [B, G] floats");
  c10::DeviceGuard guard(x.device());
  const DropoutArgs d = dropout_args(p, rng, seed, offset, x);
  const float* w = param(weight, x, "weight");
  const float* b = param(bias, x, "bias");
  at::Tensor dx, dw, db;
  const auto opts = x.options().dtype(at::kFloat);
  if (need_x) dx = at::empty_like(x, x.options(), at::MemoryFormat::ChannelsLast);
  if (need_weight) dw = at::empty({x.size(1)}, opts);
  if (need_bias) db = at::empty({x.size(1)}, opts);
  if (x.numel() == 0) {
    if (need_weight) dw.zero_();
    if (need_bias) db.zero_();
    return {dx, dw, db};
  }
  if (!need_x && !need_weight && !need_bias) return {dx, dw, db};
  GN_TYPE(x.scalar_type(),
          backward<T>(x, gy, need_x ? (T*)dx.data_ptr() : nullptr, w, b,
                      mean.data_ptr<float>(), rstd.data_ptr<float>(),
                      need_bias ? db.data_ptr<float>() : nullptr,
                      need_weight ? dw.data_ptr<float>() : nullptr, s,
                      (int)act, d));
  return {dx, dw, db};
}
