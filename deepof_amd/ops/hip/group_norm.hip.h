// Group normalisation + affine + activation (+ dropout), channels last, for
// gfx950: the kernels and their launches, for one type of values per file that
// includes this.
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
//  - tile: where a bundle of whole groups of a sample fits into half a CU's
//    LDS, a block keeps it there, so that x (and gy) are read once, in one
//    launch each way;
//  - split: else pixels are dealt to blocks, which leave partial sums, and the
//    last launch reads x (and gy) again: three launches forwards (sums, their
//    join, y), two backwards (sums, whose last blocks join them; dx).
// 64x64x192x256 bf16 with ELU (403 MB a tensor; 1.6 GB is the least that
// forward and backward move, 3.2 GB is what the split route does): sums 118 us,
// join 5, y 117; sums 194, dx 183: 5.2 TB/s over all, what a large copy reaches
// here, the sums below it and the others above.  8x24x32x512 bf16 (tile; 6.3
// MB): 9.8 us forwards, 13.3 backwards, most of it launch, first loads and the
// sums' three meetings in LDS.
// Keeping larger samples on the chip, a team of blocks each with its tile, was
// built and measured too: a team's meeting costs its blocks some 20 us, in
// which a CU's LDS holds far less than memory moves, and 64x64x192x256 bf16
// took 390 us forwards against 290 of the split route then.
//
// Sums have a fixed order everywhere, whichever block ends them: results are
// equal every time.

#pragma once

#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>
#include <torch/extension.h>

#include <algorithm>
#include <numeric>

#include "group_norm.h"
#include "philox.hip.h"
#include "vec.hip.h"

namespace {

constexpr int WAVE = 64;
constexpr int XCDS = 8;           // blocks go to them in turn, each with an L2
constexpr int THREADS = 512;      // of a block that sums
constexpr int BLOCK = 256;        // of a block that does not
using Shape = GroupNormShape;

// A sample's pixels dealt to n blocks: batches of `batch` pixels, of which
// block i takes i, i + n, ...  Blocks that run together then read neighbouring
// memory.  Forward sums of 403 MB take 109 us behind kernels that only read and
// 118 behind one that wrote; with a long piece per block they took 113.  Reading
// alone takes 62 to 71: a wave asks for its next batch only once it has summed
// the one before, which is the likely reason for the rest.
struct Deal {
  int n, batch, batches, missing;  // missing: pixels that the last batch lacks
  __device__ __forceinline__ int pixels(int i) const {
    const int k = (batches - i + n - 1) / n;
    return k * batch - ((batches - 1) % n == i ? missing : 0);
  }
  __device__ __forceinline__ int length(int k) const {  // of batch k
    return batch - (k == batches - 1 ? missing : 0);
  }
  // whether a block has more than `most` batches
  __host__ __device__ __forceinline__ bool more_than(int most) const {
    return batches > (int64_t)n * most;
  }
};

// v + v of another lane: DPP moves within 16 lanes and between them, without
// the journey through LDS that a shuffle takes.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(
                 0, __float_as_int(v), CTRL, ROWS, 0xf, true));
}

// The sum over a wave, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
  v = dpp_add<0xb1, 0xf>(v);   // lanes 1, 0, 3, 2
  v = dpp_add<0x4e, 0xf>(v);   // lanes 2, 3, 0, 1
  v = dpp_add<0x141, 0xf>(v);  // 8 lanes mirrored
  v = dpp_add<0x140, 0xf>(v);  // 16 lanes mirrored
  // the last lane of row 0 to row 1, of 2 to 3; then of rows 0, 1 to 2, 3
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x142,
                                                  0xa, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x143,
                                                  0xc, 0xf, false));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// a / b for 0 <= a < 2^20, b > 0, by a reciprocal: (a + 1/2) / b is at least
// 1 / (2 b) from the next integer, and off by less.
__device__ __forceinline__ int small_div(int a, int b) {
  return (int)(((float)a + 0.5f) * __builtin_amdgcn_rcpf((float)b));
}

// f(j, group of channel ch + j) for j < V, with one division.
template <int V, typename F>
__device__ __forceinline__ void each_group(int ch, int cg, F f) {
  int g = small_div(ch, cg), r = ch - g * cg;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    f(j, g);
    if (++r == cg) {
      r = 0;
      ++g;
    }
  }
}

// Squares that rounding has left below 0; what is no number stays none, so
// that squares beyond fp32 do not pass for a small variance.
__device__ __forceinline__ float not_below_0(float v) {
  return v < 0.0f ? 0.0f : v;
}

__device__ __forceinline__ float rstd_of(float m2, float n, float eps) {
  return 1.0f / sqrtf(m2 / n + eps);
}

// Which part of some pixels by `cols` columns of V channels a thread works
// on: one column, pixels row, row + rows, ...
struct Place {
  int cols, rows, row, col;
  bool on;
  __device__ __forceinline__ Place(int cols_, int threads) : cols(cols_) {
    rows = small_div(threads, cols);
    row = small_div(threadIdx.x, cols);
    col = threadIdx.x - row * cols;
    on = row < rows;
  }
  // pixels of this row among `pixels`
  __device__ __forceinline__ int count(int pixels) const {
    return on && row < pixels ? (pixels - row + rows - 1) / rows : 0;
  }
};

// ---------------------------------------------------------------------------
// sums over a block
// ---------------------------------------------------------------------------
// A thread's V sums, one per channel, are first added up within the groups
// that its vector touches: `units` of them, V / units channels each.  red
// holds [thread][units] of F, float or float2.
__device__ __forceinline__ void add_to(float& a, float b) { a += b; }
__device__ __forceinline__ void add_to(float2& a, float2 b) {
  a.x += b.x;
  a.y += b.y;
}
// One of many additions, as many as there are samples: what its rounding loses
// goes into the next (Kahan's sum).
__device__ __forceinline__ void add_kept(float& sum, float& lost, float v) {
  v -= lost;
  const float next = sum + v;
  lost = (next - sum) - v;
  sum = next;
}
__device__ __forceinline__ float over_wave(float v) { return wave_sum(v); }
__device__ __forceinline__ float2 over_wave(float2 v) {
  return make_float2(wave_sum(v.x), wave_sum(v.y));
}

template <int V, typename F>
__device__ __forceinline__ void put_units(F* red, int units, const F (&s)[V]) {
  F* at = red + threadIdx.x * units;
  if (units == V) {
#pragma unroll
    for (int j = 0; j < V; ++j) at[j] = s[j];
  } else if (units == 1) {
    F t = s[0];
#pragma unroll
    for (int j = 1; j < V; ++j) add_to(t, s[j]);
    at[0] = t;
  } else if (units == 2) {
    F t0 = s[0], t1 = s[V / 2];
#pragma unroll
    for (int j = 1; j < V / 2; ++j) {
      add_to(t0, s[j]);
      add_to(t1, s[V / 2 + j]);
    }
    at[0] = t0;
    at[1] = t1;
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      F t = s[j];
      add_to(t, s[j + (V > 1)]);
      at[j / 2] = t;
    }
  }
}

// Sums red over the rows and over each group's units.  A row is `width` =
// cols * units entries, of which unit `first` is the first in a group of `upg`
// units; groups g0 .. lie in the row, possibly cut off at its ends.
// done(group, sum) is called by one lane.
template <typename F, typename Done>
__device__ __forceinline__ void sum_groups(const F* red, const Place& pl,
                                           int width, int first, int upg,
                                           Done done) {
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int last = first + width;
  for (int g = small_div(first, upg) + wave; g * upg < last;
       g += THREADS / WAVE) {
    const int lo = max(g * upg, first) - first;
    const int here = min((g + 1) * upg, last) - first - lo;
    // a lane's next entry is 64 further: so many rows and so many units
    const int skip_r = small_div(WAVE, here), skip_u = WAVE - skip_r * here;
    int r = small_div(lane, here), u = lane - r * here;
    F sum{};
    while (r < pl.rows) {
      add_to(sum, red[r * width + lo + u]);
      r += skip_r;
      u += skip_u;
      if (u >= here) {
        u -= here;
        ++r;
      }
    }
    sum = over_wave(sum);
    if (lane == 0) done(g, sum);
  }
}

// A thread's mean and squares about it, per channel.  Values are summed in runs
// about what the mean was before the run, the first about the thread's first
// value, and the runs are joined: a mean far from 0 costs no digits, as
// differences alone are summed.  The first value may itself lie far from all
// others, so the first run is short, and later ones are about a mean that has
// left it behind.  (One sum of squares about the first value adds up nearly
// equal numbers then, whose roundings all go one way: of 768 values, 0 but for
// the first, it had the variance wrong by 2e-2, and this by 1e-6.)
constexpr int FIRST_RUN = 8, RUN = 64;  // multiples of what walk loads ahead

template <int V>
struct Moments {
  float mean[V], rest[V];  // the mean is their sum: rest is mean's rounding
  float m2[V];             // squares about it
  float s1[V], s2[V];      // of the run, about mean
  int n, run;              // values joined, and in the run
  __device__ __forceinline__ void begin() {
    n = run = 0;
#pragma unroll
    for (int j = 0; j < V; ++j)
      mean[j] = rest[j] = m2[j] = s1[j] = s2[j] = 0.0f;
  }
  __device__ __forceinline__ void about(const float (&v)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) mean[j] = v[j];
  }
  __device__ __forceinline__ void add(const float (&v)[V]) {
    ++run;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = v[j] - mean[j];
      s1[j] += d;
      s2[j] = fmaf(d, d, s2[j]);
    }
  }
  __device__ __forceinline__ void join() {
    if (run == 0) return;
    const float a = (float)n, b = (float)run;
    const float inv = __builtin_amdgcn_rcpf(b);
    const float share = b * __builtin_amdgcn_rcpf(a + b);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float e = s1[j] * inv;     // the run's mean, less mean
      const float d = e - rest[j];     // less the mean before it
      m2[j] += fmaf(d * d, a * share, not_below_0(s2[j] - s1[j] * e));
      const float t = fmaf(d, share, rest[j]);
      const float m = mean[j] + t;
      rest[j] = t - (m - mean[j]);
      mean[j] = m;
      s1[j] = s2[j] = 0.0f;
    }
    n += run;
    run = 0;
  }
  // The value with this index, counted by the caller, ends a run.
  __device__ __forceinline__ static bool ends(int i) {
    return i == FIRST_RUN - 1 || i % RUN == RUN - 1;
  }
};

// Joins the threads' moments.  Two rounds of sums: first the groups' means,
// into mean[g]; then what rounding left of them (about the first result,
// nothing cancels) and the squares about it.  fold(g, mean, squares) is called
// by one lane per group that has values here, n_of(g) many, and decides what
// becomes of them.  red: THREADS * units float2.
template <int V, typename Count, typename Fold>
__device__ __forceinline__ void join_moments(Moments<V>& t, int count,
                                             float2* red, float* mean,
                                             const Place& pl, int c0, int cg,
                                             int units, Count n_of,
                                             Fold fold) {
  const int per = V / units;
  const int first = c0 / per, upg = cg / per, width = pl.cols * units;
  const float n = (float)count;
  float* red1 = reinterpret_cast<float*>(red);
  float a[V];
  t.join();
#pragma unroll
  for (int j = 0; j < V; ++j) a[j] = n * t.mean[j];
  if (pl.on) put_units<V>(red1, units, a);
  __syncthreads();
  sum_groups(red1, pl, width, first, upg,
             [&](int g, float sum) { mean[g] = sum / n_of(g); });
  __syncthreads();
  if (pl.on) {
    float2 q[V];
    each_group<V>(c0 + pl.col * V, cg, [&](int j, int g) {
      const float e = t.mean[j] - mean[g];
      q[j] = make_float2(n * e, fmaf(n * e, e, t.m2[j]));
    });
    if (count == 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) q[j] = make_float2(0.0f, 0.0f);
    }
    put_units<V>(red, units, q);
  }
  __syncthreads();
  sum_groups(red, pl, width, first, upg, [&](int g, float2 sum) {
    const float shift = sum.x / n_of(g);
    fold(g, mean[g] + shift, not_below_0(sum.y - sum.x * shift));
  });
  __syncthreads();
}

// Sums over the rows of a block, channel by channel.  Threads bring s1 and s2
// of their V channels; out1[c] and out2[c] (LDS) get the totals of the row's
// channels.  In rounds of up to 4 channels; red: RED_CHANNELS(V) floats.
constexpr int ROUND(int v) { return v < 4 ? v : 4; }
constexpr int RED_CHANNELS(int v) { return THREADS * 2 * ROUND(v); }

template <int V>
__device__ __forceinline__ void sum_channels(float* red, const Place& pl,
                                             const float (&s1)[V],
                                             const float (&s2)[V], float* out1,
                                             float* out2) {
  constexpr int R = ROUND(V);
  const int items = pl.cols * 2 * R;   // sums of a row
  const int subs = min(THREADS / items, pl.rows);
  const int sub = threadIdx.x / items, item = threadIdx.x - sub * items;
#pragma unroll
  for (int j = 0; j < V; j += R) {
    auto leave = [&](int i, float t) {
      const int col = i / (2 * R), q = i % (2 * R);
      (q < R ? out1 : out2)[col * V + j + q % R] = t;
    };
    if (pl.on) {
      Pack<float, 2 * R> v;
#pragma unroll
      for (int q = 0; q < R; ++q) {
        v.v[q] = s1[j + q];
        v.v[R + q] = s2[j + q];
      }
      store_pack<float, 2 * R>(red + threadIdx.x * 2 * R, v);
    }
    __syncthreads();
    if (subs <= 1) {  // few rows
      for (int i = threadIdx.x; i < items; i += THREADS) {
        float t = 0.0f;
        for (int r = 0; r < pl.rows; ++r) t += red[r * items + i];
        leave(i, t);
      }
    } else {  // a thread sums a share of an item's rows, then the shares
      float t = 0.0f;
      if (sub < subs) {
#pragma unroll 4
        for (int r = sub; r < pl.rows; r += subs) t += red[r * items + item];
      }
      __syncthreads();
      if (sub < subs) red[threadIdx.x] = t;
      __syncthreads();
      if ((int)threadIdx.x < items) {
        t = 0.0f;
#pragma unroll 4
        for (int q = 0; q < subs; ++q) t += red[q * items + threadIdx.x];
        leave(threadIdx.x, t);
      }
    }
    __syncthreads();
  }
}

// Channel sums s1[c], s2[c] (LDS, channels first .. first + width of C) ->
// the groups' sums weighted by w; fold(g, s1, s2) is called by one lane.
template <typename Fold>
__device__ __forceinline__ void weigh_groups(const float* s1, const float* s2,
                                             const float* __restrict__ w,
                                             int first, int width, int cg,
                                             Fold fold) {
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int last = first + width;
  for (int g = small_div(first, cg) + wave; g * cg < last;
       g += THREADS / WAVE) {
    const int lo = max(g * cg, first), hi = min((g + 1) * cg, last);
    float a = 0.0f, c = 0.0f;
    for (int i = lo + lane; i < hi; i += WAVE) {
      const float wi = w ? w[i] : 1.0f;
      a = fmaf(wi, s1[i - first], a);
      c = fmaf(wi, s2[i - first], c);
    }
    a = wave_sum(a);
    c = wave_sum(c);
    if (lane == 0) fold(g, a, c);
  }
}

// ---------------------------------------------------------------------------
// values
// ---------------------------------------------------------------------------
template <int V>
__device__ __forceinline__ void load_floats(float (&v)[V], const float* at) {
  const Pack<float, V> p = load_pack<float, V>(at);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = p.v[j];
}

// z = (x - m) a + o, per channel of a thread's vector: a = rstd w, o = b.
// Parameters first: they can be on their way while statistics are not known.
template <int V>
struct Affine {
  float m[V], a[V], o[V];
  __device__ __forceinline__ void params(int ch, const float* __restrict__ w,
                                         const float* __restrict__ bias) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      a[j] = 1.0f;
      o[j] = 0.0f;
    }
    if (w) load_floats<V>(a, w + ch);
    if (bias) load_floats<V>(o, bias + ch);
  }
  // from [2][b][c] of mean and rstd w
  __device__ __forceinline__ void channels(const float* chan, int64_t plane,
                                           const float* __restrict__ bias,
                                           int ch) {
    load_floats<V>(m, chan);
    load_floats<V>(a, chan + plane);
    if (bias) {
      load_floats<V>(o, bias + ch);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = 0.0f;
    }
  }
  // indexed by group; channel ch is the thread's first
  __device__ __forceinline__ void stats(int ch, int cg, const float* mean,
                                        const float* rstd) {
    each_group<V>(ch, cg, [&](int j, int g) {
      m[j] = mean[g];
      a[j] *= rstd[g];
    });
  }
};

template <typename T, int V, int ACT, bool DROP>
__device__ __forceinline__ Pack<T, V> forward_value(
    const Affine<V>& k, const Pack<T, V>& raw, int act, const DropoutArgs& d,
    const DropoutState& st, uint64_t at) {
  float v[V];
  unpack<T, V>(raw, v);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = fmaf(v[j] - k.m[j], k.a[j], k.o[j]);
  act_apply<T, ACT, V>(act, v);
  if (DROP && d.on) dropout_apply<V>(d, st, at, v);
  return pack<T, V>(v);
}

// (x, gy) -> (x - mean, gz)
template <typename T, int V, int ACT, bool DROP>
__device__ __forceinline__ void through(const Affine<V>& k,
                                        const Pack<T, V>& rx,
                                        const Pack<T, V>& rg, int act,
                                        const DropoutArgs& d,
                                        const DropoutState& st, uint64_t at,
                                        float (&e)[V], float (&g)[V]) {
  unpack<T, V>(rx, e);
  unpack<T, V>(rg, g);
  float z[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    e[j] -= k.m[j];
    z[j] = fmaf(e[j], k.a[j], k.o[j]);
  }
  act_backward<T, ACT, V>(act, z, g);
  if (DROP && d.on) dropout_apply<V>(d, st, at, g);
}

// Vectors that a thread asks for at once, of one tensor or of each of two.
template <typename T>
constexpr int AHEAD1 = sizeof(T) == 2 ? 4 : 2;
template <typename T>
constexpr int AHEAD2 = sizeof(T) == 2 ? 4 : 2;

template <typename T, int V>
struct Both {
  Pack<T, V> x, g;
};

// use(i, load(i)) for i < count, D loads ahead of their uses.  Loads stand
// under no branch, or each would be waited for before the next: load(i, false)
// is asked for something harmless past the end.
template <int D, typename Load, typename Use>
__device__ __forceinline__ void walk(int count, Load load, Use use) {
  int i = 0;
  for (; i + D <= count; i += D) {
    decltype(load(0, true)) raw[D];
#pragma unroll
    for (int q = 0; q < D; ++q) raw[q] = load(i + q, true);
#pragma unroll
    for (int q = 0; q < D; ++q) use(i + q, raw[q]);
  }
  if (i < count) {
    decltype(load(0, true)) raw[D - 1 > 0 ? D - 1 : 1];
#pragma unroll
    for (int q = 0; q < D - 1; ++q) raw[q] = load(i + q, i + q < count);
#pragma unroll
    for (int q = 0; q < D - 1; ++q)
      if (i + q < count) use(i + q, raw[q]);
  }
}

// ---------------------------------------------------------------------------
// the last block
// ---------------------------------------------------------------------------
// Blocks that work on one sum leave their parts, and the last of them to come
// adds all up, in an order that does not depend on which one that is.  Nobody
// waits.  The parts go through atomics of agent scope, past the L2s that XCDs
// do not share.  Counters are 0 before a launch: the forward launch has cleared
// them, and a last block leaves its own at 0 again.
__device__ __forceinline__ void put2(uint64_t* at, float a, float b) {
  const uint64_t v =
      (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32;
  __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ float2 get2(const uint64_t* at) {
  const uint64_t v =
      __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((uint32_t)v),
                     __uint_as_float((uint32_t)(v >> 32)));
}

// Whether this block is the last of `blocks`.  All its threads call it; their
// put2 calls are done before it counts.  flag: LDS.
//
// What orders parts and count is this machine, not the language: put2's stores
// and get2's loads go to where all XCDs meet, every wave has waited for its
// stores (vmcnt counts them until they are there) before the barrier behind
// which thread 0 counts, and loads stand behind the count's return and another
// barrier.  Counting with acquire and release at agent scope says as much, but
// writes back and drops an L2's lines at every count: 8x24x32x512 bf16 took
// 19.2 us backwards with it, not 13.2, and the sums of 64x64x192x256 205, not
// 194.
__device__ __forceinline__ bool last_of(int blocks, uint32_t* count,
                                        int* flag) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (blocks == 1) return true;
  if (threadIdx.x == 0) {
    const bool last = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED,
                                             __HIP_MEMORY_SCOPE_AGENT) ==
                      (uint32_t)(blocks - 1);
    if (last)
      __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = last;
  }
  __syncthreads();
  return *flag != 0;
}

// Every block of a forward launch clears its share of n counters.
__device__ __forceinline__ void clear_counts(uint32_t* count, int n) {
  if (!count) return;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x)
    count[i] = 0;
}

// ---------------------------------------------------------------------------
// tile route
// ---------------------------------------------------------------------------
// Tiles narrower than a cache line share lines with their neighbours.  Block
// i's tile is so chosen that neighbours go to the same XCD, whose L2 then
// fetches a line once, and writes it back whole.  (8x24x32x512 bf16, spans of
// 32 bytes: forwards 12.0 us without and 9.2 with, backwards 16.2 and 11.4.)
__device__ __forceinline__ int neighbours_together(int i, int n) {
  const int each = n / XCDS;
  return i < each * XCDS ? (i % XCDS) * each + i / XCDS : i;
}

struct Tiles {
  int span, spans;  // channels of a tile, tiles of a sample
  int groups;       // groups of a tile
  int iters;        // vectors per thread
};

// Threads of a channel that share its samples in a span's last block.
__host__ __device__ __forceinline__ int sample_shares(int span) {
  return THREADS > span ? THREADS / span : 1;
}

// LDS: the tile, red, then floats per group.
template <typename T, int V, int ACT, bool DROP>
__global__ __launch_bounds__(THREADS, 4) void gn_tile(
    const T* __restrict__ x, T* __restrict__ y, const float* __restrict__ w,
    const float* __restrict__ bias, float* __restrict__ mean_out,
    float* __restrict__ rstd_out, uint32_t* __restrict__ counts, int n_counts,
    Shape s, Tiles tiles, int units, float eps, int act, DropoutArgs d) {
  extern __shared__ char lds[];
  clear_counts(counts, n_counts);
  Pack<T, V>* slots = reinterpret_cast<Pack<T, V>*>(lds);
  float2* red = reinterpret_cast<float2*>(slots + tiles.iters * THREADS);
  float* mean = reinterpret_cast<float*>(red + THREADS * units);
  float* rstd = mean + tiles.groups;
  const int at_tile = neighbours_together(blockIdx.x, gridDim.x);
  const int span = at_tile % tiles.spans, b = at_tile / tiles.spans;
  const Place pl(tiles.span / V, THREADS);
  const int ch = span * tiles.span + pl.col * V;  // the thread's first channel
  const int64_t from = ((int64_t)b * s.hw + pl.row) * s.c + ch;
  const int64_t next = (int64_t)pl.rows * s.c;
  const int count = pl.count((int)s.hw);

  Moments<V> t;
  t.begin();
  Affine<V> k;
  if (count) {
    k.params(ch, w, bias);
    walk<AHEAD1<T>>(count, [&](int i, bool in) {
      return load_pack<T, V>(x + from + (in ? i * next : 0));
    }, [&](int i, const Pack<T, V>& raw) {
      slots[i * THREADS + threadIdx.x] = raw;
      float v[V];
      unpack<T, V>(raw, v);
      if (i == 0) t.about(v);
      t.add(v);
      if (t.ends(i)) t.join();
    });
  }
  const float n = (float)s.hw * (float)s.cg;
  join_moments<V>(t, count, red, mean, pl, 0, s.cg, units,
                  [&](int) { return n; },
                  [&](int g, float m, float m2) {
                    const float r = rstd_of(m2, n, eps);
                    mean[g] = m;
                    rstd[g] = r;
                    if (mean_out) {
                      const int64_t at =
                          (int64_t)b * s.g + span * tiles.groups + g;
                      mean_out[at] = m;
                      rstd_out[at] = r;
                    }
                  });
  if (count == 0) return;
  const DropoutState st = dropout_state(d);
  k.stats(pl.col * V, s.cg, mean, rstd);
  for (int i = 0; i < count; ++i) {
    const int64_t at = from + i * next;
    store_pack<T, V>(y + at,
                     forward_value<T, V, ACT, DROP>(
                         k, slots[i * THREADS + threadIdx.x], act, d, st,
                         (uint64_t)at));
  }
}

// LDS: x's and gy's tiles, red, then floats per channel and per group.
// sums_c: [b][c] of the samples' sums of gz and gz xhat, which the last block
// of a span adds up to the parameters' gradients; null: none is asked for.
// counts null: they are left as [2][b][c] for gn_param_grad.
template <typename T, int V, int ACT, bool DROP>
__global__ __launch_bounds__(THREADS, 4) void gn_bwd_tile(
    const T* __restrict__ x, const T* __restrict__ gy, T* __restrict__ dx,
    const float* __restrict__ w, const float* __restrict__ bias,
    const float* __restrict__ mean, const float* __restrict__ rstd,
    uint64_t* __restrict__ sums_c, uint32_t* __restrict__ counts,
    float* __restrict__ db, float* __restrict__ dw, Shape s, Tiles tiles,
    int act, DropoutArgs d) {
  extern __shared__ char lds[];
  Pack<T, V>* slots = reinterpret_cast<Pack<T, V>*>(lds);
  const int slot_g = tiles.iters * THREADS;  // gy's slots behind x's
  float* red = reinterpret_cast<float*>(slots + 2 * slot_g);
  float* sum1 = red + RED_CHANNELS(V);
  float* sum2 = sum1 + tiles.span;
  float* t1 = sum2 + tiles.span;
  float* t2 = t1 + tiles.groups;
  int* flag = reinterpret_cast<int*>(t2 + tiles.groups);
  const int at_tile = neighbours_together(blockIdx.x, gridDim.x);
  const int span = at_tile % tiles.spans, b = at_tile / tiles.spans;
  const Place pl(tiles.span / V, THREADS);
  const int c0 = span * tiles.span, ch = c0 + pl.col * V;
  const int64_t from = ((int64_t)b * s.hw + pl.row) * s.c + ch;
  const int64_t next = (int64_t)pl.rows * s.c;
  const int count = pl.count((int)s.hw);
  const DropoutState st = dropout_state(d);
  mean += (int64_t)b * s.g;
  rstd += (int64_t)b * s.g;
  Affine<V> k;

  float s1[V], s2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0f;
  if (count) {
    k.params(ch, w, bias);
    k.stats(ch, s.cg, mean, rstd);
    walk<AHEAD2<T> / 2>(count, [&](int i, bool in) {
      const int64_t at = from + (in ? i * next : 0);
      return Both<T, V>{load_pack<T, V>(x + at), load_pack<T, V>(gy + at)};
    }, [&](int i, const Both<T, V>& raw) {
      slots[i * THREADS + threadIdx.x] = raw.x;
      slots[slot_g + i * THREADS + threadIdx.x] = raw.g;
      float e[V], g[V];
      through<T, V, ACT, DROP>(k, raw.x, raw.g, act, d, st,
                               (uint64_t)(from + i * next), e, g);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s1[j] += g[j];
        s2[j] = fmaf(g[j], e[j], s2[j]);
      }
    });
  }
  if (count)
    each_group<V>(ch, s.cg, [&](int j, int g) { s2[j] *= rstd[g]; });
  sum_channels<V>(red, pl, s1, s2, sum1, sum2);
  const float inv_n = 1.0f / ((float)s.hw * (float)s.cg);
  weigh_groups(sum1, sum2, w, c0, tiles.span, s.cg,
               [&](int g, float a, float c) {
                 const float r = rstd[g];
                 t1[g - span * tiles.groups] = -r * (a * inv_n);
                 t2[g - span * tiles.groups] = -r * r * (c * inv_n);
               });
  if (sums_c) {
    const int64_t at = (int64_t)b * s.c + c0;
    float* part = reinterpret_cast<float*>(sums_c) + at;
    for (int c = threadIdx.x; c < tiles.span; c += THREADS) {
      if (counts) {
        put2(sums_c + at + c, sum1[c], sum2[c]);
      } else {
        part[c] = sum1[c];
        part[(int64_t)s.b * s.c + c] = sum2[c];
      }
    }
  }
  __syncthreads();
  if (dx && count) {
    float m1[V], m2[V];
    each_group<V>(pl.col * V, s.cg, [&](int j, int g) {
      m1[j] = t1[g];
      m2[j] = t2[g];
    });
    for (int i = 0; i < count; ++i) {
      const int64_t at = from + i * next;
      float e[V], g[V];
      through<T, V, ACT, DROP>(k, slots[i * THREADS + threadIdx.x],
                               slots[slot_g + i * THREADS + threadIdx.x], act,
                               d, st, (uint64_t)at, e, g);
#pragma unroll
      for (int j = 0; j < V; ++j)
        g[j] = fmaf(k.a[j], g[j], fmaf(e[j], m2[j], m1[j]));
      store_pack<T, V>(dx + at, pack<T, V>(g));
    }
  }
  if (!sums_c || !counts || !last_of(s.b, counts + span, flag)) return;
  // samples dealt in `shares` to threads that lie a span apart
  const int shares = sample_shares(tiles.span);
  const int share = shares > 1 ? small_div(threadIdx.x, tiles.span) : 0;
  float2* red2 = reinterpret_cast<float2*>(red);
  for (int c1 = 0; c1 < tiles.span; c1 += THREADS) {
    const int c = c1 + threadIdx.x - share * tiles.span;
    const bool in = c < tiles.span && share < shares;
    float2 sum = make_float2(0.0f, 0.0f), lost = sum;
    if (in) {
      const uint64_t* at = sums_c + c0 + c;
      constexpr int D = 8;  // asked for at once
      for (int i = share; i < s.b; i += D * shares) {
        float2 v[D];
#pragma unroll
        for (int q = 0; q < D; ++q)
          v[q] = get2(at + (int64_t)min(i + q * shares, s.b - 1) * s.c);
#pragma unroll
        for (int q = 0; q < D; ++q) {
          if (i + q * shares >= s.b) v[q] = make_float2(0.0f, 0.0f);
          add_kept(sum.x, lost.x, v[q].x);
          add_kept(sum.y, lost.y, v[q].y);
        }
      }
    }
    red2[threadIdx.x] = sum;
    __syncthreads();
    if (in && share == 0) {
      for (int q = 1; q < shares; ++q) add_to(sum, red2[q * tiles.span + c]);
      if (db) db[c0 + c] = sum.x;
      if (dw) dw[c0 + c] = sum.y;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// split route
// ---------------------------------------------------------------------------
// Block (split, sample).  part: [b][g][splits] of (mean, M2); n follows from
// the split's bounds.  Rows wider than a block are taken in chunks of columns,
// and groups that reach over chunks are joined as they come.
template <typename T, int V>
__global__ __launch_bounds__(THREADS, 4) void gn_stats(
    const T* __restrict__ x, float2* __restrict__ part,
    uint32_t* __restrict__ counts, int n_counts, Shape s, Deal deal,
    int units) {
  clear_counts(counts, n_counts);
  constexpr int D = AHEAD1<T>;
  __shared__ float2 red[THREADS * V];
  extern __shared__ float joined[];  // [4][g]: work space, then n, mean, M2
  float* mean = joined;
  float* jn = mean + s.g;
  float* jm = jn + s.g;
  float* jq = jm + s.g;
  const int split = blockIdx.x % deal.n, b = blockIdx.x / deal.n;
  const int pixels = deal.pixels(split);
  const T* base = x + (int64_t)b * s.hw * s.c;
  for (int c0 = 0; c0 < s.c; c0 += THREADS * V) {
    const Place pl(min(THREADS, (s.c - c0) / V), THREADS);
    const int64_t next = (int64_t)pl.rows * s.c;
    int count = 0, batch = 0;
    Moments<V> t;
    t.begin();
    for (int k = split; k < deal.batches; k += deal.n, ++batch) {
      const int here = pl.count(deal.length(k));
      const T* at = base + ((int64_t)k * deal.batch + pl.row) * s.c + c0 +
                    pl.col * V;
      walk<D>(here, [&](int i, bool in) {
        return load_pack<T, V>(at + (in ? i * next : 0));
      }, [&](int i, const Pack<T, V>& raw) {
        float v[V];
        unpack<T, V>(raw, v);
        if (i == 0 && batch == 0) t.about(v);
        t.add(v);
      });
      if (t.ends(batch * D + D - 1)) t.join();
      count += here;
    }
    const int last = c0 + pl.cols * V;
    // values of group g in this chunk
    auto n_of = [&](int g) {
      return (float)(min((g + 1) * s.cg, last) - max(g * s.cg, c0)) *
             (float)pixels;
    };
    join_moments<V>(t, count, red, mean, pl, c0, s.cg, units, n_of,
                    [&](int g, float m, float q) {
                      float n = n_of(g);
                      if (g * s.cg < c0) {  // begun in an earlier chunk
                        const float d = m - jm[g], sum = jn[g] + n;
                        q += jq[g] + d * d * (jn[g] * n / sum);
                        m = jm[g] + d * (n / sum);
                        n = sum;
                      }
                      jn[g] = n;
                      jm[g] = m;
                      jq[g] = q;
                    });
  }
  for (int g = threadIdx.x; g < s.g; g += THREADS)
    part[((int64_t)b * s.g + g) * deal.n + split] = make_float2(jm[g], jq[g]);
}

// A group's partial sums are joined by `lanes` neighbouring threads, a power of
// two and at most a wave, with up to MOST of them each: all are asked for at
// once, and kept for a second pass.
constexpr int MOST = 4;
constexpr int MOST_PARTS = MOST * WAVE;

struct Share {
  int lanes, lane, group;   // group: among this block's
  int groups, blocks;       // of a block, of a sample
};

__host__ __device__ __forceinline__ int share_lanes(int parts) {
  int lanes = 1;
  while (lanes * MOST < parts) lanes *= 2;
  return lanes;
}

__device__ __forceinline__ Share share_of(int lanes, int groups) {
  Share sh;
  sh.lanes = lanes;
  sh.lane = threadIdx.x & (lanes - 1);
  sh.groups = THREADS / lanes;
  sh.group = threadIdx.x / lanes;
  sh.blocks = (groups + sh.groups - 1) / sh.groups;
  return sh;
}

__device__ __forceinline__ float share_sum(int lanes, float v) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE);
  return v;
}

// This thread's parts of e[0 .. n); zeros past the end.
__device__ __forceinline__ void share_load(const Share& sh, const float2* e,
                                           int n, float2 (&v)[MOST]) {
#pragma unroll
  for (int q = 0; q < MOST; ++q) {
    const int i = sh.lane + q * sh.lanes;
    v[q] = i < n ? e[i] : make_float2(0.0f, 0.0f);
  }
}

// Block (groups, sample): joins the splits' statistics, the mean first, about
// split 0's, then squares about it.  stat: [2][b][g] mean and rstd, kept for
// the way back, or null.  chan: [2][b][c], mean and rstd w of every channel,
// which the next launch's threads load as vectors.
__global__ __launch_bounds__(THREADS) void gn_join(
    const float2* __restrict__ part, const float* __restrict__ w,
    float* __restrict__ stat, float* __restrict__ chan, Shape s, Deal deal,
    int lanes, float eps) {
  __shared__ float sums[2][THREADS];
  const Share sh = share_of(lanes, s.g);
  const int b = blockIdx.x / sh.blocks;
  const int g0 = (blockIdx.x - b * sh.blocks) * sh.groups;
  const int g = g0 + sh.group;
  if (g < s.g) {
    const float2* e = part + ((int64_t)b * s.g + g) * deal.n;
    float2 v[MOST];
    share_load(sh, e, deal.n, v);
    const float ref = e[0].x;
    float n[MOST], sm = 0.0f, sq = 0.0f;
#pragma unroll
    for (int q = 0; q < MOST; ++q) {
      const int i = sh.lane + q * sh.lanes;
      n[q] = i < deal.n ? (float)deal.pixels(i) : 0.0f;
      sm += n[q] * (v[q].x - ref);
    }
    const float mean = ref + share_sum(sh.lanes, sm) / (float)s.hw;
#pragma unroll
    for (int q = 0; q < MOST; ++q) {
      const float d = v[q].x - mean;
      sq += fmaf(n[q] * (float)s.cg, d * d, v[q].y);
    }
    sq = share_sum(sh.lanes, sq);
    if (sh.lane == 0) {
      const float r = rstd_of(sq, (float)s.hw * (float)s.cg, eps);
      sums[0][sh.group] = mean;
      sums[1][sh.group] = r;
      if (stat) {
        stat[(int64_t)b * s.g + g] = mean;
        stat[((int64_t)s.b + b) * s.g + g] = r;
      }
    }
  }
  __syncthreads();
  const int last = min(g0 + sh.groups, s.g) * s.cg;
  for (int c = g0 * s.cg + threadIdx.x; c < last; c += THREADS) {
    const int at = small_div(c, s.cg) - g0;
    chan[(int64_t)b * s.c + c] = sums[0][at];
    chan[((int64_t)s.b + b) * s.c + c] = sums[1][at] * (w ? w[c] : 1.0f);
  }
}

// Block (sample, piece of pixels, chunk of columns).  Pieces are short and in
// memory's order: blocks that run together then read and write neighbouring
// memory (403 MB copied in 145 us; by 2048 blocks, each with a long piece of
// its own, in 166 us).
struct Pieces {
  int pixels, pieces, chunks;  // pixels of a piece; pieces, column chunks
};

template <typename T, int V, int ACT, bool DROP>
__global__ __launch_bounds__(BLOCK) void gn_apply(
    const T* __restrict__ x, T* __restrict__ y,
    const float* __restrict__ chan, const float* __restrict__ bias, Shape s,
    Pieces ps, bool stream, int act, DropoutArgs d) {
  const int chunk = blockIdx.x % ps.chunks, rest = blockIdx.x / ps.chunks;
  const int piece = rest % ps.pieces, b = rest / ps.pieces;
  const int c0 = chunk * BLOCK * V;
  const Place pl(min(BLOCK, (s.c - c0) / V), BLOCK);
  const int64_t first = (int64_t)piece * ps.pixels;
  const int count = pl.count((int)min((int64_t)ps.pixels, s.hw - first));
  if (count == 0) return;
  const int ch = c0 + pl.col * V;
  const int64_t from = ((int64_t)b * s.hw + first + pl.row) * s.c + ch;
  const int64_t next = (int64_t)pl.rows * s.c;
  const DropoutState st = dropout_state(d);
  constexpr int D = AHEAD1<T>;
  Affine<V> k;
  k.channels(chan + (int64_t)b * s.c + ch, (int64_t)s.b * s.c, bias, ch);
  walk<D>(count, [&](int i, bool in) {
    return load_pack<T, V>(x + from + (in ? i * next : 0), stream);
  }, [&](int i, const Pack<T, V>& raw) {
    const int64_t at = from + i * next;
    store_pack<T, V>(y + at,
                     forward_value<T, V, ACT, DROP>(k, raw, act, d, st,
                                                    (uint64_t)at),
                     stream);
  });
}

// Block (split, sample): sums of gz and gz xhat of every channel over the
// split's pixels.  part_c: [2][b * splits][c]; part_g: [b][g][splits] of the
// same sums weighted by w and added up over the group, which the sample's last
// block joins.  Sums are held to runs of RUN values, which are then added to a
// thread's totals in LDS: in one chain roundings that go one way add up, and
// 8192 equal gradients had db wrong by 6e-5.  chan, where dx is asked for: [4][b][c], for every channel its
// mean, rstd w, and what dx adds to rstd w gz: chan2 + (x - mean) chan3.
template <typename T, int V, int ACT, bool DROP>
__global__ __launch_bounds__(THREADS, 4) void gn_bwd_sums(
    const T* __restrict__ x, const T* __restrict__ gy,
    const float* __restrict__ w, const float* __restrict__ bias,
    const float* __restrict__ stat, float* __restrict__ part_c,
    uint64_t* __restrict__ part_g, uint32_t* __restrict__ counts,
    float* __restrict__ chan, Shape s, Deal deal, int lanes, int act,
    DropoutArgs d) {
  extern __shared__ float lds_sums[];  // red; [2][channels]; [2][g]; totals
  float* red = lds_sums;
  float* sum1 = red + RED_CHANNELS(V);
  float* sum2 = sum1 + min(THREADS * V, s.c);
  float* joined = sum2 + min(THREADS * V, s.c);
  int* flag = reinterpret_cast<int*>(joined + 2 * s.g);
  constexpr int RUN_BATCHES = RUN / AHEAD2<T>;
  const bool runs = deal.more_than(RUN_BATCHES);
  float* total = joined + 2 * s.g + 1 + threadIdx.x;  // [2 V][THREADS], if runs
  const int split = blockIdx.x % deal.n, b = blockIdx.x / deal.n;
  const DropoutState st = dropout_state(d);
  const float* mean = stat + (int64_t)b * s.g;
  const float* rstd = stat + ((int64_t)s.b + b) * s.g;
  float* out1 = part_c + ((int64_t)b * deal.n + split) * s.c;
  float* out2 = out1 + (int64_t)s.b * deal.n * s.c;
  for (int c0 = 0; c0 < s.c; c0 += THREADS * V) {
    const Place pl(min(THREADS, (s.c - c0) / V), THREADS);
    const int64_t next = (int64_t)pl.rows * s.c;
    const int ch = c0 + pl.col * V;
    float s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0f;
    if (pl.on) {
      constexpr int D = AHEAD2<T> / 2;  // more would spill registers
      Affine<V> k;
      k.params(ch, w, bias);
      k.stats(ch, s.cg, mean, rstd);
      int batch = 0;
      for (int kb = split; kb < deal.batches; kb += deal.n, ++batch) {
        const int here = pl.count(deal.length(kb));
        const int64_t at = ((int64_t)b * s.hw + (int64_t)kb * deal.batch +
                            pl.row) * s.c + ch;
        walk<D>(here, [&](int i, bool in) {
          const int64_t to = at + (in ? i * next : 0);
          return Both<T, V>{load_pack<T, V>(x + to), load_pack<T, V>(gy + to)};
        }, [&](int i, const Both<T, V>& raw) {
          float e[V], g[V];
          through<T, V, ACT, DROP>(k, raw.x, raw.g, act, d, st,
                                   (uint64_t)(at + i * next), e, g);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            s1[j] += g[j];
            s2[j] = fmaf(g[j], e[j], s2[j]);
          }
        });
        if (runs && batch % RUN_BATCHES == RUN_BATCHES - 1) {
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) {
            float* at = total + j * THREADS;
            float& sum = j < V ? s1[j % V] : s2[j % V];
            *at = batch < RUN_BATCHES ? sum : *at + sum;
            sum = 0.0f;
          }
        }
      }
      if (runs) {  // every block has had one
#pragma unroll
        for (int j = 0; j < V; ++j) {
          s1[j] += total[j * THREADS];
          s2[j] += total[(V + j) * THREADS];
        }
      }
      each_group<V>(ch, s.cg, [&](int j, int g) { s2[j] *= rstd[g]; });
    }
    sum_channels<V>(red, pl, s1, s2, sum1, sum2);
    const int width = pl.cols * V;
    for (int c = threadIdx.x; c < width; c += THREADS) {
      out1[c0 + c] = sum1[c];
      out2[c0 + c] = sum2[c];
    }
    weigh_groups(sum1, sum2, w, c0, width, s.cg, [&](int g, float a, float c) {
      const bool begun = g * s.cg < c0;
      joined[g] = a + (begun ? joined[g] : 0.0f);
      joined[s.g + g] = c + (begun ? joined[s.g + g] : 0.0f);
    });
    __syncthreads();
  }
  if (!chan) return;
  uint64_t* parts = part_g + (int64_t)b * s.g * deal.n;
  for (int g = threadIdx.x; g < s.g; g += THREADS)
    put2(parts + (int64_t)g * deal.n + split, joined[g], joined[s.g + g]);
  if (!last_of(deal.n, counts + b, flag)) return;
  const int lane = threadIdx.x & (lanes - 1);
  const float inv_n = 1.0f / ((float)s.hw * (float)s.cg);
  for (int g = threadIdx.x / lanes; g < s.g; g += THREADS / lanes) {
    float2 v[MOST], sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int q = 0; q < MOST; ++q) {
      const int i = lane + q * lanes;
      v[q] = i < deal.n ? get2(parts + (int64_t)g * deal.n + i)
                        : make_float2(0.0f, 0.0f);
    }
#pragma unroll
    for (int q = 0; q < MOST; ++q) add_to(sum, v[q]);
    sum.x = share_sum(lanes, sum.x);
    sum.y = share_sum(lanes, sum.y);
    if (lane == 0) {
      joined[g] = -rstd[g] * (sum.x * inv_n);
      joined[s.g + g] = -rstd[g] * rstd[g] * (sum.y * inv_n);
    }
  }
  __syncthreads();
  const int64_t plane = (int64_t)s.b * s.c;
  for (int c = threadIdx.x; c < s.c; c += THREADS) {
    const int g = small_div(c, s.cg);
    float* at = chan + (int64_t)b * s.c + c;
    at[0] = mean[g];
    at[plane] = rstd[g] * (w ? w[c] : 1.0f);
    at[2 * plane] = joined[g];
    at[3 * plane] = joined[s.g + g];
  }
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
    float sum = 0.0f, lost = 0.0f;
    if (ch < c) {
#pragma unroll 8
      for (int64_t r = r0; r < rows; r += BLOCK / 8)
        add_kept(sum, lost, at[r * c]);
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
// others, laid out as gn_apply's, write dx.
template <typename T, int V, int ACT, bool DROP>
__global__ __launch_bounds__(BLOCK, 4) void gn_bwd_dx(
    const T* __restrict__ x, const T* __restrict__ gy, T* __restrict__ dx,
    const float* __restrict__ chan, const float* __restrict__ bias,
    const float* __restrict__ part_c, int64_t part_rows,
    float* __restrict__ db, float* __restrict__ dw, Shape s, Pieces ps,
    int param_blocks, bool stream, int act, DropoutArgs d) {
  __shared__ float red[BLOCK];
  if ((int)blockIdx.x < param_blocks) {
    param_sums(part_c, part_rows, s.c, blockIdx.x, db, dw, red);
    return;
  }
  const int block = blockIdx.x - param_blocks;
  const int chunk = block % ps.chunks, rest = block / ps.chunks;
  const int piece = rest % ps.pieces, b = rest / ps.pieces;
  const int c0 = chunk * BLOCK * V;
  const Place pl(min(BLOCK, (s.c - c0) / V), BLOCK);
  const int64_t first = (int64_t)piece * ps.pixels;
  const int count = pl.count((int)min((int64_t)ps.pixels, s.hw - first));
  if (count == 0) return;
  const int ch = c0 + pl.col * V;
  const int64_t from = ((int64_t)b * s.hw + first + pl.row) * s.c + ch;
  const int64_t next = (int64_t)pl.rows * s.c;
  const DropoutState st = dropout_state(d);
  Affine<V> k;
  float m1[V], m2[V];
  auto emit = [&](const Pack<T, V>& rx, const Pack<T, V>& rg, int64_t at) {
    float e[V], g[V];
    through<T, V, ACT, DROP>(k, rx, rg, act, d, st, (uint64_t)at, e, g);
#pragma unroll
    for (int j = 0; j < V; ++j)
      g[j] = fmaf(k.a[j], g[j], fmaf(e[j], m2[j], m1[j]));
    store_pack<T, V>(dx + at, pack<T, V>(g), stream);
  };
  constexpr int D = AHEAD2<T>;
  const int64_t plane = (int64_t)s.b * s.c;
  chan += (int64_t)b * s.c + ch;
  k.channels(chan, plane, bias, ch);
  load_floats<V>(m1, chan + 2 * plane);
  load_floats<V>(m2, chan + 3 * plane);
  walk<D>(count, [&](int i, bool in) {
    const int64_t at = from + (in ? i * next : 0);
    return Both<T, V>{load_pack<T, V>(x + at, stream),
                      load_pack<T, V>(gy + at, stream)};
  }, [&](int i, const Both<T, V>& raw) {
    emit(raw.x, raw.g, from + i * next);
  });
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
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

// A launch's threads are counted in 32 bits.
void check_launch(int64_t blocks, int threads) {
  TORCH_CHECK(blocks * threads < (1ll << 32), "group_norm: tensor too large");
}

struct Plan {
  bool tiled;
  Tiles tiles;
  int units;  // groups that a vector touches, at most
  size_t lds;
};

// LDS of a tile's block: half of a CU's 160 KB, so that one block reads while
// another writes.
constexpr size_t TILE_LDS = 80 * 1024;

// How to tile, or that it does not fit.  Spans are multiples of whole groups
// and whole vectors, of 32 bytes or more where they can be, and wider while
// that leaves four blocks per CU.
Plan plan_tiles(const Shape& s, int v, size_t value, bool back) {
  Plan p{};
  p.units = v / std::gcd(v, s.cg);
  const int64_t base = std::lcm((int64_t)s.cg, (int64_t)v);
  const int64_t widest = std::min<int64_t>(s.c, (int64_t)THREADS * v);
  const int64_t many = s.c / base;
  for (int64_t m = 1; m <= many && base * m <= widest; ++m) {
    if (many % m) continue;
    const int64_t span = base * m, spans = s.c / span;
    if (p.tiled && (int64_t)p.tiles.span * (int64_t)value >= 32 &&
        s.b * spans < 1024)
      break;
    const int64_t rows = THREADS / (span / v);
    const int64_t iters = (s.hw + rows - 1) / rows;
    const int64_t lds =
        iters * THREADS * v * (int64_t)value * (back ? 2 : 1) +
        (back ? 4 * RED_CHANNELS(v) + 8 * span + 4 : 8 * THREADS * p.units) +
        8 * (span / s.cg);
    if (lds > (int64_t)TILE_LDS) break;
    p.tiled = true;
    p.lds = (size_t)lds;
    p.tiles = {(int)span, (int)spans, (int)(span / s.cg), (int)iters};
  }
  return p;
}

// Samples that a thread of a span's last block adds up, at most: of more,
// another launch takes the sums, with more than one block's share of the
// memory's rate.  Backward passes, bf16, in us: 4096x64x4x4, 512 samples a
// thread, 92 here and 57 there; one pixel of 512 channels, 1024 samples 78 and
// 55, 4096 samples 281 and 71.  512 of those, where the host's part is longer
// than the kernels, take 53 and 57.
constexpr int64_t MOST_SAMPLES = 256;

int join_blocks(const Shape& s, int lanes) {
  const int groups = THREADS / lanes;
  return (s.g + groups - 1) / groups;
}

// Blocks per sample that sum: about 512 over the batch, two per CU
// (4x55x128x256 fp32: 1024 of them took 20 us, 512 12), with `deep` vectors per
// thread or more; at most what a join reads at once.
Deal deal_pixels(const Shape& s, int v, int deep) {
  Deal d;
  d.batch = THREADS / std::min(THREADS, s.c / v) * deep;
  d.batches = (int)((s.hw + d.batch - 1) / d.batch);
  d.missing = (int)((int64_t)d.batches * d.batch - s.hw);
  d.n = std::max(1, std::min({(512 + s.b - 1) / s.b, d.batches, MOST_PARTS}));
  // joins have at most as many blocks as a sample has groups
  check_launch((int64_t)s.b * std::max(d.n, s.g), THREADS);
  return d;
}

// Pieces of `deep` vectors per thread.
Pieces cut_pieces(const Shape& s, int v, int deep, int64_t more) {
  const int cols = std::min(BLOCK, s.c / v);
  Pieces p;
  p.pixels = BLOCK / cols * deep;
  p.chunks = (s.c / v + BLOCK - 1) / BLOCK;
  p.pieces = (int)((s.hw + p.pixels - 1) / p.pixels);
  check_launch((int64_t)s.b * p.pieces * p.chunks + more, BLOCK);
  return p;
}

// Activations, and whether there is dropout, are compiled in for whole vectors;
// narrower ones, which odd channel counts take, choose as they go.
#define GN_ACT(DROP_, ACT_, ...)                \
  {                                             \
    constexpr int V = 8, ACT = ACT_;            \
    constexpr bool DROP = DROP_;                \
    __VA_ARGS__;                                \
    break;                                      \
  }
#define GN_ACTS(DROP_, ACT_, ...)                            \
  switch (ACT_) {                                            \
    case ACT_ELU: GN_ACT(DROP_, ACT_ELU, __VA_ARGS__)        \
    case ACT_LEAKY: GN_ACT(DROP_, ACT_LEAKY, __VA_ARGS__)    \
    case ACT_RELU: GN_ACT(DROP_, ACT_RELU, __VA_ARGS__)      \
    case ACT_SILU: GN_ACT(DROP_, ACT_SILU, __VA_ARGS__)      \
    default: GN_ACT(DROP_, ACT_NONE, __VA_ARGS__)            \
  }
#define GN_VARIANT(V_, ACT_, ON_, ...)          \
  do {                                          \
    if (V_ == 8 && ON_) {                       \
      GN_ACTS(true, ACT_, __VA_ARGS__)          \
    } else if (V_ == 8) {                       \
      GN_ACTS(false, ACT_, __VA_ARGS__)         \
    } else if (V_ == 4) {                       \
      constexpr int V = 4, ACT = ACT_ANY;       \
      constexpr bool DROP = true;               \
      __VA_ARGS__;                              \
    } else {                                    \
      constexpr int V = 1, ACT = ACT_ANY;       \
      constexpr bool DROP = true;               \
      __VA_ARGS__;                              \
    }                                           \
  } while (0)

// More LDS than a launch may ask for without saying so.
template <typename K>
void allow_lds(K kernel, size_t bytes) {
  if (bytes > 64 * 1024)
    C10_HIP_CHECK(hipFuncSetAttribute(
        reinterpret_cast<const void*>(kernel),
        hipFuncAttributeMaxDynamicSharedMemorySize,
        (int)std::max(bytes, TILE_LDS)));
}

template <typename T>
void gn_forward(const at::Tensor& x, at::Tensor& y, const float* w,
                const float* bias, float* stat, uint32_t* counts, int n_counts,
                const Shape& s, float eps, int act, const DropoutArgs& d) {
  const hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
  const T* px = (const T*)x.data_ptr();
  T* py = (T*)y.data_ptr();
  const int v = vector_of<T>(s, {px, py});
  const Plan p = plan_tiles(s, v, sizeof(T), false);
  if (p.tiled) {
    check_launch((int64_t)s.b * p.tiles.spans, THREADS);
    float* rstd = stat ? stat + (int64_t)s.b * s.g : nullptr;
    GN_VARIANT(v, act, d.on, {
      auto kernel = gn_tile<T, V, ACT, DROP>;
      allow_lds(kernel, p.lds);
      hipLaunchKernelGGL(kernel, dim3(s.b * p.tiles.spans), dim3(THREADS),
                         p.lds, stream, px, py, w, bias, stat, rstd, counts,
                         n_counts, s, p.tiles, p.units, eps, act, d);
      C10_HIP_KERNEL_LAUNCH_CHECK();
    });
    return;
  }
  const Deal deal = deal_pixels(s, v, AHEAD1<T>);
  const Pieces ps = cut_pieces(s, v, 2 * AHEAD1<T>, 0);
  const int64_t parts = (int64_t)s.b * s.g * deal.n;
  const int64_t plane = (int64_t)s.b * s.c;
  // channels' values first: their vectors are aligned
  auto buf = at::empty({2 * plane + 2 * parts}, x.options().dtype(at::kFloat));
  float* chan = buf.data_ptr<float>();
  float2* part = (float2*)(chan + 2 * plane);
  const auto stats = v == 8   ? gn_stats<T, 8>
                     : v == 4 ? gn_stats<T, 4>
                              : gn_stats<T, 1>;
  const size_t lds = 4 * (size_t)s.g * 4;
  allow_lds(stats, lds + THREADS * v * 8);
  hipLaunchKernelGGL(stats, dim3(s.b * deal.n), dim3(THREADS), lds, stream, px,
                     part, counts, n_counts, s, deal, p.units);
  C10_HIP_KERNEL_LAUNCH_CHECK();
  const int lanes = share_lanes(deal.n);
  hipLaunchKernelGGL(gn_join, dim3(s.b * join_blocks(s, lanes)), dim3(THREADS),
                     0, stream, part, w, stat, chan, s, deal, lanes, eps);
  C10_HIP_KERNEL_LAUNCH_CHECK();
  const bool nt = x.numel() * (int64_t)sizeof(T) > STREAM_BYTES;
  GN_VARIANT(v, act, d.on, {
    hipLaunchKernelGGL((gn_apply<T, V, ACT, DROP>),
                       dim3(s.b * ps.pieces * ps.chunks), dim3(BLOCK), 0,
                       stream, px, py, chan, bias, s, ps, nt, act, d);
    C10_HIP_KERNEL_LAUNCH_CHECK();
  });
}

template <typename T>
void gn_backward(const at::Tensor& x, const at::Tensor& gy, at::Tensor& dx_out,
                 const float* w, const float* bias, const float* stat,
                 uint32_t* counts, float* db, float* dw, const Shape& s,
                 int act, const DropoutArgs& d) {
  const hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
  const T* px = (const T*)x.data_ptr();
  const T* pg = (const T*)gy.data_ptr();
  T* dx = dx_out.defined() ? (T*)dx_out.data_ptr() : nullptr;
  const int v = vector_of<T>(s, {px, pg, dx});
  const auto opts = x.options().dtype(at::kFloat);
  const Plan p = plan_tiles(s, v, sizeof(T), true);
  if (p.tiled) {
    check_launch((int64_t)s.b * p.tiles.spans, THREADS);
    at::Tensor buf;
    uint64_t* sums = nullptr;
    if (db || dw) {
      buf = at::empty({2 * (int64_t)s.b * s.c}, opts);
      sums = (uint64_t*)buf.data_ptr();
    }
    const float* rstd = stat + (int64_t)s.b * s.g;
    const bool many = s.b > MOST_SAMPLES * sample_shares(p.tiles.span);
    if (many) counts = nullptr;
    GN_VARIANT(v, act, d.on, {
      auto kernel = gn_bwd_tile<T, V, ACT, DROP>;
      allow_lds(kernel, p.lds);
      hipLaunchKernelGGL(kernel, dim3(s.b * p.tiles.spans), dim3(THREADS),
                         p.lds, stream, px, pg, dx, w, bias, stat, rstd, sums,
                         counts, db, dw, s, p.tiles, act, d);
      C10_HIP_KERNEL_LAUNCH_CHECK();
    });
    if (sums && many) {
      hipLaunchKernelGGL(gn_param_grad, dim3((s.c + 7) / 8), dim3(BLOCK), 0,
                         stream, (const float*)sums, (int64_t)s.b, s.c, db, dw);
      C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    return;
  }
  const int param_blocks = db || dw ? (s.c + 7) / 8 : 0;
  const Deal deal = deal_pixels(s, v, AHEAD2<T>);
  const Pieces ps = cut_pieces(s, v, 2 * AHEAD2<T>, param_blocks);
  const int64_t rows = (int64_t)s.b * deal.n, plane = (int64_t)s.b * s.c;
  auto buf = at::empty({4 * plane + 2 * rows * (s.c + s.g)}, opts);
  float* chan = buf.data_ptr<float>();
  float* part_c = chan + 4 * plane;
  uint64_t* part_g = (uint64_t*)(part_c + 2 * rows * s.c);
  const bool nt = x.numel() * (int64_t)sizeof(T) > STREAM_BYTES;
  GN_VARIANT(v, act, d.on, {
    auto sums = gn_bwd_sums<T, V, ACT, DROP>;
    const size_t lds =
        4 * (RED_CHANNELS(V) + 2 * s.g + 1 +
             2 * (size_t)std::min(THREADS * V, s.c) +
             (deal.more_than(RUN / AHEAD2<T>) ? 2 * V * THREADS : 0));
    allow_lds(sums, lds);
    hipLaunchKernelGGL(sums, dim3(s.b * deal.n), dim3(THREADS), lds, stream, px,
                       pg, w, bias, stat, part_c, part_g, counts,
                       dx ? chan : nullptr, s, deal, share_lanes(deal.n), act,
                       d);
    C10_HIP_KERNEL_LAUNCH_CHECK();
    if (dx) {
      hipLaunchKernelGGL((gn_bwd_dx<T, V, ACT, DROP>),
                         dim3(s.b * ps.pieces * ps.chunks + param_blocks),
                         dim3(BLOCK), 0, stream, px, pg, dx, chan, bias, part_c,
                         rows, db, dw, s, ps, param_blocks, nt, act, d);
    } else {
      hipLaunchKernelGGL(gn_param_grad, dim3(param_blocks), dim3(BLOCK), 0,
                         stream, part_c, rows, s.c, db, dw);
    }
    C10_HIP_KERNEL_LAUNCH_CHECK();
  });
}

}  // namespace
