// Group norm with an activation over channels-last rows: per sequence and
// group, y = act((x - mean) * rstd * weight + bias), mean and variance over
// the sequence's rows and the group's channels, all of it in fp32.
//
// Variances are sums of squared differences from a mean, never a difference of
// squares. A running sum of values far from zero is off by its own roundings
// (a clip of 6000 x 2048 values 1000.1 in one group: its mean by 0.004), so the pass
// that sums the squares of x - mean sums those differences too: their mean corrects
// both (64 clips of 750 x 512: 1 % more time in fp32, 5 % in 16 bits). A mean is kept as
// two floats, the second one part of the bias, and threads and blocks join by (count,
// mean, sum of squares about it) with means as offsets from one of them: of a mean far
// from zero a second-order rounding is left. The order of every sum is fixed.
//
// Bound by memory: x is read once and y written once. Single rows keep a group
// in the registers of 1 to 256 threads. Longer sequences are cut into blocks of
// whole groups, 64 bytes of a row or one group, and a cluster of up to sixteen
// CTAs shares a block's rows: each keeps its rows in shared memory, the CTAs
// exchange their statistics through distributed shared memory, and y is formed
// from the kept rows. Rows beyond the shared memory are read again (from L2
// mostly). 64 clips of 750 x 512 fp32 take 43 us, 69 % of the copy rate: a CTA
// loads, exchanges and stores in turn, so that only several an SM overlap. (Two
// launches over ranges of rows, which read x twice, took 57 us, and two to four
// times as long where sequences are short.)
#include <cooperative_groups.h>

#include <algorithm>

#include "fav_common.cuh"
#include "fav_ops.cuh"

namespace fav {
namespace {

namespace cg = cooperative_groups;

struct NormArgs {
  const void* x;
  void* y;
  long long x_stride, y_stride;
  const float *weight, *bias, *alpha, *recip;
  Sequences seq;
  float eps;
  int channels, groups, width;  // width: channels of a group
  int activation, wide;         // wide: 16-byte loads of the coefficients
  int group_threads;            // single rows: threads of a group
  int block_groups, blocks;     // clusters: groups of a block, blocks of a row
  int keep_rows, stats_at;      // clusters: rows of a CTA that shared memory holds, bytes up to the statistics
};

// sin(v)^2 has period pi: v - k pi lies within pi / 2 of zero, where the Taylor
// series of the sine to the 11th power is within 6e-8. pi in two parts
// (8 + 24 bits) keeps the difference exact to fp32 for |v| up to 2^14.
__device__ __forceinline__ float2 both(float c) { return make_float2(c, c); }
__device__ __forceinline__ float2 sin_squared2(float2 v) {
  const float2 t = f2fma(v, both(0.318309886f), both(12582912.f));  // 1.5 * 2^23: rounds to an integer
  const float2 k = f2add(t, both(-12582912.f));
  float2 r = f2fma(k, both(-3.140625f), v);
  r = f2fma(k, both(-9.6765358979e-4f), r);
  const float2 z = f2mul(r, r);
  float2 p = both(-2.5052108e-8f);
  p = f2fma(p, z, both(2.7557319e-6f));
  p = f2fma(p, z, both(-1.9841270e-4f));
  p = f2fma(p, z, both(8.3333333e-3f));
  p = f2fma(p, z, both(-1.6666667e-1f));
  const float2 s = f2fma(f2mul(r, z), p, r);
  return f2mul(s, s);
}
constexpr float kSineRange = 16384.f;
__device__ __noinline__ float sin_squared_far(float v) {
  const float s = sinf(v);
  return s * s;
}

// The coefficients of V neighbouring channels, and their outputs.
template <int V>
struct NormChannels {
  static constexpr int P = (V + 1) / 2;
  float2 w[P], b[P], al[P], re[P];

  __device__ __forceinline__ static void pairs(float2 (&to)[P], const float* from, int c, float none, bool wide) {
    if (!from) {
#pragma unroll
      for (int i = 0; i < P; ++i) to[i] = make_float2(none, none);
    } else if (V % 4 == 0 && wide) {
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        const float4 v = ldg4(from + c + 4 * i);
        to[2 * i] = lo2(v), to[V > 2 ? 2 * i + 1 : 0] = hi2(v);
      }
    } else {
#pragma unroll
      for (int i = 0; i < P; ++i)
        to[i] = make_float2(__ldg(from + c + (V > 1 ? 2 * i : 0)), __ldg(from + c + (V > 1 ? 2 * i + 1 : 0)));
    }
  }
  __device__ __forceinline__ void load(const NormArgs& a, int c) {
    pairs(w, a.weight, c, 1.f, a.wide);
    pairs(b, a.bias, c, 0.f, a.wide);
    if (a.activation == FAV_ACTIVATION_SNAKE) {
      pairs(al, a.alpha, c, 0.f, a.wide);
      pairs(re, a.recip, c, 0.f, a.wide);
    }
  }
  // After load(): w times rstd, so that a value takes one multiply, and the low part
  // of the mean in the bias.
  __device__ __forceinline__ void scale(float rstd, float low) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      w[i] = f2mul(w[i], make_float2(rstd, rstd));
      b[i] = f2fma(w[i], make_float2(-low, -low), b[i]);
    }
  }
  template <typename T>
  __device__ __forceinline__ Pack<T, V> apply(int activation, const Pack<T, V>& x, float mean) const {
    Pack<T, V> out;
    float2 v[P];
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = f2fma(f2add(pair_of(x, i), make_float2(-mean, -mean)), w[i], b[i]);
    if (activation == FAV_ACTIVATION_SILU) {
#pragma unroll
      for (int i = 0; i < P; ++i) v[i] = silu2<T>(v[i]);
    } else if (activation == FAV_ACTIVATION_SNAKE) {
      float2 u[P], q[P];
      float far = 0.f;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        u[i] = f2mul(al[i], v[i]);
        far = fmaxf(far, fmaxf(fabsf(u[i].x), fabsf(u[i].y)));
        q[i] = sin_squared2(u[i]);
      }
      if (far >= kSineRange) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          if (!(fabsf(u[i].x) < kSineRange)) q[i].x = sin_squared_far(u[i].x);
          if (!(fabsf(u[i].y) < kSineRange)) q[i].y = sin_squared_far(u[i].y);
        }
      }
#pragma unroll
      for (int i = 0; i < P; ++i) v[i] = f2fma(re[i], q[i], v[i]);
    }
#pragma unroll
    for (int i = 0; i < P; ++i) put_pair(out, i, v[i]);
    return out;
  }
};

// Sums over a pack's elements, the even and the odd ones apart (V = 1: the
// element alone).
template <typename T, int V>
__device__ __forceinline__ float2 add_values(const Pack<T, V>& x, float2 sum) {
  if constexpr (V == 1) return make_float2(sum.x + to_f32(x.v[0]), 0.f);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) sum = f2add(sum, pair_of(x, i));
  return sum;
}
// Sums of differences from a mean and of their squares, even and odd ones apart.
struct Moments {
  float2 sum, squares;
};
template <typename T, int V>
__device__ __forceinline__ void add_moments(const Pack<T, V>& x, float mean, Moments& m) {
  if constexpr (V == 1) {
    const float d = to_f32(x.v[0]) - mean;
    m.sum.x += d;
    m.squares.x = fmaf(d, d, m.squares.x);
    return;
  }
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const float2 d = f2add(pair_of(x, i), make_float2(-mean, -mean));
    m.sum = f2add(m.sum, d);
    m.squares = f2fma(d, d, m.squares);
  }
}
// .x: the sum of the differences, .y: of their squares.
__device__ __forceinline__ float2 total_of(const Moments& m) {
  return make_float2(m.sum.x + m.sum.y, m.squares.x + m.squares.y);
}

// Of `count` values: their mean is mean + low, their squares are about that.
struct Stats {
  float mean, low, squares;
};
// From 1 / count and sums of differences from `about` (NaN stays NaN; rounding may
// leave the squares of equal values just under zero).
__device__ __forceinline__ Stats stats_of(float inv, float about, float2 sums) {
  const float low = sums.x * inv;
  return {about, low, max_nan(fmaf(-sums.x, low, sums.y), 0.f)};
}
// Joins the statistics `b` of `more` values to those of `count`; a's mean stays the
// one that its low part counts from.
__device__ __forceinline__ void join(Stats& a, float& count, const Stats& b, float more) {
  if (more == 0.f) return;
  const float n = count + more, d = (b.mean - a.mean) + b.low - a.low, f = more / n;
  a.low = fmaf(d, f, a.low);
  a.squares += b.squares + d * d * count * f;
  count = n;
}

__device__ __forceinline__ float shuffle_add(float v, int o) { return v + __shfl_xor_sync(0xffffffffu, v, o); }
__device__ __forceinline__ float2 shuffle_add(float2 v, int o) {
  return make_float2(shuffle_add(v.x, o), shuffle_add(v.y, o));
}
__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float2 add(float2 a, float2 b) { return f2add(a, b); }

constexpr int kRowThreads = 256;  // single rows

// ------------------------------------------------------------- single rows
// `group_threads` threads (a power of two) hold a (row, group)'s values, NV
// vectors each; NV = 0 reads them again instead.
template <typename S>
__device__ __forceinline__ S group_sum(S v, int threads, S* part) {
  const int in_warp = min(threads, 32);
  for (int o = in_warp / 2; o > 0; o >>= 1) v = shuffle_add(v, o);
  if (threads > 32) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    const int first = threadIdx.x / threads * (threads / 32);
    v = part[first];
    for (int i = 1; i < threads / 32; ++i) v = add(v, part[first + i]);
  }
  return v;
}

template <typename T, int V, int NV>
__global__ void __launch_bounds__(kRowThreads) norm_rows_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float part[kRowThreads / 32];
  __shared__ float2 part2[kRowThreads / 32];
  grid_dependency_sync();
  const int threads = a.group_threads, per_block = kRowThreads / threads;
  const long long item = (long long)blockIdx.x * per_block + threadIdx.x / threads;
  const bool live = item < (long long)a.seq.rows * a.groups;
  const long long row = live ? item / a.groups : 0;
  const int g = live ? (int)(item - row * a.groups) : 0;
  const int t = threadIdx.x % threads, vecs = a.width / V, c0 = g * a.width;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride + c0;
  T* y = static_cast<T*>(a.y) + row * a.y_stride + c0;
  const float inv = 1.f / (float)a.width;
  Moments m{};
  float2 sum = make_float2(0.f, 0.f);
  if constexpr (NV > 0) {
    Pack<T, V> xv[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (t + k * threads < vecs) {
        xv[k] = load_const<T, V>(x + (t + k * threads) * V);
        sum = add_values(xv[k], sum);
      }
    const float mean = group_sum(sum.x + sum.y, threads, part) * inv;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (t + k * threads < vecs) add_moments(xv[k], mean, m);
    const Stats s = stats_of(inv, mean, group_sum(total_of(m), threads, part2));
    const float rstd = rsqrtf(s.squares * inv + a.eps);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (t + k * threads) * V;
      if (!live || t + k * threads >= vecs) continue;
      NormChannels<V> ch;
      ch.load(a, c0 + c);
      ch.scale(rstd, s.low);
      store_pack<T, V>(y + c, ch.apply(a.activation, xv[k], mean));
    }
  } else {
    for (int k = t; k < vecs; k += threads) sum = add_values(load_const<T, V>(x + (size_t)k * V), sum);
    const float mean = group_sum(sum.x + sum.y, threads, part) * inv;
    for (int k = t; k < vecs; k += threads) add_moments(load_const<T, V>(x + (size_t)k * V), mean, m);
    const Stats s = stats_of(inv, mean, group_sum(total_of(m), threads, part2));
    const float rstd = rsqrtf(s.squares * inv + a.eps);
    for (int k = t; live && k < vecs; k += threads) {
      NormChannels<V> ch;
      ch.load(a, c0 + k * V);
      ch.scale(rstd, s.low);
      store_pack<T, V>(y + (size_t)k * V, ch.apply(a.activation, load_const<T, V>(x + (size_t)k * V), mean));
    }
  }
}

constexpr int kWideThreads = 512;  // of a CTA with a large share of the rows
// Of a CTA with a small one: twice as many for fp32 (64 clips of 750 x 512: 256
// threads 43 us, 128 48 us; bf16 with SiLU 44 and 35).
constexpr int small_threads(int v) { return v == 4 ? 256 : 128; }
constexpr int kMaxCtas = 16;  // of a cluster (above 8 where the device can place them)

// --------------------------------------------------------------- sequences
// A CTA's share of one (sequence, block of groups): rows [first, first + rows)
// by vecs vectors, walked by threads in the order of e = row * vecs + vector. A
// block of several groups has at most NT vectors, and only whole
// rows of threads walk it: a thread then keeps to one vector, hence one group.
template <int NT, typename S>
__device__ __forceinline__ S block_sum(S v, S* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = shuffle_add(v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int i = 1; i < NT / 32; ++i) v = add(v, part[i]);
  return v;
}

template <typename T, int V, int NT>
__global__ void __launch_bounds__(NT, NT == kWideThreads ? 1 : 4) norm_kernel(const __grid_constant__ NormArgs a) {
  extern __shared__ __align__(16) unsigned char s_raw[];
  // A thread's statistics (several groups a block), then the groups' own.
  __shared__ float s_mean[NT], s_low[NT], s_square[NT];
  __shared__ float2 s_sums[NT / 32];
  using P = Pack<T, V>;
  P* kept = reinterpret_cast<P*>(s_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  // Statistics of this CTA's groups, read by the others of the cluster.
  Stats* s_stats = reinterpret_cast<Stats*>(s_raw + a.stats_at);
  grid_dependency_sync();
  const int item = blockIdx.x / ctas, s = item / a.blocks, block = item - s * a.blocks;
  const Span sp = span_of(a.seq, s);
  const bool bad = sp.begin > sp.end;
  if (bad && threadIdx.x == 0) record_error(a.seq.status, kDevBadOffsets);
  const int length = bad ? 0 : sp.end - sp.begin;
  const int g0 = block * a.block_groups, groups = min(a.block_groups, a.groups - g0);
  const int share = (length + ctas - 1) / ctas, before = min(rank * share, length), rows = min(share, length - before);
  const int c0 = g0 * a.width, vecs = groups * a.width / V, group_vecs = a.width / V;
  const T* x = static_cast<const T*>(a.x) + (sp.begin + before) * a.x_stride + c0;
  T* y = static_cast<T*>(a.y) + (sp.begin + before) * a.y_stride + c0;
  const int step = vecs <= NT ? NT / vecs * vecs : NT;
  const bool walks = threadIdx.x < step;
  // Row and vector of a thread, and its steps from one to the next.
  const int r0 = threadIdx.x / vecs, v0 = threadIdx.x - r0 * vecs, dr = step / vecs, dv = step - dr * vecs;
  // Vectors of this thread, the kept ones first.
  const int vectors = walks && rows > r0 ? (int)(((long long)rows * vecs - threadIdx.x - 1) / step) + 1 : 0;
  const int held = min(rows, a.keep_rows);
  const int kept_vectors = walks && held > r0 ? (held * vecs - (int)threadIdx.x - 1) / step + 1 : 0;
  float2 sums = make_float2(0.f, 0.f);
  if (dv == 0) {
    const T* p = x + r0 * a.x_stride + v0 * V;
    P* to = kept + threadIdx.x;
    const long long hop = dr * a.x_stride;
    if constexpr (V == 8) {
      // 16 vectors are on their way to their places, four of them summed at a
      // time, so that the sums of 8 hide loads (bf16 with SiLU, all rows first in
      // brackets: 4 clips of 150 x 512 6.7 us (7.7), 64 of 1500 93 (95), 64 of 750
      // 34.7 both, 64 of 12 9.7 (9.2)).
      int issued = 0;
      const auto issue = [&] {
#pragma unroll
        for (int u = 0; u < 4; ++u, ++issued, p += hop)
          if (issued < kept_vectors) copy_pack<T, V>(to + issued * step, p);
        copy_commit();
      };
      issue();
      issue();
      issue();
      for (int k = 0; k < kept_vectors; k += 4) {
        issue();
        copy_wait<3>();
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (k + u < kept_vectors) sums = add_values(to[(k + u) * step], sums);
      }
    } else {
      // All of the kept rows are on their way at once, then summed (64 clips of 750 x
      // 512 fp32 43 us, as above 45).
#pragma unroll 4
      for (int k = 0; k < kept_vectors; ++k, p += hop) copy_pack<T, V>(to + k * step, p);
      copy_commit();
      copy_wait<0>();
#pragma unroll 4
      for (int k = 0; k < kept_vectors; ++k) sums = add_values(to[k * step], sums);
    }
    p = x + r0 * a.x_stride + v0 * V + kept_vectors * hop;
#pragma unroll 4
    for (int k = kept_vectors; k < vectors; ++k, p += hop) sums = add_values(load_const<T, V>(p), sums);
  } else {
    for (int k = 0, r = r0, v = v0; k < vectors; ++k) {
      const P in = load_const<T, V>(x + r * a.x_stride + v * V);
      sums = add_values(in, sums);
      if (k < kept_vectors) kept[threadIdx.x + k * step] = in;
      r += dr, v += dv;
      if (v >= vecs) ++r, v -= vecs;
    }
  }
  // This thread's differences from `mean` and their squares.
  const auto moments_about = [&](float mean) {
    Moments m{};
#pragma unroll 4
    for (int k = 0; k < kept_vectors; ++k) add_moments(kept[threadIdx.x + k * step], mean, m);
    if (kept_vectors < vectors) {
      int r = r0, v = v0;
      for (int k = 0; k < vectors; ++k) {
        if (k >= kept_vectors) add_moments(load_const<T, V>(x + r * a.x_stride + v * V), mean, m);
        r += dr, v += dv;
        if (v >= vecs) ++r, v -= vecs;
      }
    }
    return total_of(m);
  };
  const float sum = sums.x + sums.y, inv = rows ? 1.f / ((float)rows * (float)a.width) : 0.f;
  if (groups == 1) {
    const float mean = block_sum<NT>(sum, s_square) * inv;
    const float2 total = block_sum<NT>(moments_about(mean), s_sums);
    if (threadIdx.x == 0) s_stats[0] = stats_of(inv, mean, total);
  } else {
    // A thread's squares are about its own mean. A warp joins a group's threads, as
    // seen from the mean of the group's first: the offsets give the group's mean,
    // then the squares move to it.
    Stats own{};
    if (vectors) {
      const float own_inv = 1.f / (float)(vectors * V), mean = sum * own_inv;
      own = stats_of(own_inv, mean, moments_about(mean));
    }
    s_mean[threadIdx.x] = own.mean;
    s_low[threadIdx.x] = own.low;
    s_square[threadIdx.x] = own.squares;
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int g = warp; g < groups; g += NT / 32) {
      const float origin = s_mean[g * group_vecs];
      const auto each = [&](auto&& f) {  // f(values, mean's offset, squares) of the lane's threads
        for (int i = lane; i < dr * group_vecs; i += 32) {
          const int k = i / group_vecs, t = k * vecs + g * group_vecs + i - k * group_vecs;
          // Vectors that thread t walked: rows k, k + dr, ...
          const int walked = rows > k ? (rows - k - 1) / dr + 1 : 0;
          if (walked) f((float)(walked * V), (s_mean[t] - origin) + s_low[t], s_square[t]);
        }
      };
      float total = 0.f, squares = 0.f;
      each([&](float n, float offset, float) { total = fmaf(n, offset, total); });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total = shuffle_add(total, o);
      const float low = total * inv;
      each([&](float n, float offset, float square) {
        const float d = offset - low;
        squares += fmaf(n * d, d, square);
      });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) squares = shuffle_add(squares, o);
      if (lane == 0) s_stats[g] = {origin, low, squares};
    }
  }
  if (ctas > 1)
    cluster.sync();
  else
    __syncthreads();
  // Every CTA joins all of the cluster's, in order, into its own table.
  float* s_rstd = s_square;
  if (threadIdx.x < groups) {  // at most one a thread
    const int g = threadIdx.x;
    Stats part[kMaxCtas];
#pragma unroll
    for (int i = 0; i < kMaxCtas; ++i)
      if (i < ctas) part[i] = cluster.map_shared_rank(s_stats, i)[g];
    Stats all = part[0];
    float count = (float)min(share, length) * (float)a.width;
#pragma unroll
    for (int i = 1; i < kMaxCtas; ++i)
      if (i < ctas) join(all, count, part[i], (float)(min(share, length - min(i * share, length))) * (float)a.width);
    s_mean[g] = all.mean;
    s_low[g] = all.low;
    s_rstd[g] = count > 0.f ? rsqrtf(all.squares / count + a.eps) : 0.f;
  }
  if (ctas > 1) cluster.barrier_arrive();  // done with the others' statistics
  __syncthreads();
  if (dv == 0) {
    // One vector of channels for good: its coefficients stay in registers.
    const int g = min(v0 / group_vecs, groups - 1);
    const float mean = s_mean[g];
    NormChannels<V> ch;
    if (vectors) ch.load(a, c0 + v0 * V);
    ch.scale(s_rstd[g], s_low[g]);
    T* p = y + r0 * a.y_stride + v0 * V;
    const long long hop = dr * a.y_stride;
#pragma unroll 2
    for (int k = 0; k < kept_vectors; ++k, p += hop)
      store_pack<T, V>(p, ch.apply(a.activation, kept[threadIdx.x + k * step], mean));
    const T* from = x + (r0 + (long long)kept_vectors * dr) * a.x_stride + v0 * V;
    for (int k = kept_vectors; k < vectors; ++k, p += hop, from += dr * a.x_stride)
      store_pack<T, V>(p, ch.apply(a.activation, load_const<T, V>(from), mean));
  } else {
    for (int k = 0, r = r0, v = v0; k < vectors; ++k) {
      const P in = k < kept_vectors ? kept[threadIdx.x + k * step] : load_const<T, V>(x + r * a.x_stride + v * V);
      NormChannels<V> ch;
      ch.load(a, c0 + v * V);
      ch.scale(s_rstd[0], s_low[0]);
      store_pack<T, V>(y + r * a.y_stride + v * V, ch.apply(a.activation, in, s_mean[0]));
      r += dr, v += dv;
      if (v >= vecs) ++r, v -= vecs;
    }
  }
  if (ctas > 1) cluster.barrier_wait();  // no CTA leaves while another reads its statistics
}

constexpr int kMaxNormSmem = 200 * 1024;

// Whether the device can place clusters of this size (more than 8 CTAs is not
// guaranteed).
bool clusters_fit(void (*kernel)(NormArgs), int ctas, int threads, size_t smem) {
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxNormSmem);
  cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) cudaGetLastError();
  return clusters > 0;
}

template <typename T, int V>
cudaError_t launch_rows(NormArgs a, cudaStream_t stream) {
  const int vecs = a.width / V;
  a.group_threads = 1;
  while (a.group_threads < kRowThreads && a.group_threads < vecs) a.group_threads *= 2;
  const long long per_block = kRowThreads / a.group_threads;
  const long long blocks = ((long long)a.seq.rows * a.groups + per_block - 1) / per_block;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (vecs <= a.group_threads) return launch_op(norm_rows_kernel<T, V, 1>, (unsigned)blocks, kRowThreads, 0, stream, a);
  if (vecs <= 4 * a.group_threads)
    return launch_op(norm_rows_kernel<T, V, 4>, (unsigned)blocks, kRowThreads, 0, stream, a);
  return launch_op(norm_rows_kernel<T, V, 0>, (unsigned)blocks, kRowThreads, 0, stream, a);
}

template <typename T, int V, int NT>
cudaError_t launch_cluster(const NormArgs& a, int ctas, size_t smem, cudaStream_t stream) {
  const long long blocks = (long long)a.seq.n * a.blocks * ctas;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const auto kernel = norm_kernel<T, V, NT>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxNormSmem);
  if (e != cudaSuccess) return e;
  if (ctas > 8 && (e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess)
    return e;
  return launch_op(kernel, (unsigned)blocks, NT, smem, stream, a, (unsigned)ctas);
}

template <typename T, int V>
cudaError_t launch_sequences(NormArgs a, cudaStream_t stream) {
  const int vecs = a.width / V;
  // Whole groups, 64 bytes of a row where they are narrower: short rows leave
  // a CTA's share small enough for several an SM without a larger cluster.
  a.block_groups = std::max(1, std::min(a.groups, 64 / (int)(a.width * sizeof(T))));
  while (a.block_groups > 1 && a.block_groups * vecs > 128) --a.block_groups;
  a.blocks = (a.groups + a.block_groups - 1) / a.block_groups;
  const size_t row = (size_t)a.block_groups * a.width * sizeof(T), stats = a.block_groups * sizeof(Stats);
  // Shared memory for sequences of up to twice the mean length.
  const long long rows = a.seq.offsets ? std::min<long long>(a.seq.rows, 2LL * a.seq.rows / a.seq.n + 1) : a.seq.length;
  // CTAs share a sequence while there are fewer than two an SM, or while a share
  // exceeds half an SM's shared memory.
  int ctas = 1;
  while (ctas < kMaxCtas && rows >= 32 * ctas &&
         ((long long)a.seq.n * a.blocks * ctas < 148 * 2 || (rows + ctas - 1) / ctas * row > kMaxNormSmem / 2))
    ctas *= 2;
  const auto fit = [&] {
    const long long share = (rows + ctas - 1) / ctas;
    // (15: what rounding the rows up to 16 bytes may add)
    a.keep_rows = (int)std::min<long long>(share, (kMaxNormSmem - stats - 15) / row);
    a.stats_at = (int)((a.keep_rows * row + 15) / 16 * 16);
    return a.stats_at + stats;
  };
  size_t smem = fit();
  if (ctas > 8 && !clusters_fit(norm_kernel<T, V, kWideThreads>, ctas, kWideThreads, smem)) ctas = 8, smem = fit();
  // Large shares, one CTA an SM, need its threads; small ones more CTAs.
  if (smem > 64 * 1024 || ctas > 8) return launch_cluster<T, V, kWideThreads>(a, ctas, smem, stream);
  return launch_cluster<T, V, small_threads(V)>(a, ctas, smem, stream);
}

template <typename T, int V>
cudaError_t launch_width(const NormArgs& a, cudaStream_t stream) {
  if (!a.seq.offsets && a.seq.length == 1) return launch_rows<T, V>(a, stream);
  return launch_sequences<T, V>(a, stream);
}

template <typename T>
cudaError_t launch_type(const NormArgs& a, cudaStream_t stream) {
  constexpr int kWide = 16 / sizeof(T);
  const auto fits = [&](int v) {
    return a.width % v == 0 && aligned_for(a.x, a.x_stride, sizeof(T), v) && aligned_for(a.y, a.y_stride, sizeof(T), v);
  };
  if (fits(kWide)) return launch_width<T, kWide>(a, stream);
  if (fits(2)) return launch_width<T, 2>(a, stream);
  return launch_width<T, 1>(a, stream);
}

}  // namespace

cudaError_t launch_group_norm(const fav_norm_args& c, const Sequences& seq, cudaStream_t stream) {
  NormArgs a{};
  a.x = c.x;
  a.y = c.y;
  a.x_stride = c.x_stride;
  a.y_stride = c.y_stride;
  a.weight = c.weight;
  a.bias = c.bias;
  a.alpha = c.alpha;
  a.recip = c.reciprocal;
  a.seq = seq;
  a.eps = c.eps;
  a.channels = c.channels;
  a.groups = c.groups;
  a.width = c.channels / c.groups;
  a.activation = c.activation;
  a.wide = a.width % 4 == 0 && aligned_for(c.weight, 0, 4, 4) && aligned_for(c.bias, 0, 4, 4) &&
           aligned_for(c.alpha, 0, 4, 4) && aligned_for(c.reciprocal, 0, 4, 4);
  if (c.type == FAV_TYPE_F32) return launch_type<float>(a, stream);
  if (c.type == FAV_TYPE_BF16) return launch_type<__nv_bfloat16>(a, stream);
  return launch_type<__half>(a, stream);
}

}  // namespace fav
