// Group norm with an activation over channels-last rows: per sequence and
// group, y = act((x - mean) * rstd * weight + bias), mean and variance over
// the sequence's rows and the group's channels, all of it in fp32.
//
// Variances are sums of squared differences from a mean, never a difference of
// squares: a thread centres its values on its own mean, and threads and blocks
// join by (count, mean, sum of squares about it), so a mean far from zero costs
// no digits. The order of every sum is fixed.
//
// Bound by memory: x is read once and y written once. Single rows keep a group
// in the registers of 1 to 256 threads. Longer sequences are cut into blocks of
// whole groups, about 256 bytes of a row, and a cluster of up to eight CTAs
// shares a block's rows: each keeps its rows in shared memory, the CTAs exchange
// their statistics through distributed shared memory, and y is formed from the
// kept rows. Rows beyond the shared memory are read again (from L2 mostly).
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
// series of the sine to the 13th power is exact to 1e-9. pi in two parts
// (8 + 24 bits) keeps the difference exact to fp32 for |v| up to 2^14.
__device__ __forceinline__ float2 sin_squared2(float2 v) {
  const float2 magic = make_float2(12582912.f, 12582912.f);  // 1.5 * 2^23: rounds to an integer
  const float2 t = f2fma(v, make_float2(0.318309886f, 0.318309886f), magic);
  const float2 k = f2add(t, make_float2(-12582912.f, -12582912.f));
  float2 r = f2fma(k, make_float2(-3.140625f, -3.140625f), v);
  r = f2fma(k, make_float2(-9.6765358979e-4f, -9.6765358979e-4f), r);
  const float2 z = f2mul(r, r);
  float2 p = make_float2(1.6059044e-10f, 1.6059044e-10f);
  p = f2fma(p, z, make_float2(-2.5052108e-8f, -2.5052108e-8f));
  p = f2fma(p, z, make_float2(2.7557319e-6f, 2.7557319e-6f));
  p = f2fma(p, z, make_float2(-1.9841270e-4f, -1.9841270e-4f));
  p = f2fma(p, z, make_float2(8.3333333e-3f, 8.3333333e-3f));
  p = f2fma(p, z, make_float2(-1.6666667e-1f, -1.6666667e-1f));
  const float2 s = f2fma(f2mul(r, z), p, r);
  float2 q = f2mul(s, s);
  if (!(fabsf(v.x) < 16384.f)) { const float e = sinf(v.x); q.x = e * e; }
  if (!(fabsf(v.y) < 16384.f)) { const float e = sinf(v.y); q.y = e * e; }
  return q;
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
  template <typename T>
  __device__ __forceinline__ Pack<T, V> apply(const NormArgs& a, const Pack<T, V>& x, float mean, float rstd) const {
    Pack<T, V> out;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float2 v = f2mul(f2add(pair_of(x, i), make_float2(-mean, -mean)), make_float2(rstd, rstd));
      v = f2fma(v, w[i], b[i]);
      if (a.activation == FAV_ACTIVATION_SILU)
        v = silu2(v);
      else if (a.activation == FAV_ACTIVATION_SNAKE)
        v = f2fma(re[i], sin_squared2(f2mul(al[i], v)), v);
      put_pair(out, i, v);
    }
    return out;
  }
};

template <typename T, int V>
__device__ __forceinline__ float sum_of(const Pack<T, V>& x) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) s += to_f32(x.v[i]);
  return s;
}
template <typename T, int V>
__device__ __forceinline__ float squares_about(const Pack<T, V>& x, float mean, float sum) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float d = to_f32(x.v[i]) - mean;
    sum = fmaf(d, d, sum);
  }
  return sum;
}

constexpr int kNormThreads = 256;

// ------------------------------------------------------------- single rows
// `group_threads` threads (a power of two) hold a (row, group)'s values, NV
// vectors each; NV = 0 reads them again instead.
__device__ __forceinline__ float group_sum(float v, int threads, float* part) {
  const int in_warp = min(threads, 32);
  for (int o = in_warp / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threads > 32) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    const int first = threadIdx.x / threads * (threads / 32);
    v = 0.f;
    for (int i = 0; i < threads / 32; ++i) v += part[first + i];
  }
  return v;
}

template <typename T, int V, int NV>
__global__ void __launch_bounds__(kNormThreads) norm_rows_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float part[kNormThreads / 32];
  grid_dependency_sync();
  const int threads = a.group_threads, per_block = kNormThreads / threads;
  const long long item = (long long)blockIdx.x * per_block + threadIdx.x / threads;
  const bool live = item < (long long)a.seq.rows * a.groups;
  const long long row = live ? item / a.groups : 0;
  const int g = live ? (int)(item - row * a.groups) : 0;
  const int t = threadIdx.x % threads, vecs = a.width / V, c0 = g * a.width;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride + c0;
  T* y = static_cast<T*>(a.y) + row * a.y_stride + c0;
  const float inv = 1.f / (float)a.width;
  if constexpr (NV > 0) {
    Pack<T, V> xv[NV];
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (t + k * threads < vecs) {
        xv[k] = load_const<T, V>(x + (t + k * threads) * V);
        sum += sum_of(xv[k]);
      }
    const float mean = group_sum(sum, threads, part) * inv;
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (t + k * threads < vecs) sum = squares_about(xv[k], mean, sum);
    const float rstd = rsqrtf(group_sum(sum, threads, part) * inv + a.eps);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (t + k * threads) * V;
      if (!live || t + k * threads >= vecs) continue;
      NormChannels<V> ch;
      ch.load(a, c0 + c);
      store_pack<T, V>(y + c, ch.apply(a, xv[k], mean, rstd));
    }
  } else {
    float sum = 0.f;
    for (int k = t; k < vecs; k += threads) sum += sum_of(load_const<T, V>(x + (size_t)k * V));
    const float mean = group_sum(sum, threads, part) * inv;
    sum = 0.f;
    for (int k = t; k < vecs; k += threads) sum = squares_about(load_const<T, V>(x + (size_t)k * V), mean, sum);
    const float rstd = rsqrtf(group_sum(sum, threads, part) * inv + a.eps);
    for (int k = t; live && k < vecs; k += threads) {
      NormChannels<V> ch;
      ch.load(a, c0 + k * V);
      store_pack<T, V>(y + (size_t)k * V, ch.apply(a, load_const<T, V>(x + (size_t)k * V), mean, rstd));
    }
  }
}

// --------------------------------------------------------------- sequences
// A CTA's share of one (sequence, block of groups): rows [first, first + rows)
// by vecs vectors, walked by threads in the order of e = row * vecs + vector. A
// block of several groups has at most kNormThreads vectors, and only whole
// rows of threads walk it: a thread then keeps to one vector, hence one group.
struct Stats {
  float count, mean, squares;
};

__device__ __forceinline__ Stats join(Stats a, Stats b) {
  const float n = a.count + b.count;
  if (b.count == 0.f) return a;
  const float d = b.mean - a.mean, f = b.count / n;
  return {n, fmaf(d, f, a.mean), a.squares + b.squares + d * d * a.count * f};
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormThreads) norm_kernel(const __grid_constant__ NormArgs a) {
  extern __shared__ __align__(16) unsigned char s_raw[];
  __shared__ float s_sum[kNormThreads], s_square[kNormThreads];
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
  const int step = vecs <= kNormThreads ? kNormThreads / vecs * vecs : kNormThreads;
  const bool walks = threadIdx.x < step;
  // Row and vector of a thread, and its steps from one to the next.
  const int r0 = threadIdx.x / vecs, v0 = threadIdx.x - r0 * vecs, dr = step / vecs, dv = step - dr * vecs;
  constexpr int U = 8;  // vectors on their way at once

  float sum = 0.f, count = 0.f;
  for (int r = r0, v = v0; walks && r < rows;) {
    P in[U];
    int n = 0;
    int rr = r, vv = v;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (rr < rows) {
        in[u] = load_const<T, V>(x + rr * a.x_stride + vv * V);
        n = u + 1;
      }
      rr += dr, vv += dv;
      if (vv >= vecs) ++rr, vv -= vecs;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u < n) {
        sum += sum_of(in[u]);
        count += V;
        if (r < a.keep_rows) kept[r * vecs + v] = in[u];
      }
      r += dr, v += dv;
      if (v >= vecs) ++r, v -= vecs;
    }
  }
  // The thread's own mean, and its squares about it.
  const float own = count > 0.f ? sum / count : 0.f;
  float square = 0.f;
  for (int r = r0, v = v0; walks && r < rows;) {
    const P in = r < a.keep_rows ? kept[r * vecs + v] : load_const<T, V>(x + r * a.x_stride + v * V);
    square = squares_about(in, own, square);
    r += dr, v += dv;
    if (v >= vecs) ++r, v -= vecs;
  }
  s_sum[threadIdx.x] = sum;
  s_square[threadIdx.x] = square;
  __syncthreads();
  // A warp joins a group's threads: the sum gives the mean, then the squares
  // move from the threads' means to it.
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int used = vecs <= kNormThreads ? step / vecs : 1, across = vecs <= kNormThreads ? group_vecs : kNormThreads;
  for (int g = warp; g < groups; g += kNormThreads / 32) {
    float total = 0.f;
    for (int i = lane; i < used * across; i += 32) {
      const int k = i / across, t = k * (vecs <= kNormThreads ? vecs : 0) + g * group_vecs + (i - k * across);
      total += s_sum[t];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const float all = (float)rows * (float)a.width, mean = rows > 0 ? total / all : 0.f;
    float squares = 0.f;
    for (int i = lane; i < used * across; i += 32) {
      const int k = i / across, t = k * (vecs <= kNormThreads ? vecs : 0) + g * group_vecs + (i - k * across);
      // Vectors that thread t walked: every step-th of rows * vecs from t on.
      const long long left = (long long)rows * vecs - t;
      const float n = left > 0 ? (float)((left + step - 1) / step * V) : 0.f;
      if (n > 0.f) {
        const float d = s_sum[t] / n - mean;
        squares += fmaf(n * d, d, s_square[t]);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, o);
    if (lane == 0) s_stats[g] = {all, mean, squares};
  }
  if (ctas > 1)
    cluster.sync();
  else
    __syncthreads();
  // Every CTA joins all of the cluster's, in order, into its own table.
  float* s_mean = s_sum;
  float* s_rstd = s_square;
  if (threadIdx.x < groups) {  // at most kNormThreads
    const int g = threadIdx.x;
    Stats all = ctas > 1 ? cluster.map_shared_rank(s_stats, 0)[g] : s_stats[g];
    for (int i = 1; i < ctas; ++i) all = join(all, cluster.map_shared_rank(s_stats, i)[g]);
    s_mean[g] = all.mean;
    s_rstd[g] = all.count > 0.f ? rsqrtf(all.squares / all.count + a.eps) : 0.f;
  }
  __syncthreads();
  if (walks) {
    if (dv == 0) {
      // One vector of channels for good: its coefficients stay in registers.
      const int g = v0 / group_vecs;
      const float mean = s_mean[g], rstd = s_rstd[g];
      NormChannels<V> ch;
      if (r0 < rows) ch.load(a, c0 + v0 * V);
#pragma unroll 4
      for (int r = r0; r < rows; r += dr) {
        const P in = r < a.keep_rows ? kept[r * vecs + v0] : load_const<T, V>(x + r * a.x_stride + v0 * V);
        store_pack<T, V>(y + r * a.y_stride + v0 * V, ch.apply(a, in, mean, rstd));
      }
    } else {
      for (int r = r0, v = v0; r < rows;) {
        const P in = r < a.keep_rows ? kept[r * vecs + v] : load_const<T, V>(x + r * a.x_stride + v * V);
        NormChannels<V> ch;
        ch.load(a, c0 + v * V);
        store_pack<T, V>(y + r * a.y_stride + v * V, ch.apply(a, in, s_mean[v / group_vecs], s_rstd[v / group_vecs]));
        r += dr, v += dv;
        if (v >= vecs) ++r, v -= vecs;
      }
    }
  }
  if (ctas > 1) cluster.sync();  // no CTA leaves while another reads its statistics
}

constexpr int kMaxNormSmem = 200 * 1024;

template <typename T, int V>
cudaError_t launch_rows(NormArgs a, cudaStream_t stream) {
  const int vecs = a.width / V;
  a.group_threads = 1;
  while (a.group_threads < kNormThreads && a.group_threads < vecs) a.group_threads *= 2;
  const long long per_block = kNormThreads / a.group_threads;
  const long long blocks = ((long long)a.seq.rows * a.groups + per_block - 1) / per_block;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (vecs <= a.group_threads) return launch_op(norm_rows_kernel<T, V, 1>, (unsigned)blocks, kNormThreads, 0, stream, a);
  if (vecs <= 4 * a.group_threads)
    return launch_op(norm_rows_kernel<T, V, 4>, (unsigned)blocks, kNormThreads, 0, stream, a);
  return launch_op(norm_rows_kernel<T, V, 0>, (unsigned)blocks, kNormThreads, 0, stream, a);
}

template <typename T, int V>
cudaError_t launch_sequences(NormArgs a, cudaStream_t stream) {
  const int vecs = a.width / V;
  // Whole groups, about 256 bytes of a row, one at least; several only while a
  // thread can keep to one vector.
  a.block_groups = 256 / (int)(a.width * sizeof(T));
  if (a.block_groups < 1) a.block_groups = 1;
  if (a.block_groups > a.groups) a.block_groups = a.groups;
  while (a.block_groups > 1 && a.block_groups * vecs > kNormThreads) --a.block_groups;
  a.blocks = (a.groups + a.block_groups - 1) / a.block_groups;
  const size_t row = (size_t)a.block_groups * a.width * sizeof(T);
  // Shared memory for sequences of up to twice the mean length.
  const long long rows = a.seq.offsets ? std::min<long long>(a.seq.rows, 2LL * a.seq.rows / a.seq.n + 1) : a.seq.length;
  // CTAs share a sequence while the GPU has room for more of them, and while a
  // share is larger than a quarter of an SM's shared memory.
  int ctas = 1;
  while (ctas < 8 && rows >= 32 * ctas &&
         ((long long)a.seq.n * a.blocks * ctas < 148 * 4 || (rows + ctas - 1) / ctas * row > kMaxNormSmem / 4))
    ctas *= 2;
  const size_t stats = a.block_groups * sizeof(Stats) + 16;
  const long long share = (rows + ctas - 1) / ctas;
  a.keep_rows = (int)std::min<long long>(share, (kMaxNormSmem - stats) / row);
  a.stats_at = (int)((a.keep_rows * row + 15) / 16 * 16);
  const size_t smem = a.stats_at + stats;
  const long long blocks = (long long)a.seq.n * a.blocks * ctas;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const cudaError_t e =
      cudaFuncSetAttribute(norm_kernel<T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxNormSmem);
  if (e != cudaSuccess) return e;
  return launch_op(norm_kernel<T, V>, (unsigned)blocks, kNormThreads, smem, stream, a, (unsigned)ctas);
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
