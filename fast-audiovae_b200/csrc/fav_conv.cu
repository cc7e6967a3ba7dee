// Short causal depthwise convolution with a carried history, for packed
// prompts and for single rows (one per stream), channels last:
//
//   y[t, c] = act(bias[c] + sum_j w[c, j] * x[t - (K - 1) + j, c]),  K = 2..8,
//
// rows before a sequence's first come from its slot's history (K - 1 rows, the
// most recent inputs, in x's type) or are zero. Sums run in fp32, oldest tap
// first, and round once to the output's type.
//
// A thread owns up to 4 neighbouring channels and walks down
// `rows_per_thread` rows with the last K - 1 inputs in registers, so a tile
// re-reads only the K - 1 rows above it. The next 8 rows are on their way to
// the thread's own ring in shared memory (cp.async): in registers they would
// halve the resident warps. Packs of 8 channels and rings of 16 rows leave 16
// warps an SM instead of 32 and took 4 to 24 % longer on 16-bit prompts. 33 ragged
// prompts of up to 750 x 2048 bf16 take 26 us, 57 % of the copy rate: the SiLU's
// two special functions a value alone need 12 us, its other instructions 10, and
// the resident warps overlap them in part. 64 x 2000 x 2048 without SiLU take 166
// us, 97 %. 512 single rows take 6.8 us, 4.6 with their histories in L2.
#include "fav_common.cuh"
#include "fav_ops.cuh"

namespace fav {
namespace {

constexpr int kConvThreads = 128;
constexpr int kConvDepth = 8;  // rows of x on their way to a thread

// Blocks that an SM holds at once. 64 registers a thread carry up to 4 taps;
// more taps want 128 (16 x 750 x 2048 bf16, 8 taps: 41 us, with 80 and spills 52).
template <int K>
constexpr int conv_blocks() {
  return K <= 4 ? 8 : 4;
}

struct ConvArgs {
  const void* x;
  void* y;
  long long x_stride, y_stride;
  const float* w;
  const float* bias;
  void* pool;  // [num_slots][2][K - 1][channels]
  Sequences seq;
  int channels, silu, rows_per_thread, row_tiles, step;
  int wide_weight;  // 16-byte loads of the coefficients
};

// V channels of a row in fp32, as pairs.
template <int V>
struct Row {
  float2 v[(V + 1) / 2];
};
template <typename T, int V>
__device__ __forceinline__ Row<V> widen(const Pack<T, V>& p) {
  Row<V> r;
#pragma unroll
  for (int i = 0; i < (V + 1) / 2; ++i) r.v[i] = pair_of(p, i);
  return r;
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> narrow(const Row<V>& r) {
  Pack<T, V> p;
#pragma unroll
  for (int i = 0; i < (V + 1) / 2; ++i) put_pair(p, i, r.v[i]);
  return p;
}

// A thread's coefficients, and one row of y from the K rows that end at it.
template <typename T, int V, int K, bool ACT>
struct ConvThread {
  static constexpr int P = (V + 1) / 2;
  float2 w[K][P], bias[P];

  __device__ __forceinline__ void load(const ConvArgs& a, int c) {
    float flat[V * K];
    if (V * K % 4 == 0 && a.wide_weight) {
#pragma unroll
      for (int i = 0; i < V * K / 4; ++i) {
        const float4 v = ldg4(a.w + (size_t)c * K + 4 * i);
        flat[4 * i] = v.x, flat[4 * i + 1] = v.y, flat[4 * i + 2] = v.z, flat[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V * K; ++i) flat[i] = __ldg(a.w + (size_t)c * K + i);
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int lo = 2 * p, hi = V > 1 ? 2 * p + 1 : 0;
#pragma unroll
      for (int j = 0; j < K; ++j) w[j][p] = make_float2(flat[lo * K + j], flat[hi * K + j]);
      bias[p] = a.bias ? make_float2(__ldg(a.bias + c + lo), __ldg(a.bias + c + hi)) : make_float2(0.f, 0.f);
    }
  }
  __device__ __forceinline__ Row<V> row(const Row<V>* win) const {
    Row<V> out;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float2 v = bias[p];
#pragma unroll
      for (int j = 0; j < K; ++j) v = f2fma(w[j][p], win[j].v[p], v);
      out.v[p] = ACT ? silu2<T>(v) : v;
    }
    return out;
  }
};

// Single rows, one per stream: K - 1 history rows and the new one in, the row
// of y and the advanced history out. A thread does `rows_per_thread` streams,
// two of them at a time, with one load of its coefficients.
template <typename T, int V, int K, bool ACT>
__global__ void __launch_bounds__(kConvThreads) conv_step_kernel(const __grid_constant__ ConvArgs a) {
  constexpr int H = K - 1, U = 2;
  using P = Pack<T, V>;
  grid_dependency_sync();
  const Sequences& q = a.seq;
  const int vecs = a.channels / V;
  const long long idx = (long long)blockIdx.x * kConvThreads + threadIdx.x;
  const long long tile = idx / vecs;
  if (tile >= a.row_tiles) return;
  const int c = (int)(idx - tile * vecs) * V;
  const size_t table = (size_t)H * a.channels;
  const T* x = static_cast<const T*>(a.x) + c;
  T* y = static_cast<T*>(a.y) + c;
  T* pool = static_cast<T*>(a.pool) + c;
  const int first = (int)tile * a.rows_per_thread, last = min(first + a.rows_per_thread, q.rows);
  ConvThread<T, V, K, ACT> th;
  th.load(a, c);
  for (int r0 = first; r0 < last; r0 += U) {
    P win[U][K];
    SlotRef st[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r0 + u >= last) break;
      st[u] = slot_of(q, r0 + u);
      const bool held = st[u].slot >= 0 && st[u].read >= 0;
      const T* from = pool + (2 * (size_t)max(st[u].slot, 0) + max(st[u].read, 0)) * table;
#pragma unroll
      for (int j = 0; j < H; ++j) win[u][j] = held ? load_pack<T, V>(from + (size_t)j * a.channels) : P{};
      win[u][H] = load_const<T, V>(x + (r0 + u) * a.x_stride);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r0 + u >= last || st[u].bad) continue;
      if (st[u].slot >= 0) {
        T* to = pool + (2 * (size_t)st[u].slot + st[u].write) * table;
#pragma unroll
        for (int j = 0; j < H; ++j) store_pack<T, V>(to + (size_t)j * a.channels, win[u][j + 1]);
      }
      Row<V> rows[K];
#pragma unroll
      for (int j = 0; j < K; ++j) rows[j] = widen(win[u][j]);
      store_pack<T, V>(y + (r0 + u) * a.y_stride, narrow<T, V>(th.row(rows)));
    }
  }
}

template <typename T, int V, int K, bool ACT>
__global__ void __launch_bounds__(kConvThreads, conv_blocks<K>()) conv_kernel(const __grid_constant__ ConvArgs a) {
  constexpr int H = K - 1, U = 4, D = kConvDepth;
  using P = Pack<T, V>;
  // Each thread's next D rows: it copies, waits for and reads its own alone.
  __shared__ P s_ring[D][kConvThreads];
  grid_dependency_sync();
  const Sequences& q = a.seq;
  const int vecs = a.channels / V;
  const long long idx = (long long)blockIdx.x * kConvThreads + threadIdx.x;
  const long long work = idx / vecs;
  const int c = (int)(idx - work * vecs) * V;
  const size_t table = (size_t)H * a.channels;
  const T* x = static_cast<const T*>(a.x) + c;
  T* pool = static_cast<T*>(a.pool) + c;
  if (work >= a.row_tiles) {
    // One item per sequence: checks its offsets; a sequence of no rows hands
    // its history on as it is.
    const long long s = work - a.row_tiles;
    if (s >= q.n || !q.offsets) return;
    const Span sp = span_of(q, (int)s);
    if (sp.begin > sp.end) record_error(q.status, kDevBadOffsets);
    if (sp.begin != sp.end || !a.pool) return;
    const SlotRef st = slot_of(q, (int)s);
    if (st.bad) return;
    const T* from = pool + (2 * (size_t)st.slot + (st.read < 0 ? 0 : st.read)) * table;
    T* to = pool + (2 * (size_t)st.slot + st.write) * table;
    for (int j = 0; j < H; ++j)
      store_pack<T, V>(to + (size_t)j * a.channels, st.read < 0 ? P{} : load_pack<T, V>(from + (size_t)j * a.channels));
    return;
  }
  int r = (int)(work * a.rows_per_thread);
  const int first = r, last = (int)min((long long)r + a.rows_per_thread, (long long)q.rows);
  P* ring = &s_ring[0][threadIdx.x];
  const T* px = x + r * a.x_stride;  // the next row to copy
  T* py = static_cast<T*>(a.y) + c + r * a.y_stride;
#pragma unroll
  for (int u = 0; u < D; ++u) {
    if (r + u < last) copy_pack<T, V>(ring + u * kConvThreads, px);
    copy_commit();
    px += a.x_stride;
  }
  ConvThread<T, V, K, ACT> th;
  th.load(a, c);
  Row<V> win[H + U];
  Span sp{0, 0};
  SlotRef st{-1, -1, -1, false};
  bool live = false;
  while (r < last) {
    if (r >= sp.end) {
      // The sequence that row r belongs to, and the K - 1 rows above it.
      const int s = sequence_at(q, r);
      sp = s < 0 ? Span{1, 0} : span_of(q, s);
      live = r >= sp.begin && r < sp.end;
      if (live) {
        st = slot_of(q, s);
        live = !st.bad;
        const T* hist = pool + (2 * (size_t)max(st.slot, 0) + max(st.read, 0)) * table;
#pragma unroll
        for (int j = 0; j < H; ++j) {
          const int row = r - H + j;
          if (row >= sp.begin)
            win[j] = widen(load_const<T, V>(x + row * a.x_stride));
          else if (st.slot >= 0 && st.read >= 0)
            win[j] = widen(load_pack<T, V>(hist + (size_t)(row - sp.begin + H) * a.channels));
          else
            win[j] = Row<V>{};
        }
      } else {
        sp.end = r + 1;  // a row of no sequence: left as it is
      }
    }
    const int stop = min(sp.end, last), at = (r - first) % D;
    if (at % U == 0 && r + U <= stop) {
      copy_wait<D - U>();
#pragma unroll
      for (int u = 0; u < U; ++u) win[H + u] = widen(ring[(at + u) * kConvThreads]);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (live) store_pack<T, V>(py, narrow<T, V>(th.row(win + u)));
        py += a.y_stride;
      }
      // Into the places just read: after the stores, which have waited for the reads.
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r + D + u < last) copy_pack<T, V>(ring + (at + u) * kConvThreads, px);
        copy_commit();
        px += a.x_stride;
      }
#pragma unroll
      for (int j = 0; j < H; ++j) win[j] = win[j + U];
      r += U;
    } else {
      copy_wait<D - 1>();
      win[H] = widen(ring[at * kConvThreads]);
      if (live) store_pack<T, V>(py, narrow<T, V>(th.row(win)));
      py += a.y_stride;
      if (r + D < last) copy_pack<T, V>(ring + at * kConvThreads, px);
      copy_commit();
      px += a.x_stride;
#pragma unroll
      for (int j = 0; j < H; ++j) win[j] = win[j + 1];
      ++r;
    }
    if (live && r == sp.end && st.slot >= 0) {
      T* to = pool + (2 * (size_t)st.slot + st.write) * table;
#pragma unroll
      for (int j = 0; j < H; ++j) store_pack<T, V>(to + (size_t)j * a.channels, narrow<T, V>(win[j]));
    }
  }
}

template <typename T, int V, int K, bool ACT>
cudaError_t launch_one(unsigned grid, cudaStream_t stream, const ConvArgs& a) {
  if (a.step) return launch_op(conv_step_kernel<T, V, K, ACT>, grid, kConvThreads, 0, stream, a);
  return launch_op(conv_kernel<T, V, K, ACT>, grid, kConvThreads, 0, stream, a);
}

template <typename T, int V, int K>
cudaError_t launch_act(unsigned grid, cudaStream_t stream, const ConvArgs& a) {
  return a.silu ? launch_one<T, V, K, true>(grid, stream, a) : launch_one<T, V, K, false>(grid, stream, a);
}

template <typename T, int V>
cudaError_t launch_taps(int taps, unsigned grid, cudaStream_t stream, const ConvArgs& a) {
  switch (taps) {
    case 2: return launch_act<T, V, 2>(grid, stream, a);
    case 3: return launch_act<T, V, 3>(grid, stream, a);
    case 4: return launch_act<T, V, 4>(grid, stream, a);
    case 5: return launch_act<T, V, 5>(grid, stream, a);
    case 6: return launch_act<T, V, 6>(grid, stream, a);
    case 7: return launch_act<T, V, 7>(grid, stream, a);
    case 8: return launch_act<T, V, 8>(grid, stream, a);
    default: return cudaErrorInvalidValue;
  }
}

template <typename T>
cudaError_t launch_type(int taps, int v, unsigned grid, cudaStream_t stream, const ConvArgs& a) {
  return v == 4 ? launch_taps<T, 4>(taps, grid, stream, a) : launch_taps<T, 1>(taps, grid, stream, a);
}

}  // namespace

cudaError_t launch_causal_conv(const fav_conv_args& c, const Sequences& seq, cudaStream_t stream) {
  ConvArgs a{};
  a.x = c.x;
  a.y = c.y;
  a.x_stride = c.x_stride;
  a.y_stride = c.y_stride;
  a.w = c.weight;
  a.bias = c.bias;
  a.pool = c.state_pool;
  a.seq = seq;
  a.channels = c.channels;
  a.silu = c.activation == FAV_ACTIVATION_SILU;
  const int elem = elem_bytes(c.type);
  a.step = !seq.offsets && seq.length == 1;
  const bool wide = c.channels % 4 == 0 && aligned_for(c.x, c.x_stride, elem, 4) &&
                    aligned_for(c.y, c.y_stride, elem, 4) && aligned_for(c.state_pool, 0, elem, 4);
  const int v = wide ? 4 : 1;
  const long long vecs = c.channels / v;
  a.wide_weight = aligned_for(c.weight, 0, 4, 4) && v * c.taps % 4 == 0;
  // One wave of the threads that the SMs hold, so that every thread loads its
  // coefficients and finds its sequence once; at most 64 rows a thread. Single
  // rows: up to 4 a thread, for the coefficients.
  const long long blocks_per_sm = c.taps <= 4 ? conv_blocks<4>() : conv_blocks<8>();
  const long long wave = 148LL * kConvThreads * (a.step ? 4 : blocks_per_sm), most = a.step ? 4 : 64;
  long long rpt = ((long long)seq.rows * vecs + wave - 1) / wave;
  a.rows_per_thread = (int)(rpt < 1 ? 1 : rpt > most ? most : rpt);
  a.row_tiles = (int)(((long long)seq.rows + a.rows_per_thread - 1) / a.rows_per_thread);
  const long long items = ((long long)a.row_tiles + (seq.offsets ? seq.n : 0)) * vecs;
  if (items == 0) return cudaSuccess;
  const long long blocks = (items + kConvThreads - 1) / kConvThreads;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const unsigned grid = (unsigned)blocks;
  if (c.type == FAV_TYPE_F32) return launch_type<float>(c.taps, v, grid, stream, a);
  if (c.type == FAV_TYPE_BF16) return launch_type<__nv_bfloat16>(c.taps, v, grid, stream, a);
  return launch_type<__half>(c.taps, v, grid, stream, a);
}

}  // namespace fav
