// Short causal depthwise convolution with a carried history, for packed
// prompts and for single rows (one per stream), channels last:
//
//   y[t, c] = act(bias[c] + sum_j w[c, j] * x[t - (K - 1) + j, c]),  K = 2..8,
//
// rows before a sequence's first come from its slot's history (K - 1 rows, the
// most recent inputs, in x's type) or are zero. Sums run in fp32, oldest tap
// first, and round once to the output's type.
//
// Bound by memory: it reads x and writes y once. A thread owns up to 16 bytes
// of neighbouring channels and walks down `rows_per_thread` rows with the last
// K - 1 inputs in registers, so a tile re-reads only the K - 1 rows above it;
// four rows are loaded before they are used. Fewer rows a thread when there
// are few rows in all, so that a prompt of one stream still fills the GPU.
#include "fav_ops.cuh"

namespace fav {
namespace {

constexpr int kConvThreads = 128;

struct ConvArgs {
  const void* x;
  void* y;
  long long x_stride, y_stride;
  const float* w;
  const float* bias;
  void* pool;  // [num_slots][2][K - 1][channels]
  Sequences seq;
  int channels, silu, rows_per_thread, row_tiles;
};

template <typename T, int V, int K>
struct ConvThread {
  static constexpr int H = K - 1;
  float w[K][V], bias[V];
  bool act;

  __device__ __forceinline__ void load(const ConvArgs& a, int c) {
    act = a.silu != 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int j = 0; j < K; ++j) w[j][i] = __ldg(a.w + (size_t)(c + i) * K + j);
      bias[i] = a.bias ? __ldg(a.bias + c + i) : 0.f;
    }
  }
  __device__ __forceinline__ Pack<T, V> row(const Pack<T, V>* win) const {
    Pack<T, V> out;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float v = w[0][i] * to_f32(win[0].v[i]);
#pragma unroll
      for (int j = 1; j < K; ++j) v = fmaf(w[j][i], to_f32(win[j].v[i]), v);
      v += bias[i];
      out.v[i] = from_f32<T>(act ? silu(v) : v);
    }
    return out;
  }
};

template <typename T, int V, int K>
__global__ void __launch_bounds__(kConvThreads) conv_kernel(const __grid_constant__ ConvArgs a) {
  constexpr int H = K - 1, U = 4;
  using P = Pack<T, V>;
  grid_dependency_sync();
  const Sequences& q = a.seq;
  const int vecs = a.channels / V;
  const long long idx = (long long)blockIdx.x * kConvThreads + threadIdx.x;
  const long long work = idx / vecs;
  const int c = (int)(idx - work * vecs) * V;
  const size_t table = (size_t)H * a.channels;
  const T* x = static_cast<const T*>(a.x) + c;
  T* y = static_cast<T*>(a.y) + c;
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
  int r = (int)work * a.rows_per_thread;
  const int last = min(r + a.rows_per_thread, q.rows);
  ConvThread<T, V, K> th;
  th.load(a, c);
  while (r < last) {
    int s = sequence_at(q, r);
    Span sp = s < 0 ? Span{1, 0} : span_of(q, s);
    if (r < sp.begin || r >= sp.end) {
      ++r;  // a row of no sequence: left as it is
      continue;
    }
    const int stop = min(sp.end, last);
    const SlotRef st = slot_of(q, s);
    if (st.bad) {
      r = stop;
      continue;
    }
    P win[H + U];
    const T* hist = pool + (2 * (size_t)max(st.slot, 0) + max(st.read, 0)) * table;
#pragma unroll
    for (int j = 0; j < H; ++j) {
      const int row = r - H + j;
      if (row >= sp.begin)
        win[j] = load_pack<T, V>(x + row * a.x_stride);
      else if (st.slot >= 0 && st.read >= 0)
        win[j] = load_pack<T, V>(hist + (size_t)(row - sp.begin + H) * a.channels);
      else
        win[j] = P{};
    }
    for (; r + U <= stop; r += U) {
#pragma unroll
      for (int u = 0; u < U; ++u) win[H + u] = load_pack<T, V>(x + (r + u) * a.x_stride);
#pragma unroll
      for (int u = 0; u < U; ++u) store_pack<T, V>(y + (r + u) * a.y_stride, th.row(win + u));
#pragma unroll
      for (int j = 0; j < H; ++j) win[j] = win[j + U];
    }
    for (; r < stop; ++r) {
      win[H] = load_pack<T, V>(x + r * a.x_stride);
      store_pack<T, V>(y + r * a.y_stride, th.row(win));
#pragma unroll
      for (int j = 0; j < H; ++j) win[j] = win[j + 1];
    }
    if (stop == sp.end && st.slot >= 0) {
      T* to = pool + (2 * (size_t)st.slot + st.write) * table;
#pragma unroll
      for (int j = 0; j < H; ++j) store_pack<T, V>(to + (size_t)j * a.channels, win[j]);
    }
  }
}

template <typename T, int V>
cudaError_t launch_taps(int taps, unsigned grid, cudaStream_t stream, const ConvArgs& a) {
  switch (taps) {
    case 2: return launch_op(conv_kernel<T, V, 2>, grid, kConvThreads, 0, stream, a);
    case 3: return launch_op(conv_kernel<T, V, 3>, grid, kConvThreads, 0, stream, a);
    case 4: return launch_op(conv_kernel<T, V, 4>, grid, kConvThreads, 0, stream, a);
    default: break;
  }
  if constexpr (V <= 4) {
    switch (taps) {
      case 5: return launch_op(conv_kernel<T, V, 5>, grid, kConvThreads, 0, stream, a);
      case 6: return launch_op(conv_kernel<T, V, 6>, grid, kConvThreads, 0, stream, a);
      case 7: return launch_op(conv_kernel<T, V, 7>, grid, kConvThreads, 0, stream, a);
      case 8: return launch_op(conv_kernel<T, V, 8>, grid, kConvThreads, 0, stream, a);
      default: break;
    }
  }
  return cudaErrorInvalidValue;
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
  // 16 bytes a thread where the addresses allow it; 8 for a 16-bit type with
  // more than four taps, whose coefficients would not fit the registers.
  const int elem = elem_bytes(c.type);
  int v = c.type == FAV_TYPE_F32 || c.taps > 4 ? 4 : 8;
  for (; v > 1; v = v == 8 ? 4 : 1)
    if (c.channels % v == 0 && aligned_for(c.x, c.x_stride, elem, v) && aligned_for(c.y, c.y_stride, elem, v) &&
        aligned_for(c.state_pool, 0, elem, v))
      break;
  const long long vecs = c.channels / v;
  // At least about 1024 threads per SM before a thread takes more rows; 32
  // rows a thread re-read K - 1 rows above them, a tenth at most for K = 4.
  long long rpt = (long long)seq.rows * vecs / (148 * 1024);
  a.rows_per_thread = (int)(rpt < 1 ? 1 : rpt > 32 ? 32 : rpt);
  a.row_tiles = (seq.rows + a.rows_per_thread - 1) / a.rows_per_thread;
  const long long items = ((long long)a.row_tiles + (seq.offsets ? seq.n : 0)) * vecs;
  if (items == 0) return cudaSuccess;
  const long long blocks = (items + kConvThreads - 1) / kConvThreads;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const unsigned grid = (unsigned)blocks;
  if (c.type == FAV_TYPE_F32)
    return v == 4 ? launch_taps<float, 4>(c.taps, grid, stream, a) : launch_taps<float, 1>(c.taps, grid, stream, a);
  if (c.type == FAV_TYPE_BF16)
    return v == 8   ? launch_taps<__nv_bfloat16, 8>(c.taps, grid, stream, a)
           : v == 4 ? launch_taps<__nv_bfloat16, 4>(c.taps, grid, stream, a)
                    : launch_taps<__nv_bfloat16, 1>(c.taps, grid, stream, a);
  return v == 8   ? launch_taps<__half, 8>(c.taps, grid, stream, a)
         : v == 4 ? launch_taps<__half, 4>(c.taps, grid, stream, a)
                  : launch_taps<__half, 1>(c.taps, grid, stream, a);
}

}  // namespace fav
