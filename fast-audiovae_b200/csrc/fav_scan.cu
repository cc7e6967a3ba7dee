// Selective state space scan over the rows of packed sequences, and over single
// rows of many streams, channels last. Channel c of group g keeps N states:
//
//   delta    = softplus(dt[t, c] + dt_bias[c])        (or the sum itself)
//   h[n, c]  = exp(delta * a[n, c]) * h[n, c] + delta * x[t, c] * b[t, g, n]
//   y[t, c]  = (sum_n c[t, g, n] * h[n, c] + d[c] * x[t, c]) * silu(z[t, c])
//
// h starts from the sequence's slot of the state pool (fp32, [slot][2][N][C])
// or from zero and goes to the slot's other table. All of it runs in fp32 and
// y rounds once to its type. The decay is 2^(delta * a * log2 e): one multiply
// and one ex2 a state.
#include "fav_ops.cuh"

namespace fav {
namespace {

struct ScanArgs {
  const void *x, *dt, *z, *b, *c;
  void* y;
  long long x_stride, dt_stride, z_stride, b_stride, b_group, c_stride, c_group, y_stride;
  const float *a, *d, *dt_bias;
  float* pool;
  Sequences seq;
  int channels, states, groups, softplus;
  // Prompts: rows of a piece, pieces, 64-channel blocks of a group, and the
  // pieces' own results when sequences are split ([pieces][N][C], [pieces][C]).
  int piece_rows, pieces, group_blocks;
  float* piece_state;
  float* piece_delta;
};

// log(1 + e^v), exact to a few fp32 roundings on both sides of zero.
__device__ __forceinline__ float softplus_f32(float v) { return fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))); }

__device__ __forceinline__ float delta_of(const ScanArgs& a, float dt, int c) {
  const float v = a.dt_bias ? dt + __ldg(a.dt_bias + c) : dt;
  return a.softplus ? softplus_f32(v) : v;
}

// ------------------------------------------------------------- single rows
// One row per stream. Reading and writing the states is the whole cost (8 * N
// bytes a channel), so a thread moves V = 4 neighbouring channels of a state
// with 16-byte accesses; L lanes of a warp share a channel's states where
// there are too few channels and streams to fill the GPU.
constexpr int kStepThreads = 128;

template <typename T, int V, int L>
__global__ void __launch_bounds__(kStepThreads) scan_step_kernel(const __grid_constant__ ScanArgs a) {
  constexpr int W = 32 / L;  // channel vectors of a warp
  grid_dependency_sync();
  const Sequences& q = a.seq;
  const int vecs = a.channels / V;
  const int lane = threadIdx.x & 31, l = lane / W;
  const long long warp = ((long long)blockIdx.x * kStepThreads + threadIdx.x) >> 5;
  const long long item = warp * W + lane % W, items = (long long)q.n * vecs;
  const bool live = item < items;
  const int s = live ? (int)(item / vecs) : 0;
  const int c = live ? (int)(item - (long long)s * vecs) * V : 0;
  const int g = c / (a.channels / a.groups);
  SlotRef st{-1, -1, -1, false};
  if (live) st = slot_of(q, s);
  const size_t table = (size_t)a.states * a.channels;
  const float* from = a.pool + (2 * (size_t)max(st.slot, 0) + max(st.read, 0)) * table + c;
  float* to = a.pool + (2 * (size_t)max(st.slot, 0) + max(st.write, 0)) * table + c;
  const Pack<T, V> xv = load_pack<T, V>(static_cast<const T*>(a.x) + s * a.x_stride + c);
  const Pack<T, V> dv = load_pack<T, V>(static_cast<const T*>(a.dt) + s * a.dt_stride + c);
  const T* bp = static_cast<const T*>(a.b) + s * a.b_stride + g * a.b_group;
  const T* cp = static_cast<const T*>(a.c) + s * a.c_stride + g * a.c_group;
  float scale[V], dx[V], y[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float delta = delta_of(a, to_f32(dv.v[i]), c + i);
    scale[i] = delta * kLog2e;
    dx[i] = delta * to_f32(xv.v[i]);
    y[i] = 0.f;
  }
  const bool held = st.slot >= 0 && st.read >= 0, keep = live && st.slot >= 0;
#pragma unroll 4
  for (int n = l; n < a.states; n += L) {
    const Pack<float, V> av = load_pack<float, V>(a.a + (size_t)n * a.channels + c);
    Pack<float, V> h = held ? load_pack<float, V>(from + (size_t)n * a.channels) : Pack<float, V>{};
    const float bn = to_f32(bp[n]), cn = to_f32(cp[n]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      h.v[i] = fmaf(ex2_approx(scale[i] * av.v[i]), h.v[i], dx[i] * bn);
      y[i] = fmaf(h.v[i], cn, y[i]);
    }
    if (keep) store_pack<float, V>(to + (size_t)n * a.channels, h);
  }
#pragma unroll
  for (int o = W; o < 32; o *= 2)
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] += __shfl_xor_sync(0xffffffffu, y[i], o);
  if (!live || st.bad || l != 0) return;
  Pack<T, V> out, zv{};
  if (a.z) zv = load_pack<T, V>(static_cast<const T*>(a.z) + s * a.z_stride + c);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float v = a.d ? fmaf(__ldg(a.d + c + i), to_f32(xv.v[i]), y[i]) : y[i];
    if (a.z) v *= silu(to_f32(zv.v[i]));
    out.v[i] = from_f32<T>(v);
  }
  store_pack<T, V>(static_cast<T*>(a.y) + s * a.y_stride + c, out);
}

// ----------------------------------------------------------------- prompts
// A block owns CH neighbouring channels of one group over one piece (a whole
// sequence, or a run of its rows). L lanes share a channel, eight states each
// in registers. Per tile of 32 rows all threads first form delta and delta * x
// (the softplus once per value, not once per state) and widen b and c in shared
// memory; then each thread steps through the rows, and y replaces delta in
// place; then all threads add d * x, gate and store.
//
// Bound by ex2: T * C * N of them at 16 a clock and SM.
constexpr int kTileRows = 32;
constexpr int kLaneStates = 8;

// A piece: rows [begin, end) of sequence ``seq``; pieces ``first``.. of the
// same sequence precede it.
struct Piece {
  int seq, first, begin, end;
  bool ok, last;
};

__device__ __forceinline__ Piece piece_at(const ScanArgs& a, int p) {
  const Sequences& q = a.seq;
  const int R = a.piece_rows;
  Piece r{0, 0, 0, 0, false, false};
  if (!q.offsets) {
    const int per = (q.length - 1) / R + 1;
    r.seq = p / per;
    r.first = r.seq * per;
    const int base = r.seq * q.length, end = base + q.length;
    r.begin = base + (p - r.first) * R;
    r.end = min(r.begin + R, end);
    r.last = r.end == end;
    r.ok = true;
    return r;
  }
  // Pieces of packed sequences end where the sequence or a run of R rows of
  // the whole does. Sequence s owns the numbers from offsets[s] / R + s on:
  // they grow with s, and every sequence has one, an empty one too.
  int lo = -1, hi = q.n - 1;
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if ((long long)(q.offsets[mid] / R) + mid <= p)
      lo = mid;
    else
      hi = mid - 1;
  }
  if (lo < 0) return r;
  const Span sp = span_of(q, lo);
  if (sp.begin > sp.end) return r;
  r.seq = lo;
  r.first = sp.begin / R + lo;
  const int k = p - r.first;
  const long long tile = (long long)(sp.begin / R + k) * R;
  if (k > 0 && tile >= sp.end) return r;
  r.begin = k ? (int)tile : sp.begin;
  r.end = (int)min((long long)sp.end, tile + R);
  r.last = r.end == sp.end;
  r.ok = true;
  return r;
}

// PARTIAL: the state a piece reaches by itself and its sum of delta, for the
// pieces behind it; no y.
template <typename T, int V, int L, int CH, bool PARTIAL>
__global__ void __launch_bounds__(CH* L) scan_kernel(const __grid_constant__ ScanArgs a) {
  constexpr int NT = CH * L, S = kLaneStates, NP = S * L, R = kTileRows;
  constexpr int VPT = (R * CH / V + NT - 1) / NT;  // vectors of a tile per thread
  __shared__ __align__(16) float s_delta[R][CH];
  __shared__ __align__(16) float s_dx[R][CH];
  __shared__ __align__(16) float s_b[R][NP];
  __shared__ __align__(16) float s_c[PARTIAL ? 1 : R][NP];
  grid_dependency_sync();
  const Sequences& q = a.seq;
  const int blocks = a.group_blocks * a.groups;
  const int p = blockIdx.x / blocks, cb = blockIdx.x - p * blocks;
  const int g = cb / a.group_blocks, width = a.channels / a.groups;
  const int c_in = (cb - g * a.group_blocks) * CH;  // first channel inside the group
  const int c0 = g * width + c_in, count = min(CH, width - c_in);
  if (!PARTIAL && cb == 0 && p < q.n && threadIdx.x == 0) {
    const Span sp = span_of(q, p);
    if (sp.begin > sp.end) record_error(q.status, kDevBadOffsets);
  }
  const Piece pc = piece_at(a, p);
  if (!pc.ok || (PARTIAL && pc.last)) return;
  const SlotRef st = slot_of(q, pc.seq);
  if (st.bad) return;
  const int ch = threadIdx.x / L, l = threadIdx.x % L;
  const bool mine = ch < count;
  const int c = c0 + (mine ? ch : 0);
  const size_t table = (size_t)a.states * a.channels;
  float decay[S], h[S];
#pragma unroll
  for (int j = 0; j < S; ++j) {
    const int n = l * S + j;
    decay[j] = n < a.states ? __ldg(a.a + (size_t)n * a.channels + c) * kLog2e : 0.f;
    h[j] = 0.f;
  }
  if (p == pc.first) {
    if (st.slot >= 0 && st.read >= 0) {
      const float* from = a.pool + (2 * (size_t)st.slot + st.read) * table + c;
#pragma unroll
      for (int j = 0; j < S; ++j)
        if (l * S + j < a.states) h[j] = from[(size_t)(l * S + j) * a.channels];
    }
  } else if (!PARTIAL) {
    // Join the pieces before this one, in order.
    for (int k = pc.first; k < p; ++k) {
      const float sum = a.piece_delta[(size_t)k * a.channels + c];
      const float* from = a.piece_state + (size_t)k * table + c;
#pragma unroll
      for (int j = 0; j < S; ++j) {
        const float v = l * S + j < a.states ? from[(size_t)(l * S + j) * a.channels] : 0.f;
        h[j] = k == pc.first ? v : fmaf(ex2_approx(sum * decay[j]), h[j], v);
      }
    }
  }
  float total = 0.f;  // PARTIAL: sum of delta
  const T* xb = static_cast<const T*>(a.x) + c0;
  const T* db = static_cast<const T*>(a.dt) + c0;
  const T* zb = static_cast<const T*>(a.z) + c0;
  T* yb = static_cast<T*>(a.y) + c0;
  const T* bb = static_cast<const T*>(a.b) + g * a.b_group;
  const T* cc = static_cast<const T*>(a.c) + g * a.c_group;
  for (int t0 = pc.begin; t0 < pc.end; t0 += R) {
    const int rows = min(R, pc.end - t0);
    Pack<T, V> xv[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int e = (k * NT + threadIdx.x) * V, r = e / CH, i = e % CH;
      if (R * CH / V % NT && r >= R) continue;
      const bool in = r < rows && i < count;
      Pack<T, V> dv{};
      xv[k] = Pack<T, V>{};
      if (in) {
        xv[k] = load_pack<T, V>(xb + (t0 + r) * a.x_stride + i);
        dv = load_pack<T, V>(db + (t0 + r) * a.dt_stride + i);
      }
      Pack<float, V> delta, dx;
#pragma unroll
      for (int u = 0; u < V; ++u) {
        // A row behind the last: delta = 0 keeps every state as it is.
        delta.v[u] = in ? delta_of(a, to_f32(dv.v[u]), c0 + i + u) : 0.f;
        dx.v[u] = in ? delta.v[u] * to_f32(xv[k].v[u]) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < V; ++u) {
        s_delta[r][i + u] = delta.v[u];
        s_dx[r][i + u] = dx.v[u];
      }
    }
    for (int e = threadIdx.x; e < R * NP; e += NT) {
      const int r = e / NP, n = e % NP;
      const bool in = r < rows && n < a.states;
      s_b[r][n] = in ? to_f32(bb[(t0 + r) * a.b_stride + n]) : 0.f;
      if (!PARTIAL) s_c[r][n] = in ? to_f32(cc[(t0 + r) * a.c_stride + n]) : 0.f;
    }
    __syncthreads();
#pragma unroll 4
    for (int r = 0; r < R; ++r) {
      const float delta = s_delta[r][ch], dx = s_dx[r][ch];
      float y = 0.f;
#pragma unroll
      for (int j = 0; j < S; j += 4) {
        const float4 bv = *reinterpret_cast<const float4*>(&s_b[r][l * S + j]);
        h[j] = fmaf(ex2_approx(delta * decay[j]), h[j], dx * bv.x);
        h[j + 1] = fmaf(ex2_approx(delta * decay[j + 1]), h[j + 1], dx * bv.y);
        h[j + 2] = fmaf(ex2_approx(delta * decay[j + 2]), h[j + 2], dx * bv.z);
        h[j + 3] = fmaf(ex2_approx(delta * decay[j + 3]), h[j + 3], dx * bv.w);
        if constexpr (!PARTIAL) {
          const float4 cv = *reinterpret_cast<const float4*>(&s_c[r][l * S + j]);
          y = fmaf(h[j], cv.x, y);
          y = fmaf(h[j + 1], cv.y, y);
          y = fmaf(h[j + 2], cv.z, y);
          y = fmaf(h[j + 3], cv.w, y);
        }
      }
      if constexpr (PARTIAL) {
        total += delta;
      } else {
#pragma unroll
        for (int o = 1; o < L; o *= 2) y += __shfl_xor_sync(0xffffffffu, y, o);
        if (l == 0) s_delta[r][ch] = y;  // the channel's lanes have all read delta: they are in one warp
      }
    }
    __syncthreads();
    if constexpr (!PARTIAL) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int e = (k * NT + threadIdx.x) * V, r = e / CH, i = e % CH;
        if (r >= rows || i >= count) continue;
        Pack<T, V> out, zv{};
        if (a.z) zv = load_pack<T, V>(zb + (t0 + r) * a.z_stride + i);
#pragma unroll
        for (int u = 0; u < V; ++u) {
          const float y = s_delta[r][i + u];
          float v = a.d ? fmaf(__ldg(a.d + c0 + i + u), to_f32(xv[k].v[u]), y) : y;
          if (a.z) v *= silu(to_f32(zv.v[u]));
          out.v[u] = from_f32<T>(v);
        }
        store_pack<T, V>(yb + (t0 + r) * a.y_stride + i, out);
      }
      __syncthreads();
    }
  }
  if (!mine) return;
  if (PARTIAL) {
    float* to = a.piece_state + (size_t)p * table + c;
#pragma unroll
    for (int j = 0; j < S; ++j)
      if (l * S + j < a.states) to[(size_t)(l * S + j) * a.channels] = h[j];
    if (l == 0) a.piece_delta[(size_t)p * a.channels + c] = total;
  } else if (pc.last && st.slot >= 0) {
    float* to = a.pool + (2 * (size_t)st.slot + st.write) * table + c;
#pragma unroll
    for (int j = 0; j < S; ++j)
      if (l * S + j < a.states) to[(size_t)(l * S + j) * a.channels] = h[j];
  }
}

template <typename T, int V>
cudaError_t launch_step(const ScanArgs& a, cudaStream_t stream) {
  const long long items = (long long)a.seq.n * (a.channels / V);
  // Lanes per channel vector: more while the call has under 1024 threads an SM
  // and every lane still has states.
  int lanes = 1;
  while (lanes < 16 && items * lanes < 148 * 1024 && lanes * 4 <= a.states) lanes *= 4;
  const long long blocks = (items * lanes + kStepThreads - 1) / kStepThreads;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (lanes == 16) return launch_op(scan_step_kernel<T, V, 16>, (unsigned)blocks, kStepThreads, 0, stream, a);
  if (lanes == 4) return launch_op(scan_step_kernel<T, V, 4>, (unsigned)blocks, kStepThreads, 0, stream, a);
  return launch_op(scan_step_kernel<T, V, 1>, (unsigned)blocks, kStepThreads, 0, stream, a);
}

template <typename T, int V, int L, int CH>
cudaError_t launch_pieces(const ScanArgs& a, cudaStream_t stream) {
  const long long blocks = (long long)a.pieces * a.group_blocks * a.groups;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (a.piece_state) {
    const cudaError_t e = launch_op(scan_kernel<T, V, L, CH, true>, (unsigned)blocks, CH * L, 0, stream, a);
    if (e != cudaSuccess) return e;
  }
  return launch_op(scan_kernel<T, V, L, CH, false>, (unsigned)blocks, CH * L, 0, stream, a);
}

int lanes_for(int states) {
  int lanes = 1;
  while (lanes * kLaneStates < states) lanes *= 2;
  return lanes;
}
int block_channels(int lanes) { return lanes <= 8 ? 64 : 32; }

template <typename T, int V>
cudaError_t launch_lanes(const ScanArgs& a, cudaStream_t stream) {
  switch (lanes_for(a.states)) {
    case 1: return launch_pieces<T, V, 1, 64>(a, stream);
    case 2: return launch_pieces<T, V, 2, 64>(a, stream);
    case 4: return launch_pieces<T, V, 4, 64>(a, stream);
    case 8: return launch_pieces<T, V, 8, 64>(a, stream);
    default: return launch_pieces<T, V, 16, 32>(a, stream);
  }
}

template <typename T>
cudaError_t launch_type(const ScanArgs& a, bool step, bool wide, cudaStream_t stream) {
  if (step) return wide ? launch_step<T, 4>(a, stream) : launch_step<T, 1>(a, stream);
  return wide ? launch_lanes<T, 4>(a, stream) : launch_lanes<T, 1>(a, stream);
}

// How the rows are cut: piece_rows and pieces.
struct Split {
  int piece_rows, pieces;
  bool split;
};

Split split_of(const fav_scan_args& c, const Sequences& q) {
  const int lanes = lanes_for(c.states), ch = block_channels(lanes);
  const int width = c.channels / c.groups;
  const long long blocks = (long long)c.groups * ((width + ch - 1) / ch);
  const int warps = ch * lanes / 32;
  // A split scan forms every decay twice. It pays where whole sequences would
  // leave most of the GPU idle.
  const long long have = blocks * q.n * warps;
  const long long longest = q.offsets ? q.rows : q.length;
  if (have >= 148 * 8 || longest <= 2 * kTileRows) return {q.rows + 1, q.n, false};
  long long want = (148 * 24 + blocks * warps - 1) / (blocks * warps);
  long long rows = (q.rows + want - 1) / want;
  rows = (rows + kTileRows - 1) / kTileRows * kTileRows;
  if (rows < kTileRows) rows = kTileRows;
  if (q.offsets) return {(int)rows, (int)(q.rows / rows) + q.n, true};
  const long long per = (q.length - 1) / rows + 1;
  return {(int)rows, (int)(per * q.n), per > 1};
}

}  // namespace

size_t scan_workspace_bytes(const fav_scan_args& c, const Sequences& q) {
  if (q.rows == 0 || (!q.offsets && q.length == 1)) return 0;
  const Split s = split_of(c, q);
  return s.split ? (size_t)s.pieces * c.channels * (c.states + 1) * sizeof(float) : 0;
}

cudaError_t launch_selective_scan(const fav_scan_args& c, const Sequences& seq, cudaStream_t stream) {
  ScanArgs a{};
  a.x = c.x;
  a.dt = c.dt;
  a.z = c.z;
  a.b = c.b;
  a.c = c.c;
  a.y = c.y;
  a.x_stride = c.x_stride;
  a.dt_stride = c.dt_stride;
  a.z_stride = c.z_stride;
  a.y_stride = c.y_stride;
  a.b_stride = c.b_stride;
  a.b_group = c.b_group_stride;
  a.c_stride = c.c_stride;
  a.c_group = c.c_group_stride;
  a.a = c.a;
  a.d = c.d;
  a.dt_bias = c.dt_bias;
  a.pool = c.state_pool;
  a.seq = seq;
  a.channels = c.channels;
  a.states = c.states;
  a.groups = c.groups;
  a.softplus = c.softplus;
  if (seq.n == 0) return cudaSuccess;
  const bool step = !seq.offsets && seq.length == 1;
  const int elem = elem_bytes(c.type), width = c.channels / c.groups;
  const bool wide = width % 4 == 0 && aligned_for(c.x, c.x_stride, elem, 4) && aligned_for(c.dt, c.dt_stride, elem, 4) &&
                    aligned_for(c.z, c.z_stride, elem, 4) && aligned_for(c.y, c.y_stride, elem, 4) &&
                    aligned_for(c.a, 0, 4, 4) && aligned_for(c.state_pool, 0, 4, 4);
  if (!step) {
    const Split s = split_of(c, seq);
    a.piece_rows = s.piece_rows;
    a.pieces = s.pieces;
    const int ch = block_channels(lanes_for(c.states));
    a.group_blocks = (width + ch - 1) / ch;
    if (s.split) {
      a.piece_state = static_cast<float*>(c.workspace);
      a.piece_delta = a.piece_state + (size_t)s.pieces * c.channels * c.states;
    }
  }
  if (c.type == FAV_TYPE_F32) return launch_type<float>(a, step, wide, stream);
  if (c.type == FAV_TYPE_BF16) return launch_type<__nv_bfloat16>(a, step, wide, stream);
  return launch_type<__half>(a, step, wide, stream);
}

}  // namespace fav
