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
#include <algorithm>

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
  // Prompts: rows of a piece, pieces, blocks of channels of a group, and the
  // pieces' own results when sequences are split ([pieces][N][C], [pieces][C]).
  int piece_rows, pieces, group_blocks, by_length;
  float* piece_state;
  float* piece_delta;
};

// log(1 + e^v) = max(v, 0) + log(1 + e), e = e^-|v| in (0, 1]; the logarithm is
// 2 atanh(s), s = e / (2 + e) <= 1/3, whose series to s^13 is within 2e-8. No
// digits are lost where e is small, as they would be in the logarithm of 1 + e.
__device__ __forceinline__ float softplus_f32(float v) {
  const float e = ex2_approx(-kLog2e * fabsf(v));
  const float s = e * rcp_approx(2.f + e), q = s * s;
  float p = fmaf(q, 0.153846154f, 0.181818182f);  // 2/13, 2/11, ...
  p = fmaf(p, q, 0.222222222f);
  p = fmaf(p, q, 0.285714286f);
  p = fmaf(p, q, 0.4f);
  p = fmaf(p, q, 0.666666667f);
  p = fmaf(p, q, 2.f);
  return fmaf(p, s, max_nan(v, 0.f));
}

__device__ __forceinline__ float delta_of(const ScanArgs& a, float dt, int c) {
  const float v = a.dt_bias ? dt + __ldg(a.dt_bias + c) : dt;
  return a.softplus ? softplus_f32(v) : v;
}

// h * 2^p over the rows of a piece, as row after row would give it: by thirds, whose
// powers stay in range where 2^p does not and the product does (a growing state that
// is still zero would become inf * 0). Beyond 2^+-378 any h but 0 is inf or 0.
__device__ __forceinline__ float times_power(float h, float p) {
  const float e = ex2_approx(min_nan(max_nan(p * 0.333333333f, -126.f), 126.f));
  return h * e * e * e;
}

// ------------------------------------------------------------- single rows
// One row per stream. Reading and writing the states is the whole cost (8 * N
// bytes a channel), so a thread moves V = 4 neighbouring channels of a state
// with 16-byte accesses; L lanes of a warp share a channel's states where
// there are too few channels and streams to fill the GPU. 512 streams of 2048 x 16
// take 27 us, 71 % of the copy rate; without the hint that a state is not used
// again 30. (Holding `a` in registers over several streams took 51 us: the
// registers cost more warps than the reads of `a` time.)
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
  constexpr int B = 4;  // states of a lane on their way at once (four: 26.7 us, eight, with fewer warps: 27.3)
  for (int n0 = l; n0 < a.states; n0 += B * L) {
    Pack<float, V> h[B];
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const int n = n0 + k * L;
      h[k] = held && n < a.states ? load_once<float, V>(from + (size_t)n * a.channels) : Pack<float, V>{};
    }
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const int n = n0 + k * L;
      if (n >= a.states) break;
      const Pack<float, V> av = load_const<float, V>(a.a + (size_t)n * a.channels + c);
      const float bn = to_f32(bp[n]), cn = to_f32(cp[n]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        h[k].v[i] = fmaf(ex2_approx(scale[i] * av.v[i]), h[k].v[i], dx[i] * bn);
        y[i] = fmaf(h[k].v[i], cn, y[i]);
      }
      if (keep) store_once<float, V>(to + (size_t)n * a.channels, h[k]);
    }
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
    if (a.z) v *= silu<T>(to_f32(zv.v[i]));
    out.v[i] = from_f32<T>(v);
  }
  store_pack<T, V>(static_cast<T*>(a.y) + s * a.y_stride + c, out);
}

// ----------------------------------------------------------------- prompts
// A block owns CH neighbouring channels of one group over one piece (a whole
// sequence, or a run of its rows). L lanes share a channel, S states each in
// registers as pairs; every lane forms the channel's delta, so that nothing but
// b and c passes through shared memory in fp32. Tiles of 16 rows of x, dt and z
// are copied ahead of their use (cp.async) into two buffers, and y takes x's
// place in them until the tile is stored.
//
// Bound by the special function unit: T * C * N times ex2 at 16 a clock and SM,
// and four more a value for softplus and gate. 32 ragged prompts of up to 750 x
// 1536 x 16 in fp32 need 100 us of it and take 168: it is busy two thirds of the
// time on the SMs that have work, and the SMs' shares differ. (A quarter of the
// powers by a polynomial on the FMA pipe took 10 % longer: the instructions it
// adds are as scarce.)
constexpr int kTileRows = 16;
constexpr int kBlockChannels = 64;

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
    r.end = (int)min((long long)r.begin + R, (long long)end);  // the sum may pass 32 bits
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

// The sequence that is number `rank` by length, longest first (n <= NT): the
// blocks that start last are then the short ones (33 prompts of up to 750 rows
// 226 us in their own order, 171 in this one).
template <int NT>
__device__ __forceinline__ int sequence_by_length(const Sequences& q, int rank) {
  __shared__ int s_length[NT], s_pick;
  const int t = threadIdx.x;
  int length = -1;
  if (t < q.n) {
    const Span sp = span_of(q, t);
    length = max(sp.end - sp.begin, -1);
  }
  s_length[t] = length;
  __syncthreads();
  if (t < q.n) {
    int before = 0;
    for (int j = 0; j < q.n; ++j) before += s_length[j] > length || (s_length[j] == length && j < t);
    if (before == rank) s_pick = t;
  }
  __syncthreads();
  return s_pick;
}

// PARTIAL: the state a piece reaches by itself and its sum of delta, for the
// pieces behind it; no y.
template <typename T, bool WIDE, int S, int L, bool PARTIAL>
__global__ void __launch_bounds__(kBlockChannels* L, L == 2 ? 3 : 1) scan_kernel(const __grid_constant__ ScanArgs a) {
  constexpr int CH = kBlockChannels, R = kTileRows, Q = 8, NT = CH * L, NP = S * L, H = S / 2;
  constexpr int V = WIDE ? 16 / (int)sizeof(T) : 1;
  constexpr int kMaps = R * NP / NT;  // values of b (and of c) of a tile per thread
  static_assert(kMaps * NT == R * NP, "tile split");
  struct Tile {
    T x[R][CH], dt[R][CH], z[PARTIAL ? 1 : R][CH];
  };
  struct Maps {
    float b[R][NP], c[PARTIAL ? 1 : R][NP];
  };
  extern __shared__ __align__(16) unsigned char s_raw[];
  Tile* s_tile = reinterpret_cast<Tile*>(s_raw);                    // two
  Maps* s_maps = reinterpret_cast<Maps*>(s_raw + 2 * sizeof(Tile));  // two
  grid_dependency_sync();
  const Sequences& q = a.seq;
  const int blocks = a.group_blocks * a.groups;
  const int turn = blockIdx.x / blocks, cb = blockIdx.x - turn * blocks;
  const int p = a.by_length && !PARTIAL ? sequence_by_length<NT>(q, turn) : turn;
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

  const T* xb = static_cast<const T*>(a.x) + c0;
  const T* db = static_cast<const T*>(a.dt) + c0;
  const T* zb = static_cast<const T*>(a.z) + c0;
  const T* bb = static_cast<const T*>(a.b) + g * a.b_group;
  const T* cc = static_cast<const T*>(a.c) + g * a.c_group;
  const bool gate = !PARTIAL && a.z != nullptr;
  T maps_b[kMaps], maps_c[kMaps];
  // Where this thread's vectors of a tile lie, kVecs of them kHop rows apart, and
  // its values of b and c, kMaps of them kMapHop rows apart.
  constexpr int kAcross = CH / V, kVecs = (R * kAcross + NT - 1) / NT, kHop = NT / kAcross, kMapHop = NT / NP;
  static_assert(NT % kAcross == 0 && NT % NP == 0, "a thread keeps to one column");
  const int vr = threadIdx.x / kAcross, vi = threadIdx.x % kAcross * V;
  const int mr = threadIdx.x / NP, mn = threadIdx.x % NP;
  const bool v_in = vi < count, m_in = mn < a.states;
  const T* px = xb + (pc.begin + vr) * a.x_stride + vi;
  const T* pd = db + (pc.begin + vr) * a.dt_stride + vi;
  const T* pz = gate ? zb + (pc.begin + vr) * a.z_stride + vi : nullptr;
  const T* pb = bb + (pc.begin + mr) * a.b_stride + mn;
  const T* pq = cc + (pc.begin + mr) * a.c_stride + mn;
  // Starts the copies of the next tile, of `rows` rows, into buffer `to`, and its
  // b and c into registers.
  const auto fetch = [&](int rows, int to) {
    Tile& tile = s_tile[to];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int r = vr + k * kHop;
      if (v_in && r < rows) {
        copy_pack<T, V>(reinterpret_cast<Pack<T, V>*>(&tile.x[r][vi]), px + k * kHop * a.x_stride);
        copy_pack<T, V>(reinterpret_cast<Pack<T, V>*>(&tile.dt[r][vi]), pd + k * kHop * a.dt_stride);
        if constexpr (!PARTIAL)
          if (gate) copy_pack<T, V>(reinterpret_cast<Pack<T, V>*>(&tile.z[r][vi]), pz + k * kHop * a.z_stride);
      }
    }
    copy_commit();
#pragma unroll
    for (int k = 0; k < kMaps; ++k) {
      const bool in = m_in && mr + k * kMapHop < rows;
      maps_b[k] = in ? pb[k * kMapHop * a.b_stride] : from_f32<T>(0.f);
      if constexpr (!PARTIAL) maps_c[k] = in ? pq[k * kMapHop * a.c_stride] : from_f32<T>(0.f);
    }
    px += R * a.x_stride, pd += R * a.dt_stride, pb += R * a.b_stride;
    if constexpr (!PARTIAL) pz += gate ? R * a.z_stride : 0, pq += R * a.c_stride;
  };
  if (pc.begin < pc.end) fetch(min(R, pc.end - pc.begin), 0);

  const int ch = threadIdx.x / L, l = threadIdx.x % L;
  const bool mine = ch < count;
  const int c = c0 + (mine ? ch : 0);
  const size_t table = (size_t)a.states * a.channels;
  // State j of this lane is number l * S + j.
  const auto each = [&](auto&& f) {
#pragma unroll
    for (int j = 0; j < S; ++j)
      if (l * S + j < a.states) f(j, (size_t)(l * S + j) * a.channels);
  };
  float decay[S], h[S];
#pragma unroll
  for (int j = 0; j < S; ++j) decay[j] = h[j] = 0.f;
  // (finite, so that a row of delta = 0 keeps the state even where a is not)
  each([&](int j, size_t at) { decay[j] = max_nan(__ldg(a.a + at + c) * kLog2e, -3e38f); });
  if (p == pc.first) {
    if (st.slot >= 0 && st.read >= 0) {
      const float* from = a.pool + (2 * (size_t)st.slot + st.read) * table + c;
      each([&](int j, size_t at) { h[j] = from[at]; });
    }
  } else if (!PARTIAL) {
    // Join the pieces before this one, in order.
    const float* from = a.piece_state + (size_t)pc.first * table + c;
    const float* sums = a.piece_delta + (size_t)pc.first * a.channels + c;
    each([&](int j, size_t at) { h[j] = from[at]; });
#pragma unroll 4
    for (int k = pc.first + 1; k < p; ++k) {
      from += table;
      sums += a.channels;
      const float sum = *sums;
      each([&](int j, size_t at) { h[j] = times_power(h[j], sum * decay[j]) + from[at]; });
    }
  }
  const float bias = a.dt_bias ? __ldg(a.dt_bias + c) : 0.f, skip = !PARTIAL && a.d ? __ldg(a.d + c) : 0.f;
  float2 decay2[H], h2[H];
#pragma unroll
  for (int j = 0; j < H; ++j) {
    decay2[j] = make_float2(decay[2 * j], decay[2 * j + 1]);
    h2[j] = make_float2(h[2 * j], h[2 * j + 1]);
  }
  T* py = static_cast<T*>(a.y) + c0 + (pc.begin + vr) * a.y_stride + vi;
  float total = 0.f;  // PARTIAL: sum of delta
  int buffer = 0;
  for (int t0 = pc.begin; t0 < pc.end; t0 += R, buffer ^= 1) {
    const int rows = min(R, pc.end - t0);
    Tile& tile = s_tile[buffer];
    Maps& maps = s_maps[buffer];
#pragma unroll
    for (int k = 0; k < kMaps; ++k) {
      maps.b[mr + k * kMapHop][mn] = to_f32(maps_b[k]);
      if constexpr (!PARTIAL) maps.c[mr + k * kMapHop][mn] = to_f32(maps_c[k]);
    }
    copy_wait<0>();
    __syncthreads();
    if (t0 + R < pc.end) fetch(min(R, pc.end - t0 - R), buffer ^ 1);
    // Q rows at a time: their deltas together, then the states row by row, then
    // their outputs together, so that only the states' own chain is serial. A row
    // behind the last has delta = 0 and keeps every state as it is.
    for (int r0 = 0; r0 < rows; r0 += Q) {
      // Lane l forms delta of the rows u with u % L = l for the channel's others.
      float own_delta[Q / L], own_dx[Q / L], y[Q];
#pragma unroll
      for (int k = 0; k < Q / L; ++k) {
        const int r = r0 + k * L + l;
        const float v = to_f32(tile.dt[r][ch]) + bias;
        own_delta[k] = r < rows ? (a.softplus ? softplus_f32(v) : v) : 0.f;
        own_dx[k] = r < rows ? own_delta[k] * to_f32(tile.x[r][ch]) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < Q; ++u) {
        float delta = own_delta[u / L], dx = own_dx[u / L];
        if constexpr (L > 1) {
          delta = __shfl_sync(0xffffffffu, delta, u % L, L);
          dx = __shfl_sync(0xffffffffu, dx, u % L, L);
        }
        const float2 delta2 = make_float2(delta, delta), dx2 = make_float2(dx, dx);
        float2 y2 = make_float2(0.f, 0.f), y3 = y2;
#pragma unroll
        for (int j = 0; j < H; j += 2) {
          const float4 bv = *reinterpret_cast<const float4*>(&maps.b[r0 + u][l * S + 2 * j]);
          const float2 p0 = f2mul(delta2, decay2[j]), p1 = f2mul(delta2, decay2[j + 1]);
          h2[j] = f2fma(make_float2(ex2_approx(p0.x), ex2_approx(p0.y)), h2[j], f2mul(dx2, make_float2(bv.x, bv.y)));
          h2[j + 1] =
              f2fma(make_float2(ex2_approx(p1.x), ex2_approx(p1.y)), h2[j + 1], f2mul(dx2, make_float2(bv.z, bv.w)));
          if constexpr (!PARTIAL) {
            const float4 cv = *reinterpret_cast<const float4*>(&maps.c[r0 + u][l * S + 2 * j]);
            y2 = f2fma(h2[j], make_float2(cv.x, cv.y), y2);
            y3 = f2fma(h2[j + 1], make_float2(cv.z, cv.w), y3);
          }
        }
        if constexpr (PARTIAL) {
          total += delta;
        } else {
          y2 = f2add(y2, y3);
          y[u] = y2.x + y2.y;
        }
      }
      if constexpr (!PARTIAL) {
        // Sums over the lanes, row u's to lane u % L: each step halves the rows that
        // a lane has left.
#pragma unroll
        for (int o = 1, left = Q; o < L; o *= 2, left /= 2)
#pragma unroll
          for (int k = 0; k < left / 2; ++k) {
            const bool odd = l & o;
            const float send = odd ? y[2 * k] : y[2 * k + 1];
            y[k] = (odd ? y[2 * k + 1] : y[2 * k]) + __shfl_xor_sync(0xffffffffu, send, o);
          }
#pragma unroll
        for (int k = 0; k < Q / L; ++k) {
          const int r = r0 + k * L + l;
          float v = fmaf(skip, to_f32(tile.x[r][ch]), y[k]);
          if (gate) v *= silu<T>(to_f32(tile.z[r][ch]));
          tile.x[r][ch] = from_f32<T>(v);  // read by this lane alone
        }
      }
    }
    if constexpr (!PARTIAL) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        const int r = vr + k * kHop;
        if (v_in && r < rows)
          store_pack<T, V>(py + k * kHop * a.y_stride, *reinterpret_cast<const Pack<T, V>*>(&tile.x[r][vi]));
      }
      py += R * a.y_stride;
    }
  }
  if (!mine) return;
#pragma unroll
  for (int j = 0; j < H; ++j) h[2 * j] = h2[j].x, h[2 * j + 1] = h2[j].y;
  if (PARTIAL) {
    float* to = a.piece_state + (size_t)p * table + c;
    each([&](int j, size_t at) { to[at] = h[j]; });
    if (l == 0) a.piece_delta[(size_t)p * a.channels + c] = total;
  } else if (pc.last && st.slot >= 0) {
    float* to = a.pool + (2 * (size_t)st.slot + st.write) * table + c;
    each([&](int j, size_t at) { to[at] = h[j]; });
  }
}

template <typename T, int V>
cudaError_t launch_step(const ScanArgs& a, cudaStream_t stream) {
  const long long items = (long long)a.seq.n * (a.channels / V);
  // Four lanes per channel vector while one would leave an SM under 1024 threads,
  // sixteen while four would leave it under 128 (1 x 1024 channels 2.4 us, not 2.9).
  const int lanes = items >= 148 * 1024 ? 1 : items >= 148 * 32 ? 4 : 16;
  const long long blocks = (items * lanes + kStepThreads - 1) / kStepThreads;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (lanes == 16) return launch_op(scan_step_kernel<T, V, 16>, (unsigned)blocks, kStepThreads, 0, stream, a);
  if (lanes == 4) return launch_op(scan_step_kernel<T, V, 4>, (unsigned)blocks, kStepThreads, 0, stream, a);
  return launch_op(scan_step_kernel<T, V, 1>, (unsigned)blocks, kStepThreads, 0, stream, a);
}

template <typename T, bool WIDE, int S, int L, bool PARTIAL>
cudaError_t launch_scan(const ScanArgs& a, unsigned blocks, cudaStream_t stream) {
  constexpr int R = kTileRows;
  const size_t tile = (size_t)R * kBlockChannels * sizeof(T), maps = (size_t)R * S * L * sizeof(float);
  const size_t smem = PARTIAL ? 2 * (2 * tile + kBlockChannels * sizeof(T) + maps + S * L * sizeof(float))
                              : 2 * (3 * tile + 2 * maps);
  const auto kernel = scan_kernel<T, WIDE, S, L, PARTIAL>;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  return launch_op(kernel, blocks, kBlockChannels * L, smem, stream, a);
}

template <typename T, bool WIDE, int S, int L>
cudaError_t launch_pieces(const ScanArgs& a, cudaStream_t stream) {
  const long long blocks = (long long)a.pieces * a.group_blocks * a.groups;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (a.piece_state) {
    const cudaError_t e = launch_scan<T, WIDE, S, L, true>(a, (unsigned)blocks, stream);
    if (e != cudaSuccess) return e;
  }
  return launch_scan<T, WIDE, S, L, false>(a, (unsigned)blocks, stream);
}

// Lanes of a channel: 4 states each up to 8, 8 up to 64, 16 above. (16 states in
// one lane take a seventh fewer instructions, but leave too few warps: ragged
// prompts of 16 states 238 us, against 170 us with two lanes.)
int lanes_for(int states) {
  int lanes = 2;
  while (lanes < 8 && lanes * 8 < states) lanes *= 2;
  return lanes;
}

template <typename T, bool WIDE>
cudaError_t launch_lanes(const ScanArgs& a, cudaStream_t stream) {
  if (a.states <= 8) return launch_pieces<T, WIDE, 4, 2>(a, stream);
  switch (lanes_for(a.states)) {
    case 2: return launch_pieces<T, WIDE, 8, 2>(a, stream);
    case 4: return launch_pieces<T, WIDE, 8, 4>(a, stream);
    default: break;
  }
  return a.states <= 64 ? launch_pieces<T, WIDE, 8, 8>(a, stream) : launch_pieces<T, WIDE, 16, 8>(a, stream);
}

template <typename T>
cudaError_t launch_type(const ScanArgs& a, bool step, bool wide, cudaStream_t stream) {
  if (step) return wide ? launch_step<T, 4>(a, stream) : launch_step<T, 1>(a, stream);
  return wide ? launch_lanes<T, true>(a, stream) : launch_lanes<T, false>(a, stream);
}

// How the rows are cut: piece_rows and pieces.
struct Split {
  int piece_rows, pieces;
  bool split;
};

Split split_of(const fav_scan_args& c, const Sequences& q) {
  const int width = c.channels / c.groups;
  const long long blocks = (long long)c.groups * ((width + kBlockChannels - 1) / kBlockChannels);
  const int warps = kBlockChannels * lanes_for(c.states) / 32;
  // A split scan forms every decay twice: it pays where whole sequences leave an
  // SM fewer than six warps. Twelve an SM then: fewer leave it idle (one prompt of
  // 6000 x 1024: 88 us, with eight 130), more pieces take longer to join.
  const long long have = blocks * q.n * warps;
  const long long longest = q.offsets ? q.rows : q.length;
  if (have >= 148 * 6 || longest <= 4 * kTileRows) return {q.rows + 1, q.n, false};
  const long long want = (148 * 12 + blocks * warps - 1) / (blocks * warps);
  long long rows = (q.rows + want - 1) / want;
  rows = (rows + kTileRows - 1) / kTileRows * kTileRows;
  if (rows < 2 * kTileRows) rows = 2 * kTileRows;
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
  // Steps move four channels at a time, prompts 16 bytes.
  const int v = step ? 4 : 16 / elem;
  const bool wide = width % v == 0 && aligned_for(c.x, c.x_stride, elem, v) && aligned_for(c.dt, c.dt_stride, elem, v) &&
                    aligned_for(c.z, c.z_stride, elem, v) && aligned_for(c.y, c.y_stride, elem, v) &&
                    (!step || (aligned_for(c.a, 0, 4, 4) && aligned_for(c.state_pool, 0, 4, 4)));
  if (!step) {
    const Split s = split_of(c, seq);
    a.piece_rows = s.piece_rows;
    a.pieces = s.pieces;
    a.by_length = seq.offsets && !s.split && seq.n <= kBlockChannels;
    a.group_blocks = (width + kBlockChannels - 1) / kBlockChannels;
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
