// Shared by the stream operators (fav_conv.cu, fav_scan.cu, fav_norm.cu,
// fav_int4.cu): element types, vector loads and stores, and how packed rows
// belong to sequences and sequences to state slots.
#pragma once
#include "../../include/fast_audiovae_cuda.h"
#include "fav_device.cuh"
#include "fav_internal.h"

namespace fav {

// Codes an operator records in the caller's status word (first error wins).
constexpr uint32_t kDevBadOffsets = 0x201;  // offsets decrease or leave the rows
constexpr uint32_t kDevBadSlot = 0x202;     // a slot code names no slot of the pool

// ------------------------------------------------------------ element types
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

// The one rounding of a result to its stored type (nearest, ties to even).
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// V consecutive elements, moved by one access of V * sizeof(T) bytes.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}
// The same of memory that no thread writes during the kernel.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_const(const T* p) {
  constexpr int B = sizeof(T) * V;
  Pack<T, V> r;
  if constexpr (B == 16)
    *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(p));
  else if constexpr (B == 8)
    *reinterpret_cast<uint2*>(&r) = __ldg(reinterpret_cast<const uint2*>(p));
  else if constexpr (B == 4)
    *reinterpret_cast<uint32_t*>(&r) = __ldg(reinterpret_cast<const uint32_t*>(p));
  else
    *reinterpret_cast<uint16_t*>(&r) = __ldg(reinterpret_cast<const uint16_t*>(p));
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) {
  *reinterpret_cast<Pack<T, V>*>(p) = v;
}

// The same of memory that is not read or written again soon: it leaves the caches
// first.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_once(const T* p) {
  constexpr int B = sizeof(T) * V;
  Pack<T, V> r;
  if constexpr (B == 16)
    *reinterpret_cast<uint4*>(&r) = __ldcs(reinterpret_cast<const uint4*>(p));
  else if constexpr (B == 8)
    *reinterpret_cast<uint2*>(&r) = __ldcs(reinterpret_cast<const uint2*>(p));
  else if constexpr (B == 4)
    *reinterpret_cast<uint32_t*>(&r) = __ldcs(reinterpret_cast<const uint32_t*>(p));
  else
    *reinterpret_cast<uint16_t*>(&r) = __ldcs(reinterpret_cast<const uint16_t*>(p));
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_once(T* p, const Pack<T, V>& v) {
  constexpr int B = sizeof(T) * V;
  if constexpr (B == 16)
    __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&v));
  else if constexpr (B == 8)
    __stcs(reinterpret_cast<uint2*>(p), *reinterpret_cast<const uint2*>(&v));
  else if constexpr (B == 4)
    __stcs(reinterpret_cast<uint32_t*>(p), *reinterpret_cast<const uint32_t*>(&v));
  else
    __stcs(reinterpret_cast<uint16_t*>(p), *reinterpret_cast<const uint16_t*>(&v));
}

// A pack from global into shared memory, asynchronously; without an
// asynchronous copy of that size (2 bytes) at once.
template <typename T, int V>
__device__ __forceinline__ void copy_pack(Pack<T, V>* to, const T* from) {
  if constexpr (sizeof(T) * V == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
  else if constexpr (sizeof(T) * V >= 4)
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(to)), "l"(from), "n"(sizeof(T) * V)
                 : "memory");
  else
    *to = load_const<T, V>(from);
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Elements 2 i and 2 i + 1 of a pack in fp32, and back. V = 1: element 0 twice.
template <typename T, int V>
__device__ __forceinline__ float2 pair_of(const Pack<T, V>& p, int i) {
  return make_float2(to_f32(p.v[V > 1 ? 2 * i : 0]), to_f32(p.v[V > 1 ? 2 * i + 1 : 0]));
}
template <typename T, int V>
__device__ __forceinline__ void put_pair(Pack<T, V>& p, int i, float2 v) {
  p.v[V > 1 ? 2 * i : 0] = from_f32<T>(v.x);
  if constexpr (V > 1) p.v[2 * i + 1] = from_f32<T>(v.y);
}

__device__ __forceinline__ float ex2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float rcp_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// e^v, |v| <= 100, and of two. The argument of 2^x is off by the rounding of v log2 e,
// which grows with v (25 units of e^v at 20): in fp32 (T) what that and the rounding of
// log2 e itself lost is put back, e^v (1 + lost ln 2). Outputs of 16 bits do without.
constexpr float kLog2eLow = 1.9259629911266175e-8f;  // log2 e less the float
constexpr float kLn2 = 0.6931471805599453f;
template <typename T>
__device__ __forceinline__ float exp_for(float v) {
  const float t = v * kLog2e, e = ex2_approx(t);
  if constexpr (sizeof(T) < 4) return e;
  return e * fmaf(fmaf(v, kLog2eLow, fmaf(v, kLog2e, -t)), kLn2, 1.f);  // (infinity stays)
}
template <typename T>
__device__ __forceinline__ float2 exp_pair(float2 v) {
  const float2 t = f2mul(v, make_float2(kLog2e, kLog2e)), e = make_float2(ex2_approx(t.x), ex2_approx(t.y));
  if constexpr (sizeof(T) < 4) return e;
  const float2 lost = f2fma(v, make_float2(kLog2eLow, kLog2eLow),
                            f2fma(v, make_float2(kLog2e, kLog2e), make_float2(-t.x, -t.y)));
  return f2mul(e, f2fma(lost, make_float2(kLn2, kLn2), make_float2(1.f, 1.f)));
}

// v / (1 + e^-v) by the hardware's 2^x and 1/x (2 and 1 units in the last
// place). Below -100, where e^-v overflows, v stands at -100: the result is
// then 0, its limit, at -inf too. A NaN stays one.
template <typename T>
__device__ __forceinline__ float silu(float v) {
  v = max_nan(v, -100.f);
  return v * rcp_approx(1.f + exp_for<T>(sizeof(T) < 4 ? -v : -min_nan(v, 100.f)));
}
// The same of two, the multiplies and the sum packed.
template <typename T>
__device__ __forceinline__ float2 silu2(float2 v) {
  v = make_float2(max_nan(v.x, -100.f), max_nan(v.y, -100.f));
  const float2 m = sizeof(T) < 4 ? make_float2(-v.x, -v.y) : make_float2(-min_nan(v.x, 100.f), -min_nan(v.y, 100.f));
  const float2 s = f2add(exp_pair<T>(m), make_float2(1.f, 1.f));
  return f2mul(v, make_float2(rcp_approx(s.x), rcp_approx(s.y)));
}

// --------------------------------------------------------------- sequences
// Rows [begin, end) of one sequence; begin > end marks a bad pair of offsets.
struct Span {
  int begin, end;
};

struct Sequences {
  const int* offsets;  // device [n + 1], or nullptr: every sequence has ``length`` rows
  const int* codes;    // device [n], or nullptr: no states
  int n, length, rows, num_slots;
  uint32_t* status;
};

__device__ __forceinline__ Span span_of(const Sequences& q, int s) {
  if (!q.offsets) return {s * q.length, (s + 1) * q.length};
  const int b = q.offsets[s], e = q.offsets[s + 1];
  return b >= 0 && b <= e && e <= q.rows ? Span{b, e} : Span{1, 0};
}

// The last sequence that begins at or before row r (offsets increase), -1 if
// none does. Any content of ``offsets`` gives an index below n.
__device__ __forceinline__ int sequence_at(const Sequences& q, int r) {
  if (!q.offsets) return r / q.length;
  int lo = -1, hi = q.n - 1;
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (q.offsets[mid] <= r)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// A sequence's slot: where its state is read (table < 0: a fresh start, from
// zeros) and where the advanced state goes. slot < 0: no state, or a code
// outside the pool (recorded).
struct SlotRef {
  int slot, read, write;
  bool bad;
};

__device__ __forceinline__ SlotRef slot_of(const Sequences& q, int s) {
  if (!q.codes) return {-1, -1, -1, false};
  const int code = q.codes[s], slot = code >> 2;
  if (slot < 0 || slot >= q.num_slots) {
    record_error(q.status, kDevBadSlot);
    return {-1, -1, -1, true};
  }
  return {slot, code & 2 ? -1 : code & 1, (code & 1) ^ 1, false};
}

// ------------------------------------------------------------ host helpers
inline bool aligned_for(const void* p, long long stride, int elem, int width) {
  return !p || (reinterpret_cast<uintptr_t>(p) % (size_t)(elem * width) == 0 && stride % width == 0);
}

inline int elem_bytes(int type) { return type == FAV_TYPE_F32 ? 4 : 2; }

// Launches that follow one another in a stream overlap (see launch_overlapped).
template <typename Args>
inline cudaError_t launch_op(void (*kernel)(Args), dim3 grid, unsigned block, size_t smem, cudaStream_t stream,
                             const Args& a, unsigned cluster = 1) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) cudaGetLastError();  // reported here: clear it for the caller's next call
  return e;
}

}  // namespace fav
