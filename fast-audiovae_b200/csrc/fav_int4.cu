// Projection of the few rows of a step by 4-bit weights with group scales:
//
//   y[m, r] = bias[r] + sum_g scales[r, g] * sum_{k in g} x[m, k] * (q[r, k] - 8)
//
// The floor is reading the weights once (out * depth / 2 bytes: 2.8 us of 16 x
// 8192 x 4096, 0.7 us of 1 x 4096 x 2048). They take 12.4 and 4.8 us, with weights that
// are in L2 already 10.6 and 3.9: the chain of launch, weights, inputs, products and
// join, a few us long, and for more input rows the reading and arranging of inputs
// from L1. The codes minus 8 are exact in fp16 and bf16, so the inner sums run on the tensor cores with
// exact operands: mma.sync m16n8k16, 16 weight rows by 8 input rows, fp32
// accumulation (an input row or two cannot fill a tcgen05 tile, and the codes
// must pass the registers anyway to become operands). A block's sum is scaled
// and joined in fp32. fp32 inputs are cut into three bf16 parts of 8 bits each
// that add up to them exactly: three products, one accumulator.
//
// Layout. Weights stay as the caller has them, row after row. An MMA does not
// care in which order it walks k as long as both operands agree, so a lane
// takes W consecutive bytes (2 W values of k) of its two rows and the same
// values of k of its input row; four lanes make a k block of 8 W values. W is
// the widest of 16, 8 and 4 with blocks that a group's scale covers whole.
// A CTA owns 16 R rows and all of k; its NW warps take every NW-th k block and
// join through shared memory in a fixed order. Many warps with short loops hide
// more than few with long ones: a warp has U blocks of weights and inputs on
// their way at once, 16 bytes of weights a lane and row. (Twice and four times as
// much, 1 x 4096 x 2048 7.2 and 9.2 us instead of 4.8: straight code that runs once
// costs more to fetch than the wait it saves.)
// Sums of inputs times codes may leave fp32's range where the scaled ones do not
// (bf16 and fp32 inputs above 2^117; fp16 stays far below). A thread that finds
// such a sum forms it again, value by value and made smaller by 2^11: slow, but
// out of the way of every other call.
// Clusters that shared k and kept the inputs in shared memory took longer (7.0
// us): the exchange costs more than the reads it saves.
#include <type_traits>

#include "fav_ops.cuh"

namespace fav {
namespace {

struct Int4Args {
  const void* x;
  void* y;
  long long x_stride, y_stride;
  const uint8_t* weight;
  const float *scales, *bias;
  int rows, depth, out, group, groups;
};

// The MMA's operand type for inputs of type T, and the parts of an input.
template <typename T>
struct Int4Type {
  using M = T;
  static constexpr int kParts = 1;
};
template <>
struct Int4Type<float> {
  using M = __nv_bfloat16;
  static constexpr int kParts = 3;
};

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                          __nv_bfloat16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Codes j and j + 4 of a word of eight, minus 8, as a pair of operands. The
// code is put into the mantissa of 1024 (fp16) or 128 (bf16); taking 1032 or
// 136 away is exact.
__device__ __forceinline__ uint32_t code_pair(uint32_t word, int j, __half) {
  const uint32_t v = ((word >> (4 * j)) & 0x000f000fu) | 0x64006400u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), __floats2half2_rn(1032.f, 1032.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t code_pair(uint32_t word, int j, __nv_bfloat16) {
  const uint32_t v = ((word >> (4 * j)) & 0x000f000fu) | 0x43004300u;
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), __floats2bfloat162_rn(136.f, 136.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Eight consecutive inputs, and the words that the MMAs take of them: the pairs
// (0,4), (1,5), (2,6), (3,7) of each part.
template <typename T>
struct Inputs {
  uint32_t w[4 * sizeof(T) / 2];
};
template <bool WIDE, typename T>
__device__ __forceinline__ Inputs<T> load_inputs(const T* p, bool in) {
  constexpr int N = 4 * sizeof(T) / 2;
  Inputs<T> v;
  if constexpr (WIDE) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(p) + i / 4);
      v.w[i] = q.x, v.w[i + 1] = q.y, v.w[i + 2] = q.z, v.w[i + 3] = q.w;
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) v.w[i] = __float_as_uint(__ldg(p + i));
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v.w[i] = __ldg(h + 2 * i) | ((uint32_t)__ldg(h + 2 * i + 1) << 16);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v.w[i] = in ? v.w[i] : 0u;
  return v;
}

template <typename T>
__device__ __forceinline__ void input_pairs(const Inputs<T>& v, uint32_t (&b)[1][4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    b[0][2 * i] = __byte_perm(v.w[i], v.w[i + 2], 0x5410);
    b[0][2 * i + 1] = __byte_perm(v.w[i], v.w[i + 2], 0x7632);
  }
}
__device__ __forceinline__ void input_pairs(const Inputs<float>& v, uint32_t (&b)[3][4]) {
  uint32_t part[3][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // Truncation, so that the largest values do not round to infinity; what is
    // not finite stays in the first part alone (with a NaN's leading bit).
    const uint32_t bits = v.w[i];
    const bool finite = (bits & 0x7f800000u) != 0x7f800000u;
    const bool nan = !finite && (bits & 0x007fffffu);
    part[0][i] = (bits & 0xffff0000u) | (nan ? 0x00400000u : 0u);
    const float mid = __uint_as_float(bits) - __uint_as_float(bits & 0xffff0000u);
    part[1][i] = finite ? __float_as_uint(mid) & 0xffff0000u : 0u;
    part[2][i] = finite ? __float_as_uint(mid - __uint_as_float(part[1][i])) : 0u;
  }
#pragma unroll
  for (int q = 0; q < 3; ++q)
#pragma unroll
    for (int i = 0; i < 4; ++i) b[q][i] = __byte_perm(part[q][i], part[q][i + 4], 0x7632);
}

// W consecutive weight bytes of one lane and row.
template <int W>
struct Codes {
  uint32_t w[W / 4];
};
template <int W>
__device__ __forceinline__ Codes<W> load_codes(const uint8_t* p) {
  Codes<W> c;
  if constexpr (W == 16) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    c.w[0] = v.x, c.w[1] = v.y, c.w[2] = v.z, c.w[3] = v.w;
  } else if constexpr (W == 8) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    c.w[0] = v.x, c.w[1] = v.y;
  } else {
    c.w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
  return c;
}

// A warp's share of one output, k blocks `block`, `block` + step, ... of `width` values, by
// codes smaller and scales larger by 2^11, both exact: finite where the scaled sum is.
template <typename T>
__device__ __noinline__ float far_sum(const Int4Args& a, int row, int m, int block, int step, int width) {
  const T* x = static_cast<const T*>(a.x) + m * a.x_stride;
  const uint8_t* code = a.weight + (size_t)row * (a.depth / 2);
  const float* scale = a.scales + (size_t)row * a.groups;
  float sum = 0.f;
  for (int k0 = block * width; k0 < a.depth; k0 += step * width) {
    float part = 0.f;
#pragma unroll 1
    for (int k = k0; k < min(k0 + width, a.depth); ++k)
      part = fmaf(to_f32(x[k]), (float)((code[k / 2] >> (k % 2 * 4) & 15) - 8) * 0x1p-11f, part);
    sum = fmaf(scale[k0 / a.group] * 0x1p11f, part, sum);
  }
  return sum;
}

// R: tiles of 16 weight rows a warp; C: tiles of 8 input rows.
template <typename T, bool WIDE, int W, int R, int C, int NW>
__global__ void __launch_bounds__(32 * NW) int4_kernel(const __grid_constant__ Int4Args a) {
  using M = typename Int4Type<T>::M;
  constexpr int P = Int4Type<T>::kParts, KB = 8 * W, U = 16 / W;
  constexpr int kOut = 16 * R, kIn = 8 * C;
  extern __shared__ float s_dyn[];
  float (*s_sum)[kIn][kOut + 1] = reinterpret_cast<float (*)[kIn][kOut + 1]>(s_dyn);
  grid_dependency_sync();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int r0 = blockIdx.x * kOut, m0 = blockIdx.y * kIn;
  const int blocks = (a.depth + KB - 1) / KB;
  const size_t pitch = a.depth / 2;
  const uint8_t* wrow[R][2];
  const float* srow[R][2];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = min(r0 + 16 * r + 8 * h + g, a.out - 1);  // rows behind the last repeat it, unused
      wrow[r][h] = a.weight + row * pitch + t * W;
      srow[r][h] = a.scales + (size_t)row * a.groups;
    }
  const T* xrow[C];
#pragma unroll
  for (int c = 0; c < C; ++c)  // rows behind the last repeat it: their sums are not stored
    xrow[c] = static_cast<const T*>(a.x) + min(m0 + 8 * c + g, a.rows - 1) * a.x_stride;
  float sum[R][C][4] = {};
  for (int b0 = warp; b0 < blocks; b0 += NW * U) {
    Codes<W> code[U][R][2];
    float scale[U][R][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int blk = b0 + u * NW;
      const bool in = blk * KB + t * 2 * W < a.depth;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          code[u][r][h] = in ? load_codes<W>(wrow[r][h] + (size_t)blk * (KB / 2)) : Codes<W>{};
          scale[u][r][h] = blk < blocks ? __ldg(srow[r][h] + blk * KB / a.group) : 0.f;
        }
    }
    Inputs<T> in[U][W / 4][C];  // k behind the last reads as zero
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < W / 4; ++i)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const int k = (b0 + u * NW) * KB + t * 2 * W + 8 * i;
          in[u][i][c] = load_inputs<WIDE>(xrow[c] + (k < a.depth ? k : 0), k < a.depth);
        }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (b0 + u * NW >= blocks) break;
      float part[R][C][4] = {};
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        uint32_t op[R][2][4];  // two MMAs of a word of eight codes
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            op[r][j / 2][2 * (j % 2)] = code_pair(code[u][r][0].w[i], j, M{});
            op[r][j / 2][2 * (j % 2) + 1] = code_pair(code[u][r][1].w[i], j, M{});
          }
#pragma unroll
        for (int c = 0; c < C; ++c) {
          uint32_t part_in[P][4];
          input_pairs(in[u][i][c], part_in);
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int q = P - 1; q >= 0; --q) {
              mma_16816(part[r][c], op[r][0], part_in[q][0], part_in[q][1], M{});
              mma_16816(part[r][c], op[r][1], part_in[q][2], part_in[q][3], M{});
            }
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[r][c][e] = fmaf(scale[u][r][e / 2], part[r][c][e], sum[r][c][e]);
    }
  }
  // Accumulators 0, 1: weight row g, input rows 2 t and 2 t + 1; 2, 3: row g + 8.
  bool over = false;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s_sum[warp][8 * c + 2 * t + e % 2][16 * r + 8 * (e / 2) + g] = sum[r][c][e];
        over |= !(fabsf(sum[r][c][e]) < INFINITY);
      }
  if constexpr (!std::is_same<T, __half>::value) {
    if (over)
#pragma unroll 1
      for (int i = 0; i < R * C * 4; ++i) {
        const int c = 8 * (i / 4 % C) + 2 * t + i % 2, r = 16 * (i / 4 / C) + 8 * (i / 2 % 2) + g;
        float& v = s_sum[warp][c][r];
        if (!(fabsf(v) < INFINITY) && m0 + c < a.rows && r0 + r < a.out)
          v = far_sum<T>(a, r0 + r, m0 + c, warp, NW, KB);
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kIn * kOut; i += 32 * NW) {
    const int c = i / kOut, r = i % kOut, m = m0 + c, row = r0 + r;
    if (m >= a.rows || row >= a.out) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += s_sum[w][c][r];
    static_cast<T*>(a.y)[m * a.y_stride + row] = from_f32<T>(a.bias ? v + __ldg(a.bias + row) : v);
  }
}

template <typename T, bool WIDE, int W, int R, int C, int NW>
cudaError_t launch_tile(const Int4Args& a, cudaStream_t stream) {
  const long long across = ((long long)a.rows + 8 * C - 1) / (8 * C);
  if (across > 65535) return cudaErrorInvalidValue;
  const size_t smem = (size_t)NW * 8 * C * (16 * R + 1) * sizeof(float);
  if (smem > 48 * 1024) {
    const cudaError_t e =
        cudaFuncSetAttribute(int4_kernel<T, WIDE, W, R, C, NW>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  return launch_op(int4_kernel<T, WIDE, W, R, C, NW>, dim3((a.out + 16 * R - 1) / (16 * R), (unsigned)across), 32 * NW, smem,
                   stream, a);
}

template <typename T, bool WIDE, int W>
cudaError_t launch_width(const Int4Args& a, cudaStream_t stream) {
  // Up to 32 input rows share a pass over the weights. More weight rows a CTA
  // where that still gives every SM one: the inputs are then read and arranged
  // less often (16 inputs of 8192 x 4096: 16 rows 16.5 us, 32 rows 14.5, 64 rows in
  // the registers of eight warps 12.4).
  const bool many = a.out >= 148 * 32;
  if (a.rows <= 8) return many ? launch_tile<T, WIDE, W, 2, 1, 16>(a, stream) : launch_tile<T, WIDE, W, 1, 1, 16>(a, stream);
  if (a.rows <= 16) return many ? launch_tile<T, WIDE, W, 4, 2, 8>(a, stream) : launch_tile<T, WIDE, W, 2, 2, 16>(a, stream);
  return launch_tile<T, WIDE, W, 2, 4, 16>(a, stream);
}

template <typename T, bool WIDE>
cudaError_t launch_group(const Int4Args& a, cudaStream_t stream) {
  if (a.group % 128 == 0) return launch_width<T, WIDE, 16>(a, stream);
  if (a.group % 64 == 0) return launch_width<T, WIDE, 8>(a, stream);
  return launch_width<T, WIDE, 4>(a, stream);
}

template <typename T>
cudaError_t launch_type(const Int4Args& a, bool wide, cudaStream_t stream) {
  return wide ? launch_group<T, true>(a, stream) : launch_group<T, false>(a, stream);
}

}  // namespace

cudaError_t launch_project_int4(const fav_int4_args& c, cudaStream_t stream) {
  const Int4Args a{c.x, c.y, c.x_stride, c.y_stride, c.weight, c.scales, c.bias, c.rows, c.depth, c.out, c.group,
                   (int)(((long long)c.depth + c.group - 1) / c.group)};  // the sum may pass 32 bits
  const int elem = elem_bytes(c.type);
  const bool wide = aligned_for(c.x, c.x_stride, elem, 16 / elem);
  if (c.type == FAV_TYPE_F32) return launch_type<float>(a, wide, stream);
  if (c.type == FAV_TYPE_BF16) return launch_type<__nv_bfloat16>(a, wide, stream);
  return launch_type<__half>(a, wide, stream);
}

}  // namespace fav
