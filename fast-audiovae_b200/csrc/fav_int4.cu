// Projection of a few rows by 4-bit weights with group scales:
//
//   y[m, r] = bias[r] + sum_g scales[r, g] * sum_{k in g} x[m, k] * (q[r, k] - 8)
//
// Sums in fp32.
#include "fav_ops.cuh"

namespace fav {
namespace {

struct Int4Args {
  const void* x;
  void* y;
  long long x_stride, y_stride;
  const uint8_t* weight;
  const float *scales, *bias;
  int rows, depth, out, group;
};

constexpr int kInt4Threads = 128;

template <typename T>
__global__ void __launch_bounds__(kInt4Threads) int4_kernel(const __grid_constant__ Int4Args a) {
  grid_dependency_sync();
  const long long warp = ((long long)blockIdx.x * kInt4Threads + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const int m = (int)(warp / a.out), r = (int)(warp - (long long)m * a.out);
  if (m >= a.rows) return;
  const int groups = (a.depth + a.group - 1) / a.group;
  const T* x = static_cast<const T*>(a.x) + m * a.x_stride;
  const uint8_t* w = a.weight + (size_t)r * (a.depth / 2);
  float sum = 0.f;
  for (int k = 2 * lane; k < a.depth; k += 64) {
    const int byte = w[k / 2];
    const float s = a.scales[(size_t)r * groups + k / a.group];
    sum = fmaf(s, to_f32(x[k]) * (float)((byte & 15) - 8) + to_f32(x[k + 1]) * (float)((byte >> 4) - 8), sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0)
    static_cast<T*>(a.y)[m * a.y_stride + r] = from_f32<T>(a.bias ? sum + __ldg(a.bias + r) : sum);
}

}  // namespace

cudaError_t launch_project_int4(const fav_int4_args& c, cudaStream_t stream) {
  Int4Args a{c.x, c.y, c.x_stride, c.y_stride, c.weight, c.scales, c.bias, c.rows, c.depth, c.out, c.group};
  const long long blocks = ((long long)c.rows * c.out + kInt4Threads / 32 - 1) / (kInt4Threads / 32);
  if (blocks == 0) return cudaSuccess;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (c.type == FAV_TYPE_F32) return launch_op(int4_kernel<float>, (unsigned)blocks, kInt4Threads, 0, stream, a);
  if (c.type == FAV_TYPE_BF16)
    return launch_op(int4_kernel<__nv_bfloat16>, (unsigned)blocks, kInt4Threads, 0, stream, a);
  return launch_op(int4_kernel<__half>, (unsigned)blocks, kInt4Threads, 0, stream, a);
}

}  // namespace fav
