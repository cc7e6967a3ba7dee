// Group norm with an activation over channels-last rows: per sequence and
// group, y = act((x - mean) * rstd * weight + bias), mean and variance over
// the sequence's rows and the group's channels, in fp32.
#include "fav_ops.cuh"

namespace fav {
namespace {

struct NormArgs {
  const void* x;
  void* y;
  long long x_stride, y_stride;
  const float *weight, *bias, *alpha, *recip;
  Sequences seq;
  float eps;
  int channels, groups, activation;
};

__device__ __forceinline__ float activate(const NormArgs& a, float v, int c) {
  if (a.activation == FAV_ACTIVATION_SILU) return silu(v);
  if (a.activation == FAV_ACTIVATION_SNAKE) {
    const float s = sinf(__ldg(a.alpha + c) * v);
    return fmaf(__ldg(a.recip + c), s * s, v);
  }
  return v;
}

constexpr int kNormThreads = 256;

__device__ __forceinline__ float block_sum(float v, float* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < kNormThreads / 32; ++i) v += part[i];
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float part[kNormThreads / 32];
  grid_dependency_sync();
  const int s = blockIdx.x / a.groups, g = blockIdx.x - s * a.groups;
  const Span sp = span_of(a.seq, s);
  if (sp.begin > sp.end) {
    if (threadIdx.x == 0) record_error(a.seq.status, kDevBadOffsets);
    return;
  }
  const int width = a.channels / a.groups;
  const long long count = (long long)(sp.end - sp.begin) * width;
  if (count == 0) return;
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  float sum = 0.f;
  for (long long e = threadIdx.x; e < count; e += kNormThreads)
    sum += to_f32(x[(sp.begin + e / width) * a.x_stride + g * width + e % width]);
  const float mean = block_sum(sum, part) / (float)count;
  sum = 0.f;
  for (long long e = threadIdx.x; e < count; e += kNormThreads) {
    const float d = to_f32(x[(sp.begin + e / width) * a.x_stride + g * width + e % width]) - mean;
    sum = fmaf(d, d, sum);
  }
  const float rstd = rsqrtf(block_sum(sum, part) / (float)count + a.eps);
  for (long long e = threadIdx.x; e < count; e += kNormThreads) {
    const int c = g * width + (int)(e % width);
    const long long r = sp.begin + e / width;
    float v = (to_f32(x[r * a.x_stride + c]) - mean) * rstd;
    if (a.weight) v *= __ldg(a.weight + c);
    if (a.bias) v += __ldg(a.bias + c);
    y[r * a.y_stride + c] = from_f32<T>(activate(a, v, c));
  }
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
  a.activation = c.activation;
  const long long blocks = (long long)seq.n * c.groups;
  if (blocks == 0) return cudaSuccess;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (c.type == FAV_TYPE_F32) return launch_op(norm_kernel<float>, (unsigned)blocks, kNormThreads, 0, stream, a);
  if (c.type == FAV_TYPE_BF16)
    return launch_op(norm_kernel<__nv_bfloat16>, (unsigned)blocks, kNormThreads, 0, stream, a);
  return launch_op(norm_kernel<__half>, (unsigned)blocks, kNormThreads, 0, stream, a);
}

}  // namespace fav
