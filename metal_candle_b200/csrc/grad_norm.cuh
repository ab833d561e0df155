// The norm of many gradients as partial sums of squares, and the clipping factor that comes of it (grad_norm.cu, adamw.cu).
#pragma once
#include <algorithm>
#include <vector>

#include "common.cuh"

namespace mcb {
namespace gnorm {

size_t workspace_bytes(int n_tensors);
// Leaves *parts partial sums of squares of the tensors in part (workspace_bytes of room).
int launch_squares(const mcb_grad_tensor* tensors, int n, double* part, int* parts, const DeviceState* ds, cudaStream_t st, const char* who);

// Sum over a block of 256 threads, the same bits on all of them.
__device__ __forceinline__ double block_sum(double v, double* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += s[i];
  return sum;
}
// (in float64: the norm of finite float32 gradients may lie above the largest float32, and what is clipped by it must not notice)
__device__ __forceinline__ double norm_of(const double* part, int parts, double* s) {
  part = from_here(part);
  double v = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) v += __ldcg(part + i);
  return sqrt(block_sum(v, s));
}
// min(1, max_norm / (norm + 1e-6)) * scale as the product of two float32 numbers.  The second is 1 but where the product lies below 2^-100, towards
// the numbers that float32 holds with fewer digits: there it is 2^-64, and a gradient is multiplied by both in turn.
// A norm of NaN makes the factor NaN, one of inf makes it 0; a max_norm of inf never clips.
__device__ __forceinline__ float2 clip_factor(double norm, float max_norm, float scale) {
  double f = 1.0;
  if (max_norm != INFINITY) {
    f = max_norm / (norm + 1e-6);
    f = f < 1.0 || f != f ? f : 1.0;
  }
  f *= scale;
  const bool low = fabs(f) < 0x1p-100;
  return make_float2(static_cast<float>(low ? f * 0x1p64 : f), low ? 0x1p-64f : 1.0f);
}

}  // namespace gnorm
}  // namespace mcb
