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
__device__ __forceinline__ float norm_of(const double* part, int parts, double* s) {
  part = from_here(part);
  double v = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) v += __ldcg(part + i);
  return static_cast<float>(sqrt(block_sum(v, s)));
}
// A norm of NaN makes the factor NaN, one of inf makes it 0; a max_norm of inf never clips.
__device__ __forceinline__ float clip_factor(float norm, float max_norm) {
  if (max_norm == INFINITY) return 1.0f;
  const float f = max_norm / (norm + 1e-6f);
  return f < 1.0f || f != f ? f : 1.0f;
}

}  // namespace gnorm
}  // namespace mcb
