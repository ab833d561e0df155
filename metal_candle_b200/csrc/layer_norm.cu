// Layer norm over the last dimension, forward and backward (beside RMSNorm):
//   mean = sum(x) / D;  var = sum((x - mean)^2) / D;  n = (x - mean) / sqrt(var + eps);  y = n w + b
//   g = dy w;  dx = rstd (g - sum(g) / D - n sum(g n) / D) (+ the gradient of the residual path);  dw = sum over rows of dy n;  db = of dy
// The variance is taken from the differences to the mean, which are in registers by then: E[x^2] - mean^2 would lose a row whose
// mean is large against its spread.  The backward pass takes both from x again instead of reading them: x is read anyway.
//
// HBM-bound: the forward reads x and writes y, the backward reads x and dy (and the residual) and writes dx.  A row is read once,
// into registers, by TPR threads (32 to 512, so that a thread has at most four 16-byte vectors of it); rows of more than 512
// x 4 vectors are read again from L2 instead.  Blocks walk over rows; a thread's columns stay its own, so that its parts of
// dw and db are registers until the block writes them out, a line of partial sums each that a last kernel adds up in order: no atomics.
#include "common.cuh"

namespace mcb {
namespace lnorm {
namespace {

constexpr int kMaxVec = 4;

struct Params {
  const void *x, *w, *b, *dy, *res;
  void* out;                // y or dx
  float *mean, *rstd;       // forward, or null
  float *part;              // backward: [blocks][2][D], or null
  int64_t rows;
  int D;
  float eps;
};

// Sum over the TPR threads of a row, the same bits on all of them.  `buf`: two floats a warp of the block, by turns.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* buf) {
  v = warp_sum(v);
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x >> 5;
    constexpr int W = TPR / 32;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) buf[warp] = v;
    __syncthreads();
    const int first = warp / W * W;
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) v += buf[first + i];
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float2 v, float2* buf) {
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x >> 5;
    constexpr int W = TPR / 32;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) buf[warp] = v;
    __syncthreads();
    const int first = warp / W * W;
    v = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < W; ++i) { v.x += buf[first + i].x; v.y += buf[first + i].y; }
  }
  return v;
}

// N elements at column c of a row: one 16-byte vector, or (N == 1) the element itself
template <typename T, int N>
__device__ __forceinline__ void load_n(float* f, const T* p) {
  if constexpr (N == 1) {
    f[0] = to_f32(*p);
  } else {
    Vec16<T> v;
    v.raw = *reinterpret_cast<const decltype(v.raw)*>(p);
    v.to_float(f);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T* p, const float* f) {
  if constexpr (N == 1) {
    *p = from_f32<T>(f[0]);
  } else {
    Vec16<T> v;
    v.from_float(f);
    *reinterpret_cast<decltype(v.raw)*>(p) = v.raw;
  }
}

// A thread has elements [N * (lane + TPR * k), + N) of a row for k < K.
template <typename T, int TPR, int K, int N>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) ln_fwd_kernel(const Params p) {
  constexpr int kBlock = TPR < 128 ? 128 : TPR, kRows = kBlock / TPR;
  __shared__ float buf[kBlock / 32];
  const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const T *x = static_cast<const T*>(p.x), *w = static_cast<const T*>(p.w), *b = static_cast<const T*>(p.b);
  T* y = static_cast<T*>(p.out);
  const float inv = 1.0f / static_cast<float>(p.D);
  grid_launch_dependents();
  grid_dependency_wait();
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRows; r0 < p.rows; r0 += static_cast<int64_t>(gridDim.x) * kRows) {
    const int64_t row = r0 + slot;
    const bool have = row < p.rows;
    float v[K][N];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = N * (lane + TPR * k);
#pragma unroll
      for (int e = 0; e < N; ++e) v[k][e] = 0.0f;
      if (have && c < p.D) load_n<T, N>(v[k], x + row * p.D + c);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e) sum += v[k][e];
    const float mean = row_sum<TPR>(sum, buf) * inv;
    float sq = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (N * (lane + TPR * k) < p.D) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          v[k][e] -= mean;
          sq = fmaf(v[k][e], v[k][e], sq);
        }
      }
    const float rstd = rsqrtf(row_sum<TPR>(sq, buf) * inv + p.eps);
    if (!have) continue;   // (no barrier follows within the round)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = N * (lane + TPR * k);
      if (c >= p.D) continue;
      float f[N];
#pragma unroll
      for (int e = 0; e < N; ++e) v[k][e] *= rstd;
      if (w != nullptr) {
        load_n<T, N>(f, w + c);
#pragma unroll
        for (int e = 0; e < N; ++e) v[k][e] *= f[e];
      }
      if (b != nullptr) {
        load_n<T, N>(f, b + c);
#pragma unroll
        for (int e = 0; e < N; ++e) v[k][e] += f[e];
      }
      store_n<T, N>(y + row * p.D + c, v[k]);
    }
    if (lane == 0) {
      if (p.mean != nullptr) p.mean[row] = mean;
      if (p.rstd != nullptr) p.rstd[row] = rstd;
    }
  }
}

template <typename T, int TPR, int K, int N>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) ln_bwd_kernel(const Params p) {
  constexpr int kBlock = TPR < 128 ? 128 : TPR, kRows = kBlock / TPR;
  extern __shared__ float sums[];   // [2][D] of the block's row slots, where it has several
  __shared__ float buf[kBlock / 32];
  __shared__ float2 buf2[kBlock / 32];
  const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const T *x = static_cast<const T*>(p.x), *w = static_cast<const T*>(p.w), *dy = static_cast<const T*>(p.dy), *res = static_cast<const T*>(p.res);
  T* dx = static_cast<T*>(p.out);
  const float inv = 1.0f / static_cast<float>(p.D);
  grid_launch_dependents();
  grid_dependency_wait();
  float gw[K][N], gb[K][N];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < N; ++e) gw[k][e] = gb[k][e] = 0.0f;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRows; r0 < p.rows; r0 += static_cast<int64_t>(gridDim.x) * kRows) {
    const int64_t row = r0 + slot;
    const bool have = row < p.rows;
    float v[K][N], d[K][N];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = N * (lane + TPR * k);
#pragma unroll
      for (int e = 0; e < N; ++e) v[k][e] = d[k][e] = 0.0f;
      if (have && c < p.D) {
        load_n<T, N>(v[k], x + row * p.D + c);
        load_n<T, N>(d[k], dy + row * p.D + c);
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e) sum += v[k][e];
    const float mean = row_sum<TPR>(sum, buf) * inv;
    float sq = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (N * (lane + TPR * k) < p.D) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          v[k][e] -= mean;
          sq = fmaf(v[k][e], v[k][e], sq);
        }
      }
    const float rstd = rsqrtf(row_sum<TPR>(sq, buf) * inv + p.eps);
    float2 s2 = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = N * (lane + TPR * k);
      float f[N];
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = 1.0f;
      if (w != nullptr && c < p.D) load_n<T, N>(f, w + c);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        v[k][e] *= rstd;
        gw[k][e] = fmaf(d[k][e], v[k][e], gw[k][e]);
        gb[k][e] += d[k][e];
        d[k][e] *= f[e];
        s2.x += d[k][e];
        s2.y = fmaf(d[k][e], v[k][e], s2.y);
      }
    }
    s2 = row_sum2<TPR>(s2, buf2);
    const float a = s2.x * inv, q = s2.y * inv;
    if (!have) continue;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = N * (lane + TPR * k);
      if (c >= p.D) continue;
      float f[N];
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = 0.0f;
      if (res != nullptr) load_n<T, N>(f, res + row * p.D + c);
#pragma unroll
      for (int e = 0; e < N; ++e) d[k][e] = fmaf(fmaf(-v[k][e], q, d[k][e] - a), rstd, f[e]);
      store_n<T, N>(dx + row * p.D + c, d[k]);
    }
  }
  if (p.part == nullptr) return;
  float* out = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.D;
  if constexpr (kRows > 1) {
    for (int s = 0; s < kRows; ++s) {
      __syncthreads();
      if (slot != s) continue;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int c = N * (lane + TPR * k) + e;
          if (c < p.D) {
            sums[c] = (s ? sums[c] : 0.0f) + gw[k][e];
            sums[p.D + c] = (s ? sums[p.D + c] : 0.0f) + gb[k][e];
          }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.D; i += kBlock) out[i] = sums[i];
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int c = N * (lane + TPR * k) + e;
        if (c < p.D) { out[c] = gw[k][e]; out[p.D + c] = gb[k][e]; }
      }
  }
}

// Rows of any length, element by element, read again for each sum; the columns' sums of a block's rows likewise.
template <typename T, bool BWD>
__global__ void __launch_bounds__(512) ln_long_kernel(const Params p) {
  __shared__ float buf[16];
  __shared__ float2 buf2[16];
  const T *x = static_cast<const T*>(p.x), *w = static_cast<const T*>(p.w), *b = static_cast<const T*>(p.b), *dy = static_cast<const T*>(p.dy),
          *res = static_cast<const T*>(p.res);
  T* out = static_cast<T*>(p.out);
  const float inv = 1.0f / static_cast<float>(p.D);
  grid_launch_dependents();
  grid_dependency_wait();
  float* part = p.part == nullptr ? nullptr : p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.D;
  if (BWD && part != nullptr)
    for (int c = threadIdx.x; c < p.D; c += 512) part[c] = part[p.D + c] = 0.0f;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const int64_t at = row * p.D;
    float sum = 0.0f, sq = 0.0f;
    for (int c = threadIdx.x; c < p.D; c += 512) sum += to_f32(x[at + c]);
    const float mean = row_sum<512>(sum, buf) * inv;
    for (int c = threadIdx.x; c < p.D; c += 512) {
      const float v = to_f32(x[at + c]) - mean;
      sq = fmaf(v, v, sq);
    }
    const float rstd = rsqrtf(row_sum<512>(sq, buf) * inv + p.eps);
    if constexpr (!BWD) {
      for (int c = threadIdx.x; c < p.D; c += 512) {
        float v = (to_f32(x[at + c]) - mean) * rstd;
        if (w != nullptr) v *= to_f32(w[c]);
        if (b != nullptr) v += to_f32(b[c]);
        out[at + c] = from_f32<T>(v);
      }
      if (threadIdx.x == 0) {
        if (p.mean != nullptr) p.mean[row] = mean;
        if (p.rstd != nullptr) p.rstd[row] = rstd;
      }
    } else {
      float2 s2 = make_float2(0.0f, 0.0f);
      for (int c = threadIdx.x; c < p.D; c += 512) {
        const float n = (to_f32(x[at + c]) - mean) * rstd, d = to_f32(dy[at + c]), g = w != nullptr ? d * to_f32(w[c]) : d;
        s2.x += g;
        s2.y = fmaf(g, n, s2.y);
        if (part != nullptr) {   // (this thread's own columns)
          part[c] = fmaf(d, n, part[c]);
          part[p.D + c] += d;
        }
      }
      s2 = row_sum2<512>(s2, buf2);
      for (int c = threadIdx.x; c < p.D; c += 512) {
        const float n = (to_f32(x[at + c]) - mean) * rstd, d = to_f32(dy[at + c]), g = w != nullptr ? d * to_f32(w[c]) : d;
        const float r = res != nullptr ? to_f32(res[at + c]) : 0.0f;
        out[at + c] = from_f32<T>(fmaf(fmaf(-n, s2.y * inv, g - s2.x * inv), rstd, r));
      }
    }
  }
}

// dw and db from the blocks' sums, in block order: 32 columns a block of 32 x 8, eight strands of blocks to a column.
__global__ void __launch_bounds__(256) ln_reduce_kernel(const float* part, int blocks, int D, float* dw, float* db, int accumulate) {
  __shared__ float s[8][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), strand = threadIdx.x >> 5;
  grid_launch_dependents();
  grid_dependency_wait();
  part = from_here(part);
  float v = 0.0f;
  if (c < 2 * D)
    for (int i = strand; i < blocks; i += 8) v += part[static_cast<int64_t>(i) * 2 * D + c];
  s[strand][threadIdx.x & 31] = v;
  __syncthreads();
  if (strand != 0 || c >= 2 * D) return;
  for (int i = 1; i < 8; ++i) v += s[i][threadIdx.x];
  float* out = c < D ? dw : db;
  if (out == nullptr) return;
  const int k = c < D ? c : c - D;
  out[k] = accumulate ? out[k] + v : v;
}

constexpr int kMaxBlocks = 1184;   // 8 x 148

int blocks_for(int64_t rows, int per_block, int sms, int per_sm) {
  const int64_t want = (rows + per_block - 1) / per_block;
  int64_t most = static_cast<int64_t>(sms) * per_sm;
  if (most > kMaxBlocks) most = kMaxBlocks;
  return static_cast<int>(want < most ? want : most);
}

// A row's threads and vectors: as few threads as have at most kMaxVec vectors each.
template <typename T, int N, bool BWD, int TPR, int K>
int launch_k(const Params& p, int sms, cudaStream_t st, int* blocks) {
  constexpr int kBlock = TPR < 128 ? 128 : TPR, kRows = kBlock / TPR;
  *blocks = blocks_for(p.rows, kRows, sms, 2048 / kBlock < 8 ? 2048 / kBlock : 8);
  if constexpr (BWD) {
    const size_t smem = p.part != nullptr && kRows > 1 ? 2 * static_cast<size_t>(p.D) * 4 : 0;
    MCB_CHECK_CUDA(launch_kernel(ln_bwd_kernel<T, TPR, K, N>, dim3(*blocks), dim3(kBlock), smem, st, chained_launch(), p));
  } else {
    MCB_CHECK_CUDA(launch_kernel(ln_fwd_kernel<T, TPR, K, N>, dim3(*blocks), dim3(kBlock), 0, st, chained_launch(), p));
  }
  MCB_CHECK_LAUNCH("layer_norm");
  return MCB_OK;
}
template <typename T, int N, bool BWD, int TPR>
int launch_tpr(const Params& p, int vecs, int sms, cudaStream_t st, int* blocks) {
  const int k = (vecs + TPR - 1) / TPR;
  if (k <= 1) return launch_k<T, N, BWD, TPR, 1>(p, sms, st, blocks);
  if (k == 2) return launch_k<T, N, BWD, TPR, 2>(p, sms, st, blocks);
  if (k == 3) return launch_k<T, N, BWD, TPR, 3>(p, sms, st, blocks);
  return launch_k<T, N, BWD, TPR, 4>(p, sms, st, blocks);
}
template <typename T, bool BWD>
int launch(const Params& p, bool vec, int sms, cudaStream_t st, int* blocks) {
  constexpr int N = Vec16<T>::N;
  if (vec && p.D <= 512 * kMaxVec * N) {
    const int vecs = p.D / N;
    if (vecs <= 32 * kMaxVec) return launch_tpr<T, N, BWD, 32>(p, vecs, sms, st, blocks);
    if (vecs <= 128 * kMaxVec) return launch_tpr<T, N, BWD, 128>(p, vecs, sms, st, blocks);
    return launch_tpr<T, N, BWD, 512>(p, vecs, sms, st, blocks);
  }
  if (!vec && p.D <= 512 * kMaxVec) {
    if (p.D <= 32 * kMaxVec) return launch_tpr<T, 1, BWD, 32>(p, p.D, sms, st, blocks);
    if (p.D <= 128 * kMaxVec) return launch_tpr<T, 1, BWD, 128>(p, p.D, sms, st, blocks);
    return launch_tpr<T, 1, BWD, 512>(p, p.D, sms, st, blocks);
  }
  *blocks = blocks_for(p.rows, 1, sms, 4);
  MCB_CHECK_CUDA(launch_kernel(ln_long_kernel<T, BWD>, dim3(*blocks), dim3(512), 0, st, chained_launch(), p));
  MCB_CHECK_LAUNCH("layer_norm");
  return MCB_OK;
}

int check(const char* who, int64_t rows, int64_t D, float eps, int dtype) {
  if (dtype != MCB_F32 && dtype != MCB_BF16) return fail(MCB_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (rows <= 0 || D <= 0 || D > 0x3fffffff) return fail(MCB_ERR_SHAPE, "%s: rows=%lld D=%lld", who, (long long)rows, (long long)D);
  if (!(eps >= 0.0f && eps - eps == 0.0f)) return fail(MCB_ERR_SHAPE, "%s: eps must be finite and not negative", who);
  return MCB_OK;
}

}  // namespace
}  // namespace lnorm
}  // namespace mcb

using namespace mcb;

extern "C" int mcb_layernorm_fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows, int64_t D,
                                 float eps, int dtype, void* stream) {
  MCB_NVTX_RANGE("mcb_layernorm_fwd");
  if (!x || !y) return fail(MCB_ERR_NULL, "layernorm_fwd: x or y is null");
  if (int rc = lnorm::check("layernorm_fwd", rows, D, eps, dtype)) return rc;
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  lnorm::Params p = {};
  p.x = x; p.w = w; p.b = b; p.out = y; p.mean = mean; p.rstd = rstd;
  p.rows = rows; p.D = static_cast<int>(D); p.eps = eps;
  const int size = dtype == MCB_F32 ? 4 : 2;
  const bool vec = D * size % 16 == 0 && aligned16(x) && aligned16(y) && aligned16(w) && aligned16(b);
  int blocks = 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == MCB_F32 ? lnorm::launch<float, false>(p, vec, ds->sm_count, st, &blocks)
                          : lnorm::launch<__nv_bfloat16, false>(p, vec, ds->sm_count, st, &blocks);
}

extern "C" size_t mcb_layernorm_bwd_workspace_bytes(int64_t rows, int64_t D) {
  if (rows <= 0 || D <= 0) return 0;
  const int64_t blocks = rows < lnorm::kMaxBlocks ? rows : lnorm::kMaxBlocks;
  return static_cast<size_t>(blocks) * 2 * D * 4;
}

extern "C" int mcb_layernorm_bwd(const void* x, const void* w, const void* dy, const void* dx_residual, void* dx, float* dw, float* db,
                                 int accumulate, int64_t rows, int64_t D, float eps, int dtype, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  MCB_NVTX_RANGE("mcb_layernorm_bwd");
  if (!x || !dy || !dx) return fail(MCB_ERR_NULL, "layernorm_bwd: x, dy or dx is null");
  if (int rc = lnorm::check("layernorm_bwd", rows, D, eps, dtype)) return rc;
  const bool sums = dw != nullptr || db != nullptr;
  if (sums && (!workspace || workspace_bytes < mcb_layernorm_bwd_workspace_bytes(rows, D) || !aligned16(workspace)))
    return fail(MCB_ERR_WORKSPACE, "layernorm_bwd: workspace of %zu bytes, 16-byte aligned, needed", mcb_layernorm_bwd_workspace_bytes(rows, D));
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  lnorm::Params p = {};
  p.x = x; p.w = w; p.dy = dy; p.res = dx_residual; p.out = dx; p.part = sums ? static_cast<float*>(workspace) : nullptr;
  p.rows = rows; p.D = static_cast<int>(D); p.eps = eps;
  const int size = dtype == MCB_F32 ? 4 : 2;
  const bool vec = D * size % 16 == 0 && aligned16(x) && aligned16(dx) && aligned16(w) && aligned16(dy) && aligned16(dx_residual);
  int blocks = 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = dtype == MCB_F32 ? lnorm::launch<float, true>(p, vec, ds->sm_count, st, &blocks)
                                : lnorm::launch<__nv_bfloat16, true>(p, vec, ds->sm_count, st, &blocks)) return rc;
  if (!sums) return MCB_OK;
  MCB_CHECK_CUDA(launch_kernel(lnorm::ln_reduce_kernel, dim3(static_cast<unsigned>((2 * D + 31) / 32)), dim3(256), 0, st, chained_launch(),
                               static_cast<const float*>(p.part), blocks, p.D, dw, db, accumulate));
  MCB_CHECK_LAUNCH("layer_norm_reduce");
  return MCB_OK;
}
