// Layer norm over the last dimension, forward and backward (beside RMSNorm):
//   mean = sum(x) / D;  var = sum((x - mean)^2) / D;  n = (x - mean) / sqrt(var + eps);  y = n w + b
//   g = dy w;  dx = rstd (g - sum(g) / D - n sum(g n) / D) (+ the gradient of the residual path);  dw = sum over rows of dy n;  db = of dy
// The variance is taken from the differences to the mean, which are in registers by then: E[x^2] - mean^2 would lose a row whose
// mean is large against its spread.  The backward pass takes both from x again instead of reading them: x is read anyway.
//
// HBM-bound: the forward reads x and writes y, the backward reads x and dy (and the residual) and writes dx.  A row is read once,
// into registers, by TPR threads (32 to 512, so that a thread has at most four 16-byte vectors of it, or eight elements of a row that
// is not made of whole, aligned vectors); longer rows are read again from L2 instead.  Blocks walk over rows; a thread's columns stay its own, so that its parts of
// dw and db are registers until the block writes them out, a line of partial sums each that a last kernel adds up in order: no atomics.
#include <type_traits>

#include "common.cuh"

namespace mcb {
namespace lnorm {
namespace {

struct Params {
  const void *x, *w, *b, *dy, *res;
  void* out;                // y or dx
  float *mean, *rstd;       // forward, or null
  float *part;              // backward: [blocks][2][D], or null
  int64_t rows;
  int D;
  float eps;
};

// Sums over the TPR threads of a row, the same bits on all of them.  `buf` has a place for each warp of the block; a call with another
// buffer lies between two with the same one, whose barrier keeps them apart.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* buf) {
  v = warp_sum(v);
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x >> 5;
    constexpr int W = TPR / 32;
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
__device__ __forceinline__ float3 row_sum3(float3 v, float3* buf) {
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  v.z = warp_sum(v.z);
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x >> 5;
    constexpr int W = TPR / 32;
    if ((threadIdx.x & 31) == 0) buf[warp] = v;
    __syncthreads();
    const int first = warp / W * W;
    v = make_float3(0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < W; ++i) { v.x += buf[first + i].x; v.y += buf[first + i].y; v.z += buf[first + i].z; }
  }
  return v;
}

// N elements of a row as they lie in memory: one 16-byte vector, or (N == 1) the element itself
template <typename T, int N>
struct Piece {
  using Raw = std::conditional_t<N == 1, T, decltype(Vec16<T>::raw)>;
  Raw raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
  __device__ __forceinline__ void zero() { raw = Raw(); }
  __device__ __forceinline__ void to_float(float (&f)[N]) const {
    if constexpr (N == 1) f[0] = to_f32(raw);
    else { Vec16<T> v; v.raw = raw; v.to_float(f); }
  }
  __device__ __forceinline__ void from_float(const float (&f)[N]) {
    if constexpr (N == 1) raw = from_f32<T>(f[0]);
    else { Vec16<T> v; v.from_float(f); raw = v.raw; }
  }
};

// ---- rows on their way -------------------------------------------------------------------------------------------------
// A block has `STAGES - 1` rounds of rows on their way from memory while it works on one (cp.async): the bytes in flight are what the
// bandwidth is made of, and shared memory has room for them where registers have not.  A thread has the elements [N * (lane + TPR * k), + N) of a row.
// N > 1 (rows of whole, aligned 16-byte vectors): every thread fetches its own vectors and waits for nobody.  N == 1: rows that start
// anywhere are fetched as the 16-byte granules that cover them, and the row's threads meet once a round.
__device__ __forceinline__ void cp_async16(void* dst, const void* src, int bytes) {
  const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

constexpr int block_of(int tpr) { return tpr < 128 ? 128 : tpr; }
constexpr int stages_of(int tpr, int k) { return k * block_of(tpr) > 1024 ? 2 : 3; }   // (three would not fit for three operands)

template <typename T, int TPR, int K, int N>
struct Feed {
  static constexpr int kBlock = block_of(TPR), kRows = kBlock / TPR, STAGES = stages_of(TPR, K);
  uint8_t* ring;
  int lane, slot, D, nt, row_bytes;
  int64_t rows;
  __host__ __device__ static int bytes_of_row(int D) { return ((D * static_cast<int>(sizeof(T)) + 15) & ~15) + 16; }
  __host__ static size_t smem(int D, int nt) {
    return static_cast<size_t>(STAGES) * nt * (N > 1 ? K * kBlock * 16 : kRows * bytes_of_row(D));
  }
  __device__ __forceinline__ Feed(void* smem_base, int lane_, int slot_, const Params& p, int nt_)
      : ring(static_cast<uint8_t*>(smem_base)), lane(lane_), slot(slot_), D(p.D), nt(nt_), row_bytes(bytes_of_row(p.D)), rows(p.rows) {}
  __device__ __forceinline__ uint8_t* at(int stage, int t) const {
    if constexpr (N > 1) return ring + (static_cast<size_t>(stage * nt + t) * K * kBlock + threadIdx.x) * 16;
    else return ring + (static_cast<size_t>(stage * nt + t) * kRows + slot) * row_bytes;
  }
  __device__ __forceinline__ void fetch(int stage, int t, const T* x, int64_t row) const {
    if (row >= rows) return;
    if constexpr (N > 1) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = N * (lane + TPR * k);
        if (c < D) cp_async16(at(stage, t) + k * kBlock * 16, x + row * D + c, 16);
      }
    } else {
      const uintptr_t from = reinterpret_cast<uintptr_t>(x + row * D), first = from & ~static_cast<uintptr_t>(15);
      const uintptr_t end = reinterpret_cast<uintptr_t>(x + rows * D), row_end = from + static_cast<uintptr_t>(D) * sizeof(T);
      for (uintptr_t g = first + 16 * lane; g < row_end; g += 16 * TPR)   // nothing behind the tensor is read
        cp_async16(at(stage, t) + (g - first), reinterpret_cast<const void*>(g), end - g < 16 ? static_cast<int>(end - g) : 16);
    }
  }
  __device__ __forceinline__ void get(int stage, int t, const T* x, int64_t row, float (&v)[K][N]) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = N * (lane + TPR * k);
#pragma unroll
      for (int e = 0; e < N; ++e) v[k][e] = 0.0f;
      if (row < rows && c < D) {
        Piece<T, N> piece;
        if constexpr (N > 1) piece.load(reinterpret_cast<const T*>(at(stage, t) + k * kBlock * 16));
        else piece.load(reinterpret_cast<const T*>(at(stage, t) + (reinterpret_cast<uintptr_t>(x + row * D) & 15)) + c);
        piece.to_float(v[k]);
      }
    }
  }
  // The round's rows are here (and, N == 1, nobody reads the stage that is filled next).
  __device__ __forceinline__ void arrived() const {
    cp_async_wait<STAGES - 2>();
    if constexpr (N == 1) {
      if constexpr (TPR > 32) __syncthreads();
      else __syncwarp();
    }
  }
};

template <typename T, int TPR, int K, int N>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) ln_fwd_kernel(const Params p) {
  extern __shared__ uint4 smem4[];
  using F = Feed<T, TPR, K, N>;
  __shared__ float buf[2][F::kBlock / 32];
  const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const T *x = static_cast<const T*>(p.x), *w = static_cast<const T*>(p.w), *b = static_cast<const T*>(p.b);
  T* y = static_cast<T*>(p.out);
  const float inv = 1.0f / static_cast<float>(p.D);
  const int64_t step = static_cast<int64_t>(gridDim.x) * F::kRows;
  int64_t r0 = static_cast<int64_t>(blockIdx.x) * F::kRows;
  const F feed(smem4, lane, slot, p, 1);
  grid_launch_dependents();
  grid_dependency_wait();
#pragma unroll
  for (int i = 0; i < F::STAGES - 1; ++i) {
    feed.fetch(i, 0, x, r0 + slot + i * step);
    cp_async_commit();
  }
  for (int stage = 0; r0 < p.rows; r0 += step) {
    const int64_t row = r0 + slot;
    float v[K][N];
    float sum = 0.0f;
    feed.arrived();
    feed.fetch(stage == 0 ? F::STAGES - 1 : stage - 1, 0, x, row + (F::STAGES - 1) * step);
    cp_async_commit();
    feed.get(stage, 0, x, row, v);
    if (++stage == F::STAGES) stage = 0;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e) sum += v[k][e];
    const float mean = row_sum<TPR>(sum, buf[0]) * inv;
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
    const float rstd = rsqrtf(row_sum<TPR>(sq, buf[1]) * inv + p.eps);
    if (row >= p.rows) continue;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = N * (lane + TPR * k);
      if (c >= p.D) continue;
      Piece<T, N> t;
      float f[N];
#pragma unroll
      for (int e = 0; e < N; ++e) v[k][e] *= rstd;
      if (w != nullptr) {
        t.load(w + c);
        t.to_float(f);
#pragma unroll
        for (int e = 0; e < N; ++e) v[k][e] *= f[e];
      }
      if (b != nullptr) {
        t.load(b + c);
        t.to_float(f);
#pragma unroll
        for (int e = 0; e < N; ++e) v[k][e] += f[e];
      }
      t.from_float(v[k]);
      t.store(y + row * p.D + c);
    }
    if (lane == 0) {
      if (p.mean != nullptr) p.mean[row] = mean;
      if (p.rstd != nullptr) p.rstd[row] = rstd;
    }
  }
}

// After the mean one more round of sums does: of (x - mean)^2, of g and of g (x - mean), from which rstd and both means of the backward
// formula follow.  SUMS: dw and db are asked for.
template <typename T, int TPR, int K, int N, bool SUMS>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) ln_bwd_kernel(const Params p) {
  extern __shared__ uint4 smem4[];
  using F = Feed<T, TPR, K, N>;
  __shared__ float buf[F::kBlock / 32];
  __shared__ float3 buf3[F::kBlock / 32];
  const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const T *x = static_cast<const T*>(p.x), *w = static_cast<const T*>(p.w), *dy = static_cast<const T*>(p.dy), *res = static_cast<const T*>(p.res);
  T* dx = static_cast<T*>(p.out);
  const float inv = 1.0f / static_cast<float>(p.D);
  const int64_t step = static_cast<int64_t>(gridDim.x) * F::kRows;
  int64_t r0 = static_cast<int64_t>(blockIdx.x) * F::kRows;
  const F feed(smem4, lane, slot, p, res != nullptr ? 3 : 2);
  auto fetch = [&](int stage, int64_t row) {
    feed.fetch(stage, 0, x, row);
    feed.fetch(stage, 1, dy, row);
    if (res != nullptr) feed.fetch(stage, 2, res, row);
    cp_async_commit();
  };
  grid_launch_dependents();
  grid_dependency_wait();
  float gw[SUMS ? K : 1][N], gb[SUMS ? K : 1][N];
#pragma unroll
  for (int k = 0; k < (SUMS ? K : 1); ++k)
#pragma unroll
    for (int e = 0; e < N; ++e) gw[k][e] = gb[k][e] = 0.0f;
#pragma unroll
  for (int i = 0; i < F::STAGES - 1; ++i) fetch(i, r0 + slot + i * step);
  int stage = 0;
  for (; r0 < p.rows; r0 += step) {
    const int64_t row = r0 + slot;
    float v[K][N], d[K][N];
    float sum = 0.0f;
    feed.arrived();
    const int here = stage;
    fetch(stage == 0 ? F::STAGES - 1 : stage - 1, row + (F::STAGES - 1) * step);
    if (++stage == F::STAGES) stage = 0;
    feed.get(here, 0, x, row, v);
    feed.get(here, 1, dy, row, d);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e) sum += v[k][e];
    const float mean = row_sum<TPR>(sum, buf) * inv;
    float3 s = make_float3(0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = N * (lane + TPR * k);
      if (c >= p.D) continue;
      float f[N];
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = 1.0f;
      if (w != nullptr) {
        Piece<T, N> t;
        t.load(w + c);
        t.to_float(f);
      }
#pragma unroll
      for (int e = 0; e < N; ++e) {
        v[k][e] -= mean;
        const float g = d[k][e] * f[e];
        s.x = fmaf(v[k][e], v[k][e], s.x);
        s.y += g;
        s.z = fmaf(g, v[k][e], s.z);
      }
    }
    s = row_sum3<TPR>(s, buf3);
    const float rstd = rsqrtf(s.x * inv + p.eps);
    const float a = s.y * inv, q = s.z * inv * rstd;
    if (row >= p.rows) continue;
    float r[K][N];
    if (res != nullptr) feed.get(here, 2, res, row, r);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = N * (lane + TPR * k);
      if (c >= p.D) continue;
      Piece<T, N> t;
      float f[N];
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = 1.0f;
      if (w != nullptr) {   // (from L1: registers for it would cost occupancy)
        t.load(w + c);
        t.to_float(f);
      }
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float n = v[k][e] * rstd;
        if constexpr (SUMS) {
          gw[k][e] = fmaf(d[k][e], n, gw[k][e]);
          gb[k][e] += d[k][e];
        }
        f[e] = fmaf(fmaf(-n, q, fmaf(d[k][e], f[e], -a)), rstd, res != nullptr ? r[k][e] : 0.0f);
      }
      t.from_float(f);
      t.store(dx + row * p.D + c);
    }
  }
  if constexpr (SUMS) {
    float* out = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.D;
    if constexpr (F::kRows > 1) {
      cp_async_wait<0>();
      float* sums = reinterpret_cast<float*>(smem4);   // [2][D] of the block's row slots, over the ring
      for (int s = 0; s < F::kRows; ++s) {
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
      for (int i = threadIdx.x; i < 2 * p.D; i += F::kBlock) out[i] = sums[i];
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
}

// Rows of any length, element by element, read again for each sum; the columns' sums of a block's rows likewise.
template <typename T, bool BWD>
__global__ void __launch_bounds__(512) ln_long_kernel(const Params p) {
  __shared__ float buf[2][16];
  __shared__ float3 buf3[16];
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
    const float mean = row_sum<512>(sum, buf[0]) * inv;
    for (int c = threadIdx.x; c < p.D; c += 512) {
      const float v = to_f32(x[at + c]) - mean;
      sq = fmaf(v, v, sq);
    }
    const float rstd = rsqrtf(row_sum<512>(sq, buf[1]) * inv + p.eps);
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
      float3 s2 = make_float3(0.0f, 0.0f, 0.0f);
      for (int c = threadIdx.x; c < p.D; c += 512) {
        const float n = (to_f32(x[at + c]) - mean) * rstd, d = to_f32(dy[at + c]), g = w != nullptr ? d * to_f32(w[c]) : d;
        s2.x += g;
        s2.y = fmaf(g, n, s2.y);
        if (part != nullptr) {   // (this thread's own columns)
          part[c] = fmaf(d, n, part[c]);
          part[p.D + c] += d;
        }
      }
      s2 = row_sum3<512>(s2, buf3);
      for (int c = threadIdx.x; c < p.D; c += 512) {
        const float n = (to_f32(x[at + c]) - mean) * rstd, d = to_f32(dy[at + c]), g = w != nullptr ? d * to_f32(w[c]) : d;
        const float r = res != nullptr ? to_f32(res[at + c]) : 0.0f;
        out[at + c] = from_f32<T>(fmaf(fmaf(-n, s2.y * inv, g - s2.x * inv), rstd, r));
      }
    }
  }
}

// dw and db from the blocks' sums: 32 columns a block of 32 x 32, thirty-two strands of blocks to a column that are added up in order.
__global__ void __launch_bounds__(1024) ln_reduce_kernel(const float* part, int blocks, int D, float* dw, float* db, int accumulate) {
  __shared__ float s[32][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), strand = threadIdx.x >> 5;
  grid_launch_dependents();
  grid_dependency_wait();
  part = from_here(part);
  float v = 0.0f;
  if (c < 2 * D)
#pragma unroll 4
    for (int i = strand; i < blocks; i += 32) v += part[static_cast<int64_t>(i) * 2 * D + c];
  s[strand][threadIdx.x & 31] = v;
  __syncthreads();
  if (strand != 0 || c >= 2 * D) return;
#pragma unroll
  for (int i = 1; i < 32; ++i) v += s[i][threadIdx.x];
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

// As many blocks as are on the device at once: the rows' sums are kept by block.
template <typename K>
int resident(K kernel, int threads, size_t smem, int64_t want, int sms, int* blocks) {
  int per_sm = 0;
  MCB_CHECK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem));
  *blocks = blocks_for(want, 1, sms, per_sm < 1 ? 1 : per_sm);
  return MCB_OK;
}
template <typename T, int N, bool BWD, int TPR, int K>
int launch_k(const Params& p, int sms, cudaStream_t st, int* blocks) {
  using F = Feed<T, TPR, K, N>;
  size_t smem = F::smem(p.D, !BWD ? 1 : p.res != nullptr ? 3 : 2);
  if (BWD && F::kRows > 1 && smem < 2 * static_cast<size_t>(p.D) * 4) smem = 2 * static_cast<size_t>(p.D) * 4;
  void (*kernel)(const Params) = ln_fwd_kernel<T, TPR, K, N>;
  if constexpr (BWD) kernel = p.part != nullptr ? ln_bwd_kernel<T, TPR, K, N, true> : ln_bwd_kernel<T, TPR, K, N, false>;
  MCB_CHECK_CUDA(cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  if (int rc = resident(kernel, F::kBlock, smem, (p.rows + F::kRows - 1) / F::kRows, sms, blocks)) return rc;
  MCB_CHECK_CUDA(launch_kernel(kernel, dim3(*blocks), dim3(F::kBlock), smem, st, chained_launch(), p));
  MCB_CHECK_LAUNCH("layer_norm");
  return MCB_OK;
}
template <typename T, int N, bool BWD, int TPR>
int launch_tpr(const Params& p, int pieces, int sms, cudaStream_t st, int* blocks) {
  const int k = (pieces + TPR - 1) / TPR;
  if (k <= 1) return launch_k<T, N, BWD, TPR, 1>(p, sms, st, blocks);
  if (k == 2) return launch_k<T, N, BWD, TPR, 2>(p, sms, st, blocks);
  if constexpr (N > 1) {
    if (k == 3) return launch_k<T, N, BWD, TPR, 3>(p, sms, st, blocks);
    return launch_k<T, N, BWD, TPR, 4>(p, sms, st, blocks);
  } else {
    if (k <= 4) return launch_k<T, N, BWD, TPR, 4>(p, sms, st, blocks);
    return launch_k<T, N, BWD, TPR, 8>(p, sms, st, blocks);
  }
}
// A row's threads: as few as have at most four 16-byte pieces (or eight elements) of it each.
template <typename T, bool BWD, int N>
int launch_n(const Params& p, int sms, cudaStream_t st, int* blocks) {
  const int pieces = p.D / N;
  constexpr int most = N > 1 ? 4 : 8;
  if (pieces <= 32 * most) return launch_tpr<T, N, BWD, 32>(p, pieces, sms, st, blocks);
  if (pieces <= 128 * most) return launch_tpr<T, N, BWD, 128>(p, pieces, sms, st, blocks);
  if (pieces <= 512 * most) return launch_tpr<T, N, BWD, 512>(p, pieces, sms, st, blocks);
  *blocks = blocks_for(p.rows, 1, sms, 4);
  MCB_CHECK_CUDA(launch_kernel(ln_long_kernel<T, BWD>, dim3(*blocks), dim3(512), 0, st, chained_launch(), p));
  MCB_CHECK_LAUNCH("layer_norm");
  return MCB_OK;
}
template <typename T, bool BWD>
int launch(const Params& p, bool vec, int sms, cudaStream_t st, int* blocks) {
  return vec ? launch_n<T, BWD, Vec16<T>::N>(p, sms, st, blocks) : launch_n<T, BWD, 1>(p, sms, st, blocks);
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
  MCB_CHECK_CUDA(launch_kernel(lnorm::ln_reduce_kernel, dim3(static_cast<unsigned>((2 * D + 31) / 32)), dim3(1024), 0, st, chained_launch(),
                               static_cast<const float*>(p.part), blocks, p.D, dw, db, accumulate));
  MCB_CHECK_LAUNCH("layer_norm_reduce");
  return MCB_OK;
}
