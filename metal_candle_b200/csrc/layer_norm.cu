// Layer norm over the last dimension, forward and backward (beside RMSNorm):
//   mean = sum(x) / D;  var = sum((x - mean)^2) / D;  n = (x - mean) / sqrt(var + eps);  y = n w + b
//   g = dy w;  dx = rstd (g - sum(g) / D - n sum(g n) / D) (+ the gradient of the residual path);  dw = sum over rows of dy n;  db = of dy
// The variance is taken from the differences to the mean, which are in registers by then: E[x^2] - mean^2 would lose a row whose
// mean is large against its spread.  The backward pass takes both from x again instead of reading them: x is read anyway.
//
// HBM-bound: the forward reads x and writes y, the backward reads x and dy (and the residual) and writes dx.  A row is read once, by TPR
// threads (8 to 512, so that a thread has at most two 16-byte vectors of it, four where the row needs more than 512 x 2), with the
// next rows on their way in shared memory.  Blocks walk over rows; a thread's columns stay its own, so that its parts of dw and db
// are registers until the block writes them out, a line of partial sums each that a last kernel adds up in order: no atomics.
// Rows that are not whole vectors (D = 777) start at every alignment.  Row r starts (r D) mod N elements behind a vector boundary, which comes
// back every P = N / gcd(D, N) rows: a block takes rows of one residue mod P, and everything is the aligned case moved by a constant, with
// a ragged first and last vector.  Longer rows, and operands of different alignments, take a kernel that reads element by element.
#include <atomic>
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
  int D, period;            // rows until one starts at the same alignment again
  float eps;
};

// Sums over the TPR threads of a row, the same bits on all of them.  `buf` has a place for each warp of the block; a call with another
// buffer lies between two with the same one, whose barrier keeps them apart.
template <int TPR>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* buf) {
  v = lanes_sum<TPR>(v);
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
// Three at a time.  Where a warp has a row to itself two halves, then quarters of it take a sum each: nine exchanges instead of fifteen, in a
// longer chain (which costs the larger rows' kernels more than the exchanges do: 16384 x 1024 float32, backward: 50 us, 47 without).
template <int TPR>
__device__ __forceinline__ float3 row_sum3(float3 v, float3* buf) {
  if constexpr (TPR == 32) {
    constexpr uint32_t all = 0xffffffffu;
    const bool up = threadIdx.x & 16, right = threadIdx.x & 8;
    const float xy = (up ? v.y : v.x) + __shfl_xor_sync(all, up ? v.x : v.y, 16), z = v.z + __shfl_xor_sync(all, v.z, 16);
    float c = (right ? z : xy) + __shfl_xor_sync(all, right ? xy : z, 8);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) c += __shfl_xor_sync(all, c, o);
    return make_float3(__shfl_sync(all, c, 0), __shfl_sync(all, c, 16), __shfl_sync(all, c, 8));
  }
  v.x = lanes_sum<TPR>(v.x);
  v.y = lanes_sum<TPR>(v.y);
  v.z = lanes_sum<TPR>(v.z);
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

// Arithmetic on pairs: one instruction for two elements.
__device__ __forceinline__ float2 two(const float* v) { return make_float2(v[0], v[1]); }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ void put2(float* v, float2 x) { v[0] = x.x; v[1] = x.y; }

// ---- rows on their way -------------------------------------------------------------------------------------------------
// A block has `STAGES - 1` rounds of rows on their way from memory while it works on one (cp.async, every thread its own vectors):
// the bytes in flight are what the bandwidth is made of, and shared memory has room for them where registers have not.
__device__ __forceinline__ void cp_async16(void* dst, const void* src, int bytes) {
  const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

constexpr bool staged(int tpr, int k) { return tpr == 32 && k == 4; }   // see the backward kernel
constexpr int block_of(int tpr) { return tpr < 128 ? 128 : tpr; }
constexpr int stages_of(int tpr, int k) { return k * block_of(tpr) > 1024 ? 2 : 3; }   // (three would not fit for three operands)

// The rows of a block and a thread's part of them: vectors lane + TPR * k of a row, k < K.  Row r of the block's turn j is j * P + q.  SHIFT: a row
// begins `off` elements into its first vector.
template <typename T, int TPR, int K, bool SHIFT>
struct Rows {
  static constexpr int N = Vec16<T>::N, kBlock = block_of(TPR), kRows = kBlock / TPR, STAGES = stages_of(TPR, K);
  uint4* ring;
  int lane, nt, off, D, P, q;
  int64_t j, step, rows;
  static __host__ __device__ constexpr size_t smem(int nt) { return static_cast<size_t>(STAGES) * nt * K * kBlock * 16; }
  __device__ __forceinline__ Rows(void* base, const Params& p, int nt_) : ring(static_cast<uint4*>(base)), nt(nt_), D(p.D), P(SHIFT ? p.period : 1), rows(p.rows) {
    lane = threadIdx.x % TPR;
    q = SHIFT ? blockIdx.x % P : 0;
    j = static_cast<int64_t>(blockIdx.x / P) * kRows + threadIdx.x / TPR;
    step = static_cast<int64_t>(gridDim.x / P) * kRows;
    off = SHIFT ? static_cast<int>(((reinterpret_cast<uintptr_t>(p.x) & 15) / sizeof(T) + static_cast<int64_t>(q) * D) % N) : 0;
    // places of vectors that a row does not have are never loaded: they stay 0
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (!here(k))
        for (int i = 0; i < STAGES * nt; ++i) ring[(static_cast<size_t>(i) * K + k) * kBlock + threadIdx.x] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ int64_t row(int64_t turn) const { return turn * P + q; }
  __device__ __forceinline__ bool any(int64_t turn) const { return (turn - threadIdx.x / TPR) * P + q < rows; }   // some row of the block's
  __device__ __forceinline__ int col(int k) const { return N * (lane + TPR * k) - off; }   // of element 0 of a vector; may be below 0
  __device__ __forceinline__ bool here(int k) const { return col(k) < D; }
  __device__ __forceinline__ bool whole(int k) const { return !SHIFT || (col(k) >= 0 && col(k) + N <= D); }
  __device__ __forceinline__ bool in(int k, int e) const { return static_cast<unsigned>(col(k) + e) < static_cast<unsigned>(D); }
  __device__ __forceinline__ void fetch(int stage, int t, const T* x, int64_t turn) const {
    const int64_t r = row(turn);
    if (r >= rows) return;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (here(k)) {
        const T* from = x + r * D + col(k);
        int bytes = 16;
        if constexpr (SHIFT) {   // nothing behind the tensor is read (before it, at most the rest of its first 16 bytes)
          const int64_t left = (rows * D - (r * D + col(k))) * static_cast<int64_t>(sizeof(T));
          if (left < 16) bytes = static_cast<int>(left);
        }
        cp_async16(ring + (static_cast<size_t>(stage * nt + t) * K + k) * kBlock + threadIdx.x, from, bytes);
      }
  }
  // the vectors of a row as float32; elements outside the row are 0 (what a row that does not exist has is anything)
  __device__ __forceinline__ void get_vector(int stage, int t, int k, float (&f)[N]) const {
    load(f, reinterpret_cast<const T*>(ring + (static_cast<size_t>(stage * nt + t) * K + k) * kBlock + threadIdx.x));
  }
  __device__ __forceinline__ void get(int stage, int t, float (&v)[K][N]) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      get_vector(stage, t, k, v[k]);
      drop(v[k], k);
    }
  }
  static __device__ __forceinline__ void load(float (&f)[N], const T* p) {
    Vec16<T> v;
    v.raw = *reinterpret_cast<const decltype(v.raw)*>(p);
    v.to_float(f);
  }
  __device__ __forceinline__ void drop(float (&v)[N], int k) const {
    if constexpr (SHIFT) {
      if (!whole(k)) {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (!in(k, e)) v[e] = 0.0f;
      }
    }
  }
  // a vector of a weight [D], `none` where there is no weight
  __device__ __forceinline__ void weight(float (&f)[N], const T* w, int k, float none) const {
    if (!SHIFT && w != nullptr) return load(f, w + col(k));
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = none;
    if (w == nullptr) return;
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (in(k, e)) f[e] = to_f32(w[col(k) + e]);
  }
  __device__ __forceinline__ void store(T* out, int64_t turn, int k, const float (&f)[N]) const {
    T* to = out + row(turn) * D + col(k);
    Vec16<T> v;
    if (whole(k)) {
      v.from_float(f);
      *reinterpret_cast<decltype(v.raw)*>(to) = v.raw;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (in(k, e)) to[e] = from_f32<T>(f[e]);
    }
  }
};

template <typename T, int TPR, int K, bool SHIFT>
__global__ void __launch_bounds__(block_of(TPR)) ln_fwd_kernel(const Params p) {
  extern __shared__ uint4 smem4[];
  using R = Rows<T, TPR, K, SHIFT>;
  constexpr int N = R::N;
  __shared__ float buf[2][R::kBlock / 32];
  const T *x = static_cast<const T*>(p.x), *w = static_cast<const T*>(p.w), *b = static_cast<const T*>(p.b);
  T* y = static_cast<T*>(p.out);
  const float inv = 1.0f / static_cast<float>(p.D);
  R rows(smem4, p, 1);
  grid_launch_dependents();
  grid_dependency_wait();
#pragma unroll
  for (int i = 0; i < R::STAGES - 1; ++i) {
    rows.fetch(i, 0, x, rows.j + i * rows.step);
    cp_async_commit();
  }
  // a moved weight is read element by element: once, into registers
  float fw[SHIFT ? K : 1][N], fb[SHIFT ? K : 1][N];
  if constexpr (SHIFT) {
#pragma unroll
    for (int k = 0; k < K; ++k) { rows.weight(fw[k], w, k, 1.0f); rows.weight(fb[k], b, k, 0.0f); }
  }
  int stage = 0;
  for (int64_t j = rows.j; rows.any(j); j += rows.step) {
    float v[K][N];
    cp_async_wait<R::STAGES - 2>();
    rows.get(stage, 0, v);
    rows.fetch(stage == 0 ? R::STAGES - 1 : stage - 1, 0, x, j + (R::STAGES - 1) * rows.step);
    cp_async_commit();
    if (++stage == R::STAGES) stage = 0;
    float2 sum = both(0.0f), sq = sum;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < N; e += 2) sum = __fadd2_rn(two(&v[k][e]), sum);
    const float mean = row_sum<TPR>(sum.x + sum.y, buf[0]) * inv;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (rows.here(k)) {
#pragma unroll
        for (int e = 0; e < N; e += 2) put2(&v[k][e], __fadd2_rn(two(&v[k][e]), both(-mean)));
        rows.drop(v[k], k);
#pragma unroll
        for (int e = 0; e < N; e += 2) sq = __ffma2_rn(two(&v[k][e]), two(&v[k][e]), sq);
      }
    const float rstd = rsqrtf(row_sum<TPR>(sq.x + sq.y, buf[1]) * inv + p.eps);
    const int64_t row = rows.row(j);
    if (row >= p.rows) continue;   // (no barrier follows within the round)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!rows.here(k)) continue;
      float f[N], g[N];
      if constexpr (!SHIFT) { rows.weight(f, w, k, 1.0f); rows.weight(g, b, k, 0.0f); }
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const float2 n = __fmul2_rn(two(&v[k][e]), both(rstd));
        put2(&v[k][e], __ffma2_rn(n, two(SHIFT ? &fw[k][e] : &f[e]), two(SHIFT ? &fb[k][e] : &g[e])));
      }
      rows.store(y, j, k, v[k]);
    }
    if (rows.lane == 0) {
      if (p.mean != nullptr) p.mean[row] = mean;
      if (p.rstd != nullptr) p.rstd[row] = rstd;
    }
  }
}

// After the mean one more round of sums does: of (x - mean)^2, of g and of g (x - mean), from which rstd and both means of the backward
// formula follow.  SUMS: dw and db are asked for.
template <typename T, int TPR, int K, bool SHIFT, bool SUMS>
__global__ void __launch_bounds__(block_of(TPR), TPR == 256 ? 2 : 1) ln_bwd_kernel(const Params p) {
  extern __shared__ uint4 smem4[];
  using R = Rows<T, TPR, K, SHIFT>;
  constexpr int N = R::N;
  __shared__ float buf[R::kBlock / 32];
  __shared__ float3 buf3[R::kBlock / 32];
  const T *x = static_cast<const T*>(p.x), *w = static_cast<const T*>(p.w), *dy = static_cast<const T*>(p.dy), *res = static_cast<const T*>(p.res);
  T* dx = static_cast<T*>(p.out);
  const float inv = 1.0f / static_cast<float>(p.D);
  R rows(smem4, p, res != nullptr ? 3 : 2);
  auto fetch = [&](int stage, int64_t turn) {
    rows.fetch(stage, 0, x, turn);
    rows.fetch(stage, 1, dy, turn);
    if (res != nullptr) rows.fetch(stage, 2, res, turn);
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
  for (int i = 0; i < R::STAGES - 1; ++i) fetch(i, rows.j + i * rows.step);
  // the weight of a vector: where a thread has four, float32 in shared memory behind the ring; else from L1, or, where the row's vectors are not the
  // weight's, read element by element into registers once
  constexpr bool STAGED = staged(TPR, K), KEPT = SHIFT && !STAGED;
  float fw[KEPT ? K : 1][N];
  float* ws = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(smem4) + R::smem(rows.nt));
  if constexpr (KEPT) {
#pragma unroll
    for (int k = 0; k < K; ++k) rows.weight(fw[k], w, k, 1.0f);
  }
  if constexpr (STAGED) {
    for (int i = threadIdx.x; i < TPR * K * N; i += R::kBlock) {
      const int c = i - rows.off;
      ws[i] = static_cast<unsigned>(c) >= static_cast<unsigned>(p.D) ? 0.0f : w != nullptr ? to_f32(w[c]) : 1.0f;
    }
    __syncthreads();
  }
  auto weight = [&](float (&f)[N], int k) {
    if constexpr (STAGED) {
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        const float4 v = *reinterpret_cast<const float4*>(ws + N * (rows.lane + TPR * k) + e);
        f[e] = v.x; f[e + 1] = v.y; f[e + 2] = v.z; f[e + 3] = v.w;
      }
    } else if constexpr (KEPT) {
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = fw[k][e];
    } else {
      rows.weight(f, w, k, 1.0f);
    }
  };
  int stage = 0;
  for (int64_t j = rows.j; rows.any(j); j += rows.step) {
    float v[K][N], d[K][N];
    cp_async_wait<R::STAGES - 2>();
    rows.get(stage, 0, v);
    rows.get(stage, 1, d);
    const int now = stage;
    fetch(stage == 0 ? R::STAGES - 1 : stage - 1, j + (R::STAGES - 1) * rows.step);
    if (++stage == R::STAGES) stage = 0;
    float2 sum = both(0.0f);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < N; e += 2) sum = __fadd2_rn(two(&v[k][e]), sum);
    const float mean = row_sum<TPR>(sum.x + sum.y, buf) * inv;
    float2 sx = both(0.0f), sy = sx, sz = sx;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!rows.here(k)) continue;
      float f[N];
      weight(f, k);
#pragma unroll
      for (int e = 0; e < N; e += 2) put2(&v[k][e], __fadd2_rn(two(&v[k][e]), both(-mean)));
      rows.drop(v[k], k);
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const float2 o = two(&v[k][e]), g = __fmul2_rn(two(&d[k][e]), two(&f[e]));
        sx = __ffma2_rn(o, o, sx);
        sy = __fadd2_rn(g, sy);
        sz = __ffma2_rn(g, o, sz);
      }
    }
    const float3 s = row_sum3<TPR>(make_float3(sx.x + sx.y, sy.x + sy.y, sz.x + sz.y), buf3);
    const float rstd = rsqrtf(s.x * inv + p.eps);
    const float a = s.y * inv, q = s.z * inv * rstd;
    if (rows.row(j) >= p.rows) continue;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!rows.here(k)) continue;
      float f[N];
      weight(f, k);   // (again: registers for it would cost occupancy)
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const float2 n = __fmul2_rn(two(&v[k][e]), both(rstd)), g = two(&d[k][e]);
        if constexpr (SUMS) {
          put2(&gw[k][e], __ffma2_rn(g, n, two(&gw[k][e])));
          put2(&gb[k][e], __fadd2_rn(g, two(&gb[k][e])));
        }
        put2(&f[e], __ffma2_rn(n, both(-q), __ffma2_rn(g, two(&f[e]), both(-a))));
      }
      if (res != nullptr) {
        float r[N];
        rows.get_vector(now, 2, k, r);
#pragma unroll
        for (int e = 0; e < N; e += 2) put2(&f[e], __ffma2_rn(two(&f[e]), both(rstd), two(&r[e])));
      } else {
#pragma unroll
        for (int e = 0; e < N; e += 2) put2(&f[e], __fmul2_rn(two(&f[e]), both(rstd)));
      }
      rows.store(dx, j, k, f);
    }
  }
  if constexpr (SUMS) {
    float* out = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.D;
    if constexpr (R::kRows > 1) {
      cp_async_wait<0>();
      float* sums = reinterpret_cast<float*>(smem4);   // [2][D] of the block's row slots, over the ring
      for (int s = 0; s < R::kRows; ++s) {
        __syncthreads();
        if (static_cast<int>(threadIdx.x / TPR) != s) continue;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (rows.in(k, e)) {
              const int c = rows.col(k) + e;
              sums[c] = (s ? sums[c] : 0.0f) + gw[k][e];
              sums[p.D + c] = (s ? sums[p.D + c] : 0.0f) + gb[k][e];
            }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * p.D; i += R::kBlock) out[i] = sums[i];
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (rows.in(k, e)) { out[rows.col(k) + e] = gw[k][e]; out[p.D + rows.col(k) + e] = gb[k][e]; }
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
#pragma unroll 8
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

template <typename T, bool BWD, bool SHIFT, int TPR, int K>
int launch_k(const Params& p, int sms, cudaStream_t st, int* blocks) {
  using R = Rows<T, TPR, K, SHIFT>;
  constexpr size_t kWeight = BWD && staged(TPR, K) ? static_cast<size_t>(TPR) * K * R::N * 4 : 0;
  const size_t smem = R::smem(!BWD ? 1 : p.res != nullptr ? 3 : 2) + kWeight;
  static_assert(!BWD || R::kRows == 1 || 2 * sizeof(float) * TPR * K * R::N <= R::smem(2), "dw and db of the block's row slots lie over the ring");
  void (*kernel)(const Params) = ln_fwd_kernel<T, TPR, K, SHIFT>;
  if constexpr (BWD) kernel = p.part != nullptr ? ln_bwd_kernel<T, TPR, K, SHIFT, true> : ln_bwd_kernel<T, TPR, K, SHIFT, false>;
  // as many blocks as are on the device at once (each leaves a line of sums), a whole number of rounds of the alignments; asked once for
  // every kernel, number of operands and device
  static std::atomic<int> answer[4][64];
  int dev = 0;
  MCB_CHECK_CUDA(cudaGetDevice(&dev));
  if (dev >= 64) return fail(MCB_ERR_SHAPE, "layer norm: device %d out of range", dev);
  std::atomic<int>& known = answer[(BWD && p.part != nullptr) + 2 * (BWD && p.res != nullptr)][dev];
  int per_sm = known.load(std::memory_order_relaxed);
  if (per_sm == 0) {
    const size_t most = R::smem(BWD ? 3 : 1) + kWeight;   // (of any call of this kernel: another thread's launch must not find less)
    MCB_CHECK_CUDA(cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most)));
    MCB_CHECK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, R::kBlock, smem));
    if (per_sm < 1) per_sm = 1;
    known.store(per_sm, std::memory_order_relaxed);
  }
  const int64_t turns = (p.rows + p.period - 1) / p.period;   // rows of an alignment
  const int each = blocks_for(turns, R::kRows, sms, per_sm), most = blocks_for(p.rows, 1, sms, per_sm) / p.period;
  *blocks = p.period * (each < most || most < 1 ? each : most);
  MCB_CHECK_CUDA(launch_kernel(kernel, dim3(*blocks), dim3(R::kBlock), smem, st, chained_launch(), p));
  MCB_CHECK_LAUNCH("layer_norm");
  return MCB_OK;
}
// A row's threads: as few as have at most two vectors of it each, but a warp for up to four where that was the faster: forward (32768 x 896
// bfloat16, us: 32 threads with four 23, 64 with two 27), and backward of aligned bfloat16 rows, with the weight in shared memory (with the residual,
// reduction included: 55, 64 with two 60, 128 with one 69; aligned float32 30000 x 512: 57, 64 with two 54; moved bfloat16 20000 x 1001: 64 and 54).
template <typename T, bool BWD, bool SHIFT>
int launch_rows(const Params& p, int vecs, int sms, cudaStream_t st, int* blocks) {
  if (vecs <= 8) return launch_k<T, BWD, SHIFT, 8, 1>(p, sms, st, blocks);
  if (vecs <= 16) return launch_k<T, BWD, SHIFT, 8, 2>(p, sms, st, blocks);
  if (vecs <= 32) return launch_k<T, BWD, SHIFT, 32, 1>(p, sms, st, blocks);
  if (vecs <= 64) return launch_k<T, BWD, SHIFT, 32, 2>(p, sms, st, blocks);
  if constexpr (!BWD || (!SHIFT && sizeof(T) == 2))
    if (vecs <= 128) return launch_k<T, BWD, SHIFT, 32, 4>(p, sms, st, blocks);
  if (vecs <= 128) return launch_k<T, BWD, SHIFT, 64, 2>(p, sms, st, blocks);
  if (vecs <= 256) return launch_k<T, BWD, SHIFT, 128, 2>(p, sms, st, blocks);
  if (vecs <= 512) return launch_k<T, BWD, SHIFT, 256, 2>(p, sms, st, blocks);
  if (vecs <= 1024) return launch_k<T, BWD, SHIFT, 512, 2>(p, sms, st, blocks);
  return launch_k<T, BWD, SHIFT, 512, 4>(p, sms, st, blocks);
}
template <typename T, bool BWD>
int launch(Params& p, uintptr_t operands, uintptr_t weights, int sms, cudaStream_t st, int* blocks) {
  constexpr int N = Vec16<T>::N;
  // operands: the bits in which the row operands' addresses differ from one another, weights: all bits of the weights' addresses
  const bool alike = (operands & 15) == 0;
  const bool whole = p.D % N == 0 && (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && (weights & 15) == 0;
  const int vecs = whole ? p.D / N : (p.D + 2 * N - 2) / N;
  p.period = 1;
  if (alike && vecs <= 2048) {
    if (whole) return launch_rows<T, BWD, false>(p, vecs, sms, st, blocks);
    for (p.period = 1; p.D * static_cast<int64_t>(p.period) % N != 0; p.period *= 2) {}
    return launch_rows<T, BWD, true>(p, vecs, sms, st, blocks);
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
  if (!on_boundary(element_bytes(dtype), x, w, b, y) || !on_boundary(4, mean, rstd))
    return fail(MCB_ERR_ALIGN, "layernorm_fwd: a pointer is not aligned to its elements");
  const size_t row = static_cast<size_t>(D) * element_bytes(dtype), all = rows * row;
  const Range ranges[] = {{y, all}, {mean, rows * sizeof(float)}, {rstd, rows * sizeof(float)}, {y == x ? nullptr : x, all}, {w, row}, {b, row}};
  if (outputs_overlap(ranges, 3)) return fail(MCB_ERR_SHAPE, "layernorm_fwd: an output overlaps an input (but for y = x) or another output");
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  lnorm::Params p = {};
  p.x = x; p.w = w; p.b = b; p.out = y; p.mean = mean; p.rstd = rstd;
  p.rows = rows; p.D = static_cast<int>(D); p.eps = eps;
  const auto at = [](const void* v) { return reinterpret_cast<uintptr_t>(v); };
  const uintptr_t operands = at(x) ^ at(y), weights = at(w) | at(b);
  int blocks = 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == MCB_F32 ? lnorm::launch<float, false>(p, operands, weights, ds->sm_count, st, &blocks)
                          : lnorm::launch<__nv_bfloat16, false>(p, operands, weights, ds->sm_count, st, &blocks);
}

extern "C" size_t mcb_layernorm_bwd_workspace_bytes(int64_t rows, int64_t D) {
  if (rows <= 0 || D <= 0) return 0;
  const int64_t blocks = rows < 8 ? 8 : rows < lnorm::kMaxBlocks ? rows : lnorm::kMaxBlocks;   // (one an alignment at least)
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
  if (!on_boundary(element_bytes(dtype), x, w, dy, dx_residual, dx) || !on_boundary(4, dw, db))
    return fail(MCB_ERR_ALIGN, "layernorm_bwd: a pointer is not aligned to its elements");
  const size_t row = static_cast<size_t>(D) * element_bytes(dtype), all = rows * row, sum = D * sizeof(float);
  const auto other = [&](const void* v) { return dx == v ? nullptr : v; };   // (dx may be what it is made of, row for row)
  const Range ranges[] = {{dx, all}, {dw, sum}, {db, sum}, {sums ? workspace : nullptr, mcb_layernorm_bwd_workspace_bytes(rows, D)},
                          {other(x), all}, {other(dy), all}, {other(dx_residual), all}, {w, row}};
  if (outputs_overlap(ranges, 4))
    return fail(MCB_ERR_SHAPE, "layernorm_bwd: a gradient or the workspace overlaps an input (but for dx = dy or dx_residual) or one another");
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  lnorm::Params p = {};
  p.x = x; p.w = w; p.dy = dy; p.res = dx_residual; p.out = dx; p.part = sums ? static_cast<float*>(workspace) : nullptr;
  p.rows = rows; p.D = static_cast<int>(D); p.eps = eps;
  const auto at = [](const void* v) { return reinterpret_cast<uintptr_t>(v); };
  const uintptr_t operands = (at(x) ^ at(dx)) | (at(x) ^ at(dy)) | (dx_residual ? at(x) ^ at(dx_residual) : 0), weights = at(w);
  int blocks = 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = dtype == MCB_F32 ? lnorm::launch<float, true>(p, operands, weights, ds->sm_count, st, &blocks)
                                : lnorm::launch<__nv_bfloat16, true>(p, operands, weights, ds->sm_count, st, &blocks)) return rc;
  if (!sums) return MCB_OK;
  MCB_CHECK_CUDA(launch_kernel(lnorm::ln_reduce_kernel, dim3(static_cast<unsigned>((2 * D + 31) / 32)), dim3(1024), 0, st, chained_launch(),
                               static_cast<const float*>(p.part), blocks, p.D, dw, db, accumulate));
  MCB_CHECK_LAUNCH("layer_norm_reduce");
  return MCB_OK;
}
