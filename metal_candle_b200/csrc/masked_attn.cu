// Attention under document / prefix masks, with a score cap and a distance bias, and its gradients:
//   s = scale q.k;  s = cap tanh(s / cap);  s -= slope |i - j|;  o = sum over visible j of softmax(s) v
//   P = exp(s - lse);  dv = P^T do;  dS = P (do v^T - do.o) (1 - tanh^2);  dq = scale dS k;  dk = scale dS^T q
// The entry points, and kernels on CUDA cores for float32 (the validation path) and for bfloat16 heads of other sizes than 64,
// which flash_attn.cu takes to the tensor cores.
//
// CUDA-core kernels: tiles of 32 x 64, 256 threads, a thread has rows ty + 16 i and columns tx + 16 j of a product (two by four: the longest
// block's chain of tiles is what a launch takes at the sizes this is for, 12 heads x 1200 positions, forward: 184 us, 64 x 64 tiles by 256
// threads 282).  Bound by the operands' way from shared memory: 12 of 72 TFLOP/s.  Tiles are float32 rows of D + 4 elements: the
// four extra put the sixteen rows that a half warp reads on different banks for every D that is a multiple of 8.  One pass over the
// keys that some row of the tile sees, with the running maximum and sum; nothing of size seq x seq is stored and no sum uses
// atomics.  The backward pass is a kernel by query tiles (dq, and delta and lse for the other) and one by key tiles (dk, dv).
#include <cooperative_groups.h>

#include "masked_attn.cuh"

namespace cg = cooperative_groups;

namespace mcb {
namespace mattn {
namespace {

constexpr int kRows = 32, kB = 64, kThreads = 256, kLdP = 68;   // rows of a block's tile, and of the tiles it walks over
constexpr int kR = 2;   // rows of a thread: ty, ty + 16

__host__ __device__ constexpr int tile_floats(int d) { return kB * (d + 4); }
__host__ __device__ constexpr int rows_floats(int d) { return kRows * (d + 4); }
inline size_t smem_fwd(int d) { return (rows_floats(d) + 2 * tile_floats(d) + kRows * kLdP) * sizeof(float); }
inline size_t smem_bwd(int d) { return (2 * rows_floats(d) + 2 * tile_floats(d) + 2 * kRows * kLdP) * sizeof(float); }

// rows [first, first + COUNT) of a [.., S, D] plane as float32; `step` elements between rows; rows outside [0, S) are zeros
template <int COUNT, typename T>
__device__ __forceinline__ void load_tile(float* dst, const T* plane, int64_t step, int first, int S, int D) {
  // half a warp to a row of up to 64 elements, a warp to a longer one
  const int wide = D > 64 ? 32 : 16, c = threadIdx.x % wide * 4;
  if (c >= D) return;
#pragma unroll 4
  for (int r = threadIdx.x / wide; r < COUNT; r += kThreads / wide) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (first + r < S) {
      const T* s = plane + (first + r) * step + c;
      if constexpr (sizeof(T) == 4) {
        v = *reinterpret_cast<const float4*>(s);
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(s);
        v = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
      }
    }
    *reinterpret_cast<float4*>(dst + r * (D + 4) + c) = v;
  }
}

// acc[i][j] = sum_k a[ty + 16 i][k] b[tx + 16 j][k] for i < ni, j < nj (rows and columns that exist; others stay 0).  Even and odd k are summed
// apart, two multiply-adds to an instruction.
__device__ __forceinline__ void mul_nt(float (&acc)[kR][4], const float* a, const float* b, int D, int ty, int tx, int ni, int nj) {
  float2 sum[kR][4];
#pragma unroll
  for (int i = 0; i < kR; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = make_float2(0.0f, 0.0f);
  const int ld = D + 4;
  a += ty * ld;
  b += tx * ld;
  if (ni == kR && nj == 4) {
#pragma unroll 2
    for (int k = 0; k < D; k += 4) {
      float4 x[kR], y[4];
#pragma unroll
      for (int i = 0; i < kR; ++i) x[i] = *reinterpret_cast<const float4*>(a + 16 * i * ld + k);
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(b + 16 * j * ld + k);
#pragma unroll
      for (int i = 0; i < kR; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] = __ffma2_rn(make_float2(x[i].x, x[i].y), make_float2(y[j].x, y[j].y), sum[i][j]);
#pragma unroll
      for (int i = 0; i < kR; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] = __ffma2_rn(make_float2(x[i].z, x[i].w), make_float2(y[j].z, y[j].w), sum[i][j]);
    }
  } else {
    for (int k = 0; k < D; k += 4)
#pragma unroll
      for (int i = 0; i < kR; ++i) {
        if (i >= ni) break;
        const float4 x = *reinterpret_cast<const float4*>(a + 16 * i * ld + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j >= nj) break;
          const float4 y = *reinterpret_cast<const float4*>(b + 16 * j * ld + k);
          sum[i][j] = __ffma2_rn(make_float2(x.x, x.y), make_float2(y.x, y.y), sum[i][j]);
          sum[i][j] = __ffma2_rn(make_float2(x.z, x.w), make_float2(y.z, y.w), sum[i][j]);
        }
      }
  }
#pragma unroll
  for (int i = 0; i < kR; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = sum[i][j].x + sum[i][j].y;
}

// acc[i][jj] += sum_k p[ty + 16 i][k] v[k][4 (tx + 16 jj) ..] for k < K (a multiple of 4 up to 64), i < ni
template <int DV>
__device__ __forceinline__ void mul_nn(float4 (&acc)[kR][DV], const float* p, const float* v, int D, int ty, int tx, int K, int ni) {
  const int ld = D + 4;
  p += ty * kLdP;
  v += 4 * tx;
#pragma unroll 4
  for (int k = 0; k < K; k += 4) {
    float4 x[kR];
#pragma unroll
    for (int i = 0; i < kR; ++i) x[i] = i < ni ? *reinterpret_cast<const float4*>(p + 16 * i * kLdP + k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int jj = 0; jj < DV; ++jj) {
      if (4 * (tx + 16 * jj) >= D) continue;
      float4 y[4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) y[kk] = *reinterpret_cast<const float4*>(v + (k + kk) * ld + 64 * jj);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int i = 0; i < kR; ++i) {
          const float f = kk == 0 ? x[i].x : kk == 1 ? x[i].y : kk == 2 ? x[i].z : x[i].w;
          const float2 a = __ffma2_rn(make_float2(f, f), make_float2(y[kk].x, y[kk].y), make_float2(acc[i][jj].x, acc[i][jj].y));
          const float2 b = __ffma2_rn(make_float2(f, f), make_float2(y[kk].z, y[kk].w), make_float2(acc[i][jj].z, acc[i][jj].w));
          acc[i][jj] = make_float4(a.x, a.y, b.x, b.y);
        }
    }
  }
}
// sixteens of rows and of columns that a tile from position `first` has, and its positions rounded up to fours
__device__ __forceinline__ int row_sixteens(int first, int end) { return end - first > 16 ? 2 : 1; }
__device__ __forceinline__ int sixteens(int first, int end) { return end - first >= kB ? 4 : (end - first + 15) / 16; }
__device__ __forceinline__ int fours(int first, int end) { return end - first >= kB ? kB : (end - first + 3) & ~3; }

template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = v;
  } else {
    __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
  }
}
// whether the four are finite: x - x is 0 for those and NaN for the others
__device__ __forceinline__ bool finite4(float4 v) { return (v.x - v.x) + (v.y - v.y) + (v.z - v.z) + (v.w - v.w) == 0.0f; }
// over the sixteen lanes that share a row
__device__ __forceinline__ float row_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A block's item: a quarter of one of the mask's tiles, the longest tiles first, and a head.
struct Item {
  int b, first, head;
};
__device__ __forceinline__ Item item_of(const int4* work, int heads, int block) {
  const int quarter = block / heads;
  const int4 t = work[quarter >> 2];
  Item w;
  w.head = block % heads;
  w.b = t.x;
  w.first = t.y * amask::kTile + (quarter & 3) * kRows;
  return w;
}
// The intervals of the tile's rows into shared memory, and the positions that any of them covers.  All threads.
__device__ __forceinline__ int2 load_ranges(int2* rows, int* ends, const int2* all, const Call& c, const Item& w) {
  if (threadIdx.x == 0) { ends[0] = 0x7fffffff; ends[1] = 0; }
  __syncthreads();
  if (threadIdx.x < kRows) {
    const int s = w.first + threadIdx.x;
    const int2 r = s < c.S ? all[static_cast<int64_t>(w.b) * c.S + s] : make_int2(0, 0);
    rows[threadIdx.x] = r;
    if (r.x < r.y) { atomicMin(&ends[0], r.x); atomicMax(&ends[1], r.y); }
  }
  __syncthreads();
  return make_int2(ends[0], ends[1]);
}

template <typename T, int DV>
__global__ void __launch_bounds__(kThreads, 3) masked_fwd_kernel(const __grid_constant__ Call c) {
  extern __shared__ float4 smem4[];
  __shared__ int2 rows[kRows];
  __shared__ int ends[2], bad[kRows];
  float* sQ = reinterpret_cast<float*>(smem4);
  float* sK = sQ + rows_floats(c.D);
  float* sV = sK + tile_floats(c.D);
  float* sP = sV + tile_floats(c.D);
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  grid_launch_dependents();
  grid_dependency_wait();
  const Item w = item_of(c.mask.qwork, c.Hk * c.G, blockIdx.x);
  if (w.first >= c.S) return;
  const int hk = w.head / c.G, g = w.head % c.G;
  if (threadIdx.x < kRows) bad[threadIdx.x] = 0;
  const int2 range = load_ranges(rows, ends, c.mask.rows, c, w);
  load_tile<kRows>(sQ, static_cast<const T*>(c.q) + q_row(c, w.b, hk, g, 0) * c.D, c.D, w.first, c.S, c.D);
  const float slope2 = c.slopes ? c.slopes[w.head] * kLog2e : 0.0f;
  const int ni = row_sixteens(w.first, c.S);
  float m[kR], l[kR];
  float4 acc[kR][DV] = {};
#pragma unroll
  for (int i = 0; i < kR; ++i) { m[i] = kNoScore; l[i] = 0.0f; }
  for (int j0 = range.x; j0 < range.y; j0 += kB) {
    __syncthreads();
    load_tile<kB>(sK, static_cast<const T*>(c.k) + k_row(c, w.b, hk, 0) * c.D, c.D, j0, c.S, c.D);
    load_tile<kB>(sV, static_cast<const T*>(c.v) + k_row(c, w.b, hk, 0) * c.D, c.D, j0, c.S, c.D);
    __syncthreads();
    float s[kR][4];
    mul_nt(s, sQ, sK, c.D, ty, tx, ni, sixteens(j0, range.y));
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      if (i >= ni) break;
      const int2 sees = rows[ty + 16 * i];
      const int qpos = w.first + ty + 16 * i;
      float top = kNoScore;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = j0 + tx + 16 * j;
        float bent;
        s[i][j] = key >= sees.x && key < sees.y ? score2(c, s[i][j], slope2, abs(qpos - key), bent) : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
      top = fmaxf(row_max(top), m[i]);
      const float old = exp2f(m[i] - top);
      m[i] = top;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = exp2f(s[i][j] - top);
        sum += p;
        sP[(ty + 16 * i) * kLdP + tx + 16 * j] = p;
      }
      l[i] = fmaf(l[i], old, row_sum(sum));
#pragma unroll
      for (int jj = 0; jj < DV; ++jj) {
        acc[i][jj].x *= old; acc[i][jj].y *= old; acc[i][jj].z *= old; acc[i][jj].w *= old;
      }
    }
    __syncthreads();
    mul_nn<DV>(acc, sP, sV, c.D, ty, tx, fours(j0, range.y), ni);
  }
#pragma unroll
  for (int i = 0; i < kR; ++i) {
    const int s = w.first + ty + 16 * i;
    if (s >= c.S) continue;
    const bool none = l[i] == 0.0f;
    const float inv = none ? 0.0f : 1.0f / l[i];
    T* out = static_cast<T*>(c.o) + o_at(c, w.b, hk, g, s);
#pragma unroll
    for (int jj = 0; jj < DV; ++jj) {
      const int col = 4 * (tx + 16 * jj);
      if (col >= c.D) continue;
      float4 v = acc[i][jj];
      v = none ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
      if (!finite4(v) && l[i] == l[i]) bad[ty + 16 * i] = 1;   // (a sum of weights that is NaN: so is every element, by right)
      store4(out + col, v);
    }
    if (c.lse != nullptr && tx == 0) c.lse[q_row(c, w.b, hk, g, s)] = none ? -INFINITY : (m[i] + log2f(l[i])) * kLn2;
  }
  __syncthreads();
  for (int r = threadIdx.x >> 5; r < kRows; r += kThreads / 32)
    if (bad[r]) fwd_row<T>(c, w.b, hk, g, w.first + r);
}

// bfloat16: delta = sum of P dP is taken here and not from the rounded o, and what that changes put right at the end, by a second sum (see
// attn_dq_masked_kernel).
template <typename T, int DV>
__global__ void __launch_bounds__(kThreads) masked_dq_kernel(const __grid_constant__ Call c) {
  extern __shared__ float4 smem4[];
  __shared__ int2 rows[kRows];
  __shared__ int ends[2], bad[kRows];
  __shared__ float s_lse2[kRows], s_delta[kRows];
  float* sQ = reinterpret_cast<float*>(smem4);
  float* sO = sQ + rows_floats(c.D);   // d o
  float* sK = sO + rows_floats(c.D);
  float* sV = sK + tile_floats(c.D);
  float* sS = sV + tile_floats(c.D);
  float* sP = sS + kRows * kLdP;
  constexpr bool kExact = sizeof(T) == 2;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  grid_launch_dependents();
  grid_dependency_wait();
  const Item w = item_of(c.mask.qwork, c.Hk * c.G, blockIdx.x);
  if (w.first >= c.S) return;
  const int hk = w.head / c.G, g = w.head % c.G;
  if (threadIdx.x < kRows) bad[threadIdx.x] = 0;
  const int2 range = load_ranges(rows, ends, c.mask.rows, c, w);
  const int64_t o0 = o_at(c, w.b, hk, g, 0), ostep = c.o_tok ? static_cast<int64_t>(c.Hk) * c.G * c.D : c.D;
  load_tile<kRows>(sQ, static_cast<const T*>(c.q) + q_row(c, w.b, hk, g, 0) * c.D, c.D, w.first, c.S, c.D);
  load_tile<kRows>(sO, static_cast<const T*>(c.dout) + o0, ostep, w.first, c.S, c.D);
  load_tile<kRows>(sK, static_cast<const T*>(c.o_in) + o0, ostep, w.first, c.S, c.D);
  __syncthreads();
  const int64_t pitch = amask::tiles_of(c.S) * amask::kTile;
  for (int r = threadIdx.x >> 5; r < kRows; r += kThreads / 32) {
    float d = 0.0f;
    for (int e = threadIdx.x & 31; e < c.D; e += 32) d = fmaf(sO[r * (c.D + 4) + e], sK[r * (c.D + 4) + e], d);
    d = warp_sum(d);
    if ((threadIdx.x & 31) == 0) {
      const int s = w.first + r;
      float lse2 = INFINITY;   // of a row that sees nothing: P = 0
      if (s < c.S && rows[r].x < rows[r].y) {
        const float v = c.lse[q_row(c, w.b, hk, g, s)];
        if (v != -INFINITY) lse2 = v * kLog2e;
      }
      s_lse2[r] = lse2;
      s_delta[r] = d;
      const int64_t at = ((static_cast<int64_t>(w.b) * c.Hk + hk) * c.G + g) * pitch + s;
      if (!kExact) c.ndelta[at] = -d;
      c.nlse2[at] = -lse2;
    }
  }
  const float slope2 = c.slopes ? c.slopes[w.head] * kLog2e : 0.0f;
  const int ni = row_sixteens(w.first, c.S);
  float4 acc[kR][DV] = {}, acc2[kExact ? kR : 1][DV] = {};
  float exact[kR] = {};
  for (int j0 = range.x; j0 < range.y; j0 += kB) {
    __syncthreads();
    load_tile<kB>(sK, static_cast<const T*>(c.k) + k_row(c, w.b, hk, 0) * c.D, c.D, j0, c.S, c.D);
    load_tile<kB>(sV, static_cast<const T*>(c.v) + k_row(c, w.b, hk, 0) * c.D, c.D, j0, c.S, c.D);
    __syncthreads();
    float s[kR][4], dp[kR][4];
    const int nj = sixteens(j0, range.y);
    mul_nt(s, sQ, sK, c.D, ty, tx, ni, nj);
    mul_nt(dp, sO, sV, c.D, ty, tx, ni, nj);
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      if (i >= ni) break;
      const int r = ty + 16 * i;
      const int2 sees = rows[r];
      const float lse2 = s_lse2[r], delta = s_delta[r];
      const bool single = sees.y - sees.x == 1;   // P = 1 whatever the score: delta is its dP, to the bit, and dS = 0 here and in the next kernel
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = j0 + tx + 16 * j;
        float p, t, ds = 0.0f, pt = 0.0f;
        if (key >= sees.x && key < sees.y) {
          p = pair_p(c, s[i][j], slope2, abs(w.first + r - key), lse2, t);
          pt = p * t;
          if (single) p = fmaf(p, 0.0f, 1.0f);
          pt = single ? 0.0f : pt;
          ds = p * (single ? dp[i][j] * 0.0f : dp[i][j] - delta) * t;
          exact[i] = fmaf(p, dp[i][j], exact[i]);
        }
        sS[r * kLdP + tx + 16 * j] = ds;
        if (kExact) sP[r * kLdP + tx + 16 * j] = pt;
      }
    }
    __syncthreads();
    mul_nn<DV>(acc, sS, sK, c.D, ty, tx, fours(j0, range.y), ni);
    if constexpr (kExact) mul_nn<DV>(acc2, sP, sK, c.D, ty, tx, fours(j0, range.y), ni);
  }
#pragma unroll
  for (int i = 0; i < kR; ++i) {
    const int s = w.first + ty + 16 * i;
    float put_right = 0.0f;
    const float d = row_sum(exact[i]);
    const int2 sees = rows[ty + 16 * i];
    if constexpr (kExact) put_right = s_delta[ty + 16 * i] - d;
    if (kExact || sees.y - sees.x == 1) {
      if (tx == 0) c.ndelta[((static_cast<int64_t>(w.b) * c.Hk + hk) * c.G + g) * pitch + s] = -d;
    }
    if (s >= c.S) continue;
    T* out = static_cast<T*>(c.dq) + q_row(c, w.b, hk, g, s) * c.D;
#pragma unroll
    for (int jj = 0; jj < DV; ++jj) {
      const int col = 4 * (tx + 16 * jj);
      if (col >= c.D) continue;
      float4 v = acc[i][jj];
      if constexpr (kExact) {
        const float4 k = acc2[i][jj];
        v = make_float4(fmaf(put_right, k.x, v.x), fmaf(put_right, k.y, v.y), fmaf(put_right, k.z, v.z), fmaf(put_right, k.w, v.w));
      }
      v = make_float4(v.x * c.scale, v.y * c.scale, v.z * c.scale, v.w * c.scale);
      if (!finite4(v) && d == d) bad[ty + 16 * i] = 1;   // (delta, of what the row sees alone, NaN: so is every element)
      store4(out + col, v);
    }
  }
  __syncthreads();
  for (int r = threadIdx.x >> 5; r < kRows; r += kThreads / 32)
    if (bad[r]) dq_row<T>(c, w.b, hk, g, w.first + r);
}

template <typename T, int DV>
__global__ void __launch_bounds__(kThreads) masked_dkv_kernel(const __grid_constant__ Call c) {
  extern __shared__ float4 smem4[];
  __shared__ int2 rows[kRows];
  __shared__ int ends[2], bad[kRows];
  float* sK = reinterpret_cast<float*>(smem4);
  float* sV = sK + rows_floats(c.D);
  float* sQ = sV + rows_floats(c.D);
  float* sO = sQ + tile_floats(c.D);
  float* sP = sO + tile_floats(c.D);
  float* sS = sP + kRows * kLdP;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  grid_launch_dependents();
  grid_dependency_wait();
  // the blocks of a cluster share a tile's steps (a head and 64 queries each), consecutive ones each
  cg::cluster_group cl = cg::this_cluster();
  const int parts = static_cast<int>(cl.num_blocks()), part = static_cast<int>(cl.block_rank());
  const Item w = item_of(c.mask.kwork, c.Hk, blockIdx.x / parts);
  if (w.first >= c.S) return;   // (all of the cluster)
  const int hk = w.head, ni = row_sixteens(w.first, c.S);
  if (threadIdx.x < kRows) bad[threadIdx.x] = 0;
  const int2 range = load_ranges(rows, ends, c.mask.keys, c, w);
  load_tile<kRows>(sK, static_cast<const T*>(c.k) + k_row(c, w.b, hk, 0) * c.D, c.D, w.first, c.S, c.D);
  load_tile<kRows>(sV, static_cast<const T*>(c.v) + k_row(c, w.b, hk, 0) * c.D, c.D, w.first, c.S, c.D);
  const int64_t pitch = amask::tiles_of(c.S) * amask::kTile, ostep = c.o_tok ? static_cast<int64_t>(c.Hk) * c.G * c.D : c.D;
  float4 gk[kR][DV] = {}, gv[kR][DV] = {};
  const int per_head = range.y > range.x ? (range.y - range.x + kB - 1) / kB : 0;
  const int64_t steps = static_cast<int64_t>(c.G) * per_head;
  for (int64_t step = steps * part / parts; step < steps * (part + 1) / parts; ++step) {
    const int g = static_cast<int>(step / per_head), i0 = range.x + static_cast<int>(step % per_head) * kB;
    const float slope2 = c.slopes ? c.slopes[hk * c.G + g] * kLog2e : 0.0f;
    const int64_t srow = ((static_cast<int64_t>(w.b) * c.Hk + hk) * c.G + g) * pitch;
    {
      __syncthreads();
      load_tile<kB>(sQ, static_cast<const T*>(c.q) + q_row(c, w.b, hk, g, 0) * c.D, c.D, i0, c.S, c.D);
      load_tile<kB>(sO, static_cast<const T*>(c.dout) + o_at(c, w.b, hk, g, 0), ostep, i0, c.S, c.D);
      __syncthreads();
      float s[kR][4], dp[kR][4], lse2[4], delta[4];   // rows: keys, columns: queries
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int qpos = i0 + tx + 16 * j;
        lse2[j] = qpos < c.S ? -c.nlse2[srow + qpos] : INFINITY;
        delta[j] = qpos < c.S ? -c.ndelta[srow + qpos] : 0.0f;
      }
      const int nj = sixteens(i0, range.y);
      mul_nt(s, sK, sQ, c.D, ty, tx, ni, nj);
      mul_nt(dp, sV, sO, c.D, ty, tx, ni, nj);
#pragma unroll
      for (int i = 0; i < kR; ++i) {
        if (i >= ni) break;
        const int r = ty + 16 * i;
        const int2 seen = rows[r];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int qpos = i0 + tx + 16 * j;
          float p = 0.0f, ds = 0.0f;
          if (qpos >= seen.x && qpos < seen.y && lse2[j] != INFINITY)
            ds = pair_ds(c, s[i][j], dp[i][j], slope2, abs(qpos - w.first - r), lse2[j], delta[j], p);
          sP[r * kLdP + tx + 16 * j] = p;
          sS[r * kLdP + tx + 16 * j] = ds;
        }
      }
      __syncthreads();
      mul_nn<DV>(gv, sP, sO, c.D, ty, tx, fours(i0, range.y), ni);
      mul_nn<DV>(gk, sS, sQ, c.D, ty, tx, fours(i0, range.y), ni);
    }
  }
  if (parts > 1) {
    // every block's sums into its own shared memory (over Q and d O), then the first adds the others' to its own, in order
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kR; ++i)
#pragma unroll
      for (int jj = 0; jj < DV; ++jj) {
        const int col = 4 * (tx + 16 * jj);
        if (col >= c.D) continue;
        *reinterpret_cast<float4*>(sQ + (ty + 16 * i) * (c.D + 4) + col) = gk[i][jj];
        *reinterpret_cast<float4*>(sO + (ty + 16 * i) * (c.D + 4) + col) = gv[i][jj];
      }
    cl.sync();
    if (part == 0)
      for (int q = 1; q < parts; ++q) {
        const float *pk = cl.map_shared_rank(sQ, q), *pv = cl.map_shared_rank(sO, q);
#pragma unroll
        for (int i = 0; i < kR; ++i)
#pragma unroll
          for (int jj = 0; jj < DV; ++jj) {
            const int col = 4 * (tx + 16 * jj);
            if (col >= c.D || i >= ni) continue;
            const float4 x = *reinterpret_cast<const float4*>(pk + (ty + 16 * i) * (c.D + 4) + col), y = *reinterpret_cast<const float4*>(pv + (ty + 16 * i) * (c.D + 4) + col);
            gk[i][jj] = make_float4(gk[i][jj].x + x.x, gk[i][jj].y + x.y, gk[i][jj].z + x.z, gk[i][jj].w + x.w);
            gv[i][jj] = make_float4(gv[i][jj].x + y.x, gv[i][jj].y + y.y, gv[i][jj].z + y.z, gv[i][jj].w + y.w);
          }
      }
    cl.sync();   // no block leaves while the first reads its sums
    if (part != 0) return;
  }
#pragma unroll
  for (int i = 0; i < kR; ++i) {
    const int s = w.first + ty + 16 * i;
    if (s >= c.S) continue;
    const int64_t at = k_row(c, w.b, hk, s) * c.D;
#pragma unroll
    for (int jj = 0; jj < DV; ++jj) {
      const int col = 4 * (tx + 16 * jj);
      if (col >= c.D) continue;
      float4 k = gk[i][jj];
      k = make_float4(k.x * c.scale, k.y * c.scale, k.z * c.scale, k.w * c.scale);
      if (!finite4(k) || !finite4(gv[i][jj])) bad[ty + 16 * i] = 1;
      store4(static_cast<T*>(c.dk) + at + col, k);
      store4(static_cast<T*>(c.dv) + at + col, gv[i][jj]);
    }
  }
  __syncthreads();
  for (int r = threadIdx.x >> 5; r < kRows; r += kThreads / 32)
    if (bad[r]) dkv_row<T>(c, w.b, hk, w.first + r);
}

int launch_one(void (*kernel)(Call), const char* name, int64_t blocks, int cluster, size_t smem, const Call& c, cudaStream_t st) {
  if (blocks > 0x7fffffffll) return fail(MCB_ERR_SHAPE, "masked attention: %lld blocks", (long long)blocks);
  // (the most of any call: another thread's launch of the same kernel must not find less)
  MCB_CHECK_CUDA(cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_bwd(128))));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = chained_launch() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster); attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 2 : 1;
  MCB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, c));
  MCB_CHECK_LAUNCH(name);
  return MCB_OK;
}
template <typename T>
int launch_fwd(const Call& c, cudaStream_t st) {
  const int64_t quarters = 4 * amask::tiles_of(c.S) * c.B;
  return launch_one(c.D <= 64 ? masked_fwd_kernel<T, 1> : masked_fwd_kernel<T, 2>, "masked_fwd_kernel", quarters * c.Hk * c.G, 1, smem_fwd(c.D), c, st);
}
template <typename T>
int launch_bwd(const Call& c, int sms, cudaStream_t st) {
  const int64_t quarters = 4 * amask::tiles_of(c.S) * c.B;
  if (int rc = launch_one(c.D <= 64 ? masked_dq_kernel<T, 1> : masked_dq_kernel<T, 2>, "masked_dq_kernel", quarters * c.Hk * c.G, 1, smem_bwd(c.D), c, st)) return rc;
  // clusters share a key tile's steps as long as a part has one and there are not many blocks to an SM: the longest tile's chain of steps is what
  // the launch takes (2 kv heads of 7 x 1200 positions of 80, whole backward pass: 2516 us unshared, 722 by 8)
  const int64_t tiles = quarters * c.Hk, steps = static_cast<int64_t>(c.G) * ((c.S + kB - 1) / kB);
  int parts = 1;
  while (parts < 8 && tiles * parts * 2 <= 8 * sms && parts * 2 <= steps) parts *= 2;
  return launch_one(c.D <= 64 ? masked_dkv_kernel<T, 1> : masked_dkv_kernel<T, 2>, "masked_dkv_kernel", tiles * parts, parts, smem_bwd(c.D), c, st);
}

inline size_t up1k(size_t v) { return (v + 1023) & ~static_cast<size_t>(1023); }
size_t stat_bytes(const mcb_masked_attention* a) {
  return up1k(static_cast<size_t>(a->batch) * a->kv_heads * a->groups * amask::tiles_of(a->seq) * amask::kTile * 4);
}

size_t k_bytes(const mcb_masked_attention* a) { return static_cast<size_t>(a->batch) * a->kv_heads * a->seq * a->head_dim * (a->dtype == MCB_F32 ? 4 : 2); }
size_t slopes_bytes(const mcb_masked_attention* a) { return static_cast<size_t>(a->kv_heads) * a->groups * 4; }
size_t lse_bytes(const mcb_masked_attention* a) { return static_cast<size_t>(a->batch) * a->kv_heads * a->groups * a->seq * 4; }

// What flash_attn.cu takes: its tiles are built for heads of 64.
bool tensor_cores(const mcb_masked_attention* a) { return a->dtype == MCB_BF16 && a->head_dim == 64; }

int fill(Call& c, const mcb_masked_attention* a, const char* who) {
  if (!a) return fail(MCB_ERR_NULL, "%s: the call is null", who);
  if (!a->mask) return fail(MCB_ERR_NULL, "%s: mask is null", who);
  if (a->dtype != MCB_F32 && a->dtype != MCB_BF16) return fail(MCB_ERR_UNSUPPORTED, "%s: dtype %d", who, a->dtype);
  const size_t need = mcb_attention_mask_bytes(a->batch, a->seq);
  if (need == 0) return fail(MCB_ERR_SHAPE, "%s: batch=%lld seq=%lld", who, (long long)a->batch, (long long)a->seq);
  if (a->mask_bytes < need) return fail(MCB_ERR_SHAPE, "%s: a mask of %zu bytes is none of %lld x %lld positions", who, a->mask_bytes, (long long)a->batch, (long long)a->seq);
  if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8 != 0)
    return fail(MCB_ERR_UNSUPPORTED, "%s: head dimension %lld (multiples of 8 up to 128)", who, (long long)a->head_dim);
  // rows and work items are counted in 32 bits, tiles of 128 positions and up to 8 blocks to an item
  if (a->kv_heads <= 0 || a->groups <= 0 || a->kv_heads > 0x7fffffff || a->groups > 0x7fffffff / a->kv_heads ||
      a->batch * amask::tiles_of(a->seq) > 0x07ffffffll / (a->kv_heads * a->groups))
    return fail(MCB_ERR_SHAPE, "%s: batch=%lld kv_heads=%lld groups=%lld seq=%lld", who, (long long)a->batch, (long long)a->kv_heads, (long long)a->groups, (long long)a->seq);
  const auto finite = [](float v) { return v - v == 0.0f; };
  if (!(a->scale > 0.0f && finite(a->scale * kLog2e))) return fail(MCB_ERR_SHAPE, "%s: scale must be positive and finite", who);
  // (a quotient below 2^-126 has lost digits that every score would be short of)
  const float bend = a->scale / a->softcap;
  if (!(a->softcap >= 0.0f && finite(a->softcap * kLog2e) && (a->softcap == 0.0f || (finite(bend) && bend >= 0x1p-126f))))
    return fail(MCB_ERR_SHAPE, "%s: softcap must be 0 (none) or positive and finite, and scale / softcap within float32's normal numbers", who);
  if (!aligned16(a->mask) || (reinterpret_cast<uintptr_t>(a->slopes) & 3) != 0) return fail(MCB_ERR_ALIGN, "%s: alignment of the mask or the slopes", who);
  c = Call{};
  c.mask = amask::view(a->mask, a->batch, a->seq);
  c.slopes = a->slopes;
  c.B = static_cast<int>(a->batch); c.S = static_cast<int>(a->seq); c.Hk = static_cast<int>(a->kv_heads);
  c.G = static_cast<int>(a->groups); c.D = static_cast<int>(a->head_dim);
  c.o_tok = a->o_token_major != 0;
  c.scale = a->scale; c.cap = a->softcap;
  return MCB_OK;
}

}  // namespace
}  // namespace mattn
}  // namespace mcb

using namespace mcb;

extern "C" int mcb_attention_masked_fwd(const mcb_masked_attention* a, const void* q, const void* k, const void* v, void* o, float* lse,
                                        void* stream) {
  MCB_NVTX_RANGE("mcb_attention_masked_fwd");
  mattn::Call c;
  if (int rc = mattn::fill(c, a, "attention_masked_fwd")) return rc;
  if (!q || !k || !v || !o) return fail(MCB_ERR_NULL, "attention_masked_fwd: q, k, v or o is null");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o)) return fail(MCB_ERR_ALIGN, "attention_masked_fwd: 16-byte alignment");
  if (!on_boundary(4, lse)) return fail(MCB_ERR_ALIGN, "attention_masked_fwd: lse is not aligned to its elements");
  const size_t kb = mattn::k_bytes(a), qb = kb * a->groups;
  const Range ranges[] = {{o, qb}, {lse, mattn::lse_bytes(a)}, {q, qb}, {k, kb}, {v, kb}, {a->mask, mcb_attention_mask_bytes(a->batch, a->seq)},
                          {a->slopes, mattn::slopes_bytes(a)}};
  if (outputs_overlap(ranges, 2)) return fail(MCB_ERR_SHAPE, "attention_masked_fwd: o or lse overlaps an input or the other");
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  c.q = q; c.k = k; c.v = v; c.o = o; c.lse = lse; c.status = ds->status_word;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (mattn::tensor_cores(a)) return mattn::launch_fwd_umma(c, ds, st);
  return a->dtype == MCB_F32 ? mattn::launch_fwd<float>(c, st) : mattn::launch_fwd<__nv_bfloat16>(c, st);
}

extern "C" size_t mcb_attention_masked_workspace_bytes(const mcb_masked_attention* a) {
  mattn::Call c;
  if (mattn::fill(c, a, "attention_masked_workspace_bytes") != MCB_OK) return 0;
  return 2 * mattn::stat_bytes(a);
}

extern "C" int mcb_attention_masked_bwd(const mcb_masked_attention* a, const void* q, const void* k, const void* v, const void* o,
                                        const float* lse, const void* dout, void* dq, void* dk, void* dv, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  MCB_NVTX_RANGE("mcb_attention_masked_bwd");
  mattn::Call c;
  if (int rc = mattn::fill(c, a, "attention_masked_bwd")) return rc;
  if (!q || !k || !v || !o || !lse || !dout || !dq || !dk || !dv) return fail(MCB_ERR_NULL, "attention_masked_bwd: a required pointer is null");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !aligned16(dout) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv))
    return fail(MCB_ERR_ALIGN, "attention_masked_bwd: 16-byte alignment");
  if (!on_boundary(4, lse)) return fail(MCB_ERR_ALIGN, "attention_masked_bwd: lse is not aligned to its elements");
  const size_t stat = mattn::stat_bytes(a);
  if (!workspace || workspace_bytes < 2 * stat || (reinterpret_cast<uintptr_t>(workspace) & 1023u) != 0)
    return fail(MCB_ERR_WORKSPACE, "attention_masked_bwd: workspace of %zu bytes, 1024-byte aligned, needed", 2 * stat);
  const size_t kb = mattn::k_bytes(a), qb = kb * a->groups;
  const Range ranges[] = {{dq, qb}, {dk, kb}, {dv, kb}, {workspace, 2 * stat}, {q, qb}, {k, kb}, {v, kb}, {o, qb}, {dout, qb}, {lse, mattn::lse_bytes(a)},
                          {a->mask, mcb_attention_mask_bytes(a->batch, a->seq)}, {a->slopes, mattn::slopes_bytes(a)}};
  if (outputs_overlap(ranges, 4)) return fail(MCB_ERR_SHAPE, "attention_masked_bwd: a gradient or the workspace overlaps an input or one another");
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  c.q = q; c.k = k; c.v = v; c.o_in = o; c.lse = const_cast<float*>(lse); c.dout = dout; c.dq = dq; c.dk = dk; c.dv = dv;
  c.ndelta = static_cast<float*>(workspace);
  c.nlse2 = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + stat);
  c.status = ds->status_word;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (mattn::tensor_cores(a)) return mattn::launch_bwd_umma(c, ds, st);
  return a->dtype == MCB_F32 ? mattn::launch_bwd<float>(c, ds->sm_count, st) : mattn::launch_bwd<__nv_bfloat16>(c, ds->sm_count, st);
}
