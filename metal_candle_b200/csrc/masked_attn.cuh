// What the kernels of attention under a document / prefix mask share: the call, the score's shape, and one row at a time.
#pragma once
#include "attn_mask.cuh"

namespace mcb {
namespace mattn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Stands for "no score yet" as the running maximum: finite, so that a row that sees nothing has exponentials 2^(-inf - m) = 0
// and not NaN, and no finite score lies below.
constexpr float kNoScore = -3.4028235e38f;

struct Call {
  amask::View mask;
  const void *q, *k, *v, *o_in, *dout;
  void *o, *dq, *dk, *dv;
  float* lse;
  const float* slopes;   // [Hk * G] or null
  float* ndelta;         // backward scratch (see flash_attn.cu)
  float* nlse2;
  int B, S, Hk, G, D;
  int o_tok;
  float scale;           // of q.k
  float cap;             // 0: none
  int* status;
};

// tcgen05 kernels of flash_attn.cu: bfloat16, head dimension 64
int launch_fwd_umma(const Call& c, const DeviceState* ds, cudaStream_t st);
int launch_bwd_umma(const Call& c, const DeviceState* ds, cudaStream_t st);

// Row (nb, head g of its group, position s) of q, dq and lse; of k and v; of o and d o: in rows of D elements or, token-major, elements.
__device__ __forceinline__ int64_t q_row(const Call& c, int b, int hk, int g, int s) {
  return ((static_cast<int64_t>(b) * c.Hk + hk) * c.G + g) * c.S + s;
}
__device__ __forceinline__ int64_t k_row(const Call& c, int b, int hk, int s) { return (static_cast<int64_t>(b) * c.Hk + hk) * c.S + s; }
__device__ __forceinline__ int64_t o_at(const Call& c, int b, int hk, int g, int s) {
  if (!c.o_tok) return q_row(c, b, hk, g, s) * c.D;
  return ((static_cast<int64_t>(b) * c.S + s) * (c.Hk * c.G) + hk * c.G + g) * c.D;
}

// The score in units of log 2 from the dot product: scale, cap by tanh, distance bias; `bent` receives tanh (0 without a cap), whose
// square is what the cap takes off the derivative.
__device__ __forceinline__ float score2(const Call& c, float dot, float slope2, int distance, float& bent) {
  float s;
  bent = 0.0f;
  if (c.cap > 0.0f) {
    bent = tanhf(dot * (c.scale / c.cap));
    s = bent * (c.cap * kLog2e);
  } else {
    s = dot * (c.scale * kLog2e);
  }
  return slope2 != 0.0f ? fmaf(-slope2, static_cast<float>(distance), s) : s;
}

// ---- one row by one warp ------------------------------------------------------------------------------------------------
//
// A tile's product takes a masked probability of 0 times whatever lies at the masked position: an infinity or a NaN there (memory
// that nothing has written behind a document, a diverged neighbour) makes the sum NaN although the row does not see it.  A row that
// comes out not finite is therefore computed again from the positions that it sees alone, here.  With finite inputs none is, and a row
// that is NaN by right (a diverged run) is left as soon as that shows.
// 32 positions at a time: a lane takes the products of one of them by itself, then the warp adds their rows up, a lane the four elements from 4 l
// on (head dimensions up to 128).  Bound by latency: 2 heads of 16384 positions with every row taken again 45 ms forward and 107 backward,
// beside 0.2 and 0.47 where none is.  (Four rows and two pieces at a time, and no more: the kernels that call this hold its registers with theirs.
// With eight each 36 and 92, but the forward of a finite 16384 with a prefix took 447 us instead of 402.)
template <typename T>
__device__ __forceinline__ float lane_dot(const T* a, const T* b, int d) {
  constexpr int N = Vec16<T>::N;
  float s = 0.0f;
#pragma unroll 2
  for (int at = 0; at < d; at += N) {
    Vec16<T> x, y;
    x.raw = *reinterpret_cast<const decltype(x.raw)*>(a + at);
    y.raw = *reinterpret_cast<const decltype(y.raw)*>(b + at);
    float fx[N], fy[N];
    x.to_float(fx);
    y.to_float(fy);
#pragma unroll
    for (int e = 0; e < N; ++e) s = fmaf(fx[e], fy[e], s);
  }
  return s;
}
template <typename T>
__device__ __forceinline__ void load4(float (&x)[4], const T* p) {
  if constexpr (sizeof(T) == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
  }
}
// acc += the sum over the lanes i of `which` of their f times row i (`step` elements apart).  Every load is made,
// of a row and a piece that exist, so that four are on their way at a time.
template <typename T>
__device__ __forceinline__ void add_rows(float (&acc)[4], float f, uint32_t which, const T* rows, int64_t step, int d) {
  if (which == 0) return;
  const int lane = threadIdx.x & 31, some = __ffs(which) - 1;
  rows += min(4 * lane, d - 4);
  for (int i0 = 0; i0 < 32; i0 += 4) {
    if ((which >> i0 & 15u) == 0) continue;
    float x[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) load4(x[i], rows + ((which >> (i0 + i) & 1u) != 0 ? i0 + i : some) * step);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = __shfl_sync(0xffffffffu, f, i0 + i);
      if ((which >> (i0 + i) & 1u) == 0) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(w, x[i][e], acc[e]);
    }
  }
}
__device__ __forceinline__ void all_nan(float (&v)[4]) { v[0] = v[1] = v[2] = v[3] = __int_as_float(0x7fffffff); }
template <typename T>
__device__ __forceinline__ void row_store(T* p, const float (&v)[4], float f, int d) {
  const int at = 4 * (threadIdx.x & 31);
  if (at >= d) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) p[at + e] = from_f32<T>(v[e] * f);
}

template <typename T>
__device__ __noinline__ void fwd_row(const Call& c, int b, int hk, int g, int s) {
  const int2 sees = c.mask.rows[static_cast<int64_t>(b) * c.S + s];
  const int64_t kv = k_row(c, b, hk, 0) * c.D;
  const T *q = static_cast<const T*>(c.q) + q_row(c, b, hk, g, s) * c.D, *k = static_cast<const T*>(c.k) + kv, *v = static_cast<const T*>(c.v) + kv;
  const float slope2 = c.slopes ? c.slopes[hk * c.G + g] * kLog2e : 0.0f;
  float m = kNoScore, l = 0.0f, acc[4] = {};
  for (int j0 = sees.x; j0 < sees.y; j0 += 32) {
    const int j = j0 + (threadIdx.x & 31);
    const bool in = j < sees.y;
    float t = -INFINITY, bent;
    if (in) t = score2(c, lane_dot(q, k + static_cast<int64_t>(j) * c.D, c.D), slope2, abs(s - j), bent);
    const float top = fmaxf(m, warp_max(t));   // (a NaN score leaves the maximum and makes the sums NaN)
    const float old = exp2f(m - top), p = in ? exp2f(t - top) : 0.0f;
    l = fmaf(l, old, warp_sum(p));
    if (l != l) break;   // (the same on all lanes) every element is NaN
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= old;
    add_rows(acc, p, __ballot_sync(0xffffffffu, in), v + static_cast<int64_t>(j0) * c.D, c.D, c.D);
    m = top;
  }
  const bool none = l == 0.0f;
  const float inv = none ? 0.0f : 1.0f / l;
  if (none) acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
  row_store(static_cast<T*>(c.o) + o_at(c, b, hk, g, s), acc, inv, c.D);
  if (c.lse != nullptr && (threadIdx.x & 31) == 0) c.lse[q_row(c, b, hk, g, s)] = none ? -INFINITY : (m + log2f(l)) * kLn2;
}

// P of a pair from the log-sum-exp (base 2) of the query's row, and t = 1 - tanh^2
__device__ __forceinline__ float pair_p(const Call& c, float dot, float slope2, int distance, float lse2, float& t) {
  float bent;
  const float p = exp2f(score2(c, dot, slope2, distance, bent) - lse2);
  t = 1.0f - bent * bent;
  return p;
}
// and dS, with delta of that row
__device__ __forceinline__ float pair_ds(const Call& c, float dot, float dp, float slope2, int distance, float lse2, float delta, float& p) {
  float t;
  p = pair_p(c, dot, slope2, distance, lse2, t);
  return p * (dp - delta) * t;
}

template <typename T>
__device__ __noinline__ void dq_row(const Call& c, int b, int hk, int g, int s) {
  const int2 sees = c.mask.rows[static_cast<int64_t>(b) * c.S + s];
  const int64_t qr = q_row(c, b, hk, g, s), kv = k_row(c, b, hk, 0) * c.D;
  const T *q = static_cast<const T*>(c.q) + qr * c.D, *go = static_cast<const T*>(c.dout) + o_at(c, b, hk, g, s);
  const T *k = static_cast<const T*>(c.k) + kv, *v = static_cast<const T*>(c.v) + kv;
  const float slope2 = c.slopes ? c.slopes[hk * c.G + g] * kLog2e : 0.0f, lse2 = c.lse[qr] * kLog2e;
  float acc[4] = {}, delta = 0.0f;
  bool nan = false;
  for (int turn = 0; turn < 2 && !nan && lse2 != -INFINITY; ++turn) {   // delta = sum of P dP first
    float part = 0.0f;
    for (int j0 = sees.x; j0 < sees.y; j0 += 32) {
      const int j = j0 + (threadIdx.x & 31);
      const bool in = j < sees.y;
      float ds = 0.0f;
      if (in) {
        float p;
        const float dp = lane_dot(go, v + static_cast<int64_t>(j) * c.D, c.D);
        ds = pair_ds(c, lane_dot(q, k + static_cast<int64_t>(j) * c.D, c.D), dp, slope2, abs(s - j), lse2, delta, p);
        if (turn == 0) ds = part = fmaf(p, dp, part);
      }
      nan = __any_sync(0xffffffffu, ds != ds);   // delta, or a dS: every element is NaN
      if (nan) break;
      if (turn == 1) add_rows(acc, ds, __ballot_sync(0xffffffffu, in), k + static_cast<int64_t>(j0) * c.D, c.D, c.D);
    }
    delta = warp_sum(part);
  }
  if (nan) all_nan(acc);
  row_store(static_cast<T*>(c.dq) + qr * c.D, acc, c.scale, c.D);
}

// (delta and the log-sum-exp of the queries as the dq kernel has left them)
template <typename T>
__device__ __noinline__ void dkv_row(const Call& c, int b, int hk, int s) {
  const int2 seen = c.mask.keys[static_cast<int64_t>(b) * c.S + s];
  const int64_t kr = k_row(c, b, hk, s) * c.D, pitch = amask::tiles_of(c.S) * amask::kTile, ostep = c.o_tok ? static_cast<int64_t>(c.Hk) * c.G * c.D : c.D;
  const T *k = static_cast<const T*>(c.k) + kr, *v = static_cast<const T*>(c.v) + kr;
  float gk[4] = {}, gv[4] = {};
  // a query whose log-sum-exp is NaN makes every element NaN: sooner seen than from its products
  bool nan = false;
  for (int g = 0; g < c.G && !nan; ++g) {
    const float* of = c.nlse2 + ((static_cast<int64_t>(b) * c.Hk + hk) * c.G + g) * pitch;
    float sum = 0.0f;
#pragma unroll 4
    for (int i = seen.x + (threadIdx.x & 31); i < seen.y; i += 32) {
      const float x = of[i];
      if (x != x) sum = x;
    }
    nan = __any_sync(0xffffffffu, sum != sum);
  }
  for (int g = 0; g < c.G && !nan; ++g) {
    const float slope2 = c.slopes ? c.slopes[hk * c.G + g] * kLog2e : 0.0f;
    const T *q = static_cast<const T*>(c.q) + q_row(c, b, hk, g, 0) * c.D, *go = static_cast<const T*>(c.dout) + o_at(c, b, hk, g, 0);
    const int64_t first = ((static_cast<int64_t>(b) * c.Hk + hk) * c.G + g) * pitch;
    for (int i0 = seen.x; i0 < seen.y; i0 += 32) {
      const int i = i0 + (threadIdx.x & 31);
      const float lse2 = i < seen.y ? -c.nlse2[first + i] : INFINITY;
      const bool in = lse2 != INFINITY;
      float p = 0.0f, ds = 0.0f;
      if (in)
        ds = pair_ds(c, lane_dot(k, q + static_cast<int64_t>(i) * c.D, c.D), lane_dot(v, go + i * ostep, c.D), slope2, abs(s - i), lse2,
                     -c.ndelta[first + i], p);
      nan = __any_sync(0xffffffffu, p != p);   // every element of both is NaN
      if (nan) break;
      const uint32_t which = __ballot_sync(0xffffffffu, in);
      add_rows(gk, ds, which, q + static_cast<int64_t>(i0) * c.D, c.D, c.D);
      add_rows(gv, p, which, go + i0 * ostep, ostep, c.D);
    }
  }
  if (nan) { all_nan(gk); all_nan(gv); }
  row_store(static_cast<T*>(c.dk) + kr, gk, c.scale, c.D);
  row_store(static_cast<T*>(c.dv) + kr, gv, 1.0f, c.D);
}

}  // namespace mattn
}  // namespace mcb
