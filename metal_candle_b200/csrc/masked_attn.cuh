// What the kernels of attention under a document / prefix mask share: the call, the score's shape, and one row at a time.
#pragma once
#include "attn_mask.cuh"

namespace mcb {
namespace mattn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Stands for "no score yet" as the running maximum: finite, so that a row that sees nothing has exponentials 2^(-inf - m) = 0
// and not NaN, and below any score that counts.
constexpr float kNoScore = -3e38f;

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
// Head dimensions up to 128: lane l has the elements l, l + 32, l + 64, l + 96.
template <typename T>
struct RowData {
  float v[4];
  __device__ __forceinline__ RowData(const T* p, int d) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = lane + 32 * e < d ? to_f32(p[lane + 32 * e]) : 0.0f;
  }
  __device__ __forceinline__ float dot(const RowData& o) const {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fmaf(v[e], o.v[e], s);
    return warp_sum(s);
  }
};
template <typename T>
__device__ __forceinline__ void row_store(T* p, const float (&v)[4], float f, int d) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 32 * e < d) p[lane + 32 * e] = from_f32<T>(v[e] * f);
}

template <typename T>
__device__ __noinline__ void fwd_row(const Call& c, int b, int hk, int g, int s) {
  const int2 sees = c.mask.rows[static_cast<int64_t>(b) * c.S + s];
  const RowData<T> q(static_cast<const T*>(c.q) + q_row(c, b, hk, g, s) * c.D, c.D);
  const float slope2 = c.slopes ? c.slopes[hk * c.G + g] * kLog2e : 0.0f;
  float m = kNoScore, l = 0.0f, acc[4] = {};
  for (int j = sees.x; j < sees.y; ++j) {
    const int64_t kr = k_row(c, b, hk, j) * c.D;
    const RowData<T> k(static_cast<const T*>(c.k) + kr, c.D), v(static_cast<const T*>(c.v) + kr, c.D);
    float bent;
    const float t = score2(c, q.dot(k), slope2, abs(s - j), bent);
    const float top = t > m ? t : m;   // (a NaN score leaves the maximum and makes the sums NaN)
    const float old = exp2f(m - top), p = exp2f(t - top);
    l = fmaf(l, old, p);
    if (l != l) break;   // (the same on all lanes) every element is NaN
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(p, v.v[e], acc[e] * old);
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
  const int64_t qr = q_row(c, b, hk, g, s), oa = o_at(c, b, hk, g, s);
  const RowData<T> q(static_cast<const T*>(c.q) + qr * c.D, c.D), go(static_cast<const T*>(c.dout) + oa, c.D);
  const float slope2 = c.slopes ? c.slopes[hk * c.G + g] * kLog2e : 0.0f, lse2 = c.lse[qr] * kLog2e;
  float acc[4] = {};
  if (lse2 != -INFINITY) {
    float delta = 0.0f;
    for (int turn = 0; turn < 2; ++turn)   // delta = sum of P dP first
      for (int j = sees.x; j < sees.y; ++j) {
        const int64_t kr = k_row(c, b, hk, j) * c.D;
        const RowData<T> k(static_cast<const T*>(c.k) + kr, c.D), v(static_cast<const T*>(c.v) + kr, c.D);
        float p;
        const float dp = go.dot(v), ds = pair_ds(c, q.dot(k), dp, slope2, abs(s - j), lse2, delta, p);
        if (turn == 0) {
          acc[0] = fmaf(p, dp, acc[0]);
          if (acc[0] == acc[0]) {
            if (j == sees.y - 1) { delta = acc[0]; acc[0] = 0.0f; }
            continue;
          }
        }
        if (turn == 0 || ds != ds) {   // delta, or a dS, is NaN: so is every element
          acc[0] = acc[1] = acc[2] = acc[3] = turn == 0 ? acc[0] : ds;
          turn = 2;
          break;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] = fmaf(ds, k.v[e], acc[e]);
        }
      }
  }
  row_store(static_cast<T*>(c.dq) + qr * c.D, acc, c.scale, c.D);
}

// (delta and the log-sum-exp of the queries as the dq kernel has left them)
template <typename T>
__device__ __noinline__ void dkv_row(const Call& c, int b, int hk, int s) {
  const int2 seen = c.mask.keys[static_cast<int64_t>(b) * c.S + s];
  const int64_t kr = k_row(c, b, hk, s) * c.D, pitch = amask::tiles_of(c.S) * amask::kTile;
  const RowData<T> k(static_cast<const T*>(c.k) + kr, c.D), v(static_cast<const T*>(c.v) + kr, c.D);
  float gk[4] = {}, gv[4] = {};
  for (int g = 0; g < c.G; ++g) {
    const float slope2 = c.slopes ? c.slopes[hk * c.G + g] * kLog2e : 0.0f;
    for (int i = seen.x; i < seen.y; ++i) {
      const int64_t at = ((static_cast<int64_t>(b) * c.Hk + hk) * c.G + g) * pitch + i;
      const float lse2 = -c.nlse2[at];
      if (lse2 == INFINITY) continue;
      const RowData<T> q(static_cast<const T*>(c.q) + q_row(c, b, hk, g, i) * c.D, c.D), go(static_cast<const T*>(c.dout) + o_at(c, b, hk, g, i), c.D);
      float p;
      const float ds = pair_ds(c, q.dot(k), go.dot(v), slope2, abs(s - i), lse2, -c.ndelta[at], p);
      if (p != p) {   // every element of both is NaN
        g = c.G;
        for (int e = 0; e < 4; ++e) gk[e] = gv[e] = p;
        break;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        gk[e] = fmaf(ds, q.v[e], gk[e]);
        gv[e] = fmaf(p, go.v[e], gv[e]);
      }
    }
  }
  row_store(static_cast<T*>(c.dk) + kr, gk, c.scale, c.D);
  row_store(static_cast<T*>(c.dv) + kr, gv, 1.0f, c.D);
}

}  // namespace mattn
}  // namespace mcb
