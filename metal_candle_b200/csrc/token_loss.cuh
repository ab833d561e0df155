// What the losses over the logits of given tokens share: the arguments of a row, the arithmetic of its softmax, and what each
// loss makes of a row's log-probability.
//
// A row x [V] at temperature T has y = x / T, p_j = exp(y_j) / sum exp(y).  Exponentials are taken in base 2 of differences,
// 2^((x_j - m) k) with k = log2(e) / T: exact for x_j = m whatever its magnitude, and 0 for masked logits (-inf, or the type's
// lowest value, whose difference may overflow to -inf).  The target is kept out of the sum: with m, s over the other columns,
// p_t / (1 - p_t) = 2^((x_t - m) k) / s, so that neither log p_t near 0 nor 1 - p_t, the gradient's factor, is a difference of
// nearly equal numbers.
#pragma once

#include "common.cuh"

namespace mcb {
namespace tokenloss {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxTeacher = 1024;   // teacher entries a row

enum Op { kStats = 0, kUnit = 1, kPolicy = 2, kDistill = 3 };

struct RowArgs {
  const void* logits;      // row r starts (r / S) * batch_stride + (r % S) * token_stride elements in
  void* grad;              // [M, V] dense, or null
  int64_t M, S, batch_stride, token_stride;
  int V;
  float k, inv_t, temperature;
  // the target of each row (kStats, kUnit, kPolicy); -1 and, with has_ignore, `ignore` leave the row out
  const void* targets;
  int target_bytes, has_ignore;
  int64_t ignore;
  const float* weight;     // kPolicy, kDistill: [M]; 0 leaves the row out, NaN marks a target out of range
  // kPolicy
  const float* advantages; // of row r: advantages[r / advantage_rows]
  int64_t advantage_rows;
  const float* old_logp;   // null: the policy that is being trained
  const float* ref_logp;   // null: no KL term
  float ratio_min, ratio_max, kl_coef;
  // kDistill
  const void* teacher_ids; // [M, K]
  const void* teacher;     // [M, K]
  int id_bytes, teacher_f32, K;
  // what a row leaves behind
  float* logp;             // [M] (kDistill: none)
  float* lse;              // [M], or null
  float* terms;            // kPolicy: [3, M]: loss, KL, clipped; kDistill: [M]; each times the row's weight.  Null: they are summed only
};

__device__ __forceinline__ int64_t row_offset(const RowArgs& a, int64_t row) {   // (rows and S are below 2^31)
  const uint32_t r = static_cast<uint32_t>(row), b = r / static_cast<uint32_t>(a.S);
  return b * a.batch_stride + static_cast<int64_t>(r - b * static_cast<uint32_t>(a.S)) * a.token_stride;
}

// The row's target, -1 where the row is left out, -2 where it is none of the vocabulary; in two steps for a caller that asks ahead.
__device__ __forceinline__ int64_t load_target(const void* targets, int target_bytes, int64_t row) {
  return target_bytes == 8 ? static_cast<const int64_t*>(targets)[row] : static_cast<const int32_t*>(targets)[row];
}
__device__ __forceinline__ int kept_target(int64_t t, int has_ignore, int64_t ignore, int V) {
  if (t == -1 || (has_ignore && t == ignore)) return -1;
  return t >= 0 && t < V ? static_cast<int>(t) : -2;
}
__device__ __forceinline__ int read_target(const void* targets, int target_bytes, int has_ignore, int64_t ignore, int64_t row, int V) {
  return kept_target(load_target(targets, target_bytes, row), has_ignore, ignore, V);
}

// 2^x, denormal results flushed to zero (one instruction, relative error about 2^-22)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// maximum m and sum s of 2^((x - m) k) of two sets of logits; an empty or wholly masked set is (-inf, 0), or (-inf, NaN) if it
// holds nothing but NaN besides
__device__ __forceinline__ void combine(float& m, float& s, float m2, float s2, float k) {
  const float mm = fmaxf(m, m2);
  if (mm == -INFINITY) { s += s2; return; }
  s = s * ex2((m - mm) * k) + s2 * ex2((m2 - mm) * k);
  m = mm;
}

// log(1 + x) for x >= 0, with w = 1 + x as rounded: log w scaled by how far w moved from 1 (W. Kahan's form), exact to a few
// roundings where log w alone would have lost x
__device__ __forceinline__ float log_plus_one(float x, float w) {
  return w == 1.0f ? x : w > 2.0f ? logf(w) : logf(w) * __fdividef(x, w - 1.0f);
}

// A row's softmax around its target: (m, s) are those of the other columns.
struct TargetStats {
  float top, sum;       // of the whole row
  float logp, rest;     // log p_t and 1 - p_t
};
// y_t - y_m of a target so far below that (x_t - m) k is no float32 number, though y_t - y_m itself may be one (m > x_t)
__device__ __forceinline__ float far_below(float xt, float m, float k) {
  const float inv_t = k * kLn2, d = xt - m;
  if (d > -INFINITY) return d * inv_t;
  return m > 0.0f ? xt * inv_t - m * inv_t : d;   // (a difference that overflows has parts of both signs; else x_t is -inf)
}
__device__ __forceinline__ TargetStats target_stats(float m, float s, float xt, float k) {
  TargetStats r;
  if (m == -INFINITY && s == 0.0f) {   // nothing but the target (which, masked itself, has no probability: NaN)
    r.logp = r.rest = xt - xt;
    r.top = xt; r.sum = 1.0f + r.logp;
    return r;
  }
  if (xt == INFINITY) {   // an overflow, NaN as in any other column
    r.top = xt;
    r.logp = r.rest = r.sum = NAN;
    return r;
  }
  const float d = (m - xt) * k;
  if (d <= 0.0f) {
    const float odds = s * ex2(d);
    r.top = xt; r.sum = 1.0f + odds;
    r.logp = -log_plus_one(odds, r.sum);
    r.rest = __fdividef(odds, r.sum);
  } else {   // (NaN as well)
    r.top = m; r.sum = s + ex2(-d);
    r.logp = d < INFINITY ? fmaf(-d, kLn2, -logf(r.sum)) : far_below(xt, m, k) - logf(r.sum);
    r.rest = __fdividef(s, r.sum);
  }
  return r;
}

// The clipped policy term of one token and its derivative towards logp, and what is reported of it.
struct PolicyTerm {
  float loss, dlogp, kl, clipped;
};
// What the loss reads of a row besides its logits, apart so that it can be asked for ahead.
struct RowInputs {
  float weight, advantage, old_logp, ref_logp;
};
template <int OP>
__device__ __forceinline__ RowInputs row_inputs(const RowArgs& a, int64_t row) {
  RowInputs in = {};
  if constexpr (OP == kPolicy || OP == kDistill) in.weight = a.weight[row];
  if constexpr (OP == kPolicy) {
    in.advantage = a.advantages[static_cast<uint32_t>(row) / static_cast<uint32_t>(a.advantage_rows)];
    if (a.old_logp != nullptr) in.old_logp = a.old_logp[row];
    if (a.ref_logp != nullptr) in.ref_logp = a.ref_logp[row];
  }
  return in;
}
__device__ __forceinline__ PolicyTerm policy_term(const RowArgs& a, const RowInputs& in, float logp) {
  const float adv = in.advantage;
  const float ratio = a.old_logp != nullptr ? ex2((logp - in.old_logp) * kLog2e) : isnan(logp) ? logp : 1.0f;
  const float bounded = fminf(fmaxf(ratio, a.ratio_min), a.ratio_max);
  PolicyTerm t;
  // min(r A, clip(r) A): the bound holds only where it makes the term smaller
  const bool bound = adv >= 0.0f ? ratio > a.ratio_max : ratio < a.ratio_min;
  t.loss = -(bound ? bounded : ratio) * adv;
  t.dlogp = bound ? 0.0f : -adv * ratio;
  t.clipped = bound ? 1.0f : 0.0f;
  t.kl = 0.0f;
  if (a.ref_logp != nullptr) {
    // exp(d) - d - 1 >= 0 with d = ref - logp: an estimate of KL(policy || reference) that is never negative
    const float d = in.ref_logp - logp;
    const float e = expm1f(d);
    t.kl = e < INFINITY ? e - d : e;   // (d = inf, a target that the policy forbids: e - d would be NaN)
    if (a.kl_coef > 0.0f) {   // (0 times an infinite divergence is not a loss)
      t.loss += a.kl_coef * t.kl;
      t.dlogp -= a.kl_coef * e;
    }
  }
  return t;
}

// What a row's log-probability comes to: d loss / d logp / T, and the row's terms.
struct RowResult {
  float c, terms[3];
};
template <int OP>
__device__ __forceinline__ RowResult finish_target_row(const RowArgs& a, const RowInputs& in, const TargetStats& r) {
  RowResult out = {a.inv_t, {0.0f, 0.0f, 0.0f}};
  if constexpr (OP == kPolicy) {
    const float w = in.weight;
    const PolicyTerm t = policy_term(a, in, r.logp);
    out.c = w * t.dlogp * a.inv_t;
    out.terms[0] = w * t.loss; out.terms[1] = w * t.kl; out.terms[2] = w * t.clipped;
  }
  return out;
}
// What the row leaves behind, by one thread.  sums: where its terms are added up, or null.
template <int OP>
__device__ __forceinline__ void write_row(const RowArgs& a, int64_t row, float logp, float lse, const float* terms, double* sums) {
  constexpr int n = OP == kPolicy ? 3 : OP == kDistill ? 1 : 0;
  if (OP != kDistill && a.logp != nullptr) a.logp[row] = logp;
  if (OP != kDistill && a.lse != nullptr) a.lse[row] = lse;
#pragma unroll
  for (int t = 0; t < n; ++t) {
    if (a.terms != nullptr) a.terms[t * a.M + row] = terms[t];
    if (sums != nullptr) sums[t] += static_cast<double>(terms[t]);
  }
}
template <int OP>
__device__ __forceinline__ void write_target_row(const RowArgs& a, int64_t row, const TargetStats& r, const RowResult& out, double* sums) {
  write_row<OP>(a, row, r.logp, a.lse != nullptr ? r.top * a.inv_t + logf(r.sum) : 0.0f, out.terms, sums);
}
// A row that is left out (value 0) or whose target is out of range (NaN).
template <int OP>
__device__ __forceinline__ void write_left_out(const RowArgs& a, int64_t row, float value, double* sums) {
  const float terms[3] = {value, value, value};
  write_row<OP>(a, row, value, value, terms, sums);
}

__device__ __forceinline__ float read_teacher(const RowArgs& a, int64_t i) {
  return a.teacher_f32 ? static_cast<const float*>(a.teacher)[i] : to_f32(static_cast<const __nv_bfloat16*>(a.teacher)[i]);
}
__device__ __forceinline__ int64_t read_teacher_id(const RowArgs& a, int64_t i) {
  return a.id_bytes == 8 ? static_cast<const int64_t*>(a.teacher_ids)[i] : static_cast<const int32_t*>(a.teacher_ids)[i];
}

// out[t] = sum over i < count of terms[i * step + t * apart] by one block, in an order that depends on its size alone; eight loads in
// flight a thread.  warp_sums: room for a double a warp.
template <int THREADS = 0, typename V>   // (0: whatever the block has)
__device__ __forceinline__ void block_sums(const V* terms, int64_t count, int64_t step, int64_t apart, int n, float* out, double* warp_sums) {
  const int nt = THREADS > 0 ? THREADS : blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int t = 0; t < n; ++t) {
    double acc = 0.0;
    for (int64_t i = threadIdx.x; i < count; i += 8 * nt) {
      V v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = i + j * nt < count ? __ldcg(terms + t * apart + (i + j * nt) * step) : V(0);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc += static_cast<double>(v[j]);
    }
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    __syncthreads();   // warp_sums is free
    if (lane == 0) warp_sums[warp] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
      double total = 0.0;
      for (int w = 0; w < nt >> 5; ++w) total += warp_sums[w];
      out[t] = static_cast<float>(total);
    }
  }
}

// Rows in the order they are to be taken, the kept ones first (as mcb_loss_weights tells them apart), and where the sums of the rows'
// terms go.  The last block to finish makes them, in one order: of the terms, or (short rows, of which there may be many) of what each
// block has added up over its rows, which are the same from call to call.  All null for a chunk of rows.
constexpr int kMaxPartials = 2048;   // blocks of such a launch, each with 3 doubles
struct RowPlan {
  const int32_t* order;
  const int32_t* kept;
  float* sums;      // n_sums of them
  int n_sums;
  int* done;        // 0 when the kernel starts
  double* partials;
};

// kUnit and kPolicy, rows of at most 256 vectors, each held by a warp (token_stream.cu).
int launch_short_rows(int op, const RowArgs& a, const RowPlan& plan, int dtype, DeviceState* ds, cudaStream_t st, bool* taken);

// The one-pass kernel (token_resident.cu), where it takes rows of this length: *taken says whether it did.
int launch_resident_rows(int op, const RowArgs& a, const RowPlan& plan, int dtype, DeviceState* ds, cudaStream_t st, bool* taken);

// The reverse of token log-probabilities whose softmax is known: dx_j = c (1[j = t] - exp(y_j - lse)), c = dlogp / T, dlogp of row i =
// coef[i / coef_rows]; logp and lse of `a` are read.
struct GradArgs {
  RowArgs a;
  const float* coef;
  int64_t coef_rows;
};

// Where the exponents of such a row are taken from: log2 p_j = (x_j - from) k + add, with add 32 bits of log2 p_t (from the target) or of
// -lse log2(e) (from 0).  Its rounding is an error of p_j relative to p_j, and so is that of x_j k, so the smaller of the two in
// magnitude is taken: log p_t near 0 keeps its digits however large the logits are, and a target far below the rest (a token that a mask
// forbids) costs the other columns none.  Where both are large (logits of some thousand, and a target far below) the kernels take the
// row's maximum and sum again: returns false.  32: an error of 32 x 2^-24 for each of the few roundings, 1e-5.
__device__ __forceinline__ bool row_anchor(float logp, float lse, float xt, float& from, float& add) {
  const bool at_target = !(fabsf(logp) > fabsf(lse));   // (NaN: the row is NaN)
  from = at_target ? xt : 0.0f;
  add = (at_target ? logp : -lse) * kLog2e;
  return !(fminf(fabsf(logp), fabsf(lse)) > 32.0f);
}

// token_stream.cu: kStats, or kPolicy without a gradient; and the gradient, where it is not in place.
int launch_stats_rows(int op, const RowArgs& a, int dtype, DeviceState* ds, cudaStream_t st);
int launch_grad_stream(const GradArgs& ga, int dtype, DeviceState* ds, cudaStream_t st, bool* taken);

}  // namespace tokenloss
}  // namespace mcb
