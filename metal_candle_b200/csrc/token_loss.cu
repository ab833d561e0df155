// Losses over the logits [M, V] of given tokens, with their gradients: token log-probabilities, the preference loss of pairs,
// the clipped policy loss with a KL term, and distillation from a teacher's top logits.
#include <cooperative_groups.h>

#include "token_loss.cuh"

namespace cg = cooperative_groups;

namespace mcb {
namespace {
using namespace tokenloss;

constexpr int kRowThreads = 256;

__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();   // red is free
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.0f;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) t += red[w];
  return t;
}
__device__ __forceinline__ float block_max(float v, float* red) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = red[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 5); ++w) t = fmaxf(t, red[w]);
  return t;
}

// Rows longer than the one-pass kernel takes: one block a row, three sweeps (maximum, sum, gradient).  Any alignment and stride.
template <typename T, int OP>
__global__ void __launch_bounds__(kRowThreads)
token_rows_kernel(const RowArgs a) {
  __shared__ float red[32], red2[32];
  __shared__ int t_id[OP == kDistill ? kMaxTeacher : 1];
  __shared__ float t_q[OP == kDistill ? kMaxTeacher : 1], t_p[OP == kDistill ? kMaxTeacher : 1];
  grid_launch_dependents();
  grid_dependency_wait();
  const int tid = threadIdx.x, nt = blockDim.x;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* x = static_cast<const T*>(from_here(a.logits)) + row_offset(a, row);
    T* g = a.grad != nullptr ? static_cast<T*>(a.grad) + row * a.V : nullptr;
    __syncthreads();   // shared memory of the row before is free
    int tgt = -1;
    float left_out = 0.0f;
    bool out;
    if constexpr (OP == kDistill) {
      const float w = a.weight[row];
      out = w == 0.0f;
    } else {
      tgt = read_target(a.targets, a.target_bytes, a.has_ignore, a.ignore, row, a.V);
      out = tgt < 0;
      if (tgt == -2) left_out = NAN;
    }
    if (out) {
      if (tid == 0) write_left_out<OP>(a, row, left_out, nullptr);
      if (g != nullptr)
        for (int c = tid; c < a.V; c += nt) g[c] = from_f32<T>(left_out);
      continue;
    }
    float m = -INFINITY, s = 0.0f;
    for (int c = tid; c < a.V; c += nt)
      if (c != tgt) m = fmaxf(m, to_f32(x[c]));
    m = block_max(m, red);
    const float ref = m == -INFINITY ? 0.0f : m;
    for (int c = tid; c < a.V; c += nt)
      if (c != tgt) s += ex2((to_f32(x[c]) - ref) * a.k);
    s = block_sum(s, red);
    if constexpr (OP != kDistill) {
      const float xt = to_f32(x[tgt]);
      const TargetStats r = target_stats(m, s, xt, a.k);
      const RowResult res = finish_target_row<OP>(a, row_inputs<OP>(a, row), r);
      if (tid == 0) write_target_row<OP>(a, row, r, res, nullptr);
      const float c0 = res.c;
      __syncthreads();   // everyone has read the target's logit, which the gradient may lie over
      if (g != nullptr) {
        const float f = -c0 / r.sum;
        const float top = r.top == -INFINITY ? 0.0f : r.top;
        for (int c = tid; c < a.V; c += nt)
          g[c] = from_f32<T>(c == tgt ? c0 * r.rest : f * ex2((to_f32(x[c]) - top) * a.k));
      }
    } else {
      // teacher: q = softmax(t / T) over its K entries; those with -inf count for nothing, whatever their id
      const float w = a.weight[row];
      const int64_t t0 = row * a.K;
      float tm = -INFINITY, ts = 0.0f;
      for (int i = tid; i < a.K; i += nt) tm = fmaxf(tm, read_teacher(a, t0 + i));
      tm = block_max(tm, red);
      const float tref = tm == -INFINITY ? 0.0f : tm;
      for (int i = tid; i < a.K; i += nt) ts += exp2f((read_teacher(a, t0 + i) - tref) * a.k);
      ts = block_sum(ts, red);
      const bool empty = ts == 0.0f;
      const float inv_ts = 1.0f / ts, log_ts = logf(ts), log_s = logf(s);
      float loss = 0.0f;
      for (int i = tid; i < a.K; i += nt) {
        const float d = (read_teacher(a, t0 + i) - tref) * a.inv_t;   // log q = d - log_ts
        const int64_t id = read_teacher_id(a, t0 + i);
        const float q = empty ? 0.0f : exp2f((read_teacher(a, t0 + i) - tref) * a.k) * inv_ts;
        int own = -1;
        float p = 0.0f;
        if (q != 0.0f) {   // (NaN counts)
          if (id < 0 || id >= a.V) {
            loss = NAN;
          } else {
            own = static_cast<int>(id);
            const float xi = to_f32(x[own]);
            loss += q * ((d - log_ts) - ((xi - ref) * a.inv_t - log_s));
            p = exp2f((xi - ref) * a.k) / s;
          }
        }
        t_id[i] = own; t_q[i] = q; t_p[i] = p;
      }
      loss = block_sum(loss, red2);
      const float T2 = a.temperature * a.temperature;
      if (tid == 0) a.terms[row] = w * T2 * loss;
      if (g != nullptr) {
        const float c0 = empty ? 0.0f : w * a.temperature + (isnan(loss) ? NAN : 0.0f);
        const float f = c0 / s;
        for (int c = tid; c < a.V; c += nt) g[c] = from_f32<T>(empty ? 0.0f : f * ex2((to_f32(x[c]) - ref) * a.k));
        __syncthreads();   // the row's softmax is written before its teacher columns are
        for (int i = tid; i < a.K; i += nt) {
          if (t_id[i] < 0) continue;
          float q = 0.0f;
          bool first = true;
          for (int j = 0; j < a.K; ++j) {   // the same id may come twice: the first of them writes the sum
            if (t_id[j] != t_id[i]) continue;
            if (j < i) { first = false; break; }
            q += t_q[j];
          }
          if (first) g[t_id[i]] = from_f32<T>(c0 * (t_p[i] - q));
        }
      }
    }
  }
}

// Gradients in place (see GradArgs): a block a row.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
token_grad_kernel(const GradArgs ga) {
  __shared__ float red[kRowThreads / 32];
  const RowArgs& a = ga.a;
  grid_launch_dependents();
  grid_dependency_wait();
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* x = static_cast<const T*>(from_here(a.logits)) + row_offset(a, row);
    T* g = static_cast<T*>(a.grad) + row * a.V;
    const int tgt = read_target(a.targets, a.target_bytes, a.has_ignore, a.ignore, row, a.V);
    if (tgt < 0) {
      for (int c = threadIdx.x; c < a.V; c += blockDim.x) g[c] = from_f32<T>(tgt == -2 ? NAN : 0.0f);
      continue;
    }
    const float c0 = ga.coef[row / ga.coef_rows] * a.inv_t, logp = a.logp[row];
    const float at = c0 * -expm1f(logp);
    float from, add;
    if (!row_anchor(logp, a.lse[row], to_f32(x[tgt]), from, add)) {   // the same in every thread
      float m = -INFINITY, s = 0.0f;
      for (int c = threadIdx.x; c < a.V; c += blockDim.x) m = fmaxf(m, to_f32(x[c]));
      from = block_max(m, red);
      for (int c = threadIdx.x; c < a.V; c += blockDim.x) s += ex2((to_f32(x[c]) - from) * a.k);
      add = -log2f(block_sum(s, red));
    }
    __syncthreads();   // everyone has read what the gradient may lie over
    for (int c = threadIdx.x; c < a.V; c += blockDim.x)
      g[c] = from_f32<T>(c == tgt ? at : -c0 * ex2(fmaf(to_f32(x[c]) - from, a.k, add)));
  }
}

// The weight of each row in the mean: 1 / kept rows, or 1 / (kept rows of its sequence x sequences that keep any).  Kept are the
// rows whose mask is not 0, or whose target is not left out; a target out of range gets NaN.  Neither given: all rows.
// `order`, unless null: the kept rows first, in one fixed order, then the others; and info[0] = how many are kept, info[1] = 0.
// One block, or a cluster of 8 with a part of the rows each: it is the longest chain in front of the losses.  Up to 8192 rows a block the
// targets are read once and stay in registers; up to 2048 sequences are counted as their rows pass, in the first block's memory.
constexpr int kSeqCounts = 2048;
__global__ void __launch_bounds__(1024)
row_weights_kernel(const void* targets, int target_bytes, int has_ignore, int64_t ignore, const uint8_t* mask, float* weight,
                   int32_t* order, int32_t* info, int M, int S, int V, int sequence_mean) {
  __shared__ int red[32];
  __shared__ int2 totals[8];      // each block's (kept, not kept)
  __shared__ int nonempty[8];     // and sequences that keep any
  __shared__ int counts[kSeqCounts];
  constexpr int kRows = 8, kRound = 1024 * kRows;
  cg::cluster_group cl = cg::this_cluster();
  const int n = static_cast<int>(gridDim.x), rank = static_cast<int>(blockIdx.x);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sequences = M / S;
  const bool counted = sequence_mean && sequences <= kSeqCounts;
  auto all_sync = [&]() { if (n > 1) cl.sync(); else __syncthreads(); };
  auto there = [&](auto* p, int r) { return n > 1 ? cl.map_shared_rank(p, r) : p; };
  if (counted)
    for (int b = threadIdx.x; b < sequences; b += 1024) counts[b] = 0;
  all_sync();   // (every block has begun, and its counts are cleared)
  grid_launch_dependents();
  grid_dependency_wait();
  targets = from_here(targets);
  mask = from_here(mask);
  auto kept = [&](int row) {   // 0, 1, or -1 for a target out of range
    if (mask != nullptr) return mask[row] != 0 ? 1 : 0;
    if (targets == nullptr) return 1;
    const int t = read_target(targets, target_bytes, has_ignore, ignore, row, V);
    return t >= 0 ? 1 : t + 1;
  };
  const int64_t per = (static_cast<int64_t>(M) + n - 1) / n, lo = min(static_cast<int64_t>(M), rank * per), hi = min(static_cast<int64_t>(M), lo + per);
  // eight rows a thread at a time; votes: of each warp's 32, kept and not kept
  int keep[kRows], ours, theirs;
  uint32_t votes[kRows], others[kRows];
  auto look = [&](int64_t base) {
    const int64_t mine = base + threadIdx.x;
#pragma unroll
    for (int r = 0; r < kRows; ++r) keep[r] = mine + r * 1024 < hi ? kept(static_cast<int>(mine + r * 1024)) : 0;
    ours = theirs = 0;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      votes[r] = __ballot_sync(0xffffffffu, keep[r] != 0);
      others[r] = __ballot_sync(0xffffffffu, mine + r * 1024 < hi && keep[r] == 0);
      ours += __popc(votes[r]);
      theirs += __popc(others[r]);
    }
  };
  auto block_total = [&](int v) {   // of a value each warp's lanes share
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, red[lane]);
  };
  int warp_ours = 0, warp_theirs = 0;
  for (int64_t base = lo; base < hi; base += kRound) {
    look(base);
    warp_ours += ours;
    warp_theirs += theirs;
    if (!counted) continue;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (votes[r] == 0) continue;
      const int64_t row0 = base + warp * 32 + r * 1024;
      const int b0 = static_cast<int>(row0) / S;
      if (row0 + 31 < static_cast<int64_t>(b0 + 1) * S) {   // all 32 rows of one sequence
        if (lane == 0) atomicAdd(there(counts, 0) + b0, __popc(votes[r]));
      } else if (keep[r] != 0) {
        atomicAdd(there(counts, 0) + static_cast<int>(row0 + lane) / S, 1);
      }
    }
  }
  const int block_ours = block_total(warp_ours), block_theirs = block_total(warp_theirs);
  int block_sequences = 0;
  if (sequence_mean && !counted) {
    for (int64_t b = rank * 32 + warp; b < sequences; b += n * 32) {
      int c = 0;
      for (int i = lane; i < S; i += 32) c += kept(static_cast<int>(b * S) + i) != 0;
      block_sequences += __reduce_add_sync(0xffffffffu, c) > 0;
    }
    block_sequences = block_total(block_sequences);
  }
  if (static_cast<int>(threadIdx.x) < n) {
    there(totals, threadIdx.x)[rank] = make_int2(block_ours, block_theirs);
    there(nonempty, threadIdx.x)[rank] = block_sequences;
  }
  all_sync();
  int total = 0, at0 = 0, out0 = 0, with_any = 0;
  for (int r = 0; r < n; ++r) {
    total += totals[r].x;
    with_any += nonempty[r];
    if (r < rank) { at0 += totals[r].x; out0 += totals[r].y; }
  }
  if (counted) {
    int c = 0;
    for (int b = threadIdx.x; b < sequences; b += 1024) c += there(counts, 0)[b] > 0;
    with_any = block_total(__reduce_add_sync(0xffffffffu, c));
  }
  const float share = 1.0f / static_cast<float>(max(1, sequence_mean ? with_any : total));
  if (rank == 0 && threadIdx.x == 0 && info != nullptr) { info[0] = total; info[1] = 0; }
  for (int64_t base = lo; base < hi; base += kRound) {
    if (hi - lo > kRound) look(base);   // (else it has been looked at)
    __syncthreads();
    if (lane == 0) red[warp] = ours + (theirs << 16);   // (a round has 8192 of both)
    __syncthreads();
    const int c = red[lane];
    const int before = __reduce_add_sync(0xffffffffu, lane < warp ? c : 0), sum = __reduce_add_sync(0xffffffffu, c);
    int at = at0 + (before & 0xffff), out = out0 + (before >> 16);   // places from the order's ends
    at0 += sum & 0xffff;
    out0 += sum >> 16;
    const uint32_t below = (1u << lane) - 1u;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int64_t row = base + threadIdx.x + r * 1024;
      if (row < hi) {
        if (order != nullptr)
          order[keep[r] != 0 ? at + __popc(votes[r] & below) : M - 1 - (out + __popc(others[r] & below))] = static_cast<int32_t>(row);
        if (!sequence_mean || counted)
          weight[row] = keep[r] == 0 ? 0.0f : keep[r] < 0 ? NAN : counted ? share / static_cast<float>(there(counts, 0)[static_cast<int>(row) / S]) : share;
      }
      at += __popc(votes[r]);
      out += __popc(others[r]);
    }
  }
  if (sequence_mean && !counted) {
    for (int64_t b = rank * 32 + warp; b < sequences; b += n * 32) {
      int c = 0;
      for (int i = lane; i < S; i += 32) c += kept(static_cast<int>(b * S) + i) != 0;
      c = __reduce_add_sync(0xffffffffu, c);
      for (int i = lane; i < S; i += 32) {
        const int k = kept(static_cast<int>(b * S) + i);
        weight[b * S + i] = k == 0 ? 0.0f : k < 0 ? NAN : share / static_cast<float>(c);
      }
    }
  }
  if (n > 1) cl.sync();   // no peer still reads here
}

// out[i] = sum of terms[i][0 .. M), i < n <= 8, in one order: a cluster of 8 blocks with a part each, eight loads in flight a thread.
__global__ void __launch_bounds__(1024) __cluster_dims__(8, 1, 1)
sum_terms_kernel(const float* terms, int64_t M, int n, float* out) {
  __shared__ double warp_sums[32];
  __shared__ double parts[8][8];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = static_cast<int>(blockIdx.x), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  cl.sync();   // every block has begun
  grid_launch_dependents();
  grid_dependency_wait();
  terms = from_here(terms);
  const int64_t per = (M + 7) / 8, lo = min(M, rank * per), hi = min(M, lo + per);
  for (int t = 0; t < n; ++t) {
    double acc = 0.0;
    for (int64_t i = lo + threadIdx.x; i < hi; i += 8 * 1024) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = i + j * 1024 < hi ? __ldcg(terms + t * M + i + j * 1024) : 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc += static_cast<double>(v[j]);
    }
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    __syncthreads();   // warp_sums is free
    if (lane == 0) warp_sums[warp] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
      double total = 0.0;
      for (int w = 0; w < 32; ++w) total += warp_sums[w];
      *cl.map_shared_rank(&parts[t][rank], 0) = total;
    }
  }
  cl.sync();
  if (rank == 0 && static_cast<int>(threadIdx.x) < n) {
    double total = 0.0;
    for (int r = 0; r < 8; ++r) total += parts[threadIdx.x][r];
    out[threadIdx.x] = static_cast<float>(total);
  }
}

// The preference loss of pairs (sequence i chosen, pairs + i rejected) from the tokens' log-probabilities:
// L_s = sum (or mean) of a sequence's kept tokens, z = beta ((L_c - ref_c) - (L_r - ref_r)),
// loss = mean of (1 - eps) softplus(-z) + eps softplus(z), and coef[s] = d loss / d logp of every token of sequence s.
__global__ void __launch_bounds__(1024)
preference_kernel(const float* logp, const void* targets, int target_bytes, int has_ignore, int64_t ignore, const float* ref, float* seq_logp,
                  float* coef, float* loss, int64_t pairs, int64_t S, int V, float beta, float eps, int average) {
  __shared__ double red[32];
  grid_launch_dependents();
  grid_dependency_wait();
  logp = from_here(logp);
  targets = from_here(targets);
  ref = from_here(ref);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // a sequence's sum and the share of each of its tokens in it
  auto sequence = [&](int64_t b, double& total, float& per) {
    double acc = 0.0;
    int c = 0;
    for (int64_t i = lane; i < S; i += 8 * 32) {   // eight loads in flight
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = logp[b * S + min(i + 32 * j, S - 1)];
      if (average) {
        int t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = read_target(targets, target_bytes, has_ignore, ignore, b * S + min(i + 32 * j, S - 1), V);
#pragma unroll
        for (int j = 0; j < 8; ++j) c += i + 32 * j < S && t[j] != -1;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc += i + 32 * j < S ? static_cast<double>(v[j]) : 0.0;
      }
    }
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    c = __reduce_add_sync(0xffffffffu, c);
    per = average ? 1.0f / static_cast<float>(max(1, c)) : 1.0f;
    total = average ? acc / static_cast<double>(max(1, c)) : acc;
  };
  double acc = 0.0;
  for (int64_t i = warp; i < pairs; i += 32) {   // a warp a pair
    double won, lost;
    float per_won, per_lost;
    sequence(i, won, per_won);
    sequence(pairs + i, lost, per_lost);
    if (lane != 0) continue;
    // sums of some thousand nats whose difference is a few: not rounded before it is taken
    const float z = static_cast<float>(static_cast<double>(beta) * ((won - ref[i]) - (lost - ref[pairs + i])));
    const float tail = log1pf(expf(-fabsf(z)));
    // (labels that are not smoothed: 0 times the infinite loss of the label that is not there is nothing)
    acc += static_cast<double>((1.0f - eps) * (fmaxf(-z, 0.0f) + tail) + (eps > 0.0f ? eps * (fmaxf(z, 0.0f) + tail) : 0.0f));
    const float d = (eps - 1.0f / (1.0f + expf(z))) * beta / static_cast<float>(pairs);
    seq_logp[i] = static_cast<float>(won);
    seq_logp[pairs + i] = static_cast<float>(lost);
    coef[i] = per_won * d;
    coef[pairs + i] = per_lost * -d;
  }
  if (lane == 0) red[warp] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < 32; ++w) t += red[w];
    *loss = static_cast<float>(t / static_cast<double>(pairs));
  }
}

// x[row, :] *= coef[row / group], in place
template <typename T>
__global__ void __launch_bounds__(256) scale_rows_kernel(T* x, const float* coef, int64_t rows, int64_t D, int64_t group) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int64_t n = rows * D;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
    x[i] = from_f32<T>(to_f32(x[i]) * coef[i / D / group]);
}

// ---- launches ------------------------------------------------------------------------------------------------------------

int launch_sum(const float* terms, int64_t M, int n, float* out, cudaStream_t st);

constexpr int64_t kSumInside = 4096;   // rows whose terms the one-pass kernel's last block sums
template <int OP>
int launch_rows(const RowArgs& a, const RowPlan& plan, int dtype, DeviceState* ds, cudaStream_t st) {
  static_assert(OP != kStats, "launch_stats_rows");
  if (OP == kPolicy && a.grad == nullptr) {
    if (int rc = launch_stats_rows(OP, a, dtype, ds, st)) return rc;
    return plan.sums != nullptr ? launch_sum(a.terms, a.M, plan.n_sums, plan.sums, st) : MCB_OK;
  }
  bool taken = false;
  if (OP != kDistill) {
    RowArgs b = a;
    if (plan.sums != nullptr) b.terms = nullptr;   // summed on the way
    if (int rc = launch_short_rows(OP, b, plan, dtype, ds, st, &taken)) return rc;
    if (taken) return MCB_OK;
  }
  // The sums of many rows by a launch of their own: the last block alone would take 20 us for the three terms of 20000.
  const bool apart = plan.sums != nullptr && a.M > kSumInside;
  RowPlan inside = plan;
  if (apart) inside.sums = nullptr;
  if (int rc = launch_resident_rows(OP, a, inside, dtype, ds, st, &taken)) return rc;
  if (taken) return apart ? launch_sum(a.terms, a.M, plan.n_sums, plan.sums, st) : MCB_OK;
  const int64_t most = static_cast<int64_t>(ds->sm_count) * 8;
  const dim3 grid(static_cast<unsigned>(a.M < most ? a.M : most));
  if (dtype == MCB_F32)
    MCB_CHECK_CUDA(launch_kernel(token_rows_kernel<float, OP>, grid, dim3(kRowThreads), 0, st, chained_launch(), a));
  else
    MCB_CHECK_CUDA(launch_kernel(token_rows_kernel<__nv_bfloat16, OP>, grid, dim3(kRowThreads), 0, st, chained_launch(), a));
  MCB_CHECK_LAUNCH("token_rows");
  return plan.sums != nullptr ? launch_sum(a.terms, a.M, plan.n_sums, plan.sums, st) : MCB_OK;
}

int launch_grad(const GradArgs& ga, int dtype, DeviceState* ds, cudaStream_t st) {
  bool taken = false;
  if (int rc = launch_grad_stream(ga, dtype, ds, st, &taken)) return rc;
  if (taken) return MCB_OK;
  const int64_t most = static_cast<int64_t>(ds->sm_count) * 8;
  const dim3 grid(static_cast<unsigned>(ga.a.M < most ? ga.a.M : most));
  if (dtype == MCB_F32)
    MCB_CHECK_CUDA(launch_kernel(token_grad_kernel<float>, grid, dim3(kRowThreads), 0, st, chained_launch(), ga));
  else
    MCB_CHECK_CUDA(launch_kernel(token_grad_kernel<__nv_bfloat16>, grid, dim3(kRowThreads), 0, st, chained_launch(), ga));
  MCB_CHECK_LAUNCH("token_grad");
  return MCB_OK;
}

int launch_weights(const mcb_token_targets* t, const uint8_t* mask, float* weight, int32_t* order, int32_t* info, int64_t M, int64_t S,
                   int64_t V, int sequence_mean, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  const unsigned blocks = M > 2048 ? 8 : 1;   // (each thread of a block alone would take its second two rows in turn)
  cfg.gridDim = dim3(blocks); cfg.blockDim = dim3(1024); cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = chained_launch() ? 2 : 1;
  MCB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, row_weights_kernel, t ? t->targets : nullptr, t ? t->target_bytes : 0, t ? t->has_ignore : 0,
                                    t ? t->ignore_index : 0, mask, weight, order, info, static_cast<int>(M), static_cast<int>(S),
                                    static_cast<int>(V), sequence_mean));
  MCB_CHECK_LAUNCH("row_weights");
  return MCB_OK;
}

int launch_sum(const float* terms, int64_t M, int n, float* out, cudaStream_t st) {
  MCB_CHECK_CUDA(launch_kernel(sum_terms_kernel, dim3(8), dim3(1024), 0, st, chained_launch(), terms, M, n, out));
  MCB_CHECK_LAUNCH("sum_terms");
  return MCB_OK;
}

// ---- checks of arguments ---------------------------------------------------------------------------------------------------

constexpr int64_t kMaxDim = 0x7fffffff, kMaxVocab = 1 << 30;   // (columns are counted in 32 bits, a block's step past the end included)

// The stride of a dimension of one says nothing: taken as that of dense rows.
int64_t token_stride(const mcb_token_logits* l) { return l->seq == 1 ? l->vocab : l->token_stride; }
int64_t batch_stride(const mcb_token_logits* l) { return l->batch == 1 ? l->seq * l->vocab : l->batch_stride; }

int check_logits(const char* what, const mcb_token_logits* l, const void* grad) {
  if (!l || !l->logits) return fail(MCB_ERR_NULL, "%s: null pointer", what);
  if (l->batch <= 0 || l->seq <= 0 || l->vocab <= 0 || l->vocab > kMaxVocab || l->batch > kMaxDim || l->seq > kMaxDim ||
      l->batch * l->seq > kMaxDim)
    return fail(MCB_ERR_SHAPE, "%s: %lld x %lld rows of %lld logits", what, (long long)l->batch, (long long)l->seq, (long long)l->vocab);
  if (l->batch_stride < 0 || l->token_stride < 0) return fail(MCB_ERR_SHAPE, "%s: negative strides", what);
  if (!(l->temperature > 0.0f) || !(kLog2e / l->temperature <= 3e38f) || !(l->temperature <= 3e38f))
    return fail(MCB_ERR_SHAPE, "%s: temperature %g must be positive and finite", what, static_cast<double>(l->temperature));
  if (l->dtype != MCB_F32 && l->dtype != MCB_BF16) return fail(MCB_ERR_UNSUPPORTED, "%s: dtype %d", what, l->dtype);
  const uintptr_t size = l->dtype == MCB_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(l->logits) % size != 0 || reinterpret_cast<uintptr_t>(grad) % size != 0)
    return fail(MCB_ERR_ALIGN, "%s: logits and gradient must lie on whole elements", what);
  if (grad == l->logits && (token_stride(l) != l->vocab || batch_stride(l) != l->seq * l->vocab))
    return fail(MCB_ERR_SHAPE, "%s: a gradient in place needs dense logits", what);
  if (grad && grad != l->logits) {   // (elements in 128 bits: strides may be anything)
    const __int128 from = reinterpret_cast<uintptr_t>(l->logits), g = reinterpret_cast<uintptr_t>(grad);
    const __int128 n = static_cast<__int128>(l->batch - 1) * l->batch_stride + static_cast<__int128>(l->seq - 1) * l->token_stride + l->vocab;
    if (from < g + static_cast<__int128>(l->batch * l->seq) * l->vocab * size && g < from + n * size)
      return fail(MCB_ERR_SHAPE, "%s: the gradient overlaps the logits without being in place", what);
  }
  return MCB_OK;
}
int check_targets(const char* what, const mcb_token_targets* t) {
  if (!t || !t->targets) return fail(MCB_ERR_NULL, "%s: null targets", what);
  if (t->target_bytes != 4 && t->target_bytes != 8) return fail(MCB_ERR_UNSUPPORTED, "%s: targets of %d bytes", what, t->target_bytes);
  return MCB_OK;
}
int check_policy(const char* what, const mcb_policy_terms* p) {
  if (!p || !p->advantages) return fail(MCB_ERR_NULL, "%s: null advantages", what);
  if (p->advantage_rows <= 0) return fail(MCB_ERR_SHAPE, "%s: advantage_rows %lld", what, (long long)p->advantage_rows);
  if (!(p->clip_low >= 0.0f) || !(p->clip_high >= 0.0f)) return fail(MCB_ERR_SHAPE, "%s: clip bounds must not be negative", what);
  if (!(p->kl_coef >= 0.0f) || !(p->kl_coef <= 3e38f)) return fail(MCB_ERR_SHAPE, "%s: kl_coef must be finite and not negative", what);
  if (p->kl_coef > 0.0f && !p->ref_logp) return fail(MCB_ERR_NULL, "%s: a KL term needs reference log-probabilities", what);
  return MCB_OK;
}
int check_preference(const char* what, const float* ref_logp, const float* seq_logp, const float* loss, float beta, float label_smoothing) {
  if (!ref_logp || !seq_logp || !loss) return fail(MCB_ERR_NULL, "%s: null pointer", what);
  if (!(beta > 0.0f) || !(beta <= 3e38f)) return fail(MCB_ERR_SHAPE, "%s: beta must be positive and finite", what);
  if (!(label_smoothing >= 0.0f) || !(label_smoothing <= 0.5f)) return fail(MCB_ERR_SHAPE, "%s: label smoothing must be in [0, 0.5]", what);
  return MCB_OK;
}
int check_teacher(const char* what, const mcb_teacher_top* t) {
  if (!t || !t->ids || !t->logits) return fail(MCB_ERR_NULL, "%s: null teacher", what);
  if (t->top <= 0 || t->top > kMaxTeacher) return fail(MCB_ERR_SHAPE, "%s: %lld teacher entries a row (1 to %d)", what, (long long)t->top, kMaxTeacher);
  if (t->id_bytes != 4 && t->id_bytes != 8) return fail(MCB_ERR_UNSUPPORTED, "%s: ids of %d bytes", what, t->id_bytes);
  if (t->dtype != MCB_F32 && t->dtype != MCB_BF16) return fail(MCB_ERR_UNSUPPORTED, "%s: teacher dtype %d", what, t->dtype);
  return MCB_OK;
}

// Workspace of a whole loss: what the blocks leave to be summed; a weight, up to three terms and a place in the order for each row; and
// two counters.
struct LossWorkspace {
  double* partials;
  float* weight;
  float* terms;
  int32_t* order;
  int32_t* info;
  LossWorkspace(void* base, int64_t M)
      : partials(static_cast<double*>(base)), weight(reinterpret_cast<float*>(partials + 3 * kMaxPartials)), terms(weight + M), order(reinterpret_cast<int32_t*>(terms + 3 * M)), info(order + M) {}
  RowPlan plan(float* sums, int n) const { return {order, info, sums, n, info + 1, partials}; }
};

RowArgs row_args(const mcb_token_logits* l, void* grad) {
  RowArgs a = {};
  a.logits = l->logits; a.grad = grad;
  a.M = l->batch * l->seq; a.S = l->seq; a.batch_stride = batch_stride(l); a.token_stride = token_stride(l);
  a.V = static_cast<int>(l->vocab);
  a.temperature = l->temperature; a.inv_t = 1.0f / l->temperature; a.k = kLog2e / l->temperature;
  return a;
}
void set_targets(RowArgs& a, const mcb_token_targets* t) {
  a.targets = t->targets; a.target_bytes = t->target_bytes; a.has_ignore = t->has_ignore; a.ignore = t->ignore_index;
}
void set_policy(RowArgs& a, const mcb_policy_terms* p, const float* weight, float* logp, float* terms) {
  a.weight = weight;
  a.advantages = p->advantages; a.advantage_rows = p->advantage_rows < kMaxDim ? p->advantage_rows : kMaxDim; a.old_logp = p->old_logp; a.ref_logp = p->ref_logp;
  a.ratio_min = 1.0f - p->clip_low; a.ratio_max = 1.0f + p->clip_high; a.kl_coef = p->kl_coef;
  a.logp = logp; a.terms = terms;
}
void set_teacher(RowArgs& a, const mcb_teacher_top* t, const float* weight, float* terms) {
  a.weight = weight;
  a.teacher_ids = t->ids; a.teacher = t->logits; a.id_bytes = t->id_bytes; a.teacher_f32 = t->dtype == MCB_F32; a.K = static_cast<int>(t->top);
  a.terms = terms;
}

}  // namespace
}  // namespace mcb

using namespace mcb;
using namespace mcb::tokenloss;

extern "C" int mcb_token_logprob_fwd(const mcb_token_logits* logits, const mcb_token_targets* targets, float* logp, float* lse,
                                     void* unit_grad, void* stream) {
  MCB_NVTX_RANGE("mcb_token_logprob_fwd");
  if (int rc = check_logits("token_logprob_fwd", logits, unit_grad)) return rc;
  if (int rc = check_targets("token_logprob_fwd", targets)) return rc;
  if (!logp) return fail(MCB_ERR_NULL, "token_logprob_fwd: null output");
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  RowArgs a = row_args(logits, unit_grad);
  set_targets(a, targets);
  a.logp = logp; a.lse = lse;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return unit_grad ? launch_rows<kUnit>(a, {}, logits->dtype, ds, st) : launch_stats_rows(kStats, a, logits->dtype, ds, st);
}

extern "C" int mcb_token_logprob_bwd(const mcb_token_logits* logits, const mcb_token_targets* targets, const float* logp, const float* lse,
                                     const float* dlogp, int64_t dlogp_rows, void* dlogits, void* stream) {
  MCB_NVTX_RANGE("mcb_token_logprob_bwd");
  if (!dlogits) return fail(MCB_ERR_NULL, "token_logprob_bwd: null output");
  if (!logp || !lse || !dlogp) return fail(MCB_ERR_NULL, "token_logprob_bwd: null pointer");
  if (int rc = check_logits("token_logprob_bwd", logits, dlogits)) return rc;
  if (int rc = check_targets("token_logprob_bwd", targets)) return rc;
  if (dlogp_rows <= 0) return fail(MCB_ERR_SHAPE, "token_logprob_bwd: dlogp_rows %lld", (long long)dlogp_rows);
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  GradArgs ga;
  ga.a = row_args(logits, dlogits);
  set_targets(ga.a, targets);
  ga.a.logp = const_cast<float*>(logp); ga.a.lse = const_cast<float*>(lse);
  ga.coef = dlogp; ga.coef_rows = dlogp_rows < kMaxDim ? dlogp_rows : kMaxDim;
  return launch_grad(ga, logits->dtype, ds, static_cast<cudaStream_t>(stream));
}

extern "C" int mcb_loss_weights(const mcb_token_targets* targets, const uint8_t* mask, float* weight, int64_t batch, int64_t seq, int64_t vocab,
                                int sequence_mean, void* stream) {
  MCB_NVTX_RANGE("mcb_loss_weights");
  if (!weight) return fail(MCB_ERR_NULL, "loss_weights: null output");
  if (targets)
    if (int rc = check_targets("loss_weights", targets)) return rc;
  if (batch <= 0 || seq <= 0 || vocab <= 0 || vocab > kMaxDim || batch > kMaxDim || seq > kMaxDim || batch * seq > kMaxDim)
    return fail(MCB_ERR_SHAPE, "loss_weights: bad shape");
  if (!current_device_state()) return MCB_ERR_NOT_INIT;
  return launch_weights(targets, mask, weight, nullptr, nullptr, batch * seq, seq, vocab, sequence_mean, static_cast<cudaStream_t>(stream));
}

extern "C" int mcb_loss_sums(const float* terms, int64_t rows, int n, float* out, void* stream) {
  MCB_NVTX_RANGE("mcb_loss_sums");
  if (!terms || !out) return fail(MCB_ERR_NULL, "loss_sums: null pointer");
  if (rows <= 0 || rows > kMaxDim || n <= 0 || n > 8) return fail(MCB_ERR_SHAPE, "loss_sums: bad shape");
  if (!current_device_state()) return MCB_ERR_NOT_INIT;
  return launch_sum(terms, rows, n, out, static_cast<cudaStream_t>(stream));
}

extern "C" int mcb_policy_loss_rows(const mcb_token_logits* logits, const mcb_token_targets* targets, const mcb_policy_terms* policy,
                                    const float* weight, float* logp, float* terms, void* dlogits, void* stream) {
  MCB_NVTX_RANGE("mcb_policy_loss_rows");
  if (int rc = check_logits("policy_loss_rows", logits, dlogits)) return rc;
  if (int rc = check_targets("policy_loss_rows", targets)) return rc;
  if (int rc = check_policy("policy_loss_rows", policy)) return rc;
  if (!weight || !logp || !terms) return fail(MCB_ERR_NULL, "policy_loss_rows: null pointer");
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  RowArgs a = row_args(logits, dlogits);
  set_targets(a, targets);
  set_policy(a, policy, weight, logp, terms);
  return launch_rows<kPolicy>(a, {}, logits->dtype, ds, static_cast<cudaStream_t>(stream));
}

extern "C" int mcb_distill_loss_rows(const mcb_token_logits* logits, const mcb_teacher_top* teacher, const float* weight, float* terms,
                                     void* dlogits, void* stream) {
  MCB_NVTX_RANGE("mcb_distill_loss_rows");
  if (int rc = check_logits("distill_loss_rows", logits, dlogits)) return rc;
  if (int rc = check_teacher("distill_loss_rows", teacher)) return rc;
  if (!weight || !terms) return fail(MCB_ERR_NULL, "distill_loss_rows: null pointer");
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  RowArgs a = row_args(logits, dlogits);
  set_teacher(a, teacher, weight, terms);
  return launch_rows<kDistill>(a, {}, logits->dtype, ds, static_cast<cudaStream_t>(stream));
}

extern "C" size_t mcb_token_loss_workspace_bytes(int64_t batch, int64_t seq) {
  if (batch <= 0 || seq <= 0 || batch > kMaxDim || seq > kMaxDim || batch * seq > kMaxDim) return 0;
  return (static_cast<size_t>(batch * seq) * 5 + static_cast<size_t>(batch) + 64) * sizeof(float) + 3 * kMaxPartials * sizeof(double);
}

extern "C" int mcb_policy_loss(const mcb_token_logits* logits, const mcb_token_targets* targets, const mcb_policy_terms* policy, int sequence_mean,
                               float* logp, float* out, void* dlogits, void* workspace, size_t workspace_bytes, void* stream) {
  MCB_NVTX_RANGE("mcb_policy_loss");
  if (int rc = check_logits("policy_loss", logits, dlogits)) return rc;
  if (int rc = check_targets("policy_loss", targets)) return rc;
  if (int rc = check_policy("policy_loss", policy)) return rc;
  if (!logp || !out) return fail(MCB_ERR_NULL, "policy_loss: null output");
  if (!workspace || workspace_bytes < mcb_token_loss_workspace_bytes(logits->batch, logits->seq))
    return fail(MCB_ERR_WORKSPACE, "policy_loss: workspace missing or too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(MCB_ERR_ALIGN, "policy_loss: the workspace must lie on a 16-byte boundary");
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t M = logits->batch * logits->seq;
  const LossWorkspace ws(workspace, M);
  if (int rc = launch_weights(targets, nullptr, ws.weight, ws.order, ws.info, M, logits->seq, logits->vocab, sequence_mean, st)) return rc;
  RowArgs a = row_args(logits, dlogits);
  set_targets(a, targets);
  set_policy(a, policy, ws.weight, logp, ws.terms);
  return launch_rows<kPolicy>(a, ws.plan(out, 3), logits->dtype, ds, st);
}

extern "C" int mcb_distill_loss(const mcb_token_logits* logits, const mcb_teacher_top* teacher, const uint8_t* mask, float* loss, void* dlogits,
                                void* workspace, size_t workspace_bytes, void* stream) {
  MCB_NVTX_RANGE("mcb_distill_loss");
  if (int rc = check_logits("distill_loss", logits, dlogits)) return rc;
  if (int rc = check_teacher("distill_loss", teacher)) return rc;
  if (!loss) return fail(MCB_ERR_NULL, "distill_loss: null output");
  if (!workspace || workspace_bytes < mcb_token_loss_workspace_bytes(logits->batch, logits->seq))
    return fail(MCB_ERR_WORKSPACE, "distill_loss: workspace missing or too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(MCB_ERR_ALIGN, "distill_loss: the workspace must lie on a 16-byte boundary");
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t M = logits->batch * logits->seq;
  const LossWorkspace ws(workspace, M);
  if (int rc = launch_weights(nullptr, mask, ws.weight, ws.order, ws.info, M, logits->seq, logits->vocab, 0, st)) return rc;
  RowArgs a = row_args(logits, dlogits);
  set_teacher(a, teacher, ws.weight, ws.terms);
  return launch_rows<kDistill>(a, ws.plan(loss, 1), logits->dtype, ds, st);
}

extern "C" int mcb_preference_finish(const float* logp, const mcb_token_targets* targets, const float* ref_logp, float* seq_logp, float* coef,
                                     float* loss, int64_t pairs, int64_t seq, int64_t vocab, float beta, float label_smoothing, int average,
                                     void* stream) {
  MCB_NVTX_RANGE("mcb_preference_finish");
  if (int rc = check_targets("preference_finish", targets)) return rc;
  if (!logp || !coef) return fail(MCB_ERR_NULL, "preference_finish: null pointer");
  if (int rc = check_preference("preference_finish", ref_logp, seq_logp, loss, beta, label_smoothing)) return rc;
  if (pairs <= 0 || seq <= 0 || vocab <= 0 || vocab > kMaxDim || pairs > kMaxDim || seq > kMaxDim || 2 * pairs * seq > kMaxDim)
    return fail(MCB_ERR_SHAPE, "preference_finish: bad shape");
  if (!current_device_state()) return MCB_ERR_NOT_INIT;
  MCB_CHECK_CUDA(launch_kernel(preference_kernel, dim3(1), dim3(1024), 0, static_cast<cudaStream_t>(stream), chained_launch(), logp,
                               targets->targets, targets->target_bytes, targets->has_ignore, targets->ignore_index, ref_logp, seq_logp, coef, loss, pairs, seq,
                               static_cast<int>(vocab), beta, label_smoothing, average));
  MCB_CHECK_LAUNCH("preference");
  return MCB_OK;
}

extern "C" int mcb_preference_loss(const mcb_token_logits* logits, const mcb_token_targets* targets, const float* ref_logp, float beta,
                                   float label_smoothing, int average, float* seq_logp, float* loss, void* dlogits, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  MCB_NVTX_RANGE("mcb_preference_loss");
  if (int rc = check_logits("preference_loss", logits, dlogits)) return rc;
  if (int rc = check_targets("preference_loss", targets)) return rc;
  if (int rc = check_preference("preference_loss", ref_logp, seq_logp, loss, beta, label_smoothing)) return rc;
  if (logits->batch % 2 != 0) return fail(MCB_ERR_SHAPE, "preference_loss: %lld sequences are no pairs", (long long)logits->batch);
  if (!workspace || workspace_bytes < mcb_token_loss_workspace_bytes(logits->batch, logits->seq))
    return fail(MCB_ERR_WORKSPACE, "preference_loss: workspace missing or too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(MCB_ERR_ALIGN, "preference_loss: the workspace must lie on a 16-byte boundary");
  const int64_t M = logits->batch * logits->seq;
  float* logp = static_cast<float*>(workspace);
  float* lse = logp + M;
  float* coef = lse + M;
  if (int rc = mcb_token_logprob_fwd(logits, targets, logp, lse, nullptr, stream)) return rc;
  if (int rc = mcb_preference_finish(logp, targets, ref_logp, seq_logp, coef, loss, logits->batch / 2, logits->seq, logits->vocab, beta,
                                     label_smoothing, average, stream))
    return rc;
  return dlogits ? mcb_token_logprob_bwd(logits, targets, logp, lse, coef, logits->seq, dlogits, stream) : MCB_OK;
}

extern "C" int mcb_scale_rows(void* x, const float* coef, int64_t rows, int64_t D, int64_t coef_rows, int dtype, void* stream) {
  MCB_NVTX_RANGE("mcb_scale_rows");
  if (!x || !coef) return fail(MCB_ERR_NULL, "scale_rows: null pointer");
  if (rows <= 0 || D <= 0 || coef_rows <= 0 || rows > kMaxDim || D > kMaxDim) return fail(MCB_ERR_SHAPE, "scale_rows: bad shape");
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  const int64_t blocks = (rows * D + 255) / 256, most = static_cast<int64_t>(ds->sm_count) * 16;
  const dim3 grid(static_cast<unsigned>(blocks < most ? blocks : most));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == MCB_F32)
    MCB_CHECK_CUDA(launch_kernel(scale_rows_kernel<float>, grid, dim3(256), 0, st, chained_launch(), static_cast<float*>(x), coef, rows, D, coef_rows));
  else if (dtype == MCB_BF16)
    MCB_CHECK_CUDA(launch_kernel(scale_rows_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, chained_launch(), static_cast<__nv_bfloat16*>(x), coef, rows, D, coef_rows));
  else
    return fail(MCB_ERR_UNSUPPORTED, "scale_rows: dtype %d", dtype);
  MCB_CHECK_LAUNCH("scale_rows");
  return MCB_OK;
}
