// Token losses, the two streams over the logits: statistics of each row (read once), and the gradient from statistics that are
// known (read and written once).
#include <cooperative_groups.h>

#include "token_loss.cuh"

namespace cg = cooperative_groups;

namespace mcb {
namespace {
using namespace tokenloss;

constexpr int kThreads = 256, kUnroll = 8;

// A row's vectors: [fa, fb) are the row's alone, counted from the 16-byte boundary in front of the row; its first element is at
// element lo, hi is behind its last.
struct RowVecs {
  int lo, hi, fa, fb;
};
template <typename T>
__device__ __forceinline__ RowVecs vecs_of(const T* x, int V, const T*& base) {
  constexpr int N = Vec16<T>::N;
  RowVecs r;
  r.lo = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  r.hi = r.lo + V;
  base = x - r.lo;
  r.fa = r.lo > 0 ? 1 : 0;
  r.fb = max(r.fa, r.hi / N);
  return r;
}

__device__ __forceinline__ float max_of(const Vec16<__nv_bfloat16> (&v)[kUnroll]) {
  __nv_bfloat162 m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = reinterpret_cast<const __nv_bfloat162*>(&v[0].raw)[i];
#pragma unroll
  for (int j = 1; j < kUnroll; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = __hmax2(m[i], reinterpret_cast<const __nv_bfloat162*>(&v[j].raw)[i]);
  const __nv_bfloat162 r = __hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3]));
  return fmaxf(__low2float(r), __high2float(r));
}
__device__ __forceinline__ float max_of(const Vec16<float> (&v)[kUnroll]) {
  float m = v[0].raw.x;
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) m = fmaxf(m, fmaxf(fmaxf(v[j].raw.x, v[j].raw.y), fmaxf(v[j].raw.z, v[j].raw.w)));
  return m;
}
template <typename T>
__device__ __forceinline__ void fill_masked(Vec16<T>& v) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&v.raw);
  w[0] = w[1] = w[2] = w[3] = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
}

__device__ __forceinline__ void warp_combine(float& m, float& s, float k) {
  const float top = warp_max(m);
  s = warp_sum(m == -INFINITY ? s : s * ex2((m - top) * k));
  m = top;
}

__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Statistics.  Bound: HBM, one read; per thread eight 16-byte loads are in flight, whose maximum is taken first, so that the running
// sum is rescaled once in eight vectors.  A row is one block's, or with few rows a cluster's; SHORT: one warp's (20000 x 1000 bf16 as
// blocks of a warp each 41 us: as many launches of blocks as rows).
template <typename T, int OP, bool SHORT>
__global__ void __launch_bounds__(kThreads)
token_stats_kernel(const RowArgs a, int log_ctas) {
  using VT = Vec16<T>;
  using Raw = decltype(VT::raw);
  constexpr int N = VT::N;
  __shared__ float2 red[kThreads / 32];
  __shared__ float2 parts[8];
  cg::cluster_group cl = cg::this_cluster();
  const int ctas = 1 << log_ctas, rank = static_cast<int>(blockIdx.x) & (ctas - 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = SHORT ? static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + warp : static_cast<int64_t>(blockIdx.x) >> log_ctas;
  const int tid = SHORT ? lane : threadIdx.x, bd = SHORT ? 32 : blockDim.x;   // within the row's threads
  if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // (waited for before a peer's memory is touched)
  grid_launch_dependents();
  grid_dependency_wait();
  const bool real = !SHORT || row < a.M;
  const T* x = static_cast<const T*>(from_here(a.logits)) + row_offset(a, real ? row : 0);
  const int tgt = real ? read_target(from_here(a.targets), a.target_bytes, a.has_ignore, a.ignore, row, a.V) : -1;
  if (!real) {
  } else if (tgt < 0) {   // the same in every CTA of the cluster
    if (rank == 0 && tid == 0) write_left_out<OP>(a, row, tgt == -2 ? NAN : 0.0f, nullptr);
    if (ctas > 1) cluster_wait();
  } else {
    const T* base;
    const RowVecs r = vecs_of(x, a.V, base);
    const Raw* src = reinterpret_cast<const Raw*>(base);
    const int tv = (r.lo + tgt) / N;
    const int per = (r.fb - r.fa + ctas - 1) >> log_ctas;
    const int begin = r.fa + rank * per, end = min(r.fb, begin + per);
    const float2 kk = make_float2(a.k, a.k);
    const RowInputs inputs = row_inputs<OP>(a, row);
    float m = -INFINITY, s = 0.0f;
    for (int v0 = begin + tid; v0 < end; v0 += kUnroll * bd) {
      VT v[kUnroll];
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) {
        if (v0 + j * bd < end) v[j].raw = __ldg(src + v0 + j * bd);
        else fill_masked(v[j]);
      }
      const int at = tv - v0;
      if (at >= 0 && at < kUnroll * bd && at % bd == 0) {   // the target is not summed
        const int q = (r.lo + tgt) % N;
#pragma unroll
        for (int j = 0; j < kUnroll; ++j)
          if (at == j * bd) {
            float f[N];
            v[j].to_float(f);
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = i == q ? -INFINITY : f[i];
            v[j].from_float(f);
          }
      }
      const float mm = fmaxf(m, max_of(v));
      if (mm > m && m != -INFINITY) s *= ex2((m - mm) * a.k);
      m = mm;
      const float ref = m == -INFINITY ? 0.0f : m;
      const float2 neg = make_float2(-ref, -ref);
      float2 s2 = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) {
        float f[N];
        v[j].to_float(f);
#pragma unroll
        for (int q = 0; q < N; q += 2) {
          const float2 d = __fmul2_rn(__fadd2_rn(make_float2(f[q], f[q + 1]), neg), kk);
          s2 = __fadd2_rn(s2, make_float2(ex2(d.x), ex2(d.y)));
        }
      }
      s += s2.x + s2.y;
    }
    if (rank == 0 && tid < 2 * N) {   // the row's elements in vectors that it shares with its neighbours
      const int e = tid < N ? r.lo + tid : r.fb * N + tid - N;
      if ((tid < N ? e < min(r.fa * N, r.hi) : e < r.hi) && e - r.lo != tgt) {
        const float v = to_f32(base[e]);
        if (isnan(v)) s = v;
        else if (v != -INFINITY) combine(m, s, v, 1.0f, a.k);
      }
    }
    warp_combine(m, s, a.k);
    if (!SHORT) {
      if (lane == 0) red[warp] = make_float2(m, s);
      __syncthreads();
    }
    if (!SHORT && warp == 0) {
      const float2 p = lane < bd >> 5 ? red[lane] : make_float2(-INFINITY, 0.0f);
      m = p.x; s = p.y;
      warp_combine(m, s, a.k);
      if (ctas > 1) {
        cluster_wait();
        if (lane == 0) *cl.map_shared_rank(&parts[rank], 0) = make_float2(m, s);
      }
    }
    if (ctas > 1) {
      if (warp != 0) cluster_wait();
      cl.sync();
      if (warp == 0) {
        const float2 p = lane < ctas ? parts[lane] : make_float2(-INFINITY, 0.0f);
        m = p.x; s = p.y;
        warp_combine(m, s, a.k);
      }
    }
    if (rank == 0 && tid == 0) {
      const TargetStats t = target_stats(m, s, to_f32(x[tgt]), a.k);
      write_target_row<OP>(a, row, t, finish_target_row<OP>(a, inputs, t), nullptr);
    }
  }
}

// A row's maximum and -log2 of its sum of exponentials, by a block or (SHORT) a warp that reads all of it: for the rare row whose known
// statistics have not the digits (see row_anchor).
template <typename T, bool SHORT>
__device__ __forceinline__ void sweep_row(const T* x, int V, float k, int tid, int bd, float* red, float& top, float& minus_log) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto joined = [&](float v, auto join) {
    for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (SHORT) return v;
    __syncthreads();   // red is free
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = red[0];
#pragma unroll 1
    for (int w = 1; w < bd >> 5; ++w) v = join(v, red[w]);
    return v;
  };
  float m = -INFINITY, s = 0.0f;
#pragma unroll 1
  for (int c = tid; c < V; c += bd) m = fmaxf(m, to_f32(x[c]));
  top = m = joined(m, [](float a, float b) { return fmaxf(a, b); });
#pragma unroll 1
  for (int c = tid; c < V; c += bd) s += ex2((to_f32(x[c]) - m) * k);
  minus_log = -log2f(joined(s, [](float a, float b) { return a + b; }));
}

// Gradient: dx_j = c (1[j = t] - p_j).  Bound: HBM, one read and one write.  A block takes `piece` vectors of a row, all of them in
// flight at once.  The rows are taken from the last to the first: what the statistics' kernel read last may still be in L2.
// Not in place: other blocks of the row read the target's logit, or (sweep_row) all of them.
// SHORT: a warp does (a row has one piece).
template <typename T, bool SHORT>
__global__ void __launch_bounds__(kThreads, SHORT ? 4 : 5)   // (the sweep that hardly any row takes would cost 16 registers, and with them a block an SM)
token_grad_stream_kernel(const GradArgs ga, int pieces, uint32_t parts) {
  using VT = Vec16<T>;
  using Raw = decltype(VT::raw);
  constexpr int N = VT::N;
  __shared__ float red[kThreads / 32];
  const RowArgs& a = ga.a;
  grid_launch_dependents();
  grid_dependency_wait();
  const uint32_t part = SHORT ? blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5) : blockIdx.x;
  if (SHORT && part >= parts) return;
  const uint32_t b = parts - 1 - part, row = b / static_cast<uint32_t>(pieces);
  const int piece = static_cast<int>(b - row * pieces), tid = SHORT ? threadIdx.x & 31 : threadIdx.x, bd = SHORT ? 32 : blockDim.x;
  const T* x = static_cast<const T*>(from_here(a.logits)) + row_offset(a, row);
  T* g = static_cast<T*>(a.grad) + static_cast<int64_t>(row) * a.V;
  const T* base;
  const RowVecs r = vecs_of(x, a.V, base);
  const Raw* src = reinterpret_cast<const Raw*>(base);
  T* to = g - r.lo;
  const bool same = (reinterpret_cast<uintptr_t>(to) & 15u) == 0;
  const int v0 = r.fa + piece * kUnroll * bd + tid;
  const int tgt = read_target(a.targets, a.target_bytes, a.has_ignore, a.ignore, row, a.V);
  const int edge = tid < N ? r.lo + tid : r.fb * N + tid - N;   // the elements beside the row's own vectors: the first block's
  const bool edges = piece == 0 && tid < 2 * N && (tid < N ? edge < min(r.fa * N, r.hi) : edge < r.hi);
  VT v[kUnroll];
  auto put = [&](int j) {
    const int vi = v0 + j * bd;
    if (vi >= r.fb) return;
    if (same) {
      __stcs(reinterpret_cast<Raw*>(to) + vi, v[j].raw);
    } else {
      const T* e = reinterpret_cast<const T*>(&v[j].raw);
#pragma unroll
      for (int q = 0; q < N; ++q) to[vi * N + q] = e[q];
    }
  };
  if (tgt < 0) {
    float f[N];
#pragma unroll
    for (int q = 0; q < N; ++q) f[q] = tgt == -2 ? NAN : 0.0f;
    v[0].from_float(f);
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      v[j] = v[0];
      put(j);
    }
    if (edges) to[edge] = from_f32<T>(f[0]);
    return;
  }
#pragma unroll
  for (int j = 0; j < kUnroll; ++j)
    if (v0 + j * bd < r.fb) v[j].raw = __ldcs(src + v0 + j * bd);
  const float c0 = ga.coef[row / static_cast<uint32_t>(ga.coef_rows)] * a.inv_t, logp = a.logp[row];
  float ref, add;
  if (!row_anchor(logp, a.lse[row], to_f32(x[tgt]), ref, add)) {   // the same in every thread of the row
    sweep_row<T, SHORT>(x, a.V, a.k, tid, bd, red, ref, add);
#pragma unroll
    for (int j = 0; j < kUnroll; ++j)   // again, so that nothing is kept meanwhile
      if (v0 + j * bd < r.fb) v[j].raw = __ldcs(src + v0 + j * bd);
  }
  const float2 neg = make_float2(-ref, -ref), kk = make_float2(a.k, a.k), add2 = make_float2(add, add), cc = make_float2(-c0, -c0);
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {
    float f[N];
    v[j].to_float(f);
#pragma unroll
    for (int q = 0; q < N; q += 2) {
      const float2 d = __ffma2_rn(__fadd2_rn(make_float2(f[q], f[q + 1]), neg), kk, add2);
      const float2 e = __fmul2_rn(make_float2(ex2(d.x), ex2(d.y)), cc);
      f[q] = e.x; f[q + 1] = e.y;
    }
    v[j].from_float(f);
    put(j);
  }
  const float at_target = c0 * -expm1f(logp);
  const int te = r.lo + tgt, tv = te / N;
  if (tv >= r.fa && tv < r.fb && tv >= v0 && tv < v0 + kUnroll * bd && (tv - v0) % bd == 0) to[te] = from_f32<T>(at_target);   // behind the vector
  if (edges) to[edge] = from_f32<T>(edge == te ? at_target : -c0 * ex2(fmaf(to_f32(base[edge]) - ref, a.k, add)));
}

// Short rows, statistics and gradient: a row held by a warp, as it was read; its exponentials are taken twice (there are few).  (bf16: in
// registers, but for some 20 words that spill.  float32: the search for the target's vector makes the row an array in local memory, 128
// bytes a thread.)  Any row may be written over.  20000 x 1000 bf16: a policy loss 40 us, by the one-pass kernel's warps, whose every row passes
// through a ring, barriers and a table, 64.  (Distillation is left to that one: its warps wait less for the teacher's entries.)
constexpr int kShortBlocks = 3;      // blocks an SM, which take rows in turn
template <typename T, int OP>
__global__ void __launch_bounds__(kThreads, kShortBlocks)
token_short_kernel(const RowArgs a, const RowPlan plan) {
  using VT = Vec16<T>;
  using Raw = decltype(VT::raw);
  constexpr int N = VT::N, kRows = kThreads / 32;
  __shared__ double sums[kRows][3];
  __shared__ int last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < kRows * 3) sums[0][threadIdx.x] = 0.0;
  __syncthreads();
  grid_launch_dependents();
  grid_dependency_wait();
  double* mine = plan.sums != nullptr ? sums[warp] : nullptr;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows + warp, step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t next = row0 < a.M ? load_target(a.targets, a.target_bytes, row0) : -1;   // known before the row is asked for: left out, it is not read
  for (int64_t row = row0; row < a.M; row += step) {
    const int tgt = kept_target(next, a.has_ignore, a.ignore, a.V);
    if (row + step < a.M) next = load_target(a.targets, a.target_bytes, row + step);
    const T* x = static_cast<const T*>(from_here(a.logits)) + row_offset(a, row);
    T* g = static_cast<T*>(a.grad) + row * a.V;
    const T* base;
    const RowVecs r = vecs_of(x, a.V, base);
    const Raw* src = reinterpret_cast<const Raw*>(base);
    T* to = g - r.lo;
    const bool same = (reinterpret_cast<uintptr_t>(to) & 15u) == 0;
    const int edge = lane < N ? r.lo + lane : r.fb * N + lane - N;   // the elements beside the row's own vectors
    const bool edges = lane < 2 * N && (lane < N ? edge < min(r.fa * N, r.hi) : edge < r.hi);
    VT v[kUnroll];
    auto put = [&](int j) {
      const int vi = r.fa + j * 32 + lane;
      if (vi >= r.fb) return;
      if (same) {
        __stcs(reinterpret_cast<Raw*>(to) + vi, v[j].raw);
      } else {
        const T* e = reinterpret_cast<const T*>(&v[j].raw);
#pragma unroll
        for (int q = 0; q < N; ++q) to[vi * N + q] = e[q];
      }
    };
    if (tgt < 0) {   // the same in every lane
      const float value = tgt == -2 ? NAN : 0.0f;
      if (lane == 0) write_left_out<OP>(a, row, value, mine);
      float f[N];
#pragma unroll
      for (int q = 0; q < N; ++q) f[q] = value;
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) { v[j].from_float(f); put(j); }
      if (edges) to[edge] = from_f32<T>(value);
      continue;
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int vi = r.fa + j * 32 + lane;
      if (vi < r.fb) v[j].raw = src[vi];
      else fill_masked(v[j]);
    }
    const float x_edge = edges ? to_f32(base[edge]) : -INFINITY;
    const RowInputs inputs = row_inputs<OP>(a, row);
    // the target: lane, vector and element, or an edge
    const int te = r.lo + tgt, tv = te / N - r.fa, tq = te % N;
    const bool own = te / N >= r.fa && te / N < r.fb && (tv & 31) == lane, at_edge = edges && edge == te;
    float xt = at_edge ? x_edge : 0.0f;
    if (own) {
#pragma unroll
      for (int j = 0; j < kUnroll; ++j)
        if (j == tv >> 5) {   // out of the sum
          float f[N];
          v[j].to_float(f);
#pragma unroll
          for (int q = 0; q < N; ++q)
            if (q == tq) { xt = f[q]; f[q] = -INFINITY; }
          v[j].from_float(f);
        }
    }
    xt = __shfl_sync(0xffffffffu, xt, __ffs(__ballot_sync(0xffffffffu, own || at_edge)) - 1);
    const float xe = at_edge ? -INFINITY : x_edge;
    float m = fmaxf(max_of(v), xe);
    m = warp_max(m);
    const float ref = m == -INFINITY ? 0.0f : m;
    const float2 neg = make_float2(-ref, -ref), kk = make_float2(a.k, a.k);
    float2 s2 = make_float2(edges ? ex2((xe - ref) * a.k) : 0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      float f[N];
      v[j].to_float(f);
#pragma unroll
      for (int q = 0; q < N; q += 2) {
        const float2 d = __fmul2_rn(__fadd2_rn(make_float2(f[q], f[q + 1]), neg), kk);
        s2 = __fadd2_rn(s2, make_float2(ex2(d.x), ex2(d.y)));
      }
    }
    const float s = warp_sum(s2.x + s2.y);
    const TargetStats t = target_stats(m, s, xt, a.k);
    const RowResult res = finish_target_row<OP>(a, inputs, t);
    if (lane == 0) write_target_row<OP>(a, row, t, res, mine);
    const float top = t.top == -INFINITY ? 0.0f : t.top, scale = -res.c / t.sum, at_target = res.c * t.rest;   // an element's gradient is scale 2^((x - top) k)
    const float2 neg_top = make_float2(-top, -top), ss = make_float2(scale, scale);
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      float f[N];
      v[j].to_float(f);
#pragma unroll
      for (int q = 0; q < N; q += 2) {
        const float2 d = __fmul2_rn(__fadd2_rn(make_float2(f[q], f[q + 1]), neg_top), kk);
        const float2 e = __fmul2_rn(make_float2(ex2(d.x), ex2(d.y)), ss);
        f[q] = e.x; f[q + 1] = e.y;
      }
      v[j].from_float(f);
      put(j);
    }
    if (own) to[te] = from_f32<T>(at_target);   // behind the vector
    if (edges) to[edge] = from_f32<T>(at_edge ? at_target : scale * ex2((x_edge - top) * a.k));
  }
  if (plan.sums != nullptr) {
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int t = 0; t < plan.n_sums; ++t) {
        double total = 0.0;
        for (int w = 0; w < kRows; ++w) total += sums[w][t];
        plan.partials[3 * blockIdx.x + t] = total;
      }
      __threadfence();
      last = atomicAdd(plan.done, 1) == static_cast<int>(gridDim.x) - 1;
    }
    __syncthreads();
    if (last) {
      __threadfence();
      block_sums(plan.partials, gridDim.x, 3, 1, plan.n_sums, plan.sums, sums[0]);
    }
  }
}

template <typename T, int OP>
int launch_short(const RowArgs& a, const RowPlan& plan, DeviceState* ds, cudaStream_t st, bool* taken) {
  constexpr int N = Vec16<T>::N, kRows = kThreads / 32;
  *taken = a.V / N + 1 <= 32 * kUnroll;
  if (!*taken) return MCB_OK;
  const int64_t blocks = (a.M + kRows - 1) / kRows, most = kShortBlocks * static_cast<int64_t>(ds->sm_count);
  const dim3 grid(static_cast<unsigned>(blocks < most ? blocks : most < kMaxPartials ? most : kMaxPartials));
  MCB_CHECK_CUDA(launch_kernel(token_short_kernel<T, OP>, grid, dim3(kThreads), 0, st, chained_launch(), a, plan));
  MCB_CHECK_LAUNCH("token_short");
  return MCB_OK;
}

template <typename T, int OP>
int launch_stats(const RowArgs& a, DeviceState* ds, cudaStream_t st) {
  constexpr int N = Vec16<T>::N;
  const int64_t vecs = a.V / N + 1;
  int threads = static_cast<int>((vecs + kUnroll - 1) / kUnroll + 31) / 32 * 32;
  threads = threads > kThreads ? kThreads : threads < 32 ? 32 : threads;
  // A cluster a row while that leaves SMs without a block, and its CTAs have a batch of loads each.
  int log_ctas = 0;
  while (log_ctas < 3 && a.M << (log_ctas + 1) <= 2 * ds->sm_count && vecs >> (log_ctas + 1) >= kUnroll * threads) ++log_ctas;
  if (a.M << log_ctas > 0x7fffffff) return fail(MCB_ERR_SHAPE, "token_stats: too many rows");
  if (threads == 32) {
    MCB_CHECK_CUDA(launch_kernel(token_stats_kernel<T, OP, true>, dim3(static_cast<unsigned>((a.M + kThreads / 32 - 1) / (kThreads / 32))), dim3(kThreads),
                                 0, st, chained_launch(), a, 0));
    MCB_CHECK_LAUNCH("token_stats");
    return MCB_OK;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.M << log_ctas)); cfg.blockDim = dim3(static_cast<unsigned>(threads)); cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1u << log_ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = chained_launch() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, token_stats_kernel<T, OP, false>, a, log_ctas);
  if (e != cudaSuccess) return cuda_fail(e, "token_stats_kernel launch");
  MCB_CHECK_LAUNCH("token_stats");
  return MCB_OK;
}

template <typename T>
int launch_stream(const GradArgs& ga, DeviceState* ds, cudaStream_t st, bool* taken) {
  constexpr int N = Vec16<T>::N;
  const int64_t vecs = ga.a.V / N + 1;
  int threads = static_cast<int>((vecs + kUnroll - 1) / kUnroll + 31) / 32 * 32;
  threads = threads > kThreads ? kThreads : threads < 32 ? 32 : threads;
  const int64_t pieces = (vecs + kUnroll * threads - 1) / (kUnroll * threads), blocks = pieces * ga.a.M;
  *taken = ga.a.logits != ga.a.grad && blocks <= 0x7fffffff;
  if (!*taken) return MCB_OK;
  if (threads == 32)
    MCB_CHECK_CUDA(launch_kernel(token_grad_stream_kernel<T, true>, dim3(static_cast<unsigned>((blocks + kThreads / 32 - 1) / (kThreads / 32))),
                                 dim3(kThreads), 0, st, chained_launch(), ga, static_cast<int>(pieces), static_cast<uint32_t>(blocks)));
  else
    MCB_CHECK_CUDA(launch_kernel(token_grad_stream_kernel<T, false>, dim3(static_cast<unsigned>(blocks)), dim3(static_cast<unsigned>(threads)), 0, st,
                                 chained_launch(), ga, static_cast<int>(pieces), static_cast<uint32_t>(blocks)));
  MCB_CHECK_LAUNCH("token_grad_stream");
  return MCB_OK;
}

}  // namespace

namespace tokenloss {
int launch_stats_rows(int op, const RowArgs& a, int dtype, DeviceState* ds, cudaStream_t st) {
  const bool f32 = dtype == MCB_F32;
  if (op == kPolicy) return f32 ? launch_stats<float, kPolicy>(a, ds, st) : launch_stats<__nv_bfloat16, kPolicy>(a, ds, st);
  return f32 ? launch_stats<float, kStats>(a, ds, st) : launch_stats<__nv_bfloat16, kStats>(a, ds, st);
}
int launch_short_rows(int op, const RowArgs& a, const RowPlan& plan, int dtype, DeviceState* ds, cudaStream_t st, bool* taken) {
  const bool f32 = dtype == MCB_F32;
  if (op == kUnit) return f32 ? launch_short<float, kUnit>(a, plan, ds, st, taken) : launch_short<__nv_bfloat16, kUnit>(a, plan, ds, st, taken);
  return f32 ? launch_short<float, kPolicy>(a, plan, ds, st, taken) : launch_short<__nv_bfloat16, kPolicy>(a, plan, ds, st, taken);
}
int launch_grad_stream(const GradArgs& ga, int dtype, DeviceState* ds, cudaStream_t st, bool* taken) {
  return dtype == MCB_F32 ? launch_stream<float>(ga, ds, st, taken) : launch_stream<__nv_bfloat16>(ga, ds, st, taken);
}
}  // namespace tokenloss
}  // namespace mcb
