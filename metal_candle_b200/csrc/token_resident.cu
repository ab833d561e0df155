// Token losses with their gradient in one pass: a row of logits is read once, held in registers as exponentials, and written
// once as its gradient.
//
// Bound: HBM, one read and one write of the row.  The softmax of a row needs two sweeps over it, and a row (304 KB at 151936 bf16)
// is more than an SM takes.  A cluster of up to 8 CTAs shares it; each brings its share into shared memory by one bulk copy
// (one or two rows ahead, so that the copies run under the arithmetic) and from there into registers, 80 elements a thread.
// A thread takes its own maximum m_t and e_j = 2^((x_j - m_t) k) at once, and once only: when the row's maximum m and sum s are
// known, the gradient is e_j times 2^((m_t - m) k) / s times the row's coefficient, one multiplication an element.  An SM's
// special-function units give 16 exponentials a cycle, 4.5e12 a second on the chip, where the copy bandwidth asks for 1.6e12
// (bf16): with two an element, sum and gradient, they would be three quarters busy and every stall would show.
// (m_t, s_t) are combined over the CTA through one barrier and over the cluster through distributed shared memory, once a row;
// the sums have one order.
#include <cooperative_groups.h>

#include <mutex>

#include "token_loss.cuh"
#include "umma_ptx.cuh"

namespace cg = cooperative_groups;

namespace mcb {
namespace {
using namespace tokenloss;
using namespace umma;

constexpr int kEpt = 80;            // elements a thread holds
constexpr int kMaxThreads = 512, kSoloThreads = 256;
constexpr int kMaxWarps = kMaxThreads / 32;

struct Resident {
  int ctas, log_ctas, stages, slot_bytes;
  int mis;                 // elements from a 16-byte boundary to the logits' first
  uint32_t magic;          // 2^32 / threads, rounded up: v / threads = umulhi(v, magic) for the vectors of a share
  const int32_t* order;    // rows in the order they are taken, those that are kept first; null: as they lie
  const int32_t* kept;     // how many those are
  float* out;              // sums of the terms, or null
  int n_out;
  int* done;
  int* status;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// Bounded like every wait of the library, with acquire at cluster scope: the data came from a peer's store.
__device__ __forceinline__ void wait_peers(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
  const long long t0 = clock64();
  while (true) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok || *abort_flag != 0) return;
    if (clock64() - t0 > kWaitLimitCycles) { *abort_flag = 59; atomicCAS(status, 0, 59); return; }
  }
}

template <typename T>
struct Lane;   // the maximum of a vector in memory
template <>
struct Lane<__nv_bfloat16> {
  static constexpr uint32_t kMasked = 0xff80ff80u;   // -inf
  static __device__ __forceinline__ float max_of(const Vec16<__nv_bfloat16>& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v.raw);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};
template <>
struct Lane<float> {
  static constexpr uint32_t kMasked = 0xff800000u;
  static __device__ __forceinline__ float max_of(const Vec16<float>& v) { return fmaxf(fmaxf(v.raw.x, v.raw.y), fmaxf(v.raw.z, v.raw.w)); }
};

// (m, s) of a warp's lanes: the same in every lane
__device__ __forceinline__ void warp_combine(float& m, float& s, float k) {
  const float top = warp_max(m);
  s = warp_sum(m == -INFINITY ? s : s * ex2((m - top) * k));   // (nothing kept: 0, or NaN if it holds one)
  m = top;
}

// A CTA's share of a row: n vectors from a 16-byte boundary on.  Of its elements [lo, hi) are the row's, and its vectors [fa, fb) the
// row's alone; those beside them are shared with the neighbouring rows.
struct Share {
  int64_t from, to;      // where the share begins, in elements from the logits' 16-byte boundary and from the gradient's first element
  int n, lo, hi, fa, fb;
  int column;            // of the vocabulary, at the share's element 0 (negative in front of the row)
};
template <int N>
__device__ __forceinline__ Share share_of(const RowArgs& a, const Resident& p, int rank, int64_t row) {
  Share s;
  const int64_t e0 = row_offset(a, row) + p.mis;
  const int64_t v0 = e0 / N;
  const int vecs = static_cast<int>((e0 + a.V + N - 1) / N - v0), per = (vecs + p.ctas - 1) >> p.log_ctas;
  const int begin = min(vecs, rank * per);
  s.n = min(vecs, begin + per) - begin;
  s.from = (v0 + begin) * N;
  s.column = static_cast<int>(s.from - e0);
  s.to = row * a.V + s.column;
  s.lo = max(0, -s.column);
  s.hi = max(s.lo, min(s.n * N, a.V - s.column));
  s.fa = (s.lo + N - 1) / N;
  s.fb = max(s.fa, s.hi / N);
  return s;
}

// What a row needs besides its logits, brought in for many of a cluster's rows at a time: a row's own loads, each behind the one before
// (order, target, what belongs to the target), would cost it microseconds.
struct RowInfo {
  Share share;
  int row, target;   // the target: within the share, or -1
  int state;         // 0: to be computed, 1: left out, 2: out of range
  RowInputs in;
};
constexpr int kInfoRows = 64;

// SAME: every row of the gradient lies as its logits do relative to 16 bytes, so that whole vectors can be written.
template <typename T, int OP, bool SAME>
__global__ void __launch_bounds__(kMaxThreads, 1)
token_resident_kernel(const RowArgs a, const Resident p) {
  using VT = Vec16<T>;
  using Raw = decltype(VT::raw);
  constexpr int N = VT::N, NV = kEpt / N;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[2];
  __shared__ __align__(8) uint64_t slot_bars[2];
  __shared__ __align__(16) float4 slots[2][8];   // every CTA's (maximum, sum, target's logit or loss, whose target it is), by parity
  __shared__ float3 red[2][kMaxWarps];
  __shared__ RowInfo infos[kInfoRows];
  __shared__ float edge[2][2 * N];               // the share's elements in vectors that are not the row's alone, by parity
  __shared__ float target_logit[2];
  __shared__ int repeats[2];                     // an id that came twice among the row's teacher entries, by parity
  __shared__ int abort_word;
  __shared__ int last;
  volatile int* abort_flag = &abort_word;
  cg::cluster_group cl = cg::this_cluster();
  const int ctas = p.ctas, rank = static_cast<int>(cl.block_rank());
  const int first = static_cast<int>(blockIdx.x) >> p.log_ctas, step = static_cast<int>(gridDim.x) >> p.log_ctas;
  const int tid = threadIdx.x, bd = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = bd >> 5;
  const uint32_t sbase = smem_u32(smem), full0 = smem_u32(full);
  // the teacher's entries behind the slots: id within the share (or -1), probability and logit, and a bitmap of the ids; by parity
  int* t_id = reinterpret_cast<int*>(smem + p.stages * p.slot_bytes);
  float* t_q = reinterpret_cast<float*>(t_id + 2 * a.K);
  float* t_x = t_q + 2 * a.K;
  uint32_t* t_bits = reinterpret_cast<uint32_t*>(t_x + 2 * a.K);
  const int bit_words = p.slot_bytes / 16 * N / 32 + 1;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) { mbar_init(full0 + 8 * i, 1); mbar_init(smem_u32(&slot_bars[i]), ctas); repeats[i] = 0; }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
  }
  if constexpr (OP == kDistill)
    for (int i = tid; i < 2 * bit_words; i += bd) t_bits[i] = 0;
  if (ctas > 1) cl.sync(); else __syncthreads();   // every CTA's barriers exist before a peer arrives on them
  grid_launch_dependents();
  grid_dependency_wait();
  const int M = static_cast<int>(a.M);
  const int kept = p.kept != nullptr ? *from_here(p.kept) : M;
  auto row_of = [&](int64_t i) -> int { return p.order != nullptr ? from_here(p.order)[i] : static_cast<int>(i); };
  auto request = [&](const Share& s, int stage) {   // by one thread
    mbar_expect_tx(full0 + 8 * stage, s.n * 16);   // a share with nothing in it completes at once
    if (s.n > 0)
      bulk_load(sbase + stage * p.slot_bytes, static_cast<const T*>(a.logits) - p.mis + s.from, s.n * 16, full0 + 8 * stage);
  };
  if (tid == 0)
    for (int s = 0; s < p.stages; ++s)
      if (first + static_cast<int64_t>(s) * step < kept) request(share_of<N>(a, p, rank, row_of(first + static_cast<int64_t>(s) * step)), s);

  uint32_t phases = 0, slot_phase = 0;   // bit i: parity of the i-th barrier's next completion
  int stage = 0, par = 0, at = kInfoRows;
  for (int64_t i = first; i < M; i += step, ++at) {
    if (at == kInfoRows) {
      __syncthreads();   // the last of them is done with
      for (int q = tid; q < kInfoRows; q += bd) {
        const int64_t iq = i + static_cast<int64_t>(q) * step;
        if (iq < M) {
          RowInfo f;
          f.row = row_of(iq);
          f.share = share_of<N>(a, p, rank, f.row);
          f.target = -1;
          f.state = iq < kept ? 0 : 1;
          if constexpr (OP != kDistill) {
            const int t = read_target(a.targets, a.target_bytes, a.has_ignore, a.ignore, f.row, a.V);
            if (t < 0) f.state = t == -2 ? 2 : 1;
            else if (t - f.share.column >= f.share.lo && t - f.share.column < f.share.hi) f.target = t - f.share.column;
          }
          f.in = row_inputs<OP>(a, f.row);
          infos[q] = f;
        }
      }
      __syncthreads();
      at = 0;
    }
    const RowInfo& info = infos[at];
    const bool loaded = i < kept;
    // by thread 0, when the row's slot is free: the row that is to lie there next
    auto refill = [&]() {
      if (tid == 0 && i + static_cast<int64_t>(p.stages) * step < kept)
        request(at + p.stages < kInfoRows ? infos[at + p.stages].share
                                          : share_of<N>(a, p, rank, row_of(i + static_cast<int64_t>(p.stages) * step)), stage);
      if (++stage == p.stages) stage = 0;
    };
    if (info.state != 0) {   // the same in every CTA of the cluster
      const float value = info.state == 2 ? NAN : 0.0f;
      if (rank == 0 && tid == 0) write_left_out<OP>(a, info.row, value);
      if (a.grad != nullptr) {
        const Share& s = info.share;
        T* g = static_cast<T*>(a.grad) + s.to;
        if (SAME) {
          VT z;
          float f[N];
#pragma unroll
          for (int j = 0; j < N; ++j) f[j] = value;
          z.from_float(f);
          for (int vi = s.fa + tid; vi < s.fb; vi += bd) __stcs(reinterpret_cast<Raw*>(g) + vi, z.raw);
          for (int e = s.lo + tid; e < min(s.fa * N, s.hi); e += bd) g[e] = from_f32<T>(value);
          for (int e = s.fb * N + tid; e < s.hi; e += bd) g[e] = from_f32<T>(value);
        } else {
          for (int e = s.lo + tid; e < s.hi; e += bd) g[e] = from_f32<T>(value);
        }
      }
      if (loaded) {
        mbar_wait(full0 + 8 * stage, (phases >> stage) & 1u, abort_flag, 58, p.status);
        phases ^= 1u << stage;
        __syncthreads();   // everyone has waited for this completion before the barrier is used again
        refill();
      }
      continue;
    }
    // the teacher's distribution over its entries: each warp takes all of them
    float tm = -INFINITY, ts = 0.0f, x_ref = 0.0f;
    if constexpr (OP == kDistill) {
      const int64_t t0 = static_cast<int64_t>(info.row) * a.K;
      for (int q = lane; q < a.K; q += 32) tm = fmaxf(tm, read_teacher(a, t0 + q));
      tm = warp_max(tm);
      const float tref = tm == -INFINITY ? 0.0f : tm;
      int64_t best = -1;
      for (int q = lane; q < a.K; q += 32) {
        const float t = read_teacher(a, t0 + q);
        ts += exp2f((t - tref) * a.k);
        if (t == tm && best < 0) best = read_teacher_id(a, t0 + q);
      }
      ts = warp_sum(ts);
      // the student's logit where the teacher's is largest: the loss's logits are taken relative to it
      const uint32_t who = __ballot_sync(0xffffffffu, best >= 0);
      best = __shfl_sync(0xffffffffu, best, who == 0 ? 0 : __ffs(who) - 1);
      if (best >= 0 && best < a.V) x_ref = to_f32(static_cast<const T*>(a.logits)[row_offset(a, info.row) + best]);
      if (!(fabsf(x_ref) < INFINITY)) x_ref = 0.0f;
    }
    float third = 0.0f, m = -INFINITY, sw, e[kEpt];
    bool own = false;
    {
      const Share& s = info.share;
      const int n = s.n, tl = info.target;
      own = tl >= 0;
      mbar_wait(full0 + 8 * stage, (phases >> stage) & 1u, abort_flag, 58, p.status);
      phases ^= 1u << stage;
      Raw* srow = reinterpret_cast<Raw*>(smem + stage * p.slot_bytes);
      T* selem = reinterpret_cast<T*>(srow);
      // What is not to be summed (the neighbouring rows' elements, the target) becomes -inf in the slot, by the thread that reads the
      // vector below.
      auto reader = [&](int v) { return static_cast<int>(v - __umulhi(static_cast<uint32_t>(v), p.magic) * bd) == tid; };
      bool patched = false;
      if (own && reader(tl / N)) { target_logit[par] = to_f32(selem[tl]); selem[tl] = from_f32<T>(-INFINITY); patched = true; }
      if (s.lo > 0 && tid == 0) {   // (the share's first vector is thread 0's)
        for (int q = 0; q < s.lo; ++q) selem[q] = from_f32<T>(-INFINITY);
        patched = true;
      }
      if (s.hi < n * N && reader(n - 1)) {
        for (int q = s.hi; q < n * N; ++q) selem[q] = from_f32<T>(-INFINITY);
        patched = true;
      }
      if (patched) fence_proxy_async_smem();   // the slot's next copy comes behind these stores
      if (tid < 2 * N) {   // the row's elements in those vectors are written one by one
        const int el = tid < N ? s.lo + tid : s.fb * N + tid - N;
        if (tid < N ? el < min(s.fa * N, s.hi) : el < s.hi) edge[par][tid] = to_f32(selem[el]);
      }
      VT raw[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        {
          uint32_t* w = reinterpret_cast<uint32_t*>(&raw[j].raw);
          w[0] = w[1] = w[2] = w[3] = Lane<T>::kMasked;
          if (j * bd + tid < n) raw[j].raw = srow[j * bd + tid];
          m = fmaxf(m, Lane<T>::max_of(raw[j]));
        }
      }
      if constexpr (OP == kDistill) {
        const int64_t t0 = static_cast<int64_t>(info.row) * a.K;
        const float tref = tm == -INFINITY ? 0.0f : tm;
        const float inv_ts = 1.0f / ts, log_ts = logf(ts);
        uint32_t* bits = t_bits + par * bit_words;
        for (int q = tid; q < a.K; q += bd) {
          const float d = read_teacher(a, t0 + q) - tref;   // log q = d / T - log_ts
          const float prob = ts == 0.0f ? 0.0f : exp2f(d * a.k) * inv_ts;
          int el = -1;
          if (prob != 0.0f) {   // (NaN counts)
            const int64_t id = read_teacher_id(a, t0 + q);
            if (id < 0 || id >= a.V) {
              third = NAN;
            } else {
              const int64_t off = id - s.column;
              if (off >= s.lo && off < s.hi) {
                el = static_cast<int>(off);
                const float x = to_f32(selem[el]);
                third += prob * ((d * a.inv_t - log_ts) - (x - x_ref) * a.inv_t);
                t_x[par * a.K + q] = x;
                if (atomicOr(bits + (el >> 5), 1u << (el & 31)) >> (el & 31) & 1u) repeats[par] = 1;
              }
            }
          }
          t_id[par * a.K + q] = el;
          t_q[par * a.K + q] = prob;
        }
        third = warp_sum(third);
      }
      const float mref = m == -INFINITY ? 0.0f : m;
      const float2 neg_m = make_float2(-mref, -mref), kk = make_float2(a.k, a.k);
      float2 s2 = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        {
          float f[N];
          raw[j].to_float(f);
#pragma unroll
          for (int q = 0; q < N; q += 2) {
            const float2 d = __fmul2_rn(__fadd2_rn(make_float2(f[q], f[q + 1]), neg_m), kk);
            const float2 x = make_float2(ex2(d.x), ex2(d.y));
            s2 = __fadd2_rn(s2, x);
            e[j * N + q] = x.x; e[j * N + q + 1] = x.y;
          }
        }
      }
      float mw = m;
      sw = s2.x + s2.y;
      warp_combine(mw, sw, a.k);
      if (lane == 0) red[par][warp] = make_float3(mw, sw, third);
    }
    __syncthreads();
    refill();   // everyone has taken what it needs of the slot
    if (OP == kDistill && tid == 0) repeats[par ^ 1] = 0;   // the row before is done with it, the next one not begun
    float mw;
    {
      const float3 r = lane < warps ? red[par][lane] : make_float3(-INFINITY, 0.0f, 0.0f);
      mw = r.x; sw = r.y;
      warp_combine(mw, sw, a.k);
      if constexpr (OP == kDistill) third = warp_sum(r.z);
      else if (own) third = target_logit[par];
    }
    if (ctas > 1) {
      // Thread q hands this CTA's part to CTA q.  A slot is written again two rows later, when its readers have passed the
      // exchange in between.
      const uint32_t slot = smem_u32(&slots[par][rank]), bar = smem_u32(&slot_bars[par]);
      if (tid < ctas)
        asm volatile("{\n\t.reg .b32 rs, rb;\n\t"
                     "mapa.shared::cluster.u32 rs, %0, %2;\n\t"
                     "mapa.shared::cluster.u32 rb, %1, %2;\n\t"
                     "st.shared::cluster.v4.f32 [rs], {%3, %4, %5, %6};\n\t"
                     "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [rb];\n\t}"
                     ::"r"(slot), "r"(bar), "r"(tid), "f"(mw), "f"(sw), "f"(third), "f"(own ? 1.0f : 0.0f) : "memory");
      wait_peers(bar, (slot_phase >> par) & 1u, abort_flag, p.status);
      slot_phase ^= 1u << par;
      const float4 r = lane < ctas ? slots[par][lane] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
      mw = r.x; sw = r.y;
      warp_combine(mw, sw, a.k);
      if constexpr (OP == kDistill) {
        third = warp_sum(r.z);
      } else {
        const uint32_t who = __ballot_sync(0xffffffffu, r.w != 0.0f);
        third = __shfl_sync(0xffffffffu, r.z, who == 0 ? 0 : __ffs(who) - 1);
      }
    }
    const int row = info.row;
    const bool writes = rank == 0 && tid == 0;
    float f, f_top, top, c0, at_target = 0.0f;   // an element's gradient is f times its e, or f_top 2^((x - top) k)
    if constexpr (OP == kDistill) {
      const float w = info.in.weight;
      const bool empty = ts == 0.0f;
      top = mw == -INFINITY ? 0.0f : mw;
      const float loss = empty ? 0.0f : third + ((top - x_ref) * a.inv_t + logf(sw));
      if (writes) a.terms[row] = w * (a.temperature * a.temperature) * loss;
      c0 = empty ? 0.0f : w * a.temperature + (isnan(loss) ? NAN : 0.0f);
      f_top = empty ? 0.0f : c0 / sw;
    } else {
      const TargetStats r = target_stats(mw, sw, third, a.k);
      c0 = finish_target_row<OP>(a, row, info.in, r, writes);
      at_target = c0 * r.rest;
      f_top = -c0 / r.sum;
      top = r.top == -INFINITY ? 0.0f : r.top;
    }
    f = m == -INFINITY ? f_top : f_top * ex2((m - top) * a.k);   // (nothing kept in the thread: zeros, or NaN)
    if (a.grad != nullptr) {
      const Share& s = info.share;
      T* g = static_cast<T*>(a.grad) + s.to;
      const float2 ff = make_float2(f, f);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        {
          const int vi = j * bd + tid;
          float x[N];
#pragma unroll
          for (int q = 0; q < N; q += 2) {
            const float2 y = __fmul2_rn(make_float2(e[j * N + q], e[j * N + q + 1]), ff);
            x[q] = y.x; x[q + 1] = y.y;
          }
          if (vi >= s.fa && vi < s.fb) {
            if (SAME) {
              VT t;
              t.from_float(x);
              __stcs(reinterpret_cast<Raw*>(g) + vi, t.raw);
            } else {
#pragma unroll
              for (int q = 0; q < N; ++q) g[vi * N + q] = from_f32<T>(x[q]);
            }
          }
        }
      }
      const int tl = info.target;
      if (OP != kDistill && own) {
        const int tv = tl / N;
        if (tv >= s.fa && tv < s.fb && static_cast<int>(tv - __umulhi(static_cast<uint32_t>(tv), p.magic) * bd) == tid)
          g[tl] = from_f32<T>(at_target);   // behind this thread's own vector
      }
      if (tid < 2 * N) {
        const int el = tid < N ? s.lo + tid : s.fb * N + tid - N;
        if (tid < N ? el < min(s.fa * N, s.hi) : el < s.hi)
          g[el] = from_f32<T>(el == tl ? at_target : f_top * ex2((edge[par][tid] - top) * a.k));
      }
      if constexpr (OP == kDistill) {
        __syncthreads();   // the row's softmax is written before its teacher columns are
        uint32_t* bits = t_bits + par * bit_words;
        const int* ids = t_id + par * a.K;
        const bool twice = repeats[par] != 0;
        for (int q = tid; q < a.K; q += bd) {
          const int el = ids[q];
          if (el < 0) continue;
          float prob = t_q[par * a.K + q];
          bool mine = true;
          if (twice) {   // the first of those that name the same column writes the sum of them
            prob = 0.0f;
            for (int o = 0; o < a.K; ++o) {
              if (ids[o] != el) continue;
              if (o < q) { mine = false; break; }
              prob += t_q[par * a.K + o];
            }
          }
          if (mine) g[el] = from_f32<T>(c0 * (exp2f((t_x[par * a.K + q] - top) * a.k) / sw - prob));
        }
      }
    }
    if constexpr (OP == kDistill) {   // (this parity's entries are made again behind the next row's barrier)
      for (int q = tid; q < a.K; q += bd)
        if (t_id[par * a.K + q] >= 0) t_bits[par * bit_words + (t_id[par * a.K + q] >> 5)] = 0;
    }
    par ^= 1;
  }
  __syncthreads();
  if (*abort_flag != 0) {
    for (int q = 0; q < 200; ++q) __nanosleep(1000);   // loads in flight land before the shared memory is released
  }
  if (ctas > 1) cl.sync();   // no peer still writes here
  if (p.out != nullptr && rank == 0) {
    // the last cluster to finish sums what all have left, in one order whichever it is
    if (tid == 0) {
      __threadfence();
      last = atomicAdd(p.done, 1) == step - 1;
    }
    __syncthreads();
    if (last) {
      __threadfence();
      double* sums = reinterpret_cast<double*>(smem);
      for (int t = 0; t < p.n_out; ++t) {
        double acc = 0.0;
        for (int q = tid; q < M; q += bd) acc += static_cast<double>(__ldcg(a.terms + static_cast<int64_t>(t) * M + q));
        for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
        if (lane == 0) sums[warp] = acc;
        __syncthreads();
        if (tid == 0) {
          double total = 0.0;
          for (int w = 0; w < warps; ++w) total += sums[w];
          p.out[t] = static_cast<float>(total);
        }
        __syncthreads();
      }
    }
  }
}

// What a launch needs to know of the device: its resident clusters, kept for the last few shapes (the query takes microseconds).
struct ResidentKey {
  const DeviceState* ds;
  const void* kernel;
  int ctas, threads;
  size_t smem;
  bool operator==(const ResidentKey& o) const {
    return ds == o.ds && kernel == o.kernel && ctas == o.ctas && threads == o.threads && smem == o.smem;
  }
};

template <typename T, int OP>
int launch_resident(const RowArgs& a, const RowPlan& plan, DeviceState* ds, cudaStream_t st, bool* taken) {
  constexpr int N = Vec16<T>::N, NV = kEpt / N;
  *taken = false;
  const uintptr_t ai = reinterpret_cast<uintptr_t>(a.logits), ag = reinterpret_cast<uintptr_t>(a.grad);
  const int64_t vecs = (static_cast<int64_t>(a.V) + 2 * N - 2) / N;   // that cover a row at most
  int log_ctas = 0;
  auto per_cta = [&]() { return (vecs + (1 << log_ctas) - 1) >> log_ctas; };
  while (log_ctas < 3 && per_cta() > kSoloThreads * NV) ++log_ctas;
  if (per_cta() > kMaxThreads * NV) return MCB_OK;
  int threads = static_cast<int>((per_cta() + NV - 1) / NV + 31) / 32 * 32;
  Resident p;
  p.ctas = 1 << log_ctas; p.log_ctas = log_ctas;
  p.slot_bytes = static_cast<int>(per_cta() * 16);
  p.mis = static_cast<int>((ai & 15u) / sizeof(T));
  p.magic = static_cast<uint32_t>(0x100000000ull / threads + (0x100000000ull % threads != 0));
  p.order = plan.order; p.kept = plan.kept; p.out = plan.sums; p.n_out = plan.n_sums; p.done = plan.done; p.status = ds->status_word;
  const int64_t extra = 256 + (OP == kDistill ? 24 * static_cast<int64_t>(a.K) + 8 * (p.slot_bytes / 16 * N / 32 + 1) : 0);
  const int per_sm = kMaxThreads / threads;
  p.stages = per_sm * (2 * p.slot_bytes + extra + 1024) <= 224 * 1024 ? 2 : 1;
  const size_t smem = static_cast<size_t>(p.stages) * p.slot_bytes + extra;
  if (smem > 200 * 1024) return MCB_OK;

  const bool same = a.grad == nullptr || (((ai ^ ag) & 15u) == 0 && (a.token_stride - a.V) % N == 0 && (a.batch_stride - a.S * a.V) % N == 0);
  const auto kernel = same ? token_resident_kernel<T, OP, true> : token_resident_kernel<T, OP, false>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.ctas)); cfg.blockDim = dim3(static_cast<unsigned>(threads)); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.ctas); attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  int resident = 0;
  {
    static std::mutex mu;
    static ResidentKey keys[16];
    static int counts[16], next = 0;
    const ResidentKey key{ds, reinterpret_cast<const void*>(kernel), p.ctas, threads, smem};
    std::lock_guard<std::mutex> lock(mu);
    for (int i = 0; i < 16; ++i)
      if (keys[i] == key) resident = counts[i];
    if (resident == 0) {
      MCB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
      MCB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
      MCB_CHECK_CUDA(cudaOccupancyMaxActiveClusters(&resident, kernel, &cfg));
      if (resident < 1) resident = 1;
      keys[next] = key; counts[next] = resident;
      next = (next + 1) % 16;
    }
  }
  // as many clusters as are resident together: a later one would start its share of the rows when the others are done
  cfg.gridDim = dim3(static_cast<unsigned>((a.M < resident ? a.M : resident) * p.ctas));
  if (chained_launch()) cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, p);
  if (e != cudaSuccess) return cuda_fail(e, "token_resident_kernel launch");
  MCB_CHECK_LAUNCH("token_resident");
  *taken = true;
  return MCB_OK;
}

}  // namespace

namespace tokenloss {
int launch_resident_rows(int op, const RowArgs& a, const RowPlan& plan, int dtype, DeviceState* ds, cudaStream_t st, bool* taken) {
  const bool f32 = dtype == MCB_F32;
  if (op == kUnit) return f32 ? launch_resident<float, kUnit>(a, plan, ds, st, taken) : launch_resident<__nv_bfloat16, kUnit>(a, plan, ds, st, taken);
  if (op == kPolicy) return f32 ? launch_resident<float, kPolicy>(a, plan, ds, st, taken) : launch_resident<__nv_bfloat16, kPolicy>(a, plan, ds, st, taken);
  if (op == kDistill)
    return f32 ? launch_resident<float, kDistill>(a, plan, ds, st, taken) : launch_resident<__nv_bfloat16, kDistill>(a, plan, ds, st, taken);
  *taken = false;
  return MCB_OK;
}
}  // namespace tokenloss
}  // namespace mcb
