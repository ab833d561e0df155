// Token losses with their gradient in one pass: a row of logits is read once, held on chip as exponentials, and written once as its
// gradient.
//
// Bound: HBM, one read and one write of the row.  The softmax of a row needs two sweeps over it.  If both take exponentials, the
// special-function units (16 a cycle and SM, 4.5e12 a second on the chip, where the copy bandwidth asks for 1.6e12 bf16 elements) are
// three quarters busy and every stall shows; so the first sweep's are kept: with m_t the largest logit a thread has seen,
// e_j = 2^((x_j - m_t) k), and when the row's maximum m and sum s are known the gradient is e_j times 2^((m_t - m) k) / s times the row's
// coefficient, one multiplication an element.  A row of 151936 is 608 KB of them.  A cluster of up to 8 CTAs shares it, and a CTA
// keeps its share in tensor memory, 256 KB an SM that nothing else here uses: a thread writes and reads its own lane, up to 4 chunks
// of 32 columns, and a fifth chunk stays in registers.
//
// Between a row's two sweeps lie the exchange over the cluster and the row's own scalar arithmetic.  So a row takes as few CTAs and
// then as few warps as hold it: an exchange less is worth more than rows in flight.  The warps of one row are a GROUP (one to sixteen;
// more of them, and clusters, where there are few rows), with its own ring of shared-memory pieces that bulk copies fill ahead of it,
// across the end of a row, and its own barriers; short rows have several groups on an SM.  Four further warps feed the rings and work
// out the teacher's part of a distillation row ahead of it.
// 4096 rows of 151936 bf16, all kept: 784 us with the exponentials in registers alone (a row over four CTAs, two rows in flight), 661
// in tensor memory over eight CTAs with four rows in flight, 493 as here (5.05 TB/s).  Of a row's 17 thousand cycles, where its bytes
// ask HBM for 13.6: first sweep 8.2, joining the group 1.1, the cluster 0.5 to 1, the row's arithmetic and gradient scale 1.8, second
// sweep 4.9; the ring's copies run under all of it, the stores under the second sweep alone.
// One CTA takes a whole SM (its ring excludes other kernels' shared memory), so that tensor memory is its alone and taking it never
// waits: a cluster that held some of it while it waited for more could wait for a kernel that waits for the cluster.
//
// (m, s) are combined over the group through one barrier and over the cluster through distributed shared memory, once a row; all sums
// have one order.
#include <cooperative_groups.h>

#include <float.h>

#include <mutex>

#include "token_loss.cuh"
#include "umma_ptx.cuh"

namespace cg = cooperative_groups;

namespace mcb {
namespace {
using namespace tokenloss;
using namespace umma;

constexpr int kThreads = 512, kWarps = kThreads / 32;   // that take rows
constexpr int kAllThreads = kThreads + 128;              // and four warps that serve them
// Registers: 640 threads are launched with 96 each, 61440; the row warps take 112, the serving ones keep 32 (512 x 112 + 128 x 32 = 61440).
// (Distillation with 104 and 64, so that the teacher's part spills nothing: 3 % slower.)
constexpr int kRowRegs = 112, kServeRegs = 32;
constexpr int kChunk = 32;             // elements a thread takes at a time
constexpr int kTmemChunks = 4;         // chunks it keeps in tensor memory, beside one in registers
constexpr int kMaxChunks = kTmemChunks + 1;
constexpr int kMaxPieces = 6;          // ring slots of a group
constexpr uint32_t kEdges = 1u << 31;
constexpr int kInfoRows = 128;         // rows a CTA's groups look ahead at, together
constexpr int kSmem = 200 * 1024;      // dynamic shared memory, at least: with it no other kernel that uses tensor memory fits on the SM

struct Resident {
  int ctas, log_ctas;
  int group_warps, log_groups;   // warps a group; groups a CTA
  int pieces;                    // ring slots a group
  int tmem;                      // whether any row has more than one chunk
  int mis;                       // elements from a 16-byte boundary to the logits' first
  const int32_t* order;          // rows in the order they are taken, those that are kept first; null: as they lie
  const int32_t* kept;           // how many those are
  float* out;                    // sums of the terms, or null
  int n_out;
  int* done;
  int* status;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// Whether the phase is over, without waiting (the lanes of a warp look at barriers of their own).
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
               "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}

// Hands 16 bytes to CTA `to` of the cluster, at the place of `slot` here, and tells the barrier there.  (A plain store with a releasing
// arrival would first wait for the thread's gradient stores to reach memory.)
__device__ __forceinline__ void send(uint32_t slot, uint32_t bar, int to, float4 v) {
  asm volatile("{\n\t.reg .b32 rs, rb;\n\t"
               "mapa.shared::cluster.u32 rs, %0, %2;\n\t"
               "mapa.shared::cluster.u32 rb, %1, %2;\n\t"
               "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [rs], {%3, %4, %5, %6}, [rb];\n\t}"
               ::"r"(slot), "r"(bar), "r"(to), "r"(__float_as_uint(v.x)), "r"(__float_as_uint(v.y)), "r"(__float_as_uint(v.z)),
               "r"(__float_as_uint(v.w)) : "memory");
}

// Bounded like every wait of the library, with acquire at cluster scope: the data came from a peer's store.
__device__ __forceinline__ void wait_peers(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
  long long t0 = 0;
  while (true) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok || *abort_flag != 0) return;
    if (t0 == 0) t0 = clock64();
    else if (clock64() - t0 > kWaitLimitCycles) { *abort_flag = 59; atomicCAS(status, 0, 59); return; }
  }
}

template <typename T>
struct Lane;   // the maximum of vectors in memory
template <>
struct Lane<__nv_bfloat16> {
  static constexpr uint32_t kMasked = 0xff80ff80u;   // -inf
  template <int CV>
  static __device__ __forceinline__ float max_of(const Vec16<__nv_bfloat16> (&v)[CV]) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v[0].raw);
    __nv_bfloat162 m[4] = {h[0], h[1], h[2], h[3]};
#pragma unroll
    for (int j = 1; j < CV; ++j) {
      const __nv_bfloat162* g = reinterpret_cast<const __nv_bfloat162*>(&v[j].raw);
#pragma unroll
      for (int i = 0; i < 4; ++i) m[i] = __hmax2(m[i], g[i]);
    }
    const __nv_bfloat162 r = __hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3]));
    return fmaxf(__low2float(r), __high2float(r));
  }
};
template <>
struct Lane<float> {
  static constexpr uint32_t kMasked = 0xff800000u;
  template <int CV>
  static __device__ __forceinline__ float max_of(const Vec16<float> (&v)[CV]) {
    float4 m = v[0].raw;
#pragma unroll
    for (int j = 1; j < CV; ++j) {
      m.x = fmaxf(m.x, v[j].raw.x); m.y = fmaxf(m.y, v[j].raw.y);
      m.z = fmaxf(m.z, v[j].raw.z); m.w = fmaxf(m.w, v[j].raw.w);
    }
    return fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w));
  }
};

__device__ __forceinline__ void tmem_ld_wait_on16(uint32_t (&r)[16]) {   // no use of r moves above it
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :: "memory");
}

// (m, s) of a warp's first `lanes` lanes, a power of two (the others hold nothing: -inf, 0): the same in those lanes
__device__ __forceinline__ void warp_combine(float& m, float& s, float k, int lanes = 32) {
  const float top = warp_max(m);
  s = m == -INFINITY ? s : s * ex2((m - top) * k);   // (nothing kept: 0, or NaN if it holds one)
  for (int o = lanes >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
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
  uint32_t special;  // bit c: chunk c holds the target, is not full, or has vectors that are not the row's alone; kEdges: the share has such
  int state;         // 0: to be computed, 1: left out, 2: out of range
  RowInputs in;
};
// SAME: every row of the gradient lies as its logits do relative to 16 bytes, so that whole vectors can be written.
template <typename T, int OP, bool SAME>
__global__ void __launch_bounds__(kAllThreads, 1)
token_resident_kernel(const RowArgs a, const Resident p) {
  using VT = Vec16<T>;
  using Raw = decltype(VT::raw);
  constexpr int N = VT::N, CV = kChunk / N, kLogCv = CV == 4 ? 2 : 3;   // vectors of a chunk
  static_assert(CV == 1 << kLogCv, "chunks of a power of two");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kWarps][kMaxPieces], empty[kWarps][kMaxPieces], slot_bars[kWarps][2], t_full[2][2], t_empty[2][2];
  __shared__ __align__(16) float4 slots[kWarps / 2][2][8];   // by group, parity and CTA: (maximum, sum, target's logit or loss, whose target it is)
  __shared__ __align__(16) float4 row_end[kWarps / 2][2];    // what the second sweep needs: by group and parity
  __shared__ float2 red[2][kWarps];
  __shared__ float edge[kWarps][2][2 * N];                   // the share's elements in vectors that are not the row's alone
  __shared__ float target_logit[kWarps][2];
  __shared__ float refs[kTmemChunks][kThreads];              // what the chunks in tensor memory are relative to
  __shared__ int repeats[kWarps][2];                         // whether an id came twice among the row's teacher entries
  __shared__ __align__(16) float4 teachers[kWarps][2];       // its share of the loss, x_ref, whether it has no entry that counts
  __shared__ int abort_word, last;
  __shared__ uint32_t tmem_base;
  volatile int* abort_flag = &abort_word;
  cg::cluster_group cl = cg::this_cluster();
  const int ctas = p.ctas, rank = static_cast<int>(cl.block_rank());
  const int groups = 1 << p.log_groups, log_gd = 9 - p.log_groups, gd = 1 << log_gd;   // threads a group
  const int lane = threadIdx.x & 31, warp = static_cast<int>(threadIdx.x) >> 5;
  const bool serves = warp >= kWarps;
  const int group = serves ? 0 : static_cast<int>(threadIdx.x) >> log_gd;
  const int tid = serves ? threadIdx.x : threadIdx.x & (gd - 1);   // the thread within its group (those that serve are in none)
  const int first = ((static_cast<int>(blockIdx.x) >> p.log_ctas) << p.log_groups) + group;
  const int step = (static_cast<int>(gridDim.x) >> p.log_ctas) << p.log_groups;
  const int piece_bytes = CV * 16 * gd;
  // dynamic shared memory: the rows' descriptors, the rings, and (distillation) each group's teacher entries and bitmaps of ids, by parity
  RowInfo* infos = reinterpret_cast<RowInfo*>(smem) + group * (kInfoRows >> p.log_groups);
  const int info_rows = kInfoRows >> p.log_groups;
  uint8_t* ring = smem + kInfoRows * sizeof(RowInfo) + group * p.pieces * piece_bytes;
  const int bit_words = kMaxChunks * kChunk * gd / 32;
  uint8_t* teacher_smem = smem + kInfoRows * sizeof(RowInfo) + groups * p.pieces * piece_bytes;
  struct Taught { int* id; float *q, *x; uint32_t* bits; };   // entries: column in the share or -1, probability, student's logit; ids seen
  auto taught = [&](int g, int parity) {
    uint8_t* at = teacher_smem + g * (24 * a.K + 8 * bit_words);
    Taught t;
    t.id = reinterpret_cast<int*>(at) + parity * a.K;
    t.q = reinterpret_cast<float*>(at + 8 * a.K) + parity * a.K;
    t.x = reinterpret_cast<float*>(at + 16 * a.K) + parity * a.K;
    t.bits = reinterpret_cast<uint32_t*>(at + 24 * a.K) + parity * bit_words;
    return t;
  };
  const uint32_t full0 = smem_u32(full[group]), empty0 = smem_u32(empty[group]);
  auto group_sync = [&]() {
    if (p.group_warps == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(gd) : "memory");
  };
  if (threadIdx.x == 0) *abort_flag = 0;
  if (tid == 0) {
    for (int i = 0; i < p.pieces; ++i) { mbar_init(full0 + 8 * i, 1); mbar_init(empty0 + 8 * i, p.group_warps); }
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&slot_bars[group][i]), 1);
    if (group < 2)
      for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&t_full[group][i]), 1); mbar_init(smem_u32(&t_empty[group][i]), p.group_warps); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
  }
  if constexpr (OP == kDistill)
    for (int i = tid; i < 2 * bit_words && !serves; i += gd) taught(group, 0).bits[i] = 0;
  if (ctas > 1) cl.sync(); else __syncthreads();   // every CTA's barriers exist before a peer arrives on them
  grid_dependency_wait();
  if (p.tmem) {
    if (warp == 0) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(512u) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
  }
  grid_launch_dependents();
  // a warp reaches the 32 lanes of its place among four; the warps that share them have 128 columns each
  const uint32_t tmem = p.tmem ? tmem_base + (static_cast<uint32_t>(warp & 3) << 21) + (warp >> 2) * (kTmemChunks * kChunk) : 0;

  const uint32_t M = static_cast<uint32_t>(a.M);
  const uint32_t kept = p.kept != nullptr ? static_cast<uint32_t>(*from_here(p.kept)) : M;
  auto row_of = [&](uint32_t i) -> int { return p.order != nullptr ? from_here(p.order)[i] : static_cast<int>(i); };
  auto state_of = [&](uint32_t i, int row) {   // 0: to be computed, 1: left out, 2: out of range
    if (i >= kept) return 1;
    if (OP == kDistill) return p.order == nullptr && a.weight[row] == 0.0f ? 1 : 0;
    const int t = read_target(a.targets, a.target_bytes, a.has_ignore, a.ignore, row, a.V);
    return t >= 0 ? 0 : t == -2 ? 2 : 1;
  };
  auto chunks_of = [&](int n) { return max(1, (n + CV * gd - 1) >> (kLogCv + log_gd)); };

  // Distillation: a row's teacher, by one warp: q = softmax(t / T) over its entries, those with -inf counting for nothing; of the entries
  // whose column is in this share where it is (or -1), q and the student's logit; and the sum of q (log q - (x - x_ref) / T) over
  // them, with x_ref the largest of the student's logits among all entries: no difference is positive, so that a forbidden token's
  // loss may be infinite but nothing infinite cancels.
  auto teach = [&](int g, int row, const Share& s, int into) {
    const int64_t t0 = static_cast<int64_t>(row) * a.K;
    const T* x_row = static_cast<const T*>(a.logits) + row_offset(a, row);
    const Taught at = taught(g, into);
    auto id_of = [&](int64_t id) { return id >= 0 && id < a.V ? static_cast<int>(id) : -1; };
    float tm = -INFINITY, ts = 0.0f, x_ref = -INFINITY;
#pragma unroll 2
    for (int q = lane; q < a.K; q += 32) {   // (loads of the student's logits that another CTA has are the same ones it makes)
      const float t = read_teacher(a, t0 + q);
      const int id = id_of(read_teacher_id(a, t0 + q));
      const float x = id >= 0 ? to_f32(x_row[id]) : -INFINITY;
      at.x[q] = x;
      x_ref = fmaxf(x_ref, x);
      at.id[q] = id;
      at.q[q] = t;
      tm = fmaxf(tm, t);
    }
    tm = warp_max(tm);
    x_ref = warp_max(x_ref);
    if (!(fabsf(x_ref) < INFINITY)) x_ref = 0.0f;
    const float tref = tm == -INFINITY ? 0.0f : tm;
    for (int q = lane; q < a.K; q += 32) ts += ex2((at.q[q] - tref) * a.k);
    ts = warp_sum(ts);
    const float inv_ts = ts == 0.0f ? 0.0f : 1.0f / ts, log_ts = logf(ts);
    float loss = 0.0f;
    bool twice = false;
    for (int q = lane; q < a.K; q += 32) {
      const float d = at.q[q] - tref, prob = ex2(d * a.k) * inv_ts;   // log q = d / T - log_ts
      const int id = at.id[q];
      int el = -1;
      if (prob != 0.0f) {   // (NaN counts)
        if (id < 0) {
          loss = NAN;
        } else if (id - s.column >= s.lo && id - s.column < s.hi) {
          el = id - s.column;
          loss += prob * ((d * a.inv_t - log_ts) - (at.x[q] - x_ref) * a.inv_t);
          twice |= atomicOr(at.bits + (el >> 5), 1u << (el & 31)) >> (el & 31) & 1u;
        }
      }
      at.id[q] = el;
      at.q[q] = prob;
    }
    loss = warp_sum(loss);
    twice = __any_sync(0xffffffffu, twice);
    if (lane == 0) { teachers[g][into] = make_float4(loss, x_ref, ts == 0.0f ? 1.0f : 0.0f, 0.0f); repeats[g][into] = twice; }
    __syncwarp();
  };
  // The gradient of a row's teacher columns, over what the second sweep wrote there, by threads t of n; clears their bits.
  auto teacher_columns = [&](int g, int from, const Share& s, float4 row_end, int t, int n) {
    const Taught at = taught(g, from);
    const bool twice = repeats[g][from] != 0;
    T* to = static_cast<T*>(a.grad) + s.to;
    for (int q = t; q < a.K; q += n) {
      const int el = at.id[q];
      if (el < s.lo || el >= s.hi) continue;   // -1; or what an abandoned wait left there
      at.bits[el >> 5] = 0;
      if (a.grad == nullptr) continue;
      float prob = at.q[q];
      bool mine = true;
      if (twice) {   // the first of those that name the same column writes the sum of them
        prob = 0.0f;
        for (int o = 0; o < a.K; ++o) {
          if (at.id[o] != el) continue;
          if (o < q) { mine = false; break; }
          prob += at.q[o];
        }
      }
      if (mine) to[el] = from_f32<T>(row_end.z * (exp2f((at.x[q] - row_end.y) * a.k) / row_end.w - prob));
    }
  };
  // Serving warps do both where an SM has few rows in flight, one for each group: the teacher's part up to two rows ahead, and its columns
  // when every warp has written its part of the row (by the row's own warps behind a barrier: 2048 x 151936 bf16 287 us, so 278).
  // More groups hide their own.
  const bool taught_ahead = OP == kDistill && groups <= 2;

  if (serves) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kServeRegs));
    if (warp == kWarps) {
      // Lane g feeds group g's ring: pieces in the order they are taken, each when every warp has left the slot it goes to.
      uint32_t fed = ((blockIdx.x >> p.log_ctas) << p.log_groups) + lane;   // the place of the row
      bool active = lane < groups && fed < kept;
      const int g = lane & (kWarps - 1);
      const T* from = nullptr;
      int left = -1, slot = 0;   // vectors of the row's share that have not been fed; -1: the row has not been begun
      uint32_t phase = 1;
      long long idle = 0;
      while (__any_sync(0xffffffffu, active)) {
        bool moved = false;
        if (active && left < 0) {
          const int row = row_of(fed);
          if (state_of(fed, row) == 0) {
            const Share s = share_of<N>(a, p, rank, row);
            from = static_cast<const T*>(a.logits) - p.mis + s.from;
            left = s.n;
          } else {
            fed += step;
            active = fed < kept;
          }
          moved = true;
        }
        if (active && left >= 0 && mbar_test(smem_u32(&empty[g][slot]), phase)) {
          const uint32_t bar = smem_u32(&full[g][slot]);
          const int n = min(left, CV * gd);
          mbar_expect_tx(bar, n * 16);   // a piece with nothing in it completes at once
          if (n > 0)
            bulk_load(smem_u32(smem) + kInfoRows * static_cast<uint32_t>(sizeof(RowInfo)) + (g * p.pieces + slot) * piece_bytes, from, n * 16, bar);
          from += n * N;
          left -= n;
          if (++slot == p.pieces) { slot = 0; phase ^= 1; }
          if (left == 0) { left = -1; fed += step; active = fed < kept; }
          moved = true;
        }
        if (__any_sync(0xffffffffu, moved)) { idle = 0; continue; }
        const long long now = clock64();
        if (idle == 0) idle = now;
        else if (now - idle > kWaitLimitCycles) { *abort_flag = 55; atomicCAS(p.status, 0, 55); }
        if (__any_sync(0xffffffffu, *abort_flag != 0)) break;   // (all lanes or none)
      }
      __syncwarp();
    } else if (taught_ahead && warp - kWarps - 1 < groups) {
      const int g = warp - kWarps - 1;
      uint32_t parity = 1;
      int into = 0, rows[2] = {-1, -1};   // by parity: whose entries these are
      auto end_row = [&]() {   // waits for the row that has them, if any, and writes its columns
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&t_empty[g][into]), parity, abort_flag, 57, p.status))) return false;
        const int before = into == 0 ? rows[0] : rows[1];
        if (before >= 0) teacher_columns(g, into, share_of<N>(a, p, rank, before), row_end[g][into], lane, 32);
        __syncwarp();
        return true;
      };
      bool ok = true;
      for (uint32_t i = ((blockIdx.x >> p.log_ctas) << p.log_groups) + g; i < kept && ok; i += step) {
        const int row = row_of(i);
        if (state_of(i, row) != 0) continue;
        ok = end_row();
        if (!ok) break;
        teach(g, row, share_of<N>(a, p, rank, row), into);
        if (lane == 0) mbar_arrive(smem_u32(&t_full[g][into]));
        if (into == 0) rows[0] = row; else rows[1] = row;
        if (++into == 2) { into = 0; parity ^= 1; }
      }
      for (int q = 0; q < 2 && ok; ++q) {
        ok = end_row();
        if (++into == 2) { into = 0; parity ^= 1; }
      }
      __syncwarp();
    }
  } else {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegs));

  uint32_t phase = 0, slot_phase = 0, t_phase = 0;   // parities of the ring's current round, (bit i) of slot barrier i, of the teacher's
  int slot = 0, par = 0, at = info_rows;
  for (uint32_t i = first; i < M; i += step, ++at) {   // (M and the step are below 2^31)
    if (at == info_rows) {
      group_sync();   // the last of them is done with
      for (int q = tid; q < info_rows; q += gd) {
        const uint32_t iq = i + static_cast<uint32_t>(q) * step;   // (kInfoRows steps are few)
        if (iq < M && iq >= i) {
          RowInfo f;
          f.row = row_of(iq);
          f.share = share_of<N>(a, p, rank, f.row);
          f.state = state_of(iq, f.row);
          f.target = -1;
          if constexpr (OP != kDistill) {
            if (f.state == 0) {
              const int t = read_target(a.targets, a.target_bytes, a.has_ignore, a.ignore, f.row, a.V) - f.share.column;
              if (t >= f.share.lo && t < f.share.hi) f.target = t;
            }
          }
          f.special = 0;
          const int per = CV * N << log_gd;   // elements of a chunk
          if (f.target >= 0) f.special |= 1u << (f.target / per);
          if (f.share.n * N % per != 0 || f.share.n == 0) f.special |= 1u << (chunks_of(f.share.n) - 1);
          if (f.share.lo > 0 || f.share.hi < f.share.n * N) f.special |= kEdges | 1u | 1u << (chunks_of(f.share.n) - 1);
          f.in = row_inputs<OP>(a, f.row);
          infos[q] = f;
        }
      }
      group_sync();
      at = 0;
    }
    const RowInfo& info = infos[at];
    if (info.state != 0) {   // the same in every CTA of the cluster
      const float value = info.state == 2 ? NAN : 0.0f;
      if (rank == 0 && tid == 0) write_left_out<OP>(a, info.row, value, nullptr);
      if (a.grad != nullptr) {
        const Share& s = info.share;
        T* g = static_cast<T*>(a.grad) + s.to;
        if (SAME) {
          VT z;
          float f[N];
#pragma unroll
          for (int j = 0; j < N; ++j) f[j] = value;
          z.from_float(f);
          for (int vi = s.fa + tid; vi < s.fb; vi += gd) __stcs(reinterpret_cast<Raw*>(g) + vi, z.raw);
          for (int e = s.lo + tid; e < min(s.fa * N, s.hi); e += gd) g[e] = from_f32<T>(value);
          for (int e = s.fb * N + tid; e < s.hi; e += gd) g[e] = from_f32<T>(value);
        } else {
          for (int e = s.lo + tid; e < s.hi; e += gd) g[e] = from_f32<T>(value);
        }
      }
      continue;
    }
    float third = 0.0f;
    if constexpr (OP == kDistill) {
      if (!taught_ahead) {
        if (tid < 32) teach(group, info.row, info.share, par);
        group_sync();
      }
    }
    // first sweep
    const bool own = info.target >= 0;
    float m = -INFINITY, sw = 0.0f, e[kChunk];
    const int chunks = chunks_of(info.share.n);
    const float2 kk = make_float2(a.k, a.k);
    // A chunk on its way into registers; the return value is its largest logit.
    auto fetch = [&](int c, VT (&raw)[CV]) {
      const Raw* srow = reinterpret_cast<const Raw*>(ring + slot * piece_bytes) + tid;
      mbar_wait(full0 + 8 * slot, phase, abort_flag, 56, p.status);
      if (!(info.special >> c & 1u)) {
#pragma unroll
        for (int j = 0; j < CV; ++j) raw[j].raw = srow[j << log_gd];
      } else {
        const Share& s = info.share;
        const int v0 = c << (kLogCv + log_gd), n = min(s.n - v0, CV * gd), e0 = v0 * N;   // the chunk's vectors begin at v0, its elements at e0
        T* selem = reinterpret_cast<T*>(ring + slot * piece_bytes);
        const int tl = info.target - e0;
        if (own && tl >= 0 && tl < n * N) {
          if (((tl / N) & (gd - 1)) == tid) {
            target_logit[group][par] = to_f32(selem[tl]);
            selem[tl] = from_f32<T>(-INFINITY);
            fence_proxy_async_smem();   // the slot's next copy comes behind these stores
          }
        }
        if (info.special & kEdges) {
          bool patched = false;
          if (c == 0 && s.lo > 0 && tid == 0) {
            for (int q = 0; q < s.lo; ++q) selem[q] = from_f32<T>(-INFINITY);
            patched = true;
          }
          if (s.hi < s.n * N && s.n - 1 >= v0 && s.n - 1 < v0 + CV * gd && ((s.n - 1) & (gd - 1)) == tid) {
            for (int q = s.hi; q < s.n * N; ++q) selem[q - e0] = from_f32<T>(-INFINITY);
            patched = true;
          }
          if (patched) fence_proxy_async_smem();
          if (tid < 2 * N) {   // the row's elements in those vectors are written one by one
            const int el = tid < N ? s.lo + tid : s.fb * N + tid - N;
            if (el >= e0 && el < e0 + n * N && (tid < N ? el < min(s.fa * N, s.hi) : el < s.hi)) edge[group][par][tid] = to_f32(selem[el - e0]);
          }
        }
#pragma unroll
        for (int j = 0; j < CV; ++j) {
          uint32_t* w = reinterpret_cast<uint32_t*>(&raw[j].raw);
          w[0] = w[1] = w[2] = w[3] = Lane<T>::kMasked;
          if (j * gd + tid < n) raw[j].raw = srow[j << log_gd];
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty0 + 8 * slot);   // the warp has taken what it needs of the slot
      if (++slot == p.pieces) { slot = 0; phase ^= 1; }
      return Lane<T>::max_of(raw);
    };
    // Its exponentials, relative to the thread's largest logit so far, m.
    auto exponentials = [&](const VT (&raw)[CV], float cm, float (&x)[kChunk], int n = 1 << 20) {   // n: the chunk's vectors, if it may not be full
      const float mm = fmaxf(m, cm);
      const float r = mm == -INFINITY ? 0.0f : mm;
      sw *= ex2((fmaxf(m, -FLT_MAX) - r) * a.k);   // (nothing summed yet: 0, or NaN, times at most 1)
      m = mm;
      const float2 neg_m = make_float2(-r, -r);
      float2 s2 = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < CV; ++j) {
        if (j > 0 && (j << log_gd) >= n) {   // nobody has one (the last chunk)
#pragma unroll
          for (int q = 0; q < N; ++q) x[j * N + q] = 0.0f;
          continue;
        }
        float f[N];
        raw[j].to_float(f);
#pragma unroll
        for (int q = 0; q < N; q += 2) {
          const float2 d = __fmul2_rn(__fadd2_rn(make_float2(f[q], f[q + 1]), neg_m), kk);
          const float2 y = make_float2(ex2(d.x), ex2(d.y));
          s2 = __fadd2_rn(s2, y);
          x[j * N + q] = y.x; x[j * N + q + 1] = y.y;
        }
      }
      sw += s2.x + s2.y;
    };
    auto keep = [&](int c, const float (&x)[kChunk]) {   // in tensor memory
      refs[c][threadIdx.x] = m;
      uint32_t half[2][16];
#pragma unroll
      for (int q = 0; q < 16; ++q) { half[0][q] = __float_as_uint(x[q]); half[1][q] = __float_as_uint(x[16 + q]); }
      tmem_st_x16(tmem + c * kChunk, half[0]);
      tmem_st_x16(tmem + c * kChunk + 16, half[1]);
    };
    // the next chunk is fetched before this one's arithmetic, where there are registers for two
    VT raw[CV];
    float cm;
    if constexpr (sizeof(T) == 2) {
      cm = fetch(0, raw);
      VT next[CV];
      float next_cm;
      int c = 0;
#pragma unroll 1
      for (; c + 2 < chunks; c += 2) {
        float x[kChunk];
        next_cm = fetch(c + 1, next);
        exponentials(raw, cm, x);
        keep(c, x);
        cm = fetch(c + 2, raw);
        exponentials(next, next_cm, x);
        keep(c + 1, x);
      }
      if (c + 1 < chunks) {
        float x[kChunk];
        next_cm = fetch(c + 1, next);
        exponentials(raw, cm, x);
        keep(c, x);
#pragma unroll
        for (int j = 0; j < CV; ++j) raw[j] = next[j];
        cm = next_cm;
      }
    } else {
#pragma unroll 1
      for (int c = 0; c < chunks - 1; ++c) {
        float x[kChunk];
        cm = fetch(c, raw);
        exponentials(raw, cm, x);
        keep(c, x);
      }
      cm = fetch(chunks - 1, raw);
    }
    exponentials(raw, cm, e, info.share.n - ((chunks - 1) << (kLogCv + log_gd)));
    const float ref_e = m;
    float mw = m;
    warp_combine(mw, sw, a.k);
    if (chunks > 1) tmem_st_wait();
    if (p.group_warps > 1) {
      if (lane == 0) red[par][warp] = make_float2(mw, sw);
      group_sync();
      if (tid < 32) {
        const float2 r = lane < p.group_warps ? red[par][group * p.group_warps + lane] : make_float2(-INFINITY, 0.0f);
        mw = r.x; sw = r.y;
        warp_combine(mw, sw, a.k, p.group_warps);
      }
    } else {
      __syncwarp();
    }
    if constexpr (OP == kDistill) {
      if (taught_ahead) {
        mbar_wait(smem_u32(&t_full[group][par]), t_phase, abort_flag, 57, p.status);
        t_phase ^= par;   // (both have been waited for)
      }
    }
    if constexpr (OP == kDistill) third = teachers[group][par].x;
    else if (own) third = target_logit[group][par];
    const int row = info.row;
    const bool writes = rank == 0 && tid == 0;
    float f_top, top, c0, at_target = 0.0f;   // an element's gradient is f_top 2^((x - top) k)
    // The group's first warp meets the other CTAs' and works out the row's coefficient; the others wait for it.
    if (tid < 32) {
      if (ctas > 1) {
        // Thread q hands this CTA's part to CTA q.  A slot is written again two rows later, when its readers have passed the
        // exchange in between.
        const uint32_t to = smem_u32(&slots[group][par][rank]), bar = smem_u32(&slot_bars[group][par]);
        if (tid == 0) mbar_expect_tx(bar, ctas * 16);
        if (tid < ctas) send(to, bar, tid, make_float4(mw, sw, third, own ? 1.0f : 0.0f));
        wait_peers(bar, (slot_phase >> par) & 1u, abort_flag, p.status);
        slot_phase ^= 1u << par;
        const float4 r = lane < ctas ? slots[group][par][lane] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        mw = r.x; sw = r.y;
        warp_combine(mw, sw, a.k, ctas);
        if constexpr (OP == kDistill) {
          third = warp_sum(r.z);
        } else {
          const uint32_t who = __ballot_sync(0xffffffffu, r.w != 0.0f);
          third = __shfl_sync(0xffffffffu, r.z, who == 0 ? 0 : __ffs(who) - 1);
        }
      }
      if constexpr (OP == kDistill) {
        const float w = info.in.weight;
        top = mw == -INFINITY ? 0.0f : mw;
        const bool empty_teacher = teachers[group][par].z != 0.0f;
        const float loss = empty_teacher ? 0.0f : third + ((top - teachers[group][par].y) * a.inv_t + logf(sw));
        if (writes) a.terms[row] = w * (a.temperature * a.temperature) * loss;
        c0 = empty_teacher ? 0.0f : w * a.temperature + (isnan(loss) ? NAN : 0.0f);
        f_top = empty_teacher ? 0.0f : c0 / sw;
      } else {
        const TargetStats r = target_stats(mw, sw, third, a.k);
        const RowResult out = finish_target_row<OP>(a, info.in, r);
        if (writes) write_target_row<OP>(a, row, r, out, nullptr);
        c0 = out.c;
        at_target = c0 * r.rest;
        f_top = -c0 / r.sum;
        top = r.top == -INFINITY ? 0.0f : r.top;
      }
    }
    if (p.group_warps > 1) {
      if (tid == 0) row_end[group][par] = make_float4(f_top, top, OP == kDistill ? c0 : at_target, sw);
      group_sync();
      const float4 r = row_end[group][par];
      f_top = r.x; top = r.y; sw = r.w;
      if constexpr (OP == kDistill) c0 = r.z; else at_target = r.z;
    }
    // second sweep
    if (a.grad != nullptr) {
      const Share& s = info.share;
      T* g = static_cast<T*>(a.grad) + s.to;
      // vectors j0 .. j0 + count of chunk c, from their exponentials times f
      auto put = [&](int c, int j0, const float* x, int count, float f) {
        const float2 ff = make_float2(f, f);
        const int v0 = c << (kLogCv + log_gd);
        Raw* to = reinterpret_cast<Raw*>(g) + v0 + tid;
        auto scaled = [&](int j) {
          VT t;
          float y[N];
#pragma unroll
          for (int q = 0; q < N; q += 2) {
            const float2 z = __fmul2_rn(make_float2(x[j * N + q], x[j * N + q + 1]), ff);
            y[q] = z.x; y[q + 1] = z.y;
          }
          t.from_float(y);
          return t;
        };
        if (SAME && v0 >= s.fa && v0 + CV * gd <= s.fb) {   // all of the chunk's vectors are the row's alone
#pragma unroll
          for (int j = 0; j < count; ++j) __stcs(to + ((j0 + j) << log_gd), scaled(j).raw);
          return;
        }
#pragma unroll
        for (int j = 0; j < count; ++j) {
          if (j > 0 && v0 + ((j0 + j) << log_gd) >= s.fb) break;
          const VT t = scaled(j);
          const int vi = v0 + ((j0 + j) << log_gd) + tid;
          if (vi >= s.fa && vi < s.fb) {
            if (SAME) {
              __stcs(to + ((j0 + j) << log_gd), t.raw);
            } else {
              const T* y = reinterpret_cast<const T*>(&t.raw);
#pragma unroll
              for (int q = 0; q < N; ++q) g[vi * N + q] = y[q];
            }
          }
        }
      };
      auto factor = [&](float r) {   // (-inf: the thread has seen masked logits only, whose exponentials are zeros, or NaN)
        return r == -INFINITY ? f_top : f_top * ex2((r - top) * a.k);
      };
      // half a chunk is on its way from tensor memory while the one before is written
      uint32_t w0[16], w1[16];
      float x[16];
      if (chunks > 1) tmem_ld_x16(tmem, w0);
      put(chunks - 1, 0, e, CV, factor(ref_e));
#pragma unroll 1
      for (int c = 0; c < chunks - 1; ++c) {
        const float f = factor(refs[c][threadIdx.x]);
        tmem_ld_wait_on16(w0);
        tmem_ld_x16(tmem + c * kChunk + 16, w1);
#pragma unroll
        for (int q = 0; q < 16; ++q) x[q] = __uint_as_float(w0[q]);
        put(c, 0, x, CV / 2, f);
        tmem_ld_wait_on16(w1);
        if (c + 1 < chunks - 1) tmem_ld_x16(tmem + (c + 1) * kChunk, w0);
#pragma unroll
        for (int q = 0; q < 16; ++q) x[q] = __uint_as_float(w1[q]);
        put(c, CV / 2, x, CV / 2, f);
      }
      const int tl = info.target;
      if (OP != kDistill && own) {
        const int tv = tl / N;
        if (tv >= s.fa && tv < s.fb && (tv & (gd - 1)) == tid) g[tl] = from_f32<T>(at_target);   // behind this thread's own vector
      }
      if ((info.special & kEdges) && tid < 2 * N) {
        const int el = tid < N ? s.lo + tid : s.fb * N + tid - N;
        if (tid < N ? el < min(s.fa * N, s.hi) : el < s.hi)
          g[el] = from_f32<T>(el == tl ? at_target : f_top * ex2((edge[group][par][tid] - top) * a.k));
      }
    }
    if constexpr (OP == kDistill) {
      if (taught_ahead) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&t_empty[group][par]));   // this warp has written its part
      } else {
        group_sync();   // the row's softmax is written
        teacher_columns(group, par, info.share, make_float4(f_top, top, c0, sw), tid, gd);
        if (p.group_warps == 1) __syncwarp();   // (these entries are made again behind the next row's first barrier)
      }
    }
    par ^= 1;
  }
  }   // (not the serving warps)
  tcgen05_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    for (int q = 0; q < 200; ++q) __nanosleep(1000);   // loads in flight land before the shared memory is released
  }
  if (p.tmem && warp == 0) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
  if (ctas > 1) cl.sync();   // no peer still writes here
  if (OP != kUnit && p.out != nullptr && rank == 0) {
    // the last cluster to finish sums what all have left, in one order whichever it is
    if (threadIdx.x == 0) {
      __threadfence();
      last = atomicAdd(p.done, 1) == (static_cast<int>(gridDim.x) >> p.log_ctas) - 1;
    }
    __syncthreads();
    if (last) {
      __threadfence();
      block_sums<kAllThreads>(a.terms, a.M, 1, a.M, p.n_out, p.out, reinterpret_cast<double*>(smem));
    }
  }
}

template <typename T, int OP>
int launch_resident(const RowArgs& a, const RowPlan& plan, DeviceState* ds, cudaStream_t st, bool* taken) {
  constexpr int N = Vec16<T>::N, CV = kChunk / N;
  *taken = false;
  const uintptr_t ai = reinterpret_cast<uintptr_t>(a.logits), ag = reinterpret_cast<uintptr_t>(a.grad);
  const int64_t vecs = (static_cast<int64_t>(a.V) + 2 * N - 2) / N;   // that cover a row at most
  Resident p;
  p.log_ctas = 0; p.group_warps = 1;
  auto fits = [&]() { return (vecs + (1 << p.log_ctas) - 1) >> p.log_ctas <= static_cast<int64_t>(kMaxChunks) * CV * 32 * p.group_warps; };
  // As few CTAs a row as can hold it, then as few warps: a row's exchange costs more than the rows in flight gain
  // (2048 x 151936 bf16 over 8 CTAs with four rows in flight 345 us, over 4 with two 324, over 2 with one 292; 4000 x 32000 over 2 and four
  // 144 us, by one CTA with two 115, with one 138).
  while (!fits()) {
    if (p.group_warps < kWarps) p.group_warps *= 2;
    else if (p.log_ctas < 3) ++p.log_ctas;
    else return MCB_OK;
  }
  // Few rows: more of the SMs for each, first a whole SM (down to two vectors a thread), then a cluster (down to four).
  while (true) {
    const int64_t busy = (a.M * p.group_warps + kWarps - 1) / kWarps << p.log_ctas;
    const int64_t each = vecs / (static_cast<int64_t>(p.group_warps) * 32 << p.log_ctas);   // vectors a thread
    if (2 * busy > ds->sm_count) break;
    if (p.group_warps < kWarps && each >= 4) p.group_warps *= 2;
    else if (p.group_warps == kWarps && p.log_ctas < 3 && each >= 8) ++p.log_ctas;
    else break;
  }
  p.tmem = (vecs + (1 << p.log_ctas) - 1) >> p.log_ctas > static_cast<int64_t>(CV) * 32 * p.group_warps;
  p.ctas = 1 << p.log_ctas;
  p.log_groups = 0;
  while ((kWarps / p.group_warps) >> (p.log_groups + 1)) ++p.log_groups;
  p.mis = static_cast<int>((ai & 15u) / sizeof(T));
  p.order = plan.order; p.kept = plan.kept; p.out = plan.sums; p.n_out = plan.n_sums; p.done = plan.done; p.status = ds->status_word;
  const int64_t fixed = kInfoRows * sizeof(RowInfo), most = 210 * 1024;
  const int64_t slot = static_cast<int64_t>(kThreads) * kChunk * sizeof(T);   // one ring slot of every group
  auto teacher = [&]() { return OP == kDistill ? (kWarps / p.group_warps) * (24 * static_cast<int64_t>(a.K) + 8 * kMaxChunks * kChunk * p.group_warps) : 0; };
  while (fixed + teacher() + 2 * slot > most) {
    if (p.group_warps == kWarps) return MCB_OK;
    p.group_warps *= 2;
    --p.log_groups;
  }
  p.pieces = static_cast<int>((most - fixed - teacher()) / slot);
  p.pieces = p.pieces > kMaxPieces ? kMaxPieces : p.pieces < 2 ? 2 : p.pieces;
  int64_t smem = fixed + p.pieces * slot + teacher();
  if (smem < kSmem) smem = kSmem;
  const bool same = a.grad == nullptr || (((ai ^ ag) & 15u) == 0 && (a.token_stride - a.V) % N == 0 && (a.batch_stride - a.S * a.V) % N == 0);
  const auto kernel = same ? token_resident_kernel<T, OP, true> : token_resident_kernel<T, OP, false>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.ctas)); cfg.blockDim = dim3(kAllThreads); cfg.dynamicSmemBytes = static_cast<size_t>(smem); cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.ctas); attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  int resident = 0;   // clusters that the device runs at once, asked for once a cluster size (the query takes microseconds)
  {
    struct Known { const DeviceState* ds; int clusters[4]; };
    static std::mutex mu;
    static Known known[64][2];   // by place of first use; a device is known by its state
    std::lock_guard<std::mutex> lock(mu);
    Known* k = nullptr;
    for (int i = 0; i < 64 && k == nullptr; ++i)
      if (known[i][same].ds == ds || known[i][same].ds == nullptr) k = &known[i][same];
    if (k->ds == nullptr) {
      MCB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most)));
      MCB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
      k->ds = ds;
    }
    if (k->clusters[p.log_ctas] == 0) {
      int n = 0;
      MCB_CHECK_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
      k->clusters[p.log_ctas] = n > 0 ? n : 1;
    }
    resident = k->clusters[p.log_ctas];
  }
  // as many clusters as are resident together: a later one would start its share of the rows when the others are done
  const int64_t wanted = (a.M + (1 << p.log_groups) - 1) >> p.log_groups;
  cfg.gridDim = dim3(static_cast<unsigned>((wanted < resident ? wanted : resident) * p.ctas));
  if (chained_launch()) cfg.numAttrs = 2;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, a, p);
  if (err != cudaSuccess) return cuda_fail(err, "token_resident_kernel launch");
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
  return f32 ? launch_resident<float, kDistill>(a, plan, ds, st, taken) : launch_resident<__nv_bfloat16, kDistill>(a, plan, ds, st, taken);
}
}  // namespace tokenloss
}  // namespace mcb
