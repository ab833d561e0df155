// Embedding lookup with scaling, and the gradient of its table (beside mcb_embedding_fwd, whose table is frozen):
//   out[i] = scale table[ids[i]];   grad[v] = scale sum of dout[i] over ids[i] = v
// An id outside [0, vocab) (padding) gives a row of zeros and has no gradient.
//
// The gradient goes by sorted tokens: the ids are sorted once with their positions (stable, so a row's terms stay in token order), then
// every run of equal ids is one sum, held in registers and written once.  Nothing uses floating-point atomics: the same
// tokens give the same bits, and a token that comes a thousand times costs no more than a thousand different ones.
//   1. sort (one cluster): radix sort of ceil(log2(vocab + 1)) bits, up to 9 a pass.  A warp owns consecutive tokens; within 32 of them
//      equal digits are ranked by match; counts of digits go from warp to block to cluster through shared memory.  The launch's other
//      blocks write zeros meanwhile; the rest of the table's are written beside the sums, but for the rows that get one.
//   2. sums: a tile of 8 to 32 sorted tokens by as many threads as the columns take; a run that ends inside its tile is written out, one
//      that goes on leaves its part.  3. The tile where such a run begins adds up the parts, in order.
// HBM-bound by the table's gradient (float32, written whole) where it is not accumulated.
#include <cooperative_groups.h>

#include <type_traits>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace mcb {
namespace embed {
namespace {

constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32, kDigits = 512, kMaxTile = 32, kThreads = 128, kJoinThreads = 256, kZeroRows = 64;
constexpr int64_t kEarlyBytes = 64 << 20;   // of zeros beside the sort: about what its 10 us are enough for
constexpr uint32_t kFull = 0xffffffffu;

// ---- forward -----------------------------------------------------------------------------------------------------------
// `tx` threads share a row (16 bytes, or one element, at a time), kThreads / tx rows to a block.
template <typename T, typename I, int N>
__global__ void __launch_bounds__(kThreads) embed_fwd_kernel(const I* ids, const T* table, T* out, int64_t M, int64_t H, int64_t vocab, float scale, int tx) {
  grid_launch_dependents();
  grid_dependency_wait();
  ids = from_here(ids);
  table = from_here(table);
  const int x = threadIdx.x % tx, y = threadIdx.x / tx, rows = kThreads / tx;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * rows + y; row < M; row += static_cast<int64_t>(gridDim.x) * rows) {
    const int64_t id = static_cast<int64_t>(ids[row]);
    const bool have = id >= 0 && id < vocab;
    const T* src = table + (have ? id : 0) * H;
    for (int64_t c = N * static_cast<int64_t>(x); c < H; c += N * tx) {
      if constexpr (N == 1) {
        out[row * H + c] = have ? from_f32<T>(to_f32(src[c]) * scale) : from_f32<T>(0.0f);
      } else {
        Vec16<T> v;
        float f[N];
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = 0.0f;
        if (have) {
          v.raw = *reinterpret_cast<const decltype(v.raw)*>(src + c);
          v.to_float(f);
#pragma unroll
          for (int e = 0; e < N; ++e) f[e] *= scale;
        }
        v.from_float(f);
        *reinterpret_cast<decltype(v.raw)*>(out + row * H + c) = v.raw;
      }
    }
  }
}

// ---- sort ----------------------------------------------------------------------------------------------------------------
struct SortParams {
  const void* ids;
  uint32_t *key[2], *pos[2];   // the result of pass p is in buffer p & 1
  float* zero;                 // zeros for the blocks behind the cluster to write, zero_n elements
  int64_t zero_n;
  int64_t vocab;
  int M, passes, digit_bits;
};

template <typename I>
__device__ __forceinline__ uint32_t key_of(const SortParams& p, const uint32_t* before, int pass, int i) {
  if (pass > 0) return __ldcg(before + i);
  const int64_t id = static_cast<int64_t>(static_cast<const I*>(p.ids)[i]);
  return id >= 0 && id < p.vocab ? static_cast<uint32_t>(id) : static_cast<uint32_t>(p.vocab);   // the others behind all
}

// KEEP: a warp has at most KEEP x 32 tokens, and keeps keys, positions and ranks in registers between the two walks of a pass.
// 0: any number, read again.
template <typename I, int KEEP>
__global__ void __launch_bounds__(kSortThreads) sort_kernel(const __grid_constant__ SortParams p) {
  __shared__ uint32_t hist[kSortWarps][kDigits];   // of a warp: counts, then where its next token of a digit goes
  __shared__ uint32_t total[kDigits];              // of the block; read by the others of the cluster
  __shared__ uint32_t scan[kSortThreads / 32];
  cg::cluster_group cl = cg::this_cluster();
  const int C = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockIdx.x >= static_cast<unsigned>(C)) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int64_t n4 = p.zero_n >> 2, step = static_cast<int64_t>(gridDim.x - C) * kSortThreads;
    const int64_t at = static_cast<int64_t>(blockIdx.x - C) * kSortThreads + threadIdx.x;
    for (int64_t i = at; i < n4; i += step) __stcs(reinterpret_cast<float4*>(p.zero) + i, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    for (int64_t i = (n4 << 2) + at; i < p.zero_n; i += step) p.zero[i] = 0.0f;
    return;
  }
  const int warps = C * kSortWarps;
  const int per = ((p.M + warps - 1) / warps + 31) & ~31;   // tokens of a warp
  const int64_t begin = static_cast<int64_t>(rank * kSortWarps + warp) * per;
  const int end = static_cast<int>(begin + per < p.M ? begin + per : p.M);
  const int digits = 1 << p.digit_bits;
  for (int d = lane; d < digits; d += 32) hist[warp][d] = 0;
  grid_launch_dependents();
  grid_dependency_wait();
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.digit_bits;
    const uint32_t mask = static_cast<uint32_t>(digits) - 1u;
    const uint32_t *from_key = from_here(p.key[(pass + 1) & 1]), *from_pos = from_here(p.pos[(pass + 1) & 1]);   // what the pass before has left
    uint32_t key[KEEP + 1], at[KEEP + 1], before_me[KEEP + 1];
    // a walk over 32 tokens: counts their digits into the warp's, and says how many of its digit the warp has had before a token
    auto count = [&](uint32_t d, uint32_t have) -> uint32_t {
      const uint32_t peers = __match_any_sync(have, d), base = hist[warp][d];
      __syncwarp(have);
      if (lane == __ffs(peers) - 1) hist[warp][d] = base + __popc(peers);
      return base + __popc(peers & ((1u << lane) - 1u));
    };
    if constexpr (KEEP > 0) {
#pragma unroll
      for (int n = 0; n < KEEP; ++n) {
        const int64_t i = begin + 32 * n + lane;
        key[n] = at[n] = 0;
        if (i < end) {
          key[n] = key_of<I>(p, from_key, pass, static_cast<int>(i));
          at[n] = pass > 0 ? __ldcg(from_pos + i) : static_cast<uint32_t>(i);
        }
      }
#pragma unroll
      for (int n = 0; n < KEEP; ++n) {
        const bool in = begin + 32 * n + lane < end;
        const uint32_t have = __ballot_sync(kFull, in);
        if (in) before_me[n] = count((key[n] >> shift) & mask, have);
        __syncwarp();
      }
    } else {
      for (int64_t i0 = begin; i0 < end; i0 += 32) {
        const int i = static_cast<int>(i0) + lane;
        const uint32_t have = __ballot_sync(kFull, i < end);
        if (i < end) count((key_of<I>(p, from_key, pass, i) >> shift) & mask, have);
        __syncwarp();
      }
    }
    __syncthreads();
    // counts of the warps before, within the block; kDigits == kSortThreads: one digit a thread
    uint32_t sum = 0;
    if (static_cast<int>(threadIdx.x) < digits) {
      uint32_t n[kSortWarps];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) n[w] = hist[w][threadIdx.x];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        hist[w][threadIdx.x] = sum;
        sum += n[w];
      }
      total[threadIdx.x] = sum;
    }
    cl.sync();
    uint32_t all = 0, before = 0;   // tokens of this digit in the cluster, and in the blocks before this one
    if (static_cast<int>(threadIdx.x) < digits)
      for (int r = 0; r < C; ++r) {
        const uint32_t n = *cl.map_shared_rank(&total[threadIdx.x], r);
        if (r < rank) before += n;
        all += n;
      }
    // exclusive sum over the digits
    uint32_t inc = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(kFull, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    uint32_t base = inc - all + before;
    for (int w = 0; w < warp; ++w) base += scan[w];
    if (static_cast<int>(threadIdx.x) < digits) {
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) hist[w][threadIdx.x] += base;
    }
    __syncthreads();
    uint32_t *to_key = p.key[pass & 1], *to_pos = p.pos[pass & 1];
    if constexpr (KEEP > 0) {
#pragma unroll
      for (int n = 0; n < KEEP; ++n)
        if (begin + 32 * n + lane < end) {
          const uint32_t to = hist[warp][(key[n] >> shift) & mask] + before_me[n];
          to_key[to] = key[n];
          to_pos[to] = at[n];
        }
      __syncwarp();
    } else {
      for (int64_t i0 = begin; i0 < end; i0 += 32) {
        const int i = static_cast<int>(i0) + lane;
        const uint32_t have = __ballot_sync(kFull, i < end);
        if (i < end) {
          const uint32_t k = key_of<I>(p, from_key, pass, i), to = count((k >> shift) & mask, have);
          to_key[to] = k;
          to_pos[to] = pass > 0 ? __ldcg(from_pos + i) : static_cast<uint32_t>(i);
        }
        __syncwarp();
      }
    }
    for (int d = lane; d < digits; d += 32) hist[warp][d] = 0;
    __threadfence();
    cl.sync();   // the pass is in memory, and nobody reads this block's totals any more
  }
}

// ---- sums ------------------------------------------------------------------------------------------------------------------
struct SumParams {
  const uint32_t *key, *pos;
  const void* dout;
  float* grad;
  float* part;      // [tiles][2][H]: of the tile's first run where it began before, of its last where it goes on (a run that
                    // does both is in the first)
  int64_t H;
  int64_t vocab, early;   // early: rows that hold zeros already
  int M, tile, tiles, tx, accumulate;   // tile: sorted tokens of one, 8 to kMaxTile
  int cols, sum_blocks;                 // blocks to a tile's columns, and of sums in all: the blocks behind them write zeros
  float scale;
};

template <int N>
__device__ __forceinline__ void put(float* p, const float (&v)[N]) {
  if constexpr (N == 1) {
    p[0] = v[0];
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 4) *reinterpret_cast<float4*>(p + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
  }
}
template <int N>
__device__ __forceinline__ void get_add(const float* p, float (&v)[N]) {
  if constexpr (N == 1) {
    v[0] += p[0];
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      const float4 x = *reinterpret_cast<const float4*>(p + e);
      v[e] += x.x; v[e + 1] += x.y; v[e + 2] += x.z; v[e + 3] += x.w;
    }
  }
}
template <int N>
__device__ __forceinline__ void finish(const SumParams& p, uint32_t id, int64_t c, float (&v)[N]) {
  float* g = p.grad + static_cast<int64_t>(id) * p.H + c;
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] *= p.scale;
  if (p.accumulate) get_add<N>(g, v);
  put<N>(g, v);
}

// Zeros for the rows [first, first + kZeroRows) of the table that no token names, past the L2 (the parts of long runs wait there).
__device__ __forceinline__ void zero_rows(const SumParams& p, const uint32_t* keys, int64_t first, uint32_t* named) {
  const int64_t end = first + kZeroRows < p.vocab ? first + kZeroRows : p.vocab;
  if (threadIdx.x < kZeroRows / 32) named[threadIdx.x] = 0;
  __syncthreads();
  // from the first sorted token that names a row of these on, mark what the tokens name, 32 of them at a time; 32 of one row are followed by a jump
  // behind the last of that row, so that a row named by half of all tokens takes some looks more and not one for every 32 of them (65536 tokens, half of
  // them the same: the whole gradient 882 us without, 476 with)
  if (threadIdx.x < 32) {
    // the first token from lo on whose row is not below `bound`, by 32 looks at a time
    auto seek = [&](int64_t lo, int64_t bound) {
      int64_t hi = p.M;   // keys before lo are below bound, keys from hi on are not
      while (lo < hi) {
        const int64_t step = (hi - lo + 31) / 32, q = lo + step * (threadIdx.x + 1) - 1;
        const int n = __popc(__ballot_sync(kFull, q < hi && __ldcg(keys + q) < bound));
        lo += step * n;
        hi = lo + step - 1 < hi ? lo + step - 1 : hi;
      }
      return lo;
    };
    int64_t lo = seek(0, first);
    for (;;) {
      const int64_t i = lo + threadIdx.x;
      const uint32_t key = i < p.M ? __ldcg(keys + i) : static_cast<uint32_t>(p.vocab);
      const bool in = key < end;
      const uint32_t r = key - static_cast<uint32_t>(first), one = __shfl_sync(kFull, r, 0);
      if (__all_sync(kFull, in && r == one)) {
        if (threadIdx.x == 0) atomicOr(&named[one >> 5], 1u << (one & 31));
        lo = seek(lo + 32, first + one + 1);
        continue;
      }
      if (in) atomicOr(&named[r >> 5], 1u << (r & 31));
      if (!__all_sync(kFull, in)) break;
      lo += 32;
    }
  }
  __syncthreads();
  const bool vec = p.H % 4 == 0;
  uint32_t any = 0;
  for (int i = 0; i < kZeroRows / 32; ++i) any |= named[i];
  if (any == 0 && vec) {   // all of them, without the rows between
    float4* to = reinterpret_cast<float4*>(p.grad + first * p.H);
    for (int64_t i = threadIdx.x; i < (end - first) * p.H / 4; i += kThreads) __stcs(to + i, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    return;
  }
  for (int64_t r = first; r < end; ++r) {
    const int k = static_cast<int>(r - first);
    if (named[k >> 5] >> (k & 31) & 1u) continue;
    float* row = p.grad + r * p.H;
    if (vec)
      for (int64_t i = threadIdx.x; i < p.H / 4; i += kThreads) __stcs(reinterpret_cast<float4*>(row) + i, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    else
      for (int64_t i = threadIdx.x; i < p.H; i += kThreads) row[i] = 0.0f;
  }
}

template <typename T>
struct One {   // (as Vec16)
  T raw;
  __device__ __forceinline__ void to_float(float* f) const { f[0] = to_f32(raw); }
};
__host__ __device__ constexpr int list_words(int tile) { return 2 * tile + 2; }

template <typename T, int N>
__global__ void __launch_bounds__(kThreads) sum_kernel(const __grid_constant__ SumParams p) {
  extern __shared__ uint32_t lists[];   // by tile of the block: its keys with one on either side, its positions
  const int x = threadIdx.x % p.tx, y = threadIdx.x / p.tx, ty = kThreads / p.tx;
  const int64_t t = static_cast<int64_t>(blockIdx.x / p.cols) * ty + y;
  grid_launch_dependents();
  grid_dependency_wait();
  const uint32_t *keys = from_here(p.key), *places = from_here(p.pos);
  if (blockIdx.x >= static_cast<unsigned>(p.sum_blocks)) {
    zero_rows(p, keys, p.early + static_cast<int64_t>(blockIdx.x - p.sum_blocks) * kZeroRows, lists);
    return;
  }
  uint32_t *s_key = lists + y * list_words(p.tile), *s_pos = s_key + p.tile + 2;
  const int64_t i0 = t * p.tile;
  const int n = t < p.tiles ? static_cast<int>(i0 + p.tile < p.M ? p.tile : p.M - i0) : 0;
  const uint32_t none = static_cast<uint32_t>(p.vocab);
  // keys of the tile with one on either side
  for (int i = x; i < n + 2 && n > 0; i += p.tx) {
    const int64_t at = i0 + i - 1;
    s_key[i] = at >= 0 && at < p.M ? __ldcg(keys + at) : none;
    if (i >= 1 && i <= n) s_pos[i - 1] = __ldcg(places + at);
  }
  __syncthreads();
  if (n == 0) return;
  const int64_t c = N * (static_cast<int64_t>(blockIdx.x % p.cols) * p.tx + x);
  if (c >= p.H) return;
  const T* dout = static_cast<const T*>(p.dout) + c;
  const bool began = s_key[0] == s_key[1], goes_on = s_key[n] == s_key[n + 1] && i0 + n < p.M;
  float acc[N] = {};
  bool first = true;   // still in the tile's first run
  constexpr int kAhead = 8;
  for (int b = 0; b < n; b += kAhead) {
    std::conditional_t<N == 1, One<T>, Vec16<T>> v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if constexpr (N == 1) v[k].raw = from_f32<T>(0.0f);
      else v[k].raw = {};
      if (b + k < n && s_key[b + k + 1] != none)
        v[k].raw = *reinterpret_cast<const decltype(v[k].raw)*>(dout + static_cast<int64_t>(s_pos[b + k]) * p.H);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = b + k;
      if (i >= n) break;
      const uint32_t id = s_key[i + 1];
      float f[N];
      v[k].to_float(f);
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += f[e];
      const bool last = i == n - 1;
      if (!last && s_key[i + 2] == id) continue;
      // the run ends here, or goes on behind the tile
      if (id != none) {
        if (first && began && i0 > 0) put<N>(p.part + (2 * t) * p.H + c, acc);
        else if (last && goes_on) put<N>(p.part + (2 * t + 1) * p.H + c, acc);
        else finish<N>(p, id, c, acc);
      }
      first = false;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = 0.0f;
    }
  }
}

// The runs that go on behind the tile in which they begin, a block to a tile (most have nothing to do and leave).  kJoinThreads / width groups of
// threads share the parts of a run, consecutive ones each, and add their sums up in order: a token of a thousand rows waits for memory
// a few times and not a hundred.  A run of kShare parts or more has its columns shared as well, by the blocks of its first tiles: kSlice threads wide each, so
// that there are 32 groups (896 columns, 32768 tokens of one id, this kernel: 330 us by one block, 29 so; below 64 parts the looks that
// the other blocks need are what the shares save).
constexpr int kShare = 64, kSlice = 8;
static_assert(kThreads / kSlice <= 32 && kThreads / kSlice <= kShare, "one look finds the run's begin, and it has a block for every slice");
template <int N>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ SumParams p) {
  __shared__ float sums[kJoinThreads * N];
  __shared__ int64_t found[2];   // the tiles in which the run begins and ends
  const int t = blockIdx.x;
  grid_launch_dependents();
  grid_dependency_wait();
  const uint32_t* keys = from_here(p.key);
  const int64_t i0 = static_cast<int64_t>(t) * p.tile, i1 = i0 + p.tile;
  if (i1 >= p.M) return;
  const uint32_t id = __ldcg(keys + i1 - 1), next = __ldcg(keys + i1), before = i0 > 0 ? __ldcg(keys + i0 - 1) : static_cast<uint32_t>(p.vocab);
  if (id >= static_cast<uint32_t>(p.vocab) || next != id) return;   // no run goes on behind this tile
  const int slices = p.tx > kSlice ? p.tx / kSlice : 1;
  if (before == id && slices == 1) return;   // it begins before, and is not shared
  if (threadIdx.x < 32) {
    int64_t begin = t;
    if (before == id) {
      // this tile and the n before it begin with the id
      const int64_t q = t - 1 - static_cast<int64_t>(threadIdx.x);
      begin -= __popc(__ballot_sync(kFull, q >= 0 && __ldcg(keys + q * p.tile) == id));
      if (begin > 0 && __ldcg(keys + begin * p.tile - 1) == id) --begin;
    }
    // the last tile that it reaches: tile q does where its first key is this id.  32 tiles a look, or 32 groups of 32 where they are not enough
    int64_t last = t + 1;
    for (int64_t step = 1; t - begin < slices;) {
      const int64_t q = last + step * (threadIdx.x + 1);
      const int n = __popc(__ballot_sync(kFull, q < p.tiles && __ldcg(keys + q * p.tile) == id));
      last += step * n;
      if (n == 32) step *= 32;
      else if (step == 1) break;
      else step /= 32;
    }
    if (threadIdx.x == 0) { found[0] = begin; found[1] = last; }
  }
  __syncthreads();
  const int64_t begin = found[0], count = found[1] - begin;   // parts behind the first tile's own
  const bool shared = count >= kShare && slices > 1;
  if (t - begin >= (shared ? slices : 1)) return;
  const int width = shared ? kSlice : p.tx, x = threadIdx.x % width, g = threadIdx.x / width, groups = count < 8 ? 1 : kJoinThreads / width;
  const int64_t c = N * (static_cast<int64_t>(blockIdx.y) * p.tx + (t - begin) * width + x);
  float acc[N] = {};
  if (g < groups && c < p.H) {
    if (g == 0) get_add<N>(p.part + (2 * begin + 1) * p.H + c, acc);
    const int64_t to = begin + 1 + count * (g + 1) / groups;
#pragma unroll 8
    for (int64_t q = begin + 1 + count * g / groups; q < to; ++q) get_add<N>(p.part + 2 * q * p.H + c, acc);
  }
  if (groups > 1) {
    put<N>(sums + threadIdx.x * N, acc);
    __syncthreads();
    if (g == 0)
      for (int o = 1; o < groups; ++o) get_add<N>(sums + (o * width + x) * N, acc);
  }
  if (g == 0 && c < p.H) finish<N>(p, id, c, acc);
}

inline size_t up256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }
// Sorted tokens of a tile: short tiles keep all SMs busy with few tokens (sums of 8192 tokens of 896, us: 16 with tiles of 8, 25 with 32), long ones leave
// fewer parts to join.
inline int tile_of(int64_t M) { return M <= 16384 ? 8 : M <= 65536 ? 16 : kMaxTile; }
inline int64_t tiles_of(int64_t M) { return (M + tile_of(M) - 1) / tile_of(M); }
// threads that share a row of `n` pieces: a power of two up to kThreads
inline int row_threads(int64_t n) {
  int t = 1;
  while (t < kThreads && t < n) t <<= 1;
  return t;
}

template <typename I>
int launch_sort(const SortParams& p, int sms, cudaStream_t st) {
  // few tokens: a block alone ranks them sooner than eight that wait for one another three times a pass
  const int C = p.M <= 1024 ? 1 : 8;
  cudaLaunchConfig_t cfg = {};
  int64_t fill = (p.zero_n / 4 + kSortThreads * 4 - 1) / (kSortThreads * 4);
  if (p.zero_n > 0 && fill == 0) fill = 1;
  if (fill > 2 * sms) fill = 2 * sms;
  cfg.gridDim = dim3(static_cast<unsigned>(C + (fill + C - 1) / C * C));
  cfg.blockDim = dim3(kSortThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = chained_launch() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 2;
  const bool few = p.M <= C * kSortWarps * 128;
  MCB_CHECK_CUDA(few ? cudaLaunchKernelEx(&cfg, sort_kernel<I, 4>, p) : cudaLaunchKernelEx(&cfg, sort_kernel<I, 0>, p));
  MCB_CHECK_LAUNCH("embedding_sort");
  return MCB_OK;
}

template <typename T, int N>
int launch_sums(SumParams& p, cudaStream_t st) {
  p.tx = row_threads((p.H + N - 1) / N);
  const int ty = kThreads / p.tx;
  const int64_t cols = (p.H + static_cast<int64_t>(N) * p.tx - 1) / (static_cast<int64_t>(N) * p.tx);
  const int64_t sums = (p.tiles + ty - 1) / ty * cols, zeros = (p.vocab - p.early + kZeroRows - 1) / kZeroRows;
  if (cols > 65535 || sums + zeros > 0x7fffffff) return fail(MCB_ERR_SHAPE, "embedding_bwd: H=%lld", (long long)p.H);
  p.cols = static_cast<int>(cols); p.sum_blocks = static_cast<int>(sums);
  MCB_CHECK_CUDA(launch_kernel(sum_kernel<T, N>, dim3(static_cast<unsigned>(sums + zeros)), dim3(kThreads),
                               static_cast<size_t>(ty) * list_words(p.tile) * 4, st, chained_launch(), p));
  MCB_CHECK_LAUNCH("embedding_sum");
  if (p.tiles > 1) {
    MCB_CHECK_CUDA(launch_kernel(join_kernel<N>, dim3(static_cast<unsigned>(p.tiles), static_cast<unsigned>(cols)), dim3(kJoinThreads), 0, st, chained_launch(), p));
    MCB_CHECK_LAUNCH("embedding_join");
  }
  return MCB_OK;
}

int check(const char* who, int id_bytes, int64_t M, int64_t H, int64_t vocab, float scale, int dtype) {
  if (dtype != MCB_F32 && dtype != MCB_BF16) return fail(MCB_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (id_bytes != 4 && id_bytes != 8) return fail(MCB_ERR_UNSUPPORTED, "%s: ids of %d bytes (4 or 8)", who, id_bytes);
  if (M <= 0 || M > 0x3fffffff || H <= 0 || H > 0x7fffff || vocab <= 0 || vocab > 0x3fffffff)
    return fail(MCB_ERR_SHAPE, "%s: M=%lld H=%lld vocab=%lld", who, (long long)M, (long long)H, (long long)vocab);
  if (!(scale - scale == 0.0f)) return fail(MCB_ERR_SHAPE, "%s: scale is not finite", who);
  return MCB_OK;
}

template <typename T, typename I>
int launch_fwd(const void* ids, const void* table, void* out, int64_t M, int64_t H, int64_t vocab, float scale, int sms, cudaStream_t st) {
  constexpr int N = Vec16<T>::N;
  const bool vec = H % N == 0 && aligned16(table) && aligned16(out);
  const int tx = row_threads(vec ? H / N : H);
  const int64_t want = (M + kThreads / tx - 1) / (kThreads / tx), most = 16ll * sms;
  const dim3 grid(static_cast<unsigned>(want < most ? want : most));
  if (vec)
    MCB_CHECK_CUDA(launch_kernel(embed_fwd_kernel<T, I, N>, grid, dim3(kThreads), 0, st, chained_launch(), static_cast<const I*>(ids),
                                 static_cast<const T*>(table), static_cast<T*>(out), M, H, vocab, scale, tx));
  else
    MCB_CHECK_CUDA(launch_kernel(embed_fwd_kernel<T, I, 1>, grid, dim3(kThreads), 0, st, chained_launch(), static_cast<const I*>(ids),
                                 static_cast<const T*>(table), static_cast<T*>(out), M, H, vocab, scale, tx));
  MCB_CHECK_LAUNCH("embedding_scaled_fwd");
  return MCB_OK;
}

}  // namespace
}  // namespace embed
}  // namespace mcb

using namespace mcb;

extern "C" int mcb_embedding_scaled_fwd(const void* ids, int id_bytes, const void* table, void* out, int64_t M, int64_t H, int64_t vocab,
                                        float scale, int dtype, void* stream) {
  MCB_NVTX_RANGE("mcb_embedding_scaled_fwd");
  if (!ids || !table || !out) return fail(MCB_ERR_NULL, "embedding_scaled_fwd: null pointer");
  if (int rc = embed::check("embedding_scaled_fwd", id_bytes, M, H, vocab, scale, dtype)) return rc;
  if (!on_boundary(id_bytes, ids) || !on_boundary(element_bytes(dtype), table, out))
    return fail(MCB_ERR_ALIGN, "embedding_scaled_fwd: a pointer is not aligned to its elements");
  const size_t row = static_cast<size_t>(H) * element_bytes(dtype);
  const Range ranges[] = {{out, M * row}, {table, vocab * row}, {ids, static_cast<size_t>(M) * id_bytes}};
  if (outputs_overlap(ranges, 1)) return fail(MCB_ERR_SHAPE, "embedding_scaled_fwd: the output overlaps an input");
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == MCB_F32)
    return id_bytes == 4 ? embed::launch_fwd<float, int32_t>(ids, table, out, M, H, vocab, scale, ds->sm_count, st)
                         : embed::launch_fwd<float, int64_t>(ids, table, out, M, H, vocab, scale, ds->sm_count, st);
  return id_bytes == 4 ? embed::launch_fwd<__nv_bfloat16, int32_t>(ids, table, out, M, H, vocab, scale, ds->sm_count, st)
                       : embed::launch_fwd<__nv_bfloat16, int64_t>(ids, table, out, M, H, vocab, scale, ds->sm_count, st);
}

extern "C" size_t mcb_embedding_bwd_workspace_bytes(int64_t M, int64_t H) {
  if (M <= 0 || H <= 0 || M > 0x3fffffff || H > 0x7fffff) return 0;
  return 4 * embed::up256(static_cast<size_t>(M) * 4) + static_cast<size_t>(embed::tiles_of(M)) * 2 * H * 4;
}

extern "C" int mcb_embedding_bwd(const void* ids, int id_bytes, const void* dout, float* dtable, int accumulate, int64_t M, int64_t H,
                                 int64_t vocab, float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  MCB_NVTX_RANGE("mcb_embedding_bwd");
  if (!ids || !dout || !dtable) return fail(MCB_ERR_NULL, "embedding_bwd: null pointer");
  if (int rc = embed::check("embedding_bwd", id_bytes, M, H, vocab, scale, dtype)) return rc;
  if (!aligned16(dtable)) return fail(MCB_ERR_ALIGN, "embedding_bwd: the table's gradient is not 16-byte aligned");
  if (!on_boundary(id_bytes, ids) || !on_boundary(element_bytes(dtype), dout))
    return fail(MCB_ERR_ALIGN, "embedding_bwd: a pointer is not aligned to its elements");
  if (!workspace || workspace_bytes < mcb_embedding_bwd_workspace_bytes(M, H) || !aligned16(workspace))
    return fail(MCB_ERR_WORKSPACE, "embedding_bwd: workspace of %zu bytes, 16-byte aligned, needed", mcb_embedding_bwd_workspace_bytes(M, H));
  const Range ranges[] = {{dtable, static_cast<size_t>(vocab) * H * sizeof(float)}, {workspace, mcb_embedding_bwd_workspace_bytes(M, H)},
                          {dout, static_cast<size_t>(M) * H * element_bytes(dtype)}, {ids, static_cast<size_t>(M) * id_bytes}};
  if (outputs_overlap(ranges, 2)) return fail(MCB_ERR_SHAPE, "embedding_bwd: the gradient or the workspace overlaps an input or one another");
  DeviceState* ds = current_device_state();
  if (!ds) return MCB_ERR_NOT_INIT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* w = static_cast<uint8_t*>(workspace);
  const size_t list = embed::up256(static_cast<size_t>(M) * 4);
  embed::SortParams s = {};
  s.ids = ids;
  for (int i = 0; i < 2; ++i) {
    s.key[i] = reinterpret_cast<uint32_t*>(w + 2 * i * list);
    s.pos[i] = reinterpret_cast<uint32_t*>(w + (2 * i + 1) * list);
  }
  // what the sort's launch can write while it sorts, the rows behind that with the sums
  int64_t early = accumulate ? vocab : embed::kEarlyBytes / (H * 4);
  if (early > vocab) early = vocab;
  if (!accumulate) { s.zero = dtable; s.zero_n = early * H; }
  s.vocab = vocab; s.M = static_cast<int>(M);
  int bits = 1;
  while ((vocab >> bits) != 0) ++bits;   // of vocab itself, which stands for the ids that count for nothing
  s.passes = (bits + 8) / 9;
  s.digit_bits = (bits + s.passes - 1) / s.passes;
  if (int rc = id_bytes == 4 ? embed::launch_sort<int32_t>(s, ds->sm_count, st) : embed::launch_sort<int64_t>(s, ds->sm_count, st)) return rc;
  embed::SumParams p = {};
  p.key = s.key[(s.passes - 1) & 1]; p.pos = s.pos[(s.passes - 1) & 1];
  p.dout = dout; p.grad = dtable; p.part = reinterpret_cast<float*>(w + 4 * list);
  p.H = H; p.vocab = vocab; p.early = early; p.M = static_cast<int>(M); p.tile = embed::tile_of(M); p.tiles = static_cast<int>(embed::tiles_of(M)); p.accumulate = accumulate; p.scale = scale;
  const int n = dtype == MCB_F32 ? 4 : 8;
  const bool vec = H % n == 0 && aligned16(dout);
  if (dtype == MCB_F32) return vec ? embed::launch_sums<float, 4>(p, st) : embed::launch_sums<float, 1>(p, st);
  return vec ? embed::launch_sums<__nv_bfloat16, 8>(p, st) : embed::launch_sums<__nv_bfloat16, 1>(p, st);
}
