// The mask of packed documents as intervals (see attn_mask.cuh).
//
// A document is a maximal run of equal, non-negative ids; negative ids are padding, which sees nothing and is seen by nothing.
// The first positions of a document that are marked as prefix are seen by the whole document, every other one by itself and
// what follows.  With a the run's first position, e the one behind its last and p the one behind its leading prefix
// (a where it has none):  query i sees the keys [a, max(i + 1, p)), key j is seen by the queries [j < p ? a : j, e).
//
// a, e and p are the nearest set bits of two bitmaps (a run begins here; this position is no prefix) before or behind a position.
// Three levels of 32 positions to a word answer that in at most five loads within 32768 positions, so that every position finds its own and
// there is no scan over the sequence.  The intervals are reduced to tile ranges, and the tiles are listed by falling work: documents
// make some tiles many times as long as others, and persistent kernels that take the longest first end together.
// Sequences up to 32768 take one launch, a cluster to a sequence with its bitmaps in shared memory; the list takes the longest tile of each
// sequence, then the second of each.  Longer ones take two: one writes the bitmaps, the other has a block to a tile, whose last one
// sorts all tiles.
#include <cooperative_groups.h>

#include "attn_mask.cuh"

namespace cg = cooperative_groups;

namespace mcb {
namespace amask {
namespace {

struct MaskParams {
  const void* ids;          // [batch, seq] or null: one document
  const uint8_t* prefix;    // [batch, seq] or null: none
  int* block;
  Layout l;
  int S, B, chunks;
};

struct Bits {
  const uint32_t* w;   // level 1: chunks * 1024 words, level 2: chunks * 32, level 3: chunks; in shared or global memory
  int chunks;
  __device__ __forceinline__ uint32_t l1(int i) const { return w[i]; }
  __device__ __forceinline__ uint32_t l2(int i) const { return w[chunks * 1024 + i]; }
  __device__ __forceinline__ uint32_t l3(int i) const { return w[chunks * 1056 + i]; }
};
__device__ __forceinline__ uint32_t above(int bit) { return bit == 31 ? 0u : ~0u << (bit + 1); }
__device__ __forceinline__ uint32_t below(int bit) { return (1u << bit) - 1u; }

// first set position >= from, or S
__device__ int next_set(const Bits& b, int from, int S) {
  if (from >= S) return S;
  const int w1 = from >> 5, w2 = w1 >> 5;
  uint32_t m = b.l1(w1) & (~0u << (from & 31));
  if (m) return w1 * 32 + __ffs(m) - 1;
  m = b.l2(w2) & above(w1 & 31);
  if (!m) {
    int c = w2 >> 5;
    uint32_t m3 = b.l3(c) & above(w2 & 31);
    while (!m3) {
      if (++c >= b.chunks) return S;
      m3 = b.l3(c);
    }
    const int v2 = c * 32 + __ffs(m3) - 1;
    m = b.l2(v2);
    const int v1 = v2 * 32 + __ffs(m) - 1;
    return v1 * 32 + __ffs(b.l1(v1)) - 1;
  }
  const int v1 = w2 * 32 + __ffs(m) - 1;
  return v1 * 32 + __ffs(b.l1(v1)) - 1;
}
// last set position <= from; position 0 is always set in the bitmap this is asked of
__device__ int prev_set(const Bits& b, int from) {
  const int w1 = from >> 5, w2 = w1 >> 5;
  uint32_t m = b.l1(w1) & (below(from & 31) | (1u << (from & 31)));
  if (m) return w1 * 32 + 31 - __clz(m);
  m = b.l2(w2) & below(w1 & 31);
  if (!m) {
    int c = w2 >> 5;
    uint32_t m3 = b.l3(c) & below(w2 & 31);
    while (!m3) {
      if (--c < 0) return 0;
      m3 = b.l3(c);
    }
    const int v2 = c * 32 + 31 - __clz(m3);
    m = b.l2(v2);
    const int v1 = v2 * 32 + 31 - __clz(m);
    return v1 * 32 + 31 - __clz(b.l1(v1));
  }
  const int v1 = w2 * 32 + 31 - __clz(m);
  return v1 * 32 + 31 - __clz(b.l1(v1));
}

template <typename I>
__device__ __forceinline__ int64_t id_at(const void* ids, int64_t i) {
  return static_cast<int64_t>(__ldg(static_cast<const I*>(ids) + i));
}

// Whether the bitmap (kind 0: a run begins, 1: no prefix) is set at position pos of a sequence whose first element is `row`.
template <typename I>
__device__ __forceinline__ bool bit_of(int kind, const void* ids, const uint8_t* prefix, int64_t row, int64_t pos, int S) {
  if (pos >= S) return false;
  if (kind == 1) return prefix == nullptr || prefix[row + pos] == 0;
  return pos == 0 || (ids != nullptr && id_at<I>(ids, row + pos) != id_at<I>(ids, row + pos - 1));
}
// What position i sees and by what it is seen.
__device__ __forceinline__ void intervals(const Bits& runs, const Bits& open, bool marked, int i, int S, int2& sees, int2& seen) {
  const int a = prev_set(runs, i), e = next_set(runs, i + 1, S);
  const int lead = marked ? min(next_set(open, a, S), e) : a;
  sees = make_int2(a, max(i + 1, lead));
  seen = make_int2(i < lead ? a : i, e);
}
__device__ __forceinline__ int2 blocks_of(int lo, int hi) {
  return hi > 0 ? make_int2(lo / kStep, (hi + kStep - 1) / kStep - lo / kStep) : make_int2(0, 0);
}

// Sequences up to 32768: a cluster does all of a sequence.  Each of its blocks takes whole thousands of positions, gives its bits to all the
// others, and later its tiles' ranges.
template <typename I>
__global__ void __launch_bounds__(1024) mask_short_kernel(const MaskParams p) {
  __shared__ uint32_t words[2][1024 + 32 + 1];
  __shared__ int2 lo[kChunk / kTile], hi[kChunk / kTile];   // x: keys of the query tile, y: queries of the key tile
  cg::cluster_group cl = cg::this_cluster();
  const int C = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank());
  const int b = blockIdx.x / C, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tiles = static_cast<int>(tiles_of(p.S));
  const int per = ((p.S + 1023) / 1024 + C - 1) / C * 1024, first = min(rank * per, p.S), last = min(first + per, p.S);
  if (threadIdx.x < kChunk / kTile) {
    lo[threadIdx.x] = make_int2(0x7fffffff, 0x7fffffff);
    hi[threadIdx.x] = make_int2(0, 0);
  }
  words[0][threadIdx.x] = words[1][threadIdx.x] = 0;
  grid_launch_dependents();
  grid_dependency_wait();
  const int64_t row = static_cast<int64_t>(b) * p.S;
  const void* ids = from_here(p.ids);
  const uint8_t* prefix = from_here(p.prefix);
  const int kinds = prefix == nullptr ? 1 : 2;
  cl.sync();
  for (int kind = 0; kind < kinds; ++kind)
    for (int at = first; at < last; at += 4096) {   // four loads on their way at a time
      bool set[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) set[u] = at + 1024 * u < last && bit_of<I>(kind, ids, prefix, row, at + 1024 * u + threadIdx.x, p.S);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t word = __ballot_sync(0xffffffffu, set[u]);
        if (lane < C && at + 1024 * u < last) *cl.map_shared_rank(&words[kind][(at >> 5) + 32 * u + warp], lane) = word;
      }
    }
  cl.sync();
  for (int kind = 0; kind < kinds; ++kind) {
    const uint32_t two = __ballot_sync(0xffffffffu, words[kind][threadIdx.x] != 0);
    if (lane == 0) words[kind][1024 + warp] = two;
  }
  __syncthreads();
  if (warp < kinds) {
    const uint32_t three = __ballot_sync(0xffffffffu, words[warp][1024 + lane] != 0);
    if (lane == 0) words[warp][1056] = three;
  }
  __syncthreads();
  const Bits runs{words[0], 1}, open{words[1], 1};
  int2 *rows = reinterpret_cast<int2*>(p.block + p.l.rows) + row, *keys = reinterpret_cast<int2*>(p.block + p.l.keys) + row;
  for (int i0 = first; i0 < last; i0 += 1024) {
    const int i = i0 + threadIdx.x;
    int2 sees = make_int2(i, i), seen = sees;
    const bool real = i < last && (ids == nullptr || id_at<I>(ids, row + i) >= 0);
    if (real) intervals(runs, open, kinds == 2, i, p.S, sees, seen);
    // a warp's 32 positions are of one tile: reduced first, an atomic by each of them on the same word would take its turn
    const int lo0 = __reduce_min_sync(0xffffffffu, real ? sees.x : 0x7fffffff), hi0 = __reduce_max_sync(0xffffffffu, real ? sees.y : 0);
    const int lo1 = __reduce_min_sync(0xffffffffu, real ? seen.x : 0x7fffffff), hi1 = __reduce_max_sync(0xffffffffu, real ? seen.y : 0);
    if (lane == 0 && i < last) {
      const int t = i / kTile;
      atomicMin(&lo[t].x, lo0); atomicMax(&hi[t].x, hi0);
      atomicMin(&lo[t].y, lo1); atomicMax(&hi[t].y, hi1);
    }
    if (i < last) {
      rows[i] = sees;
      keys[i] = seen;
    }
  }
  __syncthreads();
  const int t0 = first / kTile, mine = (last - first + kTile - 1) / kTile;
  for (int i = threadIdx.x; i < mine * C; i += 1024) {
    const int t = t0 + i / C, to = i % C;
    if (to == rank) continue;
    *cl.map_shared_rank(&lo[t], to) = lo[t];
    *cl.map_shared_rank(&hi[t], to) = hi[t];
  }
  cl.sync();
  // a tile's place in its sequence's order: the tiles that are longer, and as long but earlier
  for (int i = warp; i < 2 * mine; i += 32) {
    const bool k = i >= mine;
    const int t = t0 + (k ? i - mine : i);
    const int2 range = k ? blocks_of(lo[t].y, hi[t].y) : blocks_of(lo[t].x, hi[t].x);
    int place = 0;
    for (int u = lane; u < tiles; u += 32) {
      const int n = k ? blocks_of(lo[u].y, hi[u].y).y : blocks_of(lo[u].x, hi[u].x).y;
      place += n > range.y || (n == range.y && u < t);
    }
    place = __reduce_add_sync(0xffffffffu, place);
    if (lane != 0) continue;
    reinterpret_cast<int2*>(p.block + (k ? p.l.ktiles : p.l.qtiles))[static_cast<int64_t>(b) * tiles + t] = range;
    reinterpret_cast<int4*>(p.block + (k ? p.l.kwork : p.l.qwork))[static_cast<int64_t>(place) * p.B + b] = make_int4(b, t, range.x, range.y);
  }
}

// Longer ones.  One block per 32768 positions of a sequence and bitmap.
template <typename I>
__global__ void __launch_bounds__(1024) mask_bits_kernel(const MaskParams p) {
  __shared__ uint32_t words[1024];
  const int c = blockIdx.x, b = blockIdx.y, kind = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_launch_dependents();
  grid_dependency_wait();
  const int64_t row = static_cast<int64_t>(b) * p.S;
  const void* ids = from_here(p.ids);
  const uint8_t* prefix = from_here(p.prefix);
  words[threadIdx.x] = 0;
  __syncthreads();
  const int first = c * kChunk, last = min(kChunk, p.S - first);
  for (int it = 0; it * 1024 < last; ++it) {
    const int64_t pos = static_cast<int64_t>(first) + it * 1024 + threadIdx.x;
    const uint32_t word = __ballot_sync(0xffffffffu, bit_of<I>(kind, ids, prefix, row, pos, p.S));
    if (lane == 0) words[it * 32 + warp] = word;
  }
  __syncthreads();
  uint32_t* out = reinterpret_cast<uint32_t*>(p.block + p.l.bits) + (2 * static_cast<int64_t>(b) + kind) * p.l.bits_per_seq;
  const uint32_t mine = words[threadIdx.x];
  out[c * 1024 + threadIdx.x] = mine;
  const uint32_t two = __ballot_sync(0xffffffffu, mine != 0);
  __syncthreads();
  if (lane == 0) {
    out[p.chunks * 1024 + c * 32 + warp] = two;
    words[warp] = two;
  }
  __syncthreads();
  if (warp == 0) {
    const uint32_t three = __ballot_sync(0xffffffffu, words[lane] != 0);
    if (lane == 0) out[p.chunks * 1056 + c] = three;
    if (lane == 0 && c == 0 && b == 0 && kind == 0) p.block[p.l.ticket] = 0;
  }
}

// Tiles by falling block count: a counting sort over 1024 classes of counts, by one block of 128 threads.
__device__ void sort_tiles(const int2* tiles, int4* work, int n, int per_seq, int* bins, int* most) {
  tiles = from_here(tiles);
  if (threadIdx.x == 0) *most = 0;
  for (int i = threadIdx.x; i < 1024; i += kTile) bins[i] = 0;
  __syncthreads();
  int m = 0;
  for (int i = threadIdx.x; i < n; i += kTile) m = max(m, __ldcg(&tiles[i].y));
  atomicMax(most, m);
  __syncthreads();
  const int64_t top = max(1, *most);
  for (int i = threadIdx.x; i < n; i += kTile) atomicAdd(&bins[1023 - static_cast<int>(__ldcg(&tiles[i].y) * 1023ll / top)], 1);
  __syncthreads();
  // exclusive sums: eight bins a thread
  __shared__ int part[kTile];
  int sum = 0;
  for (int k = 0; k < 8; ++k) sum += bins[threadIdx.x * 8 + k];
  part[threadIdx.x] = sum;
  __syncthreads();
  for (int d = 1; d < kTile; d <<= 1) {
    const int v = threadIdx.x >= d ? part[threadIdx.x - d] : 0;
    __syncthreads();
    part[threadIdx.x] += v;
    __syncthreads();
  }
  int at = part[threadIdx.x] - sum;
  for (int k = 0; k < 8; ++k) {
    const int n_here = bins[threadIdx.x * 8 + k];
    bins[threadIdx.x * 8 + k] = at;
    at += n_here;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kTile) {
    const int first = __ldcg(&tiles[i].x), count = __ldcg(&tiles[i].y);
    work[atomicAdd(&bins[1023 - static_cast<int>(count * 1023ll / top)], 1)] = make_int4(i / per_seq, i % per_seq, first, count);
  }
  __syncthreads();
}

// One block per tile of 128 positions; the last one to finish sorts the tiles.
template <typename I>
__global__ void __launch_bounds__(kTile) mask_rows_kernel(const MaskParams p) {
  __shared__ int lo[2], hi[2], bins[1024], most, last;
  const int tiles = static_cast<int>(tiles_of(p.S)), b = blockIdx.x / tiles, t = blockIdx.x % tiles;
  grid_launch_dependents();
  if (threadIdx.x < 2) { lo[threadIdx.x] = 0x7fffffff; hi[threadIdx.x] = 0; }
  grid_dependency_wait();
  __syncthreads();
  const uint32_t* bits = reinterpret_cast<const uint32_t*>(p.block + p.l.bits) + 2 * static_cast<int64_t>(b) * p.l.bits_per_seq;
  bits = from_here(bits);
  const Bits runs{bits, p.chunks}, open{bits + p.l.bits_per_seq, p.chunks};
  const int64_t pos = static_cast<int64_t>(t) * kTile + threadIdx.x, at = static_cast<int64_t>(b) * p.S + pos;
  const int i = static_cast<int>(pos);
  int2 sees = make_int2(i, i), seen = sees;
  const bool real = pos < p.S && (p.ids == nullptr || id_at<I>(from_here(p.ids), at) >= 0);
  if (real) intervals(runs, open, p.prefix != nullptr, i, p.S, sees, seen);
  const int lo0 = __reduce_min_sync(0xffffffffu, real ? sees.x : 0x7fffffff), hi0 = __reduce_max_sync(0xffffffffu, real ? sees.y : 0);
  const int lo1 = __reduce_min_sync(0xffffffffu, real ? seen.x : 0x7fffffff), hi1 = __reduce_max_sync(0xffffffffu, real ? seen.y : 0);
  if ((threadIdx.x & 31) == 0) {
    atomicMin(&lo[0], lo0); atomicMax(&hi[0], hi0);
    atomicMin(&lo[1], lo1); atomicMax(&hi[1], hi1);
  }
  if (pos < p.S) {
    reinterpret_cast<int2*>(p.block + p.l.rows)[at] = sees;
    reinterpret_cast<int2*>(p.block + p.l.keys)[at] = seen;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    const int k = threadIdx.x;
    reinterpret_cast<int2*>(p.block + (k ? p.l.ktiles : p.l.qtiles))[blockIdx.x] = blocks_of(lo[k], hi[k]);
    __threadfence();
  }
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(p.block + p.l.ticket, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  const int n = p.B * tiles;
  sort_tiles(reinterpret_cast<const int2*>(p.block + p.l.qtiles), reinterpret_cast<int4*>(p.block + p.l.qwork), n, tiles, bins, &most);
  sort_tiles(reinterpret_cast<const int2*>(p.block + p.l.ktiles), reinterpret_cast<int4*>(p.block + p.l.kwork), n, tiles, bins, &most);
}

template <typename I>
int launch(const MaskParams& p, cudaStream_t st) {
  if (p.S <= kChunk) {
    // a thousand positions a block, more from 8192 on
    const int C = p.S <= 1024 ? 1 : p.S <= 2048 ? 2 : p.S <= 4096 ? 4 : 8;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.B * C));
    cfg.blockDim = dim3(1024);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = chained_launch() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(C); attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    MCB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, mask_short_kernel<I>, p));
    MCB_CHECK_LAUNCH("mask_short_kernel");
    return MCB_OK;
  }
  MCB_CHECK_CUDA(launch_kernel(mask_bits_kernel<I>, dim3(p.chunks, p.B, p.prefix == nullptr ? 1 : 2), dim3(1024), 0, st, chained_launch(), p));
  MCB_CHECK_LAUNCH("mask_bits_kernel");
  MCB_CHECK_CUDA(launch_kernel(mask_rows_kernel<I>, dim3(static_cast<unsigned>(p.B * tiles_of(p.S))), dim3(kTile), 0, st, chained_launch(), p));
  MCB_CHECK_LAUNCH("mask_rows_kernel");
  return MCB_OK;
}

}  // namespace
}  // namespace amask
}  // namespace mcb

using namespace mcb;

extern "C" size_t mcb_attention_mask_bytes(int64_t batch, int64_t seq) {
  if (batch <= 0 || seq <= 0 || batch > 65535 || seq > 0x3fffffffll || batch * seq > 0x7fffffffll) return 0;
  return (static_cast<size_t>(amask::layout(batch, seq).words) * 4 + 15) & ~static_cast<size_t>(15);
}

extern "C" int mcb_attention_mask(const void* document_ids, int id_bytes, const uint8_t* prefix, void* mask, size_t mask_bytes,
                                  int64_t batch, int64_t seq, void* stream) {
  MCB_NVTX_RANGE("mcb_attention_mask");
  if (!mask) return fail(MCB_ERR_NULL, "attention_mask: mask is null");
  const size_t need = mcb_attention_mask_bytes(batch, seq);
  if (need == 0) return fail(MCB_ERR_SHAPE, "attention_mask: batch=%lld seq=%lld (batch up to 65535, batch * seq below 2^31)", (long long)batch, (long long)seq);
  if (id_bytes != 4 && id_bytes != 8) return fail(MCB_ERR_UNSUPPORTED, "attention_mask: document ids of %d bytes (4 or 8)", id_bytes);
  if (!aligned16(mask) || (reinterpret_cast<uintptr_t>(document_ids) & (id_bytes - 1)) != 0) return fail(MCB_ERR_ALIGN, "attention_mask: alignment");
  if (mask_bytes < need) return fail(MCB_ERR_WORKSPACE, "attention_mask: %zu bytes given, %zu needed", mask_bytes, need);
  if (!current_device_state()) return MCB_ERR_NOT_INIT;
  amask::MaskParams p;
  p.ids = document_ids; p.prefix = prefix; p.block = static_cast<int*>(mask);
  p.l = amask::layout(batch, seq);
  p.S = static_cast<int>(seq); p.B = static_cast<int>(batch);
  p.chunks = static_cast<int>((seq + amask::kChunk - 1) / amask::kChunk);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return id_bytes == 4 ? amask::launch<int32_t>(p, st) : amask::launch<int64_t>(p, st);
}
