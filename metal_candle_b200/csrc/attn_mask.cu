// The mask of packed documents as intervals (see attn_mask.cuh).
//
// A document is a maximal run of equal, non-negative ids; negative ids are padding, which sees nothing and is seen by nothing.
// The first positions of a document that are marked as prefix are seen by the whole document, every other one by itself and
// what follows.  With a the run's first position, e the one behind its last and p the one behind its leading prefix
// (a where it has none):  query i sees the keys [a, max(i + 1, p)), key j is seen by the queries [j < p ? a : j, e).
//
// a, e and p are the nearest set bits of two bitmaps (a run begins here; this position is no prefix) before or behind a position.
// Three levels of 32 positions to a word answer that in at most five loads within 32768 positions, so that every position finds
// its own: two launches, no scan over the sequence.
// The second launch also reduces the intervals to tile ranges, and its last block sorts the tiles by the work that they are:
// documents make some tiles many times as long as others, and persistent kernels that take the longest first end together.
#include "attn_mask.cuh"

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
  const uint32_t* w;   // level 1: chunks * 1024 words, level 2: chunks * 32, level 3: chunks
  int chunks;
  __device__ __forceinline__ uint32_t l1(int i) const { return __ldcg(w + i); }
  __device__ __forceinline__ uint32_t l2(int i) const { return __ldcg(w + chunks * 1024 + i); }
  __device__ __forceinline__ uint32_t l3(int i) const { return __ldcg(w + chunks * 1056 + i); }
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

// One block per 32768 positions of a sequence and bitmap (z: 0 run begins, 1 no prefix).
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
    bool set = false;
    if (pos < p.S) {
      if (kind == 1) set = prefix == nullptr || prefix[row + pos] == 0;
      else set = pos == 0 || (ids != nullptr && id_at<I>(ids, row + pos) != id_at<I>(ids, row + pos - 1));
    }
    const uint32_t word = __ballot_sync(0xffffffffu, set);
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
  const int64_t pos = static_cast<int64_t>(t) * kTile + threadIdx.x;
  if (pos < p.S) {
    const int i = static_cast<int>(pos);
    const int64_t at = static_cast<int64_t>(b) * p.S + i;
    int2 sees = make_int2(i, i), seen = make_int2(i, i);
    if (p.ids == nullptr || id_at<I>(from_here(p.ids), at) >= 0) {
      const int a = prev_set(runs, i), e = next_set(runs, i + 1, p.S);
      const int lead = p.prefix == nullptr ? a : min(next_set(open, a, p.S), e);
      sees = make_int2(a, max(i + 1, lead));
      seen = make_int2(i < lead ? a : i, e);
      atomicMin(&lo[0], sees.x); atomicMax(&hi[0], sees.y);
      atomicMin(&lo[1], seen.x); atomicMax(&hi[1], seen.y);
    }
    reinterpret_cast<int2*>(p.block + p.l.rows)[at] = sees;
    reinterpret_cast<int2*>(p.block + p.l.keys)[at] = seen;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    const int k = threadIdx.x;
    int2 range = make_int2(0, 0);
    if (hi[k] > 0) {
      range.x = lo[k] / kStep;
      range.y = (hi[k] + kStep - 1) / kStep - range.x;
    }
    reinterpret_cast<int2*>(p.block + (k ? p.l.ktiles : p.l.qtiles))[blockIdx.x] = range;
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
