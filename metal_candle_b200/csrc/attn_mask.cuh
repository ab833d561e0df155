// What a document / prefix mask comes to: which keys a query sees is one interval of positions, and so is which queries see a
// key.  mcb_attention_mask works these out once for a batch, with the tiles' ranges and an order of the tiles, for all the
// attention calls that run under the mask (attn_mask.cu writes the block, masked_attn.cu and flash_attn.cu read it).
#pragma once
#include "common.cuh"

namespace mcb {
namespace amask {

constexpr int kTile = 128;          // positions of a tile: queries of a forward tile, keys of a dK / dV tile
constexpr int kStep = 64;           // positions of a block on the other side
constexpr int kChunk = 32768;       // positions under one word of the third bitmap level

// The mask block, all offsets in 4-byte words from its 16-byte aligned start.
struct Layout {
  int64_t rows;     // int2 [batch, seq]: the keys [x, y) that query position i sees; x == y: none
  int64_t keys;     // int2 [batch, seq]: the queries [x, y) that see key position i
  int64_t qtiles;   // int2 [batch, tiles]: first key block (of 64) and number of blocks that the tile's queries see
  int64_t ktiles;   // int2 [batch, tiles]: first query block (of 64) and number of blocks that see the tile's keys
  int64_t qwork;    // int4 [batch * tiles]: the query tiles, the most key blocks first (of each sequence): sequence, tile, first block, blocks
  int64_t kwork;    // int4 [batch * tiles]: the key tiles, the most query blocks first
  int64_t ticket;   // int: tiles that are done while the block is being made
  int64_t bits;     // two three-level bitmaps per sequence: where runs begin, where a position is no prefix (of sequences beyond kChunk)
  int64_t bits_per_seq;
  int64_t words;    // in all
};
__host__ __device__ inline int64_t tiles_of(int64_t seq) { return (seq + kTile - 1) / kTile; }
__host__ __device__ inline Layout layout(int64_t batch, int64_t seq) {
  Layout l;
  const int64_t n = batch * seq, t = batch * tiles_of(seq), chunks = (seq + kChunk - 1) / kChunk;
  l.rows = 0;
  l.keys = l.rows + 2 * n;
  l.qtiles = l.keys + 2 * n;
  l.ktiles = l.qtiles + 2 * t;
  l.qwork = (l.ktiles + 2 * t + 3) & ~static_cast<int64_t>(3);   // 16-byte records
  l.kwork = l.qwork + 4 * t;
  l.ticket = l.kwork + 4 * t;
  l.bits = l.ticket + 1;
  l.bits_per_seq = seq > kChunk ? chunks * (1024 + 32 + 1) : 0;   // (shorter ones' bitmaps are in shared memory)
  l.words = l.bits + 2 * batch * l.bits_per_seq;
  return l;
}

struct View {
  const int2* rows;
  const int2* keys;
  const int4* qwork;
  const int4* kwork;
};
inline View view(const void* mask, int64_t batch, int64_t seq) {
  const Layout l = layout(batch, seq);
  const int* w = static_cast<const int*>(mask);
  View v;
  v.rows = reinterpret_cast<const int2*>(w + l.rows);
  v.keys = reinterpret_cast<const int2*>(w + l.keys);
  v.qwork = reinterpret_cast<const int4*>(w + l.qwork);
  v.kwork = reinterpret_cast<const int4*>(w + l.kwork);
  return v;
}

}  // namespace amask
}  // namespace mcb
