// Stream-K schedule of the attention kernels: equal shares of the tile plan's
// cost-ordered work, walked piece by piece.  Params provides hkv, pairs,
// group, n_qtiles, blk_prefix, blk_count and tile_order.
#pragma once

#include "common.cuh"

namespace hsd {
namespace attn {

// A piece: blocks [b0, b1) of one item (query tile x head pair).
struct Piece {
  int qt, kvh, h0, nslot, b0, b1, nblk, item, start;
  int lo = -1, hp = 0;  // ordered tile index and head pair of the piece (lo < 0: none yet)
};

// Next piece of the work range [w, w1) (advances w).  Items are the query
// tiles in tile_order, each split into hkv x pairs head-pair items of
// blk_count[tile] blocks; W = sum of all items' blocks.  pc holds the
// previous piece of the walk (pc.lo < 0 before the first), which ended at an
// item boundary unless the range is exhausted.
template <class Params>
__device__ __forceinline__ bool next_piece(const Params& p, int& w, int w1, Piece& pc) {
  if (w >= w1) return false;
  const int per_tile = p.hkv * p.pairs;
  int lo, hp, c, b0;
  if (pc.lo >= 0) {
    // the walk continues where the previous piece ended (an item boundary):
    // the next head pair of the same tile, or the next non-empty tile
    b0 = 0;
    lo = pc.lo;
    c = pc.nblk;
    hp = pc.hp + 1;
    if (hp == per_tile) {
      hp = 0;
      do {
        ++lo;
        c = p.blk_prefix[lo + 1] - p.blk_prefix[lo];
      } while (c == 0);
      pc.qt = p.tile_order[lo];
    }
  } else {
    lo = 0;
    int hi = p.n_qtiles - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.blk_prefix[mid] * per_tile <= w)
        lo = mid;
      else
        hi = mid - 1;
    }
    pc.qt = p.tile_order[lo];
    c = p.blk_count[pc.qt];
    const int off = w - p.blk_prefix[lo] * per_tile;
    hp = off / c;
    b0 = off - hp * c;
  }
  pc.lo = lo;
  pc.hp = hp;
  pc.nblk = c;
  pc.b0 = b0;
  pc.b1 = min(c, b0 + (w1 - w));
  pc.item = lo * per_tile + hp;
  pc.start = w - b0;
  pc.kvh = hp / p.pairs;
  const int pair = hp - pc.kvh * p.pairs;
  pc.h0 = pc.kvh * p.group + 2 * pair;
  pc.nslot = (2 * pair + 1 < p.group) ? 2 : 1;
  w += pc.b1 - pc.b0;
  return true;
}

// First work index of CTA k in stream-K mode.
__device__ __forceinline__ int range_start(int k, int total, int g) {
  return int((int64_t(k) * total) / g);
}

}  // namespace attn
}  // namespace hsd
