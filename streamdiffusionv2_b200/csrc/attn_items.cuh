// How the attention kernels over caches with one length per row find their share of the work.
#pragma once
#include <stdint.h>

#include "sdv2_internal.h"

namespace sdv2 {
namespace attnx {

struct Item {
  int b, h, tile;         // row, head, query tile
  int len;                // keys of the row (plans by length)
  int part, parts, slot;  // part < 0: the whole key range, written to the output directly
};

// Item i of a plan made by plan_lens().
__device__ __forceinline__ Item find_item_lens(const AttnXParams& p, int i) {
  Item it;
  it.part = -1;
  it.parts = 1;
  it.slot = 0;
  int tile = i;
  if (i >= p.n_full) {
    const int k = i - p.n_full;
    int r = p.rows - 1;
    while (r > 0 && p.by_length[r].item0 > k) --r;
    it.parts = p.by_length[r].parts;
    const int local = k - p.by_length[r].item0;
    tile = p.by_length[r].tail_tile0 + local / it.parts;
    if (it.parts > 1) it.part = local % it.parts;
    it.slot = k;
  }
  it.tile = tile % p.pair_tiles;
  const int hb = tile / p.pair_tiles;
  it.h = hb % p.heads;
  it.b = p.by_length[hb / p.heads].row;
  it.len = p.by_length[hb / p.heads].len;
  return it;
}

// The first item of tail tile t.
__device__ __forceinline__ int first_item_lens(const AttnXParams& p, int t) {
  const int tile = p.n_full + t;
  int r = p.rows - 1;
  while (r > 0 && p.by_length[r].tail_tile0 > tile) --r;
  return p.n_full + p.by_length[r].item0 + (tile - p.by_length[r].tail_tile0) * p.by_length[r].parts;
}

__device__ __forceinline__ float exp2_int(int e) {  // 2^e, e clamped to fp32's normal range
  return __int_as_float((min(max(e, -126), 127) + 127) << 23);
}

}  // namespace attnx
}  // namespace sdv2
