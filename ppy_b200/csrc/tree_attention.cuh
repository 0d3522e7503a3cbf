// What the two tree-attention kernels share: how long a sequence is, how a batch of sequences of
// different lengths is dealt to CTAs, and where a part leaves its result for the join.
#pragma once

#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/ppyb200.h"
#include "ppyb200_device.cuh"

namespace ppyb200 {
namespace tree {

using Args = ppyb200_tree_attention_args;

__device__ __forceinline__ void raise(int32_t* status) {
  if (status != nullptr) atomicMax(status, PPYB200_DEVICE_RAISED);
}

// The cache length and node count of a sequence, held inside the buffers whatever the device
// arrays say: nodes that do not fit behind the length are dropped, and the status raised.
__device__ __forceinline__ void sequence_extent(const Args& a, int b, int64_t& length,
                                                int& count, int32_t* status) {
  int64_t l = a.lengths[b];
  int64_t n = a.counts != nullptr ? a.counts[b] : (int32_t)a.nodes;
  bool bad = l < 0 || l > a.capacity || n < 0 || n > a.nodes;
  l = l < 0 ? 0 : (l > a.capacity ? a.capacity : l);
  n = n < 0 ? 0 : (n > a.nodes ? a.nodes : n);
  if (l + n > a.capacity) {
    n = a.capacity - l;
    bad = true;
  }
  if (bad) raise(status);
  length = l;
  count = (int)n;
}

// How the key tiles of all sequences are dealt to `slots` parts (slots >= batch): parts of up to
// C tiles, C the smallest size of at least `least` tiles that the slots suffice for whatever the
// lengths are. Sequence b takes ceil(T_b / C) consecutive parts of nearly equal size, so long
// and short sequences give parts alike. (sum ceil(T_b / C) < sum T_b / C + batch, so C =
// ceil(sum T / (slots - batch + 1)) is enough.)
struct Deal {
  int slots;
  int least;
  int streams;  // results a part leaves: 2 where a CTA's two streams split its keys
};

struct Part {
  int b = -1;         // -1: no work for this slot
  int64_t length;     // the sequence's extent
  int count;
  int64_t first, tiles;  // key tiles of this part
  int index, parts;      // which part of the sequence's, and how many
};

// Key tiles of a sequence: the cache's, and the nodes' in tiles of their own when `apart`.
template <int TILE, bool APART>
__device__ __forceinline__ int64_t key_tiles(int64_t length, int count) {
  if (count == 0) return 0;
  return APART ? (length + TILE - 1) / TILE + (count + TILE - 1) / TILE
               : (length + count + TILE - 1) / TILE;
}

template <int TILE, bool APART>
__device__ __forceinline__ int64_t part_size(const Args& a, const Deal& deal, int lane,
                                             int32_t* status) {
  int64_t total = 0;
  for (int b = lane; b < (int)a.batch; b += 32) {
    int64_t length;
    int count;
    sequence_extent(a, b, length, count, status);
    total += key_tiles<TILE, APART>(length, count);
  }
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) total += __shfl_xor_sync(0xffffffffu, total, w);
  const int64_t spare = deal.slots - a.batch + 1;
  const int64_t size = (total + spare - 1) / spare;
  return size > deal.least ? size : deal.least;
}

// The part of slot `slot` (a warp together; every lane gets it). Extents that were out of range
// raise `status`.
template <int TILE, bool APART>
__device__ __forceinline__ Part part_of(const Args& a, const Deal& deal, int slot, int32_t* status) {
  const int lane = threadIdx.x & 31;
  const int64_t size = part_size<TILE, APART>(a, deal, lane, status);
  Part part;
  int before = 0;
  for (int b0 = 0; b0 < (int)a.batch; b0 += 32) {
    int64_t length = 0, tiles = 0;
    int count = 0;
    if (b0 + lane < (int)a.batch) {
      sequence_extent(a, b0 + lane, length, count, nullptr);
      tiles = key_tiles<TILE, APART>(length, count);
    }
    const int mine = (int)((tiles + size - 1) / size);
    int run = mine;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, run, w);
      if (lane >= w) run += up;
    }
    const int first = before + run - mine;
    const unsigned hit = __ballot_sync(0xffffffffu, slot >= first && slot < first + mine);
    if (hit != 0) {
      const int l = __ffs(hit) - 1;
      part.b = b0 + l;
      part.length = __shfl_sync(0xffffffffu, length, l);
      part.count = __shfl_sync(0xffffffffu, count, l);
      tiles = __shfl_sync(0xffffffffu, tiles, l);
      part.parts = __shfl_sync(0xffffffffu, mine, l);
      part.index = slot - __shfl_sync(0xffffffffu, first, l);
      part.first = part.index * tiles / part.parts;
      part.tiles = (part.index + 1) * tiles / part.parts - part.first;
      return part;
    }
    before += __shfl_sync(0xffffffffu, run, 31);
  }
  return part;
}

// The slots of sequence b's parts: the first, and how many (a warp together).
template <int TILE, bool APART>
__device__ __forceinline__ int2 parts_of(const Args& a, const Deal& deal, int b) {
  const int lane = threadIdx.x & 31;
  const int64_t size = part_size<TILE, APART>(a, deal, lane, nullptr);
  int before = 0, mine = 0;
  for (int i = lane; i <= b; i += 32) {
    int64_t length;
    int count;
    sequence_extent(a, i, length, count, nullptr);
    const int parts = (int)((key_tiles<TILE, APART>(length, count) + size - 1) / size);
    if (i < b) before += parts;
    else mine = parts;
  }
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, w);
    mine += __shfl_xor_sync(0xffffffffu, mine, w);
  }
  return make_int2(before, mine);
}

// The workspace: unnormalised outputs [slots * streams][kv_heads][rows][D] f32 (rows = nodes x
// query heads a key head), then maximum (in powers of two) and sum [..][..][rows][2].
struct Results {
  float* out;
  float2* top;
  int64_t rows;
  int kv_heads;
  __host__ __device__ __forceinline__ Results(void* workspace, const Args& a, const Deal& deal,
                                              int dim) {
    rows = a.nodes * (a.heads / a.kv_heads);
    kv_heads = (int)a.kv_heads;
    out = static_cast<float*>(workspace);
    top = reinterpret_cast<float2*>(out + (int64_t)deal.slots * deal.streams * kv_heads * rows *
                                              dim);
  }
  __host__ __device__ __forceinline__ int64_t at(int64_t slot, int kvh, int64_t row) const {
    return (slot * kv_heads + kvh) * rows + row;
  }
  static int64_t bytes(const Args& a, const Deal& deal, int dim) {
    return (int64_t)deal.slots * deal.streams * a.nodes * a.heads * (dim + 2) * 4;
  }
};

}  // namespace tree
}  // namespace ppyb200
