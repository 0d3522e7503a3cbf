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
__device__ __forceinline__ void sequence_extent(const Args& a, int b, int& length, int& count,
                                                int32_t* status) {
  const int capacity = (int)a.capacity, nodes = (int)a.nodes;
  const int l = a.lengths[b], n = a.counts != nullptr ? a.counts[b] : nodes;
  length = min(max(l, 0), capacity);
  count = min(min(max(n, 0), nodes), capacity - length);
  if (length != l || count != n) raise(status);
}

// Zeros as the results of the nodes from `count` on that did not fit behind the length.
__device__ __forceinline__ void clear_dropped(const Args& a, int b, int count) {
  const int nodes = (int)a.nodes, n = a.counts != nullptr ? min(a.counts[b], nodes) : nodes;
  uint16_t* out = static_cast<uint16_t*>(a.out) + b * a.out_strides[0];
#pragma unroll 1
  for (int node = count; node < n; ++node)
#pragma unroll 1
    for (int head = 0; head < (int)a.heads; ++head) {
      uint16_t* row = out + node * a.out_strides[1] + head * a.out_strides[2];
#pragma unroll 1
      for (int x = 0; x < (int)a.head_dim; x += 8)
        *reinterpret_cast<uint4*>(row + x) = make_uint4(0, 0, 0, 0);
      if (a.lse != nullptr) a.lse[((int64_t)b * a.heads + head) * nodes + node] = 0.f;
    }
}

// How the work is dealt to CTAs. An item is a piece of one sequence's rows (item_rows of them) under
// one key head; its work is the key tiles it reads. All items, key head by key head, lie on one
// axis of tiles, and CTA c of G takes the tiles [c W / G, (c + 1) W / G) of it: equal shares
// whatever the lengths are, walked as segments of one item each. At most the first and the last
// segment of a CTA are less than an item; those leave their unnormalised results in the workspace
// for the join, a whole item is written out by its CTA. Where a CTA's streams split an
// item's keys, every segment leaves several results.
struct Deal {
  int grid;       // CTAs at most; fewer when each would have less than `least` tiles
  int least;
  int items;      // items a sequence and key head
  int item_rows;
  int group;      // query heads a key head
  int streams;    // results a segment leaves: several where streams or copies split its keys
  bool join;      // results go through the workspace; without it there is none to write to
};

struct Segment {
  int b, kvh;
  int row0;              // the item's first row
  int length, count;     // the sequence's extent
  int first, tiles;      // the key tiles to walk
  bool starts, whole;    // from the item's first tile; all of them, by one stream
  int number;            // the item's on the axis
  int last_cta;          // of those that share the item (where this segment starts it)
  int64_t result;        // the first in the workspace, unless whole
};

// a / b of numbers that are not negative: in 32 bits where they fit, several times as fast.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

// Key tiles of an item: the cache's, and the nodes' (in tiles of their own when APART), up to the
// last row's node where the nodes are a chain.
template <int TILE, bool APART>
__device__ __forceinline__ int item_tiles(const Args& a, const Deal& deal, int length, int count,
                                          int r) {
  const int row0 = r * deal.item_rows;
  if (row0 >= count * deal.group) return 0;
  int last = count;
  if (a.parents == nullptr)
    last = min(count, (row0 + deal.item_rows + deal.group - 1) / deal.group);
  return APART ? (length + TILE - 1) / TILE + (last + TILE - 1) / TILE
               : (length + last + TILE - 1) / TILE;
}

// The axis: tiles of one key head's items (`span`), the CTAs that share it, and a CTA's place.
template <int TILE, bool APART>
struct Walk {
  int64_t span, place;  // `place`: of the next tile, on the axis
  int own;              // tiles of the lane-th item, for `enter`
  int left, offset, ctas, cta, kvh, item;

  // A warp together. The first CTA's warps report extents that are out of range.
  __device__ __forceinline__ void measure(const Args& a, const Deal& deal, bool report) {
    const int lane = threadIdx.x & 31, items = (int)a.batch * deal.items;
    span = 0;
    own = 0;
#pragma unroll 1
    for (int i = lane; i < items; i += 32) {
      int length, count;
      sequence_extent(a, i / deal.items, length, count, report ? a.status : nullptr);
      if (report && count < (int)a.nodes) clear_dropped(a, i / deal.items, count);
      const int tiles = item_tiles<TILE, APART>(a, deal, length, count, i % deal.items);
      if (i < 32) own = tiles;
      span += tiles;
    }
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) span += __shfl_xor_sync(0xffffffffu, span, w);
    const int64_t most = quotient(span * a.kv_heads, deal.least);
    ctas = most < 1 ? 1 : most < deal.grid ? (int)most : deal.grid;
  }
  __device__ __forceinline__ int64_t start_of(const Args& a, int c) const {
    return quotient(c * (span * a.kv_heads), ctas);
  }
  // The CTA whose share holds tile w of the axis.
  __device__ __forceinline__ int cta_of(const Args& a, int64_t w) const {
    return (int)quotient((w + 1) * ctas - 1, span * a.kv_heads);
  }
  // The first of the results that CTA c leaves of an item (one a stream): a CTA has at most one
  // segment that continues an item and one that starts an item without ending it, and c + the
  // item's number on the axis tells all segments apart.
  __device__ __forceinline__ static int64_t result_of(const Deal& deal, int c, int number,
                                                      bool starts) {
    return deal.streams == 1 ? 2 * (int64_t)c + (starts ? 1 : 0)
                             : deal.streams * ((int64_t)c + number);
  }
  // To the start of CTA c's share (a warp together).
  __device__ __forceinline__ void enter(const Args& a, const Deal& deal, int c) {
    const int lane = threadIdx.x & 31, items = (int)a.batch * deal.items;
    cta = c;
    left = 0;
    kvh = item = 0;
    offset = 0;
    if (c >= ctas || span == 0) return;
    const int64_t start = start_of(a, c);
    place = start;
    left = (int)(start_of(a, c + 1) - start);
    kvh = (int)quotient(start, span);
    int64_t rest = start - kvh * span;
#pragma unroll 1
    for (int i0 = 0; i0 < items; i0 += 32) {
      int64_t tiles = i0 == 0 ? own : 0;
      if (i0 > 0 && i0 + lane < items) {
        int length, count;
        sequence_extent(a, (i0 + lane) / deal.items, length, count, nullptr);
        tiles = item_tiles<TILE, APART>(a, deal, length, count, (i0 + lane) % deal.items);
      }
      int64_t run = tiles;
#pragma unroll
      for (int w = 1; w < 32; w <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, run, w);
        if (lane >= w) run += up;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, rest < run);
      if (hit != 0) {
        const int l = __ffs(hit) - 1;
        item = i0 + l;
        offset = (int)(rest - __shfl_sync(0xffffffffu, run - tiles, l));
        return;
      }
      rest -= __shfl_sync(0xffffffffu, run, 31);
    }
  }
  // The next segment of the share; false behind its end.
  __device__ __forceinline__ bool next(const Args& a, const Deal& deal, Segment& s) {
    while (left > 0) {
      s.b = item / deal.items;
      const int r = item - s.b * deal.items;
      sequence_extent(a, s.b, s.length, s.count, nullptr);
      const int tiles = item_tiles<TILE, APART>(a, deal, s.length, s.count, r);
      if (offset < tiles) {
        s.kvh = kvh;
        s.row0 = r * deal.item_rows;
        s.first = offset;
        s.tiles = min(tiles - offset, left);
        s.starts = offset == 0;
        s.whole = s.tiles == tiles && deal.streams == 1;
        s.number = kvh * (int)a.batch * deal.items + item;
        s.result = result_of(deal, cta, s.number, s.starts);
        s.last_cta = s.tiles == tiles ? cta : cta_of(a, place + tiles - 1);
        place += s.tiles;
        left -= s.tiles;
        offset += s.tiles;
        return true;
      }
      offset = 0;
      if (++item == (int)a.batch * deal.items) {
        item = 0;
        ++kvh;
      }
    }
    return false;
  }
};

// The nodes whose first row lies in an item are appended by the segment that starts the item: nodes
// [x, y), none where the segment does not.
__device__ __forceinline__ int2 appended(const Deal& deal, const Segment& s) {
  if (!s.starts) return make_int2(0, 0);
  const int to = (s.row0 + deal.item_rows + deal.group - 1) / deal.group;
  return make_int2((s.row0 + deal.group - 1) / deal.group, min(s.count, to));
}

// Appends them, by `threads` threads of which this is the `thread`-th, four pieces in flight each.
template <class T>
__device__ __forceinline__ void append(const Args& a, const Deal& deal, const Segment& s,
                                       int thread, int threads) {
  const int2 nodes = appended(deal, s);
  const int from = nodes.x, to = nodes.y;
  if (from >= to) return;
  const T* k_new = static_cast<const T*>(a.k_new) + s.b * a.k_new_strides[0] +
                   s.kvh * a.k_new_strides[2];
  const T* v_new = static_cast<const T*>(a.v_new) + s.b * a.v_new_strides[0] +
                   s.kvh * a.v_new_strides[2];
  T* keys = static_cast<T*>(a.keys) + s.b * a.keys_strides[0] + s.kvh * a.keys_strides[1];
  T* values = static_cast<T*>(a.values) + s.b * a.values_strides[0] + s.kvh * a.values_strides[1];
  const int pieces = (int)a.head_dim / 8, total = (to - from) * pieces * 2;
  for (int i0 = thread; i0 < total; i0 += 4 * threads) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {  // keys and values in turn
      const int i = i0 + u * threads;
      const int64_t n = from + (i >> 1) / pieces;
      const int x = (i >> 1) % pieces * 8;
      if (i < total)
        v[u] = *reinterpret_cast<const uint4*>((i & 1) == 0 ? k_new + n * a.k_new_strides[1] + x
                                                            : v_new + n * a.v_new_strides[1] + x);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * threads;
      const int64_t n = from + (i >> 1) / pieces, j = s.length + n;
      const int x = (i >> 1) % pieces * 8;
      if (i < total)
        *reinterpret_cast<uint4*>((i & 1) == 0 ? keys + j * a.keys_strides[2] + x
                                               : values + j * a.values_strides[2] + x) = v[u];
    }
  }
}

// The workspace: unnormalised outputs of each result in f32, then maximum (in powers of two) and
// sum [results][rows][2], then the first and last CTA of each item on the axis. The outputs lie in
// blocks of eight rows, [rows / 8][D / 4][8][4]: threads with a row each then write whole lines
// (into rows 256 bytes apart a store of 32 lanes touched 32 lines, 2.3 us for 256 rows of 64).
struct Results {
  float* out;
  float2* top;
  int2* ctas;
  int rows, dim;  // of a result, the rows in eights
  __host__ __device__ __forceinline__ static int64_t count(const Args& a, const Deal& deal) {
    return deal.streams == 1 ? 2 * (int64_t)deal.grid
                             : deal.streams * (deal.grid + a.kv_heads * a.batch * deal.items);
  }
  __device__ __forceinline__ Results(const Args& a, const Deal& deal, int dim)
      : rows((deal.item_rows + 7) & ~7), dim(dim) {
    out = static_cast<float*>(a.workspace);
    top = reinterpret_cast<float2*>(out + count(a, deal) * rows * dim);
    ctas = reinterpret_cast<int2*>(top + count(a, deal) * rows);
  }
  __device__ __forceinline__ float2& top_of(int64_t result, int row) const {
    return top[result * rows + row];
  }
  // four columns of a row; the next four lie 32 further
  __device__ __forceinline__ float* out_of(int64_t result, int row, int piece) const {
    return out + (result * rows + (row & ~7)) * dim + piece * 32 + (row & 7) * 4;
  }
  static int64_t bytes(const Args& a, const Deal& deal, int dim) {
    return count(a, deal) * ((deal.item_rows + 7) & ~7) * (dim + 2) * 4 +
           a.kv_heads * a.batch * deal.items * 8;
  }
};

}  // namespace tree
}  // namespace ppyb200
