// How a tree-attention call is laid out, on the host: which kernel takes it, how its rows lie in
// tiles, how many CTAs share the key tiles, and what workspace their results need.
#pragma once

#include "tree_attention.cuh"

namespace ppyb200 {
namespace tree {

constexpr int kNarrowTile = 64, kNarrowRows = 16;  // the narrow kernel: keys a tile, rows a CTA
constexpr int kKeysTile = 128;  // the wide kernel: keys a tile
constexpr int kRowsTile = 128;  // and rows a stream

struct WideRows {
  int tile_nodes;  // nodes of a row tile (tile_nodes x group <= 128 / copies)
  bool share;      // two row tiles an item, sharing the key tiles; else two streams over the keys
  int copies;      // of the rows in a query tile (1 when shared)
};

// How the rows lie in tiles; tile_nodes 0 when a key head's group does not fit a tile.
inline WideRows wide_rows(const Args& a) {
  WideRows w;
  const int group = (int)(a.heads / a.kv_heads);
  w.copies = a.nodes <= 32 / group ? 4 : a.nodes <= 64 / group ? 2 : 1;
  w.tile_nodes = kRowsTile / w.copies / group;
  w.share = w.tile_nodes > 0 && a.nodes > w.tile_nodes;
  if (w.tile_nodes > a.nodes) w.tile_nodes = (int)a.nodes;
  return w;
}

struct Plan {
  bool wide;
  WideRows rows;  // of the wide kernel
  Deal deal;
  int64_t workspace;
};

inline int padded_dim(int64_t head_dim) { return head_dim <= 64 ? 64 : 128; }

// What the tensor-core kernel takes: a positive scale (it keeps maxima of unscaled scores), query
// heads a key head that fit a row tile, and tensors that tensor maps describe.
inline bool wide_fits(const Args& a) {
  return a.heads / a.kv_heads <= kRowsTile && a.head_dim > 32;
}
inline bool strides_fit(const int64_t (&strides)[3], int64_t n0, int64_t n1, int64_t n2) {
  const int64_t n[3] = {n0, n1, n2};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (strides[i] <= 0 || strides[i] >= (1ll << 39))) return false;
  return true;
}

// Which kernel is the faster, by the bytes of a full cache (the lengths are on the device). The
// narrow kernel starts and ends an item in about 2 us where the wide one takes 6, and reads the
// cache once per 16 rows at up to 4.6 TB/s, the wide one once at up to 5.5. Measured, wide
// against narrow, us: one row, 12 heads of 64, 1 sequence of 1000 entries (3 MB) 19.7 / 10.0,
// 64 of 750 (144 MB) 71.8 / 51.5; 4 rows, 8 heads of 128, 64 of 1500 (384 MB) 95.8 / 93.1, 16 of
// 8000 (504 MB) 95.7 / 109.7; trees of 32 nodes, 12 heads of 64, 8 of 1000 (26 MB) 26.3 / 28.7; of
// 64 nodes, 2 sequences (6 MB) 21.7 / 23.6, 4 (13 MB) 22.5 / 29.5, 64 (204 MB) 110 / 249. A cache
// that is mostly empty counts as a full one: 64 of 750 entries in slots for 16384 go to the wide
// kernel, 73.3 / 52.4.
inline bool narrow_faster(const Args& a) {
  const int64_t rows = a.nodes * (a.heads / a.kv_heads), item = a.capacity * a.head_dim * 4;
  const int64_t cache = a.batch * a.kv_heads * item, tiles = (rows + kNarrowRows - 1) / kNarrowRows;
  if (tiles <= 1) return item < (1 << 20) || cache < (256 << 20);
  return tiles <= 4 && cache * tiles * tiles < (160 << 20);
}

inline bool wide_takes(const Args& a) {
  return wide_fits(a) && !narrow_faster(a) && a.scale > 0 && a.capacity > 0 &&
         strides_fit(a.q_strides, a.batch, a.nodes, a.heads) &&
         strides_fit(a.k_new_strides, a.batch, a.nodes, a.kv_heads) &&
         strides_fit(a.v_new_strides, a.batch, a.nodes, a.kv_heads) &&
         strides_fit(a.keys_strides, a.batch, a.kv_heads, a.capacity) &&
         strides_fit(a.values_strides, a.batch, a.kv_heads, a.capacity);
}

inline Plan plan_for(const Args& a, bool wide, int sm_count) {
  Plan p = {};
  p.wide = wide;
  const int64_t group = a.heads / a.kv_heads, rows = a.nodes * group;
  p.deal.group = (int)group;
  p.deal.least = 2;
  if (wide) {
    p.rows = wide_rows(a);
    p.deal.streams = p.rows.share ? 1 : 2 * p.rows.copies;
    p.deal.item_rows = (int)(p.rows.tile_nodes * group * (p.rows.share ? 2 : 1));
    p.deal.grid = sm_count;
  } else {
    p.deal.streams = 1;
    p.deal.item_rows = kNarrowRows;
    p.deal.grid = sm_count * (a.head_dim <= 64 ? 4 : 2);
  }
  p.deal.items = (int)((rows + p.deal.item_rows - 1) / p.deal.item_rows);
  // no more CTAs than a full cache has work for
  const int64_t tile = wide ? kKeysTile : kNarrowTile;
  const int64_t work = a.batch * a.kv_heads * p.deal.items *
                       ((a.capacity + tile - 1) / tile + (wide ? (a.nodes + tile - 1) / tile : 0));
  const int64_t most = work / p.deal.least;
  if (p.deal.grid > most) p.deal.grid = most < 1 ? 1 : (int)most;
  // some item may have several results; one CTA writes whole items, and no workspace
  p.deal.join = p.deal.streams > 1 || p.deal.grid > 1;
  p.workspace = p.deal.join ? Results::bytes(a, p.deal, padded_dim(a.head_dim)) : 0;
  return p;
}

}  // namespace tree
}  // namespace ppyb200
