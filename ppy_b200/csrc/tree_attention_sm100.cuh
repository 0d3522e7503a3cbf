// The tree attention's tensor-core kernel, for key heads with many query rows (nodes x the
// query heads that share the key head): tcgen05 products with TMEM accumulators, fed by TMA.
//
// A CTA an SM walks its share of the work (Walk): segments of key tiles (128 keys each: the cache's,
// then the nodes' own) of one sequence and key head, with two streams, each a query tile of 128
// rows with its own softmax warpgroup and MMA issuer, so that one stream's products run while the
// other's softmax does:
//   rows > 128   the streams hold two row tiles and share every key tile (read once for 256 rows)
//   rows <= 128  the streams hold the same rows and take the key tiles in turn
//   rows <= 64   the same, and a query tile holds its rows twice (four times up to 32 rows): each
//                copy weighs a half (a quarter) of a tile's keys, with zeros for the others, so
//                that all eight softmax warps have rows and each less to do
// Streams that split an item's keys, and copies, leave results of their own for the join.
// Per key tile and stream:
//   S = Q K^T   M = 128, N = 128, both operands K-major with the 128-byte swizzle; the query rows
//               of a tile come as one box [nodes][heads of the group][64 columns]
//   softmax     a row a thread, f32, the running maximum moved only when a score exceeds it by
//               2^kMove (the weights of the tile are at most that then, exact for the quotient)
//   O += P V    P from TMEM in the values' type (rounded to half a step, as the prompt
//               attention's), V as it lies in the cache: [keys][64 columns] boxes are the
//               MN-major form of the operand, no transposed copy
// TMEM: D = 64: S 2 x 128 columns, O 2 x 64, P 2 x 64, and S of the next tile runs during the
// softmax. D = 128: S 2 x 128, O 2 x 128, and P lies over its S; S of the next tile follows the
// product that reads P (MMAs of one thread run in order).
//
// Tiles with masked keys (the cache's last, and the nodes') have their hidden values cleaned in
// shared memory before the product: rows behind the sequence are zeroed, and so are single
// values of nodes that are not finite, which the last step adds to the rows that see them.
//
//   warps 0-7  softmax (warpgroup t = stream t; warp w reads TMEM lanes 32 (w % 4) ...)
//   warp 8     TMA loads of Q, K and V (a ring of K and V tiles in turn), by one thread
//   warps 9,10 one thread each: the MMAs of stream 0 and 1; warp 9 owns the TMEM
//   warp 11    appends a segment's nodes to the cache, unless they are many
//
// Every mbarrier wait is bounded: on giving up the CTA raises the status, every role leaves its
// loop, copies and MMAs in flight are drained and the TMEM is freed. Rows left without a result get
// NaN, so that a caller without a status word does not take old memory for one.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "gemm_sm100.cuh"
#include "mma16.cuh"
#include "tmem.cuh"
#include "tree_attention.cuh"
#include "tree_attention_plan.cuh"

namespace ppyb200 {
namespace tree {

using namespace tmem;
using gemm::mbar_arrive;
using gemm::mbar_drain_wait;
using gemm::mbar_expect_tx;
using gemm::mbar_init;
using gemm::mbar_try_wait;
using gemm::tc_fence_after;
using gemm::tc_fence_before;
using mma16::exp2_sfu;
using mma16::finite_only;
using mma16::Kind;

constexpr int kWideThreads = 384;
// Registers a thread after the split (setmaxnreg): the softmax warpgroups hold a row of 128 scores
// and take what the third warpgroup gives up. The launch holds kLaunchRegs x 384, and the split
// must not ask for more: launch_wide checks the compiled count, since a split that the pool
// cannot meet would never return.
constexpr uint32_t kLaunchRegs = 168, kSoftmaxRegs = 224, kSupportRegs = 56;
static_assert(2 * 128 * kSoftmaxRegs + 128 * kSupportRegs <= kWideThreads * kLaunchRegs,
              "register split above the launch's registers");
constexpr uint32_t kWaitLimit = 1u << 22;  // tries of an mbarrier wait, unless a test sets others
// The running maximum moves when a score exceeds it by more than 2^kMove, and weights are held
// times 2^kLift until they are divided by their sum (lifted too): the two together stay within
// f16's 2^15, whose small weights would vanish without the lift; bf16 has f32's range. A slack of
// 2^4 in place of 2^8 costs f16 nothing measurable: maxima settle within the first tiles.
template <class T>
constexpr float kMove = std::is_same<T, __half>::value ? 4.f : 8.f;
template <class T>
constexpr float kLift = std::is_same<T, __half>::value ? 11.f : 0.f;

constexpr int kBox = 128 * 64 * 2;  // 128 rows of 64 16-bit columns: one TMA box

template <int D>
struct WideShape {
  static constexpr int kBoxes = D / 64;
  static constexpr int kTileBytes = kBoxes * kBox;  // a K, V or Q tile
  static constexpr int kSlots = D == 64 ? 10 : 5;   // K and V tiles in the ring
  static constexpr int kTrees = D == 64 ? 8 : 4;    // more than the segments in the ring
  static constexpr bool kOver = D == 128;           // P lies over S
  static constexpr uint32_t kOCol = 256;
  static constexpr uint32_t kPCol = kOver ? 0 : 384;
  static constexpr uint32_t kPStep = kOver ? 128 : 64;
};

template <int D>
struct WideShared {
  alignas(1024) uint8_t q[2][WideShape<D>::kTileBytes];
  alignas(1024) uint8_t ring[WideShape<D>::kSlots][WideShape<D>::kTileBytes];
  alignas(8) uint64_t q_full, q_empty, full[WideShape<D>::kSlots], empty[WideShape<D>::kSlots];
  alignas(8) uint64_t s_full[2], s_free[2], p_full[2], o_done[2], turn[2], drain[2];
  uint32_t tmem_base;
  int abort;
  // a value among a segment's node tiles is not finite: the segment's mark, in turns of eight (the
  // ring holds five tiles, so no stream is eight segments ahead of the other)
  int spoiled[8];
  uint8_t parents[WideShape<D>::kTrees][256];  // of the last segments with node tiles
};

__device__ __forceinline__ void support_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSupportRegs));
}
__device__ __forceinline__ void softmax_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
}

// The ring's entries. Streams that share their tiles take every entry in one order. Streams that do
// not have slots of their own (the first kSlots - kSlots / 2, and the rest): loads complete in
// any order, and a stream that came round to a slot of the other's could take the completion
// before last for its own, the barrier's phases being told apart by parity only.
template <int D>
struct Entry {
  int slot;
  uint32_t parity;
  static constexpr int kAll = WideShape<D>::kSlots, kRest = kAll / 2, kFirst = kAll - kRest;
  __device__ __forceinline__ static int slots(bool share, int t) {
    return share ? kAll : t == 0 ? kFirst : kRest;
  }
  __device__ __forceinline__ Entry(bool share, int t, int e) {
    const int round = share ? e / kAll : t == 0 ? e / kFirst : e / kRest;
    slot = e - round * slots(share, t) + (share || t == 0 ? 0 : kFirst);
    parity = (uint32_t)(round & 1);
  }
};

// The launch's tensor maps: [columns][slots or nodes][key heads][batch], and for q [columns]
// [heads][nodes][batch].
struct WideMaps {
  CUtensorMap q, keys, values, k_new, v_new;
};

template <class Layout>
__device__ __forceinline__ bool wide_wait(Layout& s, uint64_t* bar, uint32_t parity,
                                          int32_t* status, uint32_t limit) {
  for (uint32_t tries = 0; tries < limit; ++tries) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*(volatile int*)&s.abort) return false;
  }
  *(volatile int*)&s.abort = 1;
  raise(status);
  return false;
}
template <class Layout>
__device__ __forceinline__ bool wide_warp_wait(Layout& s, uint64_t* bar, uint32_t parity,
                                               int32_t* status, uint32_t limit) {
  return __all_sync(0xffffffffu, wide_wait(s, bar, parity, status, limit)) != 0;
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int32_t x, int32_t y, int32_t z, int32_t w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// An MN-major tile with the 128-byte swizzle: 64-column boxes kBox bytes apart (leading offset),
// 1024 bytes between groups of eight keys (stride offset).
__device__ __forceinline__ uint64_t smem_desc_mn(const void* tile) {
  const uint64_t addr = smem_u32(tile);
  return ((addr & 0x3FFFFull) >> 4) | ((uint64_t)(kBox >> 4) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

template <class T>
constexpr uint32_t type_bits() {  // a and b format: 0 f16, 1 bf16
  return sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
}
template <class T>
constexpr uint32_t idesc_s() {
  return (1u << 4) | type_bits<T>() | ((uint32_t)(kKeysTile >> 3) << 17) |
         ((uint32_t)(kRowsTile >> 4) << 24);
}
template <class T, int D>
constexpr uint32_t idesc_o() {  // B (the values) MN-major
  return (1u << 4) | type_bits<T>() | (1u << 16) | ((uint32_t)(D >> 3) << 17) |
         ((uint32_t)(kRowsTile >> 4) << 24);
}

// Which keys of a tile a row sees, a bit each.
struct Sight {
  uint64_t lo, hi;
  __device__ __forceinline__ static Sight first(int n) {  // keys 0 .. n - 1
    Sight s;
    s.lo = n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1;
    n -= 64;
    s.hi = n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1;
    return s;
  }
  __device__ __forceinline__ void add(int key) {
    if (key < 64) lo |= 1ull << key;
    else hi |= 1ull << (key - 64);
  }
  __device__ __forceinline__ bool has(int key) const {
    return (((key < 64 ? lo : hi) >> (key & 63)) & 1ull) != 0;
  }
};

// What node `node` sees of the node tile that starts at node n0 (parents null: of a chain).
__device__ __forceinline__ Sight node_sight(const uint8_t* parents, int node, int n0, int count) {
  if (parents == nullptr) return Sight::first(min(node + 1, count) - n0);
  Sight s = Sight::first(0);
  for (int i = node;;) {
    if (i >= n0 && i < n0 + kKeysTile) s.add(i - n0);
    const int p = parents[i];
    if (p == 255) return s;  // a root
    i = p;
  }
}

// After a wait that gave up: NaN as the result of a softmax thread's row of every segment of the CTA's,
// those that it had finished among them. A function of its own, for the registers' sake.
template <class T, int D, int COPIES>
__device__ __noinline__ void leave_nan(const Args& a, const Deal& deal, const WideRows& wide) {
  const int lane_row = threadIdx.x % 128, t = threadIdx.x / 128;
  const int row = lane_row % (128 / COPIES), copy = lane_row / (128 / COPIES);
  const float nan = __uint_as_float(0x7fc00000u);
  const Results results(a, deal, D);
  Walk<kKeysTile, true> walk;
  walk.measure(a, deal, false);
  walk.enter(a, deal, blockIdx.x);
  Segment seg;
  while (walk.next(a, deal, seg)) {
    const int tile_row = (wide.share ? t * wide.tile_nodes * deal.group : 0) + row;
    const int node = (seg.row0 + tile_row) / deal.group;
    const int head = seg.kvh * deal.group + tile_row % deal.group;
    if (row >= wide.tile_nodes * deal.group || node >= seg.count) continue;
    if (!seg.whole) {
      results.top_of(seg.result + (wide.share ? 0 : t * COPIES + copy), tile_row) =
          make_float2(nan, nan);
      continue;
    }
    T* out = static_cast<T*>(a.out) + seg.b * a.out_strides[0] + node * a.out_strides[1] +
             head * a.out_strides[2];
    for (int x = 0; x < (int)a.head_dim; x += 2)
      *reinterpret_cast<uint32_t*>(out + x) = Kind<T>::pack(nan, nan);
    if (a.lse != nullptr) a.lse[((int64_t)seg.b * a.heads + head) * a.nodes + node] = nan;
  }
}

template <class T, int D, int COPIES>
__global__ void __launch_bounds__(kWideThreads, 1)
wide_kernel(const __grid_constant__ WideMaps maps, const __grid_constant__ Args a,
            const __grid_constant__ Deal deal, const __grid_constant__ WideRows wide,
            const uint32_t limit) {
  using Shape = WideShape<D>;
  constexpr int kSpan = 128 / COPIES;  // rows of a copy, and keys of a tile that it weighs
  extern __shared__ uint8_t smem_raw[];
  WideShared<D>& s = *reinterpret_cast<WideShared<D>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&s.q_full, 1);
    mbar_init(&s.q_empty, 2);
    for (int i = 0; i < Shape::kSlots; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], wide.share ? 2 : 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s.s_full[t], 1);
      mbar_init(&s.s_free[t], 4);
      mbar_init(&s.p_full[t], 4);
      mbar_init(&s.o_done[t], 1);
      mbar_init(&s.turn[t], 4);
      mbar_init(&s.drain[t], 1);
    }
    s.abort = 0;
    for (int i = 0; i < 8; ++i) s.spoiled[i] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&s.tmem_base)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  // the set-up above overlaps the previous kernel; its results are needed from here on
  pdl_wait();
  Walk<kKeysTile, true> walk;
  walk.measure(a, deal, blockIdx.x == 0);
  walk.enter(a, deal, blockIdx.x);
  const int group = deal.group, d = (int)a.head_dim;
  // Stream t of a segment walks its tiles t, t + 2, ..., or all of them when the streams share
  // them. Rows of the second row tile may be missing (`both` false): its stream is idle then.
  auto both_of = [&](const Segment& seg) {
    return !wide.share || seg.row0 + wide.tile_nodes * group < seg.count * group;
  };
  auto count_of = [&](const Segment& seg, int t) -> int {
    if (wide.share) return t == 0 || both_of(seg) ? seg.tiles : 0;
    return (seg.tiles - t + 1) / 2;
  };
  auto index_of = [&](int t, int k) { return wide.share ? k : 2 * k + t; };
  auto cache_tiles_of = [&](const Segment& seg) {
    return (seg.length + kKeysTile - 1) / kKeysTile;
  };
  // Up to 1024 elements of K and V one warp appends (two rounds of loads and stores) while the others
  // walk a tile. The softmax warps do more than that, while the segment's first loads are under way:
  // 64 nodes of 64 took the one warp 6 us, past the end of a short segment.
  auto many_of = [&](const Segment& seg) {
    const int2 nodes = appended(deal, seg);
    return (nodes.y - nodes.x) * d > 1024;
  };
  Segment seg;

  if (warp == 8) {
    support_registers();
    // ---- loader: lane 0 loads a segment's Q, then K and V of its tiles (K of the CTA's i-th tile
    // is entry 2 i of the ring, its V entry 2 i + 1); the warp together leaves a tree's parents in
    // shared memory before the first node tile
    const uint32_t q_bytes = (uint32_t)(COPIES * Shape::kBoxes * wide.tile_nodes * group * 128);
    int loaded[2] = {0, 0}, segments = 0;  // entries of each stream (of both, when they share)
    bool ok = true;
    for (; ok && walk.next(a, deal, seg); ++segments) {
      const int cache_tiles = cache_tiles_of(seg);
      const bool tree = a.parents != nullptr && seg.first + seg.tiles > cache_tiles;
      int parent[8];
      if (tree) {
        const int32_t* from = a.parents + (int64_t)seg.b * a.parents_stride;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          parent[i] = i * 32 + lane < seg.count ? from[i * 32 + lane] : -1;
      }
      if (lane == 0) {
        ok = wide_wait(s, &s.q_empty, (uint32_t)((segments & 1) ^ 1), a.status, limit);
        if (ok) {
          const int streams = both_of(seg) ? 2 : 1;
          const int node0 = seg.row0 / group;
          mbar_expect_tx(&s.q_full, streams * q_bytes);
          for (int t = 0; t < streams; ++t)
            for (int x = 0; x < Shape::kBoxes * COPIES; ++x)
              tma_load_4d(s.q[t] + x * (kBox / COPIES), &maps.q, &s.q_full, x / COPIES * 64,
                          seg.kvh * group, node0 + (wide.share ? t * wide.tile_nodes : 0),
                          seg.b);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      if (!ok) break;
      for (int part = 0; part < 2; ++part) {  // the cache's tiles, then the nodes'
        const bool own = part == 1;
        const int from = own ? max(seg.first, cache_tiles) : seg.first;
        const int to = own ? seg.first + seg.tiles : min(seg.first + seg.tiles, cache_tiles);
        if (own && tree) {
          // up to 256 nodes: each parent a byte, 255 for a root, as any that is no earlier node
          // is taken
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int node = i * 32 + lane, p = parent[i];
            if (p < -1 || (p >= node && node < seg.count)) raise(a.status);
            s.parents[segments % Shape::kTrees][node] =
                p >= 0 && p < node ? (uint8_t)p : (uint8_t)255;
          }
          __syncwarp();
        }
        if (lane == 0) {
          for (int tile = from; tile < to && ok; ++tile) {
            const int at = (own ? tile - cache_tiles : tile) * kKeysTile;
            const int t = wide.share ? 0 : (tile - seg.first) & 1;
            for (int v = 0; v < 2; ++v) {
              const Entry<D> entry(wide.share, t, t == 0 ? loaded[0] : loaded[1]);
              if (!wide_wait(s, &s.empty[entry.slot], entry.parity ^ 1, a.status, limit)) {
                ok = false;
                break;
              }
              const CUtensorMap* map = own ? (v == 0 ? &maps.k_new : &maps.v_new)
                                           : (v == 0 ? &maps.keys : &maps.values);
              mbar_expect_tx(&s.full[entry.slot], Shape::kTileBytes);
              for (int x = 0; x < Shape::kBoxes; ++x)
                tma_load_4d(s.ring[entry.slot] + x * kBox, map, &s.full[entry.slot], x * 64, at,
                            seg.kvh, seg.b);
              if (t == 0) ++loaded[0];
              else ++loaded[1];
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      }
    }
    if (lane == 0) {
      // the copies issued here land before the CTA may leave
      for (int t = 0; t < 2; ++t)
        for (int e = max(0, loaded[t] - Entry<D>::slots(wide.share, t)); e < loaded[t]; ++e) {
          const Entry<D> entry(wide.share, t, e);
          mbar_drain_wait(&s.full[entry.slot], entry.parity);
        }
      if (segments > 0) mbar_drain_wait(&s.q_full, (uint32_t)((segments - 1) & 1));
    }
  } else if (warp == 9 || warp == 10) {
    support_registers();
    if (lane == 0) {
      // ---- MMA issuer of stream t. tcgen05.commit tracks the products of the committing thread:
      // a commit to `empty` frees a ring entry of this stream's; for an entry (and a Q) that it has
      // no product of, where the other stream has, it arrives once the load is there, so that
      // the arrival falls in the phase it belongs to.
      const int t = warp - 9;
      const uint32_t s_col = tmem + (uint32_t)(t * kKeysTile);
      const uint32_t o_col = tmem + Shape::kOCol + (uint32_t)(t * D);
      const uint32_t p_col = tmem + Shape::kPCol + (uint32_t)(t * Shape::kPStep);
      int base = 0, n = 0, segments = 0;  // tiles so far: of both streams, and of this one
      bool ok = true;
      auto full = [&](const Entry<D>& entry) {
        return wide_wait(s, &s.full[entry.slot], entry.parity, a.status, limit);
      };
      auto entry_of = [&](int k, int v) {  // K (v = 0) or V of this stream's tile k
        return Entry<D>(wide.share, t, 2 * ((wide.share ? base : n) + k) + v);
      };
      // S = Q K^T of this stream's tile k of the segment, its (n + k)-th in all
      auto scores = [&](int k) -> bool {
        const Entry<D> entry = entry_of(k, 0);
        if (!full(entry)) return false;
        if (!Shape::kOver && n + k > 0 &&
            !wide_wait(s, &s.s_free[t], (uint32_t)((n + k - 1) & 1), a.status, limit))
          return false;
        tc_fence_after();
        const uint8_t* key = s.ring[entry.slot];
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int box = kk >> 2, off = (kk & 3) * 2;
          mma(s_col, gemm::smem_desc(s.q[t] + box * kBox) + (uint64_t)off,
              gemm::smem_desc(key + box * kBox) + (uint64_t)off, idesc_s<T>(),
              kk > 0 ? 1u : 0u);
        }
        commit(&s.s_full[t]);
        commit(&s.empty[entry.slot]);
        return true;
      };
      // O += P V of tile k
      auto product = [&](int k) -> bool {
        const Entry<D> entry = entry_of(k, 1);
        if (!full(entry) || !wide_wait(s, &s.p_full[t], (uint32_t)((n + k) & 1), a.status, limit))
          return false;
        tc_fence_after();
        const uint64_t value = smem_desc_mn(s.ring[entry.slot]);
#pragma unroll
        for (int kk = 0; kk < kKeysTile / 16; ++kk)  // 16 keys: two groups of 1024 bytes
          mma_ts(o_col, p_col + (uint32_t)(kk * 8), value + (uint64_t)(kk * (2048 >> 4)),
                 idesc_o<T, D>(), k > 0 || kk > 0 ? 1u : 0u);
        commit(&s.o_done[t]);
        commit(&s.empty[entry.slot]);
        return true;
      };
      for (; ok && walk.next(a, deal, seg); ++segments) {
        const int mine = count_of(seg, t);
        if (!wide_wait(s, &s.q_full, (uint32_t)(segments & 1), a.status, limit)) break;
        if (mine == 0) {
          mbar_arrive(&s.q_empty);
          for (int i = 0; wide.share && ok && i < 2 * seg.tiles; ++i) {
            const Entry<D> entry = entry_of(i >> 1, i & 1);
            ok = full(entry);
            if (ok) mbar_arrive(&s.empty[entry.slot]);
          }
        } else {
          ok = scores(0);
          for (int k = 0; k < mine && ok; ++k) {
            if (k + 1 == mine) commit(&s.q_empty);
            if (!Shape::kOver && k + 1 < mine) ok = scores(k + 1);
            ok = ok && product(k);
            if (Shape::kOver && k + 1 < mine) ok = ok && scores(k + 1);
          }
        }
        base += seg.tiles;
        n += mine;
      }
      commit(&s.drain[t]);
      mbar_drain_wait(&s.drain[t], 0);
    }
  } else if (warp == 11) {
    support_registers();
    // ---- append, and where the join finds an item's results
    while (walk.next(a, deal, seg)) {
      if (deal.join && seg.starts && lane == 0)
        Results(a, deal, D).ctas[seg.number] = make_int2(blockIdx.x, seg.last_cta);
      if (!many_of(seg)) append<T>(a, deal, seg, lane, 32);
    }
  } else {
    softmax_registers();
    // ---- softmax: warpgroup t, thread = row (a TMEM lane) and, when cleaning, a key
    const int t = warp >> 2;
    const int lane_row = (warp & 3) * 32 + lane;
    const int row = lane_row % kSpan;                   // of the row tile
    const int key0 = (warp & 3) * 32 / kSpan * kSpan;  // first of the tile's keys that it weighs
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lane_addr + (uint32_t)(t * kKeysTile);
    const uint32_t o_addr = tmem + lane_addr + Shape::kOCol + (uint32_t)(t * D);
    const uint32_t p_addr = tmem + lane_addr + Shape::kPCol + (uint32_t)(t * Shape::kPStep);
    const float scale_log2 = (float)a.scale * mma16::kLog2e;
    const uint64_t scale2 = f2(scale_log2, scale_log2);
    const Results results(a, deal, D);
    if (COPIES > 1 && !Shape::kOver) {
      // the weights of the keys that other copies weigh: zero throughout
      const uint32_t zeros[16] = {};
#pragma unroll
      for (int q = 0; q < 4; ++q) tmem_st16(p_addr + (uint32_t)(q * 16), zeros);
      tmem_wait_st();
    }
    int base = 0, n = 0;  // as the MMA issuer's
    int mark = 1;             // this segment's, in `spoiled`
    int turn = 0;         // tiles of shared segments so far
    bool ok = true;
    while (ok && walk.next(a, deal, seg)) {
      if (many_of(seg)) append<T>(a, deal, seg, threadIdx.x, 256);
      const int mine = count_of(seg, t);
      const bool turns = Shape::kOver && wide.share && both_of(seg);
      const int cache_tiles = cache_tiles_of(seg);
      const int tile_row = (wide.share ? t * wide.tile_nodes * group : 0) + row;  // of the item
      const int node = (seg.row0 + tile_row) / group;
      const int first_node = (seg.row0 + tile_row - row) / group;  // of the stream's rows
      const bool real = row < wide.tile_nodes * group && node < seg.count;
      const bool busy = __any_sync(0xffffffffu, real) != 0;  // the warp has rows
      // the loader's, there before the first node tile's keys
      const uint8_t* parents =
          a.parents == nullptr ? nullptr : s.parents[(mark - 1) % Shape::kTrees];
      const T* v_new = static_cast<const T*>(a.v_new) + seg.b * a.v_new_strides[0] +
                       seg.kvh * a.v_new_strides[2];
      float m = -INFINITY, l = 0.f;  // m in raw score units
      for (int k = 0; k < mine; ++k) {
        const uint32_t phase = (uint32_t)((n + k) & 1);
        if (!wide_warp_wait(s, &s.s_full[t], phase, a.status, limit)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int tile = seg.first + index_of(t, k);
        const bool own = tile >= cache_tiles;
        const int left = own ? 0 : seg.length - tile * kKeysTile;
        // a chain's node tiles before the stream's first node are seen whole
        const bool ragged =
            own ? a.parents != nullptr || (tile - cache_tiles + 1) * kKeysTile > first_node + 1
                : left < kKeysTile;
        if (busy) {
          float sv[kSpan];
#pragma unroll
          for (int c = 0; c < kSpan / 32; ++c)
            tmem_ld32_nowait(s_addr + (uint32_t)(key0 + c * 32), sv + c * 32);
          tmem_wait_ld();
          if (!Shape::kOver) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.s_free[t]);
          }
          if (ragged) {
            const Sight sees =
                !own ? Sight::first(left)
                     : real ? node_sight(parents, node, (tile - cache_tiles) * kKeysTile,
                                         seg.count)
                            : Sight::first(0);
            const uint64_t low = key0 < 64 ? sees.lo >> key0 : sees.hi >> (key0 - 64);
#pragma unroll
            for (int c = 0; c < kSpan; ++c)
              if ((((c < 64 ? low : sees.hi) >> (c & 63)) & 1ull) == 0) sv[c] = -INFINITY;
            __syncwarp();  // the walks differ; tensor memory is accessed by whole warps
          }
          float mx[4] = {m, m, m, m};
#pragma unroll
          for (int c = 0; c < kSpan; c += 8) {
            mx[0] = max3(mx[0], sv[c + 0], sv[c + 1]);
            mx[1] = max3(mx[1], sv[c + 2], sv[c + 3]);
            mx[2] = max3(mx[2], sv[c + 4], sv[c + 5]);
            mx[3] = max3(mx[3], sv[c + 6], sv[c + 7]);
          }
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          // the maximum moves by more than 2^kMove, or stays; a row that has seen nothing yet
          // stays at -inf, its weights 2^-inf = 0
          const bool move = top != -INFINITY && !((top - m) * scale_log2 <= kMove<T>);
          float alpha = 1.f;
          if (move) {
            alpha = m == -INFINITY ? 0.f : exp2_sfu((m - top) * scale_log2);
            m = top;
            l *= alpha;
          }
          __syncwarp();
          const float shift = m == -INFINITY ? 0.f : kLift<T> - m * scale_log2;
          const uint64_t shift2 = f2(shift, shift);
          if (!Shape::kOver && k > 0) {
            // the product before this tile's reads P, which the stores below replace
            if (!wide_warp_wait(s, &s.o_done[t], phase ^ 1, a.status, limit)) {
              ok = false;
              break;
            }
            tc_fence_after();
          }
          // Streams that share their tiles take turns at the exponentials: both at once would each
          // take twice as long and leave the tensor core idle for as long.
          if (turns && (t == 1 || turn > 0) &&
              !wide_warp_wait(s, &s.turn[t], (uint32_t)((turn - (t == 0 ? 1 : 0)) & 1),
                              a.status, limit)) {
            ok = false;
            break;
          }
          uint64_t sum2[4] = {0, 0, 0, 0};
#pragma unroll
          for (int quarter = 0; quarter < kSpan / 32; ++quarter) {
            uint32_t pk[16];
#pragma unroll
            for (int c = quarter * 32; c < quarter * 32 + 32; c += 2) {
              float lo, hi;
              unf2(fma2(f2(sv[c], sv[c + 1]), scale2, shift2), lo, hi);
              const float e0 = exp2_sfu(lo), e1 = exp2_sfu(hi);
              sum2[(c >> 1) & 3] = add2(sum2[(c >> 1) & 3], f2(e0, e1));
              pk[(c >> 1) & 15] = Kind<T>::pack(e0, e1);
            }
            tmem_st16(p_addr + (uint32_t)(key0 / 2 + quarter * 16), pk);
          }
          if (COPIES > 1 && Shape::kOver) {
            // P lies over S: zeros over the scores that other copies weigh
            const uint32_t zeros[16] = {};
#pragma unroll
            for (int quarter = kSpan / 32; quarter < 4; ++quarter)
              tmem_st16(p_addr + (uint32_t)((key0 / 2 + quarter * 16) % 64), zeros);
          }
          if (turns) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.turn[t ^ 1]);
          }
          float s0, s1, s2, s3;
          unf2(add2(sum2[0], sum2[1]), s0, s1);
          unf2(add2(sum2[2], sum2[3]), s2, s3);
          l += (s0 + s1) + (s2 + s3);
          if (k > 0 && __any_sync(0xffffffffu, move)) {
            // scale O of the rows whose maximum moved. Every product before this tile's is
            // complete: S of this tile was issued behind the last (D = 128), or its barrier was
            // waited for above.
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float o[32];
              tmem_ld32_nowait(o_addr + (uint32_t)(c * 32), o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] *= alpha;
              tmem_st32(o_addr + (uint32_t)(c * 32), o);
            }
          }
          tmem_wait_st();
        } else {
          // no rows in this warp: it only keeps the barriers' counts (its P rows are never read
          // by a row that leaves the CTA), in step with the others: two arrivals of one warp in
          // a phase of p_full would stand for another's
          if (!Shape::kOver) {
            if (lane == 0) mbar_arrive(&s.s_free[t]);
            if (k > 0 && !wide_warp_wait(s, &s.o_done[t], phase ^ 1, a.status, limit)) {
              ok = false;
              break;
            }
          }
          if (turns) {
            if ((t == 1 || turn > 0) &&
                !wide_warp_wait(s, &s.turn[t], (uint32_t)((turn - (t == 0 ? 1 : 0)) & 1),
                                a.status, limit)) {
              ok = false;
              break;
            }
            if (lane == 0) mbar_arrive(&s.turn[t ^ 1]);
          }
        }
        turn += turns ? 1 : 0;
        if (ragged) {
          // clean the tile's values: thread = key
          const Entry<D> entry(wide.share, t, 2 * ((wide.share ? base : n) + k) + 1);
          if (!wide_warp_wait(s, &s.full[entry.slot], entry.parity, a.status, limit)) {
            ok = false;
            break;
          }
          uint8_t* line = s.ring[entry.slot] + lane_row * 128;
          const int real_keys =
              own ? seg.count - (tile - cache_tiles) * kKeysTile : left;
          // piece by piece in the order that lies in different banks for neighbouring keys
#pragma unroll 1
          for (int x = 0; x < Shape::kBoxes; ++x)
#pragma unroll 2
            for (int e = 0; e < 8; ++e) {
              uint4* piece = reinterpret_cast<uint4*>(line + x * kBox + ((e ^ (lane & 7)) << 4));
              if (lane_row >= real_keys) {
                *piece = make_uint4(0, 0, 0, 0);
              } else if (own) {
                const uint4 w = *piece;
                const uint4 clean = make_uint4(finite_only<T>(w.x), finite_only<T>(w.y),
                                               finite_only<T>(w.z), finite_only<T>(w.w));
                if (clean.x != w.x || clean.y != w.y || clean.z != w.z || clean.w != w.w) {
                  *(volatile int*)&s.spoiled[mark & 7] = mark;  // before the value goes
                  *piece = clean;
                }
              }
            }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full[t]);
      }
      // the row's result, once the stream's last product has completed
      if (ok && mine > 0) {
        ok = wide_warp_wait(s, &s.o_done[t], (uint32_t)((n + mine - 1) & 1), a.status, limit);
        tc_fence_after();
      }
      if (ok && busy) {
        const bool spoiled = mine > 0 && *(volatile int*)&s.spoiled[mark & 7] == mark;
        const int64_t result = seg.result + (wide.share ? 0 : t * COPIES + key0 / kSpan);
        const int head = seg.kvh * group + tile_row % group;
        const float inv = 1.f / l;
        T* out = static_cast<T*>(a.out) + seg.b * a.out_strides[0] + node * a.out_strides[1] +
                 (int64_t)head * a.out_strides[2];
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          __syncwarp();  // rows differ in what they store; a tensor memory load is the whole warp's
          if (mine > 0) {
            tmem_ld32_nowait(o_addr + (uint32_t)(c * 32), o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
          if (spoiled && real) {
            // add what the cleaning took out, to the rows that see it
            for (int k = 0; k < mine; ++k) {
              const int tile = seg.first + index_of(t, k) - cache_tiles;
              if (tile < 0) continue;
              const int n0 = tile * kKeysTile;
              const Sight sees = node_sight(parents, node, n0, seg.count);
              for (int key = key0; key < key0 + kSpan && n0 + key < seg.count; ++key) {
                if (!sees.has(key)) continue;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  if (c * 32 + e >= d) continue;
                  const float v = (float)v_new[(n0 + key) * a.v_new_strides[1] + c * 32 + e];
                  if (!isfinite(v)) o[e] += v;
                }
              }
            }
          }
          if (real && seg.whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              if (c * 32 + e < d)
                *reinterpret_cast<uint4*>(out + c * 32 + e) = make_uint4(
                    Kind<T>::pack(o[e] * inv, o[e + 1] * inv),
                    Kind<T>::pack(o[e + 2] * inv, o[e + 3] * inv),
                    Kind<T>::pack(o[e + 4] * inv, o[e + 5] * inv),
                    Kind<T>::pack(o[e + 6] * inv, o[e + 7] * inv));
          } else if (real) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(results.out_of(result, tile_row, c * 8 + e / 4)) =
                  make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        const float m_log2 = m == -INFINITY ? m : m * scale_log2 - kLift<T>;
        if (real && seg.whole) {
          if (a.lse != nullptr)
            a.lse[((int64_t)seg.b * a.heads + head) * a.nodes + node] =
                (m_log2 + log2f(l)) * mma16::kLn2;
        } else if (real) {
          results.top_of(result, tile_row) = make_float2(m_log2, l);
        }
      }
      __syncwarp();
      tc_fence_before();  // O has been read before the next segment's first product
      base += seg.tiles;
      n += mine;
      ++mark;
    }
    __syncwarp();
    if (!ok) leave_nan<T, D, COPIES>(a, deal, wide);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// ---------------------------------------------------------------- host

// [columns][n1][n2][n3] 16-bit elements with strides s1, s2, s3 (elements) as boxes of 64 columns
// x box1 x box2. A dimension of one gets a stride of its own, whatever the tensor's says.
inline bool wide_map(CUtensorMap* map, const void* base, bool bf16, int64_t columns, int64_t n1,
                     int64_t s1, int box1, int64_t n2, int64_t s2, int box2, int64_t n3,
                     int64_t s3) {
  gemm::EncodeTiled encode = gemm::encode_tiled();
  if (encode == nullptr) return false;
  const int64_t n[3] = {n1, n2, n3}, s[3] = {s1, s2, s3};
  cuuint64_t dims[4] = {(cuuint64_t)columns, 0, 0, 0}, strides[3];
  for (int i = 0; i < 3; ++i) {
    if (n[i] <= 0 || n[i] > INT32_MAX) return false;
    const int64_t stride = n[i] == 1 ? (columns + 7) / 8 * 8 : s[i];
    if (stride <= 0 || stride * 2 >= (1ll << 40)) return false;
    dims[i + 1] = (cuuint64_t)n[i];
    strides[i] = (cuuint64_t)(stride * 2);
  }
  const cuuint32_t box[4] = {64, (cuuint32_t)box1, (cuuint32_t)box2, 1};
  const cuuint32_t elem[4] = {1, 1, 1, 1};
  return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                4, const_cast<void*>(base), dims, strides, box, elem,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int D, int COPIES>
inline cudaError_t launch_wide(const Args& a, const Deal& deal, const WideRows& w,
                               uint32_t wait_limit, cudaStream_t stream) {
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  const int64_t d = a.head_dim, kv = a.kv_heads;
  WideMaps maps;
  if (!wide_map(&maps.q, a.q, bf16, d, a.heads, a.q_strides[2], deal.group, a.nodes,
                a.q_strides[1], w.tile_nodes, a.batch, a.q_strides[0]) ||
      !wide_map(&maps.keys, a.keys, bf16, d, a.capacity, a.keys_strides[2], kKeysTile, kv,
                a.keys_strides[1], 1, a.batch, a.keys_strides[0]) ||
      !wide_map(&maps.values, a.values, bf16, d, a.capacity, a.values_strides[2], kKeysTile, kv,
                a.values_strides[1], 1, a.batch, a.values_strides[0]) ||
      !wide_map(&maps.k_new, a.k_new, bf16, d, a.nodes, a.k_new_strides[1], kKeysTile, kv,
                a.k_new_strides[2], 1, a.batch, a.k_new_strides[0]) ||
      !wide_map(&maps.v_new, a.v_new, bf16, d, a.nodes, a.v_new_strides[1], kKeysTile, kv,
                a.v_new_strides[2], 1, a.batch, a.v_new_strides[0]))
    return cudaErrorInvalidValue;
  static DeviceOnce once;
  constexpr int smem = (int)sizeof(WideShared<D>) + 1024;
  auto kernel = wide_kernel<T, D, COPIES>;
  int ready = 0;
  const cudaError_t e = once.get(
      [&](int* value) {
        cudaFuncAttributes attributes;
        cudaError_t r = cudaFuncGetAttributes(&attributes, kernel);
        if (r != cudaSuccess) return r;
        // the register split needs the launch's full count (setmaxnreg would wait for good)
        *value = attributes.numRegs == (int)kLaunchRegs ? 1 : 2;
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      },
      &ready);
  if (e != cudaSuccess) return e;
  if (ready != 1) return cudaErrorInvalidKernelImage;
  return launch_pdl(kernel, dim3((unsigned)deal.grid), dim3(kWideThreads), smem, stream, maps, a,
                    deal, w, wait_limit);
}

}  // namespace tree
}  // namespace ppyb200
