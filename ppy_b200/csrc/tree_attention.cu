// Attention of a few query rows over a long cache: the nodes of a drafted tree (a single token
// is a tree of one node, a prompt piece a chain) attend to every entry of their sequence's
// cache and to their own ancestors, and the nodes' keys and values are appended to the cache.
//
//   visible(i) = {j < length} and {length + a : a an ancestor of node i, or i}
//   s_ij = scale q_i . k_j,  lse_i = log sum_visible e^{s_ij},  out_i = sum e^{s_ij - lse_i} v_j
//
// The rows of one key head (nodes x the query heads that share it) form the M side of the
// products. Two kernels: the one here streams tiles of 64 keys through shared memory for 16 rows
// a CTA with warp-level products, and tree_attention_sm100.cuh holds the tensor-core
// kernel for many rows. Both keep a running maximum and sum (f32). The key tiles of all sequences
// are dealt to the CTAs in parts of equal size; a sequence of several parts is joined by a
// second kernel in the order of its parts, so results do not depend on timing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>
#include <type_traits>

#include "../../include/ppyb200.h"
#include "mma16.cuh"
#include "ppyb200_device.cuh"
#include "tree_attention.cuh"
#include "tree_attention_plan.cuh"
#include "tree_attention_sm100.cuh"

namespace {

using namespace ppyb200::mma16;
using ppyb200::tree::Args;
using ppyb200::tree::Deal;
using ppyb200::tree::Plan;
using ppyb200::tree::Results;
using ppyb200::tree::Segment;
using ppyb200::tree::Walk;
using ppyb200::tree::plan_for;
using ppyb200::tree::raise;
using ppyb200::tree::sequence_extent;
using ppyb200::tree::wide_fits;
using ppyb200::tree::wide_takes;

constexpr int kTile = ppyb200::tree::kNarrowTile;
constexpr int kRows = ppyb200::tree::kNarrowRows;
constexpr int kStages = 3;      // tiles in flight
constexpr int kWarps = 4;       // along a tile's keys
constexpr int kJoinRows = 8;    // rows of an item that a CTA joins
constexpr int kTreeWords = PPYB200_TREE_NODES / 32;

// Shared memory rows of D elements: 16-byte pieces XORed with the row's low bits, so that the
// eight rows an ldmatrix reads lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t row_piece(int row, int piece) {
  return (uint32_t)(row * D * 2 + ((piece ^ (row & 7)) << 4));
}

// Weights are held times 2^kLift until they are divided by their sum, which is lifted too: f16 ends
// at 2^-24, and where a long cache has many small weights, what they lose together would show
// (60000 weights of e^-18 beside one of 1 were zeros). 2^15 is f16's last power of two.
template <class T>
constexpr float kLift = std::is_same<T, __half>::value ? 15.f : 0.f;

// A row's result from its sums, by a warp: lane l holds columns 64 i + 2 l, +1.
template <class T, int D>
__device__ __forceinline__ void write_row(const Args& a, int b, int node, int head, int lane,
                                          float m, float l, const float (&sum)[D / 32]) {
  const float inv = 1.f / l;
  T* out = static_cast<T*>(a.out) + b * a.out_strides[0] + node * a.out_strides[1] +
           (int64_t)head * a.out_strides[2];
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const int col = i * 64 + lane * 2;
    if (col < a.head_dim)
      *reinterpret_cast<uint32_t*>(out + col) =
          Kind<T>::pack(sum[2 * i] * inv, sum[2 * i + 1] * inv);
  }
  if (lane == 0 && a.lse != nullptr)
    a.lse[((int64_t)b * a.heads + head) * a.nodes + node] = (m + log2f(l)) * kLn2;
}

// Sixteen rows a CTA; the four warps take sixteen keys each of every tile and are joined at the
// end: splitting the keys and not the head dimension leaves each warp whole scores, so the warps
// meet once an item. Each key and value is read once for up to 16 rows, and the few products cost
// less than the loads: what bounds it is memory where the caches are large (64 sequences of up to
// 1000 entries, 12 heads of 64: 170 MB in 55 us with the join, 3.1 TB/s; 525 MB at 4.6 TB/s), and
// the chain of its steps where they are small (one sequence of 1000 entries: 10 us with the
// join, of which the loads themselves would take half a microsecond).
template <class T, int D>
__global__ void __launch_bounds__(32 * kWarps, D == 64 ? 4 : 2)
narrow_kernel(const __grid_constant__ Args a, const Deal deal) {
  constexpr int kThreads = 32 * kWarps, kPieces = D / 8;
  constexpr int kKeys = kTile / kWarps;  // keys of a tile that one warp takes
  constexpr int kTileBytes = kTile * D * 2;
  extern __shared__ __align__(128) uint8_t smem[];  // kStages x (K tile, V tile)
  __shared__ uint32_t below[kRows][kTreeWords];     // ancestors of each row's node, by bit
  __shared__ unsigned long long spoiled;            // tail keys with a value that is not finite

  ppyb200::pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gid = lane >> 2, tig = lane & 3;
  const int group = deal.group, d = (int)a.head_dim;
  Walk<kTile, false> walk;
  walk.measure(a, deal, blockIdx.x == 0);
  walk.enter(a, deal, blockIdx.x);
  Segment seg;
  while (walk.next(a, deal, seg)) {
    const int b = seg.b, kvh = seg.kvh;
    const int64_t length = seg.length, total = length + seg.count;
    const int row0 = seg.row0, rows = seg.count * group;
    const int64_t t0 = seg.first, t1 = t0 + seg.tiles;
    __syncthreads();  // the last segment's shared memory has been read

    const T* q = static_cast<const T*>(a.q) + b * a.q_strides[0];
    const T* k_new = static_cast<const T*>(a.k_new) + b * a.k_new_strides[0] +
                     kvh * a.k_new_strides[2];
    const T* v_new = static_cast<const T*>(a.v_new) + b * a.v_new_strides[0] +
                     kvh * a.v_new_strides[2];
    const T* keys = static_cast<T*>(a.keys) + b * a.keys_strides[0] + kvh * a.keys_strides[1];
    const T* values =
        static_cast<T*>(a.values) + b * a.values_strides[0] + kvh * a.values_strides[1];

    const uint32_t base = shared_address(smem);
    auto load_tile = [&](int64_t tile, int stage) {
      const uint32_t ks = base + stage * 2 * kTileBytes, vs = ks + kTileBytes;
      for (int i = tid; i < kTile * kPieces; i += kThreads) {
        const int row = i / kPieces, piece = i % kPieces;
        const int64_t j = tile * kTile + row;
        const bool valid = j < total && piece * 8 < d;
        const T *ksrc = keys, *vsrc = values;
        if (valid) {
          if (j < length) {
            ksrc = keys + j * a.keys_strides[2] + piece * 8;
            vsrc = values + j * a.values_strides[2] + piece * 8;
          } else {
            ksrc = k_new + (j - length) * a.k_new_strides[1] + piece * 8;
            vsrc = v_new + (j - length) * a.v_new_strides[1] + piece * 8;
          }
        }
        const uint32_t at = row_piece<D>(row, piece);
        copy16(ks + at, ksrc, valid);
        copy16(vs + at, vsrc, valid);
      }
    };

#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
      if (t0 + s < t1) load_tile(t0 + s, s);
      copies_commit();
    }

    ppyb200::tree::append<T>(a, deal, seg, tid, kThreads);

    if (deal.join && seg.starts && tid == 0)
      Results(a, deal, D).ctas[seg.number] = make_int2(blockIdx.x, seg.last_cta);

    // query fragments: the 16 rows, zero beyond the rows and the head size
    const int ra = row0 + gid, rb = ra + 8;
    uint32_t qf[D / 16][4];
    {
      const T* qa = ra < rows ? q + (ra / group) * a.q_strides[1] +
                                    (int64_t)(kvh * group + ra % group) * a.q_strides[2] : nullptr;
      const T* qb = rb < rows ? q + (rb / group) * a.q_strides[1] +
                                    (int64_t)(kvh * group + rb % group) * a.q_strides[2] : nullptr;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        const int c = s * 16 + tig * 2;
        qf[s][0] = qa != nullptr && c < d ? *reinterpret_cast<const uint32_t*>(qa + c) : 0u;
        qf[s][1] = qb != nullptr && c < d ? *reinterpret_cast<const uint32_t*>(qb + c) : 0u;
        qf[s][2] = qa != nullptr && c + 8 < d ? *reinterpret_cast<const uint32_t*>(qa + c + 8) : 0u;
        qf[s][3] = qb != nullptr && c + 8 < d ? *reinterpret_cast<const uint32_t*>(qb + c + 8) : 0u;
      }
    }

    // ancestors of this tile's rows, where the CTA reads node slots of a tree
    const bool tree = a.parents != nullptr;
    if (tree && t1 * kTile > length) {
      const int32_t* parents = a.parents + b * a.parents_stride;
      for (int r = tid; r < kRows; r += kThreads) {
#pragma unroll
        for (int w = 0; w < kTreeWords; ++w) below[r][w] = 0;
        if (row0 + r < rows) {
          int i = (row0 + r) / group;
          below[r][i >> 5] |= 1u << (i & 31);
          for (;;) {
            const int p = parents[i];
            if (p < 0 || p >= i) {  // a root; an index that is no earlier node raises
              if (p != -1) raise(a.status);
              break;
            }
            i = p;
            below[r][i >> 5] |= 1u << (i & 31);
          }
        }
      }
    }
    if (tid == 0) spoiled = 0;

    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[n][c] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    const float scale = (float)a.scale * kLog2e;  // scores in powers of two
    // the last node that rows gid and gid + 8 may see
    const int last0 = ra >= rows ? -1 : tree ? seg.count - 1 : ra / group;
    const int last1 = rb >= rows ? -1 : tree ? seg.count - 1 : rb / group;

    for (int64_t t = t0; t < t1; ++t) {
      const int stage = (int)((t - t0) % kStages);
      copies_wait<kStages - 2>();
      __syncthreads();
      if (t + kStages - 1 < t1) load_tile(t + kStages - 1, (int)((t - t0 + kStages - 1) % kStages));
      copies_commit();
      const uint32_t ks = base + stage * 2 * kTileBytes, vs = ks + kTileBytes;

      // S = Q K^T: this warp's rows against its keys of the tile
      float s[kKeys / 8][4];
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n) {
        s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
        const int row = warp * kKeys + n * 8 + (lane & 7);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {  // 32 columns: four 8 x 8 tiles
          uint32_t kf[4];
          load4(kf, ks + row_piece<D>(row, c * 4 + (lane >> 3)));
          Kind<T>::mma(s[n], qf[2 * c], kf[0], kf[1]);
          Kind<T>::mma(s[n], qf[2 * c + 1], kf[2], kf[3]);
        }
      }
      const bool tail = (t + 1) * kTile > length;
      const int rel = (int)(t * kTile - length);  // the node of the tile's first slot, or negative
      if (tail) {
        // values that are not finite must not meet the zero weights of rows that do not see
        // them: zero them here, and add them below to the rows that do
        const int from = max(0, -rel) * kPieces, to = min(kTile, seg.count - rel) * kPieces;
#pragma unroll 1
        for (int i = from + tid; i < to; i += kThreads) {
          const int row = i / kPieces;
          uint4* at = reinterpret_cast<uint4*>(smem + (vs - base) + row_piece<D>(row, i % kPieces));
          const uint4 v = *at;
          const uint4 clean = make_uint4(finite_only<T>(v.x), finite_only<T>(v.y),
                                         finite_only<T>(v.z), finite_only<T>(v.w));
          if (clean.x != v.x || clean.y != v.y || clean.z != v.z || clean.w != v.w) {
            *at = clean;
            atomicOr(&spoiled, 1ull << row);
          }
        }
        __syncthreads();
      }
      // whether row gid (half 0) or gid + 8 (half 1) sees node n; a chain's rows see those up to
      // their own, and every row the cache's entries (n < 0)
      auto sees = [&](int half, int n) {
        const int last = half == 0 ? last0 : last1;
        if (!tree || n < 0) return n <= last;
        return n <= last && ((below[gid + 8 * half][n >> 5] >> (n & 31)) & 1u) != 0;
      };
      float x0 = m0, x1 = m1;
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          s[n][c] *= scale;
          if (tail) {
            if (!sees(c >> 1, rel + warp * kKeys + n * 8 + tig * 2 + (c & 1)))
              s[n][c] = -INFINITY;
          }
          if (c < 2) x0 = fmaxf(x0, s[n][c]);
          else x1 = fmaxf(x1, s[n][c]);
        }
#pragma unroll
      for (int w = 1; w < 4; w <<= 1) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, w));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, w));
      }
      // a row that has seen nothing yet keeps its maximum at -inf; its terms are 2^-inf = 0
      const float u0 = x0 == -INFINITY ? 0.f : x0, u1 = x1 == -INFINITY ? 0.f : x1;
      const float f0 = exp2_sfu(m0 - u0), f1 = exp2_sfu(m1 - u1);
      const float v0 = u0 - kLift<T>, v1 = u1 - kLift<T>;
      m0 = x0;
      m1 = x1;
      l0 *= f0;
      l1 *= f1;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        o[n][0] *= f0;
        o[n][1] *= f0;
        o[n][2] *= f1;
        o[n][3] *= f1;
      }
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n) {
        s[n][0] = exp2_sfu(s[n][0] - v0);
        s[n][1] = exp2_sfu(s[n][1] - v0);
        s[n][2] = exp2_sfu(s[n][2] - v1);
        s[n][3] = exp2_sfu(s[n][3] - v1);
        l0 += s[n][0] + s[n][1];
        l1 += s[n][2] + s[n][3];
      }
      // O += P V, P rounded to the values' type (half a step, 2^-9 or 2^-12 of each weight, as
      // the prompt attention rounds it); the sum above takes the unrounded weights
#pragma unroll
      for (int kk = 0; kk < kKeys / 16; ++kk) {
        const uint32_t pf[4] = {
            Kind<T>::pack(s[2 * kk][0], s[2 * kk][1]), Kind<T>::pack(s[2 * kk][2], s[2 * kk][3]),
            Kind<T>::pack(s[2 * kk + 1][0], s[2 * kk + 1][1]),
            Kind<T>::pack(s[2 * kk + 1][2], s[2 * kk + 1][3])};
        const int row = warp * kKeys + kk * 16 + (lane & 15);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {  // 16 columns: keys 0-7 and 8-15 of two 8-wide tiles
          uint32_t vf[4];
          load4_transposed(vf, vs + row_piece<D>(row, c * 2 + (lane >> 4)));
          Kind<T>::mma(o[2 * c], pf, vf[0], vf[1]);
          Kind<T>::mma(o[2 * c + 1], pf, vf[2], vf[3]);
        }
      }
      if (tail && spoiled != 0) {
#pragma unroll 1
        for (int key = warp * kKeys; key < (warp + 1) * kKeys; ++key) {
          if (((spoiled >> key) & 1ull) == 0) continue;
          const T* v = v_new + (int64_t)(rel + key) * a.v_new_strides[1];
          const bool see0 = sees(0, rel + key), see1 = sees(1, rel + key);
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int col = n * 8 + tig * 2 + c;
              if (col >= d) continue;
              const float value = (float)v[col];
              if (isfinite(value)) continue;
              if (see0) o[n][c] += value;
              if (see1) o[n][2 + c] += value;
            }
        }
      }
      if (tail) {
        __syncthreads();
        if (tid == 0) spoiled = 0;
      }
    }
    copies_wait<0>();
    m0 -= kLift<T>;  // from here on the reference that the sums go by
    m1 -= kLift<T>;
#pragma unroll
    for (int w = 1; w < 4; w <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, w);
      l1 += __shfl_xor_sync(0xffffffffu, l1, w);
    }

    // join the warps in shared memory: [kWarps][kRows][D + 2]
    float* box = reinterpret_cast<float*>(smem);
    constexpr int kLine = D + 2;
    __syncthreads();
    float* mine = box + (warp * kRows + gid) * kLine;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      const int col = n * 8 + tig * 2;
      *reinterpret_cast<float2*>(mine + col) = make_float2(o[n][0], o[n][1]);
      *reinterpret_cast<float2*>(mine + 8 * kLine + col) = make_float2(o[n][2], o[n][3]);
    }
    if (tig == 0) {
      *reinterpret_cast<float2*>(mine + D) = make_float2(m0, l0);
      *reinterpret_cast<float2*>(mine + 8 * kLine + D) = make_float2(m1, l1);
    }
    __syncthreads();
    // a warp a row at a time, a lane two columns of every 64
    const Results results(a, deal, D);
    for (int r = warp; r < kRows && row0 + r < rows; r += kWarps) {
      float m = -INFINITY, l = 0.f, sum[D / 32];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, box[(w * kRows + r) * kLine + D]);
      const float u = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) sum[i] = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* from = box + (w * kRows + r) * kLine;
        const float f = exp2_sfu(from[D] - u);
        l += f * from[D + 1];
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const float2 v = *reinterpret_cast<const float2*>(from + i * 64 + lane * 2);
          sum[2 * i] += f * v.x;
          sum[2 * i + 1] += f * v.y;
        }
      }
      const int node = (row0 + r) / group, head = kvh * group + (row0 + r) % group;
      if (seg.whole) {
        write_row<T, D>(a, b, node, head, lane, m, l, sum);
      } else {
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
          *reinterpret_cast<float2*>(results.out_of(seg.result, r, i * 16 + lane / 2) +
                                     lane % 2 * 2) = make_float2(sum[2 * i], sum[2 * i + 1]);
        if (lane == 0) results.top_of(seg.result, r) = make_float2(m, l);
      }
    }
  }
}

// One column of a row whose values are not all finite, from those alone: the infinity that they add
// up to, or NaN. For sums that came out as NaN because a result held an infinity times zero: a copy
// of the rows weighs the keys of the others with zero.
template <class T>
__device__ __noinline__ float odd_value(const Args& a, int b, int kvh, int length, int node,
                                        int col) {
  const T* values = static_cast<const T*>(a.values) + b * a.values_strides[0] +
                    kvh * a.values_strides[1] + col;
  const T* v_new = static_cast<const T*>(a.v_new) + b * a.v_new_strides[0] +
                   kvh * a.v_new_strides[2] + col;
  float sum = 0.f;
#pragma unroll 8
  for (int64_t j = 0; j < length; ++j) {
    const float v = (float)values[j * a.values_strides[2]];
    if (!isfinite(v)) sum += v;
  }
#pragma unroll 1
  for (int i = node; i >= 0;) {  // the node and its ancestors
    const float v = (float)v_new[i * a.v_new_strides[1]];
    if (!isfinite(v)) sum += v;
    const int p = a.parents == nullptr ? i - 1 : a.parents[b * a.parents_stride + i];
    i = p < i ? p : -1;
  }
  return isfinite(sum) ? __uint_as_float(0x7fc00000u) : sum;
}

// Joins the unnormalised results of an item's segments in their order, a thread four columns of a
// row. What it costs is the latency of its loads one after another, so the outputs of the first
// eight results are under way before the maxima are known.
template <class T, int D>
__global__ void __launch_bounds__(kJoinRows * D / 4) join_kernel(const __grid_constant__ Args a,
                                                                 const Deal deal) {
  ppyb200::pdl_wait();
  const int number = blockIdx.x, piece = threadIdx.x / kJoinRows;
  const int r = blockIdx.y * kJoinRows + threadIdx.x % kJoinRows;
  const int items = (int)a.batch * deal.items, kvh = number / items, item = number - kvh * items;
  const int b = item / deal.items, row = (item - b * deal.items) * deal.item_rows + r;
  const int node = row / deal.group;
  const Results results(a, deal, D);
  const int2 ctas = results.ctas[number];  // meaningless where the item has no rows
  int length, count;
  sequence_extent(a, b, length, count, nullptr);
  if (r >= deal.item_rows || node >= count) return;
  if (deal.streams == 1 && ctas.x == ctas.y) return;  // whole: written by its CTA
  const int parts = (ctas.y - ctas.x + 1) * deal.streams;
  int cta = ctas.x, stream = 0;  // of the next result
  constexpr int kBatch = 8;
  float m = -INFINITY, l = 0.f, sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < parts; i0 += kBatch) {
    float4 v[kBatch];
    float2 top[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      top[i] = make_float2(-INFINITY, 0.f);
      if (i0 + i < parts) {
        // the first segment starts the item, the others continue it
        const int64_t at =
            Walk<kTile, false>::result_of(deal, cta, number, cta == ctas.x) + stream;
        if (++stream == deal.streams) {
          stream = 0;
          ++cta;
        }
        v[i] = *reinterpret_cast<const float4*>(results.out_of(at, r, piece));
        top[i] = results.top_of(at, r);
      }
    }
    float most = m;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) most = fmaxf(most, top[i].x);
    const float u = most == -INFINITY ? 0.f : most, f = exp2_sfu(m - u);
    m = most;
    l *= f;
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] *= f;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float g = exp2_sfu(top[i].x - u);
      l += g * top[i].y;
      sum[0] += g * v[i].x;
      sum[1] += g * v[i].y;
      sum[2] += g * v[i].z;
      sum[3] += g * v[i].w;
    }
  }
  const int head = kvh * deal.group + row % deal.group;
  const float inv = 1.f / l;
  if (piece * 4 < a.head_dim) {
    const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    if (all != all && l == l) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (sum[k] != sum[k]) sum[k] = odd_value<T>(a, b, kvh, length, node, piece * 4 + k);
    }
    T* out = static_cast<T*>(a.out) + b * a.out_strides[0] + node * a.out_strides[1] +
             (int64_t)head * a.out_strides[2] + piece * 4;
    *reinterpret_cast<uint2*>(out) = make_uint2(Kind<T>::pack(sum[0] * inv, sum[1] * inv),
                                                Kind<T>::pack(sum[2] * inv, sum[3] * inv));
  }
  if (piece == 0 && a.lse != nullptr)
    a.lse[((int64_t)b * a.heads + head) * a.nodes + node] = (m + log2f(l)) * kLn2;
}

// ---------------------------------------------------------------- host

template <class T, int D>
cudaError_t join(const Args& a, const Plan& p, cudaStream_t stream) {
  const dim3 grid((unsigned)(a.kv_heads * a.batch * p.deal.items),
                  (unsigned)((p.deal.item_rows + kJoinRows - 1) / kJoinRows));
  return ppyb200::launch_pdl(join_kernel<T, D>, grid, dim3(kJoinRows * D / 4), 0, stream, a, p.deal);
}

template <class T, int D>
cudaError_t launch_narrow(const Args& a, const Plan& p, cudaStream_t stream) {
  static ppyb200::DeviceOnce once;
  constexpr int smem = kStages * 2 * kTile * D * 2;
  int ready = 0;
  auto kernel = narrow_kernel<T, D>;
  const cudaError_t e = once.get([&](int* value) {
    *value = 1;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  }, &ready);
  if (e != cudaSuccess) return e;
  return ppyb200::launch_pdl(kernel, dim3((unsigned)p.deal.grid), dim3(32 * kWarps), smem, stream,
                             a, p.deal);
}

std::atomic<uint32_t> wait_limit{ppyb200::tree::kWaitLimit};

template <class T, int D>
cudaError_t launch_dim(const Args& a, const Plan& p, cudaStream_t stream) {
  using ppyb200::tree::launch_wide;
  const uint32_t limit = wait_limit.load(std::memory_order_relaxed);
  const cudaError_t e =
      !p.wide ? launch_narrow<T, D>(a, p, stream)
      : p.rows.copies == 4 ? launch_wide<T, D, 4>(a, p.deal, p.rows, limit, stream)
      : p.rows.copies == 2 ? launch_wide<T, D, 2>(a, p.deal, p.rows, limit, stream)
                           : launch_wide<T, D, 1>(a, p.deal, p.rows, limit, stream);
  return e == cudaSuccess && p.deal.join ? join<T, D>(a, p, stream) : e;
}

template <class T>
cudaError_t launch_type(const Args& a, const Plan& p, cudaStream_t stream) {
  return a.head_dim <= 64 ? launch_dim<T, 64>(a, p, stream) : launch_dim<T, 128>(a, p, stream);
}

bool rows16(const void* p, const int64_t (&strides)[3]) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && strides[0] % 8 == 0 &&
         strides[1] % 8 == 0 && strides[2] % 8 == 0;
}

// nullptr when the arguments are in order, else what is wrong with them
const char* refusal(const ppyb200_tree_attention_args& a) {
  if (a.dtype != PPYB200_BF16 && a.dtype != PPYB200_F16) return "dtype is bf16 or f16";
  if (a.batch < 0 || a.nodes < 0 || a.capacity < 0 || a.heads <= 0 || a.kv_heads <= 0 ||
      a.heads % a.kv_heads != 0)
    return "heads is a multiple of kv_heads, and no size is negative";
  if (a.head_dim <= 0 || a.head_dim > 128 || a.head_dim % 8 != 0)
    return "head_dim is a multiple of 8 up to 128";
  if (a.parents != nullptr && a.nodes > PPYB200_TREE_NODES)
    return "a tree has at most PPYB200_TREE_NODES nodes (a chain may be longer)";
  if (a.batch > 65535 || a.capacity > INT32_MAX || a.nodes * (a.heads / a.kv_heads) > INT32_MAX ||
      a.batch * ((a.nodes * (a.heads / a.kv_heads) + 15) / 16) > INT32_MAX / 2 ||
      a.batch * a.heads * a.nodes > INT32_MAX)
    return "batch up to 65535, rows (batch x heads x nodes) and capacity below 2^31";
  if (!rows16(a.q, a.q_strides) || !rows16(a.k_new, a.k_new_strides) ||
      !rows16(a.v_new, a.v_new_strides) || !rows16(a.keys, a.keys_strides) ||
      !rows16(a.values, a.values_strides) || !rows16(a.out, a.out_strides))
    return "every row of q, k, v, the cache and out starts on a 16-byte boundary";
  return nullptr;
}

}  // namespace

extern "C" {

void ppyb200_tree_attention_wait_limit(int64_t tries) {
  wait_limit.store(tries < 0 || tries > ppyb200::tree::kWaitLimit ? ppyb200::tree::kWaitLimit
                                                                  : (uint32_t)tries,
                   std::memory_order_relaxed);
}

int64_t ppyb200_tree_attention_workspace(const ppyb200_tree_attention_args* args) {
  if (args == nullptr || refusal(*args) != nullptr || args->batch == 0 || args->nodes == 0)
    return 0;
  // enough for either kernel: strides and scale, which choose one, are not among the sizes
  const int sm_count = ppyb200_sm_count();
  const int64_t narrow = plan_for(*args, false, sm_count).workspace;
  const int64_t wide = wide_fits(*args) ? plan_for(*args, true, sm_count).workspace : 0;
  return narrow > wide ? narrow : wide;
}

int32_t ppyb200_tree_attention(const ppyb200_tree_attention_args* args) {
  if (args == nullptr) {
    ppyb200_set_error("ppyb200_tree_attention: no arguments");
    return PPYB200_RAISED;
  }
  const ppyb200_tree_attention_args& a = *args;
  const char* wrong = refusal(a);
  if (wrong != nullptr) {
    char text[256];
    snprintf(text, sizeof text, "ppyb200_tree_attention: %s", wrong);
    ppyb200_set_error(text);
    return PPYB200_RAISED;
  }
  if (a.batch == 0 || a.nodes == 0) return PPYB200_OK;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(ppyb200_stream());
  const Plan p = plan_for(a, wide_takes(a), ppyb200_sm_count());
  if (p.workspace > 0 && (a.workspace == nullptr || a.workspace_bytes < p.workspace ||
                          (reinterpret_cast<uintptr_t>(a.workspace) & 15u) != 0)) {
    ppyb200_set_error("ppyb200_tree_attention: a 16-byte aligned workspace of "
                      "ppyb200_tree_attention_workspace bytes required");
    return PPYB200_RAISED;
  }
  const cudaError_t e = a.dtype == PPYB200_BF16 ? launch_type<__nv_bfloat16>(a, p, stream)
                                                : launch_type<__half>(a, p, stream);
  if (e != cudaSuccess) return ppyb200_check((int32_t)e, "ppyb200_tree_attention");
  ppyb200_count_launches(p.deal.join ? 2 : 1);
  return PPYB200_OK;
}

}  // extern "C"
