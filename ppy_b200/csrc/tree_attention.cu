// Attention of a few query rows over a long cache: the nodes of a drafted tree (a single token
// is a tree of one node, a prompt piece a chain) attend to every entry of their sequence's
// cache and to their own ancestors, and the nodes' keys and values are appended to the cache.
//
//   visible(i) = {j < length} and {length + a : a an ancestor of node i, or i}
//   s_ij = scale q_i . k_j,  lse_i = log sum_visible e^{s_ij},  out_i = sum e^{s_ij - lse_i} v_j
//
// The rows of one key head (nodes x the query heads that share it) form the M side of the
// products; tiles of 64 keys stream through shared memory once per 16, 32, 64 or 128 rows with
// a running maximum and sum (f32). A long axis of keys is split over CTAs: each leaves its
// unnormalised f32 output with its maximum and sum in the workspace, and a second kernel joins
// them in split order, so results do not depend on timing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/ppyb200.h"
#include "mma16.cuh"
#include "ppyb200_device.cuh"

namespace {

using namespace ppyb200::mma16;

constexpr int kTile = 64;       // keys a tile
constexpr int kStages = 3;      // tiles in flight
constexpr int kTreeWords = PPYB200_TREE_NODES / 32;

struct Shape {
  int splits;     // CTAs along the keys
  int row_tiles;  // CTAs along the rows of one key head
  int group;      // query heads a key head
};

__device__ __forceinline__ void raise(int32_t* status) {
  if (status != nullptr) atomicMax(status, PPYB200_DEVICE_RAISED);
}

// The cache length and node count of a sequence, held inside the buffers whatever the device
// arrays say: nodes that do not fit behind the length are dropped, and the status raised.
__device__ __forceinline__ void sequence_extent(const ppyb200_tree_attention_args& a, int b,
                                                int64_t& length, int& count, int32_t* status) {
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

// Shared memory rows of D elements: 16-byte pieces XORed with the row's low bits, so that the
// eight rows an ldmatrix reads lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t row_piece(int row, int piece) {
  return (uint32_t)(row * D * 2 + ((piece ^ (row & 7)) << 4));
}

// WM warps along the rows (16 each), WK warps along a tile's keys.
template <class T, int D, int WM, int WK>
__global__ void __launch_bounds__(32 * WM * WK)
tree_attention_kernel(const ppyb200_tree_attention_args a, const Shape shape, float* partial) {
  constexpr int kThreads = 32 * WM * WK, kRows = 16 * WM, kPieces = D / 8;
  constexpr int kKeys = kTile / WK;      // keys of a tile that one warp takes
  constexpr int kTileBytes = kTile * D * 2;
  extern __shared__ __align__(128) uint8_t smem[];  // kStages x (K tile, V tile)
  __shared__ uint32_t below[kRows][kTreeWords];     // ancestors of each row's node, by bit
  __shared__ unsigned long long spoiled;            // tail keys with a value that is not finite

  ppyb200::pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wm = warp / WK, wk = warp % WK;
  const int gid = lane >> 2, tig = lane & 3;
  const int b = blockIdx.z;
  const int kvh = blockIdx.y / shape.row_tiles, rt = blockIdx.y % shape.row_tiles;
  const int group = shape.group, d = (int)a.head_dim;
  int64_t length;
  int count;
  sequence_extent(a, b, length, count, blockIdx.x == 0 && blockIdx.y == 0 && tid == 0
                                           ? a.status : nullptr);
  const int rows = count * group, row0 = rt * kRows;
  if (row0 >= rows) return;
  const int64_t total = length + count;
  const int64_t tiles = (total + kTile - 1) / kTile;
  const int64_t per = (tiles + shape.splits - 1) / shape.splits;
  const int64_t t0 = blockIdx.x * per, t1 = min(tiles, t0 + per);

  const T* q = static_cast<const T*>(a.q) + b * a.q_strides[0];
  const T* k_new = static_cast<const T*>(a.k_new) + b * a.k_new_strides[0] +
                   kvh * a.k_new_strides[2];
  const T* v_new = static_cast<const T*>(a.v_new) + b * a.v_new_strides[0] +
                   kvh * a.v_new_strides[2];
  T* keys = static_cast<T*>(a.keys) + b * a.keys_strides[0] + kvh * a.keys_strides[1];
  T* values = static_cast<T*>(a.values) + b * a.values_strides[0] + kvh * a.values_strides[1];

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

  // append: the CTAs of the first row tile write the nodes whose slots they read
  if (rt == 0 && t1 * kTile > length) {
    const int64_t first = max(t0 * kTile, length), last = min(t1 * kTile, total);
    const int pieces = d / 8;
    for (int64_t i = tid; i < (last - first) * pieces; i += kThreads) {
      const int64_t j = first + i / pieces, n = j - length;
      const int piece = (int)(i % pieces);
      *reinterpret_cast<uint4*>(keys + j * a.keys_strides[2] + piece * 8) =
          *reinterpret_cast<const uint4*>(k_new + n * a.k_new_strides[1] + piece * 8);
      *reinterpret_cast<uint4*>(values + j * a.values_strides[2] + piece * 8) =
          *reinterpret_cast<const uint4*>(v_new + n * a.v_new_strides[1] + piece * 8);
    }
  }

  // query fragments: this warp's 16 rows, zero beyond the rows and the head size
  const int ra = row0 + wm * 16 + gid, rb = ra + 8;
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
      const int row = wk * kKeys + n * 8 + (lane & 7);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {  // 32 columns: four 8 x 8 tiles
        uint32_t kf[4];
        load4(kf, ks + row_piece<D>(row, c * 4 + (lane >> 3)));
        Kind<T>::mma(s[n], qf[2 * c], kf[0], kf[1]);
        Kind<T>::mma(s[n], qf[2 * c + 1], kf[2], kf[3]);
      }
    }
    const bool tail = (t + 1) * kTile > length;
    if (tail) {
      // values that are not finite must not meet the zero weights of rows that do not see
      // them: zero them here, and add them below to the rows that do
      for (int i = tid; i < kTile * D / 2; i += kThreads) {
        const int row = i / (D / 2), word = i % (D / 2);
        if (t * kTile + row < length) continue;
        uint32_t* at = reinterpret_cast<uint32_t*>(smem + (vs - base) +
                                                   row_piece<D>(row, word / 4) + (word % 4) * 4);
        const float2 v = Kind<T>::unpack(*at);
        if (!isfinite(v.x) || !isfinite(v.y)) {
          *at = Kind<T>::pack(isfinite(v.x) ? v.x : 0.f, isfinite(v.y) ? v.y : 0.f);
          atomicOr(&spoiled, 1ull << row);
        }
      }
      __syncthreads();
    }
    auto sees = [&](int r, int64_t j) {  // row r (in the tile of rows) and slot j
      if (j < length) return true;
      if (j >= total || row0 + r >= rows) return false;
      const int n = (int)(j - length);
      return tree ? ((below[r][n >> 5] >> (n & 31)) & 1u) != 0 : n <= (row0 + r) / group;
    };
    float x0 = m0, x1 = m1;
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[n][c] *= scale;
        if (tail) {
          const int64_t j = t * kTile + wk * kKeys + n * 8 + tig * 2 + (c & 1);
          if (!sees(wm * 16 + gid + (c >> 1) * 8, j)) s[n][c] = -INFINITY;
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
      s[n][0] = exp2_sfu(s[n][0] - u0);
      s[n][1] = exp2_sfu(s[n][1] - u0);
      s[n][2] = exp2_sfu(s[n][2] - u1);
      s[n][3] = exp2_sfu(s[n][3] - u1);
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
      const int row = wk * kKeys + kk * 16 + (lane & 15);
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {  // 16 columns: keys 0-7 and 8-15 of two 8-wide tiles
        uint32_t vf[4];
        load4_transposed(vf, vs + row_piece<D>(row, c * 2 + (lane >> 4)));
        Kind<T>::mma(o[2 * c], pf, vf[0], vf[1]);
        Kind<T>::mma(o[2 * c + 1], pf, vf[2], vf[3]);
      }
    }
    if (tail && spoiled != 0) {
      for (int key = wk * kKeys; key < (wk + 1) * kKeys; ++key) {
        if (((spoiled >> key) & 1ull) == 0) continue;
        const int64_t j = t * kTile + key;
        const T* v = v_new + (j - length) * a.v_new_strides[1];
        const bool see0 = sees(wm * 16 + gid, j), see1 = sees(wm * 16 + gid + 8, j);
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
#pragma unroll
  for (int w = 1; w < 4; w <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, w);
    l1 += __shfl_xor_sync(0xffffffffu, l1, w);
  }

  // join the warps along the keys in shared memory
  if (WK > 1) {
    float* box = reinterpret_cast<float*>(smem);  // [WK][kRows][D + 2]
    constexpr int kLine = D + 2;
    __syncthreads();
    float* mine = box + (wk * kRows + wm * 16 + gid) * kLine;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      const int col = n * 8 + tig * 2;
      mine[col] = o[n][0];
      mine[col + 1] = o[n][1];
      mine[8 * kLine + col] = o[n][2];
      mine[8 * kLine + col + 1] = o[n][3];
    }
    if (tig == 0) {
      mine[D] = m0;
      mine[D + 1] = l0;
      mine[8 * kLine + D] = m1;
      mine[8 * kLine + D + 1] = l1;
    }
    __syncthreads();
    if (wk != 0) return;
    float y0 = -INFINITY, y1 = -INFINITY;
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float* from = box + (w * kRows + wm * 16 + gid) * kLine;
      y0 = fmaxf(y0, from[D]);
      y1 = fmaxf(y1, from[8 * kLine + D]);
    }
    const float z0 = y0 == -INFINITY ? 0.f : y0, z1 = y1 == -INFINITY ? 0.f : y1;
    l0 = l1 = 0.f;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float* from = box + (w * kRows + wm * 16 + gid) * kLine;
      const float f0 = exp2_sfu(from[D] - z0), f1 = exp2_sfu(from[8 * kLine + D] - z1);
      l0 += f0 * from[D + 1];
      l1 += f1 * from[8 * kLine + D + 1];
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        const int col = n * 8 + tig * 2;
        o[n][0] += f0 * from[col];
        o[n][1] += f0 * from[col + 1];
        o[n][2] += f1 * from[8 * kLine + col];
        o[n][3] += f1 * from[8 * kLine + col + 1];
      }
    }
    m0 = y0;
    m1 = y1;
  }

#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = half == 0 ? ra : rb;
    if (r >= rows) continue;
    const float m = half == 0 ? m0 : m1, l = half == 0 ? l0 : l1;
    const int node = r / group, head = kvh * group + r % group;
    if (shape.splits == 1) {
      T* out = static_cast<T*>(a.out) + b * a.out_strides[0] + node * a.out_strides[1] +
               (int64_t)head * a.out_strides[2];
      const float inv = 1.f / l;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        const int col = n * 8 + tig * 2;
        if (col < d)
          *reinterpret_cast<uint32_t*>(out + col) =
              Kind<T>::pack(o[n][2 * half] * inv, o[n][2 * half + 1] * inv);
      }
      if (tig == 0 && a.lse != nullptr)
        a.lse[((int64_t)b * a.heads + head) * a.nodes + node] = (m + log2f(l)) * kLn2;
    } else {
      // partial [batch][heads][nodes][splits][D + 2]
      float* to = partial + ((((int64_t)b * a.heads + head) * a.nodes + node) * shape.splits +
                             blockIdx.x) * (D + 2);
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
        *reinterpret_cast<float2*>(to + n * 8 + tig * 2) =
            make_float2(o[n][2 * half], o[n][2 * half + 1]);
      if (tig == 0) *reinterpret_cast<float2*>(to + D) = make_float2(m, l);
    }
  }
}

// One warp a row: joins the splits' unnormalised outputs in split order.
template <class T, int D>
__global__ void __launch_bounds__(128) join_kernel(const ppyb200_tree_attention_args a,
                                                   const int splits, const float* partial) {
  ppyb200::pdl_wait();
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= a.batch * a.heads * a.nodes) return;
  const int node = (int)(row % a.nodes);
  const int head = (int)(row / a.nodes % a.heads), b = (int)(row / a.nodes / a.heads);
  int64_t length;
  int count;
  sequence_extent(a, b, length, count, nullptr);
  if (node >= count) return;
  const float* from = partial + row * splits * (D + 2);
  float m = -INFINITY;
  for (int s = lane; s < splits; s += 32) m = fmaxf(m, from[s * (D + 2) + D]);
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
  const float u = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float* p = from + s * (D + 2);
    const float f = exp2_sfu(p[D] - u);
    l += f * p[D + 1];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const float2 v = *reinterpret_cast<const float2*>(p + i * 64 + lane * 2);
      o[2 * i] += f * v.x;
      o[2 * i + 1] += f * v.y;
    }
  }
  const float inv = 1.f / l;
  T* out = static_cast<T*>(a.out) + b * a.out_strides[0] + node * a.out_strides[1] +
           (int64_t)head * a.out_strides[2];
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const int col = i * 64 + lane * 2;
    if (col < a.head_dim)
      *reinterpret_cast<uint32_t*>(out + col) = Kind<T>::pack(o[2 * i] * inv, o[2 * i + 1] * inv);
  }
  if (lane == 0 && a.lse != nullptr) a.lse[row] = (m + log2f(l)) * kLn2;
}

// ---------------------------------------------------------------- host

struct Plan {
  int wm, wk;  // warps along rows and keys
  Shape shape;
  int64_t workspace;
};

int padded_dim(int64_t head_dim) { return head_dim <= 64 ? 64 : 128; }

Plan plan_for(const ppyb200_tree_attention_args& a, int sm_count) {
  Plan p;
  p.shape.group = (int)(a.heads / a.kv_heads);
  const int64_t rows = a.nodes * p.shape.group;
  p.wm = rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 64 ? 4 : 8;
  p.wk = p.wm == 1 ? 4 : p.wm == 2 ? 2 : 1;
  p.shape.row_tiles = (int)((rows + 16 * p.wm - 1) / (16 * p.wm));
  const int64_t ctas = a.batch * a.kv_heads * p.shape.row_tiles;
  const int64_t tiles = (a.capacity + kTile - 1) / kTile;
  // enough CTAs for four on every SM, each with at least two tiles of a full cache
  int64_t splits = (4 * (int64_t)sm_count + ctas - 1) / ctas;
  splits = splits < 1 ? 1 : splits > (tiles + 1) / 2 ? (tiles + 1) / 2 : splits;
  p.shape.splits = (int)splits;
  p.workspace = splits == 1 ? 0 : a.batch * a.heads * a.nodes * splits *
                                      (padded_dim(a.head_dim) + 2) * 4;
  return p;
}

template <class T, int D, int WM, int WK>
cudaError_t launch_rows(const ppyb200_tree_attention_args& a, const Plan& p, cudaStream_t stream) {
  static ppyb200::DeviceOnce once;
  constexpr int smem = kStages * 2 * kTile * D * 2;
  int ready = 0;
  auto kernel = tree_attention_kernel<T, D, WM, WK>;
  cudaError_t e = once.get([&](int* value) {
    *value = 1;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  }, &ready);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)p.shape.splits, (unsigned)(a.kv_heads * p.shape.row_tiles),
                  (unsigned)a.batch);
  e = ppyb200::launch_pdl(kernel, grid, dim3(32 * WM * WK), smem, stream, a, p.shape,
                          static_cast<float*>(a.workspace));
  if (e != cudaSuccess || p.shape.splits == 1) return e;
  const int64_t rows = a.batch * a.heads * a.nodes;
  return ppyb200::launch_pdl(join_kernel<T, D>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0,
                             stream, a, p.shape.splits, static_cast<const float*>(a.workspace));
}

template <class T, int D>
cudaError_t launch_dim(const ppyb200_tree_attention_args& a, const Plan& p, cudaStream_t stream) {
  switch (p.wm) {
    case 1: return launch_rows<T, D, 1, 4>(a, p, stream);
    case 2: return launch_rows<T, D, 2, 2>(a, p, stream);
    case 4: return launch_rows<T, D, 4, 1>(a, p, stream);
    default: return launch_rows<T, D, 8, 1>(a, p, stream);
  }
}

template <class T>
cudaError_t launch_type(const ppyb200_tree_attention_args& a, const Plan& p,
                        cudaStream_t stream) {
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
      a.kv_heads * ((a.nodes * (a.heads / a.kv_heads) + 127) / 128) > 65535)
    return "batch up to 65535, kv_heads x row tiles of 128 up to 65535, capacity below 2^31";
  if (!rows16(a.q, a.q_strides) || !rows16(a.k_new, a.k_new_strides) ||
      !rows16(a.v_new, a.v_new_strides) || !rows16(a.keys, a.keys_strides) ||
      !rows16(a.values, a.values_strides) || !rows16(a.out, a.out_strides))
    return "every row of q, k, v, the cache and out starts on a 16-byte boundary";
  return nullptr;
}

}  // namespace

extern "C" {

int64_t ppyb200_tree_attention_workspace(const ppyb200_tree_attention_args* args) {
  if (args == nullptr || refusal(*args) != nullptr || args->batch == 0 || args->nodes == 0)
    return 0;
  return plan_for(*args, ppyb200_sm_count()).workspace;
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
  const Plan p = plan_for(a, ppyb200_sm_count());
  if (p.workspace > 0 && (a.workspace == nullptr || a.workspace_bytes < p.workspace ||
                          (reinterpret_cast<uintptr_t>(a.workspace) & 15u) != 0)) {
    ppyb200_set_error("ppyb200_tree_attention: a 16-byte aligned workspace of "
                      "ppyb200_tree_attention_workspace bytes required");
    return PPYB200_RAISED;
  }
  const cudaError_t e = a.dtype == PPYB200_BF16 ? launch_type<__nv_bfloat16>(a, p, stream)
                                                : launch_type<__half>(a, p, stream);
  if (e != cudaSuccess) return ppyb200_check((int32_t)e, "ppyb200_tree_attention");
  ppyb200_count_launches(p.shape.splits == 1 ? 1 : 2);
  return PPYB200_OK;
}

}  // extern "C"
