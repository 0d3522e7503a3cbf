// The cache behind the tree attention: accepting the verified path of a tree, and evicting
// entries by accumulated attention weight.
//
// accept    Path nodes p_0 < p_1 < ... of a sequence (a_b of them) were verified. Every entry's
//           accumulated weight grows by the attention that those rows paid to it,
//             w_j += sum over the key head's query heads and u < a_b of e^{s(p_u, j) - lse(p_u)},
//           the path's own entries starting from zero (entry t is seen by steps u >= t), and
//           their rows of K and V move from slots length + p_t to length + t.
// evict     Each key head keeps `budget` entries: those at the last `recent` positions first,
//           then by weight. Survivors in slots behind the budget fill the holes before it, both
//           in ascending order; the entries carry their positions, so order in the cache means
//           nothing. Sources lie behind the budget and holes before it: rows move in parallel,
//           and only the rows that have to move do.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include <type_traits>

#include <cooperative_groups.h>

#include "../../include/ppyb200.h"
#include "mma16.cuh"
#include "ppyb200_device.cuh"

namespace {

using namespace ppyb200::mma16;

__device__ __forceinline__ void raise(int32_t* status) {
  if (status != nullptr) atomicMax(status, PPYB200_DEVICE_RAISED);
}

int32_t refuse(const char* who, const char* what) {
  char text[256];
  snprintf(text, sizeof text, "%s: %s", who, what);
  ppyb200_set_error(text);
  return PPYB200_RAISED;
}

// ---------------------------------------------------------------- accept

constexpr int kAcceptThreads = 128;

// Sixteen keys of a warp against the path's rows: the sums of e^{s - lse} over the rows for key
// gid (sum0) and gid + 8 (sum1), complete in every lane of the quad. A fragments come straight
// from global memory: lane tig of a quad holds 16-byte pieces tig, tig + 4, ... of its rows, and
// since a product may take the head dimension in any order, columns 8 p .. 8 p + 3 of piece p
// serve as its columns (2 tig, +1, +8, +9) of one 16-deep step and the next four of another; the
// query fragments in shared memory are laid out to match.
template <class T, int D>
struct KeyRows {
  uint32_t a[D / 16][4];
  __device__ __forceinline__ void load(const T* lo, const T* hi, int d, int tig) {
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const int col = (c * 4 + tig) * 8;
      uint4 x = make_uint4(0, 0, 0, 0), y = x;
      if (lo != nullptr && col < d) x = __ldg(reinterpret_cast<const uint4*>(lo + col));
      if (hi != nullptr && col < d) y = __ldg(reinterpret_cast<const uint4*>(hi + col));
      a[2 * c][0] = x.x;
      a[2 * c][1] = y.x;
      a[2 * c][2] = x.y;
      a[2 * c][3] = y.y;
      a[2 * c + 1][0] = x.z;
      a[2 * c + 1][1] = y.z;
      a[2 * c + 1][2] = x.w;
      a[2 * c + 1][3] = y.w;
    }
  }
  // first0, first1: the first row that sees key gid and gid + 8
  __device__ __forceinline__ void weigh(const uint2* qf, const float* lse, int rows, float scale,
                                        int lane, int first0, int first1, float& sum0,
                                        float& sum1) const {
    const int tig = lane & 3;
    sum0 = sum1 = 0.f;
    for (int n = 0; n * 8 < rows; ++n) {
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        const uint2 b = qf[(n * (D / 16) + s) * 32 + lane];
        Kind<T>::mma(c, a[s], b.x, b.y);
      }
      const int r = n * 8 + tig * 2;
      const float2 l = *reinterpret_cast<const float2*>(lse + r);
      if (r >= first0 && r < rows) sum0 += exp2_sfu(fmaf(c[0], scale, -l.x));
      if (r + 1 >= first0 && r + 1 < rows) sum0 += exp2_sfu(fmaf(c[1], scale, -l.y));
      if (r >= first1 && r < rows) sum1 += exp2_sfu(fmaf(c[2], scale, -l.x));
      if (r + 1 >= first1 && r + 1 < rows) sum1 += exp2_sfu(fmaf(c[3], scale, -l.y));
    }
#pragma unroll
    for (int w = 1; w < 4; w <<= 1) {
      sum0 += __shfl_xor_sync(0xffffffffu, sum0, w);
      sum1 += __shfl_xor_sync(0xffffffffu, sum1, w);
    }
  }
};

// A CTA takes a stretch of one key head's entries and runs all the path's rows against them: keys
// are read once, straight into fragments, values not at all (only the path's own rows move). Bound
// by memory: 1152 key heads of 1700 to 4000 entries, 64 wide, 81 us, 5.1 TB/s.
template <class T, int D>
__global__ void __launch_bounds__(kAcceptThreads, D == 64 ? 8 : 5)
accept_kernel(const __grid_constant__ ppyb200_accept_args a,
              const __grid_constant__ ppyb200_accept_part_args part, const int chunks,
              const int chunk_keys) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int path[PPYB200_PATH_STEPS];
  __shared__ int valid;  // steps up to the first that is not in order
  ppyb200::pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gid = lane >> 2, tig = lane & 3;
  const int layer = blockIdx.z / (int)a.batch, b = blockIdx.z % (int)a.batch;
  const int kvh = blockIdx.y, group = (int)(a.heads / a.kv_heads), d = (int)a.head_dim;
  const bool last = (int)blockIdx.x == chunks;  // the CTA of the path's own entries

  // the piece's steps: none where the piece before was cut
  const int first = (int)part.first, steps = (int)a.steps;
  const int before = first > 0 ? part.taken_before[b] : 0;
  int64_t length = a.lengths[b];
  int n = a.accepted[b];
  const int shortest = before == first ? first : 0;
  bool bad = length < shortest || length > a.capacity || n < 0 || n > part.path_steps;
  n = before != first || length < first ? 0 : min(max(n - first, 0), steps);
  length = length < 0 ? 0 : (length > a.capacity ? a.capacity : length);
  const int64_t nodes_at = length - first;  // the slot of the attention's first node
  const int nodes = part.counts == nullptr ? (int)a.nodes : min((int)a.nodes, part.counts[b]);
  if (tid == 0) valid = n;
  __syncthreads();
  for (int t = tid; t < n; t += kAcceptThreads) {
    const int32_t* from = a.path + b * part.path_stride + first + t;
    const int p = from[0];
    path[t] = p;
    if (p <= (first + t > 0 ? from[-1] : -1) || p >= nodes || nodes_at + p >= a.capacity)
      atomicMin(&valid, t);
  }
  __syncthreads();
  if (valid < n) bad = true;
  n = valid;
  if (last && kvh == 0 && tid == 0) {
    if (bad) raise(a.status);
    if (layer == 0 && part.taken != nullptr) part.taken[b] = before + n;
  }
  if (n <= 0) return;
  const int64_t j0 = (int64_t)blockIdx.x * chunk_keys;
  if (!last && j0 >= length) return;

  const int rows = n * group, blocks = (rows + 7) / 8;
  uint2* qf = reinterpret_cast<uint2*>(smem);
  float* lse = reinterpret_cast<float*>(smem + (size_t)blocks * 8 * D * 2);
  if (a.weights != nullptr) {
    const T* q = static_cast<const T*>(a.q) + layer * a.q_strides[0] + b * a.q_strides[1];
    for (int i = tid; i < blocks * (D / 16) * 32; i += kAcceptThreads) {
      const int l = i & 31, s = (i >> 5) % (D / 16), r = (i / (32 * (D / 16))) * 8 + (l >> 2);
      const int col = ((s >> 1) * 4 + (l & 3)) * 8 + (s & 1) * 4;
      uint2 v = make_uint2(0, 0);
      if (r < rows && col < d)
        v = *reinterpret_cast<const uint2*>(q + path[r / group] * a.q_strides[2] +
                                            (int64_t)(kvh * group + r % group) * a.q_strides[3] +
                                            col);
      qf[i] = v;
    }
    for (int r = tid; r < blocks * 8; r += kAcceptThreads) {
      lse[r] = r < rows
                   ? a.lse[(((int64_t)layer * a.batch + b) * a.heads + kvh * group + r % group) *
                               a.nodes + path[r / group]] * kLog2e
                   : 0.f;
    }
    __syncthreads();
  }
  const float scale = (float)a.scale * kLog2e;
  T* keys = static_cast<T*>(a.keys) + layer * a.keys_strides[0] + b * a.keys_strides[1] +
            kvh * a.keys_strides[2];
  float* weights = a.weights == nullptr ? nullptr
                                        : a.weights + layer * a.weights_strides[0] +
                                              b * a.weights_strides[1] +
                                              kvh * a.weights_strides[2];
  if (!last) {
    const int64_t end = min(j0 + chunk_keys, length);
    // sixteen keys a warp at a time, the next sixteen and their weights under way meanwhile
    constexpr int kStep = kAcceptThreads / 2;
    KeyRows<T, D> k;
    auto load = [&](int64_t j, KeyRows<T, D>& to, float& weight) {
      const int64_t ja = j + gid, jb = ja + 8;
      to.load(ja < end ? keys + ja * a.keys_strides[3] : nullptr,
              jb < end ? keys + jb * a.keys_strides[3] : nullptr, d, tig);
      const int64_t mine = tig == 0 ? ja : jb;  // lanes 0 and 1 of a quad have a key each
      weight = tig < 2 && mine < end ? weights[mine] : 0.f;
    };
    float weight;
    load(j0 + warp * 16, k, weight);
#pragma unroll 1
    for (int64_t j = j0 + warp * 16; j < end; j += kStep) {
      KeyRows<T, D> next;
      float next_weight;
      load(j + kStep, next, next_weight);
      float s0, s1;
      k.weigh(qf, lse, rows, scale, lane, 0, 0, s0, s1);
      const int64_t mine = j + gid + (tig == 0 ? 0 : 8);
      if (tig < 2 && mine < end) weights[mine] = weight + (tig == 0 ? s0 : s1);
      k = next;
      weight = next_weight;
    }
    return;
  }

  // the path's own entries: their weights while the keys are where the attention left them ...
  if (weights != nullptr) {
    for (int t = warp * 16; t < n; t += kAcceptThreads / 2) {
      const int ta = t + gid, tb = ta + 8;
      KeyRows<T, D> k;
      k.load(ta < n ? keys + (nodes_at + path[ta]) * a.keys_strides[3] : nullptr,
             tb < n ? keys + (nodes_at + path[tb]) * a.keys_strides[3] : nullptr, d, tig);
      float s0, s1;
      k.weigh(qf, lse, rows, scale, lane, ta * group, tb * group, s0, s1);
      if (tig == 0 && ta < n) weights[length + ta] = s0;
      if (tig == 1 && tb < n) weights[length + tb] = s1;
    }
  }
  if (a.positions != nullptr) {
    int32_t* positions = a.positions + layer * a.weights_strides[0] + b * a.weights_strides[1] +
                         kvh * a.weights_strides[2];
    for (int t = tid; t < n; t += kAcceptThreads) positions[length + t] = a.seen[b] + t;
  }
  // ... then the rows, through shared memory, since a row's new slot may be another's old one
  T* values = static_cast<T*>(a.values) + layer * a.values_strides[0] + b * a.values_strides[1] +
              kvh * a.values_strides[2];
  uint4* box = reinterpret_cast<uint4*>(smem);
  const int pieces = d / 8;
  __syncthreads();
  for (int i = tid; i < n * pieces * 2; i += kAcceptThreads) {
    const int piece = i % pieces, t = (i / pieces) >> 1;
    const int64_t slot = nodes_at + path[t];
    box[i] = ((i / pieces) & 1) == 0
                 ? *reinterpret_cast<const uint4*>(keys + slot * a.keys_strides[3] + piece * 8)
                 : *reinterpret_cast<const uint4*>(values + slot * a.values_strides[3] +
                                                   piece * 8);
  }
  __syncthreads();
  for (int i = tid; i < n * pieces * 2; i += kAcceptThreads) {
    const int piece = i % pieces, t = (i / pieces) >> 1;
    const int64_t slot = length + t;
    if (((i / pieces) & 1) == 0)
      *reinterpret_cast<uint4*>(keys + slot * a.keys_strides[3] + piece * 8) = box[i];
    else
      *reinterpret_cast<uint4*>(values + slot * a.values_strides[3] + piece * 8) = box[i];
  }
}

template <class T, int D>
cudaError_t launch_accept(const ppyb200_accept_args& a, const ppyb200_accept_part_args& part,
                          cudaStream_t stream) {
  static ppyb200::DeviceOnce once;
  const int64_t rows = (a.steps * (a.heads / a.kv_heads) + 7) / 8 * 8;
  const int64_t queries = rows * (D * 2 + 4), box = a.steps * a.head_dim * 4;
  const size_t smem = (size_t)(queries > box ? queries : box);
  int ready = 0;
  auto kernel = accept_kernel<T, D>;
  cudaError_t e = once.get([&](int* value) {
    *value = 1;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                PPYB200_PATH_ROWS * (D * 2 + 4));
  }, &ready);
  if (e != cudaSuccess) return e;
  // Two waves of eight CTAs an SM over full caches, 128 to 4096 keys each: a CTA's start (lengths,
  // path, queries: loads that follow one another) costs as much as some hundred keys.
  const int64_t heads = a.layers * a.batch * a.kv_heads;
  int64_t chunk = heads * a.capacity / (16 * (int64_t)ppyb200_sm_count());
  chunk = chunk < 128 ? 128 : chunk > 4096 ? 4096 : (chunk + 63) / 64 * 64;
  const int chunks = a.weights == nullptr ? 0 : (int)((a.capacity + chunk - 1) / chunk);
  return ppyb200::launch_pdl(kernel,
                             dim3((unsigned)chunks + 1, (unsigned)a.kv_heads,
                                  (unsigned)(a.layers * a.batch)),
                             dim3(kAcceptThreads), smem, stream, a, part, chunks, (int)chunk);
}

// ---------------------------------------------------------------- evict

constexpr int kSelectThreads = 256;
constexpr int kBins = 2048;           // of a digit of a rank
constexpr int kCachedRanks = 16384;   // ranks a CTA keeps in shared memory
constexpr int kMoveRows = 32;  // rows a CTA moves

// An entry's rank as an unsigned number: protected entries above every weight, weights in
// order (the two zeros alike), NaN below them all.
__device__ __forceinline__ uint32_t entry_key(float w, int32_t position, int64_t protect_from) {
  if (position >= protect_from) return 0xffffffffu;
  if (w != w) return 0u;
  const uint32_t bits = __float_as_uint(w + 0.f);
  return (bits >> 31) != 0 ? ~bits : bits | 0x80000000u;
}

// Adds one to each lane's bin; lanes that share the first lane's bin (entries that never gathered
// any weight fall into one) add once for all.
__device__ __forceinline__ void count_bins(uint32_t* bins, uint32_t bin, bool valid) {
  const uint32_t first = __shfl_sync(0xffffffffu, bin, 0);
  const unsigned same = __ballot_sync(0xffffffffu, valid && bin == first);
  if (valid && bin == first) {
    if ((threadIdx.x & 31) == __ffs(same) - 1) atomicAdd(&bins[first], __popc(same));
  } else if (valid) {
    atomicAdd(&bins[bin], 1u);
  }
}

// Exclusive prefix sums of 32 kPer numbers in shared memory, by one warp; returns their sum.
template <int kPer>
__device__ __forceinline__ uint32_t warp_prefix(uint32_t* numbers) {
  const int lane = threadIdx.x & 31;
  uint32_t mine[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    mine[i] = numbers[lane * kPer + i];
    sum += mine[i];
  }
  uint32_t run = sum;
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, run, w);
    if (lane >= w) run += up;
  }
  uint32_t before = run - sum;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    numbers[lane * kPer + i] = before;
    before += mine[i];
  }
  return __shfl_sync(0xffffffffu, run, 31);
}

constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kWalkRows = 8;  // rows of kSelectThreads entries that the walk takes at once
constexpr int kWalkParts = kWalkRows * kSelectWarps;

struct SelectShared {
  alignas(16) uint32_t bins[2][kBins];  // of a digit, read by the whole cluster
  uint32_t sums[kSelectWarps];
  uint32_t equal[kWalkParts], holes[kWalkParts], sources[kWalkParts];  // by row and warp
  uint32_t all[3];     // of the rows together
  uint32_t counts[4];  // entries above / equal to the threshold, before / behind the budget
  uint32_t slice;      // entries in this CTA's slice of the bins
  uint32_t picked, rest;
};

// A cluster a key head; each CTA takes a stretch of its entries and keeps their ranks in shared
// memory where they fit (`cached` of them). The budget-th rank is found digit by digit (11, 11
// and 10 bits): every CTA counts its own entries, adds up a slice of the bins over the cluster from
// the others' shared memory, and reads the slice that holds the digit. Then each walks its entries
// in slot order, writes the tables of those that stay in front of the budget, and lists holes and
// sources; the lists filled, the holes' tables follow.
// Each weight is read from memory once (64 heads of 40001-65000 entries: 27 MB in, 21 MB out); the
// 62 us there are the steps that follow one another: three digits with a cluster barrier each,
// and the counting in shared memory between them.
// Loops stay rolled: a kernel of some microseconds waits for each line of its code once.
__global__ void __launch_bounds__(kSelectThreads, 4) evict_select_kernel(const ppyb200_evict_args a,
                                                                     const int64_t most,
                                                                     const int cached) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ SelectShared s;
  ppyb200::pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = (int)blockIdx.x / ranks, kv_heads = (int)a.kv_heads, batch = (int)a.batch;
  const int row = head / kv_heads, h = head - row * kv_heads;
  const int layer = row / batch, b = row - layer * batch;
  int length = a.lengths[b];
  if (length < 0 || length > a.capacity) {
    if (layer == 0 && h == 0 && tid == 0) raise(a.status);
    length = length < 0 ? 0 : (int)a.capacity;
  }
  const int budget = (int)a.budget;
  const int64_t protect_from = (int64_t)a.seen[b] - a.recent;
  const int64_t at = layer * a.weights_strides[0] + b * a.weights_strides[1] +
                     h * a.weights_strides[2];
  const int64_t out_at = layer * a.out_strides[0] + b * a.out_strides[1] + h * a.out_strides[2];
  const float* weights = a.weights + at;
  const int32_t* positions = a.positions + at;
  float* weights_out = a.weights_out + out_at;
  int32_t* positions_out = a.positions_out + out_at;
  int32_t* kept = a.kept + (int64_t)head * budget;
  int32_t* moves = static_cast<int32_t*>(a.workspace);  // counts, then holes and sources
  int32_t* holes = moves + a.layers * a.batch * a.kv_heads + head * 2 * most;
  int32_t* sources = holes + most;
  const int step = kSelectThreads * ranks, first_thread = rank * kSelectThreads + tid;
  auto sync_all = [&] {
    if (ranks == 1) __syncthreads();
    else cluster.sync();
  };

  if (length <= budget) {  // nothing to evict
    for (int64_t j = first_thread; j < budget; j += step) {
      kept[j] = j < length ? (int32_t)j : -1;
      if (j < length) {
        const float w = weights[j];
        const int32_t p = positions[j];
        weights_out[j] = w;
        positions_out[j] = p;
      }
    }
    if (rank == 0 && tid == 0) moves[head] = 0;
    return;  // the whole cluster
  }

  const int stretch = (length + ranks - 1) / ranks;
  const int begin = min(rank * stretch, length), end = min(begin + stretch, length);
  const int in_cache = min(end - begin, cached);
  auto key_of = [&](int j) {
    return j - begin < in_cache ? keys[j - begin]
                                : entry_key(weights[j], positions[j], protect_from);
  };
  // four entries from j on, begin + a multiple of four
  auto keys_of = [&](int j) {
    if (j - begin + 3 < in_cache) return *reinterpret_cast<const uint4*>(keys + (j - begin));
    return make_uint4(j < end ? key_of(j) : 0u, j + 1 < end ? key_of(j + 1) : 0u,
                      j + 2 < end ? key_of(j + 2) : 0u, j + 3 < end ? key_of(j + 3) : 0u);
  };
  if (tid < 4) s.counts[tid] = 0;

  uint32_t prefix = 0;
  uint32_t need = (uint32_t)budget;  // entries to take among those that share the prefix
#pragma unroll 1
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
    const int bins = digit == 2 ? kBins / 2 : kBins;
    const uint32_t known = ~0u << (digit == 1 ? 21 : 10);
    // The third digit has the first's memory: every CTA had read it before the second's barrier.
    uint32_t* mine = s.bins[digit & 1];
#pragma unroll 1
    for (int i = tid; i < kBins / 4; i += kSelectThreads)
      reinterpret_cast<uint4*>(mine)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (digit == 0) {
#pragma unroll 1
      for (int j0 = begin; j0 < end; j0 += 8 * kSelectThreads) {
        float w[8];
        int32_t p[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {  // all loads first
          const int j = j0 + u * kSelectThreads + tid;
          w[u] = j < end ? weights[j] : 0.f;
          p[u] = j < end ? positions[j] : 0;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int j = j0 + u * kSelectThreads + tid;
          const uint32_t key = entry_key(w[u], p[u], protect_from);
          if (j < end && j - begin < in_cache) keys[j - begin] = key;
          count_bins(mine, key >> 21, j < end);
        }
      }
    } else {
#pragma unroll 1
      for (int j0 = begin; j0 < end; j0 += 4 * kSelectThreads) {
        const uint4 four = keys_of(j0 + 4 * tid);
        const uint32_t key[4] = {four.x, four.y, four.z, four.w};
        bool counts[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          counts[u] = j0 + 4 * tid + u < end && ((key[u] ^ prefix) & known) == 0;
        if (__any_sync(0xffffffffu, counts[0] || counts[1] || counts[2] || counts[3]))
#pragma unroll
          for (int u = 0; u < 4; ++u)
            count_bins(mine, (key[u] >> shift) & (uint32_t)(bins - 1), counts[u]);
      }
    }
    sync_all();
    const int slice = bins / ranks;
    if (ranks > 1) {
      uint32_t sum = 0;
#pragma unroll 1
      for (int i = rank * slice + tid; i < (rank + 1) * slice; i += kSelectThreads) {
        uint32_t c = 0;
#pragma unroll 1
        for (int q = 0; q < ranks; ++q) c += cluster.map_shared_rank(mine, q)[i];
        mine[i] = c;  // no other CTA reads this slice of this CTA's before the next barrier
        sum += c;
      }
      sum = __reduce_add_sync(0xffffffffu, sum);
      if (lane == 0) s.sums[warp] = sum;
      __syncthreads();
      if (tid == 0) {
        uint32_t all = 0;
        for (int w = 0; w < kSelectWarps; ++w) all += s.sums[w];
        s.slice = all;
      }
      cluster.sync();
    }
    // the slice that holds the need-th entry from the top, then its bins from the top
    uint32_t above = 0;
    int owner = ranks - 1;
#pragma unroll 1
    for (; ranks > 1 && owner > 0; --owner) {
      const uint32_t all = *cluster.map_shared_rank(&s.slice, owner);
      if (above + all >= need) break;
      above += all;
    }
    const uint32_t* from = cluster.map_shared_rank(mine, owner) + owner * slice;
    const int each = (slice + kSelectThreads - 1) / kSelectThreads;
    const int top = slice - 1 - tid * each;  // this thread's highest bin of the slice
    uint32_t sum = 0;
#pragma unroll 1
    for (int i = 0; i < each; ++i) sum += top - i >= 0 ? from[top - i] : 0u;
    uint32_t run = sum;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, run, w);
      if (lane >= w) run += up;
    }
    if (lane == 31) s.sums[warp] = run;
    __syncthreads();
    above += run - sum;
#pragma unroll
    for (int w = 0; w < kSelectWarps; ++w) above += w < warp ? s.sums[w] : 0u;
    if (above < need && need <= above + sum) {  // one thread
#pragma unroll 1
      for (int i = 0; i < each; ++i) {
        const uint32_t c = from[top - i];
        if (need <= above + c) {
          s.picked = (uint32_t)(owner * slice + top - i);
          s.rest = need - above;
          break;
        }
        above += c;
      }
    }
    __syncthreads();
    prefix |= s.picked << shift;
    need = s.rest;
  }
  const uint32_t threshold = prefix;  // take every larger rank and the first `need` equal ones

  {  // entries of this stretch above and equal to the threshold, before and behind the budget
    uint32_t more[4] = {0, 0, 0, 0};
#pragma unroll 1
    for (int j = begin + 4 * tid; j < end; j += 4 * kSelectThreads) {
      const uint4 four = keys_of(j);
      const uint32_t key[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool above = j + u < end && key[u] > threshold;
        const bool same = j + u < end && key[u] == threshold, front = j + u < budget;
        more[0] += above && front ? 1 : 0;
        more[1] += above && !front ? 1 : 0;
        more[2] += same && front ? 1 : 0;
        more[3] += same && !front ? 1 : 0;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t sum = __reduce_add_sync(0xffffffffu, more[i]);
      if (lane == 0 && sum != 0) atomicAdd(&s.counts[i], sum);
    }
  }
  sync_all();
  // holes and sources of the earlier CTAs' stretches, and all of them; equal entries are taken in
  // slot order, so early stretches and early entries first
  uint32_t hole_count = 0, source_count = 0, all_holes = 0, equal_before = 0;
  uint32_t left = need, own_left = 0, own_equal = 0;
#pragma unroll 1
  for (int q = 0; q < ranks; ++q) {
    const uint32_t* other = cluster.map_shared_rank(s.counts, q);
    const uint32_t equal = other[2] + other[3];
    const uint32_t taken = min(left, equal), early = min(taken, other[2]);
    const int from = min(q * stretch, length), to = min(from + stretch, length);
    const uint32_t gone = (uint32_t)(min(to, max(from, budget)) - from) - other[0] - early;
    if (q < rank) {
      hole_count += gone;
      source_count += other[1] + taken - early;
      equal_before += equal;
    }
    if (q == rank) {
      own_left = taken;
      own_equal = equal;
    }
    all_holes += gone;
    left -= taken;
  }
  // in most stretches all equal entries stay or all go, and their order does not matter
  const bool ordered = own_left != 0 && own_left != own_equal;

  // Rows of kSelectThreads entries, eight at once, first those in front of the budget: a warp's
  // votes give an entry's place within its row and warp, the prefix sums over rows and warps the
  // rest.
  const unsigned below = (1u << lane) - 1u;
  auto walk = [&](auto is_front, int from, int to, uint32_t* places, int32_t* list,
                  uint32_t count) {
    constexpr bool kFront = decltype(is_front)::value;
#pragma unroll 1
    for (int j0 = from; j0 < to; j0 += kWalkRows * kSelectThreads) {
      uint32_t key[kWalkRows];
      float w[kWalkRows];
      int32_t p[kWalkRows];
#pragma unroll
      for (int i = 0; i < kWalkRows; ++i) {
        const int j = j0 + i * kSelectThreads + tid;
        key[i] = j < to ? key_of(j) : 0u;
        if (kFront && j < to) {  // under way while the places are found
          w[i] = weights[j];
          p[i] = positions[j];
        }
      }
      uint32_t keep = 0;  // a bit a row
      if (ordered) {
#pragma unroll 1
        for (int i = 0; i < kWalkRows; ++i) {
          const bool same = j0 + i * kSelectThreads + tid < to && key_of(min(
              j0 + i * kSelectThreads + tid, to - 1)) == threshold;
          const unsigned votes = __ballot_sync(0xffffffffu, same);
          if (lane == 0) s.equal[i * kSelectWarps + warp] = __popc(votes);
        }
        __syncthreads();
        if (warp == 0) {
          const uint32_t all = warp_prefix<kWalkParts / 32>(s.equal);
          if (lane == 0) s.all[0] = all;
        }
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < kWalkRows; ++i) {
        const int j = j0 + i * kSelectThreads + tid;
        const bool same = j < to && key[i] == threshold;
        bool stays = j < to && (key[i] > threshold || (same && own_left != 0));
        if (ordered) {
          const unsigned votes = __ballot_sync(0xffffffffu, same);
          if (same)
            stays = equal_before + s.equal[i * kSelectWarps + warp] + __popc(votes & below) < need;
        }
        if (stays) keep |= 1u << i;
        const unsigned moving = __ballot_sync(0xffffffffu, kFront ? j < to && !stays : stays);
        if (lane == 0) places[i * kSelectWarps + warp] = __popc(moving);
      }
      if (ordered) equal_before += s.all[0];
      __syncthreads();
      if (warp == 0) {
        const uint32_t all = warp_prefix<kWalkParts / 32>(places);
        if (lane == 0) s.all[1] = all;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kWalkRows; ++i) {
        const int j = j0 + i * kSelectThreads + tid;
        const bool stays = ((keep >> i) & 1u) != 0;
        const bool moves = kFront ? j < to && !stays : stays;
        const unsigned votes = __ballot_sync(0xffffffffu, moves);
        if (moves) list[count + places[i * kSelectWarps + warp] + __popc(votes & below)] = j;
        if (kFront && stays) {
          kept[j] = j;
          weights_out[j] = w[i];
          positions_out[j] = p[i];
        }
      }
      count += s.all[1];
    }
  };
  const int middle = min(end, max(begin, budget));
  walk(std::true_type{}, begin, middle, s.holes, holes, hole_count);
  walk(std::false_type{}, middle, end, s.sources, sources, source_count);
  if (rank == 0 && tid == 0) moves[head] = (int32_t)all_holes;
  sync_all();  // the lists are complete, and no CTA reads another's shared memory any more
  for (uint32_t r = first_thread; r < all_holes; r += step) {
    const int32_t to = holes[r], from = sources[r];
    kept[to] = from;
    weights_out[to] = weights[from];
    positions_out[to] = positions[from];
  }
}

// Rows of K and V from the sources to the holes (disjoint), kMoveRows a CTA. Bound by memory: 64
// heads of 40001 to 65000 entries of 128 cut to 16384, 111 us, 6.8 TB/s of reads and writes.
__global__ void __launch_bounds__(128) evict_move_kernel(const ppyb200_evict_args a,
                                                         const int64_t most) {
  ppyb200::pdl_wait();
  const int64_t head = blockIdx.y;
  const int32_t* moves = static_cast<const int32_t*>(a.workspace);
  const int64_t count = moves[head], r0 = (int64_t)blockIdx.x * kMoveRows;
  if (r0 >= count) return;
  const int64_t n = count - r0 < kMoveRows ? count - r0 : kMoveRows;
  const int h = (int)(head % a.kv_heads), b = (int)(head / a.kv_heads % a.batch);
  const int layer = (int)(head / a.kv_heads / a.batch);
  const int32_t* holes = moves + a.layers * a.batch * a.kv_heads + head * 2 * most + r0;
  const int32_t* sources = holes + most;
  uint16_t* keys = static_cast<uint16_t*>(a.keys) + layer * a.keys_strides[0] +
                   b * a.keys_strides[1] + h * a.keys_strides[2];
  uint16_t* values = static_cast<uint16_t*>(a.values) + layer * a.values_strides[0] +
                     b * a.values_strides[1] + h * a.values_strides[2];
  const int pieces = (int)a.head_dim / 8;
  for (int i = threadIdx.x; i < (int)n * pieces; i += 128) {
    const int r = i / pieces, piece = i % pieces;
    const int64_t from = sources[r], to = holes[r];
    const uint4 k = *reinterpret_cast<const uint4*>(keys + from * a.keys_strides[3] + piece * 8);
    const uint4 v =
        *reinterpret_cast<const uint4*>(values + from * a.values_strides[3] + piece * 8);
    *reinterpret_cast<uint4*>(keys + to * a.keys_strides[3] + piece * 8) = k;
    *reinterpret_cast<uint4*>(values + to * a.values_strides[3] + piece * 8) = v;
  }
}

// ---------------------------------------------------------------- host

bool rows16(const void* p, const int64_t* strides, int count) {
  if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0) return false;
  for (int i = 0; i < count; ++i)
    if (strides[i] % 8 != 0) return false;
  return true;
}

int64_t most_moves(const ppyb200_evict_args& a) {
  const int64_t behind = a.capacity - a.budget;
  return behind <= 0 ? 0 : behind < a.budget ? behind : a.budget;
}

// Clusters of the select kernel: twice the CTAs for a head (up to eight) while four CTAs an SM hold
// them all and a stretch keeps 2048 entries. 64 heads of 40001-65000 entries: one CTA a head
// 286 us, eight 62 us. 576 heads of 700-1000 entries have one each (20 us).
cudaError_t launch_select(const ppyb200_evict_args& a, int64_t heads, int64_t most, int sm_count,
                          cudaStream_t stream) {
  static ppyb200::DeviceOnce once;
  int ready = 0;
  cudaError_t e = once.get([](int* value) {
    *value = 1;
    return cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kCachedRanks * 4);
  }, &ready);
  if (e != cudaSuccess) return e;
  int ranks = 1;
  while (ranks < 8 && heads * ranks * 2 <= 4 * (int64_t)sm_count &&
         a.capacity >= (int64_t)ranks * 2 * 2048)
    ranks *= 2;
  const int64_t stretch = (a.capacity + ranks - 1) / ranks;
  const int cached = (int)(stretch < kCachedRanks ? stretch : kCachedRanks);
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(heads * ranks));
  config.blockDim = dim3(kSelectThreads);
  config.dynamicSmemBytes = (size_t)(cached + 3) / 4 * 16;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = (unsigned)ranks;
  attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attributes;
  config.numAttrs = ppyb200_pdl() ? 2 : 1;
  return cudaLaunchKernelEx(&config, evict_select_kernel, a, most, cached);
}

const char* refusal(const ppyb200_evict_args& a) {
  if (a.layers < 0 || a.batch < 0 || a.kv_heads <= 0 || a.capacity < 0)
    return "no size is negative";
  if (a.budget <= 0 || a.budget > a.capacity) return "a budget of 1 up to the capacity";
  if (a.recent < 0) return "recent is not negative";
  if (a.head_dim <= 0 || a.head_dim % 8 != 0) return "head_dim is a multiple of 8";
  if (a.capacity > INT32_MAX || a.layers * a.batch * a.kv_heads > 65535)
    return "capacity below 2^31, layers x batch x kv_heads up to 65535";
  if (!rows16(a.keys, a.keys_strides, 4) || !rows16(a.values, a.values_strides, 4))
    return "every row of the cache starts on a 16-byte boundary";
  return nullptr;
}

}  // namespace

extern "C" {

int32_t ppyb200_accept_part(const ppyb200_accept_args* args,
                            const ppyb200_accept_part_args* part) {
  const char* who = "ppyb200_accept";
  if (args == nullptr || part == nullptr) return refuse(who, "no arguments");
  const ppyb200_accept_args& a = *args;
  if (a.dtype != PPYB200_BF16 && a.dtype != PPYB200_F16) return refuse(who, "dtype is bf16 or f16");
  if (a.layers < 0 || a.batch < 0 || a.nodes < 0 || a.steps < 0 || a.capacity < 0 ||
      a.heads <= 0 || a.kv_heads <= 0 || a.heads % a.kv_heads != 0)
    return refuse(who, "heads is a multiple of kv_heads, and no size is negative");
  if (a.head_dim <= 0 || a.head_dim > 128 || a.head_dim % 8 != 0)
    return refuse(who, "head_dim is a multiple of 8 up to 128");
  if (a.steps > PPYB200_PATH_STEPS || a.steps * (a.heads / a.kv_heads) > PPYB200_PATH_ROWS)
    return refuse(who, "a path of up to 64 steps, steps x query heads a key head up to 512");
  if (a.layers * a.batch > 65535 || a.kv_heads > 65535 || a.capacity > INT32_MAX)
    return refuse(who, "layers x batch and kv_heads up to 65535, capacity below 2^31");
  if (!rows16(a.keys, a.keys_strides, 4) || !rows16(a.values, a.values_strides, 4) ||
      (a.weights != nullptr && !rows16(a.q, a.q_strides, 4)))
    return refuse(who, "every row of q and the cache starts on a 16-byte boundary");
  if (a.weights != nullptr && (a.q == nullptr || a.lse == nullptr))
    return refuse(who, "weights take q and lse");
  if (part->first < 0 || part->path_steps > INT32_MAX || part->path_stride < 0 ||
      part->first + a.steps > part->path_steps || (part->first > 0 && part->taken_before == nullptr))
    return refuse(who, "a piece lies within its path and follows the steps taken before it");
  if (a.layers == 0 || a.batch == 0 || a.steps == 0) return PPYB200_OK;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(ppyb200_stream());
  cudaError_t e;
  if (a.dtype == PPYB200_BF16)
    e = a.head_dim <= 64 ? launch_accept<__nv_bfloat16, 64>(a, *part, stream)
                         : launch_accept<__nv_bfloat16, 128>(a, *part, stream);
  else
    e = a.head_dim <= 64 ? launch_accept<__half, 64>(a, *part, stream)
                         : launch_accept<__half, 128>(a, *part, stream);
  if (e != cudaSuccess) return ppyb200_check((int32_t)e, who);
  ppyb200_count_launches(1);
  return PPYB200_OK;
}

int32_t ppyb200_accept(const ppyb200_accept_args* args) {
  if (args == nullptr) return refuse("ppyb200_accept", "no arguments");
  const ppyb200_accept_part_args whole = {nullptr, nullptr, nullptr, 0, args->steps, args->steps};
  return ppyb200_accept_part(args, &whole);
}

int64_t ppyb200_evict_workspace(const ppyb200_evict_args* args) {
  if (args == nullptr || refusal(*args) != nullptr) return 0;
  return args->layers * args->batch * args->kv_heads * (1 + 2 * most_moves(*args)) * 4;
}

int32_t ppyb200_evict(const ppyb200_evict_args* args) {
  if (args == nullptr) return refuse("ppyb200_evict", "no arguments");
  const ppyb200_evict_args& a = *args;
  const char* wrong = refusal(a);
  if (wrong != nullptr) return refuse("ppyb200_evict", wrong);
  const int64_t heads = a.layers * a.batch * a.kv_heads, most = most_moves(a);
  if (heads == 0) return PPYB200_OK;
  if (a.workspace == nullptr || a.workspace_bytes < ppyb200_evict_workspace(args) ||
      (reinterpret_cast<uintptr_t>(a.workspace) & 15u) != 0)
    return refuse("ppyb200_evict",
                  "a 16-byte aligned workspace of ppyb200_evict_workspace bytes required");
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(ppyb200_stream());
  cudaError_t e = launch_select(a, heads, most, ppyb200_sm_count(), stream);
  if (e == cudaSuccess && most > 0)
    e = ppyb200::launch_pdl(evict_move_kernel,
                            dim3((unsigned)((most + kMoveRows - 1) / kMoveRows), (unsigned)heads),
                            dim3(128), 0, stream, a, most);
  if (e != cudaSuccess) return ppyb200_check((int32_t)e, "ppyb200_evict");
  ppyb200_count_launches(most > 0 ? 2 : 1);
  return PPYB200_OK;
}

}  // extern "C"
