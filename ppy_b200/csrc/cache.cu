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
constexpr int kAcceptKeys = 512;  // prefix keys a CTA

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

template <class T, int D>
__global__ void __launch_bounds__(kAcceptThreads)
accept_kernel(const ppyb200_accept_args a, const int chunks) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int path[PPYB200_PATH_STEPS];
  __shared__ int valid;  // steps up to the first that is not in order
  ppyb200::pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gid = lane >> 2, tig = lane & 3;
  const int layer = blockIdx.z / (int)a.batch, b = blockIdx.z % (int)a.batch;
  const int kvh = blockIdx.y, group = (int)(a.heads / a.kv_heads), d = (int)a.head_dim;
  const bool last = (int)blockIdx.x == chunks;  // the CTA of the path's own entries

  int64_t length = a.lengths[b];
  int n = a.accepted[b];
  bool bad = length < 0 || length > a.capacity || n < 0 || n > a.steps;
  length = length < 0 ? 0 : (length > a.capacity ? a.capacity : length);
  n = n < 0 ? 0 : (n > (int)a.steps ? (int)a.steps : n);
  if (tid == 0) valid = n;
  __syncthreads();
  for (int t = tid; t < n; t += kAcceptThreads) {
    const int p = a.path[b * a.steps + t];
    const int before = t > 0 ? a.path[b * a.steps + t - 1] : -1;
    path[t] = p;
    if (p <= before || p >= a.nodes || length + p >= a.capacity) atomicMin(&valid, t);
  }
  __syncthreads();
  if (valid < n) bad = true;
  n = valid;
  if (bad && last && kvh == 0 && tid == 0) raise(a.status);
  if (n <= 0) return;
  const int64_t j0 = (int64_t)blockIdx.x * kAcceptKeys;
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
    if (weights == nullptr) return;
    const int64_t end = min(j0 + kAcceptKeys, length);
    for (int64_t j = j0 + warp * 16; j < end; j += kAcceptThreads / 2) {
      const int64_t ja = j + gid, jb = ja + 8;
      KeyRows<T, D> k;
      k.load(ja < end ? keys + ja * a.keys_strides[3] : nullptr,
             jb < end ? keys + jb * a.keys_strides[3] : nullptr, d, tig);
      float s0, s1;
      k.weigh(qf, lse, rows, scale, lane, 0, 0, s0, s1);
      if (tig == 0 && ja < end) weights[ja] += s0;
      if (tig == 1 && jb < end) weights[jb] += s1;
    }
    return;
  }

  // the path's own entries: their weights while the keys are where the attention left them ...
  if (weights != nullptr) {
    for (int t = warp * 16; t < n; t += kAcceptThreads / 2) {
      const int ta = t + gid, tb = ta + 8;
      KeyRows<T, D> k;
      k.load(ta < n ? keys + (length + path[ta]) * a.keys_strides[3] : nullptr,
             tb < n ? keys + (length + path[tb]) * a.keys_strides[3] : nullptr, d, tig);
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
    const int64_t slot = length + path[t];
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
cudaError_t launch_accept(const ppyb200_accept_args& a, cudaStream_t stream) {
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
  const int chunks = (int)((a.capacity + kAcceptKeys - 1) / kAcceptKeys);
  return ppyb200::launch_pdl(kernel,
                             dim3((unsigned)chunks + 1, (unsigned)a.kv_heads,
                                  (unsigned)(a.layers * a.batch)),
                             dim3(kAcceptThreads), smem, stream, a, chunks);
}

// ---------------------------------------------------------------- evict

constexpr int kSelectThreads = 512;
constexpr int kMoveRows = 32;  // rows a CTA moves

// An entry's rank as an unsigned number: protected entries above every weight, weights in
// order (the two zeros alike), NaN below them all.
__device__ __forceinline__ uint32_t entry_key(float w, int32_t position, int64_t protect_from) {
  if (position >= protect_from) return 0xffffffffu;
  if (w != w) return 0u;
  const uint32_t bits = __float_as_uint(w + 0.f);
  return (bits >> 31) != 0 ? ~bits : bits | 0x80000000u;
}

// Exclusive prefix sums over the block of two counts a thread (packed 16 + 16 bits; a chunk
// holds fewer than 65536 entries), and their totals.
__device__ __forceinline__ uint32_t block_prefix(uint32_t mine, uint32_t* totals,
                                                 uint32_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t run = mine;
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, run, w);
    if (lane >= w) run += up;
  }
  __syncthreads();  // the last call's totals have been read
  if (lane == 31) totals[warp] = run;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelectThreads / 32; ++w) {
    const uint32_t t = totals[w];
    if (w < warp) before += t;
    total += t;
  }
  return before + run - mine;
}

// One CTA a key head: finds the budget-th rank with four 8-bit histograms, then walks the
// entries in slot order, writes the tables of those that stay and lists holes and sources.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const ppyb200_evict_args a,
                                                                     const int64_t most) {
  __shared__ uint32_t bins[256];
  __shared__ uint32_t totals[kSelectThreads / 32];
  __shared__ uint32_t picked, rest;
  ppyb200::pdl_wait();
  const int tid = threadIdx.x;
  const int64_t head = blockIdx.x;
  const int h = (int)(head % a.kv_heads), b = (int)(head / a.kv_heads % a.batch);
  const int layer = (int)(head / a.kv_heads / a.batch);
  int64_t length = a.lengths[b];
  if (length < 0 || length > a.capacity) {
    if (layer == 0 && h == 0 && tid == 0) raise(a.status);
    length = length < 0 ? 0 : a.capacity;
  }
  const int64_t budget = a.budget, protect_from = (int64_t)a.seen[b] - a.recent;
  const int64_t at = layer * a.weights_strides[0] + b * a.weights_strides[1] +
                     h * a.weights_strides[2];
  const int64_t out_at = layer * a.out_strides[0] + b * a.out_strides[1] + h * a.out_strides[2];
  const float* weights = a.weights + at;
  const int32_t* positions = a.positions + at;
  float* weights_out = a.weights_out + out_at;
  int32_t* positions_out = a.positions_out + out_at;
  int32_t* kept = a.kept + head * budget;
  int32_t* moves = static_cast<int32_t*>(a.workspace);  // counts, then holes and sources
  int32_t* holes = moves + a.layers * a.batch * a.kv_heads + head * 2 * most;
  int32_t* sources = holes + most;

  if (length <= budget) {  // nothing to evict
    for (int64_t j = tid; j < budget; j += kSelectThreads) {
      kept[j] = j < length ? (int32_t)j : -1;
      if (j < length) {
        const float w = weights[j];
        const int32_t p = positions[j];
        weights_out[j] = w;
        positions_out[j] = p;
      }
    }
    if (tid == 0) moves[head] = 0;
    return;
  }

  // the budget-th largest key, eight bits at a time from the top
  uint32_t prefix = 0;
  int64_t need = budget;  // entries to take among those that share the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelectThreads) bins[i] = 0;
    __syncthreads();
    for (int64_t j = tid; j < length; j += kSelectThreads) {
      const uint32_t key = entry_key(weights[j], positions[j], protect_from);
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&bins[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid < 32) {  // lane l: bins 255 - 8 l down to 248 - 8 l
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) mine += bins[255 - 8 * tid - i];
      uint32_t run = mine;
#pragma unroll
      for (int w = 1; w < 32; w <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, run, w);
        if (tid >= w) run += up;
      }
      uint32_t above = run - mine;
      if ((int64_t)above < need && need <= (int64_t)run) {
        for (int i = 0; i < 8; ++i) {
          const uint32_t c = bins[255 - 8 * tid - i];
          if ((int64_t)(above + c) >= need) {
            picked = (uint32_t)(255 - 8 * tid - i);
            rest = (uint32_t)(need - above);
            break;
          }
          above += c;
        }
      }
    }
    __syncthreads();
    prefix |= picked << shift;
    need = rest;
    __syncthreads();
  }
  const uint32_t threshold = prefix;  // take every larger key and the first `need` equal ones

  constexpr int kItems = 4;
  int64_t equal_before = 0, hole_count = 0, source_count = 0;
  for (int64_t j0 = 0; j0 < length; j0 += kSelectThreads * kItems) {
    const int64_t first = j0 + tid * kItems;
    uint32_t key[kItems];
    uint32_t equal = 0;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int64_t j = first + i;
      key[i] = j < length ? entry_key(weights[j], positions[j], protect_from) : 0u;
      if (j < length && key[i] == threshold) ++equal;
    }
    uint32_t total;
    int64_t order = equal_before + block_prefix(equal, totals, total);
    equal_before += total;
    bool keep[kItems];
    uint32_t moving = 0;  // holes low, sources high
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int64_t j = first + i;
      keep[i] = j < length && key[i] > threshold;
      if (j < length && key[i] == threshold) keep[i] = order++ < need;
      if (j < budget && !keep[i]) moving += 1;
      if (j >= budget && keep[i]) moving += 1u << 16;
    }
    const uint32_t rank = block_prefix(moving, totals, total);
    int64_t hole = hole_count + (rank & 0xffffu), source = source_count + (rank >> 16);
    hole_count += total & 0xffffu;
    source_count += total >> 16;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int64_t j = first + i;
      if (j < budget) {
        if (keep[i]) {
          kept[j] = (int32_t)j;
          const float w = weights[j];
          const int32_t p = positions[j];
          weights_out[j] = w;
          positions_out[j] = p;
        } else {
          holes[hole++] = (int32_t)j;
        }
      } else if (keep[i]) {
        sources[source++] = (int32_t)j;
      }
    }
  }
  if (tid == 0) moves[head] = (int32_t)hole_count;
  __syncthreads();  // the lists are complete
  for (int64_t r = tid; r < hole_count; r += kSelectThreads) {
    const int32_t to = holes[r], from = sources[r];
    kept[to] = from;
    weights_out[to] = weights[from];
    positions_out[to] = positions[from];
  }
}

// Rows of K and V from the sources to the holes (disjoint), kMoveRows a CTA.
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

int32_t ppyb200_accept(const ppyb200_accept_args* args) {
  if (args == nullptr) return refuse("ppyb200_accept", "no arguments");
  const ppyb200_accept_args& a = *args;
  const char* who = "ppyb200_accept";
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
  if (a.layers == 0 || a.batch == 0 || a.steps == 0) return PPYB200_OK;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(ppyb200_stream());
  cudaError_t e;
  if (a.dtype == PPYB200_BF16)
    e = a.head_dim <= 64 ? launch_accept<__nv_bfloat16, 64>(a, stream)
                         : launch_accept<__nv_bfloat16, 128>(a, stream);
  else
    e = a.head_dim <= 64 ? launch_accept<__half, 64>(a, stream)
                         : launch_accept<__half, 128>(a, stream);
  if (e != cudaSuccess) return ppyb200_check((int32_t)e, who);
  ppyb200_count_launches(1);
  return PPYB200_OK;
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
  cudaError_t e = ppyb200::launch_pdl(evict_select_kernel, dim3((unsigned)heads),
                                      dim3(kSelectThreads), 0, stream, a, most);
  if (e == cudaSuccess && most > 0)
    e = ppyb200::launch_pdl(evict_move_kernel,
                            dim3((unsigned)((most + kMoveRows - 1) / kMoveRows), (unsigned)heads),
                            dim3(128), 0, stream, a, most);
  if (e != cudaSuccess) return ppyb200_check((int32_t)e, "ppyb200_evict");
  ppyb200_count_launches(most > 0 ? 2 : 1);
  return PPYB200_OK;
}

}  // extern "C"
