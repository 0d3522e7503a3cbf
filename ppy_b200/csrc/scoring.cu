// Log probabilities of given tokens, the entropy, and the likeliest alternatives of rows of
// logits, each row read from memory once.
//
//   m = max x,  Z = sum e^{x - m},  log p_i = x_i - m - log Z
//   H = - sum p log p = log Z - (sum (x - m) e^{x - m}) / Z
//
// m, Z and the sum T of (x - m) e^{x - m} run along the row with each other: when the maximum
// grows by D, Z becomes e^{-D} Z and T becomes e^{-D} (T - D Z). Everything is kept in powers of
// two (y = (x - m) log2 e), one exponential an element.
//
// The alternatives need no second pass over the row. A CTA's threads form 64 slots; the k-th
// largest of the slots' maxima is a lower bound for the k-th largest logit, and only slots whose
// maximum reaches it (about k of them) hold candidates: their elements, just read, come from L2
// again. The few candidates are ranked by counting.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/ppyb200.h"
#include "mma16.cuh"
#include "ppyb200_device.cuh"

namespace {

using ppyb200::mma16::exp2_sfu;
using ppyb200::mma16::kLn2;
using ppyb200::mma16::kLog2e;

constexpr int kSlots = PPYB200_TOP_LIMIT;
constexpr int kCandidates = 1024;
constexpr float kLeast = -200.f;  // 2^kLeast = 0 in f32: stands for -inf where 0 times it is 0

// A logit as an unsigned number in its order: NaN above all, the two zeros alike.
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t bits = __float_as_uint(x + 0.f);
  return (bits >> 31) != 0 ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float disordered(uint32_t key) {
  if (key == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((key >> 31) != 0 ? key & 0x7fffffffu : ~key);
}

template <class T>
struct Vector;
template <>
struct Vector<float> {
  static constexpr int kCount = 4;
  __device__ __forceinline__ static void load(const float* p, float (&v)[4]) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = x.x;
    v[1] = x.y;
    v[2] = x.z;
    v[3] = x.w;
  }
};
template <class T>
struct Vector16 {
  static constexpr int kCount = 8;
  __device__ __forceinline__ static void load(const T* p, float (&v)[8]) {
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = ppyb200::mma16::Kind<T>::unpack(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};
template <>
struct Vector<__nv_bfloat16> : Vector16<__nv_bfloat16> {};
template <>
struct Vector<__half> : Vector16<__half> {};

struct Sums {  // of a part of a row: maximum, Z and T in powers of two
  float m = -INFINITY, z = 0.f, t = 0.f;

  __device__ __forceinline__ void raise_to(float top) {
    const float drop = m == -INFINITY ? 0.f : fmaxf((m - top) * kLog2e, kLeast);
    const float f = exp2_sfu(drop);
    t = m == -INFINITY ? 0.f : f * (t + drop * z);
    z = m == -INFINITY ? 0.f : f * z;
    m = top;
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&v)[N]) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, v[i]);
    if (top > m) raise_to(top);
    const float u = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // the difference first: exact near the maximum, however large the logits are
      const float y = (v[i] - u) * kLog2e, e = exp2_sfu(y);
      z += e;
      t = fmaf(fmaxf(y, kLeast), e, t);
    }
  }
  __device__ __forceinline__ void join(const Sums& o) {
    Sums a = *this, b = o;
    const float top = fmaxf(a.m, b.m);
    if (top > a.m) a.raise_to(top);
    if (top > b.m) b.raise_to(top);
    m = top;
    z = a.z + b.z;
    t = a.t + b.t;
  }
};

// The elements of a row as a thread walks them: single ones up to the first 16-byte boundary,
// vectors, single ones to the end. Slot s is threads [s w, s w + w) with w = THREADS / kSlots.
template <class T>
struct Row {
  const T* x;
  int head, vectors, tail, vocab;
  static constexpr int kCount = Vector<T>::kCount;
  __device__ __forceinline__ Row(const T* row, int64_t count) : x(row), vocab((int)count) {
    const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15u) / (int)sizeof(T);
    head = off == 0 ? 0 : kCount - off;
    head = head < vocab ? head : vocab;
    vectors = (vocab - head) / kCount;
    tail = vocab - head - vectors * kCount;
  }
  __device__ __forceinline__ const T* vector(int i) const { return x + head + i * kCount; }
  __device__ __forceinline__ int tail_at() const { return vocab - tail; }
};

template <class T, int THREADS>
__global__ void __launch_bounds__(THREADS)
token_logprobs_kernel(const T* __restrict__ logits, int64_t vocab, int64_t pitch,
                      const int64_t* __restrict__ tokens, int given, int top,
                      float* __restrict__ logprobs, float* __restrict__ entropy,
                      float* __restrict__ top_logprobs, int64_t* __restrict__ top_tokens) {
  constexpr int kCount = Vector<T>::kCount, kWarps = THREADS / 32, kWidth = THREADS / kSlots;
  constexpr int kUnroll = 4;
  __shared__ Sums parts[kWarps];
  __shared__ uint32_t slot_max[kSlots];
  __shared__ uint32_t threshold, found;
  __shared__ uint64_t candidates[kCandidates];
  ppyb200::pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x;
  const Row<T> row(logits + r * pitch, vocab);

  Sums s;
  if (tid < row.head) {
    const float v[1] = {(float)row.x[tid]};
    s.add(v);
  }
  int i = tid;
  for (; i + (kUnroll - 1) * THREADS < row.vectors; i += kUnroll * THREADS) {
    float v[kUnroll][kCount];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) Vector<T>::load(row.vector(i + u * THREADS), v[u]);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) s.add(v[u]);
  }
  for (; i < row.vectors; i += THREADS) {
    float v[kCount];
    Vector<T>::load(row.vector(i), v);
    s.add(v);
  }
  if (tid < row.tail) {
    const float v[1] = {(float)row.x[row.tail_at() + tid]};
    s.add(v);
  }

  // the slots' maxima: 0 for a slot without elements; one with a NaN among them is searched
  if (top > 0) {
    uint32_t key = tid < row.head || tid < row.vectors || tid < row.tail ? ordered(s.m) : 0u;
    if (s.z != s.z) key = 0xffffffffu;  // NaN, or +inf: a bound that keeps the slot either way
#pragma unroll
    for (int w = 1; w < kWidth; w <<= 1)
      key = max(key, __shfl_xor_sync(0xffffffffu, key, w));
    if (tid % kWidth == 0) slot_max[tid / kWidth] = key;
  }
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) {
    Sums o;
    o.m = __shfl_xor_sync(0xffffffffu, s.m, w);
    o.z = __shfl_xor_sync(0xffffffffu, s.z, w);
    o.t = __shfl_xor_sync(0xffffffffu, s.t, w);
    s.join(o);
  }
  if (lane == 0) parts[warp] = s;
  if (tid == 0) found = 0;
  __syncthreads();
  s = parts[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) s.join(parts[w]);
  const float log_z = log2f(s.z) * kLn2;

  for (int c = tid; c < given; c += THREADS) {
    const int64_t token = tokens[r * given + c];
    logprobs[r * given + c] = token >= 0 && token < vocab
                                  ? ((float)row.x[token] - s.m) - log_z
                                  : __uint_as_float(0x7fc00000u);
  }
  if (tid == 0 && entropy != nullptr) entropy[r] = log_z - s.t / s.z * kLn2;
  if (top == 0) return;

  // the bound: the top-th largest slot maximum. Where a slot's maximum is only an upper bound
  // (a row with a NaN or an infinity) the slots are searched first.
  if (s.z != s.z) {
    __shared__ uint32_t exact_max[kSlots];
    if (tid < kSlots) exact_max[tid] = 0;
    __syncthreads();
    uint32_t key = 0;
    if (tid < row.head) key = max(key, ordered((float)row.x[tid]));
    for (int k = tid; k < row.vectors; k += THREADS) {
      float v[kCount];
      Vector<T>::load(row.vector(k), v);
#pragma unroll
      for (int e = 0; e < kCount; ++e) key = max(key, ordered(v[e]));
    }
    if (tid < row.tail) key = max(key, ordered((float)row.x[row.tail_at() + tid]));
    atomicMax(&exact_max[tid / kWidth], key);
    __syncthreads();
    if (tid < kSlots) slot_max[tid] = exact_max[tid];
    __syncthreads();
  }
  if (tid < kSlots) {
    const uint32_t mine = slot_max[tid];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < kSlots; ++j) {
      const uint32_t other = slot_max[j];
      rank += other > mine || (other == mine && j < tid) ? 1 : 0;
    }
    if (rank == top - 1) threshold = mine;
  }
  __syncthreads();
  const uint32_t bound = threshold;

  // a warp takes a slot: keys of at least `least` join the candidates as (key, ~index)
  auto collect = [&](uint32_t least) {
    for (int slot = warp; slot < kSlots; slot += kWarps) {
      if (slot_max[slot] < least) continue;
      auto offer = [&](float value, int index) {
        const uint32_t key = ordered(value);
        if (key < least) return;
        const uint32_t place = atomicAdd(&found, 1u);
        if (place < kCandidates) candidates[place] = ((uint64_t)key << 32) | (uint32_t)~index;
      };
      const int first = slot * kWidth;
      for (int t = first + lane; t < first + kWidth; t += 32) {
        if (t < row.head) offer((float)row.x[t], t);
        if (t < row.tail) offer((float)row.x[row.tail_at() + t], row.tail_at() + t);
      }
      constexpr int kAbreast = 32 / kWidth;
      for (int k = lane / kWidth;; k += kAbreast) {
        const int at = first + lane % kWidth + k * THREADS;
        if (at >= row.vectors) break;
        float v[kCount];
        Vector<T>::load(row.vector(at), v);
#pragma unroll
        for (int e = 0; e < kCount; ++e) offer(v[e], row.head + at * kCount + e);
      }
    }
  };
  auto write = [&](int rank, uint64_t candidate) {
    top_logprobs[r * top + rank] = (disordered((uint32_t)(candidate >> 32)) - s.m) - log_z;
    top_tokens[r * top + rank] = (int64_t)(uint32_t)~(uint32_t)candidate;
  };
  auto rank_candidates = [&](int count) {
    for (int c = tid; c < count; c += THREADS) {
      const uint64_t mine = candidates[c];
      int rank = 0;
      for (int j = 0; j < count && rank < top; ++j) rank += candidates[j] > mine ? 1 : 0;
      if (rank < top) write(rank, mine);
    }
  };
  collect(bound);
  __syncthreads();
  if (found <= kCandidates) {
    rank_candidates((int)found);
    return;
  }
  // Many elements reach the bound: usually equal ones (a row of -inf with few exceptions). Those
  // above it first, then the equal ones of lowest index, found from the front.
  __syncthreads();
  if (tid == 0) found = 0;
  __syncthreads();
  if (bound != 0xffffffffu) collect(bound + 1);
  __syncthreads();
  const int above = (int)found;
  if (above <= kCandidates) {
    rank_candidates(above);
    int taken = above;
    for (int j0 = 0; j0 < row.vocab && taken < top; j0 += THREADS) {
      const int j = j0 + tid;
      const bool equal = j < row.vocab && ordered((float)row.x[j]) == bound;
      const uint32_t votes = __ballot_sync(0xffffffffu, equal);
      __syncthreads();
      if (lane == 0) slot_max[warp] = __popc(votes);
      __syncthreads();
      int before = taken, total = 0;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += slot_max[w];
        total += slot_max[w];
      }
      before += __popc(votes & ((1u << lane) - 1u));
      if (equal && before < top)
        write(before, ((uint64_t)bound << 32) | (uint32_t)~j);
      taken += total;
    }
    return;
  }
  // More than kCandidates above the bound (a row that climbs from slot to slot): one maximum
  // after the other.
  uint64_t last = ~0ull;
  for (int k = 0; k < top; ++k) {
    uint64_t best = 0;
    for (int j = tid; j < row.vocab; j += THREADS) {
      const uint64_t candidate = ((uint64_t)ordered((float)row.x[j]) << 32) | (uint32_t)~j;
      if ((k == 0 || candidate < last) && candidate > best) best = candidate;
    }
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, best, w);
      best = other > best ? other : best;
    }
    __syncthreads();
    if (lane == 0) candidates[warp] = best;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) best = candidates[w] > best ? candidates[w] : best;
    if (tid == 0) write(k, best);
    last = best;
  }
}

template <class T>
cudaError_t launch(const void* logits, int64_t rows, int64_t vocab, int64_t pitch,
                   const int64_t* tokens, int64_t given, int64_t top, float* logprobs,
                   float* entropy, float* top_logprobs, int64_t* top_tokens,
                   cudaStream_t stream) {
  const dim3 grid((unsigned)rows);
  const T* x = static_cast<const T*>(logits);
  if (rows >= 2 * ppyb200_sm_count())
    return ppyb200::launch_pdl(token_logprobs_kernel<T, 256>, grid, dim3(256), 0, stream, x,
                               vocab, pitch, tokens, (int)given, (int)top, logprobs, entropy,
                               top_logprobs, top_tokens);
  return ppyb200::launch_pdl(token_logprobs_kernel<T, 1024>, grid, dim3(1024), 0, stream, x, vocab,
                             pitch, tokens, (int)given, (int)top, logprobs, entropy, top_logprobs,
                             top_tokens);
}

}  // namespace

extern "C" int32_t ppyb200_token_logprobs(const void* logits, int64_t dtype, int64_t rows,
                                          int64_t vocab, int64_t pitch, const int64_t* tokens,
                                          int64_t given, int64_t top, float* logprobs,
                                          float* entropy, float* top_logprobs,
                                          int64_t* top_tokens) {
  if (rows < 0 || rows > INT32_MAX || vocab <= 0 || vocab > (1 << 30) || pitch < vocab ||
      given < 0 || given > (1 << 20) || top < 0 || top > PPYB200_TOP_LIMIT || top > vocab ||
      dtype < PPYB200_F32 || dtype > PPYB200_F16) {
    ppyb200_set_error("ppyb200_token_logprobs: f32, bf16 or f16 rows of 1 to 2^30 logits, a pitch "
                      "of at least vocab, and top up to 64 and vocab required");
    return PPYB200_RAISED;
  }
  const int64_t size = dtype == PPYB200_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size != 0) {
    ppyb200_set_error("ppyb200_token_logprobs: logits aligned to their type required");
    return PPYB200_RAISED;
  }
  if (rows == 0) return PPYB200_OK;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(ppyb200_stream());
  cudaError_t e;
  if (dtype == PPYB200_F32)
    e = launch<float>(logits, rows, vocab, pitch, tokens, given, top, logprobs, entropy,
                      top_logprobs, top_tokens, stream);
  else if (dtype == PPYB200_BF16)
    e = launch<__nv_bfloat16>(logits, rows, vocab, pitch, tokens, given, top, logprobs, entropy,
                              top_logprobs, top_tokens, stream);
  else
    e = launch<__half>(logits, rows, vocab, pitch, tokens, given, top, logprobs, entropy,
                       top_logprobs, top_tokens, stream);
  if (e != cudaSuccess) return ppyb200_check((int32_t)e, "ppyb200_token_logprobs");
  ppyb200_count_launches(1);
  return PPYB200_OK;
}
