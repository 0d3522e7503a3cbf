// Log probabilities of given tokens, the entropy, and the likeliest alternatives of rows of
// logits, each row read from memory once.
//
//   m = max x,  Z = sum e^{x - m},  log p_i = x_i - m - log Z
//   H = - sum p log p = log Z - (sum (x - m) e^{x - m}) / Z
//
// Z and the sum T of (x - m) e^{x - m} run along the row with a reference m: when it grows by D, Z
// becomes e^{-D} Z and T becomes e^{-D} (T - D Z). The reference follows the maximum only when
// that is more than kSlack above it (a thread's maximum moves at every other vector, and some
// thread's of a warp at nearly each). One exponential an element, the other arithmetic on pairs.
//
// The alternatives need no second pass over the row. The k-th largest of the threads' maxima is a
// lower bound for the k-th largest logit, and only the threads whose own maximum reaches it (about
// k of 256) hold candidates: their elements, just read, come from L2 again. The few candidates are
// ranked by counting. Few rows are split over a cluster of CTAs each, whose first joins the sums
// and the alternatives of the parts.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <cooperative_groups.h>

#include "../../include/ppyb200.h"
#include "mma16.cuh"
#include "ppyb200_device.cuh"

namespace {

using ppyb200::mma16::exp2_sfu;
using ppyb200::mma16::kLn2;
using ppyb200::mma16::kLog2e;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kTop = PPYB200_TOP_LIMIT;
constexpr int kCandidates = 1024;
constexpr int kMostRanks = 8;    // CTAs of a cluster
constexpr float kSlack = 8.f;    // e^8 times as many terms as there are stay far from f32's limit
constexpr float kLeast = -200.f;  // e^kLeast = 0 in f32: stands for -inf where 0 times it is 0

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

// Sixteen bytes of logits as pairs of f32.
template <class T>
struct Vector {
  static constexpr int kCount = 8, kPairs = 4;
  __device__ __forceinline__ static void unpack(const uint4& x, float (&v)[8]) {
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
struct Vector<float> {
  static constexpr int kCount = 4, kPairs = 2;
  __device__ __forceinline__ static void unpack(const uint4& x, float (&v)[4]) {
    v[0] = __uint_as_float(x.x);
    v[1] = __uint_as_float(x.y);
    v[2] = __uint_as_float(x.z);
    v[3] = __uint_as_float(x.w);
  }
};

using ppyb200::add2;
using ppyb200::f2;
using ppyb200::fma2;
using ppyb200::mul2;
using ppyb200::unf2;

// Reference, maximum, Z and T of a part of a row; Z and T as two sums each until they are joined.
struct Sums {
  float m = -INFINITY, most = -INFINITY;
  uint64_t z = 0, t = 0;

  __device__ __forceinline__ void raise_to(float top) {
    const float drop = fmaxf(m - top, kLeast);
    const float f = exp2_sfu(drop * kLog2e);
    t = mul2(f2(f, f), fma2(f2(drop, drop), z, t));
    z = mul2(f2(f, f), z);
    m = top;
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&v)[N]) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, v[i]);
    most = fmaxf(most, top);
    if (top > m + kSlack) raise_to(top);  // -inf + kSlack: the first finite one
    const float u = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      // the difference first: exact near the maximum, however large the logits are
      const uint64_t d = add2(f2(v[i], N == 1 ? -INFINITY : v[(i + 1) % N]), f2(-u, -u));
      float y0, y1, d0, d1;
      unf2(mul2(d, f2(kLog2e, kLog2e)), y0, y1);
      unf2(d, d0, d1);
      const uint64_t e = f2(exp2_sfu(y0), exp2_sfu(y1));
      z = add2(z, e);
      t = fma2(f2(fmaxf(d0, kLeast), fmaxf(d1, kLeast)), e, t);
    }
  }
  __device__ __forceinline__ void join(float om, uint64_t oz, uint64_t ot) {
    Sums o;
    o.m = om;
    o.z = oz;
    o.t = ot;
    const float top = fmaxf(m, om);
    if (top > m) raise_to(top);
    if (top > om) o.raise_to(top);
    z = add2(z, o.z);
    t = add2(t, o.t);
  }
  __device__ __forceinline__ float total_z() const {
    float a, b;
    unf2(z, a, b);
    return a + b;
  }
  __device__ __forceinline__ float total_t() const {
    float a, b;
    unf2(t, a, b);
    return a + b;
  }
};

// The elements of a part of a row as its threads walk them: single ones up to the first 16-byte
// boundary, vectors, single ones to the end.
template <class T>
struct Row {
  const T* x;
  int head, vectors, tail, count;
  static constexpr int kCount = Vector<T>::kCount;
  __device__ __forceinline__ Row(const T* row, int n) : x(row), count(n) {
    const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15u) / (int)sizeof(T);
    head = min(off == 0 ? 0 : kCount - off, count);
    vectors = (count - head) / kCount;
    tail = count - head - vectors * kCount;
  }
  __device__ __forceinline__ uint4 raw(int i) const {
    return __ldg(reinterpret_cast<const uint4*>(x + head + i * kCount));
  }
  __device__ __forceinline__ int tail_at() const { return count - tail; }
  __device__ __forceinline__ bool has(int thread) const {
    return thread < head || thread < vectors || thread < tail;
  }
};

struct Shared {
  Sums parts[kWarps];
  Sums whole;                  // of this CTA's part, read by the cluster's first
  uint64_t candidates[kCandidates];  // (logit as a number in its order, ~index)
  uint64_t best[kTop];               // the part's alternatives, the largest first
  uint32_t found, listed;
  uint16_t list[kThreads];   // threads with candidates
  uint32_t votes[kWarps];
};

// Ranks the first `count` candidates by counting: the `top` largest into best, from place `at`.
__device__ __forceinline__ void rank_candidates(Shared& s, int count, int top) {
#pragma unroll 1
  for (int c = threadIdx.x; c < count; c += kThreads) {
    const uint64_t mine = s.candidates[c];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < count; ++j) rank += s.candidates[j] > mine ? 1 : 0;
    if (rank < top) s.best[rank] = mine;
  }
}

// The part's `top` largest logits (top <= count) into s.best, by every thread of the CTA. `odd`:
// a NaN or +inf among them, so that the threads' maxima are not their largest elements.
template <class T>
__device__ __forceinline__ void find_best(Shared& s, const Row<T>& row, int index0, int top,
                                          float max, bool odd) {
  constexpr int kCount = Vector<T>::kCount;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t key = row.has(tid) ? ordered(max) : 0u;  // 0: no elements
  if (odd) {
    if (tid < row.head) key = ::max(key, ordered((float)row.x[tid]));
    if (tid < row.tail) key = ::max(key, ordered((float)row.x[row.tail_at() + tid]));
#pragma unroll 1
    for (int i = tid; i < row.vectors; i += kThreads) {
      float v[kCount];
      Vector<T>::unpack(row.raw(i), v);
#pragma unroll
      for (int e = 0; e < kCount; ++e) key = ::max(key, ordered(v[e]));
    }
  }
  if (tid == 0) s.found = s.listed = 0;
  // The bound, bit by bit: the largest number of 20 leading bits (all 16 of 16-bit logits) that
  // `top` threads reach; the bits left out only let a few more candidates in. Fewer than `top`
  // threads with elements leave 0.
  uint32_t bound = 0;
#pragma unroll 1
  for (uint32_t bit = 1u << 31; bit >= 1u << 12; bit >>= 1)
    if (__syncthreads_count(key >= (bound | bit)) >= top) bound |= bit;

  // keys of at least `least` join the candidates: all vectors of the threads that have any, dealt
  // to all threads
  auto collect = [&](uint32_t least) {
    // what is below it as a float, most elements, needs no more than a comparison
    const float floor =
        least > 0x007fffffu && least <= 0xff800000u ? disordered(least) : -INFINITY;
    if (key >= least && row.has(tid)) s.list[atomicAdd(&s.listed, 1u)] = (uint16_t)tid;
    __syncthreads();
    auto offer = [&](float value, int index) {
      if (value < floor) return;
      const uint32_t k = ordered(value);
      if (k < least) return;
      const uint32_t place = atomicAdd(&s.found, 1u);
      if (place < kCandidates)
        s.candidates[place] = ((uint64_t)k << 32) | (uint32_t)~(index0 + index);
    };
    const int listed = (int)s.listed, each = (row.vectors + kThreads - 1) / kThreads;
    if (tid < listed) {
      const int thread = s.list[tid];
      if (thread < row.head) offer((float)row.x[thread], thread);
      if (thread < row.tail) offer((float)row.x[row.tail_at() + thread], row.tail_at() + thread);
    }
#pragma unroll 1
    for (int item = tid; item < listed * each; item += kThreads) {
      const int l = item / each, i = s.list[l] + (item - l * each) * kThreads;
      if (i >= row.vectors) continue;
      float v[kCount];
      Vector<T>::unpack(row.raw(i), v);
#pragma unroll
      for (int e = 0; e < kCount; ++e) offer(v[e], row.head + i * kCount + e);
    }
    __syncthreads();
  };
  collect(bound);
  if (s.found <= kCandidates) {
    rank_candidates(s, (int)s.found, top);
    return;
  }
  // Many elements reach the bound: usually equal ones (a row of -inf with few exceptions). The
  // bound in full, those above it first, then the equal ones of lowest index, from the front.
#pragma unroll 1
  for (uint32_t bit = 1u << 11; bit != 0; bit >>= 1)
    if (__syncthreads_count(key >= (bound | bit)) >= top) bound |= bit;
  if (tid == 0) s.found = s.listed = 0;
  __syncthreads();
  if (bound != 0xffffffffu) collect(bound + 1);
  const int above = (int)s.found;
  if (above <= kCandidates) {
    rank_candidates(s, above, top);
    int taken = above;
#pragma unroll 1
    for (int j0 = 0; j0 < row.count && taken < top; j0 += kThreads) {
      const int j = j0 + tid;
      const bool equal = j < row.count && ordered((float)row.x[j]) == bound;
      const uint32_t votes = __ballot_sync(0xffffffffu, equal);
      __syncthreads();
      if (lane == 0) s.votes[warp] = __popc(votes);
      __syncthreads();
      int before = taken;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += s.votes[w];
        taken += s.votes[w];
      }
      before += __popc(votes & ((1u << lane) - 1u));
      if (equal && before < top)
        s.best[before] = ((uint64_t)bound << 32) | (uint32_t)~(index0 + j);
    }
    return;
  }
  // More than kCandidates above the bound (elements that gather in few threads): one maximum
  // after the other.
  uint64_t last = ~0ull;
#pragma unroll 1
  for (int k = 0; k < top; ++k) {
    uint64_t most = 0;
#pragma unroll 1
    for (int j = tid; j < row.count; j += kThreads) {
      const uint64_t one =
          ((uint64_t)ordered((float)row.x[j]) << 32) | (uint32_t)~(index0 + j);
      if ((k == 0 || one < last) && one > most) most = one;
    }
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, most, w);
      most = other > most ? other : most;
    }
    __syncthreads();
    if (lane == 0) s.candidates[warp] = most;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) most = s.candidates[w] > most ? s.candidates[w] : most;
    if (tid == 0) s.best[k] = most;
    last = most;
  }
}

// Eight CTAs an SM: a row's end (joins, the bound, the candidates) loads next to nothing, and the
// other CTAs' rows keep the memory busy meanwhile (47 registers and five CTAs: 16384 rows of
// GPT-2 logits in f32 577 us, 32 registers 546, 6.0 TB/s of one read). Prefetching the next vectors
// into L2 made that 589. Rows of bf16 take as many exponentials for half the bytes: 1500 of
// 32011, 96 MB, 40 us, 2.4 TB/s.
template <class T>
__global__ void __launch_bounds__(kThreads, 8)
token_logprobs_kernel(const T* __restrict__ logits, int vocab, int64_t pitch,
                      const int64_t* __restrict__ tokens, int given, int top,
                      float* __restrict__ logprobs, float* __restrict__ entropy,
                      float* __restrict__ top_logprobs, int64_t* __restrict__ top_tokens) {
  namespace cg = cooperative_groups;
  constexpr int kCount = Vector<T>::kCount, kUnroll = 4;
  __shared__ Shared s;
  ppyb200::pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x / ranks;
  const T* whole_row = logits + r * pitch;
  // a part of the row; whole lines, so that parts start on boundaries where rows do
  const int part = ranks == 1 ? vocab : ((vocab + ranks - 1) / ranks + 63) / 64 * 64;
  const int index0 = min(rank * part, vocab);
  const Row<T> row(whole_row + index0, min(part, vocab - index0));

  Sums sums;
  if (tid < row.head) {
    const float v[1] = {(float)row.x[tid]};
    sums.add(v);
  }
  if (tid < row.tail) {
    const float v[1] = {(float)row.x[row.tail_at() + tid]};
    sums.add(v);
  }
  int i = tid;
#pragma unroll 1
  for (; i + (kUnroll - 1) * kThreads < row.vectors; i += kUnroll * kThreads) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) raw[u] = row.raw(i + u * kThreads);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float v[kCount];
      Vector<T>::unpack(raw[u], v);
      sums.add(v);
    }
  }
#pragma unroll 1
  for (; i < row.vectors; i += kThreads) {
    float v[kCount];
    Vector<T>::unpack(row.raw(i), v);
    sums.add(v);
  }

  const int local_top = min(top, row.count);
  if (local_top > 0) {
    const float z = sums.total_z();
    const bool odd = __syncthreads_or(z != z) != 0;
    find_best(s, row, index0, local_top, sums.most, odd);
  }
#pragma unroll 1
  for (int w = 16; w > 0; w >>= 1)
    sums.join(__shfl_xor_sync(0xffffffffu, sums.m, w), __shfl_xor_sync(0xffffffffu, sums.z, w),
              __shfl_xor_sync(0xffffffffu, sums.t, w));
  if (lane == 0) s.parts[warp] = sums;
  __syncthreads();
  sums = s.parts[0];
#pragma unroll 1
  for (int w = 1; w < kWarps; ++w) sums.join(s.parts[w].m, s.parts[w].z, s.parts[w].t);
  if (ranks > 1) {
    if (tid == 0) s.whole = sums;
    cluster.sync();
    if (rank == 0) {
#pragma unroll 1
      for (int q = 1; q < ranks; ++q) {
        const Sums* other = cluster.map_shared_rank(&s.whole, q);
        sums.join(other->m, other->z, other->t);
      }
      // the parts' alternatives side by side, then ranked together
      int count = 0;
#pragma unroll 1
      for (int q = 0; q < ranks && top > 0; ++q) {
        const int n = min(top, max(0, min(part, vocab - q * part)));
        const uint64_t* other = cluster.map_shared_rank(s.best, q);
        for (int c = tid; c < n; c += kThreads) s.candidates[count + c] = other[c];
        count += n;
      }
      __syncthreads();
      rank_candidates(s, count, top);
      __syncthreads();
    }
    cluster.sync();  // the others' shared memory has been read
    if (rank != 0) return;
  }
  const float z = sums.total_z(), log_z = log2f(z) * kLn2;
  if (tid == 0 && entropy != nullptr) entropy[r] = log_z - sums.total_t() / z;
#pragma unroll 1
  for (int c = tid; c < given; c += kThreads) {
    const int64_t token = tokens[r * given + c];
    logprobs[r * given + c] = token >= 0 && token < vocab
                                  ? ((float)whole_row[token] - sums.m) - log_z
                                  : __uint_as_float(0x7fc00000u);
  }
  if (tid < top) {
    const uint64_t one = s.best[tid];
    top_logprobs[r * top + tid] = (disordered((uint32_t)(one >> 32)) - sums.m) - log_z;
    top_tokens[r * top + tid] = (int64_t)(uint32_t)~(uint32_t)one;
  }
}

template <class T>
cudaError_t launch(const void* logits, int64_t rows, int64_t vocab, int64_t pitch,
                   const int64_t* tokens, int64_t given, int64_t top, float* logprobs,
                   float* entropy, float* top_logprobs, int64_t* top_tokens,
                   cudaStream_t stream) {
  // few rows: a cluster each, while the SMs have room and a part stays above 4096 logits
  const int64_t room = 2 * (int64_t)ppyb200_sm_count();
  int ranks = 1;
  while (ranks < kMostRanks && rows * ranks * 2 <= room && vocab >= ranks * 2 * 4096) ranks *= 2;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(rows * ranks));
  config.blockDim = dim3(kThreads);
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = (unsigned)ranks;
  attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attributes;
  config.numAttrs = ppyb200_pdl() ? 2 : 1;
  return cudaLaunchKernelEx(&config, token_logprobs_kernel<T>, static_cast<const T*>(logits),
                            (int)vocab, pitch, tokens, (int)given, (int)top, logprobs, entropy,
                            top_logprobs, top_tokens);
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
