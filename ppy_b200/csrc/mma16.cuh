// Warp-level building blocks of the decoding kernels: 16-bit matrix products on register
// fragments (mma.sync), fragment loads from shared memory (ldmatrix) and asynchronous 16-byte
// copies into it (cp.async). The decoding kernels read each cached key and value once for a
// few query rows, so they are bound by memory and not by the tensor pipe; fragments of 16 rows
// fit such few rows, where a tcgen05 tile has 128. Their products run at a small part of the tcgen05
// rate (about 170 TFLOP/s over the whole GPU), so kernels with many rows have no use for them.
//
// Fragments of mma.m16n8k16 (lane = 4 gid + tig):
//   A [16 x 16]: a0 (row gid, cols 2 tig, +1), a1 (row gid + 8), a2 (cols + 8), a3 (both)
//   B [16 x 8]:  b0 (rows 2 tig, +1, col gid), b1 (rows + 8)
//   C [16 x 8]:  c0, c1 (row gid, cols 2 tig, +1), c2, c3 (row gid + 8)
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace ppyb200 {
namespace mma16 {

template <class T>
struct Kind;  // conversions between a 16-bit type and f32, and its product instruction

template <>
struct Kind<__nv_bfloat16> {
  __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  __device__ __forceinline__ static float2 unpack(uint32_t v) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
  }
  __device__ __forceinline__ static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

template <>
struct Kind<__half> {
  __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  __device__ __forceinline__ static float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
  }
  __device__ __forceinline__ static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ uint32_t shared_address(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// Four 8 x 8 tiles of 16-bit elements; lane l gives the address of row l % 8 of tile l / 8.
__device__ __forceinline__ void load4(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(address)
               : "memory");
}
__device__ __forceinline__ void load4_transposed(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(address)
               : "memory");
}

// 16 bytes from global to shared memory, asynchronously; zeros instead of them unless `valid`
// (the source is not read then, but has to be a mapped address).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copies_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int PENDING>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// 2^x on the special-function unit (ex2.approx: relative error about 2^-22; 2^-inf = 0).
__device__ __forceinline__ float exp2_sfu(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two 16-bit values, zero in the place of one that is not finite (its exponent bits all ones).
template <class T>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {
  constexpr uint32_t kExponent = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  if ((w & kExponent) == kExponent) w &= 0xffff0000u;
  if (((w >> 16) & kExponent) == kExponent) w &= 0x0000ffffu;
  return w;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

}  // namespace mma16
}  // namespace ppyb200
