// Device helpers of the attention kernels.
#pragma once

#include "mma_device.cuh"

namespace b200q {
namespace {

// Four 8 x 8 matrices of 16-bit values from shared memory; lane l gives the address of row l % 8 of matrix l / 8.  A lane gets
// two neighbours of row lane / 4, or, transposed, of column lane / 4.
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// The 8 x 8 matrix of 16-bit values that the lanes hold (two neighbours of row lane / 4 each), transposed.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Two fp32 values as 16-bit ones, `lo` in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Eight 16-bit values on a 16-byte boundary, as fp32.
template <typename T>
__device__ __forceinline__ void unpack8(const T* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(e[i]);
}

// 2^x to two units in the last place, 0 for -inf; results below the smallest normal number are flushed to zero.
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two fp32 values in one 64-bit register pair, for the instructions that work on both.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 1 / sum of weights; 0 where there are none (a row that sees no key, or whose scores are all -inf, gives zeros).
__device__ __forceinline__ float inverse(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }

// 2^x of two values without the exponential unit: x = n + f with n = round(x) by adding 1.5 2^23, then 2^f on [-1/2, 1/2] by a
// polynomial of degree 4 with constant term 1 (coefficients fitted for the least largest relative error, 2.9e-6 = 2^-18.4
// in fp32), times 2^n.  x <= 127.  Below -127 (-inf too) n = -127, whose power comes out as 0; NaN stays NaN.
__device__ __forceinline__ float2 exp2_poly(uint64_t x) {
  constexpr float kShift = 12582912.f;
  const float2 v = unpair(x);
  x = pair(max_nan(v.x, -127.f), max_nan(v.y, -127.f));
  const uint64_t n = add2(x, pair(kShift, kShift));
  const uint64_t f = fma2(add2(n, pair(-kShift, -kShift)), pair(-1.f, -1.f), x);
  uint64_t y = fma2(f, pair(0.009582852944731712f, 0.009582852944731712f), pair(0.055906426161527634f, 0.055906426161527634f));
  y = fma2(y, f, pair(0.24024099111557007f, 0.24024099111557007f));
  y = fma2(y, f, pair(0.6931241750717163f, 0.6931241750717163f));
  y = fma2(y, f, pair(1.f, 1.f));
  const float2 m = unpair(n);
  return unpair(mul2(y, pair(__uint_as_float((__float_as_uint(m.x) << 23) + 0x3f800000u),
                             __uint_as_float((__float_as_uint(m.y) << 23) + 0x3f800000u))));
}

}  // namespace
}  // namespace b200q
