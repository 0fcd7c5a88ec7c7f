// The 8-bit paged KV cache: layout, scale rule and e4m3 conversions shared by its kernels.
//
//   codes  e4m3 [num_cache_layers][2 (K, V)][num_blocks][num_kv_heads][16][head_dim]
//   scales fp32 [num_cache_layers][2][num_blocks][num_kv_heads]
//
// The value a code stands for is code * scale of its (block, head). A (block, head) tile is
// contiguous (16 * head_dim bytes), so attention moves it with one bulk copy. The scale is the
// smallest power of two 2^e with amax <= 448 * 2^e: dividing by it is exact, and when a block that
// is being filled needs a larger one its old codes move by a power of two, which is exact except
// where they become e4m3 subnormals. A free (not power-of-two) scale would gain at most one bit at
// the bottom of e4m3's 17-bit range and would round every old code again at each growth.
#pragma once

#include "cdb_common.cuh"

namespace cdb {
namespace kv8 {

constexpr int kBlock = 16;
constexpr float kLog2e = 1.4426950408889634f;

// The attention kernels hold the weights of V in f16, as 2^(x + log2 s_v - M + kLift): M is a maximum that lags its
// logits by up to 8, so they reach 2^15, of f16's 65504. From 2^-21 of the largest weight on each is rounded by
// 2^-11 of itself; below, f16's steps stay 2^-24, so by 2^-32 of the largest one. Without the lift a key that
// takes the mass and whose value is near 0 pushes the others there: 2048 weights of 2^-20.7 of it were off by 1.5%.
constexpr float kLift = 7.f;
constexpr float kUnlift = 1.f / 128.f;  // 2^-kLift

// Smallest power of two s (>= 2^-126) with amax <= 448 s; 448 = 1.75 * 2^8.
__device__ __forceinline__ float block_scale(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  if (bits == 0u || e < -126) e = -126;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

__device__ __forceinline__ uint32_t cvt_e4m3x2_f16x2(uint32_t codes16) {
  uint32_t r;
  const uint16_t c = (uint16_t)codes16;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}

// Two floats to two codes (lo in the low byte), nearest even, saturating; NaN stays NaN.
__device__ __forceinline__ uint32_t cvt_f32x2_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ void unpack_f16x2(uint32_t w, float& lo, float& hi) {
  asm("{.reg .f16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
      : "=f"(lo), "=f"(hi)
      : "r"(w));
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// D += A B on f16 operands, fp32 accumulators (m16n8k16).
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

}  // namespace kv8
}  // namespace cdb
