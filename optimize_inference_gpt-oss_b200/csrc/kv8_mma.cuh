// Tensor-core pieces of the attention over the 8-bit cache: codes to fp16, fp32 to fp16 parts, and the
// warp-wide matrix instruction of the few-row kernel.
#pragma once

#include <cuda_fp16.h>

#include "kv8.cuh"

namespace gptoss {
namespace kv8 {

// A code c is stored as a signed byte.  u = c + 128 (the byte with its top bit flipped) put under the
// exponent byte 0x64 is the fp16 number 1024 + u, so c = that - 1152: three instructions for two
// codes and no conversion unit.
__device__ __forceinline__ uint32_t biased(uint32_t w) { return w ^ 0x80808080u; }
__device__ __forceinline__ uint32_t low_pair(uint32_t u) { return __byte_perm(u, 0x64646464u, 0x4140); }
__device__ __forceinline__ uint32_t high_pair(uint32_t u) { return __byte_perm(u, 0x64646464u, 0x4342); }
__device__ __forceinline__ uint32_t minus_1152(uint32_t x) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x64806480u));
  return r;
}
// (x - 1152) * mul with one rounding: mul a power of two, add = -1152 mul, both twice in a word.
__device__ __forceinline__ uint32_t scaled_pair(uint32_t x, uint32_t mul, uint32_t add) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(mul), "r"(add));
  return r;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// What the fp16 pair leaves of (lo, hi), as the next fp16 pair: together 22 bits of each.
__device__ __forceinline__ uint32_t pack_rest(uint32_t pair, float lo, float hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&pair));
  return pack_f16(lo - f.x, hi - f.y);
}

// c[16][8] += a[16][16] b[16][8], fp16 in, fp32 sums.  With g = lane / 4, t = lane % 4:
// a0 (g, 2t..), a1 (g + 8, 2t..), a2 (g, 2t + 8..), a3 (g + 8, 2t + 8..); b0 (2t.., g), b1 (2t + 8.., g);
// c0, c1 (g, 2t..), c2, c3 (g + 8, 2t..).
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// An 8x8 matrix of 16-bit values (lane: row g, columns 2t, 2t + 1) transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// Exponent field of a power-of-two scale; 0 for 0.
__device__ __forceinline__ int exponent_field(float s) { return (int)(__float_as_uint(s) >> 23) & 0xff; }
__device__ __forceinline__ float two_to(int e) { // e in [-126, 127]; below: 0
  return e < -126 ? 0.0f : __uint_as_float((uint32_t)(e + 127) << 23);
}

} // namespace kv8
} // namespace gptoss
