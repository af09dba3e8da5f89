// The paged 4-bit KV cache: block layout and number format, shared by the kernels that write, read, attend to
// and move its pages.
//
// A page holds 64 tokens of every layer and KV head.  The block of one (layer, page, KV head) is one contiguous
// run of bytes, so one bulk copy brings a whole 64-token tile of keys, values and their scales:
//   key codes   [64][hd / 2]      channel 2j of a token is the low nibble of byte j, channel 2j + 1 the high one
//   value codes [64][hd / 2]
//   key scales  [64][hd / 32]     bfloat16
//   value scales[64][hd / 32]
// A value is (nibble - 8) * scale of its 32 neighbouring channels, nibble in 1..15.  scale = amax / 7 rounded to
// nearest even with 4 significant bits:
//   * the rounding is at most 1/16, so the largest value is at most 7 * 17/16 = 7.44 steps and still rounds to 7:
//     narrowing the scale never costs a value more than half a step;
//   * nibble (4 bits) x scale (4 bits) has at most 8 significant bits: every product is exact in bfloat16, so the
//     tensor cores read the dequantised values without another rounding.
// A group whose largest magnitude is 2^122 or more, or not finite, gets a NaN scale and decodes to NaN.
#pragma once

#include "common.cuh"

namespace jxb {

constexpr int kPage = 64;                        // tokens per page
constexpr uint32_t kKv4Overflow = 0x7C800000u;   // bits of 2^122
constexpr uint32_t kKv4BadScale = 0x7B80u;       // bfloat16 2^120: every scale of a finite group is below it

__host__ __device__ __forceinline__ int kv4_block_bytes(int hd) { return kPage * hd + kPage * (hd / 32) * 4; }
__host__ __device__ __forceinline__ int kv4_scale_offset(int hd, int which) {
  return kPage * hd + which * kPage * (hd / 32) * 2;
}

// Block of a (layer, page, head).  64-bit: a pool passes 2^31 bytes.
__device__ __forceinline__ unsigned char* kv4_block(const jx_kv4_cache& c, int layer, int page, int head) {
  return c.pages + (((long long)layer * c.num_pages + page) * c.num_kv_heads + head) * kv4_block_bytes(c.head_dim);
}

// The scale of a group from the bits of its largest magnitude (an integer maximum of the magnitudes' bits, which
// orders NaN above infinity above every finite value).
__device__ __forceinline__ float kv4_scale(uint32_t amax_bits) {
  if (amax_bits >= kKv4Overflow) return __uint_as_float(0x7FC00000u);
  uint32_t b = __float_as_uint(__fdiv_rn(__uint_as_float(amax_bits), 7.0f));
  b = (b + 0x7FFFFu + ((b >> 20) & 1u)) & ~0xFFFFFu;   // 23 - 3 mantissa bits dropped, to nearest even
  return __uint_as_float(b);
}

// Nibble of a value.  The division is correctly rounded and the 4-bit scale keeps every half step representable, so
// a quotient lands on a half step only where the exact one does: no double rounding.
__device__ __forceinline__ uint32_t kv4_nibble(float x, float s) {
  if (!(s > 0.f)) return 8u;                     // zero group, or NaN scale
  const float q = fminf(fmaxf(rintf(__fdiv_rn(x, s)), -7.f), 7.f);
  return (uint32_t)((int)q + 8);
}

// Pairs of bfloat16 from nibbles.
namespace kv4 {
__device__ __forceinline__ __nv_bfloat162 as_b2(uint32_t x) { return *reinterpret_cast<__nv_bfloat162*>(&x); }
__device__ __forceinline__ uint32_t as_u(__nv_bfloat162 x) { return *reinterpret_cast<uint32_t*>(&x); }
// bfloat16 pair 128 + u of the nibbles k and k + 4 of a word (or k of two merged words).
__device__ __forceinline__ uint32_t raw2(uint32_t w, int k) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000F000F, 0x43004300, 0xEA;" : "=r"(r) : "r"(w >> (4 * k)));
  return r;
}
// Code times scale in one fused multiply-add, exact: (128 + u) s - 136 s = (u - 8) s.  136 s is 17 times a 4-bit number, at
// most 255, times a power of two: a bfloat16.
__device__ __forceinline__ uint32_t minus136(uint32_t s2) { return as_u(__hmul2(as_b2(s2), as_b2(0xC308C308u))); }
__device__ __forceinline__ uint32_t scaled2(uint32_t w, int k, uint32_t s2, uint32_t c2) {
  return as_u(__hfma2(as_b2(raw2(w, k)), as_b2(s2), as_b2(c2)));
}
}  // namespace kv4

}  // namespace jxb
