// The 4-bit key/value cache: where a code and a scale lie, and how 32 elements become one.
//
// A layer's cache is [pages][kv heads][page_size / 16][18 D] bytes: per page and kv head, units of 16 tokens of
//   K codes (8 D bytes) | V codes (8 D) | K scales (16 x D / 32 bfloat16) | V scales (16 x D / 32 bfloat16).
// 32 neighbouring elements of a head's row share a scale: s = bfloat16(max |x| / 7), an element is c s with c = x / s rounded to
// the nearest of -7 .. 7 (halves away from zero), kept as c + 8.  A scale below 2^-126 becomes 0 (the whole group reads back as
// zero); a group that holds an infinity or NaN gets the scale NaN and reads back as NaN.
//
// The order of the codes is that of the operands of mma.m16n8k16, so that the attention's lanes read theirs as whole vectors:
//   K, token j, element 32 G + 8 t + i: nibble i of the 32-bit word at j D/2 + t D/8 + 4 G          (lane (g, t): rows g, g + 8)
//   V, token j, element 32 G + 4 g + i: nibble i of the 16-bit word at ((j/8) 32 + 4 g + (j/2) % 4) D/8 + (j % 2) D/16 + 2 G
// For K a lane's words of all groups of a token lie side by side; for V the words of two neighbouring tokens do, a column pair
// of the operand.  Eight lanes hold a group of a row either way, four elements each, which is how rows are written and read.
#pragma once
#include "common.cuh"

namespace ilb {

constexpr int kKv4Unit = 16;               // tokens of a unit
constexpr int kKv4Group = 32;              // elements that share a scale

__host__ __device__ constexpr int kv4_unit_bytes(int d) { return 18 * d; }

// Byte offsets inside a unit: the 16 bits of elements 32 G + 4 l .. + 3 of token j, and its scale.
__device__ __forceinline__ int kv4_key_at(int d, int j, int G, int l) { return j * (d / 2) + (l >> 1) * (d / 8) + 4 * G + 2 * (l & 1); }
__device__ __forceinline__ int kv4_value_at(int d, int j, int G, int l) {
  return 8 * d + ((j >> 3) * 32 + 4 * l + ((j >> 1) & 3)) * (d / 8) + (j & 1) * (d / 16) + 2 * G;
}
__device__ __forceinline__ int kv4_scale_at(int d, bool value, int j, int G) { return (value ? 17 : 16) * d + (j * (d / 32) + G) * 2; }

// (x & mask) | bits, in one instruction (the compiler makes two of the expression).
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
  return y;
}

// Codes of a lane's four elements (16 bits, the first lowest) and the group's scale, from eight neighbouring lanes that hold a group.
// BY_PRODUCT: x times the reciprocal of s, raised by 2^-20, in the quotient's place, exact where the elements are bfloat16 numbers:
// x / s is then a half exactly or at least 2^-12 (relatively) away from one, the product is within 2^-22 of x / s (1 + 2^-20) and so lands
// on the side that the quotient rounds to.  A quotient of 32-bit elements may be nearer to a half than a reciprocal can tell and is
// taken in full where the definition counts to the last bit.
template <bool BY_PRODUCT>
__device__ __forceinline__ uint32_t kv4_quantise(const float (&x)[4], __nv_bfloat16& scale) {
  uint32_t top = max(max(__float_as_uint(x[0]) & 0x7fffffffu, __float_as_uint(x[1]) & 0x7fffffffu),      // (ordered like the numbers, NaN above infinity)
                     max(__float_as_uint(x[2]) & 0x7fffffffu, __float_as_uint(x[3]) & 0x7fffffffu));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 4));
  scale = __float2bfloat16_rn(__fmul_rn(__uint_as_float(top), 1.0f / 7.0f));
  const float s = __bfloat162float(scale);
  const bool none = top >= 0x7f800000u, flat = s < 1.17549435e-38f;
  scale = none ? __ushort_as_bfloat16(0x7fc0) : flat ? __ushort_as_bfloat16(0) : scale;
  uint32_t codes;
  if (BY_PRODUCT) {
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    inv = __fmul_rn(inv, 1.0f + 0x1p-20f);
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = __float_as_uint(__fmaf_rn(x[i], inv, 12582920.0f));      // 1.5 2^23 + 8: the sum's last bits are the rounded product plus 8
    codes = and_or(c[3] << 12, 0xf000u, and_or(c[2] << 8, 0xf00u, and_or(c[1] << 4, 0xf0u, c[0] & 15u)));
  } else {
    codes = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = __fdiv_rn(x[i], s), a = fabsf(y), w = truncf(a);
      const int c = min((int)w + (a - w >= 0.5f ? 1 : 0), 7);
      codes |= (uint32_t)(y < 0.f ? 8 - c : 8 + c) << (4 * i);
    }
  }
  return none || flat ? 0x8888u : codes;
}

// The same of eight bfloat16 elements a lane (by the product), from four neighbouring lanes that hold a group.
__device__ __forceinline__ uint32_t kv4_quantise8(const float (&x)[8], __nv_bfloat16& scale) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  scale = __float2bfloat16_rn(__fmul_rn(__uint_as_float(top), 1.0f / 7.0f));
  const float s = __bfloat162float(scale);
  const bool none = top >= 0x7f800000u, flat = s < 1.17549435e-38f;
  scale = none ? __ushort_as_bfloat16(0x7fc0) : flat ? __ushort_as_bfloat16(0) : scale;
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  inv = __fmul_rn(inv, 1.0f + 0x1p-20f);
  uint32_t codes = 0;
#pragma unroll
  for (int i = 7; i >= 0; --i) codes = codes << 4 | (__float_as_uint(__fmaf_rn(x[i], inv, 12582920.0f)) & 15u);
  return none || flat ? 0x88888888u : codes;
}

}  // namespace ilb
