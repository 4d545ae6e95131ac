// The quantised KV cache's number format, shared by the store, the read-back
// and the decode attention.
//
// A vector of 64 channels is two blocks of 32. A block is one scale 2^e, held
// as the byte e + 127, and 32 elements of kBits: 4 bits (sign, 2 exponent, 1
// mantissa: 0 .5 1 1.5 2 3 4 6) or 8 bits (sign, 4 exponent, 3 mantissa, to
// 448), the microscaling types that gfx950 converts in hardware. e is the
// smallest integer with max|x| <= T 2^e, T = 7 (4 bits) or 464 (8 bits): the
// largest number that rounds to the type's largest, so the block's maximum is
// never cut by more than the rounding itself. Against T = 6 and T = 8 the 4-bit
// error on normal values is 11.2% against 11.6% and 11.5% (RMS). Scales are
// powers of two, so x 2^-e is exact and each element's rounding (to nearest,
// ties to even) is decided on the exact quotient.
//
// e is held to [-126, 125] (4 bits) or [-126, 119] (8 bits), so every value a
// block stands for is finite. A block with an infinity or a NaN gets byte 255 and
// codes 0 and stands for NaN (0 times the float that byte << 23 spells). Byte 0
// (a cleared cache) with codes 0 stands for zeros.
//
// Four scale bytes (k block 0, k block 1, v block 0, v block 1) lie together per
// position: one word serves a key's and a value's product.
#pragma once

#include "common.h"

namespace lm {

constexpr int kQuantBlock = 32;
constexpr uint32_t kScaleNaN = 255;

// Bytes of one vector of 64 codes.
template <int kBits>
constexpr int code_bytes() { return 8 * kBits; }

// Scale byte `i` of a position's word as a float: 0 for byte 0, +inf for 255.
__device__ __forceinline__ float quant_scale(uint32_t word, int i) {
  return __uint_as_float(((word >> (8 * i)) & 0xffu) << 23);
}

// Eight codes: one 32-bit word (4 bits) or two (8 bits).
template <int kBits>
struct Codes8 {
  uint32_t w[kBits / 4];
};

// The unsigned maximum over aligned groups of four lanes (quad_perm xor 1, xor 2).
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));
}

// Quantises a block held by four consecutive lanes, eight channels each. Every
// lane of the four must call it together. Magnitudes are compared as their bit
// patterns, which order as the numbers do, infinities and NaN above them all.
template <int kBits>
__device__ __forceinline__ Codes8<kBits> quantise8(const float *x, uint32_t &scale_byte) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(x[i]) & 0x7fffffffu);
  a = quad_max(a);
  // T = 1.75 * 2^2 or 1.8125 * 2^8: a mantissa above T's carries into the exponent.
  constexpr uint32_t kCarry = kBits == 4 ? 0x1fffffu : 0x17ffffu;
  constexpr int kTop = kBits == 4 ? 2 : 8, kMost = kBits == 4 ? 252 : 246;
  const int byte = min(max((int)((a + kCarry) >> 23) - kTop, 1), kMost);
  const float s = __uint_as_float((uint32_t)byte << 23);
  Codes8<kBits> c;
  if constexpr (kBits == 4) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[0], x[1], s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[2], x[3], s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[4], x[5], s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[6], x[7], s, 3);
    c.w[0] = r;
  } else {
    // The 8-bit conversion gives NaN above 464 where the 4-bit one holds to
    // its largest, so a block at the clamped exponent is held here.
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    const float most = 448.f * s;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = fminf(fmaxf(x[i], -most), most);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      s16x2 r = (s16x2){0, 0};
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, y[4 * j], y[4 * j + 1], s, false);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, y[4 * j + 2], y[4 * j + 3], s, true);
      c.w[j] = __builtin_bit_cast(uint32_t, r);
    }
  }
  const bool bad = a >= 0x7f800000u;
#pragma unroll
  for (int j = 0; j < kBits / 4; ++j) c.w[j] = bad ? 0u : c.w[j];
  scale_byte = bad ? kScaleNaN : (uint32_t)byte;
  return c;
}

// Eight codes as bf16 pairs without their scale, times `unit`, a power of two: exact
// (codes have up to 2 or 4 significand bits).
template <int kBits>
__device__ __forceinline__ u32x4 codes_to_bf16(const uint32_t *w, float unit = 1.f) {
  u32x4 o;
  if constexpr (kBits == 4) {
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], unit, 0));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], unit, 1));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], unit, 2));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], unit, 3));
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      o[2 * j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[j], unit, false));
      o[2 * j + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[j], unit, true));
    }
  }
  return o;
}

}  // namespace lm
