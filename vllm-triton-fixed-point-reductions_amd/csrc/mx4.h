// The 4-bit KV cache format (mx4), shared by its writer, its reader and the
// attention over it.
//
// A row (one token, one kv head, K or V) of D elements is D / 32 blocks of 32
// elements. A block has one scale byte b, standing for s = 2^(b - 127), and an
// element a 4-bit code: sign and magnitude 0 .5 1 1.5 2 3 4 6 (the E2M1
// numbers that gfx950's v_cvt_scalef32 instructions take). The code's value
// is its magnitude times s, which every 16-bit and 32-bit float type holds
// exactly over the scale bytes that the writer gives that type:
//   bf16 / f32: 2 .. 252 (6 s is at most 1.5 * 2^127), f16: 104 .. 140 (.5 s
//   is at least f16's smallest subnormal, 6 s at most 49152).
// A reader takes a byte above its type's largest as the largest, so no byte
// pattern reads as an infinity or NaN and a masked key's V times a weight of 0
// is 0 whatever the row holds.
//
// Bytes of a row: 8-element chunk c is the 4-byte unit (c % 4) * (D / 32) +
// c / 4, element i of it in bits 4 i .. 4 i + 3. The MFMA operand of a 32-wide
// step j gives lane group kg the elements 32 j + 8 kg .. + 7: with this order
// the units of group kg are D / 8 consecutive bytes, one vector load per lane
// and row, and unit j of them is of block j.
#pragma once

#include "fxp_device.h"

namespace fxpr {
namespace mx4 {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 32;  // elements per scale

// Scale bytes of a float type (Io tags: 0 f16, 1 bf16, 2 f32).
template <int DT> struct Range { static constexpr uint32_t lo = 2, hi = 252; };
template <> struct Range<0> { static constexpr uint32_t lo = 104, hi = 140; };

// Scale j of a row's packed scale bytes w (j % 4 within the word), as the
// fp32 power of two the conversions take (they read its exponent only).
template <int DT> __device__ __forceinline__ float scale_of(uint32_t w, int j) {
  const uint32_t b = (w >> (8 * j)) & 0xffu;
  return __uint_as_float((b < Range<DT>::hi ? b : Range<DT>::hi) << 23);
}

// The eight elements of a 4-byte unit, as 16-bit floats of type DT: exact.
template <int DT> __device__ __forceinline__ u32x4 unpack8(uint32_t codes, float scale) {
  static_assert(DT == 0 || DT == 1, "16-bit types");
  u32x4 r;
  if constexpr (DT == 1) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3));
  }
  return r;
}

// The scale byte of a block whose largest magnitude has the fp32 bits `amax`
// (inf included, NaN not): the power of two with amax / s in (3.5, 7], within
// the type's range. 7 is the midpoint of 6 and the next magnitude a longer
// code would have, so saturating there is off by no more than rounding is
// between 4 and 6; a smaller limit (6) would double the step of every element
// of a block with amax / s in (6, 7].
template <int DT> __device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  // the exponent goes up where the mantissa exceeds 1.75 (0x600000)
  const int b = int((amax + 0x1fffffu) >> 23) - 2;
  constexpr int lo = Range<DT>::lo, hi = Range<DT>::hi;
  return uint32_t(b < lo ? lo : (b > hi ? hi : b));
}

}  // namespace mx4
}  // namespace fxpr
