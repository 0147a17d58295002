// 4 bits to a value: rows of a paged cache as the kernels that fill it and read it back take them.
#pragma once
#include "fba_types.h"

namespace fba {

// Exponents of a group of 32, so that every value that is held is a normal number of the type.
template <typename T>
inline constexpr int kScaleLimit = 125;
template <>
inline constexpr int kScaleLimit<_Float16> = 13;

// The largest of the four lanes that have a group, from a multiple of four on.
FBA_DEVICE uint32_t of_group(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, false));    // the lane beside, in the pair
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, false));  // the pair beside, in the four
}
FBA_DEVICE uint32_t bits_of(float x) { return __builtin_bit_cast(uint32_t, x); }

// Eight columns of a lane -> their codes; four lanes have a group.  The scale is the largest value's exponent less two, and one more from 1.75 of its binade on, so that nothing is
// beyond 7 times the scale and the largest code, 6, is off by less than a seventh; rounding is to the nearest, ties to the even code (the conversion's own).
//
// `off`: how far the values may be from what is meant.  Rounding is monotone, so a code is sure if off less and off more give the same one.
template <typename T>
struct To4Bits {
  uint32_t codes, scale;
  bool sure;  // whether no code of this lane, and not the group's scale, could be another (a value around zero may be taken for unsure)
  FBA_DEVICE static uint32_t round(const float (&x)[8], float by, float off) {
    uint32_t codes = 0;
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0] + off, x[1] + off, by, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2] + off, x[3] + off, by, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4] + off, x[5] + off, by, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6] + off, x[7] + off, by, 3);
  }
  template <bool kOff>
  FBA_DEVICE void hold(const float (&x)[8], float off) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, bits_of(x[i]) & 0x7fffffffu);
    most = of_group(most);
    const int e = min(max((int)((most + 0x200000u) >> 23) - 2, 127 - kScaleLimit<T>), 127 + kScaleLimit<T>);
    scale = most >= 0x7f800000u ? 255u : (uint32_t)e;
    const float by = __builtin_bit_cast(float, (uint32_t)e << 23);
    if constexpr (kOff) {
      codes = round(x, by, -off);
      const float largest = __builtin_bit_cast(float, most);
      sure = codes == round(x, by, off) && largest < 7.f * by - off && (largest > 3.5f * by + off || e == 127 - kScaleLimit<T>);
    } else {
      codes = round(x, by, 0.f);
    }
  }
};

template <typename T>
struct FromFp4;
template <>
struct FromFp4<__bf16> {
  template <int kByte>
  FBA_DEVICE static bf16x2 pair(uint32_t codes, float scale) { return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, kByte); }
};
template <>
struct FromFp4<_Float16> {
  template <int kByte>
  FBA_DEVICE static f16x2 pair(uint32_t codes, float scale) { return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, kByte); }
};
// A scale as the conversions take it.
FBA_DEVICE float scale_of(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }
// Eight codes -> the values, exactly.
template <typename T>
FBA_DEVICE x8_of<T> from_4_bits(uint32_t codes, float scale) {
  const auto a = FromFp4<T>::template pair<0>(codes, scale), b = FromFp4<T>::template pair<1>(codes, scale);
  const auto c = FromFp4<T>::template pair<2>(codes, scale), d = FromFp4<T>::template pair<3>(codes, scale);
  return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

// A double to a float whose last bits say whether something was cut off, so that a second rounding, to far fewer bits, is the same as a single one of the double: 21 bits are kept,
// and the last one is set if anything behind it was.  What is finite stays so.
FBA_DEVICE float cut(double x) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, x);
  const uint32_t high = (uint32_t)(bits >> 32) | ((uint32_t)bits != 0 ? 1u : 0u);
  const float f = (float)__builtin_bit_cast(double, (uint64_t)high << 32);
  return (high & 0x7ff00000u) != 0x7ff00000u ? fminf(fmaxf(f, -0x1.fffffep127f), 0x1.fffffep127f) : f;
}

}  // namespace fba
