// The building blocks of fba_common.h for kernels that take bf16 and fp16 alike, and tensors with strides.
//
// Both types have the same matrix instructions, fetches and layouts; what differs is chosen by Elem<T>.
#pragma once
#include "fba_common.h"

namespace fba {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <typename T>
struct Elem;

template <>
struct Elem<__bf16> {
  using x2 = bf16x2;
  using x4 = bf16x4;
  using x8 = bf16x8;
  FBA_DEVICE static f32x16 mfma32(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  FBA_DEVICE static f32x4 mfma16(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  FBA_DEVICE static float dot2(x2 a, x2 b, float c) { return __builtin_amdgcn_fdot2_f32_bf16(a, b, c, false); }
};

template <>
struct Elem<_Float16> {
  using x2 = f16x2;
  using x4 = f16x4;
  using x8 = f16x8;
  FBA_DEVICE static f32x16 mfma32(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  FBA_DEVICE static f32x4 mfma16(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  FBA_DEVICE static float dot2(x2 a, x2 b, float c) { return __builtin_amdgcn_fdot2(a, b, c, false); }
};

template <typename T>
using x8_of = typename Elem<T>::x8;
template <typename T>
using x4_of = typename Elem<T>::x4;

// Fetches of fba_common.h by type (they move 16-bit values, whatever these are).
template <typename T>
FBA_DEVICE x8_of<T> read_b128(LdsPtr p) { return *reinterpret_cast<const FBA_LDS x8_of<T>*>(p); }
template <typename T>
FBA_DEVICE x4_of<T> read_tr(LdsPtr p) { return __builtin_bit_cast(x4_of<T>, lds_read_tr(p)); }
template <typename T>
FBA_DEVICE x8_of<T> read_tr8(LdsPtr lo, LdsPtr hi) {
  return __builtin_shufflevector(read_tr<T>(lo), read_tr<T>(hi), 0, 1, 2, 3, 4, 5, 6, 7);
}

// fp32 -> T, to the nearest
template <typename T>
FBA_DEVICE x4_of<T> narrow4(float a0, float a1, float a2, float a3) {
  using x2 = typename Elem<T>::x2;
  return __builtin_shufflevector(__builtin_convertvector((f32x2){a0, a1}, x2), __builtin_convertvector((f32x2){a2, a3}, x2), 0, 1, 2, 3);
}
template <typename T>
FBA_DEVICE x8_of<T> narrow8(const f32x16& s, int j) {  // values 8j .. 8j + 7
  return __builtin_shufflevector(narrow4<T>(s[8 * j + 0], s[8 * j + 1], s[8 * j + 2], s[8 * j + 3]),
                                 narrow4<T>(s[8 * j + 4], s[8 * j + 5], s[8 * j + 6], s[8 * j + 7]), 0, 1, 2, 3, 4, 5, 6, 7);
}

// Copies of 32-row slabs from global memory into swizzled LDS tiles, as SlabDma, of tensors whose rows are `stride` bytes apart and whose last slab
// may be short: places behind row `last` of the sequence get that row, so that nothing outside of the sequence is read and what is not a number there
// stays there (such rows are masked).  Waves 0..3 do it together (8 rows each).
struct RowDma {
  uint32_t off[2], off_last[2];
  uint32_t wave_dst;
  int last_slab;
  FBA_DEVICE void init(int wave, int lane, uint32_t stride, int last) {
    last_slab = last >> 5;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int row = 8 * wave + 4 * g + (lane >> 4);
      const uint32_t chunk = ((lane & 15) ^ swz(row)) << 4;
      off[g] = row * stride + chunk;
      off_last[g] = min(row, last & 31) * stride + chunk;
    }
    wave_dst = wave * 8 * kRowBytes;
  }
  // src: the slab's first row, `slab` its number
  FBA_DEVICE void piece(int i, uint32_t slab_lds, const char* src, int slab) const {
    dma16(slab_lds + wave_dst + i * 4 * kRowBytes, src, slab == last_slab ? off_last[i] : off[i]);
  }
  FBA_DEVICE void copy(uint32_t slab_lds, const char* src, int slab) const {
    piece(0, slab_lds, src, slab);
    piece(1, slab_lds, src, slab);
  }
};

// store_tile_bf16 by type, to rows `stride` bytes apart; `rows` of the 32 are stored.  kLow: what rounding leaves, rounded, instead.
template <typename T, bool kLow = false>
FBA_DEVICE void store_tile(char* buf, const f32x16 (&acc)[4], float scale, char* out, uint32_t stride, int lane, int rows) {
  const int l32 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int mb = 0; mb < 4; ++mb)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float v[4] = {acc[mb][4 * g + 0] * scale, acc[mb][4 * g + 1] * scale, acc[mb][4 * g + 2] * scale, acc[mb][4 * g + 3] * scale};
      x4_of<T> value = narrow4<T>(v[0], v[1], v[2], v[3]);
      if constexpr (kLow) value = narrow4<T>(v[0] - (float)value[0], v[1] - (float)value[1], v[2] - (float)value[2], v[3] - (float)value[3]);
      *reinterpret_cast<x4_of<T>*>(buf + tile_off(l32, 4 * mb + g) + 8 * h) = value;
    }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = 4 * i + (lane >> 4);
    if (row < rows)
      *reinterpret_cast<u32x4*>(out + (int64_t)row * stride + (lane & 15) * 16) = *reinterpret_cast<const u32x4*>(buf + tile_off(row, lane & 15));
  }
}

}  // namespace fba
