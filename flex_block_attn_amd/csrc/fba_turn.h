// Rotation of a row (fba_rotary.h) by sixteen lanes, eight columns each: a lane needs the eight columns that its own are paired with, which another lane has, or, interleaved, itself.
#pragma once
#include "fba_rotary.h"
#include "fba_types.h"

namespace fba {

// sin and cos of `phase` / 2^64 turns.  The nearest quarter turn is taken off, and the rest, an eighth of a turn at most, goes into the Taylor series: up to x^10 in 32 bits (the
// next terms are below 2^-29), up to x^16 in 64 (below 2^-54).
FBA_DEVICE void sincos_of(uint64_t phase, float* sin, float* cos) {
  const uint32_t quarter = (uint32_t)((phase + (1ull << 61)) >> 62);
  const int32_t rest = (int32_t)((phase - ((uint64_t)quarter << 62)) >> 32);
  const float x = (float)rest * (float)(6.283185307179586 / 4294967296.0), y = x * x;
  const float s = x + x * y * (-1.f / 6 + y * (1.f / 120 + y * (-1.f / 5040 + y * (1.f / 362880))));
  const float c = 1.f + y * (-0.5f + y * (1.f / 24 + y * (-1.f / 720 + y * (1.f / 40320 - y * (1.f / 3628800)))));
  const float u = quarter & 1 ? c : s, v = quarter & 1 ? s : c;
  *sin = quarter & 2 ? -u : u;
  *cos = (quarter + 1) & 2 ? -v : v;
}
FBA_DEVICE void sincos_of(uint64_t phase, double* sin, double* cos) {
  const uint32_t quarter = (uint32_t)((phase + (1ull << 61)) >> 62);
  const int64_t rest = (int64_t)(phase - ((uint64_t)quarter << 62));
  const double x = (double)rest * (6.283185307179586 / 18446744073709551616.0), y = x * x;
  const double s = x + x * y * (-1. / 6 + y * (1. / 120 + y * (-1. / 5040 + y * (1. / 362880 + y * (-1. / 39916800 + y * (1. / 6227020800. - y * (1. / 1307674368000.)))))));
  const double c = 1. + y * (-0.5 + y * (1. / 24 + y * (-1. / 720 + y * (1. / 40320 + y * (-1. / 3628800 + y * (1. / 479001600. + y * (-1. / 87178291200. + y * (1. / 20922789888000.))))))));
  const double u = quarter & 1 ? c : s, v = quarter & 1 ? s : c;
  *sin = quarter & 2 ? -u : u;
  *cos = (quarter + 1) & 2 ? -v : v;
}

// What a lane's eight columns of a token's rows are multiplied by: x own + (what they are paired with) other.
template <typename F>
struct Turn {
  F own[8], other[8];
  int from;  // lane of the wave that has the columns these are paired with
  bool on;   // these columns turn at all

  // Columns 8 c .. 8 c + 7; `position`: on every axis, where the rotation says nothing.
  FBA_DEVICE void init(const Rotation& r, int64_t b, int t, int position, int c) {
    const int half = r.pairs >> 3;  // lanes that have a half of the pairs
    on = c < 2 * half;
    from = threadIdx.x & 63;
    if (!on) return;
    const bool first = c < half;
    if (!r.interleaved) from += first ? half : -half;
    const int32_t* const at = r.at != nullptr ? r.at + b * r.at_batch + (int64_t)t * r.n_axes : nullptr;
    auto pair = [&](int i, F* sin, F* cos) {
      // (an axis that there is not counts as the last)
      const int32_t p = at != nullptr ? at[min((uint32_t)r.axes[i], (uint32_t)r.n_axes - 1)] : position;
      sincos_of((uint64_t)r.turns[i] * (uint64_t)(int64_t)p, sin, cos);
      if (r.back) *sin = -*sin;
    };
    if (r.interleaved) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        F s, co;
        pair(4 * c + e / 2, &s, &co);
        own[e] = own[e + 1] = co;
        other[e] = -s;
        other[e + 1] = s;
      }
    } else {
      const int i0 = 8 * (first ? c : c - half);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        F s;
        pair(i0 + e, &s, &own[e]);
        other[e] = first ? -s : s;
      }
    }
  }
};

// The columns that a lane's own are paired with.  All sixteen lanes of the row take part.
template <typename T, typename F>
FBA_DEVICE x8_of<T> paired(x8_of<T> x, const Turn<F>& turn, bool interleaved) {
  if (interleaved) return __builtin_shufflevector(x, x, 1, 0, 3, 2, 5, 4, 7, 6);
  u32x4 bits = __builtin_bit_cast(u32x4, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) bits[i] = (uint32_t)__shfl((int)bits[i], turn.from);
  return __builtin_bit_cast(x8_of<T>, bits);
}

// A lane's columns of a row, turned in 32 bits and rounded once.
template <typename T, typename F>
FBA_DEVICE x8_of<T> turned(x8_of<T> x, const Turn<F>& turn, bool interleaved) {
  const x8_of<T> y = paired<T>(x, turn, interleaved);
  if (!turn.on) return x;
  float o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (float)x[e] * (float)turn.own[e] + (float)y[e] * (float)turn.other[e];
  return __builtin_shufflevector(narrow4<T>(o[0], o[1], o[2], o[3]), narrow4<T>(o[4], o[5], o[6], o[7]), 0, 1, 2, 3, 4, 5, 6, 7);
}

}  // namespace fba
