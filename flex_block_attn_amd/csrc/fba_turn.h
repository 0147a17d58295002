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

// Where a lane's eight columns, 8 c .. 8 c + 7, turn: their pairs, and the lane that has what they are paired with.
struct Columns {
  int half, c;  // lanes that have a half of the pairs
  FBA_DEVICE Columns(const Rotation& r, int c) : half(r.pairs >> 3), c(c) {}
  FBA_DEVICE bool on() const { return c < 2 * half; }
  FBA_DEVICE bool first() const { return c < half; }
  FBA_DEVICE int pair(const Rotation& r, int e) const { return r.interleaved ? 4 * c + e / 2 : 8 * (first() ? c : c - half) + e; }
  // (a, b) -> (a cos - b sin, b cos + a sin): whether column e is an a
  FBA_DEVICE bool leads(const Rotation& r, int e) const { return r.interleaved ? e % 2 == 0 : first(); }
  FBA_DEVICE int partner(const Rotation& r) const { return (int)(threadIdx.x & 63) + (r.interleaved || !on() ? 0 : first() ? half : -half); }
};

// The angles of `kPairs` consecutive pairs for a token, in turns times 2^64.  `position`: where it stands on every axis, where the rotation says nothing.
template <int kPairs>
FBA_DEVICE void phases_of(const Rotation& r, int i0, int64_t b, int t, int position, uint64_t (&phases)[kPairs]) {
  int32_t at[kPairs];
  if (r.at != nullptr) {  // (all axes are on their way at a time, then all coordinates)
    const int32_t* const where = r.at + b * r.at_batch + (int64_t)t * r.n_axes;
    uint32_t axes[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) axes[i] = (uint32_t)r.axes[i0 + i];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) at[i] = where[min(axes[i], (uint32_t)r.n_axes - 1)];  // (an axis that there is not counts as the last)
  } else {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) at[i] = position;
  }
#pragma unroll
  for (int i = 0; i < kPairs; ++i) phases[i] = (uint64_t)r.turns[i0 + i] * (uint64_t)(int64_t)at[i];
}

// What a lane's eight columns of a token's rows are multiplied by: x own + (what they are paired with) other.
struct Turn {
  float own[8], other[8];
  int from;  // lane of the wave that has the columns these are paired with
  bool on;   // these columns turn at all

  FBA_DEVICE void init(const Rotation& r, const Columns& columns, int64_t b, int t, int position) {
    on = columns.on();
    from = columns.partner(r);
    if (!on) return;
    if (r.interleaved) {
      uint64_t phases[4];
      phases_of(r, columns.pair(r, 0), b, t, position, phases);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        float s, co;
        sincos_of(phases[e / 2], &s, &co);
        if (r.back) s = -s;
        own[e] = own[e + 1] = co;
        other[e] = -s;
        other[e + 1] = s;
      }
    } else {
      uint64_t phases[8];
      phases_of(r, columns.pair(r, 0), b, t, position, phases);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float s;
        sincos_of(phases[e], &s, &own[e]);
        other[e] = columns.first() != (r.back != 0) ? -s : s;
      }
    }
  }
};

// The columns that a lane's own are paired with.  All sixteen lanes of the row take part.
template <typename T>
FBA_DEVICE x8_of<T> paired(x8_of<T> x, const Turn& turn, bool interleaved) {
  if (interleaved) return __builtin_shufflevector(x, x, 1, 0, 3, 2, 5, 4, 7, 6);
  u32x4 bits = __builtin_bit_cast(u32x4, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) bits[i] = (uint32_t)__shfl((int)bits[i], turn.from);
  return __builtin_bit_cast(x8_of<T>, bits);
}

// A lane's columns of a row, turned in 32 bits and rounded once.
template <typename T>
FBA_DEVICE x8_of<T> turned(x8_of<T> x, const Turn& turn, bool interleaved) {
  const x8_of<T> y = paired<T>(x, turn, interleaved);
  if (!turn.on) return x;
  float o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (float)x[e] * turn.own[e] + (float)y[e] * turn.other[e];
  return __builtin_shufflevector(narrow4<T>(o[0], o[1], o[2], o[3]), narrow4<T>(o[4], o[5], o[6], o[7]), 0, 1, 2, 3, 4, 5, 6, 7);
}

}  // namespace fba
