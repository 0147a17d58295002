// Positions by rotation: what its kernels share.
//
// Pair i of a row, columns (2i, 2i + 1) or (i, i + pairs), is turned by angle(i) = 2 pi turns[i] p[axes[i]]: (a, b) -> (a cos - b sin, a sin + b cos).  Columns from
// 2 * pairs on stay as they are.  turns are held as fractions of 2^64, so that the product with a whole position is exact modulo whole turns in 64-bit integers, however far the
// position: what is left is a fraction of a turn, and no angle ever grows.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fba_window.h"

namespace fba {

struct Rotation {
  const int64_t* turns;  // [pairs]; null: nothing turns
  const int32_t* axes;   // [pairs]
  const int32_t* at;     // null, or where every token stands: [batch, tokens, n_axes]
  int64_t at_batch;      // elements from one sequence to the next
  int n_axes, pairs, interleaved, back;
};

struct RotaryParams {
  Strided q, q_out, k, k_out;
  Rotation rotation;
  int heads, kv_heads, seq;
  uint32_t tokens, parts, per;  // of all sequences; parts that the heads are cut into, heads of a part
};

hipError_t launch_rotary(RotaryParams p, bool half, hipStream_t stream);

// How many parts the heads of `tokens` tokens are cut into: 16 lanes do one part of one token, and 2^14 parts are a wave for every place that the GPU has for one at half of its occupancy.
// 24 + 24 heads of 1000 tokens with 2^12, 2^13, 2^14, 2^15 and 2^16 parts: 6.6, 6.3, 6.9, 7.4 and 10.0 us; 8 + 2 of 6272: 8.5, 9.4, 9.4, 11.4 and 16.6; 6 of 12000 into 4 bits: 18.2, 18.4,
// 16.9, 19.3 and 25.4; with one part each 13.9, 8.6 and 18.4, and for 64 new tokens, 40 heads, 14.8 instead of 5.3.
inline uint32_t rotary_parts(int64_t tokens, int64_t heads) {
  const int64_t want = tokens > 0 ? (16384 + tokens - 1) / tokens : 1;
  return (uint32_t)(want < heads ? want : heads > 0 ? heads : 1);
}

}  // namespace fba
