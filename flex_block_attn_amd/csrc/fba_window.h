// Attention under a sliding window with sinks: parameters, launchers, and what host and kernels say alike about rows, keys and work items.
//
// Query row i stands at position p = i + Skv - Sq (with lengths, where Sq = Skv: at i).  Key j is visible to it when both are within the
// sequence's length and
//   causal:     j <= p and (p - j < window or j < sinks)
//   two-sided:  |p - j| < window or j < sinks
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fba {

struct Strided {  // a (batch, heads, rows, 128) tensor of 16-bit values; strides in bytes, the last dimension is dense
  char* ptr;
  int64_t batch, head;
  uint32_t row;
};

struct WindowParams {
  Strided q, k, v, o, d_o, dq, dk, dv;
  Strided o_low;           // what rounding o has left; ptr null: not wanted
  float* lse;              // [B, Hq, Sq], in log2 units; +inf for a row that sees nothing
  float* lse_exact;        // [B, Hq, Sq], of P before rounding, found by dQ for dK and dV
  float* neg_delta;        // [B, Hq, Sq], -rowsum(dO o O)
  const int32_t* lengths;  // null, or [B]
  float* parts;            // fp32 partial sums of dK and dV of key tiles with several items
  int B, Hq, Hkv, Sq, Skv, window, sinks, causal;
  float scale, scale_log2e;  // 1 / sqrt(128), and times log2(e)
  int tiles, items, chunk;   // tiles of a head, work items, consecutive items that one XCD gets together
  // dK/dV: keys of a tile; parts that the rows inside of a tile's window are cut into; tiles with sinks of a (batch, kv head), and the parts of the rows outside (0: there are none)
  int key_tile, band_parts, sink_tiles, sink_parts, sink_items;
};

constexpr int kWindowTile = 128;
inline __host__ __device__ int64_t part_floats(const WindowParams& p) { return 2 * 128 * p.key_tile; }  // dV tile, dK tile

// Few query rows: forward, or dQ and neg_delta.  Few key tiles: dK and dV.
bool window_takes_few(const WindowParams& p, int compute_units, bool backward);
bool window_keys_few(const WindowParams& p, int compute_units);
hipError_t launch_window_few_dkdv(WindowParams p, bool half, hipStream_t stream);
hipError_t launch_window_few(WindowParams p, bool half, bool backward, hipStream_t stream);
hipError_t launch_window_fwd(WindowParams p, bool half, hipStream_t stream);
hipError_t launch_window_dq(WindowParams p, bool half, hipStream_t stream);    // before dK and dV: works lse_exact and neg_delta out
hipError_t launch_window_dkdv(WindowParams p, bool half, hipStream_t stream);  // lse: the exact one; d_o has q's row stride
// Decides on key_tile, band_parts, sink_tiles and sink_parts; returns the bytes of `parts` that dK and dV need.
int64_t plan_window_dkdv(WindowParams& p, int compute_units);

// Work-group id -> item: consecutive items, which read the same keys, go to one XCD `chunk` at a time, so that they meet in its L2, and the XCDs take turns, so
// that each gets short and long items alike.
__device__ __forceinline__ int window_item(int wg, int chunk) {
  const int xcd = wg & 7, i = wg >> 3;
  return (i / chunk * 8 + xcd) * chunk + i % chunk;
}
inline int window_grid(int items, int chunk) { return (items + 8 * chunk - 1) / (8 * chunk) * (8 * chunk); }
inline int window_chunk(int items) { return items >= 8 * 32 ? 32 : items < 8 ? 1 : items / 8; }

}  // namespace fba
