// Work items of dK and dV of attention under a sliding window: which rows see a key tile, how they are cut into items, and where the items' sums go.  Shared by the
// kernel for 128-key tiles (fba_window_dkdv.hip) and the one for 32-key tiles (fba_window_few.hip).
#pragma once
#include "fba_types.h"
#include "fba_window.h"

namespace fba {

constexpr int kWindowSlab = 32;

// Rows of a (key tile, batch): slabs from `first` on, of which those from `cut` on are `gap` further.
struct RowSlabs {
  int first, cut, gap, n;
  __host__ __device__ int at(int i) const { return first + i + (i >= cut ? gap : 0); }
};

// Slabs of 32 rows with some row that sees one of `keys` keys from k0 on inside its window, or (outside) sees a sink among them outside.
__host__ __device__ inline RowSlabs row_slabs(int k0, int keys, int len, int rows, int shift, int window, int sinks, bool causal, bool outside) {
  const int k1 = (k0 + keys < len ? k0 + keys : len) - 1;
  RowSlabs s{0, 0x7fffffff, 0, 0};
  if (rows <= 0 || k1 < k0) return s;
  if (!outside) {
    int low = causal ? k0 - shift : k0 - window + 1 - shift, high = k1 + window - 1 - shift;
    low = low < 0 ? 0 : low;
    high = high > rows - 1 ? rows - 1 : high;
    s.first = low / kWindowSlab;
    s.n = high >= low ? high / kWindowSlab + 1 - s.first : 0;
    return s;
  }
  const int last = (k1 < sinks ? k1 : sinks - 1);  // last sink of the tile
  if (last < k0) return s;
  // behind the window of some sink: rows from k0 + window - shift on; in front of it: rows up to last - window - shift
  int behind = k0 + window - shift;
  behind = behind < 0 ? 0 : behind;
  const int front = causal ? -1 : (last - window - shift > rows - 1 ? rows - 1 : last - window - shift);
  const int n_front = front >= 0 ? front / kWindowSlab + 1 : 0;
  int from = behind / kWindowSlab;
  from = from < n_front ? n_front : from;
  const int all = (rows + kWindowSlab - 1) / kWindowSlab;
  const int n_behind = behind <= rows - 1 && all > from ? all - from : 0;
  s.first = 0;
  s.cut = n_front;
  s.gap = from - n_front;
  s.n = n_front + n_behind;
  return s;
}

// Place of an item's sums: the parts of a tile with several follow each other, inside first; tiles with sinks come first in a (batch, kv head).
__host__ __device__ inline int64_t part_place(const WindowParams& p, int64_t bh, int kt, bool outside, int part) {
  const int64_t with_sinks = (int64_t)p.sink_tiles * (p.band_parts + p.sink_parts), without = p.band_parts > 1 ? (int64_t)(p.tiles - p.sink_tiles) * p.band_parts : 0;
  const int64_t at = bh * (with_sinks + without) + (outside ? p.band_parts : 0) + part;
  return kt < p.sink_tiles ? at + (int64_t)kt * (p.band_parts + p.sink_parts) : at + with_sinks + (int64_t)(kt - p.sink_tiles) * p.band_parts;
}

// A work item: a tile with a part of the rows inside of the window, or of those outside.
struct KeyItem {
  bool outside;
  int part, kt, hkv, b, len, rows, shift, key0, s_begin, n;  // n slabs from s_begin on, over the query heads of the group one after the other
  RowSlabs slabs;
  bool in_parts;   // sums go to a place of the workspace, and not straight into dK and dV
  int64_t place;   // which
};
FBA_DEVICE KeyItem key_item(const WindowParams& p, int item) {
  KeyItem k;
  k.outside = item < p.sink_items;
  const int of = k.outside ? p.sink_parts : p.band_parts, tiles = k.outside ? p.sink_tiles : p.tiles;
  if (!k.outside) item -= p.sink_items;
  k.part = item % of;
  item /= of;
  k.kt = item % tiles;
  item /= tiles;
  k.hkv = item % p.Hkv;
  k.b = item / p.Hkv;
  k.len = p.lengths != nullptr ? min(max(const_idx(p.lengths)[k.b], 0), p.Skv) : p.Skv;
  k.rows = p.lengths != nullptr ? k.len : p.Sq;
  k.shift = p.lengths != nullptr ? 0 : p.Skv - p.Sq;
  k.key0 = k.kt * p.key_tile;
  k.slabs = row_slabs(k.key0, p.key_tile, k.len, k.rows, k.shift, p.window, p.sinks, p.causal != 0, k.outside);
  const int all = k.slabs.n * (p.Hq / p.Hkv);
  k.s_begin = (int)((int64_t)all * k.part / of);
  k.n = (int)((int64_t)all * (k.part + 1) / of) - k.s_begin;
  k.in_parts = p.band_parts > 1 || (p.sink_parts > 0 && k.kt < p.sink_tiles);
  k.place = part_place(p, (int64_t)k.b * p.Hkv + k.hkv, k.kt, k.outside, k.part);
  return k;
}

// Row r has key j in its window when j - back <= r + shift <= j + ahead (causal, of rows outside: all rows up to there count as inside).  This says it for the 32 keys
// from `key0` on, a wave's.
struct KeyMask {
  int key0, shift, limit, back, ahead, rows, outside;
  int whole_lo, whole_hi, some_lo, some_hi, last_whole;
  FBA_DEVICE KeyMask(const WindowParams& p, const KeyItem& k, int first_key) : key0(first_key), shift(k.shift), rows(k.rows), outside(k.outside) {
    limit = k.outside ? min(p.sinks, k.len) : k.len;
    back = k.outside && p.causal ? 0x20000000 : p.causal ? 0 : p.window - 1;
    ahead = p.window - 1;
    // slabs that all of the keys have inside begin at whole_lo .. whole_hi, that some of them have at some_lo .. some_hi
    whole_lo = key0 + 31 - back - shift;
    whole_hi = key0 + ahead - shift - (kWindowSlab - 1);
    some_lo = key0 - back - shift - (kWindowSlab - 1);
    some_hi = key0 + 31 + ahead - shift;
    last_whole = key0 + 31 < limit ? rows / kWindowSlab * kWindowSlab - kWindowSlab : -1;
  }
  FBA_DEVICE bool whole(int row0, int row_min) const {  // all keys see all rows of the slab
    const bool inside = row0 >= whole_lo && row0 <= whole_hi, some = row0 >= some_lo && row0 <= some_hi;
    return row_min <= row0 && row0 <= last_whole && (outside ? !some : inside);
  }
  // S and dP of a slab, or what has been made of them: zero where lane's key does not see the row.  Element 4 g + e of half-wave h is row 8 g + 4 h + e.
  FBA_DEVICE void apply(f32x16& s, f32x16& dp, int row0, int row_min, int lane) const {
    // element e: row r0 + e; inside: a .. a + back + ahead, there at all: from .. from + there - 1
    const int r0 = row0 + 4 * (lane >> 5), key = key0 + (lane & 31), a = key - back - shift - r0, from = row_min - r0;
    const uint32_t inside = back + ahead, there = key < limit ? max(0, rows - row_min) : 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int e = 8 * (r >> 2) + (r & 3);
      const bool sees = (((uint32_t)(e - a) <= inside) != (outside != 0)) && (uint32_t)(e - from) < there;
      s[r] = sees ? s[r] : 0.f;
      dp[r] = sees ? dp[r] : 0.f;
    }
  }
};

}  // namespace fba
