// Attention of one new token per sequence over a paged cache, of 16-bit rows and of 4-bit ones: what both kernels share.  How the work is cut is stated in fba_cache_attend.hip.
#pragma once
#include "fba_cache.h"
#include "fba_types.h"

namespace fba {

namespace {

constexpr int kTile = 32;
constexpr int kTileLds = kTile * kRowBytes;  // 8 KiB
constexpr int kWaves = 4;
constexpr int kLeastTiles = kWaves;          // of a share
constexpr float kLazy = 8.f, kNoReference = -3e38f;

inline int head_tiles_of(int group) { return group <= 16 ? 1 : 2; }  // query heads of a work-group, in sixteens (four do not fit the registers of two waves on a SIMD)

constexpr int kResident4 = 3;  // work-groups on a compute unit, of 4 bits and 16 heads

// Tiles of a sequence that are read: those with sinks, then those from the window's start on.
struct Tiles {
  int n_sink, first, n;
  FBA_DEVICE int at(int t) const { return t < n_sink ? t : first + t - n_sink; }
};
FBA_DEVICE Tiles tiles_of(int len, int window, int sinks) {
  const int from = max(0, len - window), s = from > 0 ? min(sinks, len) : 0;
  Tiles t;
  t.n_sink = (s + kTile - 1) / kTile;
  t.first = max(from / kTile, t.n_sink);
  t.n = t.n_sink + max(0, (len + kTile - 1) / kTile - t.first);
  return t;
}

FBA_DEVICE int length_of(const AttendParams& p, int b, bool* bad) {
  const int n = p.cache.lengths[b];
  *bad = !p.cache.holds(n);
  return *bad ? 0 : n;
}

// A pointer that every lane has alike, in scalar registers.
FBA_DEVICE const char* uniform(const char* p) {
  const uint64_t v = (uint64_t)p;
  return (const char*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// The tiles of all sequences, one behind the other, dealt to `wgs` work-groups in even shares.  A sequence's part in share w has place w + b for its results: from one part to
// the next w or b rises.
struct Shares {
  int total, wgs;
  FBA_DEVICE int begin(int w) const { return (int)((int64_t)total * w / wgs); }
  FBA_DEVICE int of(int tile) const { return (int)((((int64_t)tile + 1) * wgs - 1) / total); }
};

// A work-group's share: its number, its tiles, the sequence of the first one and that sequence's first tile.  All waves find it alike.
struct Share {
  int w, tile, end, b, start;
};
FBA_DEVICE bool find_share(const AttendParams& p, int tid, int lane, int wave, Share* share) {
  const CacheView& cache = p.cache;
  auto tiles_in = [&](int b) {
    bool bad;
    return b < cache.batch ? tiles_of(length_of(p, b, &bad), p.window, p.sinks).n : 0;
  };
  int total = 0;
  const bool one = cache.batch == 1;              // (needs no sums over the wave: 8.1 us instead of 8.5 for 768 slots)
  const int of_first = tiles_in(one ? 0 : lane);  // sequences 0 .. 63
  if (one) total = __builtin_amdgcn_readfirstlane(of_first);
  else
    for (int b0 = 0; b0 < cache.batch; b0 += 64) total += wave_sum(b0 == 0 ? of_first : tiles_in(b0 + lane));
  // (of 4 bits as many as sequences, if there are tiles for them: 64 of a tile each 9.9 us instead of 16.9; of 16 bits the last bits of results hang on where sequences are cut)
  const int least = cache.k_scales != nullptr ? min(total, cache.batch) : 0;
  const Shares shares{total, min(p.target, max(max(1, least), (total + kLeastTiles - 1) / kLeastTiles))};
  const int w = blockIdx.x;
  if (w >= shares.wgs) return false;
  int tile = shares.begin(w);
  const int end = shares.begin(w + 1);
  const bool notes = w == 0 && blockIdx.y == 0;  // writes down which shares every sequence is in
  int b = -1, start = 0;                         // the sequence of `tile`, its first tile
  if (one) {
    b = 0;
    if (notes && tid == 0) {
      p.note[0] = 0;
      p.note[1] = total > 0 ? shares.of(total - 1) + 1 : 0;
    }
  }
  for (int b0 = 0, before = 0; !one && b0 < cache.batch && (b < 0 || notes); b0 += 64) {
    const int n = b0 == 0 ? of_first : tiles_in(b0 + lane);
    int sum = n;  // of the lanes up to this one
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int other = __shfl_up(sum, d);
      if (lane >= d) sum += other;
    }
    const unsigned long long past = __builtin_amdgcn_ballot_w64(before + sum > tile);
    if (past != 0 && b < 0) {
      const int at = __builtin_ctzll(past);
      b = b0 + at;
      start = before + __builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readlane(n, at);
    }
    if (notes && wave == 0 && b0 + lane < cache.batch) {
      const int first = n > 0 ? shares.of(before + sum - n) : 0;
      p.note[2 * (b0 + lane)] = first + b0 + lane;
      p.note[2 * (b0 + lane) + 1] = n > 0 ? shares.of(before + sum - 1) - first + 1 : 0;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  *share = {w, tile, end, b, start};
  return true;
}

// The waves' sums of a sequence: to the output where the sequence is in one share, else where the second kernel joins them.  `smem`: room for kSumsLds bytes that no wave uses any more
// once it is here; free again behind the call.
constexpr int kSumsLds = kWaves * 16 * (kHeadDim + 2) * 4;
template <typename T, int kHeadTiles>
FBA_DEVICE void leave_sums(const AttendParams& p, char* smem, const f32x4 (&acc)[kHeadTiles][8], const float (&m_run)[kHeadTiles], const float (&l_run)[kHeadTiles], bool any_bad, bool alone, int b,
                           int w, int head0, int heads) {
  const int tid = threadIdx.x, l16 = tid & 15, g = (tid & 63) >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // The waves' sums: every wave's O [16 heads][128] and its references and denominators, in LDS, sixteen heads after the other.
  float* const sums = reinterpret_cast<float*>(smem);         // [kWaves][16][128]
  float* const ml = sums + kWaves * 16 * kHeadDim;            // [kWaves][16][2]
#pragma unroll
  for (int ht = 0; ht < kHeadTiles; ++ht) {
    __syncthreads();
    float l = l_run[ht];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const int row = wave * 16 + l16;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(sums + row * kHeadDim + 16 * dt + 4 * g) = acc[ht][dt];
    if (g == 0) {
      ml[2 * row] = m_run[ht];
      ml[2 * row + 1] = any_bad ? __builtin_nanf("") : l;
    }
    __syncthreads();
    const int d = tid % (kHeadDim / 4) * 4;
    for (int head = tid / (kHeadDim / 4); head < min(16, heads - 16 * ht); head += 64 * kWaves / (kHeadDim / 4)) {
      float m = kNoReference, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) m = fmaxf(m, ml[2 * (w * 16 + head)]);
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = fast_exp2(ml[2 * (w * 16 + head)] - m);
        sum += f * ml[2 * (w * 16 + head) + 1];
        o += f * *reinterpret_cast<const f32x4*>(sums + (w * 16 + head) * kHeadDim + d);
      }
      const int at_head = head0 + 16 * ht + head;
      const int64_t at = (int64_t)(w + b) * p.heads + at_head;
      if (alone) {
        const float f = sum == 0.f ? 0.f : 1.f / sum;  // (NaN stays)
        *reinterpret_cast<x4_of<T>*>(p.o.ptr + b * p.o.batch + at_head * p.o.head + 2 * d) = narrow4<T>(o[0] * f, o[1] * f, o[2] * f, o[3] * f);
      } else {
        *reinterpret_cast<f32x4*>(p.part + at * kHeadDim + d) = o;
      }
      if (d == 0) {
        p.part_ml[2 * at] = m;
        p.part_ml[2 * at + 1] = sum;
      }
    }
  }
  __syncthreads();
}

}  // namespace

}  // namespace fba
