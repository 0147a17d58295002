// What fills a paged cache and what makes room in it: gfx950.  Rows of 256 bytes are moved, 16 lanes to a row (of 64 where they are held in 4 bits, and their scales); bound by device memory, in small calls by the launch.
#include "fba_cache.h"
#include "fba_common.h"

namespace fba {

// New tokens' rows go to the slots behind the sequences' lengths.  Work-groups 0 .. batch - 1 work out the new lengths, those behind them copy rows, 16 threads to a
// row of K and of V.
__global__ __launch_bounds__(256) void cache_append_kernel(const AppendParams p) {
  const CacheView& cache = p.cache;
  const int tid = threadIdx.x;
  // how many tokens sequence b gets: -1 where its length or count makes no sense or there is no room
  auto tokens_of = [&](int b, int* len) {
    *len = cache.lengths[b];
    const int n = p.counts != nullptr ? p.counts[b] : p.tokens;
    return cache.holds(*len) && n >= 0 && n <= p.tokens && cache.holds((int64_t)*len + n) ? n : -1;
  };
  if ((int)blockIdx.x < cache.batch) {
    const int b = blockIdx.x;
    int len;
    const int n = tokens_of(b, &len);
    bool bad = n < 0;
    if (n > 0)
      for (int i = (len >> cache.page_log2) + tid; i <= (len + n - 1) >> cache.page_log2; i += 256) bad |= cache.page_of(b, i << cache.page_log2) < 0;
    const bool any = __syncthreads_or(bad);
    if (tid == 0) p.lengths_out[b] = any ? -1 : len + n;
    return;
  }
  const int64_t rows = (int64_t)cache.batch * cache.kv_heads * p.tokens;
  const int c = tid & 15;
  for (int64_t r = (int64_t)(blockIdx.x - cache.batch) * 16 + (tid >> 4); r < rows; r += (int64_t)p.row_wgs * 16) {
    const int t = r % p.tokens;
    const int bh = r / p.tokens, h = bh % cache.kv_heads, b = bh / cache.kv_heads;
    int len;
    const int n = tokens_of(b, &len);
    if (t >= n) continue;
    const int page = cache.page_of(b, len + t);
    if (page < 0) continue;
    const int64_t to = cache.row_of(page, h, len + t);
    const u32x4 kr = *reinterpret_cast<const u32x4*>(p.k.ptr + b * p.k.batch + h * p.k.head + (int64_t)t * p.k.row + c * 16);
    const u32x4 vr = *reinterpret_cast<const u32x4*>(p.v.ptr + b * p.v.batch + h * p.v.head + (int64_t)t * p.v.row + c * 16);
    *reinterpret_cast<u32x4*>(cache.k + to * kRowBytes + c * 16) = kr;
    *reinterpret_cast<u32x4*>(cache.v + to * kRowBytes + c * 16) = vr;
    if (c == 0 && cache.positions != nullptr) cache.positions[to] = (p.first != nullptr ? p.first[b] : len) + t;
    if (c == 1 && cache.weights != nullptr) cache.weights[to] = p.weights != nullptr ? p.weights[r] : 0.f;
  }
}

hipError_t launch_cache_append(AppendParams p, hipStream_t stream) {
  const int64_t rows = (int64_t)p.cache.batch * p.cache.kv_heads * p.tokens, wgs = (rows + 15) / 16;
  p.row_wgs = (int)(wgs < 8192 ? wgs : 8192);
  hipLaunchKernelGGL(cache_append_kernel, dim3(p.cache.batch + p.row_wgs), dim3(256), 0, stream, p);
  return hipGetLastError();
}

// Eviction, first kernel: which slots of a (sequence, kv head) stay.  A work-group of 1024 threads reads weights and positions once, finds the budget-th largest key by
// counting (11, 11 and 10 bits of it at a time), and lists the freed slots below the budget and the kept slots behind it, in order.  A wave has consecutive slots, 256 at a
// time, four to a lane, so that loads are dense, ballots number the slots inside of a wave and one scan over the waves does the rest.  Bound by latency, of the loads and
// some twenty barriers, and, where a sequence is long, by the arithmetic for each slot on the one compute unit that its head has (24 heads of 30720: 27 us; what moves the rows, 19 us for
// 102 MB).
//
// A slot's key orders as its weight does (NaN below everything, the two zeros alike); the slots that are held are above all of them.
namespace {
// Counters of a digit, lanes apart: weights have few exponents, and lanes that add to one counter wait for each other (4 x 6 heads of 32768 slots to 16384: 44 / 40 us with one /
// four of each; eight, whose sum takes longer, 43, and 24 instead of 20 for 32 x 6 of 8192).
constexpr int kCopies = 4;
constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64, kBins = 2048;
// Minima one after the other / the search, 32 x 6 heads of 4096 slots and 1, 2, 4, 8 more (with the launch of the second kernel): 8.5 / 13.5, 9.4 / 13.6, 10.7 / 14.1, 13.4 / 14.6 us;
// 4 x 6 of 16384: 13.8 / 22.8, 14.9 / 22.9, 17.3 / 23.4, 21.8 / 23.9; 8 of 1024: 7.8 / 11.2, 8.5 / 11.2, 10.1 / 11.4, 12.9 / 11.7.
constexpr int kFewDropped = 6;
// Rows that one head may have to move, by the table's size, up to which the first kernel moves them.  A second one / the first, 1, 64 and 256 slots over the budget: 32 x 6 heads of
// 4096 slots 8.6 / 7.2, 16.6 / 14.1, 21.5 / 17.0 us; 4 x 6 of 16384: 13.9 / 12.5, 25.0 / 23.4, 27.1 / 28.1, and with 1024 29.6 / 34.1.
constexpr int kFewMoved = 256;
FBA_DEVICE uint32_t weight_key(float w) {
  if (w != w) return 0;
  uint32_t bits = __builtin_bit_cast(uint32_t, w);
  if (bits == 0x80000000u) bits = 0;
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// Sum over the waves in front of this one, and over all of them, of a number that a wave's lanes have alike.  `of`: kSelectWaves ints that nobody else uses at the time.
FBA_DEVICE int waves_before(int x, int* of, int* total) {
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) of[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kSelectWaves; ++i) {
    const int n = of[i];
    before += i < wave ? n : 0;
    all += n;
  }
  *total = all;
  return before;
}

// Places of the set ones of 256 slots, four to a lane, in order.
struct Ranks {
  int at[4], n;  // set ones in front of each of this lane's four, and of all
  FBA_DEVICE Ranks(const bool (&on)[4], int lane) {
    const unsigned long long below = (1ull << lane) - 1;
    int before = 0, all = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned long long ballot = __builtin_amdgcn_ballot_w64(on[e]);
      before += __builtin_popcountll(ballot & below);
      all += __builtin_popcountll(ballot);
    }
    n = all;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      at[e] = before;
      before += on[e];
    }
  }
};

// One row's sixteenth, of the pool of K or of V.
FBA_DEVICE void move_piece(char* rows, bool held, int64_t to, int64_t from, int c) {
  if (held) *reinterpret_cast<uint32_t*>(rows + to * kHeldRowBytes + c * 4) = *reinterpret_cast<const uint32_t*>(rows + from * kHeldRowBytes + c * 4);
  else *reinterpret_cast<u32x4*>(rows + to * kRowBytes + c * 16) = *reinterpret_cast<const u32x4*>(rows + from * kRowBytes + c * 16);
}
FBA_DEVICE void move_scales(uint8_t* scales, int64_t to, int64_t from) {  // of a row, all four
  reinterpret_cast<uint32_t*>(scales)[to] = reinterpret_cast<const uint32_t*>(scales)[from];
}

// The i-th freed slot gets the i-th kept one from behind the budget, row, position and weight: 16 lanes to a row, i = first, first + step, ...
FBA_DEVICE void move_rows(const CacheView& cache, const int32_t* moves, int most, int b, int hkv, int c, int first, int step, int n) {
  const bool held = cache.k_scales != nullptr;
  for (int i = first; i < n; i += step) {
    const int to_slot = moves[1 + i], from_slot = moves[1 + most + i];
    const int64_t to = cache.row_of(cache.page_of(b, to_slot), hkv, to_slot), from = cache.row_of(cache.page_of(b, from_slot), hkv, from_slot);
    if (held) {
      move_piece(cache.k, true, to, from, c);
      move_piece(cache.v, true, to, from, c);
      if (c == 2) move_scales(cache.k_scales, to, from);
      if (c == 3) move_scales(cache.v_scales, to, from);
    } else {
      const u32x4 kr = *reinterpret_cast<const u32x4*>(cache.k + from * kRowBytes + c * 16), vr = *reinterpret_cast<const u32x4*>(cache.v + from * kRowBytes + c * 16);
      *reinterpret_cast<u32x4*>(cache.k + to * kRowBytes + c * 16) = kr;
      *reinterpret_cast<u32x4*>(cache.v + to * kRowBytes + c * 16) = vr;
    }
    if (c == 0) cache.positions[to] = cache.positions[from];
    if (c == 1) cache.weights[to] = cache.weights[from];
  }
}
}  // namespace

// kGroups: keys of up to kGroups times 4096 slots stay in registers (kGroups <= 8); 0: any number of slots, read again in every pass.
template <int kGroups>
__global__ __launch_bounds__(kSelectThreads) void cache_select_kernel(const EvictParams p) {
  const CacheView& cache = p.cache;
  __shared__ __attribute__((aligned(16))) int bins[kBins * kCopies];
  __shared__ int sums[6][kSelectWaves], found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hkv = blockIdx.x % cache.kv_heads, b = blockIdx.x / cache.kv_heads;
  int32_t* const moves = p.moves + (int64_t)blockIdx.x * (1 + 2 * (int64_t)p.most);
  // The table is fetched beside the length, as much as there is: what keys in registers can be of has kGroups * 256 pages at most.
  constexpr int kPages = kGroups * 256, kOwnPages = (kPages + kSelectThreads - 1) / kSelectThreads;
  __shared__ int pages[kPages > 0 ? kPages : 1];
  int page[kOwnPages > 0 ? kOwnPages : 1];
#pragma unroll
  for (int i = 0; i < kOwnPages; ++i) {
    const int at = tid + i * kSelectThreads;
    page[i] = at < cache.max_pages ? cache.table[(int64_t)b * cache.max_pages + at] : -1;
  }
  const int len = cache.lengths[b];
  bool bad = !cache.holds(len);
  const int used = bad ? 0 : (len + (1 << cache.page_log2) - 1) >> cache.page_log2;
  if constexpr (kGroups > 0) {
#pragma unroll
    for (int i = 0; i < kOwnPages; ++i) {
      const int at = tid + i * kSelectThreads;
      if (at < used) {
        pages[at] = page[i];
        bad |= page[i] < 0 || page[i] >= cache.pages;
      }
    }
  } else {
    for (int i = tid; i < used; i += kSelectThreads) bad |= cache.page_of(b, i << cache.page_log2) < 0;
  }
  bad = __syncthreads_or(bad);
  if (tid == 0 && hkv == 0) p.lengths_out[b] = bad ? -1 : min(len, p.budget);
  if (bad || len <= p.budget) {
    if (tid == 0) moves[0] = 0;
    return;
  }
  typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
  auto row_of = [&](int slot) { return cache.row_of(kGroups > 0 ? pages[slot >> cache.page_log2] : cache.page_of(b, slot), hkv, slot); };  // of four slots, which are on one page
  const int per = (len + 4 * kSelectThreads - 1) / (4 * kSelectThreads);  // groups of 256 slots that a wave has
  auto slot_of = [&](int j) { return (wave * per + j) * 256 + 4 * lane; };

  // the largest position
  int newest = -0x7fffffff - 1;
  constexpr int kHeld = kGroups > 0 ? kGroups : 1;
  f32x4 weight[kHeld];
  i32x4 at[kHeld];
  if constexpr (kGroups > 0) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (j < per && slot_of(j) < len) {
        const int64_t row = row_of(slot_of(j));
        weight[j] = *reinterpret_cast<const f32x4*>(cache.weights + row);
        at[j] = *reinterpret_cast<const i32x4*>(cache.positions + row);
      }
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j < per && slot_of(j) + e < len) newest = max(newest, at[j][e]);
  } else {
    for (int s = tid; s < len; s += kSelectThreads) newest = max(newest, cache.positions[row_of(s)]);
  }
#pragma unroll
  for (int x = 1; x < 64; x *= 2) newest = max(newest, __shfl_xor(newest, x));
  if (lane == 0) sums[0][wave] = newest;
  i32x4* const own_bins = reinterpret_cast<i32x4*>(bins + (kBins - 2 - 2 * tid) * kCopies);  // of this thread's two digits
#pragma unroll
  for (int i = 0; i < kCopies / 2; ++i) own_bins[i] = (i32x4){0, 0, 0, 0};
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSelectWaves; ++i) newest = max(newest, sums[0][i]);
  auto key_of = [&](int position, float w) -> uint32_t {  // (no position is behind the newest: the difference fits)
    return position < p.sinks || (uint32_t)newest - (uint32_t)position < (uint32_t)p.recent ? 0xffffffffu : weight_key(w);
  };
  uint32_t key[kHeld][4];
  if constexpr (kGroups > 0) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) key[j][e] = slot_of(j) + e < len ? key_of(at[j][e], weight[j][e]) : 0;
  }
  // A few over the budget, as after single tokens: as many minima of (key, slot from behind) in place of the search, and the rows move at once.
  if constexpr (kGroups > 0) {
    if (const int drop = len - p.budget; drop <= kFewDropped) {
      __shared__ unsigned long long lowest[kFewDropped];
      __shared__ int dropped[kFewDropped];
      if (tid < kFewDropped) lowest[tid] = ~0ull;
      __syncthreads();
      unsigned long long own = 0;  // this thread's lowest that is still there
      auto next = [&]() __attribute__((always_inline)) {
        unsigned long long low = ~0ull;
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned long long of = (unsigned long long)key[j][e] << 32 | (uint32_t)~(slot_of(j) + e);
            if (j < per && slot_of(j) + e < len && of > own) low = min(low, of);
          }
        own = low;
      };
      next();  // (a slot's complement is above zero)
      for (int r = 0; r < drop; ++r) {
        uint32_t low = own >> 32;
#pragma unroll
        for (int x = 1; x < 64; x *= 2) low = min(low, (uint32_t)__shfl_xor((int)low, x));
        const bool mine = own >> 32 == low;
        unsigned long long some = __builtin_amdgcn_ballot_w64(mine);
        if (some & (some - 1)) {  // equal ones: the highest slot
          uint32_t slot = mine ? (uint32_t)own : ~0u;
#pragma unroll
          for (int x = 1; x < 64; x *= 2) slot = min(slot, (uint32_t)__shfl_xor((int)slot, x));
          some = __builtin_amdgcn_ballot_w64(mine && (uint32_t)own == slot);
        }
        if (lane == __builtin_ctzll(some)) atomicMin(&lowest[r], own);
        __syncthreads();
        const unsigned long long gone = lowest[r];
        if (tid == 0) dropped[r] = (int)~(uint32_t)gone;
        if (own == gone) next();
      }
      __syncthreads();
      // lane i: the i-th dropped slot, and the i-th one behind the budget
      const int gone = lane < drop ? dropped[lane] : 0;
      const bool frees = lane < drop && gone < p.budget;
      bool late = lane < drop;
      int rank = 0;
      for (int i = 0; i < drop; ++i) {
        late = late && dropped[i] != p.budget + lane;
        rank += dropped[i] < gone;
      }
      const unsigned long long lates = __builtin_amdgcn_ballot_w64(late);
      const int late_rank = __builtin_popcountll(lates & ((1ull << lane) - 1)), n = __builtin_popcountll(lates);
      for (int i = wave; i < n; i += kSelectWaves) {
        const int to_slot = __builtin_amdgcn_readlane(gone, __builtin_ctzll(__builtin_amdgcn_ballot_w64(frees && rank == i)));
        const int from_slot = p.budget + __builtin_ctzll(__builtin_amdgcn_ballot_w64(late && late_rank == i));
        const int64_t to = row_of(to_slot), from = row_of(from_slot);
        const bool held = cache.k_scales != nullptr;
        if (lane < 32) move_piece(lane < 16 ? cache.k : cache.v, held, to, from, lane & 15);
        if (held && (lane == 34 || lane == 35)) move_scales(lane == 34 ? cache.k_scales : cache.v_scales, to, from);
        if (lane == 32) cache.positions[to] = cache.positions[from];
        if (lane == 33) cache.weights[to] = cache.weights[from];
      }
      if (tid == 0) moves[0] = 0;
      return;
    }
  }
  // f(group, this lane's four keys) for the wave's groups, in order.  Slots behind the last one have the lowest key: they are never reached, since more slots are there than stay.
  auto each = [&](auto f) {
    if constexpr (kGroups > 0) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        if (j < per && (wave * per + j) * 256 < len) f(j, key[j]);
    } else {
      for (int j = 0; j < per && (wave * per + j) * 256 < len; ++j) {
        uint32_t k[4] = {0, 0, 0, 0};
        if (slot_of(j) < len) {
          const int64_t row = row_of(slot_of(j));
          const f32x4 w = *reinterpret_cast<const f32x4*>(cache.weights + row);
          const i32x4 q = *reinterpret_cast<const i32x4*>(cache.positions + row);
#pragma unroll
          for (int e = 0; e < 4; ++e) k[e] = slot_of(j) + e < len ? key_of(q[e], w[e]) : 0;
        }
        f(j, k);
      }
    }
  };

  // The key of rank `budget` from above, and how many keys equal to it stay.
  uint32_t prefix = 0;
  int need = p.budget;
#pragma unroll
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, width = digit == 2 ? 10 : 11;
    each([&](int, const uint32_t(&k)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (digit == 0 || (k[e] >> (shift + width)) == (prefix >> (shift + width)))
          atomicAdd(&bins[(k[e] >> shift & ((1 << width) - 1)) * kCopies + (lane & (kCopies - 1))], 1);
      }
    });
    __syncthreads();
    // from the largest digit down: a thread has two
    const int d0 = kBins - 1 - 2 * tid;
    int n0 = 0, n1 = 0;
#pragma unroll
    for (int i = 0; i < kCopies / 4; ++i) {
      const i32x4 low = own_bins[i], high = own_bins[kCopies / 4 + i];
      n1 += low[0] + low[1] + low[2] + low[3];
      n0 += high[0] + high[1] + high[2] + high[3];
    }
    int upto = n0 + n1, all;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int other = __shfl_up(upto, d);
      if (lane >= d) upto += other;
    }
    const int before = upto - n0 - n1 + waves_before(__builtin_amdgcn_readlane(upto, 63), sums[1 + digit], &all);
#pragma unroll
    for (int i = 0; i < kCopies / 2; ++i) own_bins[i] = (i32x4){0, 0, 0, 0};
    if (before < need && before + n0 >= need) {
      found[0] = d0;
      found[1] = need - before;
    } else if (before + n0 < need && before + n0 + n1 >= need) {
      found[0] = d0 - 1;
      found[1] = need - before - n0;
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    need = found[1];
    __syncthreads();  // found is read
  }

  // of the keys equal to it the first `need` stay
  int equal = 0, all;
  each([&](int, const uint32_t(&k)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) equal += __builtin_popcountll(__builtin_amdgcn_ballot_w64(k[e] == prefix));
  });
  const int equal_before = waves_before(equal, sums[4], &all);
  auto staying = [&](const uint32_t(&k)[4], int* equals, bool (&stays)[4]) {  // whether this lane's four stay
    const bool same[4] = {k[0] == prefix, k[1] == prefix, k[2] == prefix, k[3] == prefix};
#pragma unroll
    for (int e = 0; e < 4; ++e) stays[e] = k[e] > prefix;
    if (__builtin_amdgcn_ballot_w64(same[0] || same[1] || same[2] || same[3]) == 0) return;
    const Ranks r(same, lane);
#pragma unroll
    for (int e = 0; e < 4; ++e) stays[e] = stays[e] || (same[e] && *equals + r.at[e] < need);
    *equals += r.n;
  };
  // Freed ones of slots below the budget, kept ones of those behind it: a group is on either side, or, one of them, on both.
  int freed = 0, late = 0, equals = equal_before;
  uint32_t kept = 0;  // four bits for each group
  each([&](int j, const uint32_t(&k)[4]) {
    bool stays[4];
    staying(k, &equals, stays);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (kGroups > 0) kept |= (uint32_t)stays[e] << (4 * j + e);
    }
    // (the group with the budget inside is on both sides)
    const int s0 = (wave * per + j) * 256, inside = p.budget - s0 - 4 * lane;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (s0 < p.budget) freed += __builtin_popcountll(__builtin_amdgcn_ballot_w64(!stays[e] && e < inside));
      if (s0 + 256 > p.budget) late += __builtin_popcountll(__builtin_amdgcn_ballot_w64(stays[e] && e >= inside));
    }
  });
  int n_freed, n_late;
  int to = waves_before(freed, sums[5], &n_freed), from = waves_before(late, sums[0], &n_late);
  equals = equal_before;
  each([&](int j, const uint32_t(&k)[4]) {
    bool stays[4];
    if constexpr (kGroups > 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) stays[e] = kept >> (4 * j + e) & 1;
    } else {
      staying(k, &equals, stays);
    }
    const int s0 = (wave * per + j) * 256;
    if (s0 < p.budget) {
      bool frees[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) frees[e] = !stays[e] && slot_of(j) + e < p.budget;
      const Ranks r(frees, lane);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (frees[e]) moves[1 + to + r.at[e]] = slot_of(j) + e;
      to += r.n;
    }
    if (s0 + 256 > p.budget) {
      bool lates[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) lates[e] = stays[e] && slot_of(j) + e >= p.budget;
      const Ranks r(lates, lane);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lates[e]) moves[1 + p.most + from + r.at[e]] = slot_of(j) + e;
      from += r.n;
    }
  });
  // (as many as n_late: budget slots stay)
  if (p.most > kFewMoved) {
    if (tid == 0) moves[0] = n_freed;
  } else {
    __syncthreads();
    move_rows(cache, moves, p.most, b, hkv, tid & 15, tid >> 4, kSelectThreads / 16, n_freed);
  }
}

// Second kernel, where rows are many.
__global__ __launch_bounds__(256) void cache_move_kernel(const EvictParams p) {
  const int tid = threadIdx.x, item = blockIdx.y;
  const int32_t* const moves = p.moves + (int64_t)item * (1 + 2 * (int64_t)p.most);
  move_rows(p.cache, moves, p.most, item / p.cache.kv_heads, item % p.cache.kv_heads, tid & 15, blockIdx.x * 16 + (tid >> 4), gridDim.x * 16, moves[0]);
}

int64_t cache_evict_bytes(EvictParams& p) {
  const int64_t behind = p.cache.slots() - p.budget;
  p.most = (int)(behind < 0 ? 0 : behind < p.budget ? behind : p.budget);
  return (int64_t)p.cache.batch * p.cache.kv_heads * (1 + 2 * (int64_t)p.most) * 4;
}

hipError_t launch_cache_evict(EvictParams p, hipStream_t stream) {
  const int items = p.cache.batch * p.cache.kv_heads;
  const int64_t groups = (p.cache.slots() + 4 * kSelectThreads - 1) / (4 * kSelectThreads);  // for the longest sequence there may be
  void (*select)(const EvictParams) = groups <= 2 ? &cache_select_kernel<2> : groups <= 8 ? &cache_select_kernel<8> : &cache_select_kernel<0>;
  hipLaunchKernelGGL(select, dim3(items), dim3(kSelectThreads), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.most <= kFewMoved) return e;
  // about 4096 work-groups, none without a row to move if all are moved
  int wgs = (p.most + 15) / 16, few = 4096 / items;
  if (few < 1) few = 1;
  hipLaunchKernelGGL(cache_move_kernel, dim3(wgs < few ? wgs : few, items), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace fba
