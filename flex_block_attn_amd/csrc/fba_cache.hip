// What fills a paged cache and what makes room in it: gfx950.  Rows of 256 bytes are moved, 16 lanes to a row; bound by device memory, in small calls by the launch.
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

// Eviction, first kernel: which slots of a (sequence, kv head) stay.  A work-group of 1024 threads finds the budget-th largest key, 8 bits at a time by counting,
// and lists the freed slots below the budget and the kept slots behind it, in order.
//
// A slot's key orders as its weight does (NaN below everything, the two zeros alike); the slots that are held are above all of them.
namespace {
constexpr int kSelectThreads = 1024;
FBA_DEVICE uint32_t weight_key(float w) {
  if (w != w) return 0;
  uint32_t bits = __builtin_bit_cast(uint32_t, w);
  if (bits == 0x80000000u) bits = 0;
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
}  // namespace

__global__ __launch_bounds__(kSelectThreads) void cache_select_kernel(const EvictParams p) {
  const CacheView& cache = p.cache;
  __shared__ int counts[256], wave_sums[3][kSelectThreads / 64], found[2], newest_of[kSelectThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int hkv = blockIdx.x % cache.kv_heads, b = blockIdx.x / cache.kv_heads;
  int32_t* const moves = p.moves + (int64_t)blockIdx.x * (1 + 2 * (int64_t)p.most);
  const int len = cache.lengths[b];
  bool bad = !cache.holds(len);
  if (!bad)
    for (int i = tid; i < (len + (1 << cache.page_log2) - 1) >> cache.page_log2; i += kSelectThreads) bad |= cache.page_of(b, i << cache.page_log2) < 0;
  bad = __syncthreads_or(bad);
  if (tid == 0 && hkv == 0) p.lengths_out[b] = bad ? -1 : min(len, p.budget);
  if (bad || len <= p.budget) {
    if (tid == 0) moves[0] = 0;
    return;
  }
  auto row_of = [&](int slot) { return cache.row_of(cache.page_of(b, slot), hkv, slot); };

  int newest = -0x7fffffff - 1;
  for (int s = tid; s < len; s += kSelectThreads) newest = max(newest, cache.positions[row_of(s)]);
#pragma unroll
  for (int x = 1; x < 64; x *= 2) newest = max(newest, __shfl_xor(newest, x));
  if (lane == 0) newest_of[wave] = newest;
  __syncthreads();
  for (int i = 0; i < kSelectThreads / 64; ++i) newest = max(newest, newest_of[i]);
  auto key_of = [&](int slot) -> uint32_t {
    const int64_t row = row_of(slot);
    const int at = cache.positions[row];
    return at < p.sinks || (int64_t)at > (int64_t)newest - p.recent ? 0xffffffffu : weight_key(cache.weights[row]);
  };

  // the key of rank `budget` from above, and how many keys equal to it stay
  uint32_t prefix = 0;
  int need = p.budget;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelectThreads) counts[i] = 0;
    __syncthreads();
    for (int s = tid; s < len; s += kSelectThreads) {
      const uint32_t key = key_of(s);
      if (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&counts[key >> shift & 255], 1);
    }
    __syncthreads();
    if (wave == 0) {  // from the largest digit down: a lane has four
      int mine[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += mine[i] = counts[255 - 4 * lane - i];
      int upto = sum;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int other = __shfl_up(upto, d);
        if (lane >= d) upto += other;
      }
      int above = upto - sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (above < need && above + mine[i] >= need) {
          found[0] = 255 - 4 * lane - i;
          found[1] = need - above;
        }
        above += mine[i];
      }
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    need = found[1];
    __syncthreads();
  }

  // slots in order, 1024 at a time: equal keys stay while there is need, then freed slots and kept ones are numbered
  int equal_before = 0, freed_before = 0, late_before = 0;
  for (int s0 = 0; s0 < len; s0 += kSelectThreads) {
    const int s = s0 + tid;
    const uint32_t key = s < len ? key_of(s) : 0;
    auto rank = [&](bool on, int which, int* total) {  // of the threads with it in front of this one
      const unsigned long long ballot = __builtin_amdgcn_ballot_w64(on);
      if (lane == 0) wave_sums[which][wave] = __builtin_popcountll(ballot);
      __syncthreads();
      int before = 0, all = 0;
      for (int i = 0; i < kSelectThreads / 64; ++i) {
        before += i < wave ? wave_sums[which][i] : 0;
        all += wave_sums[which][i];
      }
      *total = all;
      return before + __builtin_popcountll(ballot & ((1ull << lane) - 1));
    };
    int n_equal, n_freed, n_late;
    const bool equal = s < len && key == prefix;
    const int at = rank(equal, 0, &n_equal);
    const bool kept = s < len && (key > prefix || (equal && equal_before + at < need));
    const bool freed = s < len && !kept && s < p.budget, late = kept && s >= p.budget;
    const int at_freed = rank(freed, 1, &n_freed), at_late = rank(late, 2, &n_late);
    if (freed) moves[1 + freed_before + at_freed] = s;
    if (late) moves[1 + p.most + late_before + at_late] = s;
    equal_before += n_equal;
    freed_before += n_freed;
    late_before += n_late;
    __syncthreads();
  }
  if (tid == 0) moves[0] = freed_before;  // as many as late_before: budget slots stay
}

// Second kernel: the i-th freed slot gets the i-th kept one from behind the budget, row, position and weight.
__global__ __launch_bounds__(256) void cache_move_kernel(const EvictParams p) {
  const CacheView& cache = p.cache;
  const int tid = threadIdx.x, c = tid & 15, item = blockIdx.y, hkv = item % cache.kv_heads, b = item / cache.kv_heads;
  const int32_t* const moves = p.moves + (int64_t)item * (1 + 2 * (int64_t)p.most);
  const int n = moves[0];
  for (int i = blockIdx.x * 16 + (tid >> 4); i < n; i += gridDim.x * 16) {
    const int to_slot = moves[1 + i], from_slot = moves[1 + p.most + i];
    const int64_t to = cache.row_of(cache.page_of(b, to_slot), hkv, to_slot), from = cache.row_of(cache.page_of(b, from_slot), hkv, from_slot);
    const u32x4 kr = *reinterpret_cast<const u32x4*>(cache.k + from * kRowBytes + c * 16), vr = *reinterpret_cast<const u32x4*>(cache.v + from * kRowBytes + c * 16);
    *reinterpret_cast<u32x4*>(cache.k + to * kRowBytes + c * 16) = kr;
    *reinterpret_cast<u32x4*>(cache.v + to * kRowBytes + c * 16) = vr;
    if (c == 0) cache.positions[to] = cache.positions[from];
    if (c == 1) cache.weights[to] = cache.weights[from];
  }
}

int64_t cache_evict_bytes(EvictParams& p) {
  const int64_t behind = p.cache.slots() - p.budget;
  p.most = (int)(behind < 0 ? 0 : behind < p.budget ? behind : p.budget);
  return (int64_t)p.cache.batch * p.cache.kv_heads * (1 + 2 * (int64_t)p.most) * 4;
}

hipError_t launch_cache_evict(EvictParams p, hipStream_t stream) {
  const int items = p.cache.batch * p.cache.kv_heads;
  hipLaunchKernelGGL(cache_select_kernel, dim3(items), dim3(kSelectThreads), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.most == 0) return e;
  // about 4096 work-groups, none without a row to move if all are moved
  int wgs = (p.most + 15) / 16, few = 4096 / items;
  if (few < 1) few = 1;
  hipLaunchKernelGGL(cache_move_kernel, dim3(wgs < few ? wgs : few, items), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace fba
