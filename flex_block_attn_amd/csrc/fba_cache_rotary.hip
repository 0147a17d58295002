// New tokens into a paged cache with the rotation on the way, into 4 bits with it or without, and rows of a cache read back as dense tensors: gfx950.
//
// Sixteen lanes have a row, as in fba_cache.hip.  Bound by device memory, in small calls by the launch.
#include "fba_cache.h"
#include "fba_cache_held.h"
#include "fba_turn.h"

namespace fba {

// Work-groups 0 .. batch - 1 work out the new lengths; behind them sixteen lanes have a part of a token's heads, so that sines and cosines are worked out once for all of them:
// first the kv heads, K and V together, then those of q.
//
// What becomes 4 bits is what 64 bits say: an error in the last of 32 would, next to a border between two codes, be one of a whole code.  It is turned in 32, and again in 64 where a
// code or a scale is so near to a border that it could depend on it, which a wave comes to once in some hundred rows, or where angles are zero.  6 heads of 2 x 30720 tokens: 53 us for what
// a copy takes 49 for (without the rotation 50), and 65 right behind a read that has left as much to be written out (64 bits throughout: 71).
template <typename T, bool kHeld>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(4))) void cache_append_rotary_kernel(const AppendRotaryParams p) {
  const AppendParams& a = p.append;
  const CacheView& cache = a.cache;
  const int tid = threadIdx.x, c = tid & 15;
  // how many tokens sequence b gets: -1 where its length or count makes no sense or there is no room
  auto tokens_of = [&](int b, int* len) {
    *len = cache.lengths[b];
    const int n = a.counts != nullptr ? a.counts[b] : a.tokens;
    return cache.holds(*len) && n >= 0 && n <= a.tokens && cache.holds((int64_t)*len + n) ? n : -1;
  };
  if ((int)blockIdx.x < cache.batch) {
    const int b = blockIdx.x;
    int len;
    const int n = tokens_of(b, &len);
    bool bad = n < 0;
    if (n > 0)
      for (int i = (len >> cache.page_log2) + tid; i <= (len + n - 1) >> cache.page_log2; i += 256) bad |= cache.page_of(b, i << cache.page_log2) < 0;
    const bool any = __syncthreads_or(bad);
    if (tid == 0) a.lengths_out[b] = any ? -1 : len + n;
    return;
  }
  const uint32_t tokens = (uint32_t)cache.batch * (uint32_t)a.tokens;
  const uint32_t unit = (blockIdx.x - (uint32_t)cache.batch) * 16 + (tid >> 4), part = unit / tokens, at = unit - part * tokens;
  if (part >= p.parts) return;
  const int b = at / (uint32_t)a.tokens, t = at - (uint32_t)b * (uint32_t)a.tokens;
  int len;
  const int n = tokens_of(b, &len);
  const int h0 = part * p.per, end = min(h0 + (int)p.per, cache.kv_heads + p.heads);
  if (t >= n && (n >= 0 ? end <= cache.kv_heads : p.heads == 0)) return;  // behind the sequence's last one, and no q
  const int position = (int)((uint32_t)(a.first != nullptr ? a.first[b] : len) + (uint32_t)t);
  const int page = t < n ? cache.page_of(b, len + t) : -1;
  // Rows of K and V, a head or two ahead (4 bits have no registers for two at four waves on a SIMD).  Every round of the loop issues as many loads and stores, whatever its lanes have, so
  // that none waits for stores of the round before: behind the last head it is fetched again.
  constexpr int kAhead = kHeld ? 1 : 2;
  const char* const k_from = a.k.ptr + b * a.k.batch + (int64_t)t * a.k.row + c * 16;
  const char* const v_from = a.v.ptr + b * a.v.batch + (int64_t)t * a.v.row + c * 16;
  const int kv_end = page >= 0 ? min(end, cache.kv_heads) : h0;
  x8_of<T> k_rows[kAhead], v_rows[kAhead];
  auto fetch = [&](int h, int i) {
    h = min(h, kv_end - 1);
    k_rows[i] = *reinterpret_cast<const x8_of<T>*>(k_from + h * a.k.head);
    v_rows[i] = *reinterpret_cast<const x8_of<T>*>(v_from + h * a.v.head);
  };
  if (h0 < kv_end)
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch(h0 + i, i);
  Turn turn;
  const bool turns = p.rotation.turns != nullptr, interleaved = p.rotation.interleaved != 0;
  const Columns columns(p.rotation, c);
  turn.on = false;
  if (turns) turn.init(p.rotation, columns, b, t, position);
  const int64_t row0 = cache.row_of(page, h0, len + t), rows = 1ll << cache.page_log2;  // (a head's rows of a page are one behind the other)
  int64_t to = row0;
  for (int h1 = h0; h1 < kv_end; h1 += kAhead)
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = h1 + i;
      if (i > 0 && h >= kv_end) break;
      x8_of<T> kr = k_rows[i];
      const x8_of<T> vr = v_rows[i];
      fetch(h + kAhead, i);
      if constexpr (kHeld) {
        float kf[8], vf[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          kf[e] = (float)kr[e];
          vf[e] = (float)vr[e];
        }
        To4Bits<T> k4, v4;
        if (turns) {
          const x8_of<T> y = paired<T>(kr, turn, interleaved);
          float off = 0.f;  // of what is turned in 32 bits: less than 2^-21 (|a| + |b|), and 2^-124 for what is too small for them
#pragma unroll
          for (int e = 0; e < 8; ++e) off = fmaxf(off, fabsf(kf[e]));
          off += interleaved ? off : __shfl(off, turn.from);
          off = turn.on && off > 0.f ? off * 0x1p-21f + 0x1p-124f : 0.f;
          if (turn.on) {
#pragma unroll
            for (int e = 0; e < 8; ++e) kf[e] = kf[e] * turn.own[e] + (float)y[e] * turn.other[e];
          }
          k4.template hold<true>(kf, __builtin_bit_cast(float, of_group(bits_of(off))));
          if (__builtin_amdgcn_ballot_w64(!k4.sure) != 0) {
            if (turn.on) {
              int seldom = c, where = t, stands = position;  // (nothing of this is worked out ahead, in registers that the loop would go without)
              pin(seldom);
              pin(where);
              pin(stands);
              const Columns again(p.rotation, seldom);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                uint64_t phase[1];
                phases_of(p.rotation, again.pair(p.rotation, e), b, where, stands, phase);
                double sin, cos;
                sincos_of(phase[0], &sin, &cos);
                kf[e] = cut((double)(float)kr[e] * cos + (double)(float)y[e] * (again.leads(p.rotation, e) ? -sin : sin));
                __builtin_amdgcn_sched_barrier(0);
              }
            }
            k4.template hold<false>(kf, 0.f);
          }
        } else {
          k4.template hold<false>(kf, 0.f);
        }
        v4.template hold<false>(vf, 0.f);
        *reinterpret_cast<uint32_t*>(cache.k + to * kHeldRowBytes + c * 4) = k4.codes;
        *reinterpret_cast<uint32_t*>(cache.v + to * kHeldRowBytes + c * 4) = v4.codes;
        cache.k_scales[to * 4 + (c >> 2)] = (uint8_t)k4.scale;  // (by all four lanes of a group)
        cache.v_scales[to * 4 + (c >> 2)] = (uint8_t)v4.scale;
      } else {
        if (turns) kr = turned<T>(kr, turn, interleaved);
        *reinterpret_cast<x8_of<T>*>(cache.k + to * kRowBytes + c * 16) = kr;
        *reinterpret_cast<x8_of<T>*>(cache.v + to * kRowBytes + c * 16) = vr;
      }
      to += rows;
    }
  // positions and weights, sixteen heads at a time
  if (cache.positions != nullptr || cache.weights != nullptr)
    for (int h = h0 + c; h < kv_end; h += 16) {
      const int64_t row = row0 + (h - h0) * rows;
      if (cache.positions != nullptr) cache.positions[row] = position;
      if (cache.weights != nullptr) cache.weights[row] = a.weights != nullptr ? a.weights[((int64_t)b * cache.kv_heads + h) * a.tokens + t] : 0.f;
    }
  const char* const from = p.q.ptr + b * p.q.batch + (int64_t)t * p.q.row + c * 16;
  char* const q_to = p.q_out.ptr + b * p.q_out.batch + (int64_t)t * p.q_out.row + c * 16;
  for (int h = max(h0 - cache.kv_heads, 0); h < end - cache.kv_heads; ++h) {
    x8_of<T> r = *reinterpret_cast<const x8_of<T>*>(from + h * p.q.head);
    if (turns) r = turned<T>(r, turn, interleaved);
    if (n < 0)
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = (T)__builtin_nanf("");
    *reinterpret_cast<x8_of<T>*>(q_to + h * p.q_out.head) = r;
  }
}

hipError_t launch_cache_append_rotary(AppendRotaryParams p, bool half, hipStream_t stream) {
  const int64_t tokens = (int64_t)p.append.cache.batch * p.append.tokens;
  const int heads = p.append.cache.kv_heads + p.heads;
  p.parts = rotary_parts(tokens, heads);
  p.per = (heads + p.parts - 1) / p.parts;
  p.parts = (heads + p.per - 1) / p.per;
  const int64_t units = tokens * p.parts;
  const bool held = p.append.cache.k_scales != nullptr;
  void (*fn)(const AppendRotaryParams) = held ? (half ? &cache_append_rotary_kernel<_Float16, true> : &cache_append_rotary_kernel<__bf16, true>)
                                              : (half ? &cache_append_rotary_kernel<_Float16, false> : &cache_append_rotary_kernel<__bf16, false>);
  hipLaunchKernelGGL(fn, dim3((uint32_t)(p.append.cache.batch + (units + 15) / 16)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

// Rows of a (sequence, kv head) to a dense tensor, kReadRows slots to a work-group: zeros behind the sequence's length, and no numbers where its length or a page makes no sense.
template <typename T, bool kHeld>
__global__ __launch_bounds__(256) void cache_read_kernel(const ReadParams p) {
  const CacheView& cache = p.cache;
  const int tid = threadIdx.x, c = tid & 15;
  const uint32_t bh = blockIdx.x / p.chunks, chunk = blockIdx.x - bh * p.chunks;
  const int b = bh / (uint32_t)cache.kv_heads, h = bh - (uint32_t)b * (uint32_t)cache.kv_heads;
  const int len = cache.lengths[b];
  const bool bad = !cache.holds(len);
  constexpr int kRows = kReadRows / 16;
  int64_t row[kRows];
  bool there[kRows], none[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int slot = p.first + (int)chunk * kReadRows + 16 * i + (tid >> 4);
    there[i] = !bad && slot < len && slot < p.first + p.slots;
    const int page = there[i] ? cache.page_of(b, slot) : 0;
    none[i] = bad || page < 0;
    row[i] = there[i] && page >= 0 ? cache.row_of(page, h, slot) : 0;
    there[i] = there[i] && page >= 0;
  }
  x8_of<T> k[kRows], v[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) k[i][e] = v[i][e] = (T)(none[i] ? __builtin_nanf("") : 0.f);
    if (!there[i]) continue;
    if constexpr (kHeld) {
      const uint32_t k_codes = *reinterpret_cast<const uint32_t*>(cache.k + row[i] * kHeldRowBytes + c * 4), v_codes = *reinterpret_cast<const uint32_t*>(cache.v + row[i] * kHeldRowBytes + c * 4);
      k[i] = from_4_bits<T>(k_codes, scale_of(cache.k_scales[row[i] * 4 + (c >> 2)]));
      v[i] = from_4_bits<T>(v_codes, scale_of(cache.v_scales[row[i] * 4 + (c >> 2)]));
    } else {
      k[i] = *reinterpret_cast<const x8_of<T>*>(cache.k + row[i] * kRowBytes + c * 16);
      v[i] = *reinterpret_cast<const x8_of<T>*>(cache.v + row[i] * kRowBytes + c * 16);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int t = (int)chunk * kReadRows + 16 * i + (tid >> 4);
    if (t >= p.slots) break;
    *reinterpret_cast<x8_of<T>*>(p.k.ptr + b * p.k.batch + h * p.k.head + (int64_t)t * p.k.row + c * 16) = k[i];
    *reinterpret_cast<x8_of<T>*>(p.v.ptr + b * p.v.batch + h * p.v.head + (int64_t)t * p.v.row + c * 16) = v[i];
  }
}

hipError_t launch_cache_read(ReadParams p, bool half, hipStream_t stream) {
  p.chunks = (uint32_t)((p.slots + kReadRows - 1) / kReadRows);
  const bool held = p.cache.k_scales != nullptr;
  void (*fn)(const ReadParams) = held ? (half ? &cache_read_kernel<_Float16, true> : &cache_read_kernel<__bf16, true>)
                                      : (half ? &cache_read_kernel<_Float16, false> : &cache_read_kernel<__bf16, false>);
  hipLaunchKernelGGL(fn, dim3((uint32_t)p.cache.batch * (uint32_t)p.cache.kv_heads * p.chunks), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace fba
