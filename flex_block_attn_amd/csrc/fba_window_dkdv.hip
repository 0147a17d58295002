// Backward of attention under a sliding window with sinks, dK and dV: gfx950, head_dim 128, bf16 or fp16 in / fp32 accumulate, no atomics.
//
//   S = Q K^T, dP = dO V^T;  P = exp2(c S - lse2[q]),  dS = P o (dP - delta[q]);  dV^T += dO^T P,  dK^T += Q^T dS
//
// Work-group = 128 keys of one (batch, kv head), four waves of 32 keys, lane = key; two work-groups on a compute unit.  K and V rows stay in registers as B operands; slabs
// of 32 query rows travel global -> LDS into a ring of four (Q | dO | lse2 | -delta) buffers, three steps ahead, and feed all four waves, by rows (S, dP) and transposed
// (dV, dK).  A step is 32 matrix instructions for a wave; two waves on a SIMD, of work-groups that know nothing of each other, cover each other's exponentials, fetches and
// waits, and what a work-group takes before its first and behind its last slab: a tile has few of them, its window's.
// (64 keys to a wave, one wave on a SIMD, as the kernel for block lists: half the LDS bytes, but nobody to cover the ends: 2351 us instead of 1880 for H24 S30720, window 1152 to
// both sides, 384 sinks, where the matrix pipe is busy 59 % of the time.)
//
// The rows that see a key tile are those from its window, and, of a tile with sinks, all behind (and in front of) it.  A work item is a tile with a part of the rows inside
// of the window, or of those outside; where a tile has more than one they leave fp32 sums, which a small kernel adds in order.  The last slab of a sequence is moved back to
// end with it (its first rows are masked then, they were in the slab before), so that no row behind the sequence is read.
#include <type_traits>

#include "fba_types.h"
#include "fba_window.h"
#include "fba_window_keys.h"

namespace fba {

namespace {

constexpr int kSlab = kWindowSlab;
constexpr int kSlabBytes = kSlab * kRowBytes;       // 8 KiB
constexpr int kStatBytes = 2 * kSlab * 4;           // lse2[32] | -delta[32]
constexpr int kStageBytes = 2 * kSlabBytes + kStatBytes;
constexpr int kRing = 4;
constexpr int kSmemBytes = kRing * kStageBytes;
constexpr int kPartFloats = 2 * kWindowTile * kHeadDim;  // dV tile, dK tile

template <int N>
using IC = std::integral_constant<int, N>;

}  // namespace

template <typename T>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(2, 2))) void window_dkdv_kernel(const WindowParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using x8 = x8_of<T>;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int index = window_item(blockIdx.x, p.chunk);
  if (index >= p.items) return;
  const KeyItem item = key_item(p, index);
  const RowSlabs& slabs = item.slabs;
  const int b = item.b, hkv = item.hkv, group = p.Hq / p.Hkv, len = item.len, rows = item.rows, n = item.n, key0 = item.key0, wkey0 = key0 + 32 * wave;
  const bool in_parts = item.in_parts;
  float* const place = p.parts + item.place * kPartFloats;

  if (n == 0) {
    if (in_parts) {
      f32x4* out = reinterpret_cast<f32x4*>(place) + tid;
      for (int i = 0; i < kPartFloats / 4 / 256; ++i) out[i * 256] = (f32x4){0.f, 0.f, 0.f, 0.f};
    } else {
      for (int i = tid >> 4; i < kWindowTile && key0 + i < p.Skv; i += 16) {
        *reinterpret_cast<u32x4*>(p.dk.ptr + b * p.dk.batch + hkv * p.dk.head + (int64_t)(key0 + i) * p.dk.row + (tid & 15) * 16) = (u32x4){0, 0, 0, 0};
        *reinterpret_cast<u32x4*>(p.dv.ptr + b * p.dv.batch + hkv * p.dv.head + (int64_t)(key0 + i) * p.dv.row + (tid & 15) * 16) = (u32x4){0, 0, 0, 0};
      }
    }
    return;
  }

  // K and V rows of the wave as B operands: lane holds key l32, d = 16 ks + 8 h .. +7 (keys behind the last: that one, they are masked)
  x8 kreg[8], vreg[8];
  {
    const int key = min(wkey0 + l32, len - 1);
    const char* const kp = p.k.ptr + b * p.k.batch + hkv * p.k.head + (int64_t)key * p.k.row + 16 * h;
    const char* const vp = p.v.ptr + b * p.v.batch + hkv * p.v.head + (int64_t)key * p.v.row + 16 * h;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      kreg[ks] = *reinterpret_cast<const x8*>(kp + 32 * ks);
      vreg[ks] = *reinterpret_cast<const x8*>(vp + 32 * ks);
    }
  }

  // Slab s_begin + t is the t-th; requests run ahead of the arithmetic.  The common step, to the next slab of the same head, is a few additions; everything else (the next
  // head, the gap of rows inside, the last slab, the end) is worked out anew.
  struct At {
    int row0, row_min;  // the slab's first row, the first one that counts
  };
  const int tail = max(0, rows - kSlab);  // where the last slab of the rows begins
  int g_next = item.s_begin / slabs.n, i_next = item.s_begin % slabs.n, left = n;  // the next slab, and how many there are with it
  int steps = 0;                  // common steps from it on
  At next{0, 0};
  const char *q_next = p.q.ptr + b * p.q.batch + (int64_t)hkv * group * p.q.head, *d_next = p.d_o.ptr + b * p.d_o.batch + (int64_t)hkv * group * p.d_o.head;
  const char* st_next = reinterpret_cast<const char*>(p.lse + ((int64_t)b * p.Hq + hkv * group) * p.Sq);
  const int64_t q_step = (int64_t)p.q.row * kSlab, d_step = (int64_t)p.d_o.row * kSlab;
  int g_of = 0, row_of = 0;  // where the pointers are
  auto settle = [&]() __attribute__((always_inline)) {
    if (i_next >= slabs.n) {
      i_next = 0;
      ++g_next;
    }
    const bool there = left > 0;  // past the last one: that one again, into a buffer that nobody reads any more
    const int g = there ? g_next : g_of, slab = there ? slabs.at(i_next) : 0;
    if (there) next = At{min(slab * kSlab, tail), slab * kSlab};
    q_next += (g - g_of) * p.q.head + (int64_t)(next.row0 - row_of) * p.q.row;
    d_next += (g - g_of) * p.d_o.head + (int64_t)(next.row0 - row_of) * p.d_o.row;
    st_next += ((int64_t)(g - g_of) * p.Sq + next.row0 - row_of) * 4;
    g_of = g;
    row_of = next.row0;
    // slabs in a row that are not the last one of the rows
    const int end = i_next < slabs.cut ? min(slabs.cut, slabs.n) : slabs.n;
    steps = there ? max(0, min(min(end - 1 - i_next, rows / kSlab - 1 - slab), left - 1)) : 0;
  };
  auto advance = [&]() __attribute__((always_inline)) {
    --left;
    ++i_next;
    if (steps > 0) {
      --steps;
      next.row0 += kSlab;
      next.row_min += kSlab;
      row_of += kSlab;
      q_next += q_step;
      d_next += d_step;
      st_next += kSlab * 4;
    } else {
      settle();
    }
  };
  settle();

  const KeyMask mask(p, item, wkey0);

  uint32_t q_off[2], d_off[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int row = 8 * wave + 4 * g + (lane >> 4), from = min(row, rows - 1);  // (fewer rows than a slab has: the last one again)
    const uint32_t chunk = ((lane & 15) ^ swz(row)) << 4;
    q_off[g] = from * p.q.row + chunk;
    d_off[g] = from * p.d_o.row + chunk;
  }
  const uint32_t lds0 = lds_addr(smem), wave_dst = wave * 8 * kRowBytes;
  // statistics: lanes 0..31 fetch lse2[row0 + l], lanes 32..63 -delta[row0 + l - 32], which is behind all lse2
  const uint32_t stat_off = (uint32_t)(h * ((const char*)p.neg_delta - (const char*)p.lse)) + (uint32_t)min(l32, rows - 1) * 4;
  auto request = [&](int i, uint32_t dst) __attribute__((always_inline)) {  // one of five copies
    if (i < 2) dma16(dst + wave_dst + i * 4 * kRowBytes, q_next, q_off[i]);
    else if (i < 4) dma16(dst + kSlabBytes + wave_dst + (i - 2) * 4 * kRowBytes, d_next, d_off[i - 2]);
    else dma4(dst + 2 * kSlabBytes, st_next, stat_off);  // (each wave the same 256 bytes)
  };
  At at[kRing];
#pragma unroll
  for (int j = 0; j < kRing - 1; ++j) {
    at[j] = next;
#pragma unroll
    for (int i = 0; i < 5; ++i) request(i, lds0 + j * kStageBytes);
    advance();
  }
  wait_vmem<0>();
  __syncthreads();
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) { pin(kreg[ks]); pin(vreg[ks]); }

  // Per-lane fetch addresses; operand steps and column blocks only move the 16-byte chunk inside a 256-byte row, by an exclusive-or.
  static_assert(kStageBytes % 256 == 0 && kSlabBytes % 256 == 0, "the exclusive-ors below touch bits 5..7");
  const LdsPtr lds = lds_ptr(smem);
  RowMajorOffsets rm;
  rm.init(lane);
  TransposedOffsets tr;
  tr.init(lane);
  const LdsPtr q_base0 = lds + rm.rd[0], t_base0 = lds + tr.rd[0][0], st_ptr0 = lds + 2 * kSlabBytes + 16 * h;
  auto flip = [](LdsPtr ptr, uint32_t bits) { return (LdsPtr)(uintptr_t)((uint32_t)(uintptr_t)ptr ^ bits); };
  const float c = p.scale_log2e;
  f32x16 acc_k[4], acc_v[4];
#pragma unroll
  for (int mb = 0; mb < 4; ++mb)
#pragma unroll
    for (int r = 0; r < 16; ++r) { acc_k[mb][r] = 0.f; acc_v[mb][r] = 0.f; }

  // Step t (t % 4 == R): S_t, dP_t | P_t, dS_t | dV, dK.  Slab t+3 is requested into the buffer of slab t-1, between the first matrix instructions; behind the step slab t+1
  // must have landed (and has, as slab t+2): what step t requested may still fly.
  auto step = [&](int so) __attribute__((always_inline)) {
    const uint32_t into = lds0 + (so == 0 ? 3 * kStageBytes : so - kStageBytes);
    at[3] = next;
    const LdsPtr q_base = q_base0 + so, t_base = t_base0 + so, st_ptr = st_ptr0 + so;
    {
      f32x16 s, dp;
      // accumulator element 4g + e of half-wave h is row 8g + 4h + e of the slab; dP starts from -delta of its row
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 d4 = lds_read_f32x4(st_ptr + 4 * kSlab + 32 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) { s[4 * g + e] = 0.f; dp[4 * g + e] = d4[e]; }
      }
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        s = Elem<T>::mfma32(read_b128<T>(flip(q_base, 32u * ks)), kreg[ks], s);
        dp = Elem<T>::mfma32(read_b128<T>(flip(q_base, 32u * ks) + kSlabBytes), vreg[ks], dp);
        if (ks < 5) request(ks, into);
        if (ks & 1) __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 l4 = lds_read_f32x4(st_ptr + 32 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float pv = fast_exp2(__builtin_fmaf(s[4 * g + e], c, -l4[e]));
          s[4 * g + e] = pv;
          dp[4 * g + e] = pv * dp[4 * g + e];
        }
      }
      if (!mask.whole(at[0].row0, at[0].row_min)) mask.apply(s, dp, at[0].row0, at[0].row_min, lane);
      // rounded to T as the matrix instructions take them
      x8 pk[2], dsk[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        pk[j] = narrow8<T>(s, j);
        dsk[j] = narrow8<T>(dp, j);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) {
          const LdsPtr t0 = flip(t_base, (uint32_t)(mb << 6)) + 16 * j * kRowBytes, t1 = flip(t_base, (uint32_t)(mb << 6 | 32)) + (16 * j + 8) * kRowBytes;
          acc_v[mb] = Elem<T>::mfma32(read_tr8<T>(t0 + kSlabBytes, t1 + kSlabBytes), pk[j], acc_v[mb]);
          acc_k[mb] = Elem<T>::mfma32(read_tr8<T>(t0, t1), dsk[j], acc_k[mb]);
          if (mb & 1) __builtin_amdgcn_sched_barrier(0);
        }
    }
    advance();
    at[0] = at[1]; at[1] = at[2]; at[2] = at[3];
    wait_vmem<5>();
    __syncthreads();
  };
  for (int t = 0, so = 0; t < n; ++t) {
    step(so);
    so = so == 3 * kStageBytes ? 0 : so + kStageBytes;
  }
  wait_vmem<0>();
  __syncthreads();  // no copy is writing LDS any more, and everybody is done with the ring

  auto finish = [&](const f32x16(&acc)[4], const Strided& out, int which, float scale) __attribute__((always_inline)) {
    if (in_parts) {
      float* const row = place + which * (kWindowTile * kHeadDim) + (32 * wave + l32) * kHeadDim + 4 * h;
#pragma unroll
      for (int mb = 0; mb < 4; ++mb)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(row + 32 * mb + 8 * g) = (f32x4){acc[mb][4 * g + 0], acc[mb][4 * g + 1], acc[mb][4 * g + 2], acc[mb][4 * g + 3]};
    } else {
      store_tile<T>(smem + wave * 2 * kSlabBytes + which * kSlabBytes, acc, scale, out.ptr + b * out.batch + hkv * out.head + (int64_t)wkey0 * out.row, out.row, lane, p.Skv - wkey0);
    }
  };
  finish(acc_v, p.dv, 0, 1.f);
  finish(acc_k, p.dk, 1, p.scale);
}

// Sums the parts of the tiles that have several, in order.  A work-group per 8 rows, 32 threads to a row of dV or dK.
template <typename T>
__global__ __launch_bounds__(256) void window_sum_kernel(const WindowParams p) {
  const int c4 = (threadIdx.x & 31) * 4, groups = p.key_tile / 8, r = (blockIdx.x % groups) * 8 + (threadIdx.x >> 5);
  const int which = blockIdx.x / groups % 2;  // dV, dK
  const int tiles = p.band_parts > 1 ? p.tiles : p.sink_tiles, kt = blockIdx.x / (2 * groups) % tiles, bh = blockIdx.x / (2 * groups) / tiles;
  const int key = kt * p.key_tile + r;
  if (key >= p.Skv) return;
  const int hkv = bh % p.Hkv, b = bh / p.Hkv, parts = p.band_parts + (kt < p.sink_tiles ? p.sink_parts : 0);
  const float* src = p.parts + part_place(p, bh, kt, false, 0) * part_floats(p) + which * (p.key_tile * kHeadDim) + r * kHeadDim + c4;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int q = 0; q < parts; q += 8) {
    f32x4 of[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (q + i < parts) of[i] = *reinterpret_cast<const f32x4*>(src + (int64_t)(q + i) * part_floats(p));
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (q + i < parts) acc += of[i];
  }
  const Strided& out = which ? p.dk : p.dv;
  const float s = which ? p.scale : 1.f;
  *reinterpret_cast<x4_of<T>*>(out.ptr + b * out.batch + hkv * out.head + (int64_t)key * out.row + c4 * 2) = narrow4<T>(acc[0] * s, acc[1] * s, acc[2] * s, acc[3] * s);
}

// How the rows of a key tile are cut into items.
//   Inside of the window: into several where the tiles alone leave half of the compute units idle and more, so that two items come to each, with 16 slabs (tiles of 32 keys: 8)
//   to an item at least.  dQ, dK and dV, one item / several, H4/1 S2048 window 1024 (64 tiles of 32): 95 / 56 us, H8/2 S1024 window 512: 67 / 47, B2 H8/1 S1024, 400 to either
//   side: 136 / 70.
//   Outside (tiles with sinks): into as many as are about as long as the items inside, for the longest sequence there may be, of 16 slabs (tiles of 32 keys: 8) at least.
//   No more items outside than twice what is on the GPU at once (two to a compute unit), and one for each tile: every part leaves 128 KiB of sums, which are written and read again.
//   Backward, cut by length alone / once, twice, four and eight times what is on the GPU, H24 S30720: window 128, 4096 sinks 7296 / 5249, 5136, 5169, 5317 us (6.1 GB of sums / 0.2, 0.3, 0.4,
//   0.7), 1024 sinks 2390 / 2007, 1944, 1948, 2063; 1152 to either side, 4096 sinks 7919 / 7478, 7511, 7513, 7659, and with 384, which twice leaves as they are, 3418 / 3485 with once.
constexpr int kLeastSlabs = 16, kLeastSlabsFew = 8;
constexpr int64_t kSinkRounds = 2;
int64_t plan_window_dkdv(WindowParams& p, int compute_units) {
  p.key_tile = window_keys_few(p, compute_units) ? 32 : kWindowTile;
  p.tiles = (p.Skv + p.key_tile - 1) / p.key_tile;
  p.sink_tiles = (p.sinks + p.key_tile - 1) / p.key_tile;
  p.sink_parts = 0;
  const int least = p.key_tile == 32 ? kLeastSlabsFew : kLeastSlabs;
  const int shift = p.lengths != nullptr ? 0 : p.Skv - p.Sq, group = p.Hq / p.Hkv;
  int64_t outside = 0;
  for (int kt = 0; kt < p.sink_tiles; ++kt) {
    const int64_t n = (int64_t)row_slabs(kt * p.key_tile, p.key_tile, p.Skv, p.Sq, shift, p.window, p.sinks, p.causal != 0, true).n * group;
    if (n > outside) outside = n;
  }
  int64_t inside = (int64_t)row_slabs(p.tiles / 2 * p.key_tile, p.key_tile, p.Skv, p.Sq, shift, p.window, p.sinks, p.causal != 0, false).n * group;
  const int64_t items = (int64_t)p.B * p.Hkv * p.tiles;
  int64_t parts = 2 * items > compute_units ? 1 : 2 * compute_units / items < inside / least ? 2 * compute_units / items : inside / least;
  if (parts > 8) parts = 8;
  p.band_parts = parts < 2 ? 1 : (int)parts;
  inside /= p.band_parts;
  if (inside < least) inside = least;
  if (outside == 0) {
    p.sink_tiles = 0;
  } else {
    parts = (outside + inside - 1) / inside;
    const int64_t sink_tiles = (int64_t)p.B * p.Hkv * p.sink_tiles, most = (kSinkRounds * 2 * compute_units + sink_tiles - 1) / sink_tiles;
    if (parts > most) parts = most;
    p.sink_parts = (int)(parts > 64 ? 64 : parts);
  }
  return part_place(p, (int64_t)p.B * p.Hkv, 0, false, 0) * part_floats(p) * 4;
}

hipError_t launch_window_dkdv(WindowParams p, bool half, hipStream_t stream) {
  p.tiles = (p.Skv + p.key_tile - 1) / p.key_tile;
  p.sink_items = p.B * p.Hkv * p.sink_tiles * p.sink_parts;
  p.items = p.sink_items + p.B * p.Hkv * p.tiles * p.band_parts;
  p.chunk = window_chunk(p.items);
  hipError_t e;
  if (p.key_tile == 32) {
    e = launch_window_few_dkdv(p, half, stream);
  } else {
    void (*fn)(const WindowParams) = half ? &window_dkdv_kernel<_Float16> : &window_dkdv_kernel<__bf16>;
    if ((e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes)) != hipSuccess) return e;
    hipLaunchKernelGGL(fn, dim3(window_grid(p.items, p.chunk)), dim3(256), kSmemBytes, stream, p);
    e = hipGetLastError();
  }
  const int summed = p.band_parts > 1 ? p.tiles : p.sink_tiles;
  if (e != hipSuccess || summed == 0) return e;
  hipLaunchKernelGGL((half ? &window_sum_kernel<_Float16> : &window_sum_kernel<__bf16>), dim3(p.B * p.Hkv * summed * (p.key_tile / 4)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace fba
