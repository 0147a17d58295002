// Attention of one new token per sequence over a paged cache in 4 bits: gfx950, head_dim 128, bf16 or fp16 / fp32 accumulate.
//
// The same as over 16 bits (fba_cache_attend.hip: shares, softmax, sums, P in two parts), over the values that the 4 bits stand for, which the type holds exactly.  A slot is 136 bytes
// instead of 512.
//
// A lane's sixteen bytes of a K row are 32 columns of one scale, and become the A operand of four matrix instructions as they are, one conversion for two values, scale included: which
// columns an instruction sums is free as long as K and Q agree, so lane (row l16, group g) gives columns 32 g + 8 ks .. + 7 to instruction ks.  No LDS, and 16 rows are 1 KiB that a
// wave loads at once.  V is summed over slots, which are rows: decoded values go through an LDS tile of the wave's own, and come back transposed.  The next tile's K is requested behind
// the scores, its V behind its decoding.
//
// 8 streams of 115200 slots, 16 heads on 4: 501 MB in 84 us, 6.0 TB/s.  Its loads alone take 78 (72 without the scales, whose bytes are 6 % of all and come 64 at a time); what is left is
// that loads, some 200 vector instructions (23.1 M counted, 115200 tiles), 24 matrix instructions and 16 KiB through LDS for each tile, the vector unit busy for 56 % of the time and the
// matrix unit for 26, do not hide behind each other entirely.  Without LDS (wrong results) 78 us.  Measured and not kept: four waves on a SIMD, whose 128 registers spill (94); two, with
// two to four tiles ahead (88 to 91); each four columns of a matrix instruction with tiles of their own, for groups of four heads, so that softmax is a quarter of the work (91, and 44
// instead of 32 us for 64 short sequences); eight waves in step (94); a tile's scales in one load, transposed across the wave (91); LDS rows padded instead of swizzled (86).
// Scores cost 32 ragged sequences, 24 heads on 6, 52 -> 72 us: 27 MB written, read again and added up.  Stored in every lane, a tile's heads one behind the other, 71; the kernel of 16 bits,
// which shares their layout, was 2 us of 102 slower then, and it was not kept.
#include "fba_cache_attend.h"
#include "fba_cache_held.h"

namespace fba {

namespace {

// 16 bytes of a lane, of a base that every lane has alike.
FBA_DEVICE u32x4 load_codes(const char* pool, int64_t row, uint32_t off) {
  typedef const __attribute__((address_space(1))) char* GlobalPtr;
  return __builtin_nontemporal_load(reinterpret_cast<const __attribute__((address_space(1))) u32x4*>((GlobalPtr)(pool + row * kHeldRowBytes) + off));
}

// A byte of each.
FBA_DEVICE uint32_t load_scale(const uint8_t* pool, int64_t row, uint32_t off) {
  typedef const __attribute__((address_space(1))) uint8_t* GlobalPtr;
  return __builtin_nontemporal_load((GlobalPtr)(pool + row * 4) + off);
}

}  // namespace

// kHeadTiles: query heads of a work-group, in sixteens.
template <typename T, int kHeadTiles, bool kScores>
__global__ __attribute__((amdgpu_flat_work_group_size(64 * kWaves, 64 * kWaves), amdgpu_waves_per_eu(kHeadTiles == 1 ? kResident4 : 2, kHeadTiles == 1 ? kResident4 : 2))) void cache_attend4_kernel(
    const AttendParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];  // [waves][V tile], and the sums at a sequence's end
  using x8 = x8_of<T>;
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const CacheView& cache = p.cache;
  const int group = p.heads / cache.kv_heads;
  const int hkv = blockIdx.y / p.head_tiles, head0 = hkv * group + blockIdx.y % p.head_tiles * (16 * kHeadTiles);
  const int heads = min(16 * kHeadTiles, (hkv + 1) * group - head0);

  Share share;
  if (!find_share(p, tid, lane, wave, &share)) return;
  const int w = share.w, end = __builtin_amdgcn_readfirstlane(share.end);
  int tile = __builtin_amdgcn_readfirstlane(share.tile), b = __builtin_amdgcn_readfirstlane(share.b), start = __builtin_amdgcn_readfirstlane(share.start);

  // sequence by sequence
  for (; tile < end; ++b) {
    bool bad;
    const int len = __builtin_amdgcn_readfirstlane(length_of(p, b, &bad));
    const Tiles tiles = tiles_of(len, p.window, p.sinks);
    if (tiles.n == 0) continue;
    const int from = max(0, len - p.window), n_sinks = min(p.sinks, len);
    const int t0 = tile - start, t1 = min(tiles.n, end - start);
    const bool alone = t0 == 0 && t1 == tiles.n;
    tile = start + t1;
    start += tiles.n;

    x8 qreg[kHeadTiles][4];  // B operand: lane holds head l16, d = 32 g + 8 ks .. +7
#pragma unroll
    for (int i = 0; i < kHeadTiles; ++i) {
      const char* qp = p.q.ptr + b * p.q.batch + (int64_t)(head0 + min(16 * i + l16, heads - 1)) * p.q.head + 64 * g;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) qreg[i][ks] = *reinterpret_cast<const x8*>(qp + 16 * ks);
    }
    f32x4 acc[kHeadTiles][8];
    float m_run[kHeadTiles], l_run[kHeadTiles];
#pragma unroll
    for (int i = 0; i < kHeadTiles; ++i) {
      m_run[i] = kNoReference;
      l_run[i] = 0.f;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) acc[i][dt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    const float c = p.scale_log2e;

    // this wave's tiles: t0 + wave, + 4, ...; pages of the next 32 of them, a lane to a half tile (16 slots, which are on one page)
    const int mine = t1 > t0 + wave ? (t1 - t0 - wave + kWaves - 1) / kWaves : 0;
    int pages = 0;
    auto load_pages = [&](int i0) {
      const int i = i0 + (lane >> 1);
      int page = 0;
      if (i < mine) {
        const int slot = tiles.at(t0 + wave + kWaves * i) * kTile + 16 * (lane & 1);
        if (slot < len) {
          page = cache.page_of(b, slot);
          if (page < 0) {
            bad = true;
            page = 0;
          }
        }
      }
      pages = page;
    };
    const uint32_t code_off = l16 * kHeldRowBytes + g * 16;
    const uint32_t scale_off = l16 * 4 + g;
    u32x4 k[2], v[2];
    uint32_t k_scale[2], v_scale[2];
    int64_t rows[2];  // first rows of the tile whose V is next
    // Of the wave's i-th tile, or, so that every step has as many loads in flight and none waits for more than its own, of the last one again.
    auto request_k = [&](int i) {
      if ((i & 31) == 0) load_pages(i);
      const int at = min(i, mine - 1), slot = __builtin_amdgcn_readfirstlane(tiles.at(t0 + wave + kWaves * at)) * kTile;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        rows[half] = cache.row_of(__builtin_amdgcn_readlane(pages, 2 * (at & 31) + half), hkv, slot + 16 * half);
        k[half] = load_codes(cache.k, rows[half], code_off);
        k_scale[half] = load_scale(cache.k_scales, rows[half], scale_off);
      }
      asm volatile("" : : : "memory");  // loads stay in this order: what waits for K leaves V in flight
    };
    auto request_v = [&]() {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        v[half] = load_codes(cache.v, rows[half], code_off);
        v_scale[half] = load_scale(cache.v_scales, rows[half], scale_off);
      }
      asm volatile("" : : : "memory");
    };
    int v_off[8], v_to[4];
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) v_off[dt] = tile_off(4 * g + (l16 >> 2), 2 * dt + ((l16 & 3) >> 1)) + (l16 & 1) * 8;
#pragma unroll
    for (int j = 0; j < 4; ++j) v_to[j] = tile_off(l16, 4 * g + j);
    char* const stage = smem + wave * kTileLds;
    const LdsPtr vt = lds_ptr(stage);
    if (mine > 0) {
      request_k(0);
      request_v();
      for (int i = 0;;) {
        const int slot0 = __builtin_amdgcn_readfirstlane(tiles.at(t0 + wave + kWaves * i)) * kTile;
        const bool whole = slot0 + kTile <= len && (slot0 >= from || slot0 + kTile <= n_sinks);
        auto seen = [&](int slot) { return slot < len && (slot >= from || slot < n_sinks); };
        f32x4 s[kHeadTiles][2];
#pragma unroll
        for (int ht = 0; ht < kHeadTiles; ++ht) s[ht][0] = s[ht][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float scale = scale_of(k_scale[half]);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const x8 a = from_4_bits<T>(k[half][ks], scale);
#pragma unroll
            for (int ht = 0; ht < kHeadTiles; ++ht) s[ht][half] = Elem<T>::mfma16(a, qreg[ht][ks], s[ht][half]);
          }
        }
        request_k(i + 1);
        x8 p_hi[kHeadTiles], p_lo[kHeadTiles];
#pragma unroll
        for (int ht = 0; ht < kHeadTiles; ++ht) {
          // s[ht][half][e]: slot 16 half + 4 g + e of the tile
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[ht][half][e] *= c;
          if (!whole) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[ht][half][e] = seen(slot0 + 16 * half + 4 * g + e) ? s[ht][half][e] : -INFINITY;
          }
          float mx = fmaxf(fmaxf(fmaxf(s[ht][0][0], s[ht][0][1]), fmaxf(s[ht][0][2], s[ht][0][3])), fmaxf(fmaxf(s[ht][1][0], s[ht][1][1]), fmaxf(s[ht][1][2], s[ht][1][3])));
          if (__builtin_amdgcn_ballot_w64(mx - m_run[ht] > kLazy) != 0) {
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float m_new = fmaxf(m_run[ht], mx), alpha = fast_exp2(m_run[ht] - m_new);
            m_run[ht] = m_new;
            l_run[ht] *= alpha;
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) acc[ht][dt] *= alpha;
          }
          // slots in the order in which V is fetched: 4 g .. +3, then 16 + 4 g .. +3
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float pv = fast_exp2(s[ht][e >> 2][e & 3] - m_run[ht]);
            l_run[ht] += pv;
            p_hi[ht][e] = (T)pv;
            p_lo[ht][e] = (T)(pv - (float)p_hi[ht][e]);
          }
        }
        if constexpr (kScores) {
#pragma unroll
          for (int ht = 0; ht < kHeadTiles; ++ht)
            if (16 * ht + l16 < heads) {
              float* to = p.scores + ((int64_t)b * p.heads + head0 + 16 * ht + l16) * cache.slots() + slot0 + 4 * g;
              *reinterpret_cast<f32x4*>(to) = s[ht][0];
              if (slot0 + 16 < cache.slots()) *reinterpret_cast<f32x4*>(to + 16) = s[ht][1];  // (room for a whole number of pages, of 16 slots at least)
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // what is not seen may be no number: a weight of zero takes any other value
          if (!whole) v_scale[half] = seen(slot0 + 16 * half + l16) ? v_scale[half] : 127u;
          const float scale = scale_of(v_scale[half]);
#pragma unroll
          for (int j = 0; j < 4; ++j) *reinterpret_cast<x8*>(stage + half * 4096 + v_to[j]) = from_4_bits<T>(v[half][j], scale);
        }
        request_v();
        asm volatile("" : : : "memory");  // (LDS instructions of a wave are in order)
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
          const x8 a = read_tr8<T>(vt + v_off[dt], vt + v_off[dt] + 4096);
#pragma unroll
          for (int ht = 0; ht < kHeadTiles; ++ht) {
            acc[ht][dt] = Elem<T>::mfma16(a, p_hi[ht], acc[ht][dt]);
            acc[ht][dt] = Elem<T>::mfma16(a, p_lo[ht], acc[ht][dt]);
          }
        }
        asm volatile("" : : : "memory");  // the next tile goes where this one is
        if (++i == mine) break;
      }
    }
    const bool any_bad = __builtin_amdgcn_ballot_w64(bad) != 0;
    leave_sums<T, kHeadTiles>(p, smem, acc, m_run, l_run, any_bad, alone, b, w, head0, heads);
  }
}

template <typename T>
static hipError_t launch_attend4(const AttendParams& p, hipStream_t stream) {
  const int tiles = head_tiles_of(p.heads / p.cache.kv_heads);
  const bool scores = p.scores != nullptr;
  void (*fn)(const AttendParams) = tiles == 1 ? (scores ? &cache_attend4_kernel<T, 1, true> : &cache_attend4_kernel<T, 1, false>)
                                              : (scores ? &cache_attend4_kernel<T, 2, true> : &cache_attend4_kernel<T, 2, false>);
  constexpr int smem = kSumsLds;
  static_assert(smem >= kWaves * kTileLds, "room for the tiles");
  hipLaunchKernelGGL(fn, dim3(p.target, p.cache.kv_heads * p.head_tiles), dim3(64 * kWaves), smem, stream, p);
  return hipGetLastError();
}

hipError_t launch_cache_attend4(AttendParams p, bool half, hipStream_t stream) {
  hipError_t e = half ? launch_attend4<_Float16>(p, stream) : launch_attend4<__bf16>(p, stream);
  return e == hipSuccess ? launch_cache_join(p, half, stream) : e;
}

}  // namespace fba
