// Attention of one new token per sequence over a paged cache: gfx950, head_dim 128, bf16 or fp16 in / fp32 accumulate.
//
// The cache is read once and little is computed: the kernel is bound by device memory.  The tiles (32 slots) of all sequences, one behind the other, are cut into even shares,
// however long the sequences are, as many as work-groups fit the GPU at once: all are done together, and none starts late.  (Chunks of one length, a few times as many as fit:
// 154 us instead of 133 for 32 sequences of 0 to 16384 slots, 24 heads on 6; a few more work-groups than fit: 179.)  Lengths are known to the device only, so every
// work-group finds its share by itself and goes through the sequences in it.  It does one kv head for all query heads of the group (16 columns of a matrix instruction,
// or twice 16).  Its four waves take tiles in turn, each through a K tile and a V tile in LDS that nobody else touches, so that there is no barrier before a sequence's
// end.  The next K tile is requested as soon as the scores are there, the next V tile behind the second product, as streams (plain copies: 151 us instead of 133).
//   S^T[slot, q] = K Q^T,  P^T = exp2(c S^T - c m[q]),  O^T[d, q] += V^T P^T
// P goes into the second product in two parts of the type, rounded and what rounding left: the matrix pipe has time to spare here, and what is lost of P then is
// below what fp32 sums lose.  Sequences in several shares leave sums, which a second kernel joins.
// That case moves 848 MB at 6.4 TB/s; 8 streams of 115200 slots through a window of 8192 and 128 sinks, 16 heads on 4: 136 MB in 27 us; one of 768 slots: 6 us, and 3 to join.
//
// Accumulated weights need the denominator of all chunks: the first kernel leaves its scores (4 bytes for every head and slot, against 512 bytes of K and V), and the
// second adds up exp2(score - log2 denominator) over the heads of the group.
#include "fba_cache_attend.h"

#include <type_traits>

namespace fba {

namespace {

constexpr int kStage = 2 * kTileLds;  // of a wave: K tile | V tile

template <int N>
FBA_DEVICE void wait_copies() {  // until at most N are in flight; nothing moves across
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

}  // namespace

// kHeadTiles: query heads of a work-group, in sixteens.
template <typename T, int kHeadTiles, bool kScores>
__global__ __attribute__((amdgpu_flat_work_group_size(64 * kWaves, 64 * kWaves), amdgpu_waves_per_eu(2, 2))) void cache_attend_kernel(const AttendParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];  // [waves][K tile | V tile]
  using x8 = x8_of<T>;
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const CacheView& cache = p.cache;
  const int group = p.heads / cache.kv_heads;
  const int hkv = blockIdx.y / p.head_tiles, head0 = hkv * group + blockIdx.y % p.head_tiles * (16 * kHeadTiles);
  const int heads = min(16 * kHeadTiles, (hkv + 1) * group - head0);

  Share share;
  if (!find_share(p, tid, lane, wave, &share)) return;
  const int w = share.w, end = share.end;
  int tile = share.tile, b = share.b, start = share.start;

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

  x8 qreg[kHeadTiles][4];  // B operand: lane holds head l16, d = 32 ks + 8 g .. +7
#pragma unroll
  for (int i = 0; i < kHeadTiles; ++i) {
    const char* qp = p.q.ptr + b * p.q.batch + (int64_t)(head0 + min(16 * i + l16, heads - 1)) * p.q.head + 16 * g;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) qreg[i][ks] = *reinterpret_cast<const x8*>(qp + 64 * ks);
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
  const uint32_t lds0 = lds_addr(smem) + wave * kStage;
  uint32_t off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 4 * i + g;
    off[i] = row * kRowBytes + ((l16 ^ swz(row)) << 4);
  }
  const char* v_src[2] = {cache.v, cache.v};
  auto request = [&](uint32_t dst, const char* const (&src)[2]) {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int j = 0; j < 4; ++j) dma16_stream(dst + half * 4096 + j * 1024, src[half], off[j]);
  };
  auto request_k = [&](int i) {  // of the wave's i-th tile; V's place is kept for request_v
    if ((i & 31) == 0) load_pages(i);
    const int slot = tiles.at(t0 + wave + kWaves * i) * kTile;
    const char* k_src[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int64_t row = cache.row_of(__builtin_amdgcn_readlane(pages, 2 * (i & 31) + half), hkv, slot + 16 * half) * kRowBytes;
      k_src[half] = uniform(cache.k + row);
      v_src[half] = uniform(cache.v + row);
    }
    request(lds0, k_src);
  };
  auto request_v = [&]() { request(lds0 + kTileLds, v_src); };
  int k_off[4], v_off[8];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) k_off[ks] = tile_off(l16, 4 * ks + g);
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) v_off[dt] = tile_off(4 * g + (l16 >> 2), 2 * dt + ((l16 & 3) >> 1)) + (l16 & 1) * 8;

  char* const stage = smem + wave * kStage;
  const LdsPtr kt = lds_ptr(stage), vt = lds_ptr(stage + kTileLds);
  if (mine > 0) {
    request_k(0);
    request_v();
  }
  for (int i = 0; i < mine; ++i) {
    const int slot0 = tiles.at(t0 + wave + kWaves * i) * kTile;
    const bool more = i + 1 < mine;
    const bool whole = slot0 + kTile <= len && (slot0 >= from || slot0 + kTile <= n_sinks);
    auto seen = [&](int slot) { return slot < len && (slot >= from || slot < n_sinks); };
    wait_copies<8>();  // K is there, V may still fly
    f32x4 s[kHeadTiles][2];
#pragma unroll
    for (int ht = 0; ht < kHeadTiles; ++ht) s[ht][0] = s[ht][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const x8 a = read_b128<T>(kt + k_off[ks] + half * 4096);
#pragma unroll
        for (int ht = 0; ht < kHeadTiles; ++ht) s[ht][half] = Elem<T>::mfma16(a, qreg[ht][ks], s[ht][half]);
      }
    if (more) {
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // the fetches from the K tile are through
      request_k(i + 1);
    }
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
    if (more) wait_copies<8>(); else wait_copies<0>();  // V is there, the next K may still fly
    if constexpr (kScores) {
#pragma unroll
      for (int ht = 0; ht < kHeadTiles; ++ht)
        if (16 * ht + l16 < heads) {
          float* to = p.scores + ((int64_t)b * p.heads + head0 + 16 * ht + l16) * cache.slots() + slot0 + 4 * g;
          *reinterpret_cast<f32x4*>(to) = s[ht][0];
          if (slot0 + 16 < cache.slots()) *reinterpret_cast<f32x4*>(to + 16) = s[ht][1];  // (room for a whole number of pages, of 16 slots at least)
        }
    }
    if (!whole) {  // what is not seen may be anything: rows of zeros in its place
#pragma unroll
      for (int r = 0; r < kTile; r += 4)
        if (!seen(slot0 + r + g)) *reinterpret_cast<u32x4*>(stage + kTileLds + (r + g) * kRowBytes + l16 * 16) = (u32x4){0, 0, 0, 0};
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      const x8 a = read_tr8<T>(vt + v_off[dt], vt + v_off[dt] + 4096);
#pragma unroll
      for (int ht = 0; ht < kHeadTiles; ++ht) {
        acc[ht][dt] = Elem<T>::mfma16(a, p_hi[ht], acc[ht][dt]);
        acc[ht][dt] = Elem<T>::mfma16(a, p_lo[ht], acc[ht][dt]);
      }
    }
    if (more) {
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
      request_v();
    }
  }
  const bool any_bad = __builtin_amdgcn_ballot_w64(bad) != 0;

  leave_sums<T, kHeadTiles>(p, smem, acc, m_run, l_run, any_bad, alone, b, w, head0, heads);  // (the next sequence's copies go where the sums are)
  }
}

// Joins the parts of every sequence and adds up the weights.  Work-groups of 256: first one for every output row, whose 8 groups of 32 threads take parts in turn, so that all loads
// of up to eight parts are on their way together; then, with scores, those for kSpan slots of a (sequence, kv head) each.
constexpr int kSpan = 1024;
template <typename T>
__global__ __launch_bounds__(256) void cache_join_kernel(const AttendParams p, int out_wgs, int spans) {
  const CacheView& cache = p.cache;
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < out_wgs) {
    __shared__ f32x4 sums[8][32];
    __shared__ float ml[8][2];
    const int b = blockIdx.x / p.heads, head = blockIdx.x % p.heads, of = tid >> 5, d = (tid & 31) * 4;
    const int first = p.note[2 * b], parts = p.note[2 * b + 1];
    if (parts == 1) return;
    char* const out = p.o.ptr + b * p.o.batch + head * p.o.head + 2 * d;
    if (parts == 0) {  // nothing to see, or no length
      bool bad;
      length_of(p, b, &bad);
      const float f = bad ? __builtin_nanf("") : 0.f;
      if (of == 0) *reinterpret_cast<x4_of<T>*>(out) = narrow4<T>(f, f, f, f);
      return;
    }
    float m = kNoReference, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int i = of; i < parts; i += 8) {
      const int64_t at = (int64_t)(first + i) * p.heads + head;
      const f32x4 oi = *reinterpret_cast<const f32x4*>(p.part + at * kHeadDim + d);
      const float mi = p.part_ml[2 * at], li = p.part_ml[2 * at + 1];
      const float m_new = fmaxf(m, mi), f = fast_exp2(m - m_new), fi = fast_exp2(mi - m_new);
      o = o * f + oi * fi;
      l = l * f + li * fi;
      m = m_new;
    }
    sums[of][tid & 31] = o;
    if (d == 0) {
      ml[of][0] = m;
      ml[of][1] = l;
    }
    __syncthreads();
    if (of != 0) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fmaxf(m, ml[i][0]);
    float sum = 0.f;
    o = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = fast_exp2(ml[i][0] - m);
      sum += f * ml[i][1];
      o += f * sums[i][tid & 31];
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;  // (NaN stays)
    *reinterpret_cast<x4_of<T>*>(out) = narrow4<T>(o[0] * f, o[1] * f, o[2] * f, o[3] * f);
    return;
  }
  __shared__ float lse[256];
  const int i = blockIdx.x - out_wgs, span = i % spans, hkv = i / spans % cache.kv_heads, b = i / spans / cache.kv_heads;
  bool bad;
  const int len = length_of(p, b, &bad), s0 = span * kSpan;
  if (s0 >= len) return;
  const int group = p.heads / cache.kv_heads, first = p.note[2 * b], parts = p.note[2 * b + 1];
  for (int h0 = 0; h0 < group; h0 += 256) {  // heads of the group, a few hundred at a time
    const int n = min(256, group - h0);
    __syncthreads();
    // log2 of the denominators: 16 threads to a head
    for (int q = tid >> 4; q < n; q += 16) {
      const int64_t at = (int64_t)first * p.heads + hkv * group + h0 + q;
      float m = kNoReference, l = 0.f;
      for (int j = tid & 15; j < parts; j += 16) {
        const float mj = p.part_ml[2 * (at + (int64_t)j * p.heads)], lj = p.part_ml[2 * (at + (int64_t)j * p.heads) + 1], m_new = fmaxf(m, mj);
        l = l * fast_exp2(m - m_new) + lj * fast_exp2(mj - m_new);
        m = m_new;
      }
#pragma unroll
      for (int x = 1; x < 16; x *= 2) {
        const float mj = __shfl_xor(m, x), lj = __shfl_xor(l, x), m_new = fmaxf(m, mj);
        l = l * fast_exp2(m - m_new) + lj * fast_exp2(mj - m_new);
        m = m_new;
      }
      if ((tid & 15) == 0) lse[q] = m + __builtin_log2f(l);
    }
    __syncthreads();
    const int slot = s0 + tid * 4;
    if (slot < len) {
      const int page = cache.page_of(b, slot);
      f32x4 w = {0.f, 0.f, 0.f, 0.f};
      bool any = false;  // a sequence without a number adds nothing, and does not touch pages that may be another's
      const float* from = p.scores + ((int64_t)b * p.heads + hkv * group + h0) * cache.slots() + slot;
      for (int q = 0; q < n; ++q) {
        const f32x4 s = *reinterpret_cast<const f32x4*>(from + q * cache.slots());
        any = any || lse[q] == lse[q];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] += lse[q] == lse[q] ? fast_exp2(s[e] - lse[q]) : 0.f;  // (no number: a page or a query that is none)
      }
      if (page >= 0 && any) {  // four slots are on one page
        f32x4* to = reinterpret_cast<f32x4*>(cache.weights + cache.row_of(page, hkv, slot));
        f32x4 sum = *to;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = slot + e < len ? sum[e] + w[e] : sum[e];
        *to = sum;
      }
    }
  }
}

void plan_cache_attend(AttendParams& p, int compute_units) {
  const int group = p.heads / p.cache.kv_heads, per = 16 * head_tiles_of(group);
  p.head_tiles = (group + per - 1) / per;
  // Two work-groups are on a compute unit at a time (64 KiB of LDS each; of 4 bits kResident4 where a work-group has one tile of heads), and as many shares there are.
  const int rows = p.cache.kv_heads * p.head_tiles, resident = p.cache.k_scales != nullptr && head_tiles_of(group) == 1 ? kResident4 : 2;
  p.target = resident * compute_units / rows > 0 ? resident * compute_units / rows : 1;
  // no more than there may be tiles for
  int64_t most = (p.cache.batch * ((p.cache.slots() + kTile - 1) / kTile) + kLeastTiles - 1) / kLeastTiles;
  if (p.cache.k_scales != nullptr && most < p.cache.batch) most = p.cache.batch;
  if (p.target > most) p.target = (int)most;
  p.slots = p.target + p.cache.batch;
}

int64_t cache_attend_bytes(const AttendParams& p, bool accumulate) {
  const int64_t parts = (int64_t)p.slots * p.heads;
  return (parts * (kHeadDim + 2) + 2 * (int64_t)p.cache.batch + 4) / 4 * 16 + (accumulate ? (int64_t)p.cache.batch * p.heads * p.cache.slots() * 4 : 0);
}

template <typename T>
static hipError_t launch_attend(const AttendParams& p, hipStream_t stream) {
  const int tiles = head_tiles_of(p.heads / p.cache.kv_heads);
  const bool scores = p.scores != nullptr;
  void (*fn)(const AttendParams) = tiles == 1 ? (scores ? &cache_attend_kernel<T, 1, true> : &cache_attend_kernel<T, 1, false>)
                                              : (scores ? &cache_attend_kernel<T, 2, true> : &cache_attend_kernel<T, 2, false>);
  constexpr int smem = kWaves * kStage;  // (more than the sums at the end take)
  static_assert(smem >= kSumsLds, "room for the sums");
  hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(fn, dim3(p.target, p.cache.kv_heads * p.head_tiles), dim3(64 * kWaves), smem, stream, p);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  return launch_cache_join(p, std::is_same<T, _Float16>::value, stream);
}

hipError_t launch_cache_join(AttendParams p, bool half, hipStream_t stream) {
  const int out_wgs = p.cache.batch * p.heads;
  const int spans = p.scores != nullptr ? (int)((p.cache.slots() + kSpan - 1) / kSpan) : 0;
  void (*fn)(const AttendParams, int, int) = half ? &cache_join_kernel<_Float16> : &cache_join_kernel<__bf16>;
  hipLaunchKernelGGL(fn, dim3(out_wgs + spans * p.cache.kv_heads * p.cache.batch), dim3(256), 0, stream, p, out_wgs, spans);
  return hipGetLastError();
}

hipError_t launch_cache_attend(AttendParams p, bool half, hipStream_t stream) {
  return half ? launch_attend<_Float16>(p, stream) : launch_attend<__bf16>(p, stream);
}

}  // namespace fba
