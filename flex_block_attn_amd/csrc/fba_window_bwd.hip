// Backward of attention under a sliding window with sinks: gfx950, head_dim 128, bf16 or fp16 in / fp32 accumulate, no atomics.
//
// With P = exp(S/sqrt(128) - LSE), delta = rowsum(dO o O), dP = dO V^T, dS = P o (dP - delta) / sqrt(128):
//   dQ = dS K,  dV = P^T dO,  dK = dS^T Q
// Two kernels, each of which owns the rows it writes: the first walks the keys of 128 query rows (and works delta out, of which it has both factors at hand),
// the second the query rows of 128 keys.  Both form S and dP anew from what they have in LDS, 14 products where 10 are needed, and write nothing in between
// but delta.
//
// Sinks are seen from all rows, so a key tile with sinks has as many rows to add up as there are.  The second kernel cuts these in parts: one work item for the rows
// inside the window, as for every key tile, and as many of the same length as the rows outside of it take.  They leave fp32 sums, which a small kernel adds in
// order.
#include <type_traits>

#include "fba_types.h"
#include "fba_window.h"

namespace fba {

namespace {

constexpr int kSlab = 32;
constexpr int kSlabBytes = kSlab * kRowBytes;  // 8 KiB
constexpr int kRing = 4;

template <int N>
using IC = std::integral_constant<int, N>;

enum Kind { kNone, kFull, kMasked };

}  // namespace

// dQ: as forward, wave = 32 query rows, lane = row:
//   S^T = K Q^T, dP^T = V dO^T;  dS^T = exp2(c S^T - lse2) o (dP^T - delta);  dQ^T += K^T dS^T
// K and V slabs travel global -> LDS into a ring of four (K | V) buffers, three steps ahead.
template <typename T>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(2, 2))) void window_dq_kernel(const WindowParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];  // ring [4] of (K slab | V slab)
  using x8 = x8_of<T>;
  constexpr int kPairBytes = 2 * kSlabBytes;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int item = window_item(blockIdx.x, p.chunk);
  if (item >= p.items) return;
  const int group = p.Hq / p.Hkv;
  const int g = item % group;
  item /= group;
  const int tile = p.tiles - 1 - item % p.tiles;
  item /= p.tiles;
  const int hkv = item % p.Hkv, b = item / p.Hkv, hq = hkv * group + g;

  // slabs of the tile and what every row sees, as in forward
  const int len = p.lengths != nullptr ? min(max(p.lengths[b], 0), p.Skv) : p.Skv;
  const int rows = p.lengths != nullptr ? len : p.Sq;
  const int shift = p.lengths != nullptr ? 0 : p.Skv - p.Sq;
  const int row0 = tile * kWindowTile, ahead = p.causal ? 0 : p.window - 1;
  const int last_row = min(row0 + kWindowTile, rows) - 1;
  auto sinks_at = [&](int at) { return min(min(p.sinks, len), p.causal ? at + 1 : p.sinks); };
  int n_sink = 0, first = 0, n = 0;
  if (last_row >= row0 && len > 0) {
    const int low = max(0, row0 + shift - p.window + 1), high = min(len - 1, last_row + shift + ahead);
    n_sink = (max(0, sinks_at(last_row + shift)) + kSlab - 1) / kSlab;
    first = max(low / kSlab, n_sink);
    n = n_sink + (high >= low ? max(0, high / kSlab + 1 - first) : 0);
  }
  auto slab_of = [&](int t) { return t < n_sink ? t : first + t - n_sink; };
  const int wrow0 = row0 + wave * 32, row = wrow0 + l32, at = row + shift;
  const bool there = row < rows;
  const int hi = there ? min(len - 1, at + ahead) : -1, lo = at - p.window + 1, sk = there ? sinks_at(at) : 0;
  const int wave_first = wrow0 + shift, wave_last = min(wrow0 + 32, rows) - 1 + shift;
  const bool idle = wrow0 >= rows, whole = wrow0 + 32 <= rows;  // (rows of padding see nothing)
  const int all_hi = min(len - 1, wave_first + ahead), all_lo = wave_last - p.window + 1, all_sk = sinks_at(wave_first);
  const int any_hi = min(len - 1, wave_last + ahead), any_lo = wave_first - p.window + 1, any_sk = sinks_at(wave_last);
  auto kind_of = [&](int t) -> int {
    if (t >= n || idle) return kNone;
    const int k0 = slab_of(t) * kSlab, k1 = k0 + kSlab - 1;
    if (whole && ((k1 <= all_hi && k0 >= all_lo) || k1 < all_sk)) return kFull;
    return (k0 <= any_hi && k1 >= any_lo) || k0 < any_sk ? kMasked : kNone;
  };

  f32x16 acc[4];
#pragma unroll
  for (int mb = 0; mb < 4; ++mb)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[mb][r] = 0.f;

  if (last_row >= row0) {
    // Q and dO as B operands: lane holds row l32, d = 16 ks + 8 h .. +7 (rows behind the last: that one)
    x8 qreg[8], doreg[8];
    const int from = min(row, rows - 1);
    const char* const qp = p.q.ptr + b * p.q.batch + hq * p.q.head + (int64_t)from * p.q.row + 16 * h;
    const char* const dp = p.d_o.ptr + b * p.d_o.batch + hq * p.d_o.head + (int64_t)from * p.d_o.row + 16 * h;
    const char* const op = p.o.ptr + b * p.o.batch + hq * p.o.head + (int64_t)from * p.o.row + 16 * h;
    const int64_t stat = ((int64_t)b * p.Hq + hq) * p.Sq + from;
    float lse2 = p.lse[stat];
    float sum = 0.f;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      qreg[ks] = *reinterpret_cast<const x8*>(qp + 32 * ks);
      doreg[ks] = *reinterpret_cast<const x8*>(dp + 32 * ks);
      const x8 o8 = *reinterpret_cast<const x8*>(op + 32 * ks);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = __builtin_fmaf((float)doreg[ks][i], (float)o8[i], sum);
    }
    const float neg_delta = -sum_halves(sum);
    if (h == 0 && there) p.neg_delta[stat] = neg_delta;
    const char* const kp = p.k.ptr + b * p.k.batch + hkv * p.k.head;
    const char* const vp = p.v.ptr + b * p.v.batch + hkv * p.v.head;
    const int64_t k_step = (int64_t)p.k.row * kSlab, v_step = (int64_t)p.v.row * kSlab;
    const float c = p.scale_log2e;

    if (n > 0) {
      RowMajorOffsets rm;
      rm.init(lane);
      TransposedOffsets tr;
      tr.init(lane);
      RowDma k_dma, v_dma;
      k_dma.init(wave, lane, p.k.row, len - 1);
      v_dma.init(wave, lane, p.v.row, len - 1);
      const LdsPtr lds = lds_ptr(smem);
      const uint32_t dst = lds_addr(smem);
      auto slab_at = [&](int t) { return slab_of(min(t, n - 1)); };
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int slab = slab_at(j);
        k_dma.copy(dst + j * kPairBytes, kp + slab * k_step, slab);
        v_dma.copy(dst + j * kPairBytes + kSlabBytes, vp + slab * v_step, slab);
      }
      wait_vmem<0>();
      __syncthreads();
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) { pin(qreg[ks]); pin(doreg[ks]); }

      // dS^T of a slab from S^T and dP^T - delta, and what it adds to dQ.  dS is rounded to T as the matrix instruction takes it; the factor 1 / sqrt(128) comes at the end.
      auto add_dq = [&](LdsPtr pair, const f32x16& s) {
        x8 ds[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) ds[j] = narrow8<T>(s, j);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int mb = 0; mb < 4; ++mb) {
            const int roff = 16 * j * kRowBytes;
            acc[mb] = Elem<T>::mfma32(read_tr8<T>(pair + tr.rd[mb][0] + roff, pair + tr.rd[mb][1] + roff), ds[j], acc[mb]);
          }
      };
      auto form_ds = [&](LdsPtr pair, auto between) {
        f32x16 s, d;
#pragma unroll
        for (int r = 0; r < 16; ++r) { s[r] = 0.f; d[r] = neg_delta; }
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          s = Elem<T>::mfma32(read_b128<T>(pair + rm.rd[ks]), qreg[ks], s);
          d = Elem<T>::mfma32(read_b128<T>(pair + kSlabBytes + rm.rd[ks]), doreg[ks], d);
          between(ks);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fast_exp2(__builtin_fmaf(s[r], c, -lse2)) * d[r];
        return s;
      };
      // Step t (t % 4 == R): S_t, dP_t | dS_t | dQ += K_t^T dS_t.  Slab t+3 is requested into the buffer of slab t-1, between the first matrix instructions; behind the step
      // slab t+1 must have landed (and has, as slab t+2): what step t requested may still fly.
      auto step = [&](auto ring_c, int t) {
        constexpr int R = decltype(ring_c)::value;
        const int kind = kind_of(t), slab = slab_at(t + 3);
        const LdsPtr pair = lds + R * kPairBytes;
        const uint32_t into = dst + ((R + 3) & 3) * kPairBytes;
        auto request = [&](int i) {
          if (i < 2) k_dma.piece(i, into, kp + slab * k_step, slab);
          else v_dma.piece(i - 2, into + kSlabBytes, vp + slab * v_step, slab);
        };
        if (kind != kNone) {
          f32x16 s = form_ds(pair, [&](int ks) {
            if (ks < 4 && t > 0) request(ks);
          });
          if (kind == kMasked) {
            const int k0 = slab_of(t) * kSlab + 4 * h, a = lo - k0, z = hi - k0, y = sk - k0;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int e = 8 * (r >> 2) + (r & 3);
              s[r] = (e >= a && e <= z) || e < y ? s[r] : 0.f;
            }
          }
          add_dq(pair, s);
        } else if (t > 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) request(i);
        }
        wait_vmem<4>();
        __syncthreads();
      };
      // The same where all rows of the tile see slab t whole and slab t+3 is not the last one.
      const char *k_src = kp, *v_src = vp;
      auto whole_step = [&](auto ring_c) {
        constexpr int R = decltype(ring_c)::value;
        const LdsPtr pair = lds + R * kPairBytes;
        const uint32_t into = dst + ((R + 3) & 3) * kPairBytes + k_dma.wave_dst;
        const f32x16 s = form_ds(pair, [&](int ks) {
          if (ks == 0) dma16(into, k_src, k_dma.off[0]);
          if (ks == 1) dma16(into + 4 * kRowBytes, k_src, k_dma.off[1]);
          if (ks == 2) dma16(into + kSlabBytes, v_src, v_dma.off[0]);
          if (ks == 3) dma16(into + kSlabBytes + 4 * kRowBytes, v_src, v_dma.off[1]);
        });
        add_dq(pair, s);
        wait_vmem<4>();
        __syncthreads();
        k_src += k_step;
        v_src += v_step;
      };
      const int whole_lo = max(0, last_row + shift - p.window + 1), whole_hi = min(len - 1, row0 + shift + ahead);
      const int from = n_sink + max(0, (whole_lo + kSlab - 1) / kSlab - first);
      const int to = row0 + kWindowTile <= rows ? n_sink + (whole_hi + 1) / kSlab - first : 0;
      const int whole_end = min(to, n - 4);  // of the steps that whole_step takes
      for (int t = 0; t < n;) {
        if (t > 0 && t >= from && t + 4 <= whole_end) {
          k_src = kp + slab_of(t + 3) * k_step;
          v_src = vp + slab_of(t + 3) * v_step;
          do {
            whole_step(IC<0>{});
            whole_step(IC<1>{});
            whole_step(IC<2>{});
            whole_step(IC<3>{});
            t += 4;
          } while (t + 4 <= whole_end);
        }
        step(IC<0>{}, t);
        if (t + 1 < n) step(IC<1>{}, t + 1);
        if (t + 2 < n) step(IC<2>{}, t + 2);
        if (t + 3 < n) step(IC<3>{}, t + 3);
        t += 4;
      }
      wait_vmem<0>();
      __syncthreads();
    }
  }
  store_tile<T>(smem + wave * kSlabBytes, acc, p.scale, p.dq.ptr + b * p.dq.batch + hq * p.dq.head + (int64_t)wrow0 * p.dq.row, p.dq.row, lane, p.Sq - wrow0);
}

// dK and dV: work-group = 128 keys of one (batch, kv head), eight waves, two per SIMD.  Wave w works on keys 32 (w % 4) ..+31 and on every second 32-row slab
// (w / 4 = parity), lane = key:
//   S = Q K^T, dP = dO V^T             A = Q / dO slab rows, B = K / V rows, all from LDS
//   P = exp2(c S - lse2[q]),  dS = P o (dP - delta[q])
//   dV^T += dO^T P,  dK^T += Q^T dS    A = dO / Q slab through transposing fetches
// The two waves of a key group swap halves of their sums through LDS at the end: parity 0 finishes dV, parity 1 dK.
// LDS: ring of four (Q slab | dO slab | lse2 | -delta) buffers = two slab pairs, then the K tile and the V tile.
//
// Items: first the parts of the tiles with sinks (their rows outside of the window), then every key tile with the rows inside.
namespace {
constexpr int kStatBytes = 2 * kSlab * 4;
constexpr int kStageBytes = 2 * kSlabBytes + kStatBytes;
constexpr int kTileBytes = kWindowTile * kRowBytes;
constexpr int kTileBase = kRing * kStageBytes;
constexpr int kDkdvSmem = kTileBase + 2 * kTileBytes;

// Rows of a (key tile, batch): slabs from `first` on, of which those from `cut` on are `gap` further.
struct RowSlabs {
  int first, cut, gap, n;
  __host__ __device__ int at(int i) const { return first + i + (i >= cut ? gap : 0); }
};

// Slabs of 32 rows with some row that sees a key of tile `kt` inside its window, or (outside) sees a sink of it outside.
__host__ __device__ inline RowSlabs row_slabs(int kt, int len, int rows, int shift, int window, int sinks, bool causal, bool outside) {
  const int k0 = kt * kWindowTile, k1 = (k0 + kWindowTile < len ? k0 + kWindowTile : len) - 1;
  RowSlabs s{0, 0x7fffffff, 0, 0};
  if (rows <= 0 || k1 < k0) return s;
  if (!outside) {
    int low = causal ? k0 - shift : k0 - window + 1 - shift, high = k1 + window - 1 - shift;
    low = low < 0 ? 0 : low;
    high = high > rows - 1 ? rows - 1 : high;
    s.first = low / kSlab;
    s.n = high >= low ? high / kSlab + 1 - s.first : 0;
    return s;
  }
  const int last = (k1 < sinks ? k1 : sinks - 1);  // last sink of the tile
  if (last < k0) return s;
  // behind the window of some sink: rows from k0 + window - shift on; in front of it: rows up to last - window - shift
  int behind = k0 + window - shift;
  behind = behind < 0 ? 0 : behind;
  const int front = causal ? -1 : (last - window - shift > rows - 1 ? rows - 1 : last - window - shift);
  const int n_front = front >= 0 ? front / kSlab + 1 : 0;
  int from = behind / kSlab;
  from = from < n_front ? n_front : from;
  const int all = (rows + kSlab - 1) / kSlab;
  const int n_behind = behind <= rows - 1 && all > from ? all - from : 0;
  s.first = 0;
  s.cut = n_front;
  s.gap = from - n_front;
  s.n = n_front + n_behind;
  return s;
}
}  // namespace

template <typename T>
__global__ __attribute__((amdgpu_flat_work_group_size(512, 512), amdgpu_waves_per_eu(2, 2))) void window_dkdv_kernel(const WindowParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using x8 = x8_of<T>;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = wave & 3, par = wave >> 2;
  int item = window_item(blockIdx.x, p.chunk);
  if (item >= p.items) return;
  const bool outside = item < p.sink_items;  // of the window
  int part = 0, kt;
  if (outside) {
    part = item % p.sink_parts;
    item /= p.sink_parts;
    kt = item % p.sink_tiles;
    item /= p.sink_tiles;
  } else {
    item -= p.sink_items;
    kt = item % p.tiles;
    item /= p.tiles;
  }
  const int hkv = item % p.Hkv, b = item / p.Hkv, group = p.Hq / p.Hkv;
  const int len = p.lengths != nullptr ? min(max(p.lengths[b], 0), p.Skv) : p.Skv;
  const int rows = p.lengths != nullptr ? len : p.Sq;
  const int shift = p.lengths != nullptr ? 0 : p.Skv - p.Sq;
  const bool causal = p.causal != 0;
  const RowSlabs slabs = row_slabs(kt, len, rows, shift, p.window, p.sinks, causal, outside);
  const int all = slabs.n * group;
  const int s_begin = outside ? (int)((int64_t)all * part / p.sink_parts) : 0;
  const int n = (outside ? (int)((int64_t)all * (part + 1) / p.sink_parts) : all) - s_begin;
  const int key0 = kt * kWindowTile;

  f32x16 acc_k[4], acc_v[4];
#pragma unroll
  for (int mb = 0; mb < 4; ++mb)
#pragma unroll
    for (int r = 0; r < 16; ++r) { acc_k[mb][r] = 0.f; acc_v[mb][r] = 0.f; }

  // this lane's key: the rows lo .. hi have it in their window; the wave's keys
  const int key = key0 + kg * 32 + l32, wkey0 = key0 + kg * 32, wkey1 = wkey0 + 31;
  const int limit = outside ? min(p.sinks, len) : len;
  const int hi = key + p.window - 1 - shift, lo = outside ? (causal ? -0x40000000 : key - p.window + 1 - shift) : (causal ? key - shift : key - p.window + 1 - shift);
  const bool mine = key < limit;
  auto kind_of = [&](int row0) -> int {
    const int row1 = row0 + kSlab - 1;
    if (wkey0 >= limit) return kNone;
    if (!outside) {
      const int back = causal ? 0 : p.window - 1;
      if (row1 < wkey0 - back - shift || row0 > wkey1 + p.window - 1 - shift) return kNone;
      return row0 >= wkey1 - back - shift && row1 <= wkey0 + p.window - 1 - shift && row1 < rows && wkey1 < limit ? kFull : kMasked;
    }
    // outside: a row that has all of the wave's keys in its window, or in front of them (causal), sees none of them here
    const int all_lo = causal ? -0x40000000 : wkey1 - p.window + 1 - shift, all_hi = wkey0 + p.window - 1 - shift;  // rows that have all of them inside
    if (row0 >= all_lo && row1 <= all_hi) return kNone;
    const int any_lo = causal ? -0x40000000 : wkey0 - p.window + 1 - shift, any_hi = wkey1 + p.window - 1 - shift;
    return (row0 > any_hi || row1 < any_lo) && row1 < rows && wkey1 < limit ? kFull : kMasked;
  };

  if (n > 0) {
    const LdsPtr lds = lds_ptr(smem);
    const uint32_t lds0 = lds_addr(smem);
    {  // K rows by the waves of parity 0, V rows by those of parity 1: four slabs each
      const Strided& x = par ? p.v : p.k;
      RowDma dma;
      dma.init(kg, lane, x.row, len - 1);
      const char* src = x.ptr + b * x.batch + hkv * x.head;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int slab = min(4 * kt + j, dma.last_slab);  // slabs behind the last key: masked
        dma.copy(lds0 + kTileBase + par * kTileBytes + j * kSlabBytes, src + slab * ((int64_t)x.row * kSlab), slab);
      }
    }
    RowDma q_dma, do_dma;
    q_dma.init(kg, lane, p.q.row, rows - 1);
    do_dma.init(kg, lane, p.d_o.row, rows - 1);
    const int64_t q_step = (int64_t)p.q.row * kSlab, do_step = (int64_t)p.d_o.row * kSlab;
    const char* const qb = p.q.ptr + b * p.q.batch + (int64_t)hkv * group * p.q.head;
    const char* const db = p.d_o.ptr + b * p.d_o.batch + (int64_t)hkv * group * p.d_o.head;
    const int64_t stat0 = ((int64_t)b * p.Hq + hkv * group) * p.Sq;
    // statistics: lanes 0..31 fetch lse2[row0 + l], lanes 32..63 -delta[row0 + l - 32]
    const uint32_t stat_off = (uint32_t)l32 * 4, stat_last = (uint32_t)min(l32, (rows - 1) & 31) * 4;
    const uint32_t delta_at = (uint32_t)(lane >> 5);
    const int64_t delta_bytes = (const char*)p.neg_delta - (const char*)p.lse;  // one buffer, -delta behind lse
    const uint32_t half_off = delta_at ? (uint32_t)delta_bytes : 0;

    // cursors over (query head of the group, slab): what is requested next and what is worked on
    struct Cursor {
      int g, i;
    };
    auto start = [&](int s) { return Cursor{s / slabs.n, s % slabs.n}; };
    auto advance = [&](Cursor& c) {
      if (++c.i == slabs.n) { c.i = 0; ++c.g; }
    };
    Cursor ask = start(s_begin), work = ask;
    int asked = 0;  // slabs of this item
    auto issue_copy = [&](int ring, const Cursor& at) {
      const int slab = slabs.at(at.i);
      const uint32_t dst = lds0 + ring * kStageBytes;
      q_dma.copy(dst, qb + at.g * p.q.head + slab * q_step, slab);
      do_dma.copy(dst + kSlabBytes, db + at.g * p.d_o.head + slab * do_step, slab);
      dma4(dst + 2 * kSlabBytes, (const char*)(p.lse + stat0 + (int64_t)at.g * p.Sq + slab * kSlab), half_off + (slab == q_dma.last_slab ? stat_last : stat_off));
    };
    // slabs 2i, 2i + 1 -> ring buffers 2 slot, 2 slot + 1, by the four waves of each parity.  Past the last slab that one again, into buffers that nobody reads.
    auto next = [&]() {
      const Cursor at = ask;
      if (++asked < n) advance(ask);
      return at;
    };
    auto request_pair = [&](int slot) {
      const Cursor c0 = next(), c1 = next();
      issue_copy(2 * slot + par, par ? c1 : c0);
    };
    request_pair(0);
    request_pair(1);
    if (par) advance(work);
    RowMajorOffsets rm;
    rm.init(lane);
    TransposedOffsets tr;
    tr.init(lane);
    wait_vmem<0>();
    __syncthreads();

    // per-lane fetch addresses with the wave's share folded in
    LdsPtr q_ptr[8], k_ptr[8], t_ptr[4][2];
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      q_ptr[ks] = lds + rm.rd[ks] + par * kStageBytes;
      k_ptr[ks] = lds + rm.rd[ks] + kTileBase + kg * kSlabBytes;
    }
#pragma unroll
    for (int mb = 0; mb < 4; ++mb) {
      t_ptr[mb][0] = lds + tr.rd[mb][0] + par * kStageBytes;
      t_ptr[mb][1] = lds + tr.rd[mb][1] + par * kStageBytes;
    }
    const LdsPtr st_ptr = lds + par * kStageBytes + 2 * kSlabBytes + 16 * h;
    const float c = p.scale_log2e;

    auto compute = [&](auto half_c, int row0, bool masked) {
      constexpr int so = decltype(half_c)::value * 2 * kStageBytes;
      f32x16 s, dp;
      // accumulator element 4g + e of half-wave h is row 8g + 4h + e of the slab; dP starts from -delta of its row
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 d4 = lds_read_f32x4(st_ptr + so + 4 * kSlab + 32 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) { s[4 * g + e] = 0.f; dp[4 * g + e] = d4[e]; }
      }
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        s = Elem<T>::mfma32(read_b128<T>(q_ptr[ks] + so), read_b128<T>(k_ptr[ks]), s);
        dp = Elem<T>::mfma32(read_b128<T>(q_ptr[ks] + so + kSlabBytes), read_b128<T>(k_ptr[ks] + kTileBytes), dp);
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 l4 = lds_read_f32x4(st_ptr + so + 32 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float pv = fast_exp2(__builtin_fmaf(s[4 * g + e], c, -l4[e]));
          s[4 * g + e] = pv;
          dp[4 * g + e] = pv * dp[4 * g + e];
        }
      }
      if (masked) {
        const int r0 = row0 + 4 * h, a = lo - r0, z = hi - r0, end = mine ? rows - r0 : 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int e = 8 * (r >> 2) + (r & 3);
          const bool sees = ((e >= a && e <= z) != outside) && e < end;
          s[r] = sees ? s[r] : 0.f;
          dp[r] = sees ? dp[r] : 0.f;
        }
      }
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
          const int roff = so + 16 * j * kRowBytes;
          acc_v[mb] = Elem<T>::mfma32(read_tr8<T>(t_ptr[mb][0] + kSlabBytes + roff, t_ptr[mb][1] + kSlabBytes + roff), pk[j], acc_v[mb]);
          acc_k[mb] = Elem<T>::mfma32(read_tr8<T>(t_ptr[mb][0] + roff, t_ptr[mb][1] + roff), dsk[j], acc_k[mb]);
        }
    };
    auto step = [&](auto half_c, int s2) {
      if (2 * s2 + par < n) {
        const int row0 = slabs.at(work.i) * kSlab, kind = kind_of(row0);
        if (kind != kNone) compute(half_c, row0, kind == kMasked);
        advance(work);
        advance(work);
      }
      wait_vmem<0>();   // this wave's copies of the next pair have landed
      __syncthreads();  // everybody is done with this pair, and everybody's copies have landed
      request_pair(decltype(half_c)::value);
    };
    const int npairs = (n + 1) >> 1;
    for (int s2 = 0; s2 < npairs; s2 += 2) {
      step(IC<0>{}, s2);
      if (s2 + 1 < npairs) step(IC<1>{}, s2 + 1);
    }
    wait_vmem<0>();
    __syncthreads();  // no copy is writing LDS any more; K, V and the ring are free

    // the waves of a key group swap halves: parity 1 hands its dV sums to parity 0 through the first 64 KiB, parity 0 its dK sums through the next
    f32x4* send = reinterpret_cast<f32x4*>(smem + (par ? 0 : 65536) + kg * 16384) + lane;
    const f32x4* recv = reinterpret_cast<const f32x4*>(smem + (par ? 65536 : 0) + kg * 16384) + lane;
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x16& a = par ? acc_v[mb] : acc_k[mb];
        send[(mb * 4 + g) * 64] = (f32x4){a[4 * g + 0], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]};
      }
    __syncthreads();
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 r = recv[(mb * 4 + g) * 64];
        f32x16& a = par ? acc_k[mb] : acc_v[mb];
#pragma unroll
        for (int e = 0; e < 4; ++e) a[4 * g + e] += r[e];
      }
    __syncthreads();  // LDS is free for the results
  }

  f32x16 result[4];
#pragma unroll
  for (int mb = 0; mb < 4; ++mb) result[mb] = par ? acc_k[mb] : acc_v[mb];
  if (p.sink_parts > 0 && kt < p.sink_tiles) {
    // partial sums of a tile with sinks: the rows inside of the window first, then the parts outside
    const int64_t slot = (((int64_t)b * p.Hkv + hkv) * p.sink_tiles + kt) * (p.sink_parts + 1) + (outside ? 1 + part : 0);
    float* prow = p.parts + slot * kPartFloats + par * (kWindowTile * kHeadDim) + (kg * 32 + l32) * kHeadDim;
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(prow + 32 * mb + 8 * g + 4 * h) =
            (f32x4){result[mb][4 * g + 0], result[mb][4 * g + 1], result[mb][4 * g + 2], result[mb][4 * g + 3]};
    return;
  }
  const Strided& out = par ? p.dk : p.dv;
  store_tile<T>(smem + wave * kSlabBytes, result, par ? p.scale : 1.f, out.ptr + b * out.batch + hkv * out.head + (int64_t)wkey0 * out.row, out.row, lane,
                p.Skv - wkey0);
}

// Sums the parts of the tiles with sinks, in order.  A work-group per 8 rows, 32 threads to a row of dV or dK.
template <typename T>
__global__ __launch_bounds__(256) void window_sum_kernel(const WindowParams p) {
  const int c4 = (threadIdx.x & 31) * 4, r = (blockIdx.x % 16) * 8 + (threadIdx.x >> 5);
  const int which = blockIdx.x / 16 % 2;  // dV, dK
  int tile = blockIdx.x / 32;
  const float* src = p.parts + (int64_t)tile * (p.sink_parts + 1) * kPartFloats + which * (kWindowTile * kHeadDim) + r * kHeadDim + c4;
  const int kt = tile % p.sink_tiles;
  tile /= p.sink_tiles;
  const int hkv = tile % p.Hkv, b = tile / p.Hkv;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int q = 0; q <= p.sink_parts; q += 8) {
    f32x4 of[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (q + i <= p.sink_parts) of[i] = *reinterpret_cast<const f32x4*>(src + (int64_t)(q + i) * kPartFloats);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (q + i <= p.sink_parts) acc += of[i];
  }
  const int key = kt * kWindowTile + r;
  if (key >= p.Skv) return;
  const Strided& out = which ? p.dk : p.dv;
  const float s = which ? p.scale : 1.f;
  *reinterpret_cast<x4_of<T>*>(out.ptr + b * out.batch + hkv * out.head + (int64_t)key * out.row + c4 * 2) = narrow4<T>(acc[0] * s, acc[1] * s, acc[2] * s, acc[3] * s);
}

int64_t plan_window_bwd(WindowParams& p) {
  // Slabs of a tile with sinks outside of the window, for the longest sequence there may be, against those of a tile inside.
  p.sink_tiles = (p.sinks + kWindowTile - 1) / kWindowTile;
  p.sink_parts = 0;
  const int shift = p.lengths != nullptr ? 0 : p.Skv - p.Sq;
  int64_t outside = 0, inside = 1;
  for (int kt = 0; kt < p.sink_tiles; ++kt) {
    const int64_t n = row_slabs(kt, p.Skv, p.Sq, shift, p.window, p.sinks, p.causal != 0, true).n;
    if (n > outside) outside = n;
  }
  const int tiles = (p.Skv + kWindowTile - 1) / kWindowTile;
  inside = row_slabs(tiles / 2, p.Skv, p.Sq, shift, p.window, p.sinks, p.causal != 0, false).n;
  if (outside == 0) {
    p.sink_tiles = 0;
    return 0;
  }
  if (inside < 8) inside = 8;
  const int64_t parts = (outside + inside - 1) / inside;
  p.sink_parts = (int)(parts < 1 ? 1 : parts > 64 ? 64 : parts);
  return (int64_t)p.B * p.Hkv * p.sink_tiles * (p.sink_parts + 1) * kPartFloats * 4;
}

hipError_t launch_window_bwd(WindowParams p, bool half, hipStream_t stream) {
  p.tiles = (p.Sq + kWindowTile - 1) / kWindowTile;
  p.items = p.B * p.Hq * p.tiles;
  p.chunk = window_chunk(p.items);
  constexpr int kDqSmem = kRing * 2 * kSlabBytes;
  hipLaunchKernelGGL((half ? &window_dq_kernel<_Float16> : &window_dq_kernel<__bf16>), dim3(window_grid(p.items, p.chunk)), dim3(256), kDqSmem, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  p.tiles = (p.Skv + kWindowTile - 1) / kWindowTile;
  p.sink_items = p.B * p.Hkv * p.sink_tiles * p.sink_parts;
  p.items = p.sink_items + p.B * p.Hkv * p.tiles;
  p.chunk = window_chunk(p.items);
  void (*fn)(const WindowParams) = half ? &window_dkdv_kernel<_Float16> : &window_dkdv_kernel<__bf16>;
  if ((e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, kDkdvSmem)) != hipSuccess) return e;
  hipLaunchKernelGGL(fn, dim3(window_grid(p.items, p.chunk)), dim3(512), kDkdvSmem, stream, p);
  if ((e = hipGetLastError()) != hipSuccess || p.sink_items == 0) return e;
  hipLaunchKernelGGL((half ? &window_sum_kernel<_Float16> : &window_sum_kernel<__bf16>), dim3(p.B * p.Hkv * p.sink_tiles * 32), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace fba
