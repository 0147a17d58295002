// Backward of attention under a sliding window with sinks, dQ and delta: gfx950, head_dim 128, bf16 or fp16 in / fp32 accumulate.
//
// With P = exp(S/sqrt(128) - LSE), delta = rowsum(dO o O), dP = dO V^T, dS = P o (dP - delta) / sqrt(128):
//   dQ = dS K,  dV = P^T dO,  dK = dS^T Q
// Two kernels, each of which owns the rows it writes: this one walks the keys of 128 query rows (and works delta out, of which it has both factors at hand), the one in
// fba_window_dkdv.hip the query rows of 128 keys.  Both form S and dP anew from what they have in LDS, seven products where five are needed, and write nothing in between but
// statistics: dS would be 2 bytes for every row and key of its window.
//
// Bound by issue and by the fetches from LDS (three a product's operand, by 128 rows' four waves each): the matrix pipe is busy 52 % of the time.  H24 S30720, window 1152 to both
// sides, 384 sinks: 1.49 ms, 1.49 TFLOP of visible pairs in three products, 1.00 PFLOP/s.
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
  const int len = p.lengths != nullptr ? min(max(const_idx(p.lengths)[b], 0), p.Skv) : p.Skv;
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

  // The sum of a row's P as they are formed here: one, but for what forward's rounding of P has left in lse.  dQ is divided by it, and dK and dV get an lse that has it.  (Half of
  // that error is a row's own: without this dq of 150 to 600 keys in fp16 is off by 1.5 times what rounding it alone does, with it by 1.45.)
  float of_p[2] = {0.f, 0.f}, lse2 = INFINITY;
  const int64_t stat = ((int64_t)b * p.Hq + hq) * p.Sq + min(row, rows - 1);
  if (last_row >= row0) {
    // Q and dO as B operands: lane holds row l32, d = 16 ks + 8 h .. +7 (rows behind the last: that one)
    x8 qreg[8], doreg[8];
    const int from = min(row, rows - 1);
    const char* const qp = p.q.ptr + b * p.q.batch + hq * p.q.head + (int64_t)from * p.q.row + 16 * h;
    const char* const dp = p.d_o.ptr + b * p.d_o.batch + hq * p.d_o.head + (int64_t)from * p.d_o.row + 16 * h;
    const char* const op = p.o.ptr + b * p.o.batch + hq * p.o.head + (int64_t)from * p.o.row + 16 * h;
    // delta: with what rounding o has left, where that is there (a row's error in it goes into all of its dS)
    const char* const lp = p.o_low.ptr == nullptr ? op : p.o_low.ptr + b * p.o_low.batch + hq * p.o_low.head + (int64_t)from * p.o_low.row + 16 * h;
    const float low = p.o_low.ptr == nullptr ? 0.f : 1.f;
    lse2 = p.lse[stat];
    float sum = 0.f;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      qreg[ks] = *reinterpret_cast<const x8*>(qp + 32 * ks);
      doreg[ks] = *reinterpret_cast<const x8*>(dp + 32 * ks);
      const x8 o8 = *reinterpret_cast<const x8*>(op + 32 * ks), l8 = *reinterpret_cast<const x8*>(lp + 32 * ks);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = __builtin_fmaf((float)doreg[ks][i], __builtin_fmaf(low, (float)l8[i], (float)o8[i]), sum);
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
      auto form_ds = [&](LdsPtr pair, auto between, auto sees) __attribute__((always_inline)) {
        f32x16 s, d;
#pragma unroll
        for (int r = 0; r < 16; ++r) { s[r] = 0.f; d[r] = neg_delta; }
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          s = Elem<T>::mfma32(read_b128<T>(pair + rm.rd[ks]), qreg[ks], s);
          d = Elem<T>::mfma32(read_b128<T>(pair + kSlabBytes + rm.rd[ks]), doreg[ks], d);
          between(ks);
        }
        sees(s, d);
        return s;
      };
      auto unmasked = [&](f32x16& s, const f32x16& d) __attribute__((always_inline)) {  // dS from S and dP - delta
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float pv = fast_exp2(__builtin_fmaf(s[r], c, -lse2));
          of_p[r & 1] += pv;
          s[r] = pv * d[r];
        }
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
          const f32x16 ds = form_ds(pair, [&](int ks) {
            if (ks < 4 && t > 0) request(ks);
          }, [&](f32x16& s, const f32x16& d) __attribute__((always_inline)) {
            if (kind != kMasked) return unmasked(s, d);
            const int k0 = slab_of(t) * kSlab + 4 * h, a = lo - k0, z = hi - k0, y = sk - k0;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int e = 8 * (r >> 2) + (r & 3);
              const bool sees = (e >= a && e <= z) || e < y;
              const float pv = sees ? fast_exp2(__builtin_fmaf(s[r], c, -lse2)) : 0.f;
              of_p[r & 1] += pv;
              s[r] = sees ? pv * d[r] : 0.f;
            }
          });
          add_dq(pair, ds);
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
        }, unmasked);
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
  const float sum_p = sum_halves(of_p[0] + of_p[1]);
  if (h == 0 && there) p.lse_exact[stat] = sum_p > 0.f ? lse2 + __builtin_log2f(sum_p) : lse2;
  store_tile<T>(smem + wave * kSlabBytes, acc, sum_p > 0.f ? p.scale / sum_p : p.scale, p.dq.ptr + b * p.dq.batch + hq * p.dq.head + (int64_t)wrow0 * p.dq.row, p.dq.row, lane, p.Sq - wrow0);
}

hipError_t launch_window_dq(WindowParams p, bool half, hipStream_t stream) {
  constexpr int kSmem = kRing * 2 * kSlabBytes;
  p.tiles = (p.Sq + kWindowTile - 1) / kWindowTile;
  p.items = p.B * p.Hq * p.tiles;
  p.chunk = window_chunk(p.items);
  hipLaunchKernelGGL((half ? &window_dq_kernel<_Float16> : &window_dq_kernel<__bf16>), dim3(window_grid(p.items, p.chunk)), dim3(256), kSmem, stream, p);
  return hipGetLastError();
}

}  // namespace fba
