// Forward of attention under a sliding window with sinks: gfx950, head_dim 128, bf16 or fp16 in / fp32 accumulate.
//
// One work-group of 4 waves owns 128 consecutive query rows of one (batch, head); wave w owns rows [32w, 32w+32).  Its keys are the slabs of 32 that hold
// sinks some row sees, and those from the first row's window to the last row's.  Everything is transposed, as in the other forward kernels (lane = query row):
//   S^T[key, q] = K Q^T,  P^T = exp2(c S^T - c m[q]),  O^T[d, q] += V^T P^T          c = log2(e) / sqrt(128)
// with a running reference m and sum l per lane.  While the VALU turns S_t into P_t, the matrix pipe computes S_{t+1} and adds P_{t-1} V_{t-1} into O.  K and V
// slabs travel global -> LDS directly into two rings of four buffers, four steps ahead.
//
// A slab that all 32 rows of a wave see whole needs no mask, one that none of them sees no work; of a window's slabs only the first and the last two or so
// are masked, by two compares for every score.
//
// Bound by issue: the matrix pipe is busy 50 % of the time and the VALU 42, and two waves on a SIMD cover little more of each other than that (without the barriers 5 % less
// time, with longer waits for copies none).  H24 S30720, window 1152 to both sides, 384 sinks: 1.06 ms, 0.99 TFLOP of visible pairs, 930 TFLOP/s; H24/6 S69120 window 1536, 128
// sinks: 1.52 ms, 920 TFLOP/s, read from memory 0.47 GB; H24 S30720 window 128: 243 us, 0.95 GB.
#include <type_traits>

#include "fba_types.h"
#include "fba_window.h"

namespace fba {

namespace {

constexpr int kSlab = 32;
constexpr int kSlabBytes = kSlab * kRowBytes;  // 8 KiB
constexpr int kRing = 4;
constexpr float kMostSum = 256.f;         // of a lane's weights in a step (far from where fp16 ends)
constexpr float kNoReference = -3e38f;   // of a row that has met no score yet: finite, so that exp2 never sees inf - inf

template <int N>
using IC = std::integral_constant<int, N>;

enum Kind { kNone, kFull, kMasked };

}  // namespace

template <typename T>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(2, 2))) void window_fwd_kernel(const WindowParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];  // K ring [4][8 KiB] | V ring [4][8 KiB]
  using x8 = x8_of<T>;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int item = window_item(blockIdx.x, p.chunk);
  if (item >= p.items) return;
  // the query heads of a group together, then from tile to tile, late (under a long causal window: long) tiles first
  const int group = p.Hq / p.Hkv;
  const int g = item % group;
  item /= group;
  const int tile = p.tiles - 1 - item % p.tiles;
  item /= p.tiles;
  const int hkv = item % p.Hkv, b = item / p.Hkv, hq = hkv * group + g;

  const int len = p.lengths != nullptr ? min(max(const_idx(p.lengths)[b], 0), p.Skv) : p.Skv;
  const int rows = p.lengths != nullptr ? len : p.Sq;  // that are not padding
  const int shift = p.lengths != nullptr ? 0 : p.Skv - p.Sq;
  const int row0 = tile * kWindowTile, ahead = p.causal ? 0 : p.window - 1;
  const int last_row = min(row0 + kWindowTile, rows) - 1;  // below row0: all padding
  // sinks that position `at` sees
  auto sinks_at = [&](int at) { return min(min(p.sinks, len), p.causal ? at + 1 : p.sinks); };

  // slabs of the tile
  int n_sink = 0, first = 0, n = 0;
  if (last_row >= row0 && len > 0) {
    const int low = max(0, row0 + shift - p.window + 1), high = min(len - 1, last_row + shift + ahead);
    n_sink = (max(0, sinks_at(last_row + shift)) + kSlab - 1) / kSlab;
    first = max(low / kSlab, n_sink);
    n = n_sink + (high >= low ? max(0, high / kSlab + 1 - first) : 0);
  }
  auto slab_of = [&](int t) { return t < n_sink ? t : first + t - n_sink; };

  // what this lane's row sees: keys lo .. hi and those below sk; what the wave's rows see
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

  const char* const kp = p.k.ptr + b * p.k.batch + hkv * p.k.head;
  const char* const vp = p.v.ptr + b * p.v.batch + hkv * p.v.head;
  const int64_t k_step = (int64_t)p.k.row * kSlab, v_step = (int64_t)p.v.row * kSlab;

  f32x16 acc[4];
  float l_run = 0.f, m_run = kNoReference;
  const float c = p.scale_log2e;
#pragma unroll
  for (int mb = 0; mb < 4; ++mb)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[mb][r] = 0.f;

  if (n > 0) {
    // Q as the B operand: lane holds row l32, d = 16 ks + 8 h .. +7 (rows behind the last: that one)
    x8 qreg[8];
    const char* qp = p.q.ptr + b * p.q.batch + hq * p.q.head + (int64_t)min(row, rows - 1) * p.q.row;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) qreg[ks] = *reinterpret_cast<const x8*>(qp + 32 * ks + 16 * h);
    RowMajorOffsets rm;
    rm.init(lane);
    TransposedOffsets tr;
    tr.init(lane);
    RowDma k_dma, v_dma;
    k_dma.init(wave, lane, p.k.row, len - 1);
    v_dma.init(wave, lane, p.v.row, len - 1);
    const LdsPtr k_lds = lds_ptr(smem), v_lds = lds_ptr(smem + kRing * kSlabBytes);
    const uint32_t k_dst = lds_addr(smem), v_dst = k_dst + kRing * kSlabBytes;
    // past the last slab: that one again, into a buffer that nobody reads any more, so that the counter of copies in flight means the same at every wait
    auto slab_at = [&](int t) { return slab_of(min(t, n - 1)); };

#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int slab = slab_at(j);
      k_dma.copy(k_dst + j * kSlabBytes, kp + slab * k_step, slab);
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int slab = slab_at(j);
      v_dma.copy(v_dst + j * kSlabBytes, vp + slab * v_step, slab);
    }
    wait_vmem<0>();
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) pin(qreg[ks]);

    auto scores = [&](LdsPtr slab) {  // S^T of a slab
      f32x16 s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) s = Elem<T>::mfma32(read_b128<T>(slab + rm.rd[ks]), qreg[ks], s);
      return s;
    };
    int kind_before = kNone;  // of the slab before the step's
    f32x16 s_cur = scores(k_lds);
    pin(s_cur);
    __syncthreads();

    x8 p_prev[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) p_prev[j][i] = (T)0.f;

    // O += P V of the slab in `buf`; `between` runs behind the matrix instructions
    auto add_pv = [&](LdsPtr buf, auto between) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) {
          const int roff = 16 * j * kRowBytes;
          acc[mb] = Elem<T>::mfma32(read_tr8<T>(buf + tr.rd[mb][0] + roff, buf + tr.rd[mb][1] + roff), p_prev[j], acc[mb]);
          between(4 * j + mb);
        }
    };
    // p_prev := P_t against the rows' reference m.  Where they add up to more than kMostSum, m has fallen behind: it is raised, with what has been summed, and they are formed anew.
    // (The sum is there anyway; the maximum in front of every step costs H24/6 S69120 window 1536 1585 us instead of 1550, both on a card slower than that of the figures above.)
    auto weights = [&]() {
      const typename Elem<T>::x2 one2 = {(T)1.f, (T)1.f};
      float sum[2];
      auto form = [&]() __attribute__((always_inline)) {
        const float mc = m_run * c;
        f32x16 w;
#pragma unroll
        for (int r = 0; r < 16; ++r) w[r] = fast_exp2(__builtin_fmaf(s_cur[r], c, -mc));
        sum[0] = sum[1] = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          // rounded to T as the matrix instruction takes it; the denominator sums the rounded values, so that the weights still add up to one (lse, of that sum, is off by half
          // a step of T at most for it; backward finds the sum before rounding, where there is more time for sixteen additions: 25 us against 130)
          p_prev[j] = narrow8<T>(w, j);
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[j] = Elem<T>::dot2((typename Elem<T>::x2){p_prev[j][2 * i], p_prev[j][2 * i + 1]}, one2, sum[j]);
        }
        sum[0] += sum[1];
      };
      form();
      if (__builtin_amdgcn_ballot_w64(sum[0] > kMostSum) != 0) {
        float mx = s_cur[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s_cur[r]);
        // (of the rows that need it only, so that a row's result does not depend on its neighbours)
        const float top = max_halves(mx), m_new = max_halves(sum[0]) > kMostSum ? fmaxf(m_run, top) : m_run;
        const float alpha = fast_exp2((m_run - m_new) * c);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int mb = 0; mb < 4; ++mb)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[mb][r] *= alpha;
        form();
      }
      l_run += sum[0];
      pin(p_prev[0]);
      pin(p_prev[1]);
    };
    // Step t (t % 4 == R): O += P_{t-1} V_{t-1} | softmax(S_t) | S_{t+1} = K_{t+1} Q^T.  P_{t-1} was formed against the reference m of step t-1, so it reaches O before
    // step t may raise m.  The copies that a step owes, K_{t+4} into the buffer of K_t and V_{t+2} into that of V_{t-2}, go in front of the matrix instructions (between
    // them in steps without masks).  Behind it K_{t+2} and V_t must have landed; what steps t-1 and t requested may still fly.
    auto step = [&](auto ring_c, int t) {
      constexpr int R = decltype(ring_c)::value;
      const int k_slab = slab_at(t + 4), v_slab = slab_at(t + 2);
      k_dma.copy(k_dst + R * kSlabBytes, kp + k_slab * k_step, k_slab);
      if (t > 0) v_dma.copy(v_dst + ((R + 2) & 3) * kSlabBytes, vp + v_slab * v_step, v_slab);  // (the first three V slabs are there)
      if (kind_before != kNone) add_pv(v_lds + ((R + 3) & 3) * kSlabBytes, [](int) {});
      const int kind = kind_of(t);
      if (kind != kFull) {
        const int k0 = slab_of(t) * kSlab + 4 * h, a = lo - k0, z = hi - k0, y = sk - k0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int e = 8 * (r >> 2) + (r & 3);
          s_cur[r] = (e >= a && e <= z) || e < y ? s_cur[r] : -INFINITY;
        }
      }
      // (Where no row sees the slab its weights are zero, and V is not touched.  A branch around the products costs registers that are not there: what was spilled came back behind
      // the copies in flight, 4100 cycles a step instead of 1600; H24 S30720 window 128 315 us instead of 243.)
      const f32x16 s_nxt = scores(k_lds + ((R + 1) & 3) * kSlabBytes);
      weights();
      s_cur = s_nxt;
      kind_before = kind;
      wait_vmem<8>();
      __syncthreads();
    };
    // The same where all rows of the tile see slabs t-1, t and t+1 whole, and no slab that is requested is the last one.
    const char *k_src = kp, *v_src = vp;
    auto whole_step = [&](auto ring_c) {
      constexpr int R = decltype(ring_c)::value;
      const uint32_t k_into = k_dst + R * kSlabBytes, v_into = v_dst + ((R + 2) & 3) * kSlabBytes;
      add_pv(v_lds + ((R + 3) & 3) * kSlabBytes, [&](int i) {
        if (i == 0) dma16(k_into + k_dma.wave_dst, k_src, k_dma.off[0]);
        if (i == 2) dma16(k_into + k_dma.wave_dst + 4 * kRowBytes, k_src, k_dma.off[1]);
        if (i == 4) dma16(v_into + v_dma.wave_dst, v_src, v_dma.off[0]);
        if (i == 6) dma16(v_into + v_dma.wave_dst + 4 * kRowBytes, v_src, v_dma.off[1]);
      });
      const f32x16 s_nxt = scores(k_lds + ((R + 1) & 3) * kSlabBytes);
      weights();
      s_cur = s_nxt;
      wait_vmem<8>();
      __syncthreads();
      k_src += k_step;
      v_src += v_step;
    };
    // steps [from, to) of the window's slabs that are whole for all rows of the tile
    const int whole_lo = max(0, last_row + shift - p.window + 1), whole_hi = min(len - 1, row0 + shift + ahead);
    const int from = n_sink + max(0, (whole_lo + kSlab - 1) / kSlab - first);
    const int to = row0 + kWindowTile <= rows ? n_sink + (whole_hi + 1) / kSlab - first : 0;
    const int whole_end = min(to - 1, n - 5);  // of the steps that whole_step takes
    for (int t = 0; t < n;) {
      if (t > from && t + 4 <= whole_end) {
        k_src = kp + slab_of(t + 4) * k_step;
        v_src = vp + slab_of(t + 2) * v_step;
        do {
          whole_step(IC<0>{});
          whole_step(IC<1>{});
          whole_step(IC<2>{});
          whole_step(IC<3>{});
          t += 4;
        } while (t + 4 <= whole_end);
        kind_before = kFull;
      }
      step(IC<0>{}, t);
      if (t + 1 < n) step(IC<1>{}, t + 1);
      if (t + 2 < n) step(IC<2>{}, t + 2);
      if (t + 3 < n) step(IC<3>{}, t + 3);
      t += 4;
    }
    if (kind_before != kNone) add_pv(v_lds + ((n - 1) & 3) * kSlabBytes, [](int) {});
    wait_vmem<0>();   // no copy may still be writing LDS
    __syncthreads();  // and everybody is done with the rings
  }

  const float l = sum_halves(l_run);
  if (h == 0 && row < p.Sq) p.lse[((int64_t)b * p.Hq + hq) * p.Sq + row] = l > 0.f ? m_run * c + __builtin_log2f(l) : INFINITY;
  const float scale = l > 0.f ? 1.f / l : 0.f;
  store_tile<T>(smem + wave * kSlabBytes, acc, scale, p.o.ptr + b * p.o.batch + hq * p.o.head + (int64_t)wrow0 * p.o.row, p.o.row, lane, p.Sq - wrow0);
  if (p.o_low.ptr != nullptr)  // for backward
    store_tile<T, true>(smem + wave * kSlabBytes, acc, scale, p.o_low.ptr + b * p.o_low.batch + hq * p.o_low.head + (int64_t)wrow0 * p.o_low.row, p.o_low.row, lane, p.Sq - wrow0);
}

hipError_t launch_window_fwd(WindowParams p, bool half, hipStream_t stream) {
  constexpr int kSmem = 2 * kRing * kSlabBytes;
  p.tiles = (p.Sq + kWindowTile - 1) / kWindowTile;
  p.items = p.B * p.Hq * p.tiles;
  p.chunk = window_chunk(p.items);
  void (*fn)(const WindowParams) = half ? &window_fwd_kernel<_Float16> : &window_fwd_kernel<__bf16>;
  hipLaunchKernelGGL(fn, dim3(window_grid(p.items, p.chunk)), dim3(256), kSmem, stream, p);
  return hipGetLastError();
}

}  // namespace fba
