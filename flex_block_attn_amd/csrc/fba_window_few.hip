// Attention under a sliding window with sinks where there are few query rows: forward, and dQ with delta.  gfx950, head_dim 128, bf16 or fp16.
//
// The same products as in fba_window_fwd.hip and fba_window_dq.hip, dealt out otherwise: a work-group has 32 query rows, and its four waves take the slabs of 32 keys in turn,
// each through a K slab and a V slab of its own in LDS, so that there is no barrier before the end, where the four sums meet in LDS.  A launch has four times the
// work-groups, each with a quarter of the steps one after the other; K and V are read four times as often, from L2.
// For launches that leave most compute units without a 128-row tile: bound by latency, of the first loads and of each step
// (H1 S768 window 128: forward 7 us of which the launch is 3; B2 H8/2 S3136 window 384, padded: dK and dV 55).
#include "fba_types.h"
#include "fba_window.h"
#include "fba_window_keys.h"

namespace fba {

namespace {

constexpr int kSlab = 32;
constexpr int kSlabBytes = kSlab * kRowBytes;
constexpr int kRows = 32;
constexpr int kWaves = 4;
constexpr float kLazy = 8.f, kNoReference = -3e38f;

// until at most N copies are in flight; nothing moves across
template <int N>
FBA_DEVICE void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
FBA_DEVICE void wait_fetches() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

}  // namespace

template <typename T, bool kBackward>
__global__ __attribute__((amdgpu_flat_work_group_size(64 * kWaves, 64 * kWaves), amdgpu_waves_per_eu(2, 2))) void window_few_kernel(const WindowParams p) {
  __shared__ __attribute__((aligned(16))) char smem[kWaves * 2 * kSlabBytes];  // [wave][K slab | V slab]; at the end [wave][32 rows][128] floats
  __shared__ float ml[2][kWaves][kRows];
  using x8 = x8_of<T>;
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

  // slabs of the tile and what every row sees, as in the other kernels
  const int len = p.lengths != nullptr ? min(max(const_idx(p.lengths)[b], 0), p.Skv) : p.Skv;
  const int rows = p.lengths != nullptr ? len : p.Sq;
  const int shift = p.lengths != nullptr ? 0 : p.Skv - p.Sq;
  const int row0 = tile * kRows, ahead = p.causal ? 0 : p.window - 1;
  const int last_row = min(row0 + kRows, rows) - 1;
  auto sinks_at = [&](int at) { return min(min(p.sinks, len), p.causal ? at + 1 : p.sinks); };
  int n_sink = 0, first = 0, n = 0;
  if (last_row >= row0 && len > 0) {
    const int low = max(0, row0 + shift - p.window + 1), high = min(len - 1, last_row + shift + ahead);
    n_sink = (max(0, sinks_at(last_row + shift)) + kSlab - 1) / kSlab;
    first = max(low / kSlab, n_sink);
    n = n_sink + (high >= low ? max(0, high / kSlab + 1 - first) : 0);
  }
  auto slab_of = [&](int t) { return t < n_sink ? t : first + t - n_sink; };
  const int row = row0 + l32, at = row + shift;
  const bool there = row < rows;
  const int hi = there ? min(len - 1, at + ahead) : -1, lo = at - p.window + 1, sk = there ? sinks_at(at) : 0;
  const int tile_first = row0 + shift, tile_last = last_row + shift;
  const int all_hi = row0 + kRows <= rows ? min(len - 1, tile_first + ahead) : -1, all_lo = tile_last - p.window + 1, all_sk = row0 + kRows <= rows ? sinks_at(tile_first) : 0;

  f32x16 acc[4];
#pragma unroll
  for (int mb = 0; mb < 4; ++mb)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[mb][r] = 0.f;
  float m_run = kNoReference, l_run = 0.f;
  const float c = p.scale_log2e;

  if (last_row >= row0) {
    const char* const kp = p.k.ptr + b * p.k.batch + hkv * p.k.head;
    const char* const vp = p.v.ptr + b * p.v.batch + hkv * p.v.head;
    const uint32_t k_dst = lds_addr(smem) + wave * 2 * kSlabBytes;
    // a slab by one wave: 4 rows to a copy (rows behind the last key: that one, they are masked)
    auto request = [&](uint32_t dst, const char* src, uint32_t stride, int slab) __attribute__((always_inline)) {
      const int last = len - 1 - slab * kSlab;
      const char* const from = src + (int64_t)slab * kSlab * stride;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 4);
        dma16(dst + i * 4 * kRowBytes, from, (uint32_t)min(r, last) * stride + (((lane & 15) ^ swz(r)) << 4));
      }
    };
    // forward reads K, then V; backward V, then K
    if (wave < n && !kBackward) request(k_dst, kp, p.k.row, slab_of(wave));
    if (wave < n) request(k_dst + kSlabBytes, vp, p.v.row, slab_of(wave));
    if (wave < n && kBackward) request(k_dst, kp, p.k.row, slab_of(wave));
    // Q (and dO) as B operands: lane holds row l32, d = 16 ks + 8 h .. +7 (rows behind the last: that one)
    x8 qreg[8], doreg[8];
    float lse2 = 0.f, neg_delta = 0.f;
    const int from = min(row, rows - 1);
    const char* const qp = p.q.ptr + b * p.q.batch + hq * p.q.head + (int64_t)from * p.q.row + 16 * h;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) qreg[ks] = *reinterpret_cast<const x8*>(qp + 32 * ks);
    if constexpr (kBackward) {
      const char* const dp = p.d_o.ptr + b * p.d_o.batch + hq * p.d_o.head + (int64_t)from * p.d_o.row + 16 * h;
      const char* const op = p.o.ptr + b * p.o.batch + hq * p.o.head + (int64_t)from * p.o.row + 16 * h;
      const char* const lp = p.o_low.ptr == nullptr ? op : p.o_low.ptr + b * p.o_low.batch + hq * p.o_low.head + (int64_t)from * p.o_low.row + 16 * h;
      const float low = p.o_low.ptr == nullptr ? 0.f : 1.f;
      const int64_t stat = ((int64_t)b * p.Hq + hq) * p.Sq + from;
      lse2 = p.lse[stat];
      float sum = 0.f;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        doreg[ks] = *reinterpret_cast<const x8*>(dp + 32 * ks);
        const x8 o8 = *reinterpret_cast<const x8*>(op + 32 * ks), l8 = *reinterpret_cast<const x8*>(lp + 32 * ks);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = __builtin_fmaf((float)doreg[ks][i], __builtin_fmaf(low, (float)l8[i], (float)o8[i]), sum);
      }
      neg_delta = -sum_halves(sum);
      if (wave == 0 && h == 0 && there) p.neg_delta[stat] = neg_delta;
    }
    RowMajorOffsets rm;
    rm.init(lane);
    TransposedOffsets tr;
    tr.init(lane);
    const LdsPtr kt = lds_ptr(smem + wave * 2 * kSlabBytes), vt = kt + kSlabBytes;

    for (int t = wave; t < n; t += kWaves) {
      const int slab = slab_of(t), k0 = slab * kSlab;
      const bool more = t + kWaves < n, whole = (k0 + kSlab - 1 <= all_hi && k0 >= all_lo) || k0 + kSlab - 1 < all_sk;
      const int after = slab_of(min(t + kWaves, n - 1));
      f32x16 s, d;
#pragma unroll
      for (int r = 0; r < 16; ++r) { s[r] = 0.f; d[r] = neg_delta; }
      wait_copies<8>();  // the first of the two is there, the other may still fly
      if constexpr (kBackward) {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) d = Elem<T>::mfma32(read_b128<T>(vt + rm.rd[ks]), doreg[ks], d);
        wait_fetches();
        if (more) request(k_dst + kSlabBytes, vp, p.v.row, after);
        if (more) wait_copies<8>(); else wait_copies<0>();
      }
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) s = Elem<T>::mfma32(read_b128<T>(kt + rm.rd[ks]), qreg[ks], s);
      if constexpr (!kBackward) {
        wait_fetches();
        if (more) request(k_dst, kp, p.k.row, after);
      }
      if (!whole) {
        const int a = lo - k0 - 4 * h, z = hi - k0 - 4 * h, y = sk - k0 - 4 * h;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int e = 8 * (r >> 2) + (r & 3);
          s[r] = (e >= a && e <= z) || e < y ? s[r] : -INFINITY;
        }
      }
      x8 pk[2];
      if constexpr (kBackward) {
        // a masked value is zero whatever dP is there
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float pv = fast_exp2(__builtin_fmaf(s[r], c, -lse2));
          l_run += pv;
          s[r] = s[r] == -INFINITY ? 0.f : pv * d[r];
        }
      } else {
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        if (__builtin_amdgcn_ballot_w64((mx - m_run) * c > kLazy) != 0) {
          // (of the rows that need it only, so that a row's result does not depend on its neighbours)
          const float top = max_halves(mx), m_new = (top - m_run) * c > kLazy ? top : m_run, alpha = fast_exp2((m_run - m_new) * c);
          m_run = m_new;
          l_run *= alpha;
#pragma unroll
          for (int mb = 0; mb < 4; ++mb)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[mb][r] *= alpha;
        }
        const float mc = m_run * c;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fast_exp2(__builtin_fmaf(s[r], c, -mc));
      }
      // rounded to T as the matrix instruction takes it (P: the denominator sums the rounded values)
#pragma unroll
      for (int j = 0; j < 2; ++j) pk[j] = narrow8<T>(s, j);
      if constexpr (!kBackward) {
        const typename Elem<T>::x2 one2 = {(T)1.f, (T)1.f};
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) l_run = Elem<T>::dot2((typename Elem<T>::x2){pk[j][2 * i], pk[j][2 * i + 1]}, one2, l_run);
        if (more) wait_copies<8>(); else wait_copies<0>();  // V is there, the next K may still fly
      }
      const LdsPtr from_lds = kBackward ? kt : vt;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) {
          const int roff = 16 * j * kRowBytes;
          acc[mb] = Elem<T>::mfma32(read_tr8<T>(from_lds + tr.rd[mb][0] + roff, from_lds + tr.rd[mb][1] + roff), pk[j], acc[mb]);
        }
      wait_fetches();
      if (more) {
        if constexpr (kBackward) request(k_dst, kp, p.k.row, after);
        else request(k_dst + kSlabBytes, vp, p.v.row, after);
      }
    }
  }

  // The waves' sums meet in LDS, each where its slabs were: 32 rows of 512 bytes, 16-byte chunk c of row r at place c ^ r.
  wait_fetches();
  {
    char* const own = smem + wave * 2 * kSlabBytes;
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(own + l32 * 512 + (((8 * mb + 2 * i + h) ^ l32) << 4)) = (f32x4){acc[mb][4 * i + 0], acc[mb][4 * i + 1], acc[mb][4 * i + 2], acc[mb][4 * i + 3]};
    const float l = sum_halves(l_run);  // (backward: the sum of P)
    if (h == 0) {
      ml[0][wave][l32] = m_run;
      ml[1][wave][l32] = l;
    }
  }
  __syncthreads();
  const int r = tid >> 3;  // a row to 8 threads
  if (row0 + r >= p.Sq) return;
  float factor[kWaves], scale = p.scale;
  if constexpr (kBackward) {
#pragma unroll
    for (int w = 0; w < kWaves; ++w) factor[w] = 1.f;
    const float l = ml[1][0][r] + ml[1][1][r] + ml[1][2][r] + ml[1][3][r];  // as in fba_window_dq.hip
    if (l > 0.f) scale /= l;
    if ((tid & 7) == 0 && row0 + r < rows) {
      const int64_t stat = ((int64_t)b * p.Hq + hq) * p.Sq + row0 + r;
      p.lse_exact[stat] = p.lse[stat] + (l > 0.f ? __builtin_log2f(l) : 0.f);
    }
  } else {
    float m = kNoReference, l = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, ml[0][w][r]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      factor[w] = fast_exp2((ml[0][w][r] - m) * c);
      l += factor[w] * ml[1][w][r];
    }
    scale = l > 0.f ? 1.f / l : 0.f;
    if ((tid & 7) == 0) p.lse[((int64_t)b * p.Hq + hq) * p.Sq + row0 + r] = l > 0.f ? m * c + __builtin_log2f(l) : INFINITY;
  }
  const Strided& out = kBackward ? p.dq : p.o;
  char* const to = out.ptr + b * out.batch + hq * out.head + (int64_t)(row0 + r) * out.row;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int chunk = 8 * j + (tid & 7);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += factor[w] * *reinterpret_cast<const f32x4*>(smem + w * 2 * kSlabBytes + r * 512 + ((chunk ^ r) << 4));
    sum *= scale;
    const x4_of<T> value = narrow4<T>(sum[0], sum[1], sum[2], sum[3]);
    *reinterpret_cast<x4_of<T>*>(to + chunk * 8) = value;
    if (!kBackward && p.o_low.ptr != nullptr)
      *reinterpret_cast<x4_of<T>*>(p.o_low.ptr + b * p.o_low.batch + hq * p.o_low.head + (int64_t)(row0 + r) * p.o_low.row + chunk * 8) =
          narrow4<T>(sum[0] - (float)value[0], sum[1] - (float)value[1], sum[2] - (float)value[2], sum[3] - (float)value[3]);
  }
}

// dK and dV of 32 keys: the four waves take slabs of 32 query rows in turn, each through a Q slab and a dO slab of its own.  K and V rows are B operands in registers,
// lane = key; products and masks as in fba_window_dkdv.hip.
namespace {
constexpr int kStageBytes = 2 * kSlabBytes + 2 * kSlab * 4;  // Q slab | dO slab | lse2 | -delta
constexpr int kFewPartFloats = 2 * kRows * kHeadDim;
}  // namespace

template <typename T>
__global__ __attribute__((amdgpu_flat_work_group_size(64 * kWaves, 64 * kWaves), amdgpu_waves_per_eu(2, 2))) void window_few_dkdv_kernel(const WindowParams p) {
  __shared__ __attribute__((aligned(256))) char smem[kWaves * kStageBytes];  // at the end [wave][32 keys][128] floats, dV and then dK
  using x8 = x8_of<T>;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int index = window_item(blockIdx.x, p.chunk);
  if (index >= p.items) return;
  const KeyItem item = key_item(p, index);
  const RowSlabs& slabs = item.slabs;
  const int b = item.b, hkv = item.hkv, group = p.Hq / p.Hkv, len = item.len, rows = item.rows, n = item.n, key0 = item.key0;
  const KeyMask mask(p, item, key0);

  f32x16 acc_k[4], acc_v[4];
#pragma unroll
  for (int mb = 0; mb < 4; ++mb)
#pragma unroll
    for (int r = 0; r < 16; ++r) { acc_k[mb][r] = 0.f; acc_v[mb][r] = 0.f; }

  if (wave < n) {
    x8 kreg[8], vreg[8];
    {
      const int key = min(key0 + l32, len - 1);
      const char* const kp = p.k.ptr + b * p.k.batch + hkv * p.k.head + (int64_t)key * p.k.row + 16 * h;
      const char* const vp = p.v.ptr + b * p.v.batch + hkv * p.v.head + (int64_t)key * p.v.row + 16 * h;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        kreg[ks] = *reinterpret_cast<const x8*>(kp + 32 * ks);
        vreg[ks] = *reinterpret_cast<const x8*>(vp + 32 * ks);
      }
    }
    const char* const qb = p.q.ptr + b * p.q.batch + (int64_t)hkv * group * p.q.head;
    const char* const db = p.d_o.ptr + b * p.d_o.batch + (int64_t)hkv * group * p.d_o.head;
    const char* const sb = reinterpret_cast<const char*>(p.lse + ((int64_t)b * p.Hq + hkv * group) * p.Sq);
    const uint32_t dst = lds_addr(smem) + wave * kStageBytes;
    const uint32_t stat_off = (uint32_t)(h * ((const char*)p.neg_delta - (const char*)p.lse));
    // Slab s_begin + t; the last slab of the rows is moved back to end with them (its first rows are masked then).
    const int tail = max(0, rows - kSlab), least = min(31, rows - 1);
    int g = (item.s_begin + wave) / slabs.n, i_slab = (item.s_begin + wave) % slabs.n, row_min = slabs.at(i_slab) * kSlab, row0 = min(row_min, tail);
    uint32_t off[8];  // of Q and dO, whose rows are equally far apart
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 4);
      off[i] = (uint32_t)min(r, least) * p.q.row + (((lane & 15) ^ swz(r)) << 4);
      asm volatile("" : "+v"(off[i]));  // (worked out again in every step otherwise)
    }
    auto request = [&](uint32_t to, const char* from) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) dma16(to + i * 4 * kRowBytes, from, off[i]);
    };
    auto request_do = [&](int g, int row0) __attribute__((always_inline)) {
      request(dst + kSlabBytes, db + g * p.d_o.head + (int64_t)row0 * p.d_o.row);
      dma4(dst + 2 * kSlabBytes, sb + ((int64_t)g * p.Sq + row0) * 4, stat_off + min(l32, least) * 4);
    };
    auto request_q = [&](int g, int row0) __attribute__((always_inline)) { request(dst, qb + g * p.q.head + (int64_t)row0 * p.q.row); };
    request_do(g, row0);
    request_q(g, row0);

    RowMajorOffsets rm;
    rm.init(lane);
    TransposedOffsets tr;
    tr.init(lane);
    // operand steps and column blocks only move the 16-byte chunk inside a 256-byte row, by an exclusive-or
    static_assert(kStageBytes % 256 == 0 && kSlabBytes % 256 == 0, "the exclusive-ors below touch bits 5..7");
    const LdsPtr st = lds_ptr(smem + wave * kStageBytes), q_base = st + rm.rd[0], t_base = st + tr.rd[0][0], stat = st + 2 * kSlabBytes + 16 * h;
    auto flip = [](LdsPtr ptr, uint32_t bits) { return (LdsPtr)(uintptr_t)((uint32_t)(uintptr_t)ptr ^ bits); };
    const float c = p.scale_log2e;
    for (int t = wave; t < n; t += kWaves) {
      wait_copies<0>();
      f32x16 s, dp;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 d4 = lds_read_f32x4(stat + 4 * kSlab + 32 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) { s[4 * i + e] = 0.f; dp[4 * i + e] = d4[e]; }
      }
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        s = Elem<T>::mfma32(read_b128<T>(flip(q_base, 32u * ks)), kreg[ks], s);
        dp = Elem<T>::mfma32(read_b128<T>(flip(q_base, 32u * ks) + kSlabBytes), vreg[ks], dp);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 l4 = lds_read_f32x4(stat + 32 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float pv = fast_exp2(__builtin_fmaf(s[4 * i + e], c, -l4[e]));
          s[4 * i + e] = pv;
          dp[4 * i + e] = pv * dp[4 * i + e];
        }
      }
      if (!mask.whole(row0, row_min)) mask.apply(s, dp, row0, row_min, lane);
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
        }
      // (past the last slab: that one again, into places that nobody reads any more)
      if (t + kWaves < n)
        for (i_slab += kWaves; i_slab >= slabs.n; i_slab -= slabs.n) ++g;
      row_min = slabs.at(i_slab) * kSlab;
      const int next0 = min(row_min, tail);
      wait_fetches();
      request_do(g, next0);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) {
          const LdsPtr t0 = flip(t_base, (uint32_t)(mb << 6)) + 16 * j * kRowBytes, t1 = flip(t_base, (uint32_t)(mb << 6 | 32)) + (16 * j + 8) * kRowBytes;
          acc_k[mb] = Elem<T>::mfma32(read_tr8<T>(t0, t1), dsk[j], acc_k[mb]);
        }
      wait_fetches();
      request_q(g, next0);
      row0 = next0;
    }
    wait_copies<0>();
  }

  // The waves' sums meet in LDS, dV first: 32 rows of 512 bytes each, 16-byte chunk c of row r at place c ^ r.
  auto finish = [&](const f32x16(&acc)[4], int which, const Strided& out, float scale) __attribute__((always_inline)) {
    __syncthreads();
    char* const own = smem + wave * kRows * 512;
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(own + l32 * 512 + (((8 * mb + 2 * i + h) ^ l32) << 4)) = (f32x4){acc[mb][4 * i + 0], acc[mb][4 * i + 1], acc[mb][4 * i + 2], acc[mb][4 * i + 3]};
    __syncthreads();
    const int r = tid >> 3;  // a row to 8 threads
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int chunk = 8 * j + (tid & 7);
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) sum += *reinterpret_cast<const f32x4*>(smem + w * kRows * 512 + r * 512 + ((chunk ^ r) << 4));
      if (item.in_parts)
        *reinterpret_cast<f32x4*>(p.parts + item.place * kFewPartFloats + which * (kRows * kHeadDim) + r * kHeadDim + 4 * chunk) = sum;
      else if (key0 + r < p.Skv)
        *reinterpret_cast<x4_of<T>*>(out.ptr + b * out.batch + hkv * out.head + (int64_t)(key0 + r) * out.row + chunk * 8) = narrow4<T>(sum[0] * scale, sum[1] * scale, sum[2] * scale, sum[3] * scale);
    }
  };
  finish(acc_v, 0, p.dv, 1.f);
  finish(acc_k, 1, p.dk, p.scale);
}

// Which launches.  Rows: dQ where tiles of 128 rows leave half of the compute units idle and more; forward, which reads less, up to seven eighths of them, and up to all where the
// keys of a row are not many.  Keys: up to an eighth of the compute units, and up to half of them as long as a tile does not have the rows to be cut into several items.
// Tiles of 128 / of 32, in us (causal, no sinks; backward: dQ, dK and dV, replayed from a graph):
//   window, forward            128         256         512         1024        2048        4096        backward  128         512         2048
//      32 tiles (H1 S4096)     15 / 8      18 / 9      22 / 10     29 / 14     44 / 20     67 / 32               35 / 27     54 / 40     98 / 60
//     100 (B2 H2 S3136)        15 / 10     18 / 11     23 / 14     35 / 18     61 / 26                           43 / 39     60 / 52     123 / 89
//     128 (B4 H4 S1024)        15 / 10     18 / 11     23 / 14     25 / 16                                       43 / 38     59 / 49
//     200 (B2 H4 S3136)        16 / 15     18 / 18     23 / 22     35 / 30     62 / 38                           46 / 53     68 / 75     158 / 139
//     256 (H4 S8192)           16 / 16     19 / 19     24 / 24     31 / 35     46 / 57     75 / 104              51 / 58     75 / 79     160 / 171
//     384 (H6 S8192)           22 / 23     26 / 27     33 / 35     47 / 50     74 / 84     120 / 152             67 / 76     102 / 112   239 / 254
//     512 (H8 S8192)           25 / 31     29 / 36     36 / 46     49 / 66     76 / 110    121 / 200             71 / 90     107 / 126   243 / 288
//   keys, backward              window 128  512         1024        2048
//      16 tiles (H4/1 S2048)   52 / 35     55 / 46     61 / 53     81 / 62
//      20 (H8/1 S2560)         64 / 48     77 / 69     106 / 92    165 / 134
//      32 (H4/1 S4096)         59 / 42     66 / 58     76 / 74     100 / 98
//     100 (B2 H8/2 S3136)      79 / 60     110 / 103   148 / 154   216 / 242
bool window_takes_few(const WindowParams& p, int compute_units, bool backward) {
  const int64_t tiles = (int64_t)p.B * p.Hq * ((p.Sq + kWindowTile - 1) / kWindowTile);
  if (2 * tiles <= compute_units) return true;
  if (backward) return false;
  const int window = p.causal ? p.window : 2 * p.window - 1, keys = (window < p.Skv ? window : p.Skv) + p.sinks;
  return 8 * tiles <= 7 * compute_units || (tiles <= compute_units && keys <= 512);
}
bool window_keys_few(const WindowParams& p, int compute_units) {
  const int64_t tiles = (int64_t)p.B * p.Hkv * ((p.Skv + kWindowTile - 1) / kWindowTile);
  if (8 * tiles <= compute_units) return true;
  const int window = p.causal ? p.window : 2 * p.window - 1;
  const int64_t rows = (int64_t)(p.Hq / p.Hkv) * (window < p.Sq ? window : p.Sq);
  return 2 * tiles <= compute_units && rows <= 4096;
}

hipError_t launch_window_few_dkdv(WindowParams p, bool half, hipStream_t stream) {
  hipLaunchKernelGGL((half ? &window_few_dkdv_kernel<_Float16> : &window_few_dkdv_kernel<__bf16>), dim3(window_grid(p.items, p.chunk)), dim3(64 * kWaves), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_window_few(WindowParams p, bool half, bool backward, hipStream_t stream) {
  p.tiles = (p.Sq + kRows - 1) / kRows;
  p.items = p.B * p.Hq * p.tiles;
  p.chunk = window_chunk(p.items);
  void (*fn)(const WindowParams) = half ? (backward ? &window_few_kernel<_Float16, true> : &window_few_kernel<_Float16, false>)
                                        : (backward ? &window_few_kernel<__bf16, true> : &window_few_kernel<__bf16, false>);
  hipLaunchKernelGGL(fn, dim3(window_grid(p.items, p.chunk)), dim3(64 * kWaves), 0, stream, p);
  return hipGetLastError();
}

}  // namespace fba
