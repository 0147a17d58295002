// Rotary positions of q and k: gfx950, bf16 or fp16, head_dim 128.  The mathematics stand in fba_rotary.h; the gradient is the rotation back.
//
// Bound by device memory: a row is read and written once.  Sixteen lanes have a token and go through its heads, four rows in flight, so that sines and cosines are worked out once
// for all of them; where tokens are few the heads are cut into parts, each of which works them out again.
#include "fba_turn.h"

namespace fba {

template <typename T>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p) {
  const int c = threadIdx.x & 15;
  const uint32_t unit = blockIdx.x * 16 + (threadIdx.x >> 4);
  const uint32_t part = unit / p.tokens, n = unit - part * p.tokens;
  if (part >= p.parts) return;
  const uint32_t b = n / (uint32_t)p.seq;
  const int t = (int)(n - b * (uint32_t)p.seq);
  Turn turn;
  turn.init(p.rotation, Columns(p.rotation, c), b, t, t);
  const bool interleaved = p.rotation.interleaved != 0;
  const int first = part * p.per, end = min(first + (int)p.per, p.heads + p.kv_heads);
  auto rows = [&](const Strided& x, const Strided& out, int h0, int h1) {
    const char* const from = x.ptr + b * x.batch + (int64_t)t * x.row + c * 16;
    char* const to = out.ptr + b * out.batch + (int64_t)t * out.row + c * 16;
    for (int h = h0; h < h1; h += 4) {
      x8_of<T> r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (h + i < h1) r[i] = *reinterpret_cast<const x8_of<T>*>(from + (h + i) * x.head);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (h + i < h1) *reinterpret_cast<x8_of<T>*>(to + (h + i) * out.head) = turned<T>(r[i], turn, interleaved);
    }
  };
  rows(p.q, p.q_out, first, min(end, p.heads));
  rows(p.k, p.k_out, max(first - p.heads, 0), end - p.heads);
}

hipError_t launch_rotary(RotaryParams p, bool half, hipStream_t stream) {
  const int heads = p.heads + p.kv_heads;
  p.parts = rotary_parts(p.tokens, heads);
  p.per = (heads + p.parts - 1) / p.parts;
  p.parts = (heads + p.per - 1) / p.per;
  const int64_t units = (int64_t)p.tokens * p.parts;
  void (*fn)(const RotaryParams) = half ? &rotary_kernel<_Float16> : &rotary_kernel<__bf16>;
  hipLaunchKernelGGL(fn, dim3((uint32_t)((units + 15) / 16)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace fba
