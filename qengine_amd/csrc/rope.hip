// rope.hip -- rotary positions of query and key rows.
//
// (x, y) -> (x cos t - y sin t, x sin t + y cos t) for the pairs of the first rot
// elements of every head, the rest copied; the inverse turns by -t, which is also
// the gradient (the rotation is orthogonal).  One pass: each element is read and
// written once, so large calls are bound by HBM and small ones by the launch.
// 32,768 tokens of 28 heads of 128, all turned: 470 MB in 97 to 103 us (4.6 to 4.8 TB/s, the rate
// of a large copy); a decode step of eight tokens 3.9 us.  Stores past the caches were slower (146 us).
#include "qkv_device.h"
#include "qkv_launch.h"
#include "rope_device.h"

namespace qkv {

// A thread takes 16 elements (8 pairs, or 16 copied ones) of one token in HPT
// heads, so that their cosines are formed once: four, or one where that leaves few threads (eight
// tokens of 20 heads: 3.9 us with one, 4.7 with four; 8,192 tokens of 20 turned heads of 128: 19.7 and
// 17.8 us; the same from 2,000 to 4,000 tokens).
template <int HPT>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs p) {
  const long u = (long)(blockIdx.z * kGridX + blockIdx.x) * 256 + threadIdx.x;
  if (u >= (long)p.n_tok * p.units) return;
  const int tok = (int)(u / p.units), c = (int)(u - (long)tok * p.units);
  const int h0 = blockIdx.y * HPT;
  const RopeRuns run = rope_runs(c, p.rot, p.layout);
  u4_t x[HPT], y[HPT];
#pragma unroll
  for (int i = 0; i < HPT; i++) {
    const int h = min(h0 + i, p.num_q + p.num_k - 1);
    const bool isq = h < p.num_q;
    const uint16_t* in = isq ? p.q + tok * p.q_stride + (long)h * p.head_dim
                             : p.k + tok * p.k_stride + (long)(h - p.num_q) * p.head_dim;
    x[i] = *reinterpret_cast<const u4_t*>(in + run.a0);
    y[i] = *reinterpret_cast<const u4_t*>(in + run.a1);
  }
  if (run.turned) {
    float cs[8], sn[8];
    const int64_t pos = p.inverse ? -(int64_t)p.positions[tok] : p.positions[tok];
#pragma unroll
    for (int i = 0; i < 8; i++) rope_cos_sin(pos, p.turns[8 * c + i], p.amplitude, cs[i], sn[i]);
#pragma unroll
    for (int i = 0; i < HPT; i++) {
      u4_t xo, yo;
      if (p.layout == 0) turn8(x[i], y[i], cs, sn, xo, yo);
      else turn8_pairs(x[i], y[i], cs, sn, xo, yo);
      x[i] = xo;
      y[i] = yo;
    }
  }
#pragma unroll
  for (int i = 0; i < HPT; i++) {
    const int h = h0 + i;
    if (h >= p.num_q + p.num_k) break;
    const bool isq = h < p.num_q;
    uint16_t* out = isq ? p.q_out + tok * p.q_out_stride + (long)h * p.head_dim
                        : p.k_out + tok * p.k_out_stride + (long)(h - p.num_q) * p.head_dim;
    *reinterpret_cast<u4_t*>(out + run.a0) = x[i];
    *reinterpret_cast<u4_t*>(out + run.a1) = y[i];
  }
}

// Any even rot, head size, stride and alignment: a thread per pair or copied element.
__global__ __launch_bounds__(256) void rope_any_kernel(RopeArgs p) {
  const int per = p.units;   // rot / 2 pairs, then the copied elements (none in place)
  const long u = (long)(blockIdx.y * kGridX + blockIdx.x) * 256 + threadIdx.x;
  if (u >= (long)p.n_tok * (p.num_q + p.num_k) * per) return;
  const long row = u / per;
  const int i = (int)(u - row * per);
  const int tok = (int)(row / (p.num_q + p.num_k)), h = (int)(row - (long)tok * (p.num_q + p.num_k));
  const bool isq = h < p.num_q;
  const uint16_t* in = isq ? p.q + tok * p.q_stride + (long)h * p.head_dim
                           : p.k + tok * p.k_stride + (long)(h - p.num_q) * p.head_dim;
  uint16_t* out = isq ? p.q_out + tok * p.q_out_stride + (long)h * p.head_dim
                      : p.k_out + tok * p.k_out_stride + (long)(h - p.num_q) * p.head_dim;
  const int half = p.rot / 2;
  if (i >= half) {
    out[half + i] = in[half + i];
    return;
  }
  const int a0 = p.layout == 0 ? i : 2 * i, a1 = p.layout == 0 ? i + half : 2 * i + 1;
  const float x = h2f(in[a0]), y = h2f(in[a1]);
  float c, s;
  const int64_t pos = p.inverse ? -(int64_t)p.positions[tok] : p.positions[tok];
  rope_cos_sin(pos, p.turns[i], p.amplitude, c, s);
  out[a0] = __builtin_bit_cast(uint16_t, round16(__builtin_fmaf(x, c, -y * s)));
  out[a1] = __builtin_bit_cast(uint16_t, round16(__builtin_fmaf(x, s, y * c)));
}

hipError_t launch_rope(RopeArgs a, bool wide, bool in_place, hipStream_t stream) {
  const int heads = a.num_q + a.num_k;
  if (wide) {
    a.units = (in_place ? a.rot : a.head_dim) / 16;
    const long threads = (long)a.n_tok * a.units;
    const dim3 g = grid_xy((threads + 255) / 256);
    if (threads * heads <= 256 * 1024)
      hipLaunchKernelGGL(rope_kernel<1>, dim3(g.x, (unsigned)heads, g.y), dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL(rope_kernel<4>, dim3(g.x, (unsigned)((heads + 3) / 4), g.y), dim3(256), 0, stream, a);
  } else {
    a.units = in_place ? a.rot / 2 : a.head_dim - a.rot / 2;
    const long n = (long)a.n_tok * heads * a.units;
    hipLaunchKernelGGL(rope_any_kernel, grid_xy((n + 255) / 256), dim3(256), 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace qkv
