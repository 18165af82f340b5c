// norm_rope.hip -- norms of query and key heads with the rotary rotation in the same pass, and
// the gradient.
//
//   r = 1 / sqrt(mean(x^2) + eps),  u = r x w,  y = a R(p) u
//
// over the elements of a head, w a weight for each element, R(p) the rotation of rope_device.h and
// a its amplitude.  With g = a R(p)^T dy (the rotation back) and h = g w, the gradient is
//
//   dx = r (h - r x mean(h r x)),  dw = sum over rows of g r x,
//
// from x and dy alone: r is formed again, which costs less than storing it would.  Each element is
// read and written once, so large calls are bound by HBM (32,768 tokens of 36 heads of 128, 608 MB: 142 us, 4.3
// TB/s; the gradient of 8,192 tokens of 20 heads of 256, 252 MB: 54 us, 4.7 TB/s, and 5 for the sums of dw) and small
// ones by the launch (8 tokens: 4 us).  A group of lanes takes several heads of a token, whose cosines, sines and
// weights are formed once; where that leaves too few groups, one.  All sums and
// products are fp32; a row is rounded to fp16 once.  The sums of dw are formed in one order whatever
// the timing: by row inside a workgroup, then over the workgroups' partial sums.
#include <algorithm>
#include <type_traits>

#include "qkv_device.h"
#include "qkv_launch.h"
#include "rope_device.h"

namespace qkv {

namespace {

// Sum over the LPR neighbouring lanes of a row, in every lane of them.
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  if constexpr (LPR >= 2) v += dpp(v, std::integral_constant<int, 0xb1>{});    // quad_perm 1 0 3 2
  if constexpr (LPR >= 4) v += dpp(v, std::integral_constant<int, 0x4e>{});    // quad_perm 2 3 0 1
  if constexpr (LPR >= 8) v += dpp(v, std::integral_constant<int, 0x141>{});   // row_half_mirror
  if constexpr (LPR >= 16) v += dpp(v, std::integral_constant<int, 0x140>{});  // row_mirror
  if constexpr (LPR >= 32) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  if constexpr (LPR >= 64) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  return v;
}

__device__ __forceinline__ void unpack8(u4_t b, float* f) {
  const h8_t v = __builtin_bit_cast(h8_t, b);
#pragma unroll
  for (int i = 0; i < 8; i++) f[i] = (float)v[i];
}
__device__ __forceinline__ u4_t pack8(const float* f) {
  h8_t v;
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = round16(f[i]);
  return __builtin_bit_cast(u4_t, v);
}

// A lane's 16 elements are two runs of 8: the members of 8 pairs (half-split), or 8 neighbouring
// pairs, or elements that are not turned.
__device__ __forceinline__ void turn16(float* f, const float* cs, const float* sn, int layout) {
  if (layout == 0) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float a = f[i], b = f[8 + i];
      f[i] = __builtin_fmaf(a, cs[i], -b * sn[i]);
      f[8 + i] = __builtin_fmaf(a, sn[i], b * cs[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float a = f[2 * i], b = f[2 * i + 1];
      f[2 * i] = __builtin_fmaf(a, cs[i], -b * sn[i]);
      f[2 * i + 1] = __builtin_fmaf(a, sn[i], b * cs[i]);
    }
  }
}

__device__ __forceinline__ void load_weight(const float* w, const RopeRuns& run, float* f) {
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const f4_t v = w ? *reinterpret_cast<const f4_t*>(w + (i ? run.a1 : run.a0) + 4 * j) : f4_t{1.f, 1.f, 1.f, 1.f};
#pragma unroll
      for (int e = 0; e < 4; e++) f[8 * i + 4 * j + e] = v[e];
    }
}

// Query or key rows of a call
struct Side {
  const uint16_t* in;
  const uint16_t* dy;
  uint16_t* out;
  const float* w;
  long in_stride, dy_stride, out_stride;
  int heads;
};
__device__ __forceinline__ Side side_of(const NormRopeArgs& p, bool isq) {
  return isq ? Side{p.q, p.dq, p.q_out, p.q_weight, p.q_stride, p.dq_stride, p.q_out_stride, p.num_q}
             : Side{p.k, p.dk, p.k_out, p.k_weight, p.k_stride, p.dk_stride, p.k_out_stride, p.num_k};
}

__device__ __forceinline__ void angles(const NormRopeArgs& p, int tok, int c, bool back, float* cs, float* sn) {
  const int64_t pos = back ? -(int64_t)p.positions[tok] : p.positions[tok];
#pragma unroll
  for (int i = 0; i < 8; i++) rope_cos_sin(pos, p.turns[8 * c + i], p.amplitude, cs[i], sn[i]);
}

}  // namespace

// LPR lanes a row of 16 LPR elements; a lane group takes HPT heads of one token (all queries or all
// keys), whose cosines and weights are formed once.
template <int LPR, int HPT>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeArgs p) {
  const long u = (long)(blockIdx.z * kGridX + blockIdx.x) * 256 + threadIdx.x;
  if (u >= (long)p.n_tok * LPR) return;   // (whole groups of lanes)
  const int tok = (int)(u / LPR), c = (int)(u % LPR);
  const int q_chunks = (p.num_q + HPT - 1) / HPT, y = blockIdx.y;
  const bool isq = y < q_chunks;
  const Side sd = side_of(p, isq);
  const int h0 = (isq ? y : y - q_chunks) * HPT;
  const RopeRuns run = rope_runs(c, p.rot, p.layout);
  u4_t x[HPT][2];
#pragma unroll
  for (int i = 0; i < HPT; i++) {
    const uint16_t* in = sd.in + tok * sd.in_stride + (long)min(h0 + i, sd.heads - 1) * p.head_dim;
    x[i][0] = *reinterpret_cast<const u4_t*>(in + run.a0);
    x[i][1] = *reinterpret_cast<const u4_t*>(in + run.a1);
  }
  float w[16], cs[8], sn[8];
  load_weight(sd.w, run, w);
  if (run.turned) angles(p, tok, c, false, cs, sn);
  const float inv = 1.0f / (float)(16 * LPR);
#pragma unroll
  for (int i = 0; i < HPT; i++) {
    float f[16];
    unpack8(x[i][0], f);
    unpack8(x[i][1], f + 8);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 16; e++) ss = __builtin_fmaf(f[e], f[e], ss);
    const float r = rsqrtf(__builtin_fmaf(row_sum<LPR>(ss), inv, p.eps));
#pragma unroll
    for (int e = 0; e < 16; e++) f[e] = f[e] * r * w[e];
    if (run.turned) turn16(f, cs, sn, p.layout);
    if (h0 + i < sd.heads) {
      uint16_t* out = sd.out + tok * sd.out_stride + (long)(h0 + i) * p.head_dim;
      *reinterpret_cast<u4_t*>(out + run.a0) = pack8(f);
      *reinterpret_cast<u4_t*>(out + run.a1) = pack8(f + 8);
    }
  }
}

// Any even rot, head size, stride and alignment: a wave per row, which it reads twice, 2 bytes a lane, and for which it forms
// the angles again.  Bound by its instructions: 32,768 tokens of 36 heads of 96 take 353 us, of 192 with 64 turned 640 (94 and
// 189 at the copy's rate).
__global__ __launch_bounds__(256) void norm_rope_any_kernel(NormRopeArgs p) {
  const long row = (long)(blockIdx.y * kGridX + blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, heads = p.num_q + p.num_k;
  if (row >= (long)p.n_tok * heads) return;
  const int tok = (int)(row / heads), h = (int)(row - (long)tok * heads);
  const bool isq = h < p.num_q;
  const Side sd = side_of(p, isq);
  const long head = (long)(isq ? h : h - p.num_q) * p.head_dim;
  const uint16_t* in = sd.in + tok * sd.in_stride + head;
  uint16_t* out = sd.out + tok * sd.out_stride + head;
  float ss = 0.f;
  for (int e = lane; e < p.head_dim; e += 64) {
    const float v = h2f(in[e]);
    ss = __builtin_fmaf(v, v, ss);
  }
  const float r = rsqrtf(row_sum<64>(ss) / (float)p.head_dim + p.eps);
  const int half = p.rot / 2;
  for (int i = lane; i < p.head_dim - half; i += 64) {
    if (i >= half) {
      const int e = half + i;
      out[e] = __builtin_bit_cast(uint16_t, round16(h2f(in[e]) * r * (sd.w ? sd.w[e] : 1.f)));
      continue;
    }
    const int a0 = p.layout == 0 ? i : 2 * i, a1 = p.layout == 0 ? i + half : 2 * i + 1;
    const float x = h2f(in[a0]) * r * (sd.w ? sd.w[a0] : 1.f), y = h2f(in[a1]) * r * (sd.w ? sd.w[a1] : 1.f);
    float c, s;
    rope_cos_sin(p.positions[tok], p.turns[i], p.amplitude, c, s);
    out[a0] = __builtin_bit_cast(uint16_t, round16(__builtin_fmaf(x, c, -y * s)));
    out[a1] = __builtin_bit_cast(uint16_t, round16(__builtin_fmaf(x, s, y * c)));
  }
}

// The gradient: the first q_groups workgroups take the queries' rows, the others the keys', each lane
// group in turn HPT heads of a token.  A lane's elements are the same in all of its rows, so its part of
// dw stays in 16 registers; a workgroup's is summed through LDS and stored once.
template <int LPR, int HPT>
__global__ __launch_bounds__(256, 3) void norm_rope_grad_kernel(NormRopeArgs p) {
  constexpr int GROUPS = 256 / LPR, HD = 16 * LPR;
  __shared__ float part[GROUPS * HD];   // 16 KB
  const int tid = threadIdx.x, c = tid % LPR, grp = tid / LPR;
  const bool isq = (int)blockIdx.x < p.q_groups;
  const Side sd = side_of(p, isq);
  const int wg = isq ? blockIdx.x : blockIdx.x - p.q_groups, wgs = isq ? p.q_groups : gridDim.x - p.q_groups;
  const int chunks = (sd.heads + HPT - 1) / HPT;
  const RopeRuns run = rope_runs(c, p.rot, p.layout);
  float w[16], dw[16];
  load_weight(sd.w, run, w);
#pragma unroll
  for (int e = 0; e < 16; e++) dw[e] = 0.f;
  const float inv = 1.0f / (float)HD;
  const long items = (long)p.n_tok * chunks;
  for (long it = (long)wg * GROUPS + grp; it < items; it += (long)wgs * GROUPS) {
    const int tok = (int)(it / chunks), h0 = (int)(it - (long)tok * chunks) * HPT;
    u4_t x[HPT][2], y[HPT][2];
#pragma unroll
    for (int i = 0; i < HPT; i++) {
      const long head = (long)min(h0 + i, sd.heads - 1) * p.head_dim;
      const uint16_t *in = sd.in + tok * sd.in_stride + head, *dy = sd.dy + tok * sd.dy_stride + head;
      x[i][0] = *reinterpret_cast<const u4_t*>(in + run.a0);
      x[i][1] = *reinterpret_cast<const u4_t*>(in + run.a1);
      y[i][0] = *reinterpret_cast<const u4_t*>(dy + run.a0);
      y[i][1] = *reinterpret_cast<const u4_t*>(dy + run.a1);
    }
    float cs[8], sn[8];
    if (run.turned) angles(p, tok, c, true, cs, sn);
#pragma unroll
    for (int i = 0; i < HPT; i++) {
      float f[16], g[16];
      unpack8(x[i][0], f);
      unpack8(x[i][1], f + 8);
      unpack8(y[i][0], g);
      unpack8(y[i][1], g + 8);
      if (run.turned) turn16(g, cs, sn, p.layout);
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int e = 0; e < 16; e++) {
        ss = __builtin_fmaf(f[e], f[e], ss);
        dot = __builtin_fmaf(f[e], g[e] * w[e], dot);
      }
      const float r = rsqrtf(__builtin_fmaf(row_sum<LPR>(ss), inv, p.eps));
      const float m = row_sum<LPR>(dot) * r * inv;   // mean of h r x
      const bool live = h0 + i < sd.heads;
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const float xr = f[e] * r;
        if (live) dw[e] = __builtin_fmaf(g[e], xr, dw[e]);
        f[e] = r * (g[e] * w[e] - xr * m);
      }
      if (live) {
        uint16_t* out = sd.out + tok * sd.out_stride + (long)(h0 + i) * p.head_dim;
        *reinterpret_cast<u4_t*>(out + run.a0) = pack8(f);
        *reinterpret_cast<u4_t*>(out + run.a1) = pack8(f + 8);
      }
    }
  }
  if (!p.partial) return;
#pragma unroll
  for (int e = 0; e < 16; e++) part[grp * HD + (e < 8 ? run.a0 + e : run.a1 + e - 8)] = dw[e];
  __syncthreads();
  for (int e = tid; e < HD; e += 256) {
    float s = 0.f;
    for (int i = 0; i < GROUPS; i++) s += part[i * HD + e];
    p.partial[(long)blockIdx.x * HD + e] = s;
  }
}

// Any size and alignment: a wave per row, its part of dw in LDS (each element one lane's).  8,192 tokens of 20 heads of 96 take
// 137 us, of 192 308 (20 and 39 at the copy's rate).
__global__ __launch_bounds__(256) void norm_rope_grad_any_kernel(NormRopeArgs p) {
  __shared__ float part[4][kNormMaxHead];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hd = p.head_dim;
  const bool isq = (int)blockIdx.x < p.q_groups;
  const Side sd = side_of(p, isq);
  const int wg = isq ? blockIdx.x : blockIdx.x - p.q_groups, wgs = isq ? p.q_groups : gridDim.x - p.q_groups;
  for (int e = threadIdx.x; e < 4 * kNormMaxHead; e += 256) (&part[0][0])[e] = 0.f;
  __syncthreads();
  const int half = p.rot / 2;
  const long rows = (long)p.n_tok * sd.heads;
  for (long row = (long)wg * 4 + wave; row < rows; row += (long)wgs * 4) {
    const int tok = (int)(row / sd.heads);
    const long head = (row - (long)tok * sd.heads) * hd;
    const uint16_t *in = sd.in + tok * sd.in_stride + head, *dy = sd.dy + tok * sd.dy_stride + head;
    uint16_t* out = sd.out + tok * sd.out_stride + head;
    // the elements of step i (one past the turned pairs) and their gradients before the rotation
    auto step = [&](int i, int (&at)[2], float (&x)[2], float (&g)[2]) {
      const bool pair = i < half;
      at[0] = !pair ? half + i : p.layout == 0 ? i : 2 * i;
      at[1] = !pair ? at[0] : p.layout == 0 ? i + half : 2 * i + 1;
      x[0] = h2f(in[at[0]]);
      g[0] = h2f(dy[at[0]]);
      if (!pair) return 1;
      x[1] = h2f(in[at[1]]);
      g[1] = h2f(dy[at[1]]);
      float c, s;
      rope_cos_sin(-(int64_t)p.positions[tok], p.turns[i], p.amplitude, c, s);
      const float a = g[0], b = g[1];
      g[0] = __builtin_fmaf(a, c, -b * s);
      g[1] = __builtin_fmaf(a, s, b * c);
      return 2;
    };
    float ss = 0.f, dot = 0.f;
    for (int i = lane; i < hd - half; i += 64) {
      int at[2];
      float x[2], g[2];
      const int n = step(i, at, x, g);
      for (int e = 0; e < n; e++) {
        ss = __builtin_fmaf(x[e], x[e], ss);
        dot = __builtin_fmaf(x[e], g[e] * (sd.w ? sd.w[at[e]] : 1.f), dot);
      }
    }
    const float r = rsqrtf(row_sum<64>(ss) / (float)hd + p.eps);
    const float m = row_sum<64>(dot) * r / (float)hd;
    for (int i = lane; i < hd - half; i += 64) {
      int at[2];
      float x[2], g[2];
      const int n = step(i, at, x, g);
      for (int e = 0; e < n; e++) {
        const float xr = x[e] * r;
        part[wave][at[e]] = __builtin_fmaf(g[e], xr, part[wave][at[e]]);
        out[at[e]] = __builtin_bit_cast(uint16_t, round16(r * (g[e] * (sd.w ? sd.w[at[e]] : 1.f) - xr * m)));
      }
    }
  }
  if (!p.partial) return;
  __syncthreads();
  for (int e = threadIdx.x; e < hd; e += 256)
    p.partial[(long)blockIdx.x * hd + e] = part[0][e] + part[1][e] + part[2][e] + part[3][e];
}

// dw from the workgroups' sums: 16 columns a workgroup, every 64th partial sum a thread of each.
__global__ __launch_bounds__(1024) void norm_rope_dw_kernel(NormRopeArgs p, int groups) {
  constexpr int R = 64;
  __shared__ float part[R][17];
  const bool isq = blockIdx.y == 0;
  float* out = isq ? p.q_dw : p.k_dw;
  if (!out) return;
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4, e = min((int)blockIdx.x * 16 + c, p.head_dim - 1);
  const int from = isq ? 0 : p.q_groups, to = isq ? p.q_groups : groups;
  float s = 0.f;
  for (int i0 = from + r; i0 < to; i0 += 8 * R) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = p.partial[(long)min(i0 + i * R, to - 1) * p.head_dim + e];
#pragma unroll
    for (int i = 0; i < 8; i++) s += i0 + i * R < to ? v[i] : 0.f;
  }
  part[r][c] = s;
  __syncthreads();
  if (r < 8) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < R / 8; i++) s += part[r + 8 * i][c];
    part[r][c] = s;
  }
  __syncthreads();
  if (r == 0 && (int)blockIdx.x * 16 + c < p.head_dim) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) s += part[i][c];
    out[e] = s;
  }
}

hipError_t launch_norm_rope(const NormRopeArgs& a, bool wide, hipStream_t stream) {
  if (!wide) {
    const long rows = (long)a.n_tok * (a.num_q + a.num_k);
    hipLaunchKernelGGL(norm_rope_any_kernel, grid_xy((rows + 3) / 4), dim3(256), 0, stream, a);
    return hipGetLastError();
  }
  const int lpr = a.head_dim / 16;
  const dim3 g = grid_xy(((long)a.n_tok * lpr + 255) / 256);
  auto launch = [&](auto kernel, int hpt) {
    const unsigned chunks = (unsigned)((a.num_q + hpt - 1) / hpt + (a.num_k + hpt - 1) / hpt);
    hipLaunchKernelGGL(kernel, dim3(g.x, chunks, g.y), dim3(256), 0, stream, a);
  };
  const bool few = (long)a.n_tok * lpr * (a.num_q + a.num_k) <= 256 * 1024;
  switch (lpr) {
    case 4: few ? launch(norm_rope_kernel<4, 1>, 1) : launch(norm_rope_kernel<4, 4>, 4); break;
    case 8: few ? launch(norm_rope_kernel<8, 1>, 1) : launch(norm_rope_kernel<8, 4>, 4); break;
    case 16: few ? launch(norm_rope_kernel<16, 1>, 1) : launch(norm_rope_kernel<16, 4>, 4); break;
    case 32: few ? launch(norm_rope_kernel<32, 1>, 1) : launch(norm_rope_kernel<32, 4>, 4); break;
    default: few ? launch(norm_rope_kernel<64, 1>, 1) : launch(norm_rope_kernel<64, 4>, 4); break;
  }
  return hipGetLastError();
}

hipError_t launch_norm_rope_grad(NormRopeArgs a, bool wide, int groups, hipStream_t stream) {
  const int heads = a.num_q + a.num_k;
  a.q_groups = a.num_k == 0 ? groups : a.num_q == 0 ? 0 : std::min(std::max(groups * a.num_q / heads, 1), groups - 1);
  const dim3 grid((unsigned)groups), block(256);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, a); };
  if (!wide) {
    launch(norm_rope_grad_any_kernel);
  } else {
    const int lpr = a.head_dim / 16;
    switch (lpr) {
      case 4: launch(norm_rope_grad_kernel<4, 2>); break;
      case 8: launch(norm_rope_grad_kernel<8, 2>); break;
      case 16: launch(norm_rope_grad_kernel<16, 2>); break;
      case 32: launch(norm_rope_grad_kernel<32, 2>); break;
      default: launch(norm_rope_grad_kernel<64, 2>); break;
    }
  }
  if (a.partial)
    hipLaunchKernelGGL(norm_rope_dw_kernel, dim3((unsigned)((a.head_dim + 15) / 16), 2), dim3(1024), 0, stream, a, groups);
  return hipGetLastError();
}

}  // namespace qkv
