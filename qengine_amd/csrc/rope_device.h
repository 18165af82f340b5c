// rope_device.h -- the rotary arithmetic shared by rope.hip and f8_codec.hip.
//
// Pair i of a head at position p turns by p * f_i radians.  The frequency is
// held as R_i, the fraction f_i / 2 pi of a full turn in 64-bit fixed point, so
// that p * R_i mod 2^64 is the angle modulo one turn, exactly: 32 bits of fraction
// would be off by p * 2^-33 turns (2^-13 turns, 0.77 mrad, at p = 2^20), and an angle
// of 2^20 radians in fp32 by up to 0.06 rad.  The top 32 bits of the product give
// the nearest quarter turn and a remainder of at most an eighth (error 2^-32 turns).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qkv_device.h"

namespace qkv {

// cos and sin of position pos under R.  The Taylor sums about 0 on +-pi/4, cos to
// x^10 (first term left out 1.1e-10) and sin to x^9 (1.8e-9), are fp32-exact to
// a rounding or two; v_sin_f32's error (about 2^-20) would show in the last
// bit of one fp16 product in a few hundred.
__device__ __forceinline__ void rope_cos_sin(int64_t pos, uint64_t R, float amp, float& c, float& s) {
  const uint32_t ph = (uint32_t)(((uint64_t)pos * R) >> 32);
  const uint32_t quarter = (ph + 0x20000000u) >> 30;
  const int rem = (int)(ph - (quarter << 30));
  const float x = (float)rem * (6.283185307179586f / 4294967296.0f), z = x * x;
  float sn = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  sn = __builtin_fmaf(z, sn, 8.3333333e-3f);
  sn = __builtin_fmaf(z, sn, -1.6666667e-1f);
  sn = __builtin_fmaf(z * x, sn, x);
  float cs = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  cs = __builtin_fmaf(z, cs, -1.3888889e-3f);
  cs = __builtin_fmaf(z, cs, 4.1666667e-2f);
  cs = __builtin_fmaf(z, cs, -0.5f);
  cs = __builtin_fmaf(z, cs, 1.0f);
  const bool odd = quarter & 1u;
  const float a = odd ? sn : cs, b = odd ? cs : sn;
  // quarter 0: (cos, sin), 1: (-sin, cos), 2: (-cos, -sin), 3: (sin, -cos)
  c = ((quarter + 1u) & 2u) ? -a * amp : a * amp;
  s = (quarter & 2u) ? -b * amp : b * amp;
}

// fp32 to fp16 in a rounding of its own: joined with the product before it (a mixed-precision
// fused operation rounds once), the kernels would differ by what the compiler picks in each.
__device__ __forceinline__ _Float16 round16(float x) {
  asm("" : "+v"(x));
  return (_Float16)x;
}

// 8 pairs (x[i], y[i])
__device__ __forceinline__ void turn8(const u4_t xb, const u4_t yb, const float (&c)[8], const float (&s)[8],
                                      u4_t& xo, u4_t& yo) {
  const h8_t x = __builtin_bit_cast(h8_t, xb), y = __builtin_bit_cast(h8_t, yb);
  h8_t xr, yr;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float a = (float)x[i], b = (float)y[i];
    xr[i] = round16(__builtin_fmaf(a, c[i], -b * s[i]));
    yr[i] = round16(__builtin_fmaf(a, s[i], b * c[i]));
  }
  xo = __builtin_bit_cast(u4_t, xr);
  yo = __builtin_bit_cast(u4_t, yr);
}

// the pairs of an interleaved 16-element run: (x0 y0 x1 y1 ..)
__device__ __forceinline__ void turn8_pairs(const u4_t lo, const u4_t hi, const float (&c)[8], const float (&s)[8],
                                            u4_t& lo_o, u4_t& hi_o) {
  u4_t r[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const h8_t v = __builtin_bit_cast(h8_t, h ? hi : lo);
    h8_t w;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float a = (float)v[2 * i], b = (float)v[2 * i + 1];
      w[2 * i] = round16(__builtin_fmaf(a, c[4 * h + i], -b * s[4 * h + i]));
      w[2 * i + 1] = round16(__builtin_fmaf(a, s[4 * h + i], b * c[4 * h + i]));
    }
    r[h] = __builtin_bit_cast(u4_t, w);
  }
  lo_o = r[0];
  hi_o = r[1];
}

// element offsets, inside a head, of the two 8-element runs of run c: 8 pairs, or 16 elements
// past the turned ones
struct RopeRuns {
  int a0, a1;
  bool turned;
};
__device__ __forceinline__ RopeRuns rope_runs(int c, int rot, int layout) {
  const bool turned = 16 * c < rot;
  return turned && layout == 0 ? RopeRuns{8 * c, 8 * c + rot / 2, true} : RopeRuns{16 * c, 16 * c + 8, turned};
}

}  // namespace qkv
