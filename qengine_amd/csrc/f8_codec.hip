// f8_codec.hip -- append to the paged 8-bit cache.
//
// A page of one KV head holds e4m3 codes under one exponent: value = code * 2^(e - 127),
// with the smallest e >= 95 for which no new row's magnitude passes 448 * 2^(e - 127).
// Rows that continue a page keep its exponent or raise it; the page's older rows are
// then requantized by a power of two, which changes only codes that become
// subnormal.  Inputs are limited to +-61440, the largest code under the largest
// exponent that fp16 holds, and a NaN is stored as zero (the cache holds finite
// values only, as the other cache formats do).  Codes are the values' only rounding (to nearest
// even: 2^-4 of a value at most, 2^-10 of the page's largest below its normal range); a
// rotated key is first rounded to fp16, so that rotating apart gives the same bits.
//
// Bound by HBM: rows read once (2 bytes an element), codes written once (1).  25,000 rows of two
// prompts, 4 KV heads of 256: 153 MB in 32 to 33 us (4.7 TB/s, the rate of a large copy); a decode
// step of 32 slots with its rotation 5.3 us, which is latency.
#include <algorithm>

#include "f8_device.h"
#include "qkv_device.h"
#include "qkv_launch.h"
#include "rope_device.h"

namespace qkv {

namespace {

constexpr uint32_t kMaxBits = 0x7b80u;   // 61440

// fp16 bits to the stored range: NaN to zero, magnitudes limited
__device__ __forceinline__ uint32_t limit16(uint32_t b) {
  const uint32_t a = b & 0x7fffu;
  return a > 0x7c00u ? 0u : min(a, kMaxBits) | (b & 0x8000u);
}

// smallest biased exponent whose largest code holds the fp16 magnitude `bits`
__device__ __forceinline__ int f8_exponent(uint32_t bits) {
  const uint32_t f = __float_as_uint(h2f(bits));
  return max(95, (int)(f >> 23) - 8 + ((f & 0x7fffffu) > 0x600000u ? 1 : 0));   // (zero: 95)
}

}  // namespace

struct RowRope {
  const uint64_t* turns;
  float amp;
  int rot, layout;
};

// 8 elements from element 8c of a head row, rotated by position pos and rounded to fp16
__device__ __forceinline__ u4_t load_turned(const uint16_t* row, int c, int pos, const RowRope& r) {
  const u4_t own = *reinterpret_cast<const u4_t*>(row + 8 * c);
  if (8 * c >= r.rot) return own;
  const h8_t x = __builtin_bit_cast(h8_t, own);
  h8_t o;
  if (r.layout == 0) {
    const int half = r.rot / 2;
    const bool first = 8 * c < half;
    const int i0 = first ? 8 * c : 8 * c - half;
    const h8_t y = __builtin_bit_cast(h8_t, *reinterpret_cast<const u4_t*>(row + (first ? 8 * c + half : i0)));
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float cs, sn;
      rope_cos_sin(pos, r.turns[i0 + i], r.amp, cs, sn);
      const float a = (float)x[i], b = (float)y[i];
      // first half: x cos - y sin (b = y); second half: x sin + y cos (a = y, b = x)
      o[i] = round16(first ? __builtin_fmaf(a, cs, -b * sn) : __builtin_fmaf(b, sn, a * cs));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float cs, sn;
      rope_cos_sin(pos, r.turns[4 * c + i], r.amp, cs, sn);
      const float a = (float)x[2 * i], b = (float)x[2 * i + 1];
      o[2 * i] = round16(__builtin_fmaf(a, cs, -b * sn));
      o[2 * i + 1] = round16(__builtin_fmaf(a, sn, b * cs));
    }
  }
  return __builtin_bit_cast(u4_t, o);
}

__device__ __forceinline__ u4_t limit8(u4_t v) {
  u4_t o;
#pragma unroll
  for (int i = 0; i < 4; i++) o[i] = limit16(v[i] & 0xffffu) | (limit16(v[i] >> 16) << 16);
  return o;
}
__device__ __forceinline__ uint32_t max8(u4_t v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) m = max(m, max(v[i] & 0x7fffu, (v[i] >> 16) & 0x7fffu));
  return m;
}
// 8 limited fp16 values over 2^(e - 127) as e4m3 (nearest, ties to even; exact scaling)
__device__ __forceinline__ u2_t encode8(u4_t v, float inv) {
  const h8_t x = __builtin_bit_cast(h8_t, v);
  u2_t o;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32((float)x[4 * i] * inv, (float)x[4 * i + 1] * inv, 0, false);
    o[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32((float)x[4 * i + 2] * inv, (float)x[4 * i + 3] * inv, w, true);
  }
  return o;
}

// One workgroup per (slot, touched page, KV head, K or V); the workgroups past those
// rotate query rows.  The rows of a page stay in registers between the maximum and
// the store where KEEP 8-element runs a thread hold them (a 64-row page of 256).
template <int THREADS, bool ROPE>
__global__ __launch_bounds__(THREADS, ROPE || THREADS == 1024 ? 4 : 8) void f8_append_kernel(F8AppendArgs p) {
  constexpr int KEEP = 8;
  const int tid = threadIdx.x;
  const int hd = p.head_dim, cpr = hd / 8, cpr_log = hd == 256 ? 5 : 4;   // (head_dim is 128 or 256)
  const RowRope rope{p.turns, p.amplitude, p.rot, p.layout};
  long wg = blockIdx.y * kGridX + blockIdx.x;   // (in 32 bits: so are the divisions below)
  if (wg >= p.kv_wgs) {
    if (!ROPE || p.q == nullptr) return;
    // query rows: 16 elements of QH heads a thread, both sides of their pairs (they may be in place),
    // whose cosines are formed once
    constexpr int QH = 4;
    const long u = (wg - p.kv_wgs) * THREADS + tid;
    const int per_head = hd / 16, per_tok = (p.num_q + QH - 1) / QH * per_head;
    const long tok = u / per_tok;
    if (tok >= p.rows) return;
    // the slot of the token: the last whose start is not past it
    int lo = 0, hi = p.n_slots;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (p.starts[mid] <= tok) lo = mid; else hi = mid;
    }
    const int s0 = p.starts[lo];
    // (not behind the last slot, nor past what the call covers of this one)
    if (tok < s0 || tok >= p.starts[lo + 1] || tok - s0 >= p.max_tok || p.positions[lo] < 0 ||
        p.positions[lo] > kMaxPosition)
      return;
    const int r = (int)(u - tok * per_tok), c = r % per_head, h0 = r / per_head * QH;
    const RopeRuns run = rope_runs(c, rope.rot, rope.layout);
    const uint16_t* in = p.q + tok * p.q_stride;
    uint16_t* out = p.q_out + tok * p.q_out_stride;
    if (!run.turned && in == out) return;
    u4_t x[QH], y[QH];
#pragma unroll
    for (int i = 0; i < QH; i++) {
      const uint16_t* at = in + (long)min(h0 + i, p.num_q - 1) * hd;
      x[i] = *reinterpret_cast<const u4_t*>(at + run.a0);
      y[i] = *reinterpret_cast<const u4_t*>(at + run.a1);
    }
    if (run.turned) {
      const int pos = p.positions[lo] + (int)(tok - s0);
      float cs[8], sn[8];
#pragma unroll
      for (int i = 0; i < 8; i++) rope_cos_sin(pos, rope.turns[8 * c + i], rope.amp, cs[i], sn[i]);
#pragma unroll
      for (int i = 0; i < QH; i++) {
        if (rope.layout == 0) turn8(x[i], y[i], cs, sn, x[i], y[i]);
        else turn8_pairs(x[i], y[i], cs, sn, x[i], y[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < QH; i++) {
      if (h0 + i >= p.num_q) break;
      uint16_t* at = out + (long)(h0 + i) * hd;
      *reinterpret_cast<u4_t*>(at + run.a0) = x[i];
      *reinterpret_cast<u4_t*>(at + run.a1) = y[i];
    }
    return;
  }
  const bool is_v = wg & 1;
  wg >>= 1;
  const int h = (int)(wg % p.num_kv);
  wg /= p.num_kv;
  const int j = (int)(wg % p.spans), s = (int)(wg / p.spans);
  const int t0 = min(max(p.starts[s], 0), (int)p.rows);
  const int n = min(min(max(p.starts[s + 1], t0), (int)p.rows) - t0, p.max_tok);
  const int pos0 = p.positions[s];
  if (pos0 < 0 || pos0 > kMaxPosition || n <= 0) return;
  const long b = (long)pos0 / p.block_tokens + j;
  const long first = max((long)pos0, b * p.block_tokens), end = min((long)pos0 + n, (b + 1) * p.block_tokens);
  if (first >= end || b >= p.max_blocks) return;
  const int page = p.tables[(long)s * p.max_blocks + b];
  if (page < 0 || page >= p.n_pages) return;
  const int off = (int)(first - b * p.block_tokens), rows = (int)(end - first);
  const long tok0 = t0 + (first - pos0);
  const long stride = is_v ? p.v_stride : p.k_stride;
  const uint16_t* in = (is_v ? p.v : p.k) + tok0 * stride + (long)h * hd;
  const long row_bytes = (long)p.num_kv * hd;
  uint8_t* pool = (is_v ? p.v_pool : p.k_pool) + (long)page * p.block_tokens * row_bytes + (long)h * hd;
  uint8_t* exp_at = (is_v ? p.v_exp : p.k_exp) + (long)page * p.num_kv + h;
  const int was = off > 0 ? min((int)*exp_at, 254) : 0;

  const bool turn = ROPE && !is_v;
  const int units = rows * cpr;
  auto load = [&](int u) {
    const int r = u >> cpr_log, c = u & (cpr - 1);
    const uint16_t* row = in + r * stride;
    return limit8(turn ? load_turned(row, c, (int)(first + r), rope)
                       : __builtin_nontemporal_load(reinterpret_cast<const u4_t*>(row + 8 * c)));
  };
  u4_t kept[KEEP];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < KEEP; i++) {
    const int u = tid + i * THREADS;
    kept[i] = u < units ? load(u) : u4_t{0, 0, 0, 0};
    top = max(top, max8(kept[i]));
  }
  for (int u = tid + KEEP * THREADS; u < units; u += THREADS) top = max(top, max8(load(u)));
#pragma unroll
  for (int d = 32; d; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
  if constexpr (THREADS > 64) {
    __shared__ uint32_t tops[THREADS / 64];
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) top = max(top, tops[w]);
  }
  const int e = max(f8_exponent(top), was);
  const float inv = pow2_bits(254 - e);
  auto store = [&](int u, u4_t v) {
    const int r = u >> cpr_log, c = u & (cpr - 1);
    *reinterpret_cast<u2_t*>(pool + (long)(off + r) * row_bytes + 8 * c) = encode8(v, inv);
  };
#pragma unroll
  for (int i = 0; i < KEEP; i++)
    if (tid + i * THREADS < units) store(tid + i * THREADS, kept[i]);
  for (int u = tid + KEEP * THREADS; u < units; u += THREADS) store(u, load(u));
  if (off > 0 && e > was) {   // the older rows, at the raised exponent
    const float f = pow2_bits(127 - min(e - was, 126));
    for (int u = tid; u < off * cpr; u += THREADS) {
      const int r = u >> cpr_log, c = u & (cpr - 1);
      u2_t* at = reinterpret_cast<u2_t*>(pool + (long)r * row_bytes + 8 * c);
      const u2_t v = *at;
      *at = u2_t{rescale4(v[0], f), rescale4(v[1], f)};
    }
  }
  if (tid == 0) *exp_at = (uint8_t)e;
}

hipError_t launch_f8_append(F8AppendArgs a, hipStream_t stream) {
  a.spans = (a.max_tok + a.block_tokens - 2) / a.block_tokens + 1;
  const long kv = (long)a.n_slots * a.spans * a.num_kv * 2;
  const long q_units = a.q ? a.rows * ((a.num_q + 3) / 4) * (a.head_dim / 16) : 0;
  // As many threads as hold a page's new rows in their registers: a wave for up to 8 rows of 256
  // (8,192 tokens in 16-row pages of 256, which need 256: 19.0 us, 61.6 with 1,024), 256 up to 64 rows
  // (18,000 tokens: 27.5 us, 50.8 with 64, 50.0 with 1,024), else 1,024 (8,192 tokens in 256-row pages:
  // 19.9 us, 42.9 with 256).
  const long elems = (long)std::min(a.max_tok, a.block_tokens) * a.head_dim;
  const int threads = elems <= 64 * 8 * 4 ? 64 : elems <= 256 * 8 * 8 ? 256 : 1024;
  const long wgs = kv + (q_units + threads - 1) / threads;
  if (wgs > 0x7fffffffL) return hipErrorInvalidValue;
  a.kv_wgs = kv;
  const dim3 grid = grid_xy(wgs), block((unsigned)threads);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, a); };
  if (threads == 64) a.rot ? launch(f8_append_kernel<64, true>) : launch(f8_append_kernel<64, false>);
  else if (threads == 256) a.rot ? launch(f8_append_kernel<256, true>) : launch(f8_append_kernel<256, false>);
  else a.rot ? launch(f8_append_kernel<1024, true>) : launch(f8_append_kernel<1024, false>);
  return hipGetLastError();
}

}  // namespace qkv
