// beam.hip -- beam search's selection over beams and vocabulary.
//
//   S(b, v) = s_b + x_bv - log(sum_u exp(x_bu)),  the `take` largest of a request, ties to the lowest (b, v)
//
// The logits are read once: a workgroup takes a segment of one row, holds it in registers, sums its
// exponentials and keeps its `take` largest logits; a second launch joins a request's segments.  Inside a
// row the order of S is that of x, so segments compare the logits themselves, without a rounding.
// 512 rows of 131,072 fp16 logits take 31 + 11 us (21 at 6.4 TB/s), bf16 32 + 11, fp32 46 + 12 (42); the vector unit bounds the
// first launch of fp16, busy 0.71 of its time: 6 instructions a logit for its exponential, 1 for the maximum, and the
// selection's threshold, maxima of the lanes in turn, a fifth.  Eight workgroups are on a CU (five of bf16, by its registers),
// so that others load while one selects.
//
// The exponentials are taken in base 2 of the distance to the segment's maximum (exact for 16-bit logits),
// times log2(e) as two floats: their error stays near their own rounding, where a product of the logit and one
// float would be off by a common factor of x 2^-24.  Sums of segments are joined, and scores formed, in 64
// bits, so that beams compare to about 2^-24.
#include <algorithm>
#include <type_traits>

#include "qkv_device.h"
#include "qkv_launch.h"

namespace qkv {

namespace {

constexpr float kLog2eHi = 1.44269502162933349609375f;   // log2(e) to 24 bits, and what is left of it
constexpr float kLog2eLo = 1.925963033500011e-8f;
constexpr int kCap = 512, kWordCap = 128;                // candidates, and words that hold some, of a workgroup in LDS

// v of the lane that steps 1, 2, 7, 15 (mirrored in its quad, half row and row), 16 and 32 pair this one with
template <int STEP>
__device__ __forceinline__ float pair_of(float v) {
  if constexpr (STEP < 16) {
    constexpr int ctrl = STEP == 1 ? 0xb1 : STEP == 2 ? 0x4e : STEP == 7 ? 0x141 : 0x140;
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, true));
  } else {
    const uint32_t b = __float_as_uint(v);
    const auto s = STEP == 16 ? __builtin_amdgcn_permlane16_swap(b, b, false, false)
                              : __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __uint_as_float(((threadIdx.x & STEP) != 0) ? s[0] : s[1]);
  }
}
template <int STEP>
__device__ __forceinline__ double pair_of(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = __float_as_uint(pair_of<STEP>(__uint_as_float((uint32_t)b)));
  const uint64_t hi = __float_as_uint(pair_of<STEP>(__uint_as_float((uint32_t)(b >> 32))));
  return __builtin_bit_cast(double, hi << 32 | lo);
}
// Values as the selection's maxima compare them: floats by whole numbers in the same order (of which a maximum over lanes
// is one instruction a step), doubles as they are.
__device__ __forceinline__ int key_of(float v) {
  const int b = __float_as_int(v);
  return b ^ (b >> 31 & 0x7fffffff);
}
__device__ __forceinline__ float of_key(int k) { return __int_as_float(k ^ (k >> 31 & 0x7fffffff)); }
__device__ __forceinline__ double key_of(double v) { return v; }
__device__ __forceinline__ double of_key(double v) { return v; }
__device__ __forceinline__ int wave_max(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0xb1, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x4e, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xf, 0xf, true));
  const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  v = max((int)a[0], (int)a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  return max((int)b[0], (int)b[1]);
}
__device__ __forceinline__ double wave_max(double v) {   // (no NaN)
  auto larger = [](double a, double b) { return b > a ? b : a; };
  v = larger(v, pair_of<1>(v));
  v = larger(v, pair_of<2>(v));
  v = larger(v, pair_of<7>(v));
  v = larger(v, pair_of<15>(v));
  v = larger(v, pair_of<16>(v));
  return larger(v, pair_of<32>(v));
}
__device__ __forceinline__ float wave_sum(float v) {
  v += pair_of<1>(v);
  v += pair_of<2>(v);
  v += pair_of<7>(v);
  v += pair_of<15>(v);
  v += pair_of<16>(v);
  return v + pair_of<32>(v);
}

template <class V>
struct Found {   // candidates of a workgroup: values and what they stand for
  V v[kCap];
  int at[kCap];
  V low[4];
  int n;
};

template <class V>
__device__ __forceinline__ bool better(V a, int ia, V b, int ib) { return a > b || (a == b && ia < ib); }

// The k <= 64 largest of what the 256 threads hold, ties to the lowest index, as put(rank, value, index) by
// any thread; returns how many there are (at most k).  `top` is this thread's largest, each(f, low) calls
// f(value, index) for at least those of its values that are >= low; -infinity is no value.  gather(f, low) does so
// for all threads' together, in any of them.
//
// At least k threads hold a value >= the smallest, over the four waves, of the (k + 3) / 4-th largest of the
// lanes' maxima (and >= the k-th largest of any one wave's, which counts where another wave has too few).  What
// is at or above that goes to LDS, usually a few times k, and is ranked there by counting.  Where more values
// tie than LDS holds, they are found one after the other.  (The smallest maximum of k groups of lanes is found sooner, but
// more values lie above it: 35 -> 44 us for 512 rows of 131,072.)
template <class V, class Each, class Gather, class Put>
__device__ __forceinline__ int top_of_group(Found<V>& found, int k, V top, Each&& each, Gather&& gather, Put&& put) {
  const V none = -INFINITY;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  V low;
  auto mine = key_of(top);
  auto next = [&](int n) {   // the wave's n-th largest
    auto best = mine;
    for (int i = 0; i < n; i++) {
      best = wave_max(mine);
      const uint64_t m = __builtin_amdgcn_ballot_w64(mine == best);
      if (lane == (int)__builtin_ctzll(m)) mine = key_of(none);
    }
    if (lane == 0) found.low[wave] = of_key(best);
  };
  next((k + 3) / 4);
  if (tid == 0) found.n = 0;
  __syncthreads();
  low = found.low[0];
#pragma unroll
  for (int w = 1; w < 4; w++) low = found.low[w] < low ? found.low[w] : low;
  if (low == none) {   // (the same in every wave)
    __syncthreads();
    mine = key_of(top);
    next(k);
    __syncthreads();
    low = found.low[0];
#pragma unroll
    for (int w = 1; w < 4; w++) low = found.low[w] > low ? found.low[w] : low;
  }
  gather([&](V v, int at) __attribute__((always_inline)) {
    if (v >= low && v > none) {
      const int i = atomicAdd(&found.n, 1);
      if (i < kCap) {
        found.v[i] = v;
        found.at[i] = at;
      }
    }
  }, low);
  __syncthreads();
  const int n = found.n;
  if (n <= kCap) {
    for (int i = tid; i < n; i += 256) {
      const V v = found.v[i];
      const int at = found.at[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < n; j++) rank += better(found.v[j], found.at[j], v, at);
      if (rank < k) put(rank, v, at);
    }
    return min(n, k);
  }
  V last = INFINITY;
  int last_at = -1;
  for (int r = 0; r < k; r++) {
    V best = none;
    int best_at = 0x7fffffff;
    each([&](V v, int at) __attribute__((always_inline)) {
      if (better(last, last_at, v, at) && better(v, at, best, best_at)) {
        best = v;
        best_at = at;
      }
    }, none);
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      const V v = __shfl_xor(best, d);
      const int at = __shfl_xor(best_at, d);
      if (better(v, at, best, best_at)) {
        best = v;
        best_at = at;
      }
    }
    __syncthreads();   // (the entries are read by the step before)
    if (lane == 0) {
      found.v[wave] = best;
      found.at[wave] = best_at;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; w++)
      if (better(found.v[w], found.at[w], best, best_at)) {
        best = found.v[w];
        best_at = found.at[w];
      }
    if (best == none) return r;
    if (tid == 0) put(r, best, best_at);
    last = best;
    last_at = best_at;
  }
  return k;
}

// The largest, or NaN
__device__ __forceinline__ float maximum(float a, float b, float c) {
  asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(a) : "v"(a), "v"(b), "v"(c));
  return a;
}
__device__ __forceinline__ float maximum(float a, float b) { return maximum(a, b, b); }

// A word at the address of a logit of 2 or 4 bytes
typedef u4_t __attribute__((aligned(2))) word2_t;
typedef u4_t __attribute__((aligned(4))) word4_t;

// Logits of one 16-byte word
template <int TYPE>
struct Word;
template <>
struct Word<0> {   // fp16
  static constexpr int N = 8;
  static constexpr uint32_t kNone = 0xfc00u;
  __device__ static __forceinline__ float at(u4_t w, int i) { return h2f(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu); }
  // the largest, NaN where one is (pairs at a time: 6 instructions for 8 logits)
  __device__ static __forceinline__ float top(u4_t w) {
    uint32_t m;
    asm("v_pk_maximum3_f16 %0, %1, %2, %3" : "=v"(m) : "v"(w[0]), "v"(w[1]), "v"(w[2]));
    asm("v_pk_maximum3_f16 %0, %1, %2, %2" : "=v"(m) : "v"(m), "v"(w[3]));
    return maximum(h2f(m & 0xffffu), h2f(m >> 16));
  }
  // x - ref in one instruction
  __device__ static __forceinline__ float less(u4_t w, int i, float ref, float one) { return __builtin_fmaf(at(w, i), one, -ref); }
};
template <>
struct Word<1> {   // fp32
  static constexpr int N = 4;
  static constexpr uint32_t kNone = 0xff800000u;
  __device__ static __forceinline__ float at(u4_t w, int i) { return __uint_as_float(w[i]); }
  __device__ static __forceinline__ float top(u4_t w) { return maximum(maximum(at(w, 0), at(w, 1), at(w, 2)), at(w, 3)); }
  __device__ static __forceinline__ float less(u4_t w, int i, float ref, float) { return at(w, i) - ref; }
};
template <>
struct Word<2> {   // bf16
  static constexpr int N = 8;
  static constexpr uint32_t kNone = 0xff80u;
  __device__ static __forceinline__ float at(u4_t w, int i) {
    return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
  }
  __device__ static __forceinline__ float top(u4_t w) {
    float m = maximum(at(w, 0), at(w, 1));
#pragma unroll
    for (int i = 2; i < N; i += 2) {
      m = maximum(m, at(w, i), at(w, i + 1));
      asm volatile("" : "+v"(m));   // (in turn: the numbers of many words would fill the registers)
    }
    return m;
  }
  __device__ static __forceinline__ float less(u4_t w, int i, float ref, float) { return at(w, i) - ref; }
};
// NaN and +infinity to -infinity
template <int TYPE>
__device__ __forceinline__ void leave_out(u4_t& w) {
  using W = Word<TYPE>;
#pragma unroll
  for (int i = 0; i < W::N; i++) {
    if (W::at(w, i) < INFINITY) continue;
    if constexpr (W::N == 8) w[i >> 1] = (w[i >> 1] & (i & 1 ? 0xffffu : 0xffff0000u)) | (i & 1 ? W::kNone << 16 : W::kNone);
    else w[i] = W::kNone;
  }
}

__device__ __forceinline__ bool searched(const BeamArgs& p, long row) {   // a beam whose logits count
  return p.scores[row] > -INFINITY && !(p.done && p.done[row]);
}

}  // namespace

// A workgroup takes NV words a thread of a row.  Words are counted from the row's first logit, whatever its address, so
// that equal rows are cut and summed in the same order and beams of equal scores tie; the last word of a row is read by
// the logit, none past its end.
template <int TYPE, int NV>
__global__ __launch_bounds__(256, 4) void beam_rows_kernel(BeamArgs p) {
  using W = Word<TYPE>;
  constexpr int SIZE = 16 / W::N;
  __shared__ Found<float> found;
  __shared__ u4_t word_s[kWordCap];   // words that hold a candidate, and their first element's token
  __shared__ int word_at[kWordCap], n_words;
  __shared__ float part[4], sums[4];
  const long wg = (long)blockIdx.y * kGridX + blockIdx.x;
  if (wg >= (long)p.rows * p.segments) return;
  const long row = wg / p.segments;
  const int seg = (int)(wg - row * p.segments), tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  if (!searched(p, row)) return;
  typedef typename std::conditional<SIZE == 2, uint16_t, uint32_t>::type Logit;
  typedef typename std::conditional<SIZE == 2, word2_t, word4_t>::type Loaded;
  const Logit* logits = reinterpret_cast<const Logit*>(p.logits) + row * p.stride;
  const int w0 = seg * (256 * NV), whole = p.vocab / W::N, rest = p.vocab % W::N;
  u4_t raw[NV], none;
#pragma unroll
  for (int i = 0; i < 4; i++) none[i] = SIZE == 2 ? W::kNone * 0x10001u : W::kNone;
#pragma unroll
  for (int j = 0; j < NV; j++) {
    const int w = w0 + 256 * j + tid;
    raw[j] = none;
    if (w < whole) raw[j] = __builtin_nontemporal_load(reinterpret_cast<const Loaded*>(logits + (long)w * W::N));
  }
  if (rest != 0 && whole - w0 < 256 * NV) {   // (the same in every thread; whole >= w0)
    uint32_t v[W::N - 1];
#pragma unroll
    for (int i = 0; i < W::N - 1; i++) v[i] = logits[(long)whole * W::N + min(i, rest - 1)];
    u4_t last = none;
#pragma unroll
    for (int i = 0; i < W::N - 1; i++) {
      if (i >= rest) continue;
      if constexpr (SIZE == 2) last[i >> 1] = i & 1 ? (last[i >> 1] & 0xffffu) | v[i] << 16 : (last[i >> 1] & 0xffff0000u) | v[i];
      else last[i] = v[i];
    }
#pragma unroll
    for (int j = 0; j < NV; j++)
      if (w0 + 256 * j + tid == whole) raw[j] = last;
  }
  // Logits that are left out show in the maximum (+infinity or NaN): only then are all looked at.
  float tops[NV], top;
  auto look = [&]() __attribute__((always_inline)) {
    top = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      tops[j] = W::top(raw[j]);
      top = maximum(top, tops[j]);
    }
  };
  look();
  if (__builtin_amdgcn_ballot_w64(!(top < INFINITY))) {
#pragma unroll
    for (int j = 0; j < NV; j++) leave_out<TYPE>(raw[j]);
    look();
  }
  const float wmax = of_key(wave_max(key_of(top)));
  if (lane == 0) part[wave] = wmax;
  if (tid == 0) n_words = 0;
  __syncthreads();
  const float m = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])), ref = m == -INFINITY ? 0.f : m;
  float sum[4] = {0.f, 0.f, 0.f, 0.f}, one = 1.f;
  asm("" : "+v"(one));
#pragma unroll
  for (int j = 0; j < NV; j++) {
    asm("" : "+v"(raw[j]));   // (converted again, not held as floats)
#pragma unroll
    for (int i = 0; i < W::N; i++) {
      const float t = W::less(raw[j], i, ref, one);
      sum[i & 3] += __builtin_amdgcn_exp2f(__builtin_fmaf(t, kLog2eLo, t * kLog2eHi));
    }
  }
  const float l = wave_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
  if (lane == 0) sums[wave] = l;
  const long rec = wg * p.take;
  const int token0 = w0 * W::N;
  auto each = [&](auto&& f, float low) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NV; j++)
      if (tops[j] >= low) {
        u4_t w = raw[j];
        int at = token0 + (256 * j + tid) * W::N;
        asm volatile("" : "+v"(w), "+v"(at));   // (formed here: ahead of a loop they would fill the registers)
#pragma unroll
        for (int i = 0; i < W::N; i++) f(W::at(w, i), at + i);
      }
  };
  // Words go to LDS whole and are looked at by all threads: a wave of which one lane holds a candidate would look at
  // all 64 lanes' (35 -> 32 us for 512 rows of 131,072).
  auto gather = [&](auto&& f, float low) __attribute__((always_inline)) {
    if (top >= low) {
#pragma unroll
      for (int j = 0; j < NV; j++)
        if (tops[j] >= low) {
          const int i = atomicAdd(&n_words, 1);
          if (i < kWordCap) {
            word_s[i] = raw[j];
            word_at[i] = token0 + (256 * j + tid) * W::N;
          }
        }
    }
    __syncthreads();
    const int n = n_words;
    if (n > kWordCap) {
      if (top >= low) each(f, low);
      return;
    }
    for (int x = tid; x < n * W::N; x += 256) {
      const u4_t w = word_s[x / W::N];
      float v = -INFINITY;
#pragma unroll
      for (int i = 0; i < W::N; i++) v = x % W::N == i ? W::at(w, i) : v;
      f(v, word_at[x / W::N] + x % W::N);
    }
  };
  const int n = top_of_group<float>(found, p.take, top, each, gather, [&](int rank, float v, int at) {
    p.rec_x[rec + rank] = v;
    p.rec_at[rec + rank] = at;
  });
  for (int i = n + tid; i < p.take; i += 256) p.rec_x[rec + i] = -INFINITY;
  if (tid == 0) {   // (the sums were written ahead of a barrier in the selection)
    p.rec_sum[2 * wg] = m;
    p.rec_sum[2 * wg + 1] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }
}

// 2^24 requests, the most there may be, are two rows of workgroups, fewer are one, so that no workgroup has to look whether
// there is a request for it (0.3 of 16 us for 300).
constexpr uint32_t kJoinX = 1u << 23;

// A request's segments: every beam's logarithm of its sum, then the largest scores of what is left, RPT
// records a thread at a time together with the best of those before.
template <int RPT>
__global__ __launch_bounds__(256) void beam_join_kernel(BeamArgs p) {
  __shared__ Found<double> found;
  __shared__ double most[kMaxBeams], log_sum[kMaxBeams], best[kMaxTake];
  __shared__ int best_at[kMaxTake];
  __shared__ float score[kMaxBeams];
  __shared__ int state[kMaxBeams];   // 0: not alive, 1: searched, 2: done
  const long req = (long)(blockIdx.y * kJoinX + blockIdx.x), row0 = req * p.beams;
  const int tid = threadIdx.x, S = p.segments, k = p.take;
  const int per = S * k, total = p.beams * per;
  const float* rec_x = p.rec_x + row0 * per;
  const int32_t* rec_at = p.rec_at + row0 * per;
  float x[RPT];
  int at[RPT];
  // Of 256 records each wave takes 16 from every quarter: the wave's best, which bound what is looked at, are
  // then not those of one beam.
  const int mine = (tid & 3) * 64 + (tid >> 2);
  auto load = [&](int x0) {   // (records of beams that are not searched hold anything)
#pragma unroll
    for (int i = 0; i < RPT; i++) {
      const int r = min(x0 + 256 * i + mine, total - 1);
      x[i] = rec_x[r];
      at[i] = rec_at[r];
    }
  };
  load(0);
  // 4 lanes a beam or more
  const int lanes = p.beams <= 4 ? 64 : p.beams <= 8 ? 32 : p.beams <= 16 ? 16 : p.beams <= 32 ? 8 : 4;
  const int b = tid / lanes, part = tid % lanes;
  if (b < p.beams) {
    const long row = row0 + b;
    const float2* rec = reinterpret_cast<const float2*>(p.rec_sum) + row * S;
    const float2 one = rec[min(part, S - 1)];
    const float s = p.scores[row];
    const int over = p.done ? p.done[row] : 0;
    const bool alive = s > -INFINITY;
    float m = part < S ? one.x : -INFINITY;
    for (int i = part + lanes; i < S; i += lanes) m = fmaxf(m, rec[i].x);
    for (int d = lanes / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    double l = 0.0;
    for (int i = part; i < S; i += lanes) {
      const float2 r = i == part ? one : rec[i];
      l += r.x == m ? (double)r.y : (double)r.y * exp((double)r.x - (double)m);
    }
    for (int d = lanes / 2; d; d >>= 1) l += __shfl_xor(l, d);
    if (part == 0) {
      score[b] = s;
      state[b] = !alive ? 0 : over ? 2 : 1;
      most[b] = (double)m;
      log_sum[b] = log(l);   // (no logit: no record's value is one)
    }
  }
  __syncthreads();
  int n = 0;
  for (int x0 = 0; x0 < total; x0 += 256 * RPT) {
    if (x0 > 0) load(x0);
    // scores (-infinity: none) and, in one whole number, beam and token
    double v[RPT + 1], top = -INFINITY;
    int id[RPT + 1];
    v[RPT] = tid < n ? best[tid] : -INFINITY;
    id[RPT] = tid < n ? best_at[tid] : 0;
#pragma unroll
    for (int i = 0; i < RPT; i++) {
      const int r = x0 + 256 * i + mine, bi = min(r, total - 1) / per;
      const int st = r < total ? state[bi] : 0;
      v[i] = -INFINITY;
      id[i] = 0;
      if (st == 1 && x[i] > -INFINITY) {
        v[i] = (double)score[bi] + (((double)x[i] - most[bi]) - log_sum[bi]);
        id[i] = bi * p.vocab + at[i];
      }
      if (st == 2 && r == bi * per) {
        v[i] = (double)score[bi];
        id[i] = bi * p.vocab + p.end_token;
      }
    }
#pragma unroll
    for (int i = 0; i <= RPT; i++) top = v[i] > top ? v[i] : top;
    auto each = [&](auto&& f, double) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i <= RPT; i++) f(v[i], id[i]);
    };
    auto gather = [&](auto&& f, double low) __attribute__((always_inline)) {
      if (top >= low) each(f, low);
    };
    n = top_of_group<double>(found, k, top, each, gather, [&](int rank, double value, int what) {
      best[rank] = value;
      best_at[rank] = what;
    });
    __syncthreads();
  }
  for (int i = tid; i < k; i += 256) {
    const int bi = i < n ? best_at[i] / p.vocab : -1;
    p.parents[req * k + i] = i < n ? (int)(row0 + bi) : -1;
    p.tokens[req * k + i] = i < n ? best_at[i] - bi * p.vocab : -1;
    p.top[req * k + i] = i < n ? (float)best[i] : -INFINITY;
  }
}

// 16-byte words of a thread: few where few rows leave workgroups idle, unless a request's records then
// outgrow what its join holds at a time.
BeamPlan beam_plan(long rows, int beams, int vocab, int take, int type) {
  const int n = type == 1 ? 4 : 8;
  BeamPlan x{8, 0};
  for (int nv : {1, 4, 8}) {
    x.words = nv;
    x.segments = (int)((vocab + 256L * nv * n - 1) / (256L * nv * n));
    if (rows * x.segments <= kBeamGroups && (long)beams * x.segments * take <= kBeamRecords) break;
  }
  return x;
}

hipError_t launch_beam(BeamArgs a, const BeamPlan& plan, int type, hipStream_t stream) {
  a.segments = plan.segments;
  const dim3 grid = grid_xy((long)a.rows * a.segments), block(256);
  const unsigned n = (unsigned)(a.rows / a.beams);
  const dim3 requests = n < 2 * kJoinX ? dim3(n) : dim3(kJoinX, 2);
  auto launch = [&](auto t) {
    constexpr int T = decltype(t)::value;
    switch (plan.words) {
      case 1: hipLaunchKernelGGL((beam_rows_kernel<T, 1>), grid, block, 0, stream, a); break;
      case 4: hipLaunchKernelGGL((beam_rows_kernel<T, 4>), grid, block, 0, stream, a); break;
      default: hipLaunchKernelGGL((beam_rows_kernel<T, 8>), grid, block, 0, stream, a); break;
    }
  };
  if (type == 0) launch(std::integral_constant<int, 0>{});
  else if (type == 1) launch(std::integral_constant<int, 1>{});
  else launch(std::integral_constant<int, 2>{});
  if ((long)a.beams * a.segments * a.take <= 1024)
    hipLaunchKernelGGL(beam_join_kernel<4>, requests, block, 0, stream, a);
  else
    hipLaunchKernelGGL(beam_join_kernel<16>, requests, block, 0, stream, a);
  return hipGetLastError();
}

}  // namespace qkv
