// weigh_f8.hip -- attention weight of each key of the paged 8-bit cache, accumulated.
//
//   a_j = sum over rows r of w_rj,  w_rj = 2^(c q_r . k_j - m_r) / l_r,  m_r the largest c q_r . k_j (about),
//   l_r = sum_j 2^(c q_r . k_j - m_r),  c = scale log2(e)
//   W_j = (decay W_j where it stood before, else 0) + a_j
//
// over the rows r, (token, query head of the group) pairs, that a call has of a slot and KV head, each over the
// keys that it sees.  A row's m and l must be known before any sum over rows, so there are two passes over the scores.
//
// Few rows: keys are read once, the first pass stores the scores (4 bytes a row and key, beside head_dim bytes of
// codes), the second reads those.  Bound by HBM.
// Many rows: both passes form the scores by the matrix cores, 2 head_dim operations a row and key each; the first
// holds rows in registers and passes keys by (a lane's scores are one row's, so maximum and sum stay in it), the
// second holds keys and passes rows by (a lane's are one key's).  Bound by the matrix cores.
//
// Codes are converted to fp16 with their exponent (exact), products summed in fp32; weights are fp32 from the
// exponential on and never rounded to fewer bits.  All sums are taken in one order, whatever the timing.
#include <algorithm>

#include "qkv_device.h"
#include "qkv_launch.h"

namespace qkv {

namespace {

typedef float f16x_t __attribute__((ext_vector_type(16)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ h2_t cvt2(uint32_t w, float scale, bool hi) {
  return hi ? __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true))
            : __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
}
__device__ __forceinline__ h8_t cvt8(uint32_t a, uint32_t b, float scale) {
  const h2_t x = cvt2(a, scale, false), y = cvt2(a, scale, true), z = cvt2(b, scale, false), w = cvt2(b, scale, true);
  return h8_t{x[0], x[1], y[0], y[1], z[0], z[1], w[0], w[1]};
}
__device__ __forceinline__ float pow2f(uint32_t biased) { return __uint_as_float(biased << 23); }
// with the lane 16 and 32 away
__device__ __forceinline__ float other16(float x, int lane) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(lane & 16 ? s[0] : s[1]);
}
__device__ __forceinline__ float other32(float x, int lane) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(lane & 32 ? s[0] : s[1]);
}

// Maximum (log2 units) and sum of 2^(s - m) of a row's keys so far; m = -infinity: none.
struct Stat {
  float m, l;
};
__device__ __forceinline__ Stat join(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m), r = m == -INFINITY ? 0.f : m;
  // (a sum that is no number stays one, though its maximum may not show it)
  return {m, a.l * __builtin_amdgcn_exp2f(a.m - r) + b.l * __builtin_amdgcn_exp2f(b.m - r)};
}

struct BlockAt {
  int b, row;
};
__device__ __forceinline__ BlockAt block_at(const WeighArgs& p, int key) {
  const uint32_t q = __umulhi((uint32_t)key, p.bt_magic), x = (uint32_t)key - q * (uint32_t)p.block_tokens;
  return x >= (uint32_t)p.block_tokens ? BlockAt{(int)q + 1, (int)(x - (uint32_t)p.block_tokens)} : BlockAt{(int)q, (int)x};
}
__device__ __forceinline__ int token_of(const WeighArgs& p, int x) {
  const uint32_t q = __umulhi((uint32_t)x, p.gqa_magic), r = (uint32_t)x - q * (uint32_t)p.gqa;
  return (int)(r >= (uint32_t)p.gqa ? q + 1 : q);
}

// A slot's tokens: rows t0 .. t0+n-1 of q at positions pos0 .. (n = 0: none, or not of this launch), over keys
// below end
struct Slot {
  int t0, n, pos0, end;
};
__device__ __forceinline__ Slot slot_of(const WeighArgs& p, int s) {
  Slot x;
  x.t0 = min(max(p.starts[s], 0), (int)p.rows);
  x.n = min(min(max(p.starts[s + 1], x.t0), (int)p.rows) - x.t0, p.max_tok);
  x.pos0 = p.positions[s];
  if (x.pos0 < 0 || x.pos0 > kMaxPosition || x.n < p.from_tok || x.n > p.to_tok) x.n = 0;
  x.end = (int)min((long)x.pos0 + x.n, (long)p.max_ctx);
  return x;
}
__device__ __forceinline__ int page_of(const WeighArgs& p, const int32_t* table, int block) {
  const int pg = block < p.max_blocks ? table[block] : -1;
  return pg >= 0 && pg < p.n_pages ? pg : -1;
}
__device__ __forceinline__ bool sees(const WeighArgs& p, int key, int pos, int end) {
  return key <= pos && key < end && (p.window <= 0 || key > pos - p.window || key < p.sink);
}
// q's row of (token, head) row x, and its number among all (token, query head) rows
__device__ __forceinline__ long row_at(const WeighArgs& p, const Slot& x, int h, int row) {
  const int tok = token_of(p, row);
  return (long)(x.t0 + tok) * p.num_q + h * p.gqa + (row - tok * p.gqa);
}

// Workgroup x of `per` for one (slot, KV head)
struct Work {
  int x, s, h;
};
__device__ __forceinline__ bool work_of(const WeighArgs& p, Work& w) {
  const uint32_t wg = blockIdx.y * kGridX + blockIdx.x, head = wg / (uint32_t)p.per;
  w.x = (int)(wg - head * (uint32_t)p.per);
  w.s = (int)(head / (uint32_t)p.num_kv);
  w.h = (int)(head - (uint32_t)w.s * (uint32_t)p.num_kv);
  w.s += p.slot0;
  return w.s < p.slot_end;
}

// Whether no row of the slot sees a key of the 32 from k0 on (a multiple of 32) for its window.
__device__ __forceinline__ bool out_of_window(const WeighArgs& p, const Slot& x, int k0) {
  return p.window > 0 && k0 >= p.sink && k0 + 31 <= x.pos0 - p.window;
}

// Where the workspace holds a row's statistics (and scores): by its place in q, or, where a call's slots are taken
// few at a time, by its slot's among those.
__device__ __forceinline__ long place_of(const WeighArgs& p, const Slot& x, int s, int h, int row) {
  if (p.local_tok == 0) return row_at(p, x, h, row);
  const int tok = token_of(p, row);
  return ((long)(s - p.slot0) * p.local_tok + tok) * p.num_q + h * p.gqa + (row - tok * p.gqa);
}

}  // namespace

// ---------------------------------------------------------------------------
// few rows: up to 16 RT (token, head) rows of a slot and KV head
// ---------------------------------------------------------------------------
// A workgroup takes chunk_keys keys of a (slot, KV head), its four waves every fourth tile of 32: K rows are the A
// operand as loaded (lane l % 16 the key, group l / 16 the same dims of K and Q), so lane l has the scores of
// row l % 16 and keys 4 (l / 16) ..  Nothing is shared until the waves' statistics are joined at the end.
template <int HD, int RT>
__global__ __launch_bounds__(256, 2) void weigh_scores_kernel(WeighArgs p) {
  constexpr int KT = 32, W = 4, KW = HD / 64;
  __shared__ float ml[W][16 * RT][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  Work wk;
  if (!work_of(p, wk)) return;
  const int chunk = wk.x, h = wk.h, s = wk.s;
  const Slot sl = slot_of(p, s);
  const int first = chunk * p.chunk_keys, end = min(sl.end, first + p.chunk_keys);
  if (sl.n <= 0 || first >= sl.end) return;
  const int rows = sl.n * p.gqa;
  const int32_t* table = p.tables + (long)s * p.max_blocks;
  const uint32_t key_bytes = (uint32_t)p.num_kv * HD;

  u4_t kr[2][KW];
  uint32_t ke[2];
  int pg[2];
  auto load = [&](int key0) {
#pragma unroll
    for (int hf = 0; hf < 2; hf++) {
      const BlockAt x = block_at(p, key0 + 16 * hf);
      pg[hf] = key0 + 16 * hf < end ? page_of(p, table, x.b) : -1;
      const long page = max(pg[hf], 0);
      const uint8_t* src = p.k_pool + (page * p.block_tokens + x.row + m) * key_bytes + h * HD + 16 * g;
      ke[hf] = p.k_exp[page * p.num_kv + h];
#pragma unroll
      for (int i = 0; i < KW; i++) kr[hf][i] = *reinterpret_cast<const u4_t*>(src + 64 * i);
    }
  };
  auto next = [&](int k) {   // the wave's next tile from k on that some row sees
    while (k < end && out_of_window(p, sl, k)) k += KT * W;
    return k;
  };
  int key0 = next(first + KT * wave);
  if (key0 < end) load(key0);

  h8_t qf[RT][KW][2];
  int pos[RT];
  float* out[RT];
  Stat st[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = min(16 * t + m, rows - 1);
    const uint16_t* src = p.q + row_at(p, sl, h, row) * HD + 16 * g;
#pragma unroll
    for (int i = 0; i < KW; i++)
#pragma unroll
      for (int x = 0; x < 2; x++) qf[t][i][x] = *reinterpret_cast<const h8_t*>(src + 64 * i + 8 * x);
    pos[t] = sl.pos0 + token_of(p, row);
    out[t] = p.scores + place_of(p, sl, s, h, row) * p.score_pitch + 4 * g;
    st[t] = {-INFINITY, 0.f};
  }
  const int pos_hi = sl.pos0 + sl.n - 1;
  while (key0 < end) {
    const int key1 = next(key0 + KT * W);
    f4_t sc[RT][2];
#pragma unroll
    for (int t = 0; t < RT; t++) sc[t][0] = sc[t][1] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int hf = 0; hf < 2; hf++) {
      const float f = pow2f(ke[hf]);
#pragma unroll
      for (int i = 0; i < KW; i++)
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const h8_t a = cvt8(kr[hf][i][2 * x], kr[hf][i][2 * x + 1], f);
#pragma unroll
          for (int t = 0; t < RT; t++) sc[t][hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[t][i][x], sc[t][hf], 0, 0, 0);
        }
    }
    const bool whole = pg[0] >= 0 && pg[1] >= 0 && key0 + KT - 1 <= sl.pos0 && key0 + KT <= end &&
                       (p.window <= 0 || key0 > pos_hi - p.window || key0 + KT <= p.sink);
    const int here[2] = {pg[0], pg[1]};
    if (key1 < end) load(key1);
#pragma unroll
    for (int t = 0; t < RT; t++) {
      float top = -INFINITY;
#pragma unroll
      for (int x = 0; x < 8; x++) {
        float v = sc[t][x >> 2][x & 3] * p.scale_log2;
        if (!whole && !(here[x >> 2] >= 0 && sees(p, key0 + 16 * (x >> 2) + 4 * g + (x & 3), pos[t], end))) v = -INFINITY;
        sc[t][x >> 2][x & 3] = v;
        top = fmaxf(top, v);
      }
      const float mn = fmaxf(st[t].m, top), ref = mn == -INFINITY ? 0.f : mn;
      float l = st[t].l * __builtin_amdgcn_exp2f(st[t].m - ref);
#pragma unroll
      for (int x = 0; x < 8; x++) l += __builtin_amdgcn_exp2f(sc[t][x >> 2][x & 3] - ref);
      st[t] = {mn, l};
      if (16 * t + m < rows) {
        *reinterpret_cast<f4_t*>(out[t] + key0) = sc[t][0];
        if (key0 + 16 < end) *reinterpret_cast<f4_t*>(out[t] + key0 + 16) = sc[t][1];
      }
    }
    key0 = key1;
  }
#pragma unroll
  for (int t = 0; t < RT; t++) {
    st[t] = join(st[t], Stat{other16(st[t].m, lane), other16(st[t].l, lane)});
    st[t] = join(st[t], Stat{other32(st[t].m, lane), other32(st[t].l, lane)});
    if (g == 0) {
      ml[wave][16 * t + m][0] = st[t].m;
      ml[wave][16 * t + m][1] = st[t].l;
    }
  }
  __syncthreads();
  if (tid < rows) {
    Stat x{ml[0][tid][0], ml[0][tid][1]};
#pragma unroll
    for (int w = 1; w < W; w++) x = join(x, Stat{ml[w][tid][0], ml[w][tid][1]});
    *reinterpret_cast<f2_t*>(p.rec + (place_of(p, sl, s, h, tid) * p.chunks + chunk) * 2) = f2_t{x.m, x.l};
  }
}

// m and 1 / l of every row from its chunks' statistics, 16 lanes a row; (infinity, 0) where a row sees no key.
__global__ __launch_bounds__(256) void weigh_merge_kernel(WeighArgs p) {
  Work wk;
  if (!work_of(p, wk)) return;
  const int tid = threadIdx.x, part = tid & 15, s = wk.s, h = wk.h;
  const Slot sl = slot_of(p, s);
  const int row = wk.x * 16 + (tid >> 4), rows = sl.n * p.gqa;
  if (row >= rows) return;
  // the chunks that the row's tile was formed over
  const int tile_end = p.tile_rows ? min(sl.pos0 + token_of(p, min(rows, (row / p.tile_rows + 1) * p.tile_rows) - 1) + 1, p.max_ctx) : sl.end;
  const int n = (tile_end + p.chunk_keys - 1) / p.chunk_keys;
  const long at = place_of(p, sl, s, h, row);
  const f2_t* rec = reinterpret_cast<const f2_t*>(p.rec) + at * p.chunks;
  Stat x{-INFINITY, 0.f};
  for (int c = part; c < n; c += 16) x = join(x, Stat{rec[c][0], rec[c][1]});
#pragma unroll
  for (int d = 8; d; d >>= 1) x = join(x, Stat{__shfl_xor(x.m, d), __shfl_xor(x.l, d)});
  if (part == 0) *reinterpret_cast<f2_t*>(p.stat + 2 * at) = x.l == 0.f ? f2_t{INFINITY, 0.f} : f2_t{x.m, 1.f / x.l};
}

// What a key's weight becomes (a key whose page is absent has none).
__device__ __forceinline__ void put_weight(const WeighArgs& p, const int32_t* table, int h, int key, int weighed, float a) {
  const BlockAt x = block_at(p, key);
  const int pg = page_of(p, table, x.b);
  if (pg < 0) return;
  float* w = p.weights + ((long)pg * p.num_kv + h) * p.block_tokens + x.row;
  *w = key < weighed && p.decay != 0.f ? __builtin_fmaf(p.decay, *w, a) : a;
}

// Few rows: 1,024 keys a workgroup, four of a thread.
__global__ __launch_bounds__(256) void weigh_few_kernel(WeighArgs p) {
  constexpr int ROWS = 64;
  __shared__ f2_t stat[ROWS];
  __shared__ long at[ROWS];
  Work wk;
  if (!work_of(p, wk)) return;
  const int tid = threadIdx.x, h = wk.h, s = wk.s;
  const Slot sl = slot_of(p, s);
  const int key = wk.x * 1024 + 4 * tid;
  if (sl.n <= 0 || wk.x * 1024 >= sl.end) return;
  const int rows = sl.n * p.gqa;
  if (tid < rows) {
    const long x = place_of(p, sl, s, h, tid);
    at[tid] = x * p.score_pitch;
    stat[tid] = *reinterpret_cast<const f2_t*>(p.stat + 2 * x);
  }
  __syncthreads();
  if (key >= sl.end) return;
  f4_t a = {0.f, 0.f, 0.f, 0.f};
  const bool out = out_of_window(p, sl, key & ~31);   // (its scores were not stored)
  for (int r = 0; r < rows && !out; r++) {
    const f4_t v = *reinterpret_cast<const f4_t*>(p.scores + at[r] + key);
#pragma unroll
    for (int i = 0; i < 4; i++) a[i] += v[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v[i] - stat[r][0]) * stat[r][1];
  }
  const int32_t* table = p.tables + (long)s * p.max_blocks;
  const int weighed = p.weighed ? p.weighed[s] : sl.pos0;
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (key + i < sl.end) put_weight(p, table, h, key + i, weighed, a[i]);
}

// ---------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------
// Statistics: four waves of 64 rows, whose queries stay in registers, over chunk_keys keys, 32 at a time through
// LDS as fp16 (converted once for all waves).
template <int HD>
__global__ __launch_bounds__(256, 2) void weigh_stats_kernel(WeighArgs p) {
  constexpr int KT = 32, KP = HD * 2 + 16, NB = HD / 16, LD = HD / 128;   // LD: 16-byte loads of a thread and tile
  __shared__ __align__(16) uint8_t k_lds[2][KT * KP];
  __shared__ int page_lds[2][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hh = lane >> 5;
  Work wk;
  if (!work_of(p, wk)) return;
  const int tile = wk.x / p.chunks, chunk = wk.x - tile * p.chunks, h = wk.h, s = wk.s;
  const Slot sl = slot_of(p, s);
  const int rows = sl.n * p.gqa, r0 = tile * kWeighRows;
  if (sl.n <= 0 || r0 >= rows) return;
  const int tile_lo = sl.pos0 + token_of(p, r0), tile_hi = sl.pos0 + token_of(p, min(rows, r0 + kWeighRows) - 1);
  const int end = min(tile_hi + 1, p.max_ctx), first = chunk * p.chunk_keys;
  if (first >= end) return;
  const int32_t* table = p.tables + (long)s * p.max_blocks;
  const uint32_t key_bytes = (uint32_t)p.num_kv * HD;

  const int row_w = r0 + wave * 64;
  h8_t qf[2][NB];
  int pos[2];
  long at[2];
#pragma unroll
  for (int b = 0; b < 2; b++) {
    const int row = min(row_w + 32 * b + c, rows - 1);
    at[b] = row_at(p, sl, h, row);
    pos[b] = sl.pos0 + token_of(p, row);
    const uint16_t* src = p.q + at[b] * HD + 8 * hh;
#pragma unroll
    for (int i = 0; i < NB; i++) qf[b][i] = *reinterpret_cast<const h8_t*>(src + 16 * i);
  }
  const bool live = row_w < rows;
  const int pos_lo = sl.pos0 + token_of(p, min(row_w, rows - 1)), pos_hi = sl.pos0 + token_of(p, min(row_w + 64, rows) - 1);

  // tiles of the chunk that some row sees: on to the window past the sinks
  const int stop = min(end, first + p.chunk_keys);
  const int w0 = p.window > 0 ? max(0, tile_lo - p.window + 1) / KT * KT : 0;
  auto skip = [&](int k0) { return k0 >= p.sink && k0 < w0 ? max(w0, first) : k0; };

  u4_t raw[LD];
  uint32_t ex = 0;
  int pg = -1;
  const int ld_key = tid >> 3, ld_part = tid & 7;
  auto load = [&](int k0) {
    const BlockAt x = block_at(p, k0 + ld_key);
    pg = k0 + ld_key < end ? page_of(p, table, x.b) : -1;
    const long page = max(pg, 0);
    const uint8_t* src = p.k_pool + (page * p.block_tokens + x.row) * key_bytes + h * HD + ld_part * 16 * LD;
    ex = p.k_exp[page * p.num_kv + h];
#pragma unroll
    for (int i = 0; i < LD; i++) raw[i] = *reinterpret_cast<const u4_t*>(src + 16 * i);
  };
  auto store = [&](int buf) {
    const float f = pow2f(ex);
    uint8_t* dst = k_lds[buf] + ld_key * KP + ld_part * 32 * LD;
#pragma unroll
    for (int i = 0; i < LD; i++) {
      *reinterpret_cast<h8_t*>(dst + 32 * i) = cvt8(raw[i][0], raw[i][1], f);
      *reinterpret_cast<h8_t*>(dst + 32 * i + 16) = cvt8(raw[i][2], raw[i][3], f);
    }
    if ((ld_key & 15) == 0 && ld_part == 0) page_lds[buf][ld_key >> 4] = pg;
  };
  Stat st[2] = {{-INFINITY, 0.f}, {-INFINITY, 0.f}};
  int k0 = skip(first), buf = 0;
  if (k0 < stop) {
    load(k0);
    store(0);
  }
  while (k0 < stop) {
    const int next = skip(k0 + KT);
    if (next < stop) load(next);
    __syncthreads();   // (this tile is stored; the one before is done with)
    const int pg0 = page_lds[buf][0], pg1 = page_lds[buf][1];
    if (live && k0 <= pos_hi) {
      f16x_t acc[2] = {f16x_t{}, f16x_t{}};
      const uint8_t* src = k_lds[buf] + c * KP + 16 * hh;
#pragma unroll
      for (int i = 0; i < NB; i++) {
        const h8_t a = *reinterpret_cast<const h8_t*>(src + 32 * i);
#pragma unroll
        for (int b = 0; b < 2; b++) acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qf[b][i], acc[b], 0, 0, 0);
      }
      const bool whole = pg0 >= 0 && pg1 >= 0 && k0 + KT - 1 <= pos_lo && k0 + KT <= end &&
                         (p.window <= 0 || k0 > pos_hi - p.window || k0 + KT <= p.sink);
#pragma unroll
      for (int b = 0; b < 2; b++) {
        // lane c's row, keys 8 (x / 4) + 4 hh + x % 4
        float top = -INFINITY;
        uint32_t seen = 0xffffu;
        if (!whole) {
          seen = 0;
#pragma unroll
          for (int x = 0; x < 16; x++)
            seen |= (x < 8 ? pg0 : pg1) >= 0 && sees(p, k0 + 8 * (x >> 2) + 4 * hh + (x & 3), pos[b], end) ? 1u << x : 0u;
#pragma unroll
          for (int x = 0; x < 16; x++) top = fmaxf(top, seen >> x & 1 ? acc[b][x] * p.scale_log2 : -INFINITY);
        } else {
#pragma unroll
          for (int x = 0; x < 16; x++) top = fmaxf(top, acc[b][x] * p.scale_log2);
        }
        const float mn = fmaxf(st[b].m, top), ref = mn == -INFINITY ? 0.f : mn;
        float l = st[b].l * __builtin_amdgcn_exp2f(st[b].m - ref);
#pragma unroll
        for (int x = 0; x < 16; x++) {
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[b][x], p.scale_log2, -ref));
          l += whole || (seen >> x & 1) ? w : 0.f;
        }
        st[b] = {mn, l};
      }
    }
    buf ^= 1;
    if (next < stop) store(buf);
    k0 = next;
  }
#pragma unroll
  for (int b = 0; b < 2; b++) {
    const Stat x = join(st[b], Stat{other32(st[b].m, lane), other32(st[b].l, lane)});
    if (hh == 0 && row_w + 32 * b + c < rows) *reinterpret_cast<f2_t*>(p.rec + (at[b] * p.chunks + chunk) * 2) = f2_t{x.m, x.l};
  }
}

// Sums: four waves of 64 keys, which stay in registers as fp16, over kWeighSpan rows, 32 at a time through LDS.
template <int HD>
__global__ __launch_bounds__(256, 2) void weigh_sums_kernel(WeighArgs p) {
  constexpr int RT = 32, QP = HD * 2 + 16, NB = HD / 16, LD = HD / 64;   // LD: 16-byte loads of a thread and tile
  __shared__ __align__(16) uint8_t q_lds[2][RT * QP];
  __shared__ __align__(16) float m_lds[2][RT], il_lds[2][RT];
  __shared__ __align__(16) int pos_lds[2][RT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hh = lane >> 5;
  Work wk;
  if (!work_of(p, wk)) return;
  const int tile = wk.x / p.spans, span = wk.x - tile * p.spans, h = wk.h, s = wk.s;
  const Slot sl = slot_of(p, s);
  const int rows = sl.n * p.gqa, k0 = tile * kWeighKeys;
  if (sl.n <= 0 || k0 >= sl.end || span * kWeighSpan >= rows) return;
  const int32_t* table = p.tables + (long)s * p.max_blocks;
  const uint32_t key_bytes = (uint32_t)p.num_kv * HD;
  const int key_w = k0 + wave * 64;

  // rows of the span that see a key of the tile
  const int k1 = min(k0 + kWeighKeys, sl.end) - 1;
  long lo = (long)max(0, k0 - sl.pos0) * p.gqa, hi = rows;
  if (p.window > 0 && k0 >= p.sink) hi = min(hi, max(0l, (long)k1 + p.window - sl.pos0) * p.gqa);
  const int r_lo = (int)max(lo, (long)span * kWeighSpan) / RT * RT, r_hi = (int)min(hi, (long)(span + 1) * kWeighSpan);

  h8_t kf[2][NB];
  float sum[2] = {0.f, 0.f};
  if (r_lo < r_hi) {
#pragma unroll
    for (int b = 0; b < 2; b++) {
      const int key = key_w + 32 * b + c;
      const BlockAt x = block_at(p, min(key, sl.end - 1));
      const long page = max(page_of(p, table, x.b), 0);
      const uint8_t* src = p.k_pool + (page * p.block_tokens + x.row) * key_bytes + h * HD + 8 * hh;
      const float f = pow2f(p.k_exp[page * p.num_kv + h]);
#pragma unroll
      for (int i = 0; i < NB; i++) {
        const u2_t w = *reinterpret_cast<const u2_t*>(src + 16 * i);
        kf[b][i] = cvt8(w[0], w[1], f);
      }
    }
  }
  u4_t raw[LD];
  f2_t stat = {0.f, 0.f};
  int pos = 0;
  const int ld_row = tid >> 3, ld_part = tid & 7;
  auto load = [&](int r0) {
    const int row = min(r0 + ld_row, rows - 1);
    const long at = row_at(p, sl, h, row);
    const uint16_t* src = p.q + at * HD + ld_part * 8 * LD;
#pragma unroll
    for (int i = 0; i < LD; i++) raw[i] = *reinterpret_cast<const u4_t*>(src + 8 * i);
    stat = *reinterpret_cast<const f2_t*>(p.stat + 2 * at);
    pos = r0 + ld_row < r_hi ? sl.pos0 + token_of(p, row) : -1;   // (-1: no row, sees nothing)
  };
  auto store = [&](int buf) {
    uint8_t* dst = q_lds[buf] + ld_row * QP + ld_part * 16 * LD;
#pragma unroll
    for (int i = 0; i < LD; i++) *reinterpret_cast<u4_t*>(dst + 16 * i) = raw[i];
    if (ld_part == 0) {
      m_lds[buf][ld_row] = stat[0];
      il_lds[buf][ld_row] = stat[1];
      pos_lds[buf][ld_row] = pos;
    }
  };
  int buf = 0;
  if (r_lo < r_hi) {
    load(r_lo);
    store(0);
  }
  for (int r0 = r_lo; r0 < r_hi; r0 += RT) {
    if (r0 + RT < r_hi) load(r0 + RT);
    __syncthreads();
    const int pos_lo = r0 + RT <= r_hi ? pos_lds[buf][0] : -1, pos_hi = sl.pos0 + token_of(p, min(r0 + RT, rows) - 1);
    if (key_w <= pos_hi) {
      f16x_t acc[2] = {f16x_t{}, f16x_t{}};
      const uint8_t* src = q_lds[buf] + c * QP + 16 * hh;
#pragma unroll
      for (int i = 0; i < NB; i++) {
        const h8_t a = *reinterpret_cast<const h8_t*>(src + 32 * i);
#pragma unroll
        for (int b = 0; b < 2; b++) acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, kf[b][i], acc[b], 0, 0, 0);
      }
      const bool whole = key_w + 63 <= pos_lo && (p.window <= 0 || key_w > pos_hi - p.window || key_w + 64 <= p.sink);
      // lane c's key, rows 8 (x / 4) + 4 hh + x % 4
#pragma unroll
      for (int x4 = 0; x4 < 4; x4++) {
        const f4_t mr = *reinterpret_cast<const f4_t*>(&m_lds[buf][8 * x4 + 4 * hh]);
        const f4_t il = *reinterpret_cast<const f4_t*>(&il_lds[buf][8 * x4 + 4 * hh]);
        const int4 pr = *reinterpret_cast<const int4*>(&pos_lds[buf][8 * x4 + 4 * hh]);
        const int pos_r[4] = {pr.x, pr.y, pr.z, pr.w};
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int x = 0; x < 4; x++) {
            float w = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[b][4 * x4 + x], p.scale_log2, -mr[x])) * il[x];
            if (!whole && !sees(p, key_w + 32 * b + c, pos_r[x], sl.end)) w = 0.f;
            sum[b] += w;
          }
      }
    }
    buf ^= 1;
    if (r0 + RT < r_hi) store(buf);
  }
  // (both halves of the lanes have the same keys, other rows)
  float* out = p.partial + ((long)(sl.t0 * (long)p.gqa / kWeighSpan + s + span) * p.num_kv + h) * p.max_ctx;
#pragma unroll
  for (int b = 0; b < 2; b++) {
    const float a = sum[b] + other32(sum[b], lane);
    if (hh == 0 && key_w + 32 * b + c < sl.end) out[key_w + 32 * b + c] = a;
  }
}

// Many rows: the spans' sums into the weights.
__global__ __launch_bounds__(256) void weigh_many_kernel(WeighArgs p) {
  Work wk;
  if (!work_of(p, wk)) return;
  const int h = wk.h, s = wk.s, key = wk.x * 256 + (int)threadIdx.x;
  const Slot sl = slot_of(p, s);
  if (sl.n <= 0 || key >= sl.end) return;
  const int spans = (sl.n * p.gqa + kWeighSpan - 1) / kWeighSpan;
  const float* in = p.partial + ((long)(sl.t0 * (long)p.gqa / kWeighSpan + s) * p.num_kv + h) * p.max_ctx + key;
  float a = 0.f;
  for (int i = 0; i < spans; i++) a += in[(long)i * p.num_kv * p.max_ctx];
  put_weight(p, p.tables + (long)s * p.max_blocks, h, key, p.weighed ? p.weighed[s] : sl.pos0, a);
}

WeighPlan weigh_plan(int num_q, int num_kv, int n_slots, long rows, int max_tok, int max_ctx) {
  const int gqa = num_q / num_kv;
  WeighPlan x{};
  x.pitch = (max_ctx + 31l) / 32 * 32;
  // slots of up to 64 rows store their scores, as many slots at a time as kWeighScores bytes hold
  const double token = (double)num_q * x.pitch * 4;
  x.few_tok = (int)std::min((double)std::min(64 / gqa, max_tok), kWeighScores / token);
  x.many = max_tok > x.few_tok;
  if (x.many && n_slots == 1) x.few_tok = 0;
  if (x.few_tok > 0) x.few_slots = (int)std::min((double)n_slots, kWeighScores / (token * x.few_tok));
  // of these, workgroups enough for the CUs also where the slots are few, of 128 keys at least
  const long target = std::min(256l, std::max(16l, 8192l / std::max(1l, (long)x.few_slots * num_kv)));
  x.few_keys = (int)(128 * ((max_ctx + 128 * target - 1) / (128 * target)));
  x.few_chunks = (max_ctx + x.few_keys - 1) / x.few_keys;
  x.many_chunks = (max_ctx + kWeighChunk - 1) / kWeighChunk;
  const size_t few_rows = (size_t)x.few_slots * x.few_tok * num_q, all = (size_t)rows * num_q;
  const size_t many_sums = ((size_t)rows * gqa / kWeighSpan + n_slots) * num_kv * max_ctx;
  x.stat_bytes = 8 * std::max(few_rows, x.many ? all : 0);
  x.rec_bytes = 8 * std::max(few_rows * x.few_chunks, x.many ? all * x.many_chunks : 0);
  x.sum_bytes = 4 * std::max(few_rows * x.pitch, x.many ? many_sums : 0);
  return x;
}

hipError_t launch_weigh(WeighArgs a, const WeighPlan& x, int head_dim, hipStream_t stream) {
  const dim3 block(256);
  auto launch = [&](auto kernel, long per) {
    a.per = (int)per;
    hipLaunchKernelGGL(kernel, grid_xy(per * (a.slot_end - a.slot0) * a.num_kv), block, 0, stream, a);
  };
  if (x.few_tok > 0) for (a.slot0 = 0; a.slot0 < a.n_slots; a.slot0 += x.few_slots) {
    a.slot_end = std::min(a.n_slots, a.slot0 + x.few_slots);
    a.local_tok = x.few_tok;
    a.from_tok = 1;
    a.to_tok = x.few_tok;
    a.chunk_keys = x.few_keys;
    a.chunks = x.few_chunks;
    a.tile_rows = 0;
    const int rows = x.few_tok * a.gqa;
    if (head_dim == 128) {
      if (rows <= 16) launch(weigh_scores_kernel<128, 1>, a.chunks);
      else if (rows <= 32) launch(weigh_scores_kernel<128, 2>, a.chunks);
      else launch(weigh_scores_kernel<128, 4>, a.chunks);
    } else {
      if (rows <= 16) launch(weigh_scores_kernel<256, 1>, a.chunks);
      else if (rows <= 32) launch(weigh_scores_kernel<256, 2>, a.chunks);
      else launch(weigh_scores_kernel<256, 4>, a.chunks);
    }
    launch(weigh_merge_kernel, (rows + 15) / 16);
    launch(weigh_few_kernel, (a.max_ctx + 1023l) / 1024);
  }
  if (x.many) {
    a.slot0 = 0;
    a.slot_end = a.n_slots;
    a.local_tok = 0;
    a.from_tok = x.few_tok + 1;
    a.to_tok = 0x7fffffff;
    a.chunk_keys = kWeighChunk;
    a.chunks = x.many_chunks;
    a.tile_rows = kWeighRows;
    const long rows = (long)a.max_tok * a.gqa;
    a.spans = (int)((rows + kWeighSpan - 1) / kWeighSpan);
    const long tiles = (rows + kWeighRows - 1) / kWeighRows, keys = (a.max_ctx + kWeighKeys - 1l) / kWeighKeys;
    if (head_dim == 128) launch(weigh_stats_kernel<128>, tiles * a.chunks);
    else launch(weigh_stats_kernel<256>, tiles * a.chunks);
    launch(weigh_merge_kernel, (rows + 15) / 16);
    if (head_dim == 128) launch(weigh_sums_kernel<128>, keys * a.spans);
    else launch(weigh_sums_kernel<256>, keys * a.spans);
    launch(weigh_many_kernel, (a.max_ctx + 255l) / 256);
  }
  return hipGetLastError();
}

}  // namespace qkv
