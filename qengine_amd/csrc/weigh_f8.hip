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
// codes), the second reads those.  Bound by HBM: 32 single tokens over 333 MB of codes take 77 + 10 us, 5.0 TB/s (without
// the scores' 23 MB of stores 60; past the caches 79).  Two tiles of a wave under way, or the keys of all slots as one line
// of equal parts, were slower by 4 to 7.
// Many rows: both passes form the scores by the matrix cores, 2 head_dim operations a row and key each; the first
// holds rows in registers and passes keys by (a lane's scores are one row's, so maximum and sum stay in it), the
// second holds keys and passes rows by (a lane's are one key's).  Bound by the vector unit and the matrix cores together:
// 164 million scores of 128 dims take 55 + 65 us (34 each at a large library product's rate), 138 million of 256 dims 84 +
// 93 (60 each).
//
// Codes are converted to fp16 with their exponent (exact), products summed in fp32; weights are fp32 from the
// exponential on and never rounded to fewer bits.  All sums are taken in one order, whatever the timing.
#include <algorithm>

#include "f8_line.h"
#include "qkv_device.h"
#include "qkv_launch.h"

namespace qkv {

namespace {

typedef float f16x_t __attribute__((ext_vector_type(16)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(4))) const int32_t const_i32;   // (read by scalar loads)
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void glb_void;

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
  const const_i32 *starts = (const const_i32*)p.starts + s, *positions = (const const_i32*)p.positions + s;
  Slot x;
  x.t0 = min(max(starts[0], 0), (int)p.rows);
  x.n = min(min(max(starts[1], x.t0), (int)p.rows) - x.t0, p.max_tok);
  x.pos0 = positions[0];
  if (x.pos0 < 0 || x.pos0 > kMaxPosition || x.n < p.from_tok || x.n > p.to_tok) x.n = 0;
  x.end = (int)min((long)x.pos0 + x.n, (long)p.max_ctx);
  return x;
}
// (T: const_i32 for a block that the whole wave asks for, by a scalar load: a vector load's wait would be for all
// loads under way)
template <class T>
__device__ __forceinline__ int page_of(const WeighArgs& p, const T* table, int block) {
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

// Workgroup x of those for one (slot, KV head).  Workgroups go round the XCDs in order, so the pairs are turned
// by one with each x: no XCD has the same pair, or the same x, each time.
struct Work {
  int x, s, h;
};
__device__ __forceinline__ bool work_of(const WeighArgs& p, Work& w) {
  const uint32_t wg = blockIdx.y * kGridX + blockIdx.x, x = wg / (uint32_t)p.heads, head = (wg + x) % (uint32_t)p.heads;
  w.x = (int)x;
  w.s = (int)(head / (uint32_t)p.num_kv);
  w.h = (int)(head - (uint32_t)w.s * (uint32_t)p.num_kv);
  w.s += p.slot0;
  return x < (uint32_t)p.per;
}

// Whether no row of the slot sees a key of the 32 from k0 on (a multiple of 32) for its window.
__device__ __forceinline__ bool out_of_window(const WeighArgs& p, const Slot& x, int k0) {
  return p.window > 0 && k0 >= p.sink && k0 + 31 <= x.pos0 - p.window;
}

// m and 1 / l of a row; (infinity, 0) where it sees no key.
__device__ __forceinline__ void put_stat(const WeighArgs& p, long at, Stat x) {
  p.stat_m[at] = x.l == 0.f ? INFINITY : x.m;
  p.stat_il[at] = x.l == 0.f ? 0.f : 1.f / x.l;
}

// Where the workspace holds a row's statistics (and scores): by its place in q, or, where a call's slots are taken
// few at a time, by its slot's among those.
__device__ __forceinline__ long place_of(const WeighArgs& p, const Slot& x, int s, int h, int row) {
  if (p.local_tok == 0) return row_at(p, x, h, row);
  const int tok = token_of(p, row);
  return ((long)(s - p.slot0) * p.local_tok + tok) * p.num_q + h * p.gqa + (row - tok * p.gqa);
}

// Where the workspace holds the scores of a (slot, KV head): 32 keys of all its rows, then the next 32.
__device__ __forceinline__ long scores_of(const WeighArgs& p, int s, int h) {
  return ((long)(s - p.slot0) * p.num_kv + h) * (p.local_tok * p.gqa) * p.score_pitch;
}

}  // namespace

// ---------------------------------------------------------------------------
// few rows: up to 16 RT (token, head) rows of a slot and KV head
// ---------------------------------------------------------------------------
// A workgroup takes chunk_keys keys of a (slot, KV head), its four waves every fourth tile of 32.  A tile's rows are
// loaded whole lines at a time, past the caches (each byte is used once; as the operand asks for them, 64 bytes of 16
// rows at a time, 87 us, now 77), and pass through LDS of the wave's own, their 16-byte words permuted by the row's
// number.  K rows are the A operand (lane l % 16 the key, group l / 16 the same dims of K and Q), so lane l has the
// scores of row l % 16 and keys 4 (l / 16) ..  Nothing is shared until the waves' statistics are joined at the end.
template <int HD, int RT>
__global__ __launch_bounds__(256, 2) void weigh_scores_kernel(WeighArgs p) {
  constexpr int KT = 32, W = 4, KW = HD / 64, LPR = HD / 16, RL = 64 / LPR;
  __shared__ float ml[W][16 * RT][2];
  __shared__ __align__(16) uint8_t tile_s[W][KT * HD];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  Work wk;
  if (!work_of(p, wk)) return;
  const int chunk = wk.x, h = wk.h, s = wk.s;
  const Slot sl = slot_of(p, s);
  const int first = chunk * p.chunk_keys, end = min(sl.end, first + p.chunk_keys);
  if (sl.n <= 0 || first >= sl.end) return;
  const int rows = sl.n * p.gqa;
  const const_i32* table = (const const_i32*)(p.tables + (long)s * p.max_blocks);
  const uint32_t key_bytes = (uint32_t)p.num_kv * HD;

  u4_t kr[2][KW];   // RL rows each, a row's words by LPR lanes
  uint8_t ke[2];   // (widened where it is used: a wait)
  int pg[2];
  uint8_t* tile = tile_s[wave];
  auto word_at = [&](int row, int word) {   // (no two of 16 rows' same words on one bank)
    return reinterpret_cast<u4_t*>(tile + row * HD + (word ^ ((HD == 256 ? row : row >> 1) & (LPR - 1))) * 16);
  };
  auto load = [&](int key0) {
#pragma unroll
    for (int hf = 0; hf < 2; hf++) {
      const BlockAt x = block_at(p, key0 + 16 * hf);
      pg[hf] = key0 + 16 * hf < end ? page_of(p, table, x.b) : -1;
      const long page = max(pg[hf], 0);
      const uint8_t* src = p.k_pool + (page * p.block_tokens + x.row + lane / LPR) * key_bytes + h * HD + 16 * (lane % LPR);
      ke[hf] = p.k_exp[page * p.num_kv + h];
#pragma unroll
      for (int i = 0; i < KW; i++) kr[hf][i] = __builtin_nontemporal_load(reinterpret_cast<const u4_t*>(src + i * RL * key_bytes));
    }
  };
  // (a wave's accesses to LDS are in order, also of different lanes: so the compiler has to leave them)
  auto in_order = [&]() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
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
    out[t] = p.scores + scores_of(p, s, h) + 32 * row + 4 * g;
    st[t] = {-INFINITY, 0.f};
  }
  // (the queries are here: in the loop the wait for them would be one for the next tile's loads)
#pragma unroll
  for (int t = 0; t < RT; t++)
#pragma unroll
    for (int i = 0; i < KW; i++)
#pragma unroll
      for (int x = 0; x < 2; x++) asm volatile("" : "+v"(qf[t][i][x]));
  const int pos_hi = sl.pos0 + sl.n - 1;
  while (key0 < end) {
    const int key1 = next(key0 + KT * W);
    const float pow[2] = {pow2f(ke[0]), pow2f(ke[1])};
    in_order();
#pragma unroll
    for (int hf = 0; hf < 2; hf++)
#pragma unroll
      for (int i = 0; i < KW; i++) *word_at(16 * hf + i * RL + lane / LPR, lane % LPR) = kr[hf][i];
    const bool whole = pg[0] >= 0 && pg[1] >= 0 && key0 + KT - 1 <= sl.pos0 && key0 + KT <= end &&
                       (p.window <= 0 || key0 > pos_hi - p.window || key0 + KT <= p.sink);
    const int here[2] = {pg[0], pg[1]};
    if (key1 < end) load(key1);
    in_order();
    f4_t sc[RT][2];
#pragma unroll
    for (int t = 0; t < RT; t++) sc[t][0] = sc[t][1] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int hf = 0; hf < 2; hf++) {
#pragma unroll
      for (int i = 0; i < KW; i++) {
        const u4_t w = *word_at(16 * hf + m, 4 * i + g);
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const h8_t a = cvt8(w[2 * x], w[2 * x + 1], pow[hf]);
#pragma unroll
          for (int t = 0; t < RT; t++) sc[t][hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[t][i][x], sc[t][hf], 0, 0, 0);
        }
      }
    }
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
        *reinterpret_cast<f4_t*>(out[t] + (long)key0 * rows) = sc[t][0];
        if (key0 + 16 < end) *reinterpret_cast<f4_t*>(out[t] + (long)key0 * rows + 16) = sc[t][1];
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

// A row's statistics from its chunks', by 16 neighbouring lanes (lane `part` of them), in each of these.
__device__ __forceinline__ Stat join_chunks(const WeighArgs& p, const Slot& sl, long at, int part) {
  const int n = (sl.end + p.chunk_keys - 1) / p.chunk_keys;
  const f2_t* rec = reinterpret_cast<const f2_t*>(p.rec) + at * p.chunks;
  Stat x{-INFINITY, 0.f};
  for (int c = part; c < n; c += 16) x = join(x, Stat{rec[c][0], rec[c][1]});
#pragma unroll
  for (int d = 8; d; d >>= 1) x = join(x, Stat{__shfl_xor(x.m, d), __shfl_xor(x.l, d)});
  return x;
}

// The statistics of every row, where the next kernel's workgroups would be long in joining those of a slot each.
__global__ __launch_bounds__(256) void weigh_merge_kernel(WeighArgs p) {
  Work wk;
  if (!work_of(p, wk)) return;
  const int tid = threadIdx.x, s = wk.s, h = wk.h;
  const Slot sl = slot_of(p, s);
  const int row = wk.x * 16 + (tid >> 4);
  if (row >= sl.n * p.gqa) return;
  const long at = place_of(p, sl, s, h, row);
  const Stat x = join_chunks(p, sl, at, tid & 15);
  if ((tid & 15) == 0) put_stat(p, at, x);
}

// What a key's weight becomes.
__device__ __forceinline__ float weight_of(const WeighArgs& p, int key, int weighed, float old, float a) {
  return key < weighed && p.decay != 0.f ? __builtin_fmaf(p.decay, old, a) : a;
}
// (a key whose page is absent has none)
__device__ __forceinline__ void put_weight(const WeighArgs& p, const int32_t* table, int h, int key, int weighed, float a) {
  const BlockAt x = block_at(p, key);
  const int pg = page_of(p, table, x.b);
  if (pg < 0) return;
  float* w = p.weights + ((long)pg * p.num_kv + h) * p.block_tokens + x.row;
  *w = weight_of(p, key, weighed, *w, a);
}

// Few rows: 1,024 keys a workgroup, four of a thread.  MERGED: by the rows' statistics, else by their chunks'.
template <bool MERGED>
__global__ __launch_bounds__(256) void weigh_few_kernel(WeighArgs p) {
  constexpr int ROWS = 64;
  __shared__ f2_t stat[ROWS];
  Work wk;
  if (!work_of(p, wk)) return;
  const int tid = threadIdx.x, h = wk.h, s = wk.s;
  const Slot sl = slot_of(p, s);
  const int key = wk.x * 1024 + 4 * tid;
  if (sl.n <= 0 || wk.x * 1024 >= sl.end) return;
  const int rows = sl.n * p.gqa;
  // What does not wait for the statistics, ahead of them: the keys' page (4 keys lie in one), their weights, and the
  // scores of the first rows.
  constexpr int AHEAD = 4;
  const bool live = key < sl.end;
  const int key_l = live ? key : 0;
  const BlockAt bl = block_at(p, key_l);
  const int pg = page_of(p, p.tables + (long)s * p.max_blocks, bl.b);
  const int weighed = p.weighed ? p.weighed[s] : sl.pos0;
  float* w = p.weights + ((long)max(pg, 0) * p.num_kv + h) * p.block_tokens + bl.row;
  const bool out = out_of_window(p, sl, key & ~31);   // (its scores were not stored)
  const float* score = p.scores + scores_of(p, s, h) + (long)(key_l & ~31) * rows + (key_l & 31);
  f4_t old, ahead[AHEAD];
#pragma unroll
  for (int i = 0; i < 4; i++) old[i] = w[i];
#pragma unroll
  for (int r = 0; r < AHEAD; r++)
    ahead[r] = *reinterpret_cast<const f4_t*>(score + 32 * min(r, rows - 1));
  if constexpr (MERGED) {
    if (tid < rows) {
      const long x = place_of(p, sl, s, h, tid);
      stat[tid] = f2_t{p.stat_m[x], p.stat_il[x]};
    }
  } else {
    for (int r = tid >> 4; r < rows; r += 16) {
      const long x = place_of(p, sl, s, h, r);
      const Stat st = join_chunks(p, sl, x, tid & 15);
      if ((tid & 15) == 0) {
        stat[r] = st.l == 0.f ? f2_t{INFINITY, 0.f} : f2_t{st.m, 1.f / st.l};
      }
    }
  }
  __syncthreads();
  if (!live || pg < 0) return;   // (a key whose page is absent has no weight)
  f4_t a = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](const f4_t& v, int r) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; i++) a[i] += v[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v[i] - stat[r][0]) * stat[r][1];
  };
  if (!out) {
#pragma unroll
    for (int r = 0; r < AHEAD; r++)
      if (r < rows) add(ahead[r], r);
    for (int r = AHEAD; r < rows; r++) add(*reinterpret_cast<const f4_t*>(score + 32 * r), r);
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (key + i < sl.end) w[i] = weight_of(p, key + i, weighed, old[i], a[i]);
}

// ---------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------
// Both kernels: four waves of 64 stationary rows (or keys) in registers, the others 64 (or 32) at a step through a ring
// of kRing LDS tiles that are loaded past the registers, kRing - 1 steps ahead.  A tile's rows are stored as they are,
// but for their 16-byte words, which are permuted by the row's number so that 16 rows' same word lies on distinct
// banks.  Operand dims: lane l's 16-byte word of codes holds the dims of two products.
//
// What bounds them is that exponentials, sums and conversions fill the vector unit as long as products do the
// matrix cores (a score of 64 lanes: fma 4 cycles, exponential 8, sum 4, conversion 2 to 4; its products 16 of
// 128 dims), and that a wave does them in turn.  So there are as many workgroups on a CU as registers allow, 3 of
// 128 dims and 2 of 256, none of which waits for another's barrier (one of eight waves instead: 66 and 78 us for 164
// million scores of 128 dims, now 55 and 65; 90 and 107 for 138 million of 256 dims, now 84 and 93).  Adding up the
// scores before beside the next ones' products, written into one stream of instructions, needs registers
// for both: 60 us, and 87.
//
// Work: the steps of all stationary tiles, KV heads and slots form one line that is cut into equal parts, a
// workgroup's each, so ragged and causal lengths balance by themselves.  A tile that lies in one part is finished there;
// one that is cut leaves records that a second kernel joins.
constexpr int kRing = 4, kWaves = 4, kTile = 64 * kWaves, kThreads = 64 * kWaves;
constexpr int kWeighLead = 3;   // steps that a tile costs beside its own

// The tiles of a slot's rows and their steps over keys: v below n_sink are key steps v, then w0 on.
struct RowTiles {
  const WeighArgs& p;
  struct Tile {
    int steps, n_sink, w0, end;
    __device__ __forceinline__ int first(int v) const { return (v < n_sink ? v : v - n_sink + w0) * 64; }
  };
  __device__ __forceinline__ int count(const Slot& x) const { return (x.n * p.gqa + kTile - 1) / kTile; }
  __device__ __forceinline__ Tile tile(const Slot& x, int i) const {
    const int lo = x.pos0 + token_of(p, i * kTile), hi = x.pos0 + token_of(p, min(x.n * p.gqa, (i + 1) * kTile) - 1);
    Tile t;
    t.end = min(hi + 1, p.max_ctx);
    t.w0 = p.window > 0 ? max(0, lo - p.window + 1) / 64 : 0;
    t.n_sink = p.window > 0 ? min((p.sink + 63) / 64, t.w0) : 0;
    // (the window may lie past max_ctx: then the sinks alone)
    t.steps = t.n_sink + max(0, (t.end + 63) / 64 - t.w0);
    return t;
  }
};

// The tiles of a slot's keys and their steps over the rows r_lo .. r_hi-1 that see a key of the tile.
template <int STEP>
struct KeyTiles {
  const WeighArgs& p;
  struct Tile {
    int steps, r_lo, r_hi;
  };
  __device__ __forceinline__ int count(const Slot& x) const { return x.n > 0 ? (x.end + kTile - 1) / kTile : 0; }
  __device__ __forceinline__ Tile tile(const Slot& x, int i) const {
    const int k0 = i * kTile, k1 = min(k0 + kTile, x.end) - 1;
    long hi = (long)x.n * p.gqa;
    if (p.window > 0 && k0 >= p.sink) hi = min(hi, max(0l, (long)k1 + p.window - x.pos0) * p.gqa);
    Tile t;
    t.r_hi = (int)hi;
    t.r_lo = (int)min((long)max(0, k0 - x.pos0) * p.gqa / STEP * STEP, hi);
    t.steps = (t.r_hi - t.r_lo + STEP - 1) / STEP;
    return t;
  }
};

struct LineLds {
  int scan[kWaves], upto[kThreads], found[3];
};

// The line of one head, walked kThreads slots at a time: their tiles are counted, then taken up by as many threads as
// there are.
template <class Tiles>
struct TileLine {
  const WeighArgs& p;
  const Tiles& tiles;
  LineLds& lds;
  int s, i, mine, inc;         // this thread's tile of the last step, its units and the line's up to its end
  bool one = true;             // the line is one step: what the registers hold

  template <class F>
  __device__ __forceinline__ void walk(F&& done) {   // done(units so far): whether to stop
    int base = 0;
    for (int s0 = 0; s0 < p.n_slots; s0 += kThreads) {
      const int mine_s = s0 + (int)threadIdx.x;
      int n;
      const int count = mine_s < p.n_slots ? tiles.count(slot_of(p, mine_s)) : 0;
      lds.upto[threadIdx.x] = block_scan<kThreads>(count, lds.scan, n);
      __syncthreads();
      n = __builtin_amdgcn_readfirstlane(n);
      for (int x0 = 0; x0 < n; x0 += kThreads) {
        const int x = x0 + (int)threadIdx.x;
        mine = 0;
        if (x < n) {
          int lo = 0, hi = kThreads - 1;   // the first slot whose tiles end past x
          for (int w = kThreads / 2; w; w >>= 1) {
            const int mid = (lo + hi) / 2;
            if (lds.upto[mid] > x) hi = mid; else lo = mid + 1;
          }
          s = s0 + lo;
          i = x - (lo ? lds.upto[lo - 1] : 0);
          mine = kWeighLead + tiles.tile(slot_of(p, s), i).steps;
        }
        int sum;
        inc = add_units(base, block_scan<kThreads>(mine, lds.scan, sum));
        base = __builtin_amdgcn_readfirstlane(add_units(base, sum));
        if (done(base)) return;
      }
      __syncthreads();   // (upto is written again)
    }
  }
  // units of the line (0: too many, which starts in order cannot make)
  __device__ __forceinline__ int units() {
    int total = 0, steps = 0;
    walk([&](int so_far) {
      total = so_far;
      steps++;
      return false;
    });
    one = steps <= 1;
    return total < kLineMax && (long)total * p.num_kv < (1l << 31) ? total : 0;
  }
  // the tile that holds unit u of the line (u < its length), and the unit in it
  __device__ __forceinline__ void find(int u, int& slot, int& tile, int& at) {
    auto look = [&](int so_far) {
      if (u >= inc - mine && u < inc) {
        lds.found[0] = s;
        lds.found[1] = i;
        lds.found[2] = u - (inc - mine);
      }
      return so_far > u;
    };
    if (one) look(0); else walk(look);
    __syncthreads();
    slot = __builtin_amdgcn_readfirstlane(lds.found[0]);
    tile = __builtin_amdgcn_readfirstlane(lds.found[1]);
    at = __builtin_amdgcn_readfirstlane(lds.found[2]);
  }
};

// This workgroup's part: body(slot, its number, head, tile's number, tile, steps v0 .. v1-1, whether these are all,
// record) for each tile that it has steps of.  Where a part begins is noted for the second kernel: {slot (-1: no part),
// tile, head, step}.
template <class Tiles, class Body>
__device__ __forceinline__ void run_part(const WeighArgs& p, const Tiles& tiles, LineLds& lds, Body&& body) {
  TileLine<Tiles> line{p, tiles, lds};
  const int tid = threadIdx.x, lane = tid & 63;
  const int total = __builtin_amdgcn_readfirstlane(line.units());
  const Parts parts(__builtin_amdgcn_readfirstlane(total * p.num_kv), p.groups);
  // neighbouring parts (the same head's keys and rows) on one XCD, whose L2 holds them
  const int grp = (int)(blockIdx.x % 8) * (p.groups / 8) + (int)blockIdx.x / 8;
  int4* cuts = reinterpret_cast<int4*>(p.cuts);
  if (grp >= parts.n) {
    if (tid == 0) cuts[grp] = make_int4(-1, 0, 0, 0);
    return;
  }
  int u = parts.begin(grp);
  const int u_end = parts.begin(grp + 1);
  int h = u / total, s, i, at;
  line.find(u - h * total, s, i, at);
  bool first = true;
  while (u < u_end) {
    const Slot sl = slot_of(p, s);
    if (i >= tiles.count(sl)) {   // on to the next slot with tiles, 64 at a time
      uint64_t any = 0;
      int t = s + 1;
      while (true) {
        if (t >= p.n_slots) {
          t = 0;
          if (++h >= p.num_kv) return;   // (starts or positions that change under the call)
        }
        any = __builtin_amdgcn_ballot_w64(t + lane < p.n_slots && tiles.count(slot_of(p, min(t + lane, p.n_slots - 1))) > 0);
        if (any) break;
        t += 64;
      }
      s = t + (int)__builtin_ctzll(any);
      i = 0;
      continue;
    }
    const auto t = tiles.tile(sl, i);
    const int n_u = min(kWeighLead + t.steps - at, u_end - u);
    if (n_u <= 0) return;
    const int v0 = max(at - kWeighLead, 0), v1 = at + n_u - kWeighLead;   // (v1 <= v0: the next part's, or no step at all)
    if (first && tid == 0) cuts[grp] = make_int4(s, i, h, v0);
    if (v1 > v0 || (t.steps == 0 && v1 == 0)) body(sl, s, h, i, t, v0, v1, v0 == 0 && v1 == t.steps, 2 * grp + (first ? 0 : 1));
    u += n_u;
    first = false;
    at = 0;
    i++;
  }
}

// The tile that part g continues, if it was begun in part g - 1: its records are `first`, then 2 g, 2 (g + 1) .. of the
// n - 1 parts that continue it.
constexpr int kJoin = 4;   // threads a row or key, each every fourth record (one: 13 us where a tile has 100, now 8)
struct CutTile {
  int s, i, h, first, n, g;
  __device__ __forceinline__ long record(int x) const { return x == 0 ? first : 2 * (g + x - 1); }
};
__device__ __forceinline__ bool cut_tile(const WeighArgs& p, CutTile& c) {
  __shared__ int4 cuts[kWeighGroups];
  for (int x = threadIdx.x; x < p.groups; x += kJoin * kThreads) cuts[x] = reinterpret_cast<const int4*>(p.cuts)[x];
  __syncthreads();
  const int g = (int)blockIdx.x + 1;
  const int4 here = cuts[g], before = cuts[g - 1];
  auto same = [&](const int4& a) { return a.x == here.x && a.y == here.y && a.z == here.z; };
  if (here.x < 0 || here.w <= 0 || (same(before) && before.w > 0)) return false;
  c = {here.x, here.y, here.z, 2 * (g - 1) + (same(before) ? 0 : 1), 2, g};
  // (the parts that continue it are neighbours: to the first of another tile, 64 at a time)
  const int lane = (int)threadIdx.x & 63;
  for (int x = g + 1;; x += 64) {
    const uint64_t other = __builtin_amdgcn_ballot_w64(x + lane >= p.groups || !same(cuts[min(x + lane, p.groups - 1)]));
    c.n = x - g + 1 + (other ? (int)__builtin_ctzll(other) : 64);
    if (other) break;
  }
  return true;
}

// Reads of LDS beside loads into LDS.  (For a read that it knows of the compiler waits until every load into LDS has
// ended, those of later steps too.)
__device__ __forceinline__ uint32_t lds_at(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
__device__ __forceinline__ void lds_read(u4_t (&x)[4], uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %6\n\tds_read_b128 %3, %7\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]) : "v"(a), "v"(b), "v"(c), "v"(d) : "memory");
}
// (four rows' numbers of each eight from a on, and those 256 bytes past them)
__device__ __forceinline__ void lds_read(f4_t (&x)[4], f4_t (&y)[4], uint32_t a) {
  asm volatile("ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:32\n\tds_read_b128 %2, %8 offset:64\n\t"
               "ds_read_b128 %3, %8 offset:96\n\tds_read_b128 %4, %8 offset:256\n\tds_read_b128 %5, %8 offset:288\n\t"
               "ds_read_b128 %6, %8 offset:320\n\tds_read_b128 %7, %8 offset:352\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(y[0]), "=&v"(y[1]), "=&v"(y[2]), "=&v"(y[3])
               : "v"(a) : "memory");
}

// Scores to be added: of 32 keys from k on, the pages of each 16, whether every row sees all.
struct Half {
  int k, pg0, pg1;
  bool whole;
};

// Statistics of rows.  Codes are converted by each wave as it reads them.  The pages of kLook steps and their exponents
// are looked up at a time.  The reference of a row's sum need not be its maximum: it stands until the sum grows past
// 2^32 (what is lost then lies below 2^-94 of it), which saves the maximum of each score (66 -> 61 us).
template <int HD>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(HD == 128 ? 3 : 2, HD == 128 ? 3 : 2))) void weigh_stats_kernel(WeighArgs p) {
  constexpr int NB = HD / 32, TB = 64 * HD, LOADS = TB / 1024 / kWaves, RL = 1024 / HD, kLook = 128;
  __shared__ __align__(256) uint8_t ring[kRing][TB];
  // of every 16 keys: their first row's offset in the pool (absent: 0), their page (-1: none) and its exponent's power
  __shared__ __align__(16) long at_lds[kLook * 4];
  __shared__ __align__(16) int page_lds[kLook * 4];
  __shared__ __align__(16) float exp_lds[kLook * 4];
  __shared__ LineLds lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hh = lane >> 5;
  const uint32_t key_bytes = (uint32_t)p.num_kv * HD;
  // A wave loads 16 keys of a step, RL at a time: this lane's word of the first, and key
  static_assert(LOADS * RL == 16);
  const uint32_t my_word = 16 * ((lane % (HD / 16)) ^ (lane / (HD / 16))), my_key = lane / (HD / 16) * key_bytes;
  const uint32_t page_at = lds_at(page_lds), exp_at = lds_at(exp_lds) + 4 * (c >> 4), at_at = lds_at(at_lds);
  const uint32_t ring_at = lds_at(ring) + c * HD + ((hh ^ (c & (HD / 16 - 1))) * 16);   // key c's word of the first products
  run_part(p, RowTiles{p}, lds, [&](const Slot& sl, int s, int h, int i, const RowTiles::Tile& t, int v0, int v1, bool all, int rec)
                                    __attribute__((always_inline)) {
    const int rows = sl.n * p.gqa, row_w = i * kTile + wave * 64;
    h8_t qf[2][NB][2];
    const bool live = row_w < rows;
    const int pos_lo = sl.pos0 + token_of(p, min(row_w, rows - 1)), pos_hi = sl.pos0 + token_of(p, min(row_w + 64, rows) - 1);
    Stat st[2] = {{-INFINITY, 0.f}, {-INFINITY, 0.f}};
    // Sums by the reference that stands ..
    auto sums_of = [&](const f16x_t (&x)[2], float (&l)[2]) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < 2; b++) {
        l[b] = st[b].l;
#pragma unroll
        for (int i = 0; i < 16; i++) l[b] += __builtin_amdgcn_exp2f(__builtin_fmaf(x[b][i], p.scale_log2, -st[b].m));
      }
    };
    // .. by the maximum (lane c's row, keys 8 (i / 4) + 4 hh + i % 4) ..
    auto exact = [&](const f16x_t& x, Stat& st, auto&& seen) __attribute__((always_inline)) {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; i++) top = fmaxf(top, seen(i) ? x[i] * p.scale_log2 : -INFINITY);
      const float mn = fmaxf(st.m, top), ref = mn == -INFINITY ? 0.f : mn;
      float l = st.l * __builtin_amdgcn_exp2f(st.m - ref);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], p.scale_log2, -ref));
        l += seen(i) ? w : 0.f;
      }
      st = {mn, l};
    };
    // .. where that makes large numbers (or there is none yet).
    auto take = [&](const f16x_t (&x)[2], const float (&l)[2]) __attribute__((always_inline)) {
      if (__builtin_amdgcn_ballot_w64(!(l[0] < 0x1p32f && l[1] < 0x1p32f))) {
#pragma unroll
        for (int b = 0; b < 2; b++) exact(x[b], st[b], [](int) { return true; });
      } else {
        st[0].l = l[0];
        st[1].l = l[1];
      }
    };
    auto add = [&](const f16x_t (&x)[2], const Half& had) __attribute__((always_inline)) {
      if (had.whole) {
        float l[2];
        sums_of(x, l);
        take(x, l);
      } else {
#pragma unroll
        for (int b = 0; b < 2; b++) {
          // the row sees the keys above `from` (or below the sinks) and up to `upto`, and none of an absent page: a bound
          // past every key of it
          const int pos = sl.pos0 + token_of(p, min(row_w + 32 * b + c, rows - 1));
          const int from = p.window > 0 ? pos - p.window : -1, upto = min(pos, t.end - 1);
          const int k = had.k + 4 * hh, hi = upto - k, lo = from - k, sink = p.sink - k;
          const int hi0 = had.pg0 >= 0 ? hi : -64, hi1 = had.pg1 >= 0 ? hi : -64;
          exact(x[b], st[b], [&](int i) {
            const int d = 8 * (i >> 2) + (i & 3);
            return (d <= (i < 8 ? hi0 : hi1)) & ((d > lo) | (d < sink));
          });
        }
      }
    };
    for (int va = v0; va < v1; va += kLook) {
      const int vb = min(va + kLook, v1);
      __syncthreads();   // (the ring and the pages are written again)
      for (int x = tid; x < 4 * (vb - va); x += kThreads) {
        const int key = t.first(va + (x >> 2)) + 16 * (x & 3);
        const BlockAt y = block_at(p, key);
        const int pg = key < t.end ? page_of(p, p.tables + (long)s * p.max_blocks, y.b) : -1;
        at_lds[x] = pg < 0 ? 0 : ((long)pg * p.block_tokens + y.row) * key_bytes;
        page_lds[x] = pg;
        exp_lds[x] = pow2f(p.k_exp[(long)max(pg, 0) * p.num_kv + h]);
      }
      __syncthreads();
      // the wave's part of a step: LOADS times RL keys (past the last step it is loaded again, so that as many loads
      // are under way as are counted)
      auto load = [&](int buf, long at) __attribute__((always_inline)) {
        uint32_t word = my_word, key = my_key;
        asm volatile("" : "+v"(word), "+v"(key));   // (no LOADS offsets held in registers)
#pragma unroll
        for (int j = 0; j < LOADS; j++) {
          const uint8_t* src = p.k_pool + h * HD + at + (word ^ (j * RL * 16 & (HD - 1))) + (key + j * RL * key_bytes);
          __builtin_amdgcn_global_load_lds((glb_void*)src, (lds_void*)(ring[buf] + (wave * LOADS + j) * 1024), 16, 0, 0);
        }
      };
      auto entry = [&](int v) { return 4 * (min(v, vb - 1) - va) + wave; };
      long at[kRing - 1];
#pragma unroll
      for (int j = 0; j < kRing - 1; j++) at[j] = at_lds[entry(va + j)];
#pragma unroll
      for (int j = 0; j < kRing - 1; j++) load(j, at[j]);
      if (va == v0) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const uint16_t* src = p.q + row_at(p, sl, h, min(row_w + 32 * b + c, rows - 1)) * HD + 16 * hh;
#pragma unroll
          for (int j = 0; j < NB; j++)
#pragma unroll
            for (int x = 0; x < 2; x++) qf[b][j][x] = *reinterpret_cast<const h8_t*>(src + 32 * j + 8 * x);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (from here on only steps are under way)
      }
      for (int v = va; v < vb; v++) {
        const int buf = (v - va) % kRing;
        // this step has landed, for every wave, and every wave has read the one before
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kRing - 2) * LOADS) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        u4_t pages;
        f2_t pow;
        u2_t from;
        asm volatile("ds_read_b128 %0, %3\n\tds_read2_b32 %1, %4 offset1:2\n\tds_read_b64 %2, %5\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(pages), "=&v"(pow), "=&v"(from)
                     : "v"(page_at + 16 * (v - va)), "v"(exp_at + 16 * (v - va)), "v"(at_at + 8 * entry(v + kRing - 1))
                     : "memory");
        const long next = (long)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)from[1]) << 32 |
                                 (uint32_t)__builtin_amdgcn_readfirstlane((int)from[0]));
        load((v - va + kRing - 1) % kRing, next);
        const int k0 = t.first(v);
#pragma unroll
        for (int half = 0; half < 2; half++) {
          const int kh = k0 + 32 * half;
          if (!live || kh > pos_hi || kh >= t.end) continue;
          f16x_t acc[2] = {f16x_t{}, f16x_t{}};
          const uint32_t src = ring_at + buf * TB + 32 * half * HD;
#pragma unroll
          for (int j4 = 0; j4 < NB; j4 += 4) {
            u4_t w[4];
            lds_read(w, src ^ (32 * j4), src ^ (32 * j4 + 32), src ^ (32 * j4 + 64), src ^ (32 * j4 + 96));
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
              for (int x = 0; x < 2; x++) {
                const h8_t a = cvt8(w[j][2 * x], w[j][2 * x + 1], pow[half]);
#pragma unroll
                for (int b = 0; b < 2; b++) acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qf[b][j4 + j][x], acc[b], 0, 0, 0);
              }
            __builtin_amdgcn_s_setprio(0);
          }
          const int pg0 = __builtin_amdgcn_readfirstlane((int)pages[2 * half]), pg1 = __builtin_amdgcn_readfirstlane((int)pages[2 * half + 1]);
          const bool whole = pg0 >= 0 && pg1 >= 0 && kh + 31 <= pos_lo && kh + 32 <= t.end &&
                             (p.window <= 0 || kh > pos_hi - p.window || kh + 32 <= p.sink);
          add(acc, Half{kh, pg0, pg1, whole});
        }
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (no load into the ring is under way past here)
    }
#pragma unroll
    for (int b = 0; b < 2; b++) {
      const Stat x = join(st[b], Stat{other32(st[b].m, lane), other32(st[b].l, lane)});
      const int r = wave * 64 + 32 * b + c, row = i * kTile + r;
      if (hh == 0 && row < rows) {
        if (all) put_stat(p, row_at(p, sl, h, row), x);
        else *reinterpret_cast<f2_t*>(p.rec + ((long)rec * kTile + r) * 2) = f2_t{x.m, x.l};
      }
    }
  });
}

__global__ __launch_bounds__(kJoin * kThreads) void weigh_stats_join_kernel(WeighArgs p) {
  __shared__ f2_t part[kJoin][kThreads];
  CutTile c;
  if (!cut_tile(p, c)) return;
  const int t = (int)threadIdx.x % kThreads, w = (int)threadIdx.x / kThreads;
  Stat x{-INFINITY, 0.f};
#pragma unroll 4
  for (int j = w; j < c.n; j += kJoin) {
    const f2_t v = *reinterpret_cast<const f2_t*>(p.rec + (c.record(j) * kTile + t) * 2);
    x = join(x, Stat{v[0], v[1]});
  }
  part[w][t] = f2_t{x.m, x.l};
  __syncthreads();
  if (w > 0) return;
#pragma unroll
  for (int i = 1; i < kJoin; i++) x = join(x, Stat{part[i][t][0], part[i][t][1]});
  const Slot sl = slot_of(p, c.s);
  const int row = c.i * kTile + t;
  if (row < sl.n * p.gqa) put_stat(p, row_at(p, sl, c.h, row), x);
}

// Sums of keys.  A step brings its rows' statistics along.  (The ring leaves room for as many workgroups as registers do:
// 128 dims by steps of 32 rows and four of them 70 us, 66 by 64 and three.)
template <int HD>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(HD == 128 ? 3 : 2, HD == 128 ? 3 : 2))) void weigh_sums_kernel(WeighArgs p) {
  constexpr int STEP = HD == 128 ? 64 : 32, RING = HD == 128 ? 3 : 4, NB = HD / 32, RB = HD * 2, TB = STEP * RB, LOADS = TB / 1024 / kWaves, WORDS = RB / 16;
  __shared__ __align__(512) uint8_t ring[RING][TB];
  __shared__ __align__(16) float stat_lds[RING][3][64];   // m, 1 / l, and what the other waves load beside them
  __shared__ LineLds lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hh = lane >> 5;
  const uint32_t key_bytes = (uint32_t)p.num_kv * HD;
  // row c's word of the first product
  const uint32_t ring_at = lds_at(ring) + c * RB + (((2 * hh) ^ (c & 15)) * 16), stat_at = lds_at(stat_lds) + 16 * hh;
  // Bytes of this lane's words (and of a row's number) past the first token's rows of a step that begins with its row
  // `rem` and has `left` rows
  auto places = [&](int rem, int left, uint32_t (&at)[LOADS + 1]) {
    auto place = [&](int x) {
      const int y = rem + min(x, left - 1);
      return (uint32_t)(token_of(p, y) * (p.num_q - p.gqa) + y);
    };
#pragma unroll
    for (int j = 0; j < LOADS; j++) {
      const int x = (wave * LOADS + j) * (1024 / RB) + lane / WORDS;
      at[j] = place(x) * RB + 16 * ((lane % WORDS) ^ (x & 15));
    }
    at[LOADS] = 4 * place(lane);
  };
  uint32_t mine[LOADS + 1];   // (the same in most steps, all where groups divide them)
  places(0, 64, mine);
  run_part(p, KeyTiles<STEP>{p}, lds, [&](const Slot& sl, int s, int h, int i, const typename KeyTiles<STEP>::Tile& t, int v0, int v1, bool all, int rec)
                                    __attribute__((always_inline)) {
    const int rows = sl.n * p.gqa, key_w = i * kTile + wave * 64;
    const int32_t* table = p.tables + (long)s * p.max_blocks;
    float sum[2] = {0.f, 0.f};
    if (v0 < v1) {
      // the wave's part of a step, and a number for each of its rows: every wave as many loads
      auto load = [&](int v, int buf) {
        const int r0 = t.r_lo + STEP * min(v, v1 - 1), tok = token_of(p, r0), rem = r0 - tok * p.gqa;
        const long row = (long)(sl.t0 + tok) * p.num_q + h * p.gqa;
        uint32_t at[LOADS + 1];
        if (rem != 0 || rows - r0 < 64) {
          places(rem, rows - r0, at);
        } else {
#pragma unroll
          for (int j = 0; j <= LOADS; j++) at[j] = mine[j];
        }
#pragma unroll
        for (int j = 0; j < LOADS; j++)
          __builtin_amdgcn_global_load_lds((glb_void*)((const uint8_t*)(p.q + row * HD) + at[j]),
                                           (lds_void*)(ring[buf] + (wave * LOADS + j) * 1024), 16, 0, 0);
        const float* src = (wave == 1 ? p.stat_il : p.stat_m) + row;
        __builtin_amdgcn_global_load_lds((glb_void*)((const uint8_t*)src + at[LOADS]), (lds_void*)stat_lds[buf][min(wave, 2)], 4, 0, 0);
      };
      __syncthreads();   // (the ring is written again)
#pragma unroll
      for (int j = 0; j < RING - 1; j++) load(v0 + j, j);
      h8_t kf[2][NB][2];
      int from[2], upto[2];   // rows that see lane c's keys: from .. upto-1
#pragma unroll
      for (int b = 0; b < 2; b++) {
        const int key = min(key_w + 32 * b + c, sl.end - 1);
        from[b] = (int)min((long)max(0, key - sl.pos0) * p.gqa, (long)t.r_hi);
        upto[b] = p.window > 0 && key >= p.sink ? (int)min(max(0l, (long)key + p.window - sl.pos0) * p.gqa, (long)t.r_hi) : t.r_hi;
        const BlockAt x = block_at(p, key);
        const long page = max(page_of(p, table, x.b), 0);
        const uint8_t* src = p.k_pool + (page * p.block_tokens + x.row) * key_bytes + h * HD + 16 * hh;
        const float f = pow2f(p.k_exp[page * p.num_kv + h]);
#pragma unroll
        for (int j = 0; j < NB; j++) {
          const u4_t w = *reinterpret_cast<const u4_t*>(src + 32 * j);
          kf[b][j][0] = cvt8(w[0], w[1], f);
          kf[b][j][1] = cvt8(w[2], w[3], f);
        }
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (from here on only steps are under way)
      for (int v = v0; v < v1; v++) {
        const int buf = (v - v0) % RING, r0 = t.r_lo + STEP * v;
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((RING - 2) * (LOADS + 1)) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        load(v + RING - 1, (v - v0 + RING - 1) % RING);
#pragma unroll
        for (int half = 0; half < STEP / 32; half++) {
          const int rh = r0 + 32 * half;
          if (rh >= t.r_hi) continue;
          const int pos_lo = sl.pos0 + token_of(p, rh), pos_hi = sl.pos0 + token_of(p, min(rh + 32, rows) - 1);
          if (key_w > pos_hi) continue;
          f16x_t acc[2] = {f16x_t{}, f16x_t{}};
          const uint32_t src = ring_at + buf * TB + 32 * half * RB;
#pragma unroll
          for (int j = 0; j < NB; j += 2) {
            u4_t a[4];
            lds_read(a, src ^ (64 * j), src ^ (64 * j + 16), src ^ (64 * j + 64), src ^ (64 * j + 80));
#pragma unroll
            for (int x = 0; x < 4; x++)
#pragma unroll
              for (int b = 0; b < 2; b++)
                acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, a[x]), kf[b][j + x / 2][x % 2], acc[b], 0, 0, 0);
          }
          f4_t mr[4], il[4];
          lds_read(mr, il, stat_at + buf * (4 * 3 * 64) + 128 * half);
          const bool whole = rh + 32 <= t.r_hi && key_w + 63 <= pos_lo &&
                             (p.window <= 0 || key_w > pos_hi - p.window || key_w + 64 <= p.sink);
          // lane c's key, rows 8 (x / 4) + 4 hh + x % 4
#pragma unroll
          for (int x4 = 0; x4 < 4; x4++) {
            const int at = 32 * half + 8 * x4 + 4 * hh;
            float w[2][4];
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
              for (int x = 0; x < 4; x++) w[b][x] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[b][4 * x4 + x], p.scale_log2, -mr[x4][x]));
            if (whole) {
#pragma unroll
              for (int b = 0; b < 2; b++)
#pragma unroll
                for (int x = 0; x < 4; x++) sum[b] = __builtin_fmaf(w[b][x], il[x4][x], sum[b]);
            } else {
#pragma unroll
              for (int b = 0; b < 2; b++) {
                const int lo = from[b] - r0 - at, hi = upto[b] - r0 - at;
#pragma unroll
                for (int x = 0; x < 4; x++) sum[b] += x >= lo && x < hi ? w[b][x] * il[x4][x] : 0.f;
              }
            }
          }
        }
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (no load into the ring is under way past here)
    }
    // (both halves of the lanes have the same keys, other rows)
#pragma unroll
    for (int b = 0; b < 2; b++) {
      const float a = sum[b] + other32(sum[b], lane);
      const int x = wave * 64 + 32 * b + c, key = i * kTile + x;
      if (hh == 0 && key < sl.end) {
        if (all) put_weight(p, table, h, key, p.weighed ? p.weighed[s] : sl.pos0, a);
        else p.sums[(long)rec * kTile + x] = a;
      }
    }
  });
}

__global__ __launch_bounds__(kJoin * kThreads) void weigh_sums_join_kernel(WeighArgs p) {
  __shared__ float part[kJoin][kThreads];
  CutTile c;
  if (!cut_tile(p, c)) return;
  const int t = (int)threadIdx.x % kThreads, w = (int)threadIdx.x / kThreads;
  float a = 0.f;
#pragma unroll 4
  for (int j = w; j < c.n; j += kJoin) a += p.sums[c.record(j) * kTile + t];
  part[w][t] = a;
  __syncthreads();
  if (w > 0) return;
#pragma unroll
  for (int i = 1; i < kJoin; i++) a += part[i][t];
  const Slot sl = slot_of(p, c.s);
  const int key = c.i * kTile + t;
  if (key < sl.end) put_weight(p, p.tables + (long)c.s * p.max_blocks, c.h, key, p.weighed ? p.weighed[c.s] : sl.pos0, a);
}

WeighPlan weigh_plan(int num_q, int num_kv, int n_slots, long rows, int max_tok, int max_ctx) {
  const int gqa = num_q / num_kv;
  WeighPlan x{};
  x.pitch = (max_ctx + 31l) / 32 * 32;
  // slots of up to 64 rows store their scores, as many slots at a time as kWeighScores bytes hold
  const double token = (double)num_q * x.pitch * 4;
  x.few_tok = (int)std::min((double)std::min(64 / gqa, max_tok), kWeighScores / token);
  x.many = max_tok > x.few_tok;
  // (beside many rows only where the numbers say that slots differ: three launches more, 13 us)
  if (x.many && 2 * rows >= (long)n_slots * max_tok) x.few_tok = 0;
  if (x.few_tok > 0) x.few_slots = (int)std::min((double)n_slots, kWeighScores / (token * x.few_tok));
  // of these, workgroups enough for the CUs also where the slots are few, of 128 keys at least
  const long target = std::min(256l, std::max(16l, 8192l / std::max(1l, (long)x.few_slots * num_kv)));
  x.few_keys = (int)(128 * ((max_ctx + 128 * target - 1) / (128 * target)));
  x.few_chunks = (max_ctx + x.few_keys - 1) / x.few_keys;
  const size_t few_rows = (size_t)x.few_slots * x.few_tok * num_q, all = (size_t)rows * num_q;
  x.stat_rows = std::max(few_rows, x.many ? all : 0);
  x.rec_bytes = std::max(few_rows * x.few_chunks * 8, kWeighRec);
  x.sum_bytes = std::max(few_rows * x.pitch * 4, kWeighRec / 2);
  return x;
}

hipError_t launch_weigh(WeighArgs a, const WeighPlan& x, int head_dim, hipStream_t stream) {
  const dim3 block(256);
  int slots = 0;
  auto launch = [&](auto kernel, long per) {
    a.per = (int)per;
    a.heads = slots * a.num_kv;
    hipLaunchKernelGGL(kernel, grid_xy(per * a.heads), block, 0, stream, a);
  };
  if (x.few_tok > 0) for (a.slot0 = 0; a.slot0 < a.n_slots; a.slot0 += x.few_slots) {
    slots = std::min(a.n_slots - a.slot0, x.few_slots);
    a.local_tok = x.few_tok;
    a.from_tok = 1;
    a.to_tok = x.few_tok;
    a.chunk_keys = x.few_keys;
    a.chunks = x.few_chunks;
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
    if (rows * a.chunks <= 2048) {
      launch(weigh_few_kernel<false>, (a.max_ctx + 1023l) / 1024);
    } else {
      launch(weigh_merge_kernel, (rows + 15) / 16);
      launch(weigh_few_kernel<true>, (a.max_ctx + 1023l) / 1024);
    }
  }
  if (x.many) {
    a.slot0 = 0;
    a.local_tok = 0;
    a.from_tok = x.few_tok + 1;
    a.to_tok = 0x7fffffff;
    a.groups = head_dim == 128 ? 768 : 512;
    const dim3 groups(a.groups), wide(kThreads), joins(a.groups - 1), join_wide(kJoin * kThreads);
    if (head_dim == 128) hipLaunchKernelGGL(weigh_stats_kernel<128>, groups, wide, 0, stream, a);
    else hipLaunchKernelGGL(weigh_stats_kernel<256>, groups, wide, 0, stream, a);
    hipLaunchKernelGGL(weigh_stats_join_kernel, joins, join_wide, 0, stream, a);
    if (head_dim == 128) hipLaunchKernelGGL(weigh_sums_kernel<128>, groups, wide, 0, stream, a);
    else hipLaunchKernelGGL(weigh_sums_kernel<256>, groups, wide, 0, stream, a);
    hipLaunchKernelGGL(weigh_sums_join_kernel, joins, join_wide, 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace qkv
