// evict_f8.hip -- eviction from the paged 8-bit cache: of each slot and KV head the keys with the most
// accumulated weight stay, in order, moved to the front of the slot's pages.
//
// First what stays is found: the last and the first rows whatever they weigh, and the largest of the weights between, by
// radix selection on the weights' bits (ties to the lowest row), a workgroup for each (slot, KV head), or one for each
// 4,096 rows of long slots (131,072 rows by one workgroup: 232 us).  Then the rows of both pools and the weights
// are moved in place.
//
// In place, a row may go where another has not been read yet.  Rows only ever move forward (row i of what stays
// comes from row kept[i] >= i), so a chunk of rows may be written once every chunk before it has been read.
// Workgroups take chunks in that order by a counter for each (slot, KV head), read theirs whole into registers, say
// so, and only then wait for those before: nobody waits before having said it, so every wait ends.  (One counter
// for all costs 11 ns a chunk: 106 of 130 us for 9,216 of them.)
//
// Bound by latency where slots are few (one of 131,072 rows to 16,384: the selection's four launches 34 us, the rows' 30,
// of 14 at 4.8 TB/s) and by HBM where they are many (24 slots, 322 MB read and written: 20 and 85 us, 3.8 TB/s; rows of
// 128 to 256 bytes, each with the table's and the list's entries ahead of it).
//
// A page's exponent becomes the largest of those its rows had; codes of the others are requantized by a power of
// two, which rounds only those that become subnormal.
#include <algorithm>

#include "f8_device.h"
#include "qkv_device.h"
#include "qkv_launch.h"

namespace qkv {

namespace {

// Weights in one order: a NaN below all others, both zeros equal.
__device__ __forceinline__ uint32_t order_of(float w) {
  const uint32_t b = __float_as_uint(w + 0.0f);
  return w != w ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct BlockAt {
  int b, row;
};
// (magic = floor(2^32 / block_tokens): the product's high half is the quotient or one less)
__device__ __forceinline__ BlockAt block_at(uint32_t magic, int bt, int r) {
  const uint32_t q = __umulhi((uint32_t)r, magic), x = (uint32_t)r - q * (uint32_t)bt;
  return x >= (uint32_t)bt ? BlockAt{(int)q + 1, (int)(x - (uint32_t)bt)} : BlockAt{(int)q, (int)x};
}

}  // namespace

// What a (slot, KV head) asks for: of its rows the first `first` and last `last` stay, and `need` of the `rows` between.
struct Choice {
  int len, n_new, first, last, need, rows;
  bool alone;     // left alone, but for a page that is missing
};
__device__ __forceinline__ Choice choice_of(const EvictArgs& p, int s) {
  Choice c;
  const int keep = p.keep[s];
  c.len = p.lens[s];
  c.n_new = min(c.len, keep);
  c.alone = c.len < 0 || c.len > p.max_ctx || keep < 0 || c.n_new > p.max_keep ||
            (c.len + (long)p.block_tokens - 1) / p.block_tokens > p.max_blocks;
  c.last = c.alone || keep >= c.len ? 0 : min(keep, p.recent);
  c.first = c.alone || keep >= c.len ? 0 : min(keep - c.last, p.sink);
  c.need = c.alone || keep >= c.len ? 0 : keep - c.first - c.last;
  c.rows = c.alone || keep >= c.len ? 0 : c.len - c.first - c.last;
  return c;
}

// Whether a row of the slot has no page (by 1,024 threads, the same in all)
__device__ __forceinline__ bool page_missing(const EvictArgs& p, const int32_t* table, int len) {
  const int blocks = (int)((len + (long)p.block_tokens - 1) / p.block_tokens);
  bool bad = false;
  for (int b = threadIdx.x; !bad && b < blocks; b += 1024) bad = table[b] < 0 || table[b] >= p.n_pages;
  return __syncthreads_or(bad);
}

// kept of the rows that stay whatever they weigh, and the ends; the workspace of the second launch
__device__ __forceinline__ void begin_chain(const EvictArgs& p, int chain, const Choice& c, bool bad, int32_t* kept) {
  const int tid = threadIdx.x;
  for (int i = tid; i < p.chunks; i += 1024) p.flags[(long)chain * p.chunks + i] = 0;
  if (tid == 0) {
    p.chains[kEvictChain * chain] = 0;
    p.chains[kEvictChain * chain + 1] = bad || c.n_new == c.len ? 0 : c.n_new;
  }
  for (int i = (bad ? 0 : c.n_new) + tid; i < p.max_keep; i += 1024) kept[i] = -1;
  if (bad) return;
  const int same = c.n_new == c.len ? c.len : c.first;
  for (int i = tid; i < same; i += 1024) kept[i] = i;
  for (int i = tid; i < c.last; i += 1024) kept[c.n_new - c.last + i] = c.len - c.last + i;
}

__device__ __forceinline__ uint32_t weight_at(const EvictArgs& p, const int32_t* table, int h, int row) {
  const BlockAt x = block_at(p.bt_magic, p.block_tokens, row);
  return order_of(p.weights[((long)table[x.b] * p.num_kv + h) * p.block_tokens + x.row]);
}

// Of 64 * N counts, held N a lane from above (lane 0 the highest), where `need` are reached: the count's place from
// above and how many are needed of it, to found[0] and [1].
template <int N>
__device__ __forceinline__ void reach(const int (&c)[N], int need, int* found) {
  const int lane = threadIdx.x & 63;
  int n = 0;
#pragma unroll
  for (int i = 0; i < N; i++) n += c[i];
  int up = n;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(up, d);
    if (lane >= d) up += o;
  }
  int above = up - n;
#pragma unroll
  for (int i = 0; i < N; i++) {
    if (above < need && above + c[i] >= need) {
      found[0] = N * lane + i;
      found[1] = need - above;
    }
    above += c[i];
  }
}

// Short slots: 16 waves, each of which looks at a stretch of rows of its own, 64 at a time, in up to 16 steps whose
// weights stay in registers.
__global__ __launch_bounds__(1024) void evict_select_kernel(EvictArgs p) {
  constexpr int STEPS = kEvictHeld / 1024, COPIES = 32;
  // a histogram for every pair of lanes: no two lanes of an access share a bank
  __shared__ int hist[256 * COPIES];
  __shared__ int count[256], gt_s[16], eq_s[16], found[2];
  const int chain = blockIdx.x, s = chain / p.num_kv, h = chain - s * p.num_kv;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t* kept = p.kept + (long)chain * p.max_keep;
  const int32_t* table = p.tables + (long)s * p.max_blocks;
  const Choice c = choice_of(p, s);
  const bool bad = c.alone || page_missing(p, table, c.len);
  begin_chain(p, chain, c, bad, kept);
  int need = c.need;
  if (bad || need == 0) return;
  const int steps = ((c.rows + 15) / 16 + 63) / 64, lo = min(wave * steps * 64, c.rows), hi = min(lo + steps * 64, c.rows);
  // (all pages' loads, then all weights', under way together; past the wave's rows the last one again)
  uint32_t held[STEPS];
  int page[STEPS];
  auto row = [&](int t) { return block_at(p.bt_magic, p.block_tokens, c.first + min(lo + 64 * t + lane, max(hi - 1, 0))); };
#pragma unroll
  for (int t = 0; t < STEPS; t++) page[t] = table[row(t).b];
#pragma unroll
  for (int t = 0; t < STEPS; t++) held[t] = order_of(p.weights[((long)page[t] * p.num_kv + h) * p.block_tokens + row(t).row]);
  // f(row, key, whether it is one) over the wave's rows in order
  auto each = [&](auto&& f) {
#pragma unroll
    for (int t = 0; t < STEPS; t++)
      if (lo + 64 * t < hi) f(lo + 64 * t + lane, held[t], lo + 64 * t + lane < hi);
  };
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256 * COPIES; i += 1024) hist[i] = 0;
    __syncthreads();
    each([&](int, uint32_t k, bool is) {
      if (is && (shift == 24 || k >> (shift + 8) == prefix)) atomicAdd(&hist[(k >> shift & 255u) * COPIES + (lane & 31)], 1);
    });
    __syncthreads();
    {
      int n = 0;
#pragma unroll
      for (int i = 0; i < COPIES / 4; i++) n += hist[(tid >> 2) * COPIES + (tid & 3) + 4 * i];
      n += __shfl_xor(n, 1);
      n += __shfl_xor(n, 2);
      if ((tid & 3) == 0) count[tid >> 2] = n;
    }
    __syncthreads();
    if (wave == 0) {   // the digit, from above, at which `need` are reached
      int n[4];
#pragma unroll
      for (int i = 0; i < 4; i++) n[i] = count[255 - (4 * lane + i)];
      reach(n, need, found);
    }
    __syncthreads();
    prefix = prefix << 8 | (uint32_t)(255 - found[0]);
    need = found[1];
    if (need == count[255 - found[0]]) {   // (all that begin so stay: the digits below do not matter)
      prefix <<= shift;
      need = 0x7fffffff;
      break;
    }
  }
  // rows above the threshold stay, and the first `need` of those at it
  int gt = 0, eq = 0;
  each([&](int, uint32_t k, bool is) {
    gt += __popcll(__builtin_amdgcn_ballot_w64(is && k > prefix));
    eq += __popcll(__builtin_amdgcn_ballot_w64(is && k == prefix));
  });
  if (lane == 0) {
    gt_s[wave] = gt;
    eq_s[wave] = eq;
  }
  __syncthreads();
  int gt_before = 0, eq_before = 0;
  for (int w = 0; w < wave; w++) {
    gt_before += gt_s[w];
    eq_before += eq_s[w];
  }
  int at = c.first + gt_before + min(eq_before, need);
  each([&](int i, uint32_t k, bool is) {
    const uint64_t below = (1ull << lane) - 1, m = __builtin_amdgcn_ballot_w64(is && k == prefix);
    const bool stays = is && (k > prefix || (k == prefix && eq_before + __popcll(m & below) < need));
    const uint64_t n = __builtin_amdgcn_ballot_w64(stays);
    if (stays) kept[at + __popcll(n & below)] = c.first + i;
    at += __popcll(n);
    eq_before += __popcll(m);
  });
}

// Long slots: the rows between in stretches of 4,096, a workgroup each, by four launches: PASS 0 to 2 count digits of 11,
// 11 and 10 bits of the weights (in the prefix that the passes before have found) for each stretch; a launch adds up the
// counts of the one before, of all stretches, for itself.  PASS 3 writes the rows.
template <int PASS>
__global__ __launch_bounds__(1024) void evict_stretch_kernel(EvictArgs p) {
  constexpr int BINS = kEvictBins;
  __shared__ int hist[BINS];
  __shared__ int found[2], gt_s[16], eq_s[16], before_s[16][2];
  const int chain = blockIdx.x / p.stretches, g = blockIdx.x - chain * p.stretches, s = chain / p.num_kv, h = chain - s * p.num_kv;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t* table = p.tables + (long)s * p.max_blocks;
  int32_t* kept = p.kept + (long)chain * p.max_keep;
  const Choice c = choice_of(p, s);
  const int lo = g * kEvictStretch;
  if (PASS == 0) {   // (each stretch looks at all pages: none has to tell another)
    const bool bad = c.alone || page_missing(p, table, c.len);
    if (g == 0) begin_chain(p, chain, c, bad, kept);
    if (bad || c.need == 0 || lo >= c.rows) return;
  } else if (c.need == 0 || lo >= c.rows || p.chains[kEvictChain * chain + 1] == 0) {
    return;
  }
  const int stretches = (c.rows + kEvictStretch - 1) / kEvictStretch, hi = min(lo + kEvictStretch, c.rows);
  // (each wave's rows are neighbours, 64 at a step, as their order asks)
  uint32_t key[4];
#pragma unroll
  for (int i = 0; i < 4; i++) key[i] = weight_at(p, table, h, c.first + min(lo + 256 * wave + 64 * i + lane, hi - 1));
  auto row_of = [&](int i) { return lo + 256 * wave + 64 * i + lane; };

  // ---- the digits found so far: prefix of `bits` bits, and how many are needed of those in it
  uint32_t prefix = 0;
  int need = c.need, bits = 0;
  uint16_t* mine[3];
#pragma unroll
  for (int d = 0; d < 3; d++) mine[d] = p.counts + ((long)(d % 2 * p.n_slots * p.num_kv + chain) * p.stretches) * BINS;
  if constexpr (PASS > 0) {
    // what the launches before have found, but for the last
    if constexpr (PASS > 1) {
      const uint32_t* f = p.found + 4 * chain + 2 * (PASS - 2);
      prefix = f[0];
      need = (int)f[1];
    }
    // its counts, over all stretches: two bins a thread
    const uint32_t* in = reinterpret_cast<const uint32_t*>(mine[PASS - 1]) + tid;
    int a = 0, b = 0;
    for (int x0 = 0; x0 < stretches; x0 += 16) {
      uint32_t v[16];
#pragma unroll
      for (int x = 0; x < 16; x++) v[x] = in[(long)min(x0 + x, stretches - 1) * (BINS / 2)];
#pragma unroll
      for (int x = 0; x < 16; x++)
        if (x0 + x < stretches) {
          a += v[x] & 0xffffu;
          b += v[x] >> 16;
        }
    }
    hist[2 * tid] = a;
    hist[2 * tid + 1] = b;
    __syncthreads();
    if (wave == 0) {
      int n[BINS / 64];
#pragma unroll
      for (int i = 0; i < BINS / 64; i++) n[i] = hist[BINS - 1 - (BINS / 64 * lane + i)];
      reach(n, need, found);
    }
    __syncthreads();
    constexpr int B = PASS == 3 ? 10 : 11;
    prefix = prefix << B | (uint32_t)(BINS - 1 - found[0]);
    need = found[1];
    if (PASS < 3 && g == 0 && tid == 0) {
      p.found[4 * chain + 2 * (PASS - 1)] = prefix;
      p.found[4 * chain + 2 * (PASS - 1) + 1] = (uint32_t)need;
    }
    bits = PASS == 1 ? 11 : PASS == 2 ? 22 : 32;
    __syncthreads();   // (hist is written again)
  }
  if constexpr (PASS < 3) {
    constexpr int LEFT = PASS == 0 ? 32 : PASS == 1 ? 21 : 10, B = PASS == 2 ? 10 : 11;
    hist[tid] = hist[tid + 1024] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (row_of(i) < hi && (PASS == 0 || key[i] >> LEFT == prefix)) atomicAdd(&hist[key[i] >> (LEFT - B) & ((1u << B) - 1)], 1);
    __syncthreads();
    reinterpret_cast<uint32_t*>(mine[PASS] + (long)g * BINS)[tid] = (uint32_t)hist[2 * tid] | (uint32_t)hist[2 * tid + 1] << 16;
    // rows of this stretch above the prefix so far
    int gt = 0;
    if (PASS > 0) {
#pragma unroll
      for (int i = 0; i < 4; i++)
        gt += __popcll(__builtin_amdgcn_ballot_w64(row_of(i) < hi && key[i] >> (32 - bits) > prefix));
      if (lane == 0) gt_s[wave] = gt;
    }
    __syncthreads();
    if (PASS == 2 && tid == 0) {
      int n = 0;
      for (int w = 0; w < 16; w++) n += gt_s[w];
      p.above[chain * p.stretches + g] = n;
    }
    return;
  }
  // ---- rows above the threshold, and at it, in the stretches before: their counts above the 22-bit prefix, and
  // inside it by the last digit's
  if constexpr (PASS == 3) {
    const int digit = (int)(prefix & 1023u);
    int gt = 0, eq = 0;
    for (int x = wave; x < g; x += 16) {
      const uint16_t* n = mine[2] + (long)x * BINS;
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = reinterpret_cast<const uint32_t*>(n)[64 * i + lane];
      gt += lane == 0 ? p.above[chain * p.stretches + x] : 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int b = 2 * (64 * i + lane), lo_n = (int)(v[i] & 0xffffu), hi_n = (int)(v[i] >> 16);
        gt += (b > digit ? lo_n : 0) + (b + 1 > digit ? hi_n : 0);
        eq += (b == digit ? lo_n : 0) + (b + 1 == digit ? hi_n : 0);
      }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      gt += __shfl_xor(gt, d);
      eq += __shfl_xor(eq, d);
    }
    int gt_w = 0, eq_w = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const bool is = row_of(i) < hi;
      gt_w += __popcll(__builtin_amdgcn_ballot_w64(is && key[i] > prefix));
      eq_w += __popcll(__builtin_amdgcn_ballot_w64(is && key[i] == prefix));
    }
    if (lane == 0) {
      before_s[wave][0] = gt;
      before_s[wave][1] = eq;
      gt_s[wave] = gt_w;
      eq_s[wave] = eq_w;
    }
    __syncthreads();
    int gt_before = 0, eq_before = 0;
    for (int w = 0; w < 16; w++) {
      gt_before += before_s[w][0] + (w < wave ? gt_s[w] : 0);
      eq_before += before_s[w][1] + (w < wave ? eq_s[w] : 0);
    }
    int at = c.first + gt_before + min(eq_before, need);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const bool is = row_of(i) < hi;
      const uint64_t below = (1ull << lane) - 1, m = __builtin_amdgcn_ballot_w64(is && key[i] == prefix);
      const bool stays = is && (key[i] > prefix || (key[i] == prefix && eq_before + __popcll(m & below) < need));
      const uint64_t n = __builtin_amdgcn_ballot_w64(stays);
      if (stays) kept[at + __popcll(n & below)] = c.first + row_of(i);
      at += __popcll(n);
      eq_before += __popcll(m);
    }
  }
}

// A chunk of 16384 / HD rows of a (slot, KV head): 64 bytes a thread of each pool.
template <int HD>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs p) {
  constexpr int ROWS = kEvictBytes / HD, LPR = HD / 16, PER = 256 / LPR, N = ROWS / PER;
  __shared__ int ticket, exps[2][ROWS];
  const int tid = threadIdx.x;
  const uint32_t wg = blockIdx.x, chain = wg % (uint32_t)(p.n_slots * p.num_kv);
  const int s = (int)(chain / (uint32_t)p.num_kv), h = (int)(chain - (uint32_t)s * (uint32_t)p.num_kv);
  const int n = p.chains[kEvictChain * chain + 1];
  if (n == 0) return;
  if (tid == 0) ticket = atomicAdd(p.chains + kEvictChain * chain, 1);
  __syncthreads();
  const int chunk = ticket, r0 = chunk * ROWS;
  if (r0 >= n) return;   // (no chunk after it has rows: none waits for it)
  const int32_t* kept = p.kept + (long)chain * p.max_keep;
  const int32_t* table = p.tables + (long)s * p.max_blocks;
  const int rows = min(ROWS, n - r0), bt = p.block_tokens;
  auto at = [&](int r) { return block_at(p.bt_magic, bt, r); };
  const uint32_t row_bytes = (uint32_t)p.num_kv * HD;
  auto offset = [&](int page, int row) { return (long)page * bt * row_bytes + (long)row * row_bytes + h * HD; };

  // ---- the rows' codes and weights
  u4_t kv[2][N];
  int from_e[2][N], src[N], to_page[N], to_row[N];
  const int part = tid % LPR;
  bool moved = false;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int r = r0 + min(i * PER + tid / LPR, rows - 1);
    src[i] = kept[r];
    moved |= src[i] != r;
    const BlockAt x = at(src[i]), y = at(r);
    const int page = table[x.b];
    to_page[i] = table[y.b];
    to_row[i] = y.row;
    const long o = offset(page, x.row) + 16 * part;
    kv[0][i] = *reinterpret_cast<const u4_t*>(p.k_pool + o);
    kv[1][i] = *reinterpret_cast<const u4_t*>(p.v_pool + o);
    from_e[0][i] = p.k_exp[(long)page * p.num_kv + h];
    from_e[1][i] = p.v_exp[(long)page * p.num_kv + h];
  }
  float w = 0.f;
  int w_src = -1, w_page = 0, w_row = 0;
  if (tid < rows) {
    w_src = kept[r0 + tid];
    const BlockAt x = at(w_src), y = at(r0 + tid);
    w = p.weights[((long)table[x.b] * p.num_kv + h) * bt + x.row];
    w_page = table[y.b];
    w_row = y.row;
  }
  // ---- the new exponents of the pages that the chunk's rows lie in, over all of those pages' rows (131,072 rows to half:
  // 141 us in pages of 256, 164 of 1,024, 238 of 4,096)
  const int b0 = at(r0).b, b1 = at(r0 + rows - 1).b;
  for (int i = tid; i <= b1 - b0; i += 256) exps[0][i] = exps[1][i] = 0;
  __syncthreads();
  for (long r = (long)b0 * bt + tid, end = min((long)n, (long)(b1 + 1) * bt); r < end; r += 256) {
    const int page = table[at(kept[r]).b], b = at((int)r).b - b0;
    atomicMax(&exps[0][b], (int)p.k_exp[(long)page * p.num_kv + h]);
    atomicMax(&exps[1][b], (int)p.v_exp[(long)page * p.num_kv + h]);
  }
  __syncthreads();
  // rows that stay where they are need nothing, unless their page's exponent rises
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int b = at(r0 + min(i * PER + tid / LPR, rows - 1)).b - b0;
    moved |= exps[0][b] != from_e[0][i] || exps[1][b] != from_e[1][i];
  }
  // ---- all of it has been read: said, then waited for by those before
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  const bool change = __syncthreads_or(moved);
  int* flags = p.flags + (long)chain * p.chunks;
  if (tid == 0) __hip_atomic_store(flags + chunk, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (!change) return;
  // Flags of the 256 chunks before, and so on down; 2: all below that one were set too.
  for (int c = chunk - 1; c >= 0; c -= 256) {
    const int mine = c - tid;
    bool all = false;
    while (true) {
      const int f = mine >= 0 ? __hip_atomic_load(flags + mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 1;
      if (__syncthreads_and(f != 0)) {
        all = __syncthreads_or(f == 2);
        break;
      }
      __builtin_amdgcn_s_sleep(1);
    }
    if (all) break;
  }
  if (tid == 0) __hip_atomic_store(flags + chunk, 2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // ---- written
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int x = i * PER + tid / LPR;
    if (x >= rows) break;
    const int b = at(r0 + x).b - b0;
    const long o = offset(to_page[i], to_row[i]) + 16 * part;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int d = exps[j][b] - from_e[j][i];
      u4_t v = kv[j][i];
      if (d > 0) {
        const float f = pow2_bits(127 - min(d, 126));
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = rescale4(v[e], f);
      }
      // (past the caches, which the rows still to be read go through: 93 -> 85 us for 24 slots)
      if (d > 0 || src[i] != r0 + x) __builtin_nontemporal_store(v, reinterpret_cast<u4_t*>((j ? p.v_pool : p.k_pool) + o));
    }
  }
  if (tid < rows && w_src != r0 + tid) p.weights[((long)w_page * p.num_kv + h) * bt + w_row] = w;
  // a page's exponent by its last chunk: every chunk that reads it comes before
  if (tid <= b1 - b0 && (r0 + rows == n || (long)(b0 + tid + 1) * bt <= r0 + rows)) {
    const long e = (long)table[b0 + tid] * p.num_kv + h;
    p.k_exp[e] = (uint8_t)exps[0][tid];
    p.v_exp[e] = (uint8_t)exps[1][tid];
  }
}

hipError_t launch_evict(EvictArgs a, int head_dim, hipStream_t stream) {
  const int chains = a.n_slots * a.num_kv;
  const dim3 grid((unsigned)chains), block(1024), cut((unsigned)(chains * a.stretches));
  if (a.stretches == 0) {
    hipLaunchKernelGGL(evict_select_kernel, grid, block, 0, stream, a);
  } else {
    hipLaunchKernelGGL(evict_stretch_kernel<0>, cut, block, 0, stream, a);
    hipLaunchKernelGGL(evict_stretch_kernel<1>, cut, block, 0, stream, a);
    hipLaunchKernelGGL(evict_stretch_kernel<2>, cut, block, 0, stream, a);
    hipLaunchKernelGGL(evict_stretch_kernel<3>, cut, block, 0, stream, a);
  }
  const dim3 moves((unsigned)((long)chains * a.chunks));
  if (head_dim == 128) hipLaunchKernelGGL(evict_move_kernel<128>, moves, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(evict_move_kernel<256>, moves, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace qkv
