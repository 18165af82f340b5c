// evict_f8.hip -- eviction from the paged 8-bit cache: of each slot and KV head the keys with the most
// accumulated weight stay, in order, moved to the front of the slot's pages.
//
// Two launches.  The first finds what stays, a workgroup for each (slot, KV head): the last and the first rows
// whatever they weigh, and the largest of the weights between, by radix selection on the weights' bits (8 bits a
// pass; ties to the lowest row).  The second moves the rows of both pools and the weights in place.
//
// In place, a row may go where another has not been read yet.  Rows only ever move forward (row i of what stays
// comes from row kept[i] >= i), so a chunk of rows may be written once every chunk before it has been read.
// Workgroups take chunks in that order by a counter, read theirs whole into registers, say so, and only then wait
// for those before: nobody waits before having said it, so every wait ends.
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

// 16 waves; each looks at a stretch of rows of its own, 64 at a time.  HELD: up to 16 steps, whose weights stay in
// registers; else each pass reads them again, from the caches.
template <bool HELD>
__global__ __launch_bounds__(1024) void evict_select_kernel(EvictArgs p) {
  constexpr int STEPS = 16, COPIES = 32;
  // a histogram for every pair of lanes: no two lanes of an access share a bank
  __shared__ int hist[256 * COPIES];
  __shared__ int count[256], gt_s[16], eq_s[16], found[2];
  const int chain = blockIdx.x, s = chain / p.num_kv, h = chain - s * p.num_kv;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int len = p.lens[s], keep = p.keep[s];
  int32_t* kept = p.kept + (long)chain * p.max_keep;
  const int32_t* table = p.tables + (long)s * p.max_blocks;
  const int n_new = min(len, keep);
  bool bad = len < 0 || len > p.max_ctx || keep < 0 || n_new > p.max_keep;
  if (!bad) {
    const int blocks = (int)(((long)len + p.block_tokens - 1) / p.block_tokens);
    bad = blocks > p.max_blocks;
    for (int b = tid; !bad && b < blocks; b += 1024) bad = table[b] < 0 || table[b] >= p.n_pages;
  }
  bad = __syncthreads_or(bad);
  for (int i = tid; i < p.chunks; i += 1024) p.flags[(long)chain * p.chunks + i] = 0;
  if (chain == 0 && tid == 0) *p.ticket = 0;
  if (tid == 0) p.moves[chain] = bad || keep >= len ? 0 : n_new;
  const int from = bad ? 0 : n_new;
  for (int i = from + tid; i < p.max_keep; i += 1024) kept[i] = -1;
  if (bad) return;
  if (keep >= len) {
    for (int i = tid; i < n_new; i += 1024) kept[i] = i;
    return;
  }
  const int last = min(keep, p.recent), first = min(keep - last, p.sink);
  for (int i = tid; i < first; i += 1024) kept[i] = i;
  for (int i = tid; i < last; i += 1024) kept[keep - last + i] = len - last + i;
  int need = keep - first - last;      // of the rows between
  if (need == 0) return;
  const int rows = len - first - last;
  const int steps = ((rows + 15) / 16 + 63) / 64, lo = min(wave * steps * 64, rows), hi = min(lo + steps * 64, rows);
  auto weight = [&](int i) {           // of row first + i, in order
    const BlockAt x = block_at(p.bt_magic, p.block_tokens, first + i);
    return order_of(p.weights[((long)table[x.b] * p.num_kv + h) * p.block_tokens + x.row]);
  };
  uint32_t held[HELD ? STEPS : 1];
  if constexpr (HELD) {
#pragma unroll
    for (int t = 0; t < STEPS; t++) {
      const int i = lo + 64 * t + lane;
      held[t] = i < hi ? weight(i) : 0u;
    }
  }
  // f(row, key, whether it is one) over the wave's rows in order
  auto each = [&](auto&& f) {
    if constexpr (HELD) {
#pragma unroll
      for (int t = 0; t < STEPS; t++)
        if (lo + 64 * t < hi) f(lo + 64 * t + lane, held[t], lo + 64 * t + lane < hi);
    } else {
      for (int t = lo; t < hi; t += 64 * 8) {
        uint32_t k[8];
#pragma unroll
        for (int u = 0; u < 8; u++) k[u] = weight(min(t + 64 * u + lane, hi - 1));
#pragma unroll
        for (int u = 0; u < 8; u++)
          if (t + 64 * u < hi) f(t + 64 * u + lane, k[u], t + 64 * u + lane < hi);
      }
    }
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
      int c[4], n = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) n += c[i] = count[255 - (4 * lane + i)];
      int up = n;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(up, d);
        if (lane >= d) up += o;
      }
      int above = up - n;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (above < need && above + c[i] >= need) {
          found[0] = 255 - (4 * lane + i);
          found[1] = need - above;
        }
        above += c[i];
      }
    }
    __syncthreads();
    prefix = prefix << 8 | (uint32_t)found[0];
    need = found[1];
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
  int at = first + gt_before + min(eq_before, need);
  each([&](int i, uint32_t k, bool is) {
    const uint64_t below = (1ull << lane) - 1, m = __builtin_amdgcn_ballot_w64(is && k == prefix);
    const bool stays = is && (k > prefix || (k == prefix && eq_before + __popcll(m & below) < need));
    const uint64_t n = __builtin_amdgcn_ballot_w64(stays);
    if (stays) kept[at + __popcll(n & below)] = first + i;
    at += __popcll(n);
    eq_before += __popcll(m);
  });
}

// A chunk of 16384 / HD rows of a (slot, KV head): 64 bytes a thread of each pool.
template <int HD>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs p) {
  constexpr int ROWS = kEvictBytes / HD, LPR = HD / 16, PER = 256 / LPR, N = ROWS / PER;
  __shared__ int ticket, exps[2][ROWS];
  const int tid = threadIdx.x;
  if (tid == 0) ticket = atomicAdd(p.ticket, 1);
  __syncthreads();
  const int chains = p.n_slots * p.num_kv;
  const int chunk = ticket / chains, chain = ticket - chunk * chains, s = chain / p.num_kv, h = chain - s * p.num_kv;
  const int n = p.moves[chain], r0 = chunk * ROWS;
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
  // ---- the new exponents of the pages that the chunk's rows lie in, over all of those pages' rows
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
      if (d > 0 || src[i] != r0 + x) *reinterpret_cast<u4_t*>((j ? p.v_pool : p.k_pool) + o) = v;
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
  const dim3 grid((unsigned)chains), block(1024);
  if (a.max_ctx <= 16 * 16 * 64) hipLaunchKernelGGL(evict_select_kernel<true>, grid, block, 0, stream, a);
  else hipLaunchKernelGGL(evict_select_kernel<false>, grid, block, 0, stream, a);
  const dim3 moves((unsigned)((long)chains * a.chunks));
  if (head_dim == 128) hipLaunchKernelGGL(evict_move_kernel<128>, moves, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(evict_move_kernel<256>, moves, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace qkv
