// kv_pages.hip -- pages of a cache: sharing, reserving, giving back, compacting, copying.
//
// The state is two int32 arrays on the device: the block tables (a negative entry is no
// page) and a reference count per page.  A page is free when its count is 0 and the
// lowest free pages are handed out first, so there is no free list to keep in step and
// the result does not depend on any order: counts change by integer atomics only,
// everything else is written by the one workgroup that owns it.
//
// The planning kernels are bound by latency (a few dependent reads of the tables): release 2.9
// us, fork 4.1, the plan of a reserve 6.0 and of a compaction 5.8, eight slots with three children each.
// The copies are bound by HBM: read and written once, 16 KB a workgroup and step; 24 pages in
// 16 planes, 33.5 MB, 7.7 us with the tables, compacting 368 MB 82 us (4.5 TB/s).
#include <algorithm>

#include "qkv_device.h"
#include "qkv_launch.h"

namespace qkv {

namespace {

constexpr int kChunk = 16384;   // bytes a workgroup copies at a time

// Inclusive scan over the workgroup; `sum` gets the total.
template <int THREADS>
__device__ __forceinline__ int scan_sum(int v, int* lds, int& sum) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  __syncthreads();
  if (lane == 63) lds[w] = v;
  __syncthreads();
  int before = 0;
  sum = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; i++) {
    if (i < w) before += lds[i];
    sum += lds[i];
  }
  return v + before;
}

__device__ __forceinline__ bool any_of(bool v, int* lds) {   // over 256 threads
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = 0;
  const bool w = __builtin_amdgcn_ballot_w64(v) != 0;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = w;
  __syncthreads();
  return lds[0] | lds[1] | lds[2] | lds[3];
}

__device__ __forceinline__ int blocks_of(int tokens, int bt) { return (int)(((long)tokens + bt - 1) / bt); }

// One 16 KB chunk of page src to page dst of a plane.  STREAM: past the caches, for bulk moves
// (compacting 370 MB: 89 -> 82 us); a reserve's few pages are read again at once (8 against 10 us).
template <bool STREAM>
__device__ __forceinline__ void copy_chunk(uint8_t* base, uint64_t bytes, int src, int dst, uint64_t at) {
  const uint8_t* from = base + (uint64_t)src * bytes + at;
  uint8_t* to = base + (uint64_t)dst * bytes + at;
  const int n = (int)min((uint64_t)kChunk, bytes - at);
  const uint64_t align = reinterpret_cast<uintptr_t>(base) | bytes;
  const int tid = threadIdx.x;
  if ((align & 15) == 0) {
    const int q = n / 16;
    u4_t v[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (tid + 256 * i < q) {
        const u4_t* src = reinterpret_cast<const u4_t*>(from) + tid + 256 * i;
        v[i] = STREAM ? __builtin_nontemporal_load(src) : *src;
      }
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (tid + 256 * i < q) {
        u4_t* dst = reinterpret_cast<u4_t*>(to) + tid + 256 * i;
        if (STREAM) __builtin_nontemporal_store(v[i], dst);
        else *dst = v[i];
      }
  } else if ((align & 3) == 0) {
    for (int i = tid; i < n / 4; i += 256) reinterpret_cast<uint32_t*>(to)[i] = reinterpret_cast<const uint32_t*>(from)[i];
  } else {
    for (int i = tid; i < n; i += 256) to[i] = from[i];
  }
}

// Pairs (from, to) over every plane, the work spread over `wgs` workgroups; a pair out of
// range, or of a page with itself, is left out.
template <bool STREAM>
__device__ __forceinline__ void copy_pairs(const PagePlanes& pl, const int32_t* pairs, int n, int n_pages, int chunks,
                                           long wg, long wgs) {
  const long per = (long)pl.n * chunks;
  for (long x = wg; x < n * per; x += wgs) {
    const int i = (int)(x / per), r = (int)(x - i * per), k = r / chunks;
    const uint64_t at = (uint64_t)(r - k * chunks) * kChunk;
    const int src = pairs[2 * i], dst = pairs[2 * i + 1];
    if (at >= pl.bytes[k] || src < 0 || dst < 0 || src >= n_pages || dst >= n_pages || src == dst) continue;
    copy_chunk<STREAM>(pl.base[k], pl.bytes[k], src, dst, at);
  }
}

int plane_chunks(const PagePlanes& pl) {
  uint64_t most = 0;
  for (int i = 0; i < pl.n; i++) most = std::max(most, pl.bytes[i]);
  return (int)((most + kChunk - 1) / kChunk);
}
// Enough workgroups for every chunk, at most eight on each CU (then they loop).
unsigned copy_wgs(const PagePlanes& pl, long pairs, int chunks) {
  return (unsigned)std::min<long>(std::max<long>(pairs * pl.n * chunks, 0), 2048);
}

}  // namespace

// ---- fork: a workgroup per child -------------------------------------------
__global__ __launch_bounds__(256) void pages_fork_kernel(PageTables t, const int32_t* parents, const int32_t* children,
                                                         const int32_t* tokens, int n, int32_t* status, PageStatus c) {
  __shared__ int lds[4];
  const int i = blockIdx.x, tid = threadIdx.x;
  const int parent = parents[i], child = children[i], tok = tokens[i];
  const int nb = tok >= 0 ? blocks_of(tok, t.block_tokens) : 0;
  bool bad = parent < 0 || parent >= t.n_slots || child < 0 || child >= t.n_slots || tok < 0 || nb > t.max_blocks;
  // a child is named once, and is no parent of this call
  for (int j = tid; j < n; j += 256) bad |= (j < i && children[j] == child) || parents[j] == child;
  if (!any_of(bad, lds)) {
    const int32_t* from = t.tables + (long)parent * t.max_blocks;
    int32_t* to = t.tables + (long)child * t.max_blocks;
    for (int b = tid; b < t.max_blocks; b += 256) bad |= to[b] >= 0 || (b < nb && from[b] >= t.n_pages);
    if (!any_of(bad, lds)) {
      for (int b = tid; b < nb; b += 256) {
        const int page = from[b];
        to[b] = page;
        if (page >= 0) atomicAdd(t.refs + page, 1);
      }
      if (tid == 0 && status) status[i] = c.ok;
      return;
    }
  }
  if (tid == 0 && status) status[i] = c.invalid;
}

hipError_t launch_pages_fork(const PageTables& t, const int32_t* parents, const int32_t* children,
                             const int32_t* tokens, int n, int32_t* status, const PageStatus& codes,
                             hipStream_t stream) {
  hipLaunchKernelGGL(pages_fork_kernel, dim3((unsigned)n), dim3(256), 0, stream, t, parents, children, tokens, n,
                     status, codes);
  return hipGetLastError();
}

// ---- release: a workgroup per slot -----------------------------------------
__global__ __launch_bounds__(256) void pages_release_kernel(PageTables t, const int32_t* slots, const int32_t* keep,
                                                            int n, int32_t* status, PageStatus c) {
  __shared__ int lds[4];
  const int i = blockIdx.x, tid = threadIdx.x;
  const int slot = slots[i], kept = keep[i];
  bool bad = slot < 0 || slot >= t.n_slots || kept < 0;
  for (int j = tid; j < i; j += 256) bad |= slots[j] == slot;
  if (any_of(bad, lds)) {
    if (tid == 0 && status) status[i] = c.invalid;
    return;
  }
  int32_t* row = t.tables + (long)slot * t.max_blocks;
  for (int b = blocks_of(kept, t.block_tokens) + tid; b < t.max_blocks; b += 256) {
    const int page = row[b];
    if (page >= 0) {
      row[b] = -1;
      if (page < t.n_pages) atomicSub(t.refs + page, 1);
    }
  }
  if (tid == 0 && status) status[i] = c.ok;
}

hipError_t launch_pages_release(const PageTables& t, const int32_t* slots, const int32_t* keep, int n,
                                int32_t* status, const PageStatus& codes, hipStream_t stream) {
  hipLaunchKernelGGL(pages_release_kernel, dim3((unsigned)n), dim3(256), 0, stream, t, slots, keep, n, status, codes);
  return hipGetLastError();
}

// ---- reserve ---------------------------------------------------------------
// The plan, one workgroup: what each slot's blocks want (1: a page, 2: a page of its own in
// place of a shared one), the lowest free pages for all of it, and which slots are served
// (in list order while the pages last).  A page that every sharer of this call gives up
// is copied by each of them and becomes free: no order among them decides.
struct ReserveScratch {
  int32_t* pairs;   // [n][2] pages to copy
  int32_t* off;     // [n] first fresh page of a served slot, -1
  int32_t* want;    // [n][blocks]
  int32_t* fresh;   // [n * blocks]
};
__device__ __host__ inline ReserveScratch reserve_scratch(int32_t* s, int n, int blocks) {
  return {s, s + 2 * (long)n, s + 3 * (long)n, s + 3 * (long)n + (long)n * blocks};
}

__global__ __launch_bounds__(1024) void pages_plan_kernel(PageTables t, const int32_t* slots, const int32_t* positions,
                                                          const int32_t* n_new, int n, int max_new, int blocks,
                                                          int32_t* status, PageStatus c, int32_t* scratch) {
  __shared__ int slot_s[kReserveMax], need_s[kReserveMax], bad_s[kReserveMax], lds[16];
  const int tid = threadIdx.x;
  const ReserveScratch r = reserve_scratch(scratch, n, blocks);
  int pos = 0, cnt = 0;
  if (tid < n) {
    slot_s[tid] = slots[tid];
    pos = positions[tid];
    cnt = n_new[tid];
    need_s[tid] = 0;
  }
  __syncthreads();
  if (tid < n) {
    const int slot = slot_s[tid];
    bool bad = slot < 0 || slot >= t.n_slots || pos < 0 || cnt < 0 || cnt > max_new ||
               (cnt > 0 && ((long)pos + cnt - 1) / t.block_tokens >= t.max_blocks);
    for (int j = 0; j < tid; j++) bad |= slot_s[j] == slot;
    bad_s[tid] = bad;
  }
  __syncthreads();
  for (long x = tid; x < (long)n * blocks; x += 1024) {
    const int i = (int)(x / blocks), j = (int)(x - (long)i * blocks);
    int code = 0;
    if (!bad_s[i]) {
      const int p0 = positions[i], k = n_new[i];
      const long b = (long)p0 / t.block_tokens + j;
      if (k > 0 && b <= ((long)p0 + k - 1) / t.block_tokens) {
        const int page = t.tables[(long)slot_s[i] * t.max_blocks + b];
        code = page < 0 ? 1 : page >= t.n_pages ? 3 : t.refs[page] > 1 ? 2 : 0;
      }
    }
    r.want[x] = code;
    if (code == 3) atomicOr(&need_s[i], 1 << 30);   // (an entry past the pool)
    else if (code) atomicAdd(&need_s[i], 1);
  }
  __syncthreads();
  const bool mine = tid < n;
  bool bad = mine && (bad_s[tid] || need_s[tid] >= 1 << 30);
  const int need = mine && !bad ? need_s[tid] : 0;
  int total;
  const int inc = scan_sum<1024>(need, lds, total);
  // the lowest `total` free pages, in order
  int found = 0;
  for (long b = 0; b < t.n_pages && found < total; b += 4096) {
    const long p0 = b + 4 * tid;
    bool free[4];
    int k = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      free[e] = p0 + e < t.n_pages && t.refs[p0 + e] == 0;
      k += free[e];
    }
    int sum;
    int at = found + scan_sum<1024>(k, lds, sum) - k;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (free[e]) {
        if (at < total) r.fresh[at] = (int)(p0 + e);
        at++;
      }
    found += sum;
  }
  __syncthreads();
  if (!mine) return;
  const bool served = !bad && (need == 0 || inc <= found);
  const int off = served && need > 0 ? inc - need : -1;
  r.off[tid] = off;
  if (status) status[tid] = bad ? c.invalid : served ? c.ok : c.pages;
  // rows ahead of the first new one move along when its page is shared
  int src = -1, dst = -1;
  if (off >= 0 && r.want[(long)tid * blocks] == 2 && pos % t.block_tokens > 0) {
    src = t.tables[(long)slot_s[tid] * t.max_blocks + pos / t.block_tokens];
    dst = r.fresh[off];
  }
  r.pairs[2 * tid] = src;
  r.pairs[2 * tid + 1] = dst;
}

// The plan carried out: workgroups 0 .. n-1 (their first wave) the tables and counts of a
// slot each, the others the copies.
__global__ __launch_bounds__(256) void pages_apply_kernel(PageTables t, const int32_t* slots, const int32_t* positions,
                                                          int n, int blocks, PagePlanes planes, int chunks,
                                                          int32_t* scratch) {
  const ReserveScratch r = reserve_scratch(scratch, n, blocks);
  if (blockIdx.x >= (unsigned)n) {
    copy_pairs<false>(planes, r.pairs, n, t.n_pages, chunks, (long)blockIdx.x - n, (long)gridDim.x - n);
    return;
  }
  const int i = blockIdx.x, lane = threadIdx.x;
  const int off = r.off[i];
  if (off < 0 || lane >= 64) return;
  int32_t* row = t.tables + (long)slots[i] * t.max_blocks + positions[i] / t.block_tokens;
  int rank = off;
  for (int j0 = 0; j0 < blocks; j0 += 64) {
    const int j = j0 + lane;
    const int code = j < blocks ? r.want[(long)i * blocks + j] : 0;
    const uint64_t m = __builtin_amdgcn_ballot_w64(code != 0);
    if (code) {
      const int page = r.fresh[rank + __popcll(m & ((1ull << lane) - 1))];
      if (code == 2) atomicSub(t.refs + row[j], 1);
      row[j] = page;
      t.refs[page] = 1;
    }
    rank += __popcll(m);
  }
}

hipError_t launch_pages_reserve(const PageTables& t, const int32_t* slots, const int32_t* positions,
                                const int32_t* n_new, int n, int max_new, int32_t* status, const PageStatus& codes,
                                const PagePlanes& planes, int32_t* scratch, hipStream_t stream) {
  const int blocks = reserve_blocks(max_new, t.block_tokens), chunks = plane_chunks(planes);
  hipLaunchKernelGGL(pages_plan_kernel, dim3(1), dim3(1024), 0, stream, t, slots, positions, n_new, n, max_new, blocks,
                     status, codes, scratch);
  hipLaunchKernelGGL(pages_apply_kernel, dim3((unsigned)n + copy_wgs(planes, n, chunks)), dim3(256), 0, stream, t,
                     slots, positions, n, blocks, planes, chunks, scratch);
  return hipGetLastError();
}

// ---- copy ------------------------------------------------------------------
__global__ __launch_bounds__(256) void pages_copy_kernel(PagePlanes planes, const int32_t* pairs, int n, int n_pages,
                                                         int chunks) {
  copy_pairs<true>(planes, pairs, n, n_pages, chunks, blockIdx.x, gridDim.x);
}

hipError_t launch_pages_copy(const PagePlanes& planes, const int32_t* pairs, int n, int n_pages, hipStream_t stream) {
  const int chunks = plane_chunks(planes);
  hipLaunchKernelGGL(pages_copy_kernel, dim3(copy_wgs(planes, n, chunks)), dim3(256), 0, stream, planes, pairs, n,
                     n_pages, chunks);
  return hipGetLastError();
}

// ---- compact ---------------------------------------------------------------
// The plan, one workgroup: with `used` pages in use, the i-th of them at or past index
// `used` goes to the i-th free page before it.  scratch: the number of moves, a pad, pairs.
__global__ __launch_bounds__(1024) void pages_compact_plan_kernel(PageTables t, int32_t* moved, int32_t* n_used,
                                                                  int32_t* scratch) {
  __shared__ int lds[16];
  const int tid = threadIdx.x;
  int used = 0;
  for (long p = tid; p < t.n_pages; p += 1024) used += t.refs[p] > 0;
  int total;
  scan_sum<1024>(used, lds, total);
  int holes = 0, moves = 0;
  int32_t* pairs = scratch + 2;
  for (long b = 0; b < t.n_pages; b += 1024) {
    const long p = b + tid;
    const bool in = p < t.n_pages, use = in && t.refs[p] > 0;
    const bool hole = in && !use && p < total, move = use && p >= total;
    // both counts in one scan (each is at most 1024 a step)
    int sum;
    const int inc = scan_sum<1024>((hole ? 1 : 0) + (move ? 1 << 16 : 0), lds, sum);
    if (hole) pairs[2 * (holes + (inc & 0xffff) - 1) + 1] = (int)p;
    if (move) pairs[2 * (moves + (inc >> 16) - 1)] = (int)p;
    if (in) moved[p] = use ? (int)p : -1;
    holes += sum & 0xffff;
    moves += sum >> 16;
  }
  __syncthreads();
  for (long i = tid; i < moves; i += 1024) {
    const int src = pairs[2 * i], dst = pairs[2 * i + 1];
    moved[src] = dst;
    t.refs[dst] = t.refs[src];
    t.refs[src] = 0;
  }
  if (tid == 0) {
    scratch[0] = moves;
    n_used[0] = total;
  }
}

__global__ __launch_bounds__(256) void pages_compact_kernel(PageTables t, const int32_t* moved, PagePlanes planes,
                                                            int chunks, const int32_t* scratch, int table_wgs) {
  if (blockIdx.x >= (unsigned)table_wgs) {
    copy_pairs<true>(planes, scratch + 2, scratch[0], t.n_pages, chunks, (long)blockIdx.x - table_wgs,
               (long)gridDim.x - table_wgs);
    return;
  }
  const long entries = (long)t.n_slots * t.max_blocks;
  for (long x = (long)blockIdx.x * 256 + threadIdx.x; x < entries; x += (long)table_wgs * 256) {
    const int page = t.tables[x];
    if (page >= 0 && page < t.n_pages) {
      const int to = moved[page];
      if (to >= 0 && to != page) t.tables[x] = to;
    }
  }
}

hipError_t launch_pages_compact(const PageTables& t, int32_t* moved, int32_t* n_used, const PagePlanes& planes,
                                int32_t* scratch, hipStream_t stream) {
  const int chunks = plane_chunks(planes);
  hipLaunchKernelGGL(pages_compact_plan_kernel, dim3(1), dim3(1024), 0, stream, t, moved, n_used, scratch);
  const long entries = (long)t.n_slots * t.max_blocks;
  const int table_wgs = (int)std::min<long>((entries + 255) / 256, 1024);
  hipLaunchKernelGGL(pages_compact_kernel, dim3((unsigned)table_wgs + copy_wgs(planes, t.n_pages / 2, chunks)),
                     dim3(256), 0, stream, t, moved, planes, chunks, scratch, table_wgs);
  return hipGetLastError();
}

}  // namespace qkv
