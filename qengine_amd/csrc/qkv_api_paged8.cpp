// qkv_api_paged8.cpp -- the C ABI of rotary positions, the paged 8-bit cache and the page
// calls (declared in include/qkv.h): argument checks, then launches on the caller's stream.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "qkv_api_checks.h"

extern "C" {

int qkv_rope_table(int rot_dim, double base, int scaling, double factor, double original_ctx, double beta_fast,
                   double beta_slow, uint64_t* turns, float* amplitude) {
  if (rot_dim < 2 || rot_dim % 2 || !(base > 0.0) || !std::isfinite(base)) return QKV_ERR_INVALID;
  if (scaling < QKV_ROPE_PLAIN || scaling > QKV_ROPE_YARN) return QKV_ERR_INVALID;
  if (scaling != QKV_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) return QKV_ERR_INVALID;
  if (scaling == QKV_ROPE_NTK && rot_dim < 4) return QKV_ERR_INVALID;
  if (scaling == QKV_ROPE_YARN && (!(original_ctx > 0.0) || !(beta_fast > beta_slow) || !std::isfinite(original_ctx) ||
                                   !std::isfinite(beta_fast) || !std::isfinite(beta_slow)))
    return QKV_ERR_INVALID;
  if (!turns || !amplitude) return QKV_ERR_NULL;
  const long double two_pi = 6.283185307179586476925286766559L;
  long double b = base;
  if (scaling == QKV_ROPE_NTK) b *= powl(factor, (long double)rot_dim / (rot_dim - 2));
  for (int i = 0; i < rot_dim / 2; i++) {
    long double f = powl(b, -2.0L * i / rot_dim);
    if (scaling == QKV_ROPE_LINEAR) f /= factor;
    if (scaling == QKV_ROPE_YARN) {
      // dims that turn more than beta_fast times in the original context keep their
      // frequency, those below beta_slow turns are interpolated, linearly in between
      const long double full = original_ctx * f / two_pi;
      const long double keep = fminl(1.0L, fmaxl(0.0L, (full - beta_slow) / (beta_fast - beta_slow)));
      f = keep * f + (1.0L - keep) * f / factor;
    }
    long double t = f / two_pi;
    t -= floorl(t);
    const long double r = roundl(ldexpl(t, 64));
    turns[i] = r >= 18446744073709551616.0L ? 0u : (uint64_t)r;
  }
  *amplitude = scaling == QKV_ROPE_YARN ? (float)(1.0 + 0.1 * std::log(factor)) : 1.0f;
  return QKV_OK;
}

int qkv_rope(const uint16_t* q, long q_stride, uint16_t* q_out, long q_out_stride, const uint16_t* k, long k_stride,
             uint16_t* k_out, long k_out_stride, const int32_t* positions, const uint64_t* turns, float amplitude,
             int n_tok, int num_q, int num_k, int head_dim, int rot_dim, int layout, int inverse,
             hipStream_t stream) {
  if (n_tok < 0 || num_q < 0 || num_k < 0 || num_q + num_k == 0 || num_q > 1024 || num_k > 1024 || head_dim <= 0 ||
      head_dim > 8192 || rot_dim < 2 || rot_dim % 2 || rot_dim > head_dim || layout < 0 || layout > 1)
    return QKV_ERR_INVALID;
  if (n_tok == 0) return QKV_OK;
  if ((num_q && (!q || !q_out)) || (num_k && (!k || !k_out)) || !positions || !turns) return QKV_ERR_NULL;
  const long need_q = (long)num_q * head_dim, need_k = (long)num_k * head_dim;
  if (n_tok > 1 && ((num_q && (q_stride < need_q || q_out_stride < need_q)) ||
                    (num_k && (k_stride < need_k || k_out_stride < need_k))))
    return QKV_ERR_INVALID;
  if ((num_q && q == q_out && q_stride != q_out_stride) || (num_k && k == k_out && k_stride != k_out_stride))
    return QKV_ERR_INVALID;
  if (num_q && num_k && q_out == k_out) return QKV_ERR_INVALID;
  if ((num_q && (!aligned(q, 2) || !aligned(q_out, 2))) || (num_k && (!aligned(k, 2) || !aligned(k_out, 2))) ||
      !aligned(positions, 4) || !aligned(turns, 8))
    return QKV_ERR_ALIGN;
  qkv::RopeArgs a{};
  a.q = num_q ? q : nullptr;
  a.q_out = q_out;
  a.k = num_k ? k : nullptr;
  a.k_out = k_out;
  a.positions = positions;
  a.turns = turns;
  a.q_stride = q_stride;
  a.q_out_stride = q_out_stride;
  a.k_stride = k_stride;
  a.k_out_stride = k_out_stride;
  a.amplitude = amplitude;
  a.n_tok = n_tok;
  a.num_q = num_q;
  a.num_k = num_k;
  a.head_dim = head_dim;
  a.rot = rot_dim;
  a.layout = layout;
  a.inverse = inverse != 0;
  bool wide = rot_dim % 16 == 0 && head_dim % 16 == 0;
  if (num_q) wide = wide && aligned(q, 16) && aligned(q_out, 16) && q_stride % 8 == 0 && q_out_stride % 8 == 0;
  if (num_k) wide = wide && aligned(k, 16) && aligned(k_out, 16) && k_stride % 8 == 0 && k_out_stride % 8 == 0;
  const bool in_place = (!num_q || q == q_out) && (!num_k || k == k_out);
  if ((double)n_tok * (num_q + num_k) * head_dim / 256 > 2147483647.0) return QKV_ERR_UNSUPPORTED;
  return launch_status(qkv::launch_rope(a, wide, in_place, stream));
}

int qkv_f8_append_kv_paged(const uint16_t* k, long k_stride, const uint16_t* v, long v_stride, uint8_t* k_pool,
                           uint8_t* v_pool, uint8_t* k_exp, uint8_t* v_exp, int n_rows, int n_slots, int max_tok,
                           int num_kv, int head_dim, const int32_t* block_tables, int max_blocks, int block_tokens,
                           int n_pages, const int32_t* starts, const int32_t* positions, const uint16_t* q,
                           long q_stride, uint16_t* q_out, long q_out_stride, int num_q, const uint64_t* turns,
                           float amplitude, int rot_dim, int layout, hipStream_t stream) {
  const int st = check_f8_pool(num_kv, head_dim, max_blocks, block_tokens, n_pages);
  if (st != QKV_OK) return st;
  if (n_rows < 0 || n_slots < 0 || max_tok < 0) return QKV_ERR_INVALID;
  if (rot_dim < 0 || rot_dim > head_dim || layout < 0 || layout > 1 || num_q < 0 || num_q > 1024) return QKV_ERR_INVALID;
  if (rot_dim % 16) return QKV_ERR_UNSUPPORTED;
  if (num_q > 0 && rot_dim == 0) return QKV_ERR_INVALID;   // (nothing to do with the queries)
  if (n_rows == 0 || n_slots == 0 || max_tok == 0) return QKV_OK;
  if (!k || !v || !k_pool || !v_pool || !k_exp || !v_exp || !block_tables || !starts || !positions ||
      (rot_dim && !turns) || (num_q && (!q || !q_out)))
    return QKV_ERR_NULL;
  const long need = (long)num_kv * head_dim, need_q = (long)num_q * head_dim;
  if (n_rows > 1 && (k_stride < need || v_stride < need || (num_q && (q_stride < need_q || q_out_stride < need_q))))
    return QKV_ERR_INVALID;
  if (num_q && q == q_out && q_stride != q_out_stride) return QKV_ERR_INVALID;
  if (!aligned(k, 16) || !aligned(v, 16) || k_stride % 8 || v_stride % 8 || !aligned(k_pool, 16) ||
      !aligned(v_pool, 16) || !aligned(block_tables, 4) || !aligned(starts, 4) || !aligned(positions, 4) ||
      (rot_dim && !aligned(turns, 8)) ||
      (num_q && (!aligned(q, 16) || !aligned(q_out, 16) || q_stride % 8 || q_out_stride % 8)))
    return QKV_ERR_ALIGN;
  qkv::F8AppendArgs a{};
  a.k = k;
  a.v = v;
  a.q = num_q ? q : nullptr;
  a.q_out = q_out;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.k_exp = k_exp;
  a.v_exp = v_exp;
  a.tables = block_tables;
  a.starts = starts;
  a.positions = positions;
  a.turns = turns;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_stride = q_stride;
  a.q_out_stride = q_out_stride;
  a.rows = n_rows;
  a.amplitude = amplitude;
  a.n_slots = n_slots;
  a.max_tok = max_tok < n_rows ? max_tok : n_rows;
  a.max_blocks = max_blocks;
  a.block_tokens = block_tokens;
  a.n_pages = n_pages;
  a.num_q = num_q;
  a.num_kv = num_kv;
  a.head_dim = head_dim;
  a.rot = rot_dim;
  a.layout = layout;
  const double spans = ((double)a.max_tok + block_tokens) / block_tokens + 1;
  if (spans * n_slots * num_kv * 2 + (double)n_rows * num_q * head_dim / 512 > 2147483647.0) return QKV_ERR_UNSUPPORTED;
  return launch_status(qkv::launch_f8_append(a, stream));
}

static int check_f8_attn(int num_q, int num_kv, int head_dim, int n_slots, int n_rows, int max_tok, int max_ctx) {
  if (head_dim != 128 && head_dim != 256) return QKV_ERR_UNSUPPORTED;
  if (num_kv <= 0 || num_q <= 0 || num_q % num_kv != 0 || n_slots <= 0 || n_rows <= 0 || max_tok <= 0 || max_ctx <= 0)
    return QKV_ERR_INVALID;
  if (num_q / num_kv > 8 || num_q > 1024 || max_ctx > (1 << 30)) return QKV_ERR_UNSUPPORTED;
  if (max_tok > n_rows) max_tok = n_rows;
  // row tiles of the call, and the key tiles of them all with their leads (counted in 32 bits,
  // a head's in 30)
  const double gqa = num_q / num_kv, full = (double)n_slots * ((double)max_tok * gqa / 256 + 1);
  const double tiles = full < n_rows * gqa / 256 + n_slots ? full : n_rows * gqa / 256 + n_slots;
  if (full * num_kv > (double)(1 << 22) || tiles * std::max(num_kv, 2) * (max_ctx / 32.0 + 16) > 2147483000.0)
    return QKV_ERR_UNSUPPORTED;
  return QKV_OK;
}

}  // extern "C"

namespace {

// The launches of a call, one after the other in the same workspace: the slots of up to `apart`
// tokens (if any), then the others.
struct F8AttnPlans {
  int apart;
  qkv::F8AttnPlan few, rest;
  size_t total() const { return apart ? std::max(few.total, rest.total) : rest.total; }
};
F8AttnPlans f8_attn_plans(int num_q, int num_kv, int head_dim, int n_slots, int n_rows, int max_tok, int max_ctx) {
  if (max_tok > n_rows) max_tok = n_rows;
  F8AttnPlans x{};
  x.apart = qkv::f8_attn_apart(num_q, num_kv, head_dim, n_slots, n_rows, max_tok, max_ctx);
  if (x.apart) x.few = qkv::f8_attn_plan(num_q, num_kv, head_dim, n_slots, n_rows, x.apart, max_ctx);
  x.rest = qkv::f8_attn_plan(num_q, num_kv, head_dim, n_slots, n_rows, max_tok, max_ctx);
  return x;
}

}  // namespace

extern "C" {

size_t qkv_attn_f8_paged_workspace_bytes(int num_q, int num_kv, int head_dim, int n_slots, int n_rows, int max_tok,
                                         int max_ctx) {
  if (check_f8_attn(num_q, num_kv, head_dim, n_slots, n_rows, max_tok, max_ctx) != QKV_OK) return 0;
  // The largest of any call with up to these numbers.  A kernel's workspace grows with each of them, but
  // the kernel for more rows may need less than that for fewer, so each is asked for the most rows it takes.
  if (max_tok > n_rows) max_tok = n_rows;
  size_t most = qkv::f8_attn_plan(num_q, num_kv, head_dim, n_slots, n_rows, max_tok, max_ctx).total;
  const int gqa = num_q / num_kv;
  for (int rows : {16, 32, 64})
    if (rows / gqa < max_tok)
      most = std::max(most, qkv::f8_attn_plan(num_q, num_kv, head_dim, n_slots, n_rows, rows / gqa, max_ctx).total);
  return most;
}

int qkv_attn_f8_paged(const uint16_t* q, const uint8_t* k_pool, const uint8_t* v_pool, const uint8_t* k_exp,
                      const uint8_t* v_exp, uint16_t* out, int n_rows, int num_q, int num_kv, int head_dim,
                      int n_slots, int max_tok, int max_ctx, const int32_t* block_tables, int max_blocks,
                      int block_tokens, int n_pages, const int32_t* starts, const int32_t* positions, float scale,
                      int window_tok, int sink_tok, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  int st = check_f8_pool(num_kv, head_dim, max_blocks, block_tokens, n_pages);
  if (st != QKV_OK) return st;
  if (n_rows == 0 || n_slots == 0 || max_tok == 0) return QKV_OK;
  st = check_f8_attn(num_q, num_kv, head_dim, n_slots, n_rows, max_tok, max_ctx);
  if (st != QKV_OK) return st;
  if (window_tok < 0 || sink_tok < 0) return QKV_ERR_INVALID;
  if (!q || !k_pool || !v_pool || !k_exp || !v_exp || !out || !block_tables || !starts || !positions) return QKV_ERR_NULL;
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(k_pool, 16) || !aligned(v_pool, 16) ||
      !aligned(block_tables, 4) || !aligned(starts, 4) || !aligned(positions, 4))
    return QKV_ERR_ALIGN;
  if (max_tok > n_rows) max_tok = n_rows;
  const F8AttnPlans plans = f8_attn_plans(num_q, num_kv, head_dim, n_slots, n_rows, max_tok, max_ctx);
  if (!workspace || workspace_bytes < plans.total()) return QKV_ERR_WORKSPACE;
  if (!aligned(workspace, 256)) return QKV_ERR_ALIGN;
  qkv::F8AttnArgs a{};
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.q = q;
  a.out = out;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.k_exp = k_exp;
  a.v_exp = v_exp;
  a.tables = block_tables;
  a.starts = starts;
  a.positions = positions;
  a.counts = reinterpret_cast<int*>(ws);
  a.cuts = a.counts + qkv::kJoinCounts;
  a.desc = reinterpret_cast<int2*>(a.cuts);
  a.rows = n_rows;
  a.num_q = num_q;
  a.num_kv = num_kv;
  a.n_slots = n_slots;
  a.max_tok = max_tok;
  a.max_ctx = max_ctx;
  a.max_blocks = max_blocks;
  a.block_tokens = block_tokens;
  a.n_pages = n_pages;
  a.window = window_tok;
  a.sink = sink_tok < max_ctx ? sink_tok : max_ctx;   // (rounded up to tiles in 32 bits)
  a.gqa = num_q / num_kv;
  a.bt_magic = (uint32_t)((1ull << 32) / (uint64_t)block_tokens);
  a.gqa_magic = (uint32_t)std::min<uint64_t>((1ull << 32) / (uint64_t)a.gqa, 0xffffffffull);
  a.scale_log2 = scale * 1.4426950408889634f;
  auto launch = [&](const qkv::F8AttnPlan& x, int from, int to) {
    a.rec_ml = reinterpret_cast<float*>(ws + x.ml_off);
    a.rec_o = reinterpret_cast<float*>(ws + x.o_off);
    a.slot_tiles = x.slot_tiles;
    a.rec_rows = x.rec_rows;
    a.groups = x.groups;
    a.from_tok = from;
    a.to_tok = to;
    return launch_status(qkv::launch_f8_attn(a, x, head_dim, stream));
  };
  if (plans.apart) {
    const int st1 = launch(plans.few, 1, plans.apart);
    if (st1 != QKV_OK) return st1;
  }
  return launch(plans.rest, plans.apart + 1, 0x7fffffff);
}

int qkv_pages_fork(int32_t* block_tables, int n_slots, int max_blocks, int block_tokens, int32_t* ref_counts,
                   int n_pages, const int32_t* parents, const int32_t* children, const int32_t* n_tokens, int n,
                   int32_t* status, hipStream_t stream) {
  const qkv::PageTables t{block_tables, ref_counts, n_slots, max_blocks, block_tokens, n_pages};
  const int st = check_tables(t);
  if (st != QKV_OK) return st;
  if (n < 0 || n > n_slots) return QKV_ERR_INVALID;
  if (n >= kMaxList) return QKV_ERR_UNSUPPORTED;
  if (n == 0) return QKV_OK;
  if (!parents || !children || !n_tokens) return QKV_ERR_NULL;
  if (!aligned(parents, 4) || !aligned(children, 4) || !aligned(n_tokens, 4) || !aligned(status, 4)) return QKV_ERR_ALIGN;
  return launch_status(qkv::launch_pages_fork(t, parents, children, n_tokens, n, status, kPageStatus, stream));
}

int qkv_pages_release(int32_t* block_tables, int n_slots, int max_blocks, int block_tokens, int32_t* ref_counts,
                      int n_pages, const int32_t* slots, const int32_t* keep_tokens, int n, int32_t* status,
                      hipStream_t stream) {
  const qkv::PageTables t{block_tables, ref_counts, n_slots, max_blocks, block_tokens, n_pages};
  const int st = check_tables(t);
  if (st != QKV_OK) return st;
  if (n < 0 || n > n_slots) return QKV_ERR_INVALID;
  if (n >= kMaxList) return QKV_ERR_UNSUPPORTED;
  if (n == 0) return QKV_OK;
  if (!slots || !keep_tokens) return QKV_ERR_NULL;
  if (!aligned(slots, 4) || !aligned(keep_tokens, 4) || !aligned(status, 4)) return QKV_ERR_ALIGN;
  return launch_status(qkv::launch_pages_release(t, slots, keep_tokens, n, status, kPageStatus, stream));
}

size_t qkv_pages_reserve_scratch_bytes(int n, int max_new, int block_tokens) {
  if (n <= 0 || n > qkv::kReserveMax || max_new <= 0 || block_tokens <= 0) return 0;
  return 4 * qkv::reserve_scratch_ints(n, qkv::reserve_blocks(max_new, block_tokens));
}

int qkv_pages_reserve(int32_t* block_tables, int n_slots, int max_blocks, int block_tokens, int32_t* ref_counts,
                      int n_pages, const int32_t* slots, const int32_t* positions, const int32_t* n_new, int n,
                      int max_new, int32_t* status, const qkv_page_plane* planes, int n_planes, int32_t* scratch,
                      size_t scratch_bytes, hipStream_t stream) {
  const qkv::PageTables t{block_tables, ref_counts, n_slots, max_blocks, block_tokens, n_pages};
  int st = check_tables(t);
  if (st != QKV_OK) return st;
  qkv::PagePlanes pl{};
  st = take_planes(planes, n_planes, pl);
  if (st != QKV_OK) return st;
  if (n < 0 || max_new < 0) return QKV_ERR_INVALID;
  if (n > qkv::kReserveMax) return QKV_ERR_UNSUPPORTED;
  if (n == 0 || max_new == 0) return QKV_OK;
  if (max_new > (1 << 30) || (double)n * qkv::reserve_blocks(max_new, block_tokens) > (double)(1 << 28))
    return QKV_ERR_UNSUPPORTED;
  if (!slots || !positions || !n_new) return QKV_ERR_NULL;
  if (!scratch || scratch_bytes < qkv_pages_reserve_scratch_bytes(n, max_new, block_tokens)) return QKV_ERR_WORKSPACE;
  if (!aligned(slots, 4) || !aligned(positions, 4) || !aligned(n_new, 4) || !aligned(status, 4) || !aligned(scratch, 4))
    return QKV_ERR_ALIGN;
  return launch_status(
      qkv::launch_pages_reserve(t, slots, positions, n_new, n, max_new, status, kPageStatus, pl, scratch, stream));
}

int qkv_pages_copy(const qkv_page_plane* planes, int n_planes, int n_pages, const int32_t* pairs, int n,
                   hipStream_t stream) {
  qkv::PagePlanes pl{};
  const int st = take_planes(planes, n_planes, pl);
  if (st != QKV_OK) return st;
  if (n < 0 || n_pages <= 0) return QKV_ERR_INVALID;
  if (n == 0 || n_planes == 0) return QKV_OK;
  if (!pairs) return QKV_ERR_NULL;
  if (!aligned(pairs, 4)) return QKV_ERR_ALIGN;
  return launch_status(qkv::launch_pages_copy(pl, pairs, n, n_pages, stream));
}

int qkv_pages_compact(int32_t* block_tables, int n_slots, int max_blocks, int32_t* ref_counts, int n_pages,
                      int32_t* moved, int32_t* n_used, const qkv_page_plane* planes, int n_planes, int32_t* scratch,
                      size_t scratch_bytes, hipStream_t stream) {
  const qkv::PageTables t{block_tables, ref_counts, n_slots, max_blocks, 1, n_pages};
  int st = check_tables(t);
  if (st != QKV_OK) return st;
  qkv::PagePlanes pl{};
  st = take_planes(planes, n_planes, pl);
  if (st != QKV_OK) return st;
  if (!moved || !n_used) return QKV_ERR_NULL;
  if (!scratch || scratch_bytes < 4 * ((size_t)n_pages + 2)) return QKV_ERR_WORKSPACE;
  if (!aligned(moved, 4) || !aligned(n_used, 4) || !aligned(scratch, 4)) return QKV_ERR_ALIGN;
  return launch_status(qkv::launch_pages_compact(t, moved, n_used, pl, scratch, stream));
}

}  // extern "C"
