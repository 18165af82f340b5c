// qkv_api_loop.cpp -- the C ABI of the operators around the paged 8-bit cache in a decoding loop: norms
// of heads with the rotation, weighing and evicting keys, beam selection and the reordering of
// slots (declared in include/qkv.h): argument checks, then launches on the caller's stream.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "qkv_api_checks.h"

namespace {

// Rows of a call: n_tok tokens of `heads` heads, `stride` elements apart
bool stride_ok(int n_tok, int heads, int head_dim, long stride) { return n_tok <= 1 || stride >= (long)heads * head_dim; }

int check_norm(int n_tok, int num_q, int num_k, int head_dim, int rot_dim, int layout, float eps) {
  if (n_tok < 0 || num_q < 0 || num_k < 0 || num_q + num_k == 0 || num_q > 1024 || num_k > 1024 || head_dim <= 0 ||
      rot_dim < 0 || rot_dim % 2 || rot_dim > head_dim || layout < 0 || layout > 1 || !(eps > 0.f) || !std::isfinite(eps))
    return QKV_ERR_INVALID;
  if (head_dim > qkv::kNormMaxHead) return QKV_ERR_UNSUPPORTED;
  return QKV_OK;
}

// 16-byte accesses of every row
bool norm_wide(int head_dim, int rot_dim) {
  const int lanes = head_dim / 16;
  return head_dim % 16 == 0 && rot_dim % 16 == 0 && lanes >= 4 && (lanes & (lanes - 1)) == 0;
}
bool wide_rows(const void* p, long stride) { return aligned(p, 16) && stride % 8 == 0; }

// Workgroups of a gradient, the queries' and the keys' (at least one of each)
int norm_grad_groups(int n_tok, int num_q, int num_k) {
  const double rows = (double)n_tok * (num_q + num_k);
  return (int)std::min((double)qkv::kNormGradGroups, std::max(2.0, rows / 16));
}

}  // namespace

extern "C" {

int qkv_norm_rope(const uint16_t* q, long q_stride, uint16_t* q_out, long q_out_stride, const float* q_weight,
                  const uint16_t* k, long k_stride, uint16_t* k_out, long k_out_stride, const float* k_weight,
                  float eps, const int32_t* positions, const uint64_t* turns, float amplitude, int n_tok, int num_q,
                  int num_k, int head_dim, int rot_dim, int layout, hipStream_t stream) {
  const int st = check_norm(n_tok, num_q, num_k, head_dim, rot_dim, layout, eps);
  if (st != QKV_OK) return st;
  if (n_tok == 0) return QKV_OK;
  if ((num_q && (!q || !q_out)) || (num_k && (!k || !k_out)) || (rot_dim && (!positions || !turns))) return QKV_ERR_NULL;
  if ((num_q && (!stride_ok(n_tok, num_q, head_dim, q_stride) || !stride_ok(n_tok, num_q, head_dim, q_out_stride))) ||
      (num_k && (!stride_ok(n_tok, num_k, head_dim, k_stride) || !stride_ok(n_tok, num_k, head_dim, k_out_stride))))
    return QKV_ERR_INVALID;
  if ((num_q && q == q_out && q_stride != q_out_stride) || (num_k && k == k_out && k_stride != k_out_stride))
    return QKV_ERR_INVALID;
  if (num_q && num_k && q_out == k_out) return QKV_ERR_INVALID;
  if ((num_q && (!aligned(q, 2) || !aligned(q_out, 2) || !aligned(q_weight, 4))) ||
      (num_k && (!aligned(k, 2) || !aligned(k_out, 2) || !aligned(k_weight, 4))) ||
      (rot_dim && (!aligned(positions, 4) || !aligned(turns, 8))))
    return QKV_ERR_ALIGN;
  if ((double)n_tok * (num_q + num_k) * head_dim / 256 > 2147483647.0) return QKV_ERR_UNSUPPORTED;
  qkv::NormRopeArgs a{};
  a.q = num_q ? q : nullptr;
  a.q_out = q_out;
  a.k = num_k ? k : nullptr;
  a.k_out = k_out;
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.positions = positions;
  a.turns = turns;
  a.q_stride = q_stride;
  a.q_out_stride = q_out_stride;
  a.k_stride = k_stride;
  a.k_out_stride = k_out_stride;
  a.amplitude = amplitude;
  a.eps = eps;
  a.n_tok = n_tok;
  a.num_q = num_q;
  a.num_k = num_k;
  a.head_dim = head_dim;
  a.rot = rot_dim;
  a.layout = layout;
  bool wide = norm_wide(head_dim, rot_dim);
  if (num_q) wide = wide && wide_rows(q, q_stride) && wide_rows(q_out, q_out_stride) && aligned(q_weight, 16);
  if (num_k) wide = wide && wide_rows(k, k_stride) && wide_rows(k_out, k_out_stride) && aligned(k_weight, 16);
  if (!wide && (double)n_tok * (num_q + num_k) > qkv::kNormRows) return QKV_ERR_UNSUPPORTED;
  return launch_status(qkv::launch_norm_rope(a, wide, stream));
}

size_t qkv_norm_rope_grad_workspace_bytes(int n_tok, int num_q, int num_k, int head_dim) {
  if (check_norm(n_tok, num_q, num_k, head_dim, 0, 0, 1.f) != QKV_OK) return 0;
  return (size_t)norm_grad_groups(n_tok, num_q, num_k) * head_dim * 4;
}

int qkv_norm_rope_grad(const uint16_t* q, long q_stride, const uint16_t* q_dy, long q_dy_stride, uint16_t* q_dx,
                       long q_dx_stride, const float* q_weight, float* q_dw, const uint16_t* k, long k_stride,
                       const uint16_t* k_dy, long k_dy_stride, uint16_t* k_dx, long k_dx_stride, const float* k_weight,
                       float* k_dw, float eps, const int32_t* positions, const uint64_t* turns, float amplitude,
                       int n_tok, int num_q, int num_k, int head_dim, int rot_dim, int layout, void* workspace,
                       size_t workspace_bytes, hipStream_t stream) {
  const int st = check_norm(n_tok, num_q, num_k, head_dim, rot_dim, layout, eps);
  if (st != QKV_OK) return st;
  if (!num_q) q_dw = nullptr;
  if (!num_k) k_dw = nullptr;
  const bool sums = q_dw || k_dw;
  if (n_tok == 0 && !sums) return QKV_OK;
  if (n_tok && ((num_q && (!q || !q_dy || !q_dx)) || (num_k && (!k || !k_dy || !k_dx)) ||
                (rot_dim && (!positions || !turns))))
    return QKV_ERR_NULL;
  auto strides = [&](int heads, long s) { return !heads || stride_ok(n_tok, heads, head_dim, s); };
  if (!strides(num_q, q_stride) || !strides(num_q, q_dy_stride) || !strides(num_q, q_dx_stride) ||
      !strides(num_k, k_stride) || !strides(num_k, k_dy_stride) || !strides(num_k, k_dx_stride))
    return QKV_ERR_INVALID;
  // in place of the rows or of their outputs' gradients, with the same stride
  auto places = [](const uint16_t* in, long s, const uint16_t* out, long so) { return in != out || s == so; };
  if (n_tok && ((num_q && (!places(q, q_stride, q_dx, q_dx_stride) || !places(q_dy, q_dy_stride, q_dx, q_dx_stride))) ||
                (num_k && (!places(k, k_stride, k_dx, k_dx_stride) || !places(k_dy, k_dy_stride, k_dx, k_dx_stride))) ||
                (num_q && num_k && q_dx == k_dx)))
    return QKV_ERR_INVALID;
  if ((q_dw && q_dw == k_dw)) return QKV_ERR_INVALID;
  if ((num_q && (!aligned(q, 2) || !aligned(q_dy, 2) || !aligned(q_dx, 2) || !aligned(q_weight, 4) || !aligned(q_dw, 4))) ||
      (num_k && (!aligned(k, 2) || !aligned(k_dy, 2) || !aligned(k_dx, 2) || !aligned(k_weight, 4) || !aligned(k_dw, 4))) ||
      (rot_dim && (!aligned(positions, 4) || !aligned(turns, 8))))
    return QKV_ERR_ALIGN;
  if ((double)n_tok * (num_q + num_k) * head_dim / 256 > 2147483647.0) return QKV_ERR_UNSUPPORTED;
  if (sums && (!workspace || workspace_bytes < qkv_norm_rope_grad_workspace_bytes(n_tok, num_q, num_k, head_dim)))
    return QKV_ERR_WORKSPACE;
  if (sums && !aligned(workspace, 4)) return QKV_ERR_ALIGN;
  qkv::NormRopeArgs a{};
  a.q = num_q ? q : nullptr;
  a.dq = q_dy;
  a.q_out = q_dx;
  a.k = num_k ? k : nullptr;
  a.dk = k_dy;
  a.k_out = k_dx;
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.q_dw = q_dw;
  a.k_dw = k_dw;
  a.partial = sums ? static_cast<float*>(workspace) : nullptr;
  a.positions = positions;
  a.turns = turns;
  a.q_stride = q_stride;
  a.dq_stride = q_dy_stride;
  a.q_out_stride = q_dx_stride;
  a.k_stride = k_stride;
  a.dk_stride = k_dy_stride;
  a.k_out_stride = k_dx_stride;
  a.amplitude = amplitude;
  a.eps = eps;
  a.n_tok = n_tok;
  a.num_q = num_q;
  a.num_k = num_k;
  a.head_dim = head_dim;
  a.rot = rot_dim;
  a.layout = layout;
  bool wide = norm_wide(head_dim, rot_dim);
  if (num_q)
    wide = wide && wide_rows(q, q_stride) && wide_rows(q_dy, q_dy_stride) && wide_rows(q_dx, q_dx_stride) && aligned(q_weight, 16);
  if (num_k)
    wide = wide && wide_rows(k, k_stride) && wide_rows(k_dy, k_dy_stride) && wide_rows(k_dx, k_dx_stride) && aligned(k_weight, 16);
  return launch_status(qkv::launch_norm_rope_grad(a, wide, norm_grad_groups(n_tok, num_q, num_k), stream));
}

static int check_weigh(int num_q, int num_kv, int head_dim, int n_slots, int n_rows, int max_tok, int max_ctx) {
  if (head_dim != 128 && head_dim != 256) return QKV_ERR_UNSUPPORTED;
  if (num_kv <= 0 || num_q <= 0 || num_q % num_kv != 0 || n_slots <= 0 || n_rows <= 0 || max_tok <= 0 || max_ctx <= 0)
    return QKV_ERR_INVALID;
  if (num_q / num_kv > 8 || num_q > 1024 || max_ctx > (1 << 30)) return QKV_ERR_UNSUPPORTED;
  // workgroups of a launch, rows of a slot and KV head, and steps of the line of all tiles (by rows, then by keys),
  // counted in 31 bits, a head's steps in 30
  const double gqa = num_q / num_kv, tok = std::min(max_tok, n_rows), rows = tok * gqa, heads = (double)n_slots * num_kv;
  const double row_tiles = std::min(n_slots * (rows / 256 + 1), n_rows * gqa / 256 + n_slots);
  const double by_rows = row_tiles * (max_ctx / 64.0 + 6), by_keys = (max_ctx / 256.0 + 1) * (n_rows * gqa / 32 + 6.0 * n_slots);
  if (heads * std::max(rows / 16 + 1, max_ctx / 128.0 + 1) > 2147480000.0 || rows > (double)(1 << 30) ||
      std::max(by_rows, by_keys) * std::max(num_kv, 2) > 2147480000.0)
    return QKV_ERR_UNSUPPORTED;
  return QKV_OK;
}

static size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }
constexpr size_t kWeighCuts = 16 * qkv::kWeighGroups;
static size_t weigh_total(const qkv::WeighPlan& x) {
  return kWeighCuts + 2 * round256(4 * x.stat_rows) + round256(x.rec_bytes) + round256(x.sum_bytes);
}

size_t qkv_weigh_f8_paged_workspace_bytes(int num_q, int num_kv, int head_dim, int n_slots, int n_rows, int max_tok,
                                          int max_ctx) {
  if (check_weigh(num_q, num_kv, head_dim, n_slots, n_rows, max_tok, max_ctx) != QKV_OK) return 0;
  if (max_tok > n_rows) max_tok = n_rows;
  const qkv::WeighPlan x = qkv::weigh_plan(num_q, num_kv, n_slots, n_rows, max_tok, max_ctx);
  // Calls with smaller numbers: their scores need at most kWeighScores bytes and at most those of up to 64 rows a
  // slot at this context, their records a 64th of it (8 bytes for 128 scores or more) and 8 bytes a row; the
  // other sizes grow with each number.
  const double pitch = (max_ctx + 31.0) / 32 * 32, tokens = std::min(64 / (num_q / num_kv), max_tok);
  const size_t few_rows = (size_t)((double)n_slots * tokens * num_q);
  const size_t most = (size_t)std::min((double)qkv::kWeighScores, (double)few_rows * pitch * 4);
  return kWeighCuts + 2 * round256(4 * std::max(x.stat_rows, few_rows)) + round256(std::max(x.rec_bytes, most / 64 + 8 * few_rows)) +
         round256(std::max(x.sum_bytes, most));
}

int qkv_weigh_f8_paged(const uint16_t* q, const uint8_t* k_pool, const uint8_t* k_exp, float* weights, int n_rows,
                       int num_q, int num_kv, int head_dim, int n_slots, int max_tok, int max_ctx,
                       const int32_t* block_tables, int max_blocks, int block_tokens, int n_pages, const int32_t* starts,
                       const int32_t* positions, const int32_t* weighed, float decay, float scale, int window_tok,
                       int sink_tok, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  int st = check_f8_pool(num_kv, head_dim, max_blocks, block_tokens, n_pages);
  if (st != QKV_OK) return st;
  if (n_rows == 0 || n_slots == 0 || max_tok == 0) return QKV_OK;
  st = check_weigh(num_q, num_kv, head_dim, n_slots, n_rows, max_tok, max_ctx);
  if (st != QKV_OK) return st;
  if (window_tok < 0 || sink_tok < 0 || !std::isfinite(decay)) return QKV_ERR_INVALID;
  if (!q || !k_pool || !k_exp || !weights || !block_tables || !starts || !positions) return QKV_ERR_NULL;
  if (!aligned(q, 16) || !aligned(k_pool, 16) || !aligned(weights, 4) || !aligned(block_tables, 4) || !aligned(starts, 4) ||
      !aligned(positions, 4) || !aligned(weighed, 4))
    return QKV_ERR_ALIGN;
  if (max_tok > n_rows) max_tok = n_rows;
  const qkv::WeighPlan x = qkv::weigh_plan(num_q, num_kv, n_slots, n_rows, max_tok, max_ctx);
  if (!workspace || workspace_bytes < weigh_total(x)) return QKV_ERR_WORKSPACE;
  if (!aligned(workspace, 256)) return QKV_ERR_ALIGN;
  qkv::WeighArgs a{};
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.q = q;
  a.k_pool = k_pool;
  a.k_exp = k_exp;
  a.weights = weights;
  a.tables = block_tables;
  a.starts = starts;
  a.positions = positions;
  a.weighed = weighed;
  const size_t stat = round256(4 * x.stat_rows);
  a.cuts = reinterpret_cast<int*>(ws);
  a.stat_m = reinterpret_cast<float*>(ws + kWeighCuts);
  a.stat_il = reinterpret_cast<float*>(ws + kWeighCuts + stat);
  a.rec = reinterpret_cast<float*>(ws + kWeighCuts + 2 * stat);
  a.scores = reinterpret_cast<float*>(ws + kWeighCuts + 2 * stat + round256(x.rec_bytes));
  a.sums = a.scores;   // (the one kind's launches are done before the other's)
  a.rows = n_rows;
  a.score_pitch = x.pitch;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.decay = decay;
  a.num_q = num_q;
  a.num_kv = num_kv;
  a.n_slots = n_slots;
  a.max_tok = max_tok;
  a.max_ctx = max_ctx;
  a.max_blocks = max_blocks;
  a.block_tokens = block_tokens;
  a.n_pages = n_pages;
  a.window = window_tok;
  a.sink = sink_tok < max_ctx ? sink_tok : max_ctx;
  a.gqa = num_q / num_kv;
  a.bt_magic = (uint32_t)((1ull << 32) / (uint64_t)block_tokens);
  a.gqa_magic = (uint32_t)std::min<uint64_t>((1ull << 32) / (uint64_t)a.gqa, 0xffffffffull);
  return launch_status(qkv::launch_weigh(a, x, head_dim, stream));
}

static int check_evict(int n_slots, int num_kv, int block_tokens, int max_ctx, int max_keep) {
  if (n_slots < 0 || num_kv <= 0 || block_tokens <= 0 || max_ctx < 0 || max_keep < 0) return QKV_ERR_INVALID;
  // chunks of all slots and heads are workgroups of 256 threads of one launch, stretches of 1,024
  const double chains = (double)n_slots * num_kv;
  if (max_ctx > (1 << 30) || max_keep > (1 << 30) || chains * (max_ctx / (double)qkv::kEvictStretch + 1) >= (double)(1 << 22) ||
      chains * (max_keep / 64 + 1.0) >= (double)(1 << 24))
    return QKV_ERR_UNSUPPORTED;
  return QKV_OK;
}

static int evict_stretches(int max_ctx) {
  return max_ctx <= qkv::kEvictHeld ? 0 : (max_ctx + qkv::kEvictStretch - 1) / qkv::kEvictStretch;
}

size_t qkv_evict_f8_paged_workspace_bytes(int n_slots, int num_kv, int block_tokens, int max_ctx, int max_keep) {
  if (n_slots == 0 || check_evict(n_slots, num_kv, block_tokens, max_ctx, max_keep) != QKV_OK) return 0;
  // by slot and KV head: chunks taken and rows to move, flags, and for long slots the digits found, counts above and
  // two of a digit
  const size_t each = 4 * qkv::kEvictChain + 4 * (size_t)(max_keep / 64 + 1) + 16, stretch = 4 + 2 * 2 * qkv::kEvictBins;
  return (size_t)n_slots * num_kv * (each + evict_stretches(max_ctx) * stretch);
}

int qkv_evict_f8_paged(uint8_t* k_pool, uint8_t* v_pool, uint8_t* k_exp, uint8_t* v_exp, float* weights, int n_slots,
                       int num_kv, int head_dim, int max_ctx, int max_keep, const int32_t* block_tables, int max_blocks,
                       int block_tokens, int n_pages, const int32_t* lens, const int32_t* keep, int sink_tok,
                       int recent_tok, int32_t* kept, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  int st = check_f8_pool(num_kv, head_dim, max_blocks, block_tokens, n_pages);
  if (st != QKV_OK) return st;
  st = check_evict(n_slots, num_kv, block_tokens, max_ctx, max_keep);
  if (st != QKV_OK) return st;
  if (sink_tok < 0 || recent_tok < 0) return QKV_ERR_INVALID;
  if (n_slots == 0 || max_keep == 0) return QKV_OK;
  if (!k_pool || !v_pool || !k_exp || !v_exp || !weights || !block_tables || !lens || !keep || !kept) return QKV_ERR_NULL;
  if (!aligned(k_pool, 16) || !aligned(v_pool, 16) || !aligned(weights, 4) || !aligned(block_tables, 4) ||
      !aligned(lens, 4) || !aligned(keep, 4) || !aligned(kept, 4))
    return QKV_ERR_ALIGN;
  if (!workspace || workspace_bytes < qkv_evict_f8_paged_workspace_bytes(n_slots, num_kv, block_tokens, max_ctx, max_keep))
    return QKV_ERR_WORKSPACE;
  if (!aligned(workspace, 4)) return QKV_ERR_ALIGN;
  qkv::EvictArgs a{};
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.k_exp = k_exp;
  a.v_exp = v_exp;
  a.weights = weights;
  a.tables = block_tables;
  a.lens = lens;
  a.keep = keep;
  a.kept = kept;
  a.chains = static_cast<int*>(workspace);
  const size_t chains = (size_t)n_slots * num_kv;
  a.stretches = evict_stretches(max_ctx);
  a.counts = reinterpret_cast<uint16_t*>(a.chains + qkv::kEvictChain * chains);
  a.found = reinterpret_cast<uint32_t*>(a.counts + 2 * chains * a.stretches * qkv::kEvictBins);
  a.above = reinterpret_cast<int*>(a.found + 4 * chains);
  a.flags = a.above + chains * a.stretches;
  a.n_slots = n_slots;
  a.num_kv = num_kv;
  a.max_ctx = max_ctx;
  a.max_keep = max_keep;
  a.max_blocks = max_blocks;
  a.block_tokens = block_tokens;
  a.n_pages = n_pages;
  a.sink = sink_tok;
  a.recent = recent_tok;
  const int rows = qkv::kEvictBytes / head_dim;
  a.chunks = (max_keep + rows - 1) / rows;
  a.bt_magic = (uint32_t)((1ull << 32) / (uint64_t)block_tokens);
  return launch_status(qkv::launch_evict(a, head_dim, stream));
}

static int check_beam(int n, int beams, int vocab, int take) {
  if (n < 0 || beams <= 0 || vocab <= 0 || take <= 0) return QKV_ERR_INVALID;
  // (beam and token of a request are one whole number of 31 bits; rows are workgroups of a launch)
  if (beams > qkv::kMaxBeams || take > qkv::kMaxTake || (double)beams * vocab > 2147483647.0 ||
      (double)n * beams > (double)(1 << 24))
    return QKV_ERR_UNSUPPORTED;
  return QKV_OK;
}

size_t qkv_beam_select_workspace_bytes(int n, int beams, int vocab, int take) {
  if (n <= 0 || check_beam(n, beams, vocab, take) != QKV_OK) return 0;
  // rows are cut finer only up to kBeamGroups segments in all: the coarsest cut's, or those
  const double coarse = (double)n * beams * ((vocab + 3.0) / (256 * 8 * 4) + 1);
  return (size_t)(std::max(coarse, (double)qkv::kBeamGroups) + 1) * 8 * (take + 1);
}

int qkv_beam_select(const void* logits, int logits_type, long stride, const float* scores, const int32_t* done,
                    int end_token, int n, int beams, int vocab, int take, int32_t* parents, int32_t* tokens,
                    float* top_scores, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  const int st = check_beam(n, beams, vocab, take);
  if (st != QKV_OK) return st;
  if (logits_type < QKV_LOGITS_F16 || logits_type > QKV_LOGITS_BF16) return QKV_ERR_INVALID;
  if (done && (end_token < 0 || end_token >= vocab)) return QKV_ERR_INVALID;
  if (n == 0) return QKV_OK;
  if ((double)n * beams > 1 && stride < vocab) return QKV_ERR_INVALID;
  if (!logits || !scores || !parents || !tokens || !top_scores) return QKV_ERR_NULL;
  if (!aligned(logits, logits_type == QKV_LOGITS_F32 ? 4 : 2) || !aligned(scores, 4) || !aligned(done, 4) ||
      !aligned(parents, 4) || !aligned(tokens, 4) || !aligned(top_scores, 4))
    return QKV_ERR_ALIGN;
  if (!workspace || workspace_bytes < qkv_beam_select_workspace_bytes(n, beams, vocab, take)) return QKV_ERR_WORKSPACE;
  if (!aligned(workspace, 8)) return QKV_ERR_ALIGN;
  qkv::BeamArgs a{};
  a.logits = logits;
  a.scores = scores;
  a.done = done;
  a.parents = parents;
  a.tokens = tokens;
  a.top = top_scores;
  a.stride = stride;
  a.rows = (long)n * beams;
  a.beams = beams;
  a.vocab = vocab;
  a.take = take;
  a.end_token = end_token;
  const qkv::BeamPlan plan = qkv::beam_plan(a.rows, beams, vocab, take, logits_type);
  const size_t segments = (size_t)a.rows * plan.segments;
  a.rec_sum = static_cast<float*>(workspace);
  a.rec_x = a.rec_sum + 2 * segments;
  a.rec_at = reinterpret_cast<int32_t*>(a.rec_x + segments * take);
  return launch_status(qkv::launch_beam(a, plan, logits_type, stream));
}

int qkv_pages_reorder(int32_t* block_tables, int n_slots, int max_blocks, int block_tokens, int32_t* ref_counts,
                      int n_pages, const int32_t* slots, const int32_t* parents, const int32_t* n_tokens, int n,
                      int32_t* status, const qkv_page_plane* states, int n_states, hipStream_t stream) {
  const qkv::PageTables t{block_tables, ref_counts, n_slots, max_blocks, block_tokens, n_pages};
  int st = check_tables(t);
  if (st != QKV_OK) return st;
  qkv::PagePlanes pl{};
  st = take_planes(states, n_states, pl);
  if (st != QKV_OK) return st;
  if (n < 0 || n > n_slots) return QKV_ERR_INVALID;
  if (n > qkv::kReorderMax) return QKV_ERR_UNSUPPORTED;
  if (n == 0) return QKV_OK;
  if (!slots || !parents || !n_tokens) return QKV_ERR_NULL;
  if (!aligned(slots, 4) || !aligned(parents, 4) || !aligned(n_tokens, 4) || !aligned(status, 4)) return QKV_ERR_ALIGN;
  return launch_status(qkv::launch_pages_reorder(t, slots, parents, n_tokens, n, status, kPageStatus, pl, stream));
}

}  // extern "C"
