// qkv_launch.h -- host launchers of the gfx950 kernels (internal; the public
// surface is include/qkv.h).  Arguments are validated by qkv_api.cpp.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qkv {

// `wgs` workgroups over x and y: a dimension of a launch holds fewer than 2^32 threads (what is
// past them is dropped without an error).  A workgroup's number (below 2^32) is
// y * kGridX + x; those from `wgs` on have nothing to do.
constexpr uint32_t kGridX = 1u << 21;   // (of up to 1,024 threads)
inline dim3 grid_xy(long wgs) {
  return wgs <= kGridX ? dim3((unsigned)wgs) : dim3(kGridX, (unsigned)((wgs + kGridX - 1) / kGridX));
}

// Row mapping of a paged append: input block i (token i / blocks_per_row,
// slot token / n_tok, position positions[slot] + token % n_tok) goes to
// pool row block_tables[slot * max_blocks + pos / block_tokens] *
// block_tokens + pos % block_tokens; rows outside [0, pool_rows) are skipped.
struct PagedRows {
  const int32_t* block_tables;
  const int32_t* positions;
  int max_blocks, block_tokens, blocks_per_row, n_tok;
  long pool_rows;
};

// sc0/sc1 non-null: in0/in1 are DFK2 int8 rows with one fp16 scale per
// 128-element block (re-quantizing append)
hipError_t launch_tq3_append(const void* in0, void* out0, const void* in1, void* out1,
                             int n_blocks, int n_tensors, hipStream_t stream,
                             const PagedRows* paged = nullptr, const uint16_t* sc0 = nullptr,
                             const uint16_t* sc1 = nullptr);
hipError_t launch_tq3_dequant(const void* in, void* out, int n_blocks, hipStream_t stream);
hipError_t launch_q8_append(const void* in0, void* out0, const void* in1, void* out1,
                            int n_blocks, int n_tensors, hipStream_t stream,
                            const uint16_t* sc0 = nullptr, const uint16_t* sc1 = nullptr);
// DFK2 int8 rows (group-128 fp16 scales) to fp16; n_elems a multiple of 128
hipError_t launch_dfk2_dequant(const void* q, const uint16_t* sc, void* out, long n_elems,
                               hipStream_t stream);
hipError_t launch_q8_dequant(const void* in, void* out, int n_blocks, hipStream_t stream);
// Zero-fill of `bytes` (a multiple of 4) bytes by a kernel (graph-capture safe).
hipError_t launch_fill_zero(void* p, size_t bytes, hipStream_t stream);
hipError_t launch_ws_status(const void* workspace, int* status, int ok_value, int timeout_value,
                            hipStream_t stream);

// Token-row moves inside one slot of one layer's cache (kv_move.hip): row
// slot_row0 + to[i] := row slot_row0 + from[i] for i = 0..n-1, K and V.
constexpr int kMoveMax = 64;
struct MoveArgs {
  uint8_t* k;
  uint8_t* v;
  uint32_t k_row_bytes, v_row_bytes;   // multiples of 4
  long slot_row0;
  int n;
  int from[kMoveMax], to[kMoveMax];
};
hipError_t launch_kv_move(const MoveArgs& a, bool ordered, hipStream_t stream);

// Paged slot snapshot (gather) / restore (scatter), kv_move.hip.  Tensor t
// (0: K, 1: V) has rows of row_bytes[t] (a multiple of 4).
struct PageCopyArgs {
  uint8_t* pool[2];
  uint8_t* flat[2];
  uint32_t row_bytes[2];
  const int32_t* table;      // the slot's block-table row
  int max_blocks, block_tokens, n_rows, n_tensors;
  long pool_rows;
  bool aligned16;            // every pointer 16-byte aligned
};
hipError_t launch_kv_page_copy(const PageCopyArgs& a, bool scatter, hipStream_t stream);

// Block-sparse TQ3 verify (sparse_tq3.hip): K-pool signatures and the top-k
// block index.  Pools are fp16 [num_kv][stride][256].
struct KpoolArgs {
  const uint32_t* k;         // slot-base TQ3 key cache
  uint16_t* k_pool;
  uint16_t* k_pool_max;
  int num_kv, total_kv, blk_lo, cur_blocks, stride, bsn;
};
hipError_t launch_tq3_kpool(const KpoolArgs& a, hipStream_t stream);
struct BlockIndexArgs {
  const uint16_t* q;         // [sub_n][num_q][256]
  const uint16_t* k_pool;
  const uint16_t* k_pool_max;
  int32_t* block_index;      // [num_kv][sub_n_max][top_k]
  int num_q, num_kv, sub_n, sub_n_max, start_pos, top_k, bsn, n_blocks, stride;
  float beta;
  float inv_gqa;             // 1.0f / GQA (the reference's compile-time constant)
};
// scores: workspace of block_index_workspace_bytes (block scores [num_kv][sub_n][n_blocks])
hipError_t launch_block_index(const BlockIndexArgs& a, float* scores, hipStream_t stream);

// Chunked prefill over a TQ3 cache (prefill_tq3.hip).  Workspace pieces:
// kx  keys [num_kv][h_pad + n_pad][256] fp16: the history rows dequantized
//     exactly as the reference's bulk dequantization, padded to whole 64-row
//     tiles, then the chunk's own keys
// vt  values in 32-key tiles [num_kv][(h_pad + n_pad)/32][256 dims][32] fp16
// part_ml / part_o  key-split partials {m (log2 units), l} and o
//                   [n_split][n_tok][num_q] (x 256 for o)
struct PrefillArgs {
  const uint32_t* k_cache;   // slot-base TQ3 caches, rows 0 .. hist-1
  const uint32_t* v_cache;
  uint16_t* kx;
  uint16_t* vt;
  float* part_ml;
  float* part_o;
  int num_q, num_kv, start_pos, n_tok;
  int hist;                  // cache rows attended: start_pos, or start_pos + n_tok (verify)
  int h_pad;                 // hist rounded up to 64
  int n_pad;                 // chunk rows staged: n_tok rounded up to 64, 0 in verify mode
  int tok_groups;            // 32-token groups of an attention workgroup: 1 or 2
  int seg_tiles;             // most 32-key tiles of one attention workgroup
  int n_split;               // most key segments of a query row
  int from_cache;            // 1: the chunk's keys are cache rows too (verify)
  float scale_log2;
};
struct PrefillGeom {
  int n_pad, h_pad;
  int max_split;             // key segments per query row that the partial area holds
  size_t kx_off, vt_off, ml_off, o_off, total;
};
PrefillGeom prefill_geom(int num_q, int num_kv, int n_tok, int start_pos);
// Token groups and key segments of a call (a.hist, h_pad, n_pad, from_cache set)
// into a.tok_groups, a.seg_tiles, a.n_split <= max_split.
void prefill_schedule(PrefillArgs& a, int max_split);
hipError_t launch_prefill_tq3(const PrefillArgs& a, int max_split, int gqa, const uint16_t* q, const uint16_t* k,
                              const uint16_t* v, uint16_t* out, hipStream_t stream);

// Rotary positions (rope.hip).  Strides in elements between tokens; heads of a
// token are head_dim apart.
struct RopeArgs {
  const uint16_t* q;
  uint16_t* q_out;
  const uint16_t* k;
  uint16_t* k_out;
  const int32_t* positions;
  const uint64_t* turns;     // [rot / 2] fractions of a turn a position, 64-bit fixed point
  long q_stride, q_out_stride, k_stride, k_out_stride;
  float amplitude;
  int n_tok, num_q, num_k, head_dim, rot;
  int layout;                // 0: pairs (i, i + rot / 2), 1: (2i, 2i + 1)
  int inverse;
  int units;                 // set by the launcher
};
// wide: 16-byte accesses (rot and head_dim multiples of 16, pointers and strides aligned)
hipError_t launch_rope(RopeArgs a, bool wide, bool in_place, hipStream_t stream);

// Norms of heads with the rotation, and the gradient (norm_rope.hip).  dq, dk and their strides, the
// sums of the weights' gradients (q_dw, k_dw) and the partial sums are the gradient's alone.
constexpr int kNormMaxHead = 1024;
constexpr double kNormRows = 17179869184.0;   // of a call by a wave a row, four a workgroup, whose number is one of 32 bits
constexpr int kNormGradGroups = 768;   // workgroups of a gradient: the 3 that fit each CU
struct NormRopeArgs {
  const uint16_t* q;
  const uint16_t* dq;
  uint16_t* q_out;
  const uint16_t* k;
  const uint16_t* dk;
  uint16_t* k_out;
  const float* q_weight;     // [head_dim], nullptr: ones
  const float* k_weight;
  float* q_dw;               // [head_dim], nullptr: not wanted
  float* k_dw;
  float* partial;            // [groups][head_dim], nullptr: neither wanted
  const int32_t* positions;
  const uint64_t* turns;
  long q_stride, dq_stride, q_out_stride, k_stride, dk_stride, k_out_stride;
  float amplitude, eps;
  int n_tok, num_q, num_k, head_dim, rot, layout;
  int q_groups;              // workgroups of the queries' rows (set by the launcher)
};
// wide: 16-byte accesses, head_dim 16 times a power of two from 4 to 64, rot a multiple of 16
hipError_t launch_norm_rope(const NormRopeArgs& a, bool wide, hipStream_t stream);
hipError_t launch_norm_rope_grad(NormRopeArgs a, bool wide, int groups, hipStream_t stream);

// Append to the paged 8-bit cache (f8_codec.hip), K and with them the queries
// rotated where rot > 0.  rows: tokens the input tensors hold.
struct F8AppendArgs {
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* q;         // nullptr: no queries
  uint16_t* q_out;
  uint8_t* k_pool;
  uint8_t* v_pool;
  uint8_t* k_exp;
  uint8_t* v_exp;
  const int32_t* tables;     // [n_slots][max_blocks]
  const int32_t* starts;     // [n_slots + 1]
  const int32_t* positions;  // [n_slots]
  const uint64_t* turns;
  long k_stride, v_stride, q_stride, q_out_stride, rows, kv_wgs;
  float amplitude;
  int n_slots, max_tok, max_blocks, block_tokens, n_pages, num_q, num_kv, head_dim, rot, layout;
  int spans;                 // pages that a slot's new rows may touch (set by the launcher)
};
hipError_t launch_f8_append(F8AppendArgs a, hipStream_t stream);

// Attention over the paged 8-bit cache (attn_f8.hip).
constexpr int kMaxPosition = 1 << 30;   // of a paged 8-bit slot's first row
struct F8AttnArgs {
  const uint16_t* q;         // [rows][num_q][head_dim]
  uint16_t* out;
  const uint8_t* k_pool;     // [n_pages][block_tokens][num_kv][head_dim]
  const uint8_t* v_pool;
  const uint8_t* k_exp;      // [n_pages][num_kv]
  const uint8_t* v_exp;
  const int32_t* tables;
  const int32_t* starts;
  const int32_t* positions;
  int* counts;               // workspace, its first kJoinCounts ints: zero between calls
  int2* desc;                // workspace: [n_slots][num_kv] {parts, first record} of a row tile (few rows)
  int* cuts;                 // workspace, the same place: [groups][4] where each part begins, then
                             // the units of all heads (many rows)
  float* rec_ml;             // workspace: {m (log2 units), l} of a partial row
  float* rec_o;              // workspace: its unnormalised sums
  long rows;
  int num_q, num_kv, n_slots, max_tok, max_ctx, max_blocks, block_tokens, n_pages, window, sink;
  int from_tok, to_tok;      // the slots of this launch: those that own so many rows
  int slot_tiles;            // row tiles of a slot with max_tok tokens
  int rec_rows;              // rows of a record
  int groups;                // workgroups
  int gqa;                   // num_q / num_kv
  uint32_t bt_magic;         // floor(2^32 / block_tokens)
  uint32_t gqa_magic;        // the same of gqa, below 2^32
  float scale_log2;
};
// Workspaces begin with these counts, whatever the call's numbers, so that calls of different
// shapes can share one.
constexpr int kJoinCounts = 1024;
struct F8AttnPlan {
  bool many;                 // the kernel for more than 64 (token, head) rows a slot
  int row_tiles;             // 16-row tiles of the other one: 1, 2 or 4
  int slot_tiles, rec_rows, groups;
  bool join;                 // records joined in the launch
  bool merges;               // whether any row can be in several workgroups
  size_t ml_off, o_off, total;
};
F8AttnPlan f8_attn_plan(int num_q, int num_kv, int head_dim, int n_slots, long rows, int max_tok, int max_ctx);
// Tokens of a slot up to which it goes to a launch of its own kind beside the one for many rows
// (0: one launch for all).
int f8_attn_apart(int num_q, int num_kv, int head_dim, int n_slots, long rows, int max_tok, int max_ctx);
hipError_t launch_f8_attn(const F8AttnArgs& a, const F8AttnPlan& plan, int head_dim, hipStream_t stream);

// Attention weights of the keys of the paged 8-bit cache, accumulated (weigh_f8.hip).
constexpr int kWeighGroups = 768;                          // workgroups of the kernels for many rows, at most
constexpr size_t kWeighRec = 2 * kWeighGroups * 256 * 8;   // bytes of their records of rows, twice those of keys
constexpr long kWeighScores = 256l << 20;           // bytes of scores that a call may store
struct WeighArgs {
  const uint16_t* q;         // [rows][num_q][head_dim]
  const uint8_t* k_pool;
  const uint8_t* k_exp;
  float* weights;            // [n_pages][num_kv][block_tokens]
  const int32_t* tables;
  const int32_t* starts;
  const int32_t* positions;
  const int32_t* weighed;    // [n_slots] keys whose weights stand, nullptr: positions
  float* rec;                // workspace: {m, l} [rows of the launch][chunks], or of cut tiles (many rows)
  float* stat_m;             // workspace: m and 1 / l of the launch's rows
  float* stat_il;
  float* scores;             // workspace: [(slot, KV head) of the launch][score_pitch / 32][rows][32] (few rows)
  float* sums;               // workspace, the same place: of cut tiles (many rows)
  int groups;                // workgroups of the kernels for many rows
  int* cuts;                 // workspace: [kWeighGroups][4] where each part begins
  long rows, score_pitch;
  float scale_log2, decay;
  int num_q, num_kv, n_slots, max_tok, max_ctx, max_blocks, block_tokens, n_pages, window, sink;
  int gqa;
  uint32_t bt_magic, gqa_magic;   // as in F8AttnArgs
  // set by the launcher
  int from_tok, to_tok;      // the slots of a launch: those that own so many rows
  int slot0, heads;          // from here on, heads = slots * num_kv
  int local_tok;             // tokens of a slot in the workspace; 0: rows lie there as in q
  int chunk_keys, chunks;    // keys of a record, records of a row
  int per;                   // workgroups of a (slot, KV head)
};
struct WeighPlan {
  int few_tok;               // slots of up to so many tokens store their scores,
  int few_slots;             // so many slots at a time
  bool many;                 // whether there may be others
  int few_keys, few_chunks;
  long pitch;
  size_t stat_rows, rec_bytes, sum_bytes;
};
WeighPlan weigh_plan(int num_q, int num_kv, int n_slots, long rows, int max_tok, int max_ctx);
hipError_t launch_weigh(WeighArgs a, const WeighPlan& plan, int head_dim, hipStream_t stream);

// Eviction from the paged 8-bit cache (evict_f8.hip).
constexpr int kEvictBytes = 16384;   // codes of a chunk of rows, of each pool
constexpr int kEvictChain = 32;      // ints apart, on lines of their own
constexpr int kEvictHeld = 16384;    // rows of a slot that one workgroup chooses from
constexpr int kEvictStretch = 4096, kEvictBins = 2048;   // rows, digits of a workgroup of those for longer slots
struct EvictArgs {
  uint8_t* k_pool;
  uint8_t* v_pool;
  uint8_t* k_exp;
  uint8_t* v_exp;
  float* weights;            // [n_pages][num_kv][block_tokens]
  const int32_t* tables;
  const int32_t* lens;       // [n_slots] rows of a slot
  const int32_t* keep;       // [n_slots] rows that stay
  int32_t* kept;             // [n_slots][num_kv][max_keep]
  int* chains;               // workspace: [n_slots * num_kv][kEvictChain] chunks taken, rows to write (0: none)
  int* flags;                // workspace: [n_slots * num_kv][chunks] 1: read, 2: all before too
  uint32_t* found;           // workspace: [n_slots * num_kv][4] digits and what is needed, after the first and second
  int* above;                // workspace: [n_slots * num_kv][stretches] rows above the first two digits
  uint16_t* counts;          // workspace: [2][n_slots * num_kv][stretches][kEvictBins] of the digits, in turn
  int stretches;             // of max_ctx rows; 0: one workgroup a slot and KV head
  int n_slots, num_kv, max_ctx, max_keep, max_blocks, block_tokens, n_pages, sink, recent;
  int chunks;                // of max_keep rows
  uint32_t bt_magic;         // floor(2^32 / block_tokens)
};
hipError_t launch_evict(EvictArgs a, int head_dim, hipStream_t stream);

// Beam search's selection (beam.hip): rows = requests * beams.
constexpr int kMaxBeams = 64, kMaxTake = 64;
constexpr int kBeamGroups = 2048;   // workgroups of a call, and records of a request, below which a row
constexpr int kBeamRecords = 4096;  // is cut finer
struct BeamArgs {
  const void* logits;        // [rows][vocab], `stride` elements between rows
  const float* scores;       // [rows], -infinity: no beam
  const int32_t* done;       // [rows], nullptr: none
  int32_t* parents;          // [requests][take]
  int32_t* tokens;
  float* top;
  float* rec_x;              // workspace: [rows][segments][take] the largest logits of a segment
  int32_t* rec_at;           // and their tokens
  float* rec_sum;            // workspace: [rows][segments] {largest logit m, sum of e^(x - m)}
  long stride, rows;
  int beams, vocab, take, end_token;
  int segments;              // set by the launcher
};
struct BeamPlan {
  int words;                 // 16-byte words a thread holds
  int segments;              // workgroups of a row
};
// type 0: fp16, 1: fp32, 2: bf16
BeamPlan beam_plan(long rows, int beams, int vocab, int take, int type);
hipError_t launch_beam(BeamArgs a, const BeamPlan& plan, int type, hipStream_t stream);

// Pages of a cache (kv_pages.hip): tables [n_slots][max_blocks] with a negative
// entry where there is no page, ref_counts [n_pages] (0: free).
constexpr int kMaxPlanes = 128;
struct PagePlanes {
  uint8_t* base[kMaxPlanes];
  uint64_t bytes[kMaxPlanes];   // of a page
  int n;
};
struct PageTables {
  int32_t* tables;
  int32_t* refs;
  int n_slots, max_blocks, block_tokens, n_pages;
};
struct PageStatus {
  int ok, invalid, pages;
};
hipError_t launch_pages_fork(const PageTables& t, const int32_t* parents, const int32_t* children,
                             const int32_t* tokens, int n, int32_t* status, const PageStatus& codes,
                             hipStream_t stream);
hipError_t launch_pages_release(const PageTables& t, const int32_t* slots, const int32_t* keep, int n,
                                int32_t* status, const PageStatus& codes, hipStream_t stream);
constexpr int kReserveMax = 1024;   // slots of one reserve call
inline int reserve_blocks(int max_new, int block_tokens) {
  return (int)(((long)max_new + block_tokens - 2) / block_tokens + 1);
}
// scratch: reserve_scratch_ints(n, blocks) int32, the copied pairs [n][2] first
inline size_t reserve_scratch_ints(int n, int blocks) { return 3 * (size_t)n + 2 * (size_t)n * blocks; }
hipError_t launch_pages_reserve(const PageTables& t, const int32_t* slots, const int32_t* positions,
                                const int32_t* n_new, int n, int max_new, int32_t* status, const PageStatus& codes,
                                const PagePlanes& planes, int32_t* scratch, hipStream_t stream);
hipError_t launch_pages_copy(const PagePlanes& planes, const int32_t* pairs, int n, int n_pages, hipStream_t stream);
// Slots take over their parents' pages and rows of `states` (bytes: of a slot); n <= kReorderMax.
constexpr int kReorderMax = 1024;
hipError_t launch_pages_reorder(const PageTables& t, const int32_t* slots, const int32_t* parents,
                                const int32_t* tokens, int n, int32_t* status, const PageStatus& codes,
                                const PagePlanes& states, hipStream_t stream);
// scratch: n_pages + 2 int32
hipError_t launch_pages_compact(const PageTables& t, int32_t* moved, int32_t* n_used, const PagePlanes& planes,
                                int32_t* scratch, hipStream_t stream);

}  // namespace qkv
