// attn_f8.hip -- attention over the paged 8-bit cache (e4m3 codes, one power-of-two
// exponent per page and KV head): ragged batches of one token to whole prompts a slot.
//
//   o_t = sum_j w_j v_j / sum_j w_j,  w_j = 2^(scale log2(e) q_t . k_j - m)
//
// over the keys j that query t sees, in one pass: m is the reference maximum of the keys so
// far, and raising it rescales both sums.  Single tokens and verify blocks read 2 * head_dim
// bytes a key and KV head and are bound by HBM; prompts do 4 * head_dim operations a (head,
// visible pair) and are bound by the matrix cores.
//
// Rows.  The rows of a (slot, KV head) are its (token, query head of the group) pairs,
// row = token * gqa + head, so that a K/V tile read once serves the whole group.
// Operands are swapped: S^T = K Q^T and O^T = V^T P^T, so that a lane's scores of a
// row are exactly the key octet that it supplies as the second product's operand and
// the softmax statistics of a row stay in its lanes.  Codes are converted to fp16 with
// their exponent (exact: a stored value has 4 significant bits and lies in fp16's
// range); both products run on the fp16 matrix cores with fp32 sums.
//
// Work.  The key tiles of all row tiles, heads and slots form one line that is cut
// into equal parts, one per workgroup, so ragged lengths balance by themselves.  A
// row tile that lies in one part is stored as output; one that is cut leaves records
// (m, l, O) that the merge kernel joins.  A part has at most two cut ends, hence two
// records a workgroup.
#include <algorithm>
#include <type_traits>

#include "attn_common.h"
#include "qkv_device.h"
#include "qkv_launch.h"

namespace qkv {

namespace {

typedef float f16x_t __attribute__((ext_vector_type(16)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void glb_void;
typedef __attribute__((address_space(4))) const int32_t const_i32;   // (read by scalar loads)

// The weights are taken against a reference maximum that is raised only when a row's
// maximum passes it by more than this (log2 units): they stay below 2^12, inside
// fp16, and most tiles need no rescaling of the sums.
constexpr float kSlack = 12.0f;

__device__ __forceinline__ h2_t cvt2(uint32_t w, float scale, bool hi) {
  return hi ? __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true))
            : __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
}
__device__ __forceinline__ h8_t join8(h2_t a, h2_t b, h2_t c, h2_t d) {
  return h8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// l + the 8 rounded weights
__device__ __forceinline__ float add8(h8_t w, float l) {
  const h2_t one = {(_Float16)1.f, (_Float16)1.f};
#pragma unroll
  for (int i = 0; i < 4; i++) l = __builtin_amdgcn_fdot2(h2_t{w[2 * i], w[2 * i + 1]}, one, l, false);
  return l;
}
__device__ __forceinline__ float pow2f(uint32_t biased) { return __uint_as_float(biased << 23); }
__device__ __forceinline__ float max32(float x) {   // with the lane 32 away
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float max16(float x) {   // with the lane 16 away
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float sum32(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ float sum16(float x) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Block of a key and the key's row in it (bt_magic = floor(2^32 / block_tokens): the product's
// high half is the quotient or one less).
struct BlockRow {
  int b, row;
};
__device__ __forceinline__ BlockRow block_row(const F8AttnArgs& p, int key) {
  const uint32_t q = __umulhi((uint32_t)key, p.bt_magic), r = (uint32_t)key - q * (uint32_t)p.block_tokens;
  const bool more = r >= (uint32_t)p.block_tokens;
  return {(int)(more ? q + 1 : q), (int)(more ? r - (uint32_t)p.block_tokens : r)};
}

// Token of a (token, head) row x >= 0 (the same way; the compiler's division is five times as long)
__device__ __forceinline__ int token_of(const F8AttnArgs& p, int x) {
  const uint32_t q = __umulhi((uint32_t)x, p.gqa_magic), r = (uint32_t)x - q * (uint32_t)p.gqa;
  return (int)(r >= (uint32_t)p.gqa ? q + 1 : q);
}

// Inclusive sums over the lanes, none above `top`
__device__ __forceinline__ int scan64(int v, int top) {
  auto add = [&](int o) { v = min(v + o, top); };
  add(__builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));   // within rows of 16, from 1, 2, 4, 8 lanes below
  add(__builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));   // the row before, the half before
  add(__builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
  return v;
}

// A slot's tokens: rows t0 .. t0+n-1 of q at positions pos0 .. (n = 0: none, or not of this launch)
struct Slot {
  int t0, n, pos0;
};
__device__ __forceinline__ Slot slot_of(const F8AttnArgs& p, int s) {
  Slot x;
  x.t0 = min(max(p.starts[s], 0), (int)p.rows);
  x.n = min(min(max(p.starts[s + 1], x.t0), (int)p.rows) - x.t0, p.max_tok);
  x.pos0 = p.positions[s];
  if (x.pos0 < 0 || x.pos0 > kMaxPosition || x.n < p.from_tok || x.n > p.to_tok) x.n = 0;
  return x;
}

// The same for a slot that the whole wave asks for: by scalar loads, so that what follows from it
// stays out of the vector registers
__device__ __forceinline__ Slot slot_at(const F8AttnArgs& p, int s) {
  const const_i32 *starts = (const const_i32*)p.starts + s, *positions = (const const_i32*)p.positions + s;
  Slot x;
  x.t0 = min(max(starts[0], 0), (int)p.rows);
  x.n = min(min(max(starts[1], x.t0), (int)p.rows) - x.t0, p.max_tok);
  x.pos0 = positions[0];
  if (x.pos0 < 0 || x.pos0 > kMaxPosition || x.n < p.from_tok || x.n > p.to_tok) x.n = 0;
  return x;
}

// Row tile i of a slot, ROWS (token, head) rows each, over key tiles of KT keys: keys
// lo .. end-1 and below the sinks.  Tile v of `tiles` is key tile v below n_sink, then w0 on.
struct RowTile {
  int tiles, n_sink, w0;
  int end;              // keys that exist for the tile's last row
  int pos_lo, pos_hi;   // positions of the first and last row's tokens
  __device__ __forceinline__ int key0(int v, int kt) const { return (v < n_sink ? v : v - n_sink + w0) * kt; }
};
template <int ROWS, int KT>
__device__ __forceinline__ RowTile row_tile(const F8AttnArgs& p, const Slot& x, int i, int gqa) {
  RowTile r;
  const int rows = x.n * gqa;
  r.pos_lo = x.pos0 + token_of(p, i * ROWS);
  r.pos_hi = x.pos0 + token_of(p, min(rows, (i + 1) * ROWS) - 1);
  r.end = min(r.pos_hi + 1, p.max_ctx);
  r.w0 = p.window > 0 ? max(0, r.pos_lo - p.window + 1) / KT : 0;
  r.n_sink = p.window > 0 ? min((p.sink + KT - 1) / KT, r.w0) : 0;
  // (the window may lie past max_ctx: then the sinks alone; a tile past every key is masked)
  r.tiles = max(1, r.n_sink + max(0, (r.end + KT - 1) / KT - r.w0));
  return r;
}

// Where a workgroup's part begins: entry, and units of it before the part
struct Part {
  int entry, at;
};

// Sums stop at kLineMax: starts that are not in order can name the same rows many times, and the
// line of them all may pass 32 bits.
constexpr int kLineMax = (1 << 30) - 1;
__device__ __forceinline__ int add_units(int a, int b) { return min(a + b, kLineMax); }

template <int THREADS>
__device__ __forceinline__ int block_scan(int v, int* lds, int& sum) {   // inclusive
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  v = scan64(v, kLineMax);
  __syncthreads();
  if (lane == 63) lds[w] = v;
  __syncthreads();
  int before = 0;
  sum = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; i++) {
    if (i < w) before = add_units(before, lds[i]);
    sum = add_units(sum, lds[i]);
  }
  return add_units(v, before);
}

// The line of one head: the row tiles of the slots in order, ROWS rows and key tiles of KT keys,
// each LEAD units for what it costs beside its key tiles (queries, first loads, output) and one
// for each of those.  Walked THREADS slots at a time: their row tiles are counted, then taken up by as
// many threads as there are (most slots of a batch may hold none here).
template <int ROWS, int KT, int LEAD, int THREADS>
struct RowLine {
  const F8AttnArgs& p;
  int gqa;
  int *lds, *upto;             // THREADS / 64 and THREADS ints of LDS
  int entry, mine, inc;        // this thread's row tile of the last step (slot * slot_tiles + tile), its
                               // units and the line's up to its end
  bool one = true;             // the line is one step: what the registers hold

  template <class F>
  __device__ __forceinline__ void walk(F&& done) {   // done(units so far): whether to stop
    int base = 0;
    for (int s0 = 0; s0 < p.n_slots; s0 += THREADS) {
      const int s = s0 + (int)threadIdx.x;
      int n;
      const int tiles = s < p.n_slots ? (slot_of(p, s).n * gqa + ROWS - 1) / ROWS : 0;
      upto[threadIdx.x] = block_scan<THREADS>(tiles, lds, n);
      __syncthreads();
      n = __builtin_amdgcn_readfirstlane(n);
      for (int x0 = 0; x0 < n; x0 += THREADS) {
        const int x = x0 + (int)threadIdx.x;
        mine = 0;
        if (x < n) {
          int lo = 0, hi = THREADS - 1;   // the first slot whose tiles end past x
#pragma unroll
          for (int w = THREADS / 2; w; w >>= 1) {
            const int mid = (lo + hi) / 2;
            if (upto[mid] > x) hi = mid; else lo = mid + 1;
          }
          const int i = x - (lo ? upto[lo - 1] : 0);
          entry = (s0 + lo) * p.slot_tiles + i;
          mine = LEAD + row_tile<ROWS, KT>(p, slot_of(p, s0 + lo), i, gqa).tiles;
        }
        int sum;
        inc = add_units(base, block_scan<THREADS>(mine, lds, sum));
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
  // the row tile that holds unit u of the line (u < its length)
  __device__ __forceinline__ Part find(int u, int* found) {
    auto look = [&](int so_far) {
      if (u >= inc - mine && u < inc) {
        found[0] = entry;
        found[1] = u - (inc - mine);
      }
      return so_far > u;
    };
    if (one) look(0); else walk(look);
    __syncthreads();
    return {__builtin_amdgcn_readfirstlane(found[0]), __builtin_amdgcn_readfirstlane(found[1])};
  }
};
// Parts of the line: at most a workgroup's each and none empty, the first `more` of them one
// unit longer (the units of all heads stay below 2^31: the host sees to it).
struct Parts {
  int n, q, more;
  __device__ __forceinline__ Parts(int units, int groups) {
    n = min(units, groups);
    q = n > 0 ? units / n : 0;
    more = units - q * n;
  }
  __device__ __forceinline__ int begin(int g) const { return g * q + min(g, more); }
  __device__ __forceinline__ int of(int x) const {   // the part that holds unit x
    const int lo = more * (q + 1);
    return x < lo ? x / (q + 1) : more + (x - lo) / q;
  }
};

// The maximum that a record carries (l = 0: no key).  A sum that is no number, from a query that is
// not finite, is joined above every other and so reaches the output.
__device__ __forceinline__ float rec_max(float m, float l) { return l != l ? INFINITY : m; }

__device__ __forceinline__ bool sees(int key, int pos, int end, int window, int sink) {
  return key <= pos && key < end && (window <= 0 || key > pos - window || key < sink);
}

}  // namespace

// ---------------------------------------------------------------------------
// few rows: up to 16 (token, head) rows of a slot and KV head
// ---------------------------------------------------------------------------
// One row tile a slot; the line of units is held 64 slots at a time in the lanes of each
// wave (no LDS, no barrier ahead of the first loads of keys).
template <int ROWS, int KT, int PER>
struct SlotLine {
  const F8AttnArgs& p;
  int gqa, lane, base;   // lane l holds slot base + l
  Slot mine;
  int units, inc;

  __device__ __forceinline__ SlotLine(const F8AttnArgs& args, int g) : p(args), gqa(g), lane(threadIdx.x & 63), base(-1) {}
  __device__ __forceinline__ void load(int b) {
    if (b == base) return;
    base = b;
    mine = b + lane < p.n_slots ? slot_of(p, b + lane) : Slot{0, 0, 0};
    units = mine.n > 0 ? (row_tile<ROWS, KT>(p, mine, 0, gqa).tiles + PER - 1) / PER : 0;
    inc = scan64(units, 0x7fffffff);
  }
  // units of all slots
  __device__ __forceinline__ int total() {
    int t = 0;
    for (int b = 0; b < p.n_slots; b += 64) {
      load(b);
      t += __builtin_amdgcn_readlane(inc, 63);
    }
    return t;
  }
  // the slot (lane of the loaded ones) that holds unit u of the line, and the unit in it
  __device__ __forceinline__ int find(int u, int& at) {
    for (int b = 0;; b += 64) {
      load(b);
      const int n = __builtin_amdgcn_readlane(inc, 63);
      if (u < n || b + 64 >= p.n_slots) break;
      u -= n;
    }
    const int e = min(63, (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(inc > u) | 1ull << 63));
    at = u - (__builtin_amdgcn_readlane(inc, e) - __builtin_amdgcn_readlane(units, e));
    return e;
  }
  // the next slot with units after lane e (from the first one on again: `wrapped`)
  __device__ __forceinline__ int next(int e, bool& wrapped) {
    wrapped = false;
    uint64_t m = __builtin_amdgcn_ballot_w64(units > 0) & (e < 63 ? ~0ull << (e + 1) : 0ull);
    while (m == 0) {
      const int b = base + 64 < p.n_slots ? base + 64 : 0;
      if (b == 0) {
        if (wrapped) return 0;   // (none: see `rows` below)
        wrapped = true;
      }
      load(b);
      m = __builtin_amdgcn_ballot_w64(units > 0);
    }
    return __builtin_ctzll(m);
  }
  // units of the line ahead of lane e's slot (one load of lanes: at most 64 slots)
  __device__ __forceinline__ int before(int e) const {
    return __builtin_amdgcn_readlane(inc, e) - __builtin_amdgcn_readlane(units, e);
  }
  __device__ __forceinline__ Slot slot(int e) const {
    return {__builtin_amdgcn_readlane(mine.t0, e), __builtin_amdgcn_readlane(mine.n, e),
            __builtin_amdgcn_readlane(mine.pos0, e)};
  }
};

// The two 16-key halves of a 32-key tile: first key, pages (-1: none) and first rows in them.
struct Tile {
  int key0, pg[2], row[2];
};
__device__ __forceinline__ Tile tile_at(const F8AttnArgs& p, const const_i32* table, int key0, int end) {
  Tile t;
  t.key0 = key0;
#pragma unroll
  for (int hf = 0; hf < 2; hf++) {
    const int key = key0 + 16 * hf;
    const BlockRow x = block_row(p, key);
    const int pg = key < end && x.b < p.max_blocks ? table[x.b] : -1;
    t.pg[hf] = pg >= 0 && pg < p.n_pages ? pg : -1;
    t.row[hf] = x.row;
  }
  return t;
}

// Four waves, each with key tiles of its own (every fourth of the part's 32-key tiles), joined
// through LDS at the end: nothing is shared on the way, so a wave waits only for its
// own loads, and K, V of the next tile are in flight while this one is computed
// (16 KB a wave at head_dim 256; 128 KB a CU at two workgroups).  K rows are the A operand as
// loaded: lane l%16 is the key, and the group l/16 takes the same dims of K and Q.  V comes
// four keys by a run of dims, and byte permutes pair the keys ahead of the conversion.
// Bound by HBM: one slot at 131,072 keys, GQA 4, 4 KV heads of 256, 268 MB in 48 to 50 us (5.5 TB/s; a
// kernel that only reads reaches 6.4), 5 us of merge after it; 32 slots of 500 to 32,768 keys in
// 16-row pages of 128, 358 MB in 64 to 67 us.  Parts for 256, 768 or 1,024 workgroups were slower than
// for 512 (two a CU).
// JOIN: short contexts, whose records the last workgroup of a tile joins in this launch: there latency
// is all (a call at 700 keys 8.8 us, with the merge's launch 11.1 to 13.1; by one workgroup of eight
// waves a KV head 13.4).
constexpr int kJoinKeys = 1024, kJoinStep = 8;
constexpr int kCoherent = 1 | 16;   // sc0 | sc1: where every XCD sees it, as device-wide atomics go
template <int HD, bool JOIN>
__global__ __launch_bounds__(256, 2) void f8_few_kernel(F8AttnArgs p) {
  constexpr int KT = 32, ROWS = 16, W = 4, PER = 4, THREADS = 64 * W;
  constexpr int KW = HD / 64;        // 16-byte key loads of a lane and 16-key half
  constexpr int VD = HD / 64;        // value dwords of a lane and key
  constexpr int DB = HD / 16;        // 16-dim blocks of the output
  constexpr int PITCH = HD + 4;
  __shared__ float red[W * 16 * PITCH];
  __shared__ float ml[W][ROWS][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  const int gqa = p.gqa;

  const int recs = JOIN ? 2 * p.groups * p.rec_rows : 0;
  const __amdgpu_buffer_rsrc_t rec_ml = __builtin_amdgcn_make_buffer_rsrc(p.rec_ml, 0, recs * 8, kBufferRsrcWord3);
  const __amdgpu_buffer_rsrc_t rec_o = __builtin_amdgcn_make_buffer_rsrc(p.rec_o, 0, recs * HD * 4, kBufferRsrcWord3);

  SlotLine<ROWS, KT, PER> line(p, gqa);
  const int total = line.total();
  const Parts parts(total * p.num_kv, p.groups);
  const int grp = blockIdx.x;
  if (grp >= parts.n) return;
  int u = parts.begin(grp);
  const int u_end = parts.begin(grp + 1);
  int h = __builtin_amdgcn_readfirstlane(u / total), at;
  int e = line.find(u - h * total, at);
  bool first_seg = true;
  const uint32_t key_bytes = (uint32_t)p.num_kv * HD;
  const uint32_t k_off = m * key_bytes + 16 * g, v_off = 4 * g * key_bytes + m * (4 * VD);

  while (true) {
    const Slot sl = line.slot(e);
    const RowTile rt = row_tile<ROWS, KT>(p, sl, 0, gqa);
    const int units = (rt.tiles + PER - 1) / PER;
    const int n_u = min(units - at, u_end - u);
    const int rows = sl.n * gqa;
    if (rows <= 0 || n_u <= 0) return;   // (starts or positions that change under the call: no loop without end)
    const int v_end = min((at + n_u) * PER, rt.tiles);
    const const_i32* table = (const const_i32*)(p.tables + (long)(line.base + e) * p.max_blocks);
    // for the merge: the parts that hold the tile, and its first record
    if (!JOIN && at == 0 && tid == 0) {
      const int n = parts.of(u + units - 1) - grp + 1;
      p.desc[(line.base + e) * p.num_kv + h] = make_int2(n, 2 * grp + (first_seg ? 0 : 1));
    }

    u4_t kr[2][KW];
    uint32_t vr[8][VD];
    uint32_t ke[2], ve[2];
    auto load_k = [&](const Tile& t) {
#pragma unroll
      for (int hf = 0; hf < 2; hf++) {
        const long pg = max(t.pg[hf], 0);
        const uint8_t* base = p.k_pool + (pg * p.block_tokens + t.row[hf]) * key_bytes + (long)h * HD;
        ke[hf] = p.k_exp[pg * p.num_kv + h];
#pragma unroll
        for (int i = 0; i < KW; i++) kr[hf][i] = *reinterpret_cast<const u4_t*>(base + k_off + 64 * i);
      }
    };
    auto load_v = [&](const Tile& t) {
#pragma unroll
      for (int hf = 0; hf < 2; hf++) {
        const long pg = max(t.pg[hf], 0);
        const uint8_t* base = p.v_pool + (pg * p.block_tokens + t.row[hf]) * key_bytes + (long)h * HD;
        ve[hf] = p.v_exp[pg * p.num_kv + h];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          // (each byte is used once: past the caches; K's rows come in four pieces of a line)
          const uint8_t* src = base + (long)i * key_bytes + v_off;
          if constexpr (VD == 4) {
            const u4_t w = __builtin_nontemporal_load(reinterpret_cast<const u4_t*>(src));
#pragma unroll
            for (int d = 0; d < 4; d++) vr[4 * hf + i][d] = w[d];
          } else {
            const u2_t w = __builtin_nontemporal_load(reinterpret_cast<const u2_t*>(src));
#pragma unroll
            for (int d = 0; d < 2; d++) vr[4 * hf + i][d] = w[d];
          }
        }
      }
    };

    int v = at * PER + wave;
    Tile cur{}, nxt{};
    if (v < v_end) {
      cur = tile_at(p, table, rt.key0(v, KT), rt.end);
      load_k(cur);
      load_v(cur);
    }

    // ---- queries: row m, dims 64 i + 16 g + 8 half ..
    h8_t qf[KW][2];
    const int rc = min(m, rows - 1), tok = token_of(p, rc);
    const int pos_r = sl.pos0 + tok;
    {
      const uint16_t* src = p.q + ((long)(sl.t0 + tok) * p.num_q + h * gqa + (rc - tok * gqa)) * HD + 16 * g;
#pragma unroll
      for (int i = 0; i < KW; i++)
#pragma unroll
        for (int x = 0; x < 2; x++) qf[i][x] = *reinterpret_cast<const h8_t*>(src + 64 * i + 8 * x);
    }
    if (v + W < v_end) nxt = tile_at(p, table, rt.key0(v + W, KT), rt.end);

    f4_t acc[DB];
    float mx = -INFINITY, ls = 0.f;
#pragma unroll
    for (int d = 0; d < DB; d++) acc[d] = f4_t{0.f, 0.f, 0.f, 0.f};

    for (; v < v_end; v += W) {
      const bool more = v + W < v_end;
      // ---- scores: lane m's row, keys 16 hf + 4 g + i
      f4_t sc[2];
#pragma unroll
      for (int hf = 0; hf < 2; hf++) {
        const float f = pow2f(ke[hf]);
        f4_t a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KW; i++)
#pragma unroll
          for (int x = 0; x < 2; x++)
            a = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                join8(cvt2(kr[hf][i][2 * x], f, false), cvt2(kr[hf][i][2 * x], f, true),
                      cvt2(kr[hf][i][2 * x + 1], f, false), cvt2(kr[hf][i][2 * x + 1], f, true)),
                qf[i][x], a, 0, 0, 0);
        sc[hf] = a * p.scale_log2;
      }
      const bool whole = cur.pg[0] >= 0 && cur.pg[1] >= 0 && cur.key0 + KT - 1 <= rt.pos_lo && cur.key0 + KT <= rt.end &&
                         (p.window <= 0 || cur.key0 > rt.pos_hi - p.window || cur.key0 + KT <= p.sink);
      if (more) load_k(nxt);
      if (!whole) {
#pragma unroll
        for (int hf = 0; hf < 2; hf++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int key = cur.key0 + 16 * hf + 4 * g + i;
            const bool there = cur.pg[hf] >= 0 && key < rt.end;
            sc[hf][i] = there && sees(key, pos_r, rt.end, p.window, p.sink) ? sc[hf][i] : -INFINITY;
            // rows past the last key hold whatever the page held before
#pragma unroll
            for (int d = 0; d < VD; d++) vr[4 * hf + i][d] = there ? vr[4 * hf + i][d] : 0u;
          }
      }
      float t = sc[0][0];
#pragma unroll
      for (int i = 1; i < 8; i++) t = fmaxf(t, sc[i >> 2][i & 3]);
      t = max32(max16(t));
      if (__builtin_amdgcn_ballot_w64(t > mx + kSlack) != 0) {
        const float mn = fmaxf(mx, t);
        const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - mn);
        ls *= f;
#pragma unroll
        for (int d = 0; d < DB; d++) acc[d] *= f;
        mx = mn;
      }
      const float base = mx == -INFINITY ? 0.f : mx;
      // Weights as two fp16 parts: one part's rounding would put as much error into the output as
      // the output's own, and the second products hide beside the loads (128K keys: 53.5 and 53.9 us;
      // 17 to 64 rows keep one part, where they would cost 10%).
      h8_t pb, pl;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float w = __builtin_amdgcn_exp2f(sc[i >> 2][i & 3] - base);
        ls += w;
        pb[i] = (_Float16)w;
        pl[i] = (_Float16)(w - (float)pb[i]);
      }
      // ---- O^T += V^T P^T: dims m * HD/16 + 4 d + j
      // (an absent page's exponent is not one: zeros times it may be no number)
      const float v0 = pow2f(cur.pg[0] < 0 ? 127 : ve[0]), v1 = pow2f(cur.pg[1] < 0 ? 127 : ve[1]);
#pragma unroll
      for (int d = 0; d < VD; d++) {
        uint32_t w[4][2];   // key pairs x byte pairs
#pragma unroll
        for (int k = 0; k < 4; k++) {
          w[k][0] = __builtin_amdgcn_perm(vr[2 * k + 1][d], vr[2 * k][d], 0x05010400u);
          w[k][1] = __builtin_amdgcn_perm(vr[2 * k + 1][d], vr[2 * k][d], 0x07030602u);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const h8_t a = join8(cvt2(w[0][j >> 1], v0, j & 1), cvt2(w[1][j >> 1], v0, j & 1),
                               cvt2(w[2][j >> 1], v1, j & 1), cvt2(w[3][j >> 1], v1, j & 1));
          acc[4 * d + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pb, acc[4 * d + j], 0, 0, 0);
          acc[4 * d + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl, acc[4 * d + j], 0, 0, 0);
        }
      }
      if (more) {
        load_v(nxt);
        cur = nxt;
        if (v + 2 * W < v_end) nxt = tile_at(p, table, rt.key0(v + 2 * W, KT), rt.end);
      }
    }

    // ---- join the waves; lane m, group g holds dims (4 g + i) * HD/16 + d of row m
    const bool complete = n_u == units;
    const int rec = 2 * grp + (first_seg ? 0 : 1);
    ls = sum32(sum16(ls));
    if (g == 0) {
      ml[wave][m][0] = mx;
      ml[wave][m][1] = ls;
    }
    if (m < rows) {
      float* dst = red + (wave * 16 + m) * PITCH;
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int d = 0; d < DB; d += 4)
          *reinterpret_cast<f4_t*>(dst + (4 * g + i) * DB + d) =
              f4_t{acc[d][i], acc[d + 1][i], acc[d + 2][i], acc[d + 3][i]};
    }
    __syncthreads();
    for (int x = tid * 4; x < rows * HD; x += THREADS * 4) {
      const int r = x / HD, d = x - r * HD;
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < W; w++) M = fmaxf(M, ml[w][r][0]);
      f4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < W; w++) {
        const float f = ml[w][r][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[w][r][0] - M);
        L += ml[w][r][1] * f;
        o += f * *reinterpret_cast<const f4_t*>(red + (16 * w + r) * PITCH + d);
      }
      if (complete) {
        o *= L > 0.f ? 1.f / L : 0.f;
        const int t = token_of(p, r);
        *reinterpret_cast<u2_t*>(p.out + ((long)(sl.t0 + t) * p.num_q + h * gqa + (r - t * gqa)) * HD + d) =
            u2_t{f2h(o[0]) | (f2h(o[1]) << 16), f2h(o[2]) | (f2h(o[3]) << 16)};
      } else {
        const int at_r = rec * p.rec_rows + r;   // (at most 2 x 512 records of 16 rows)
        if constexpr (JOIN) {   // (to where every XCD sees it)
          __builtin_amdgcn_raw_buffer_store_b128(o, rec_o, (uint32_t)(at_r * HD + d) * 4, 0, kCoherent);
          if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(f2_t{rec_max(M, L), L}, rec_ml, (uint32_t)at_r * 8, 0, kCoherent);
        } else {
          *reinterpret_cast<f4_t*>(p.rec_o + (long)at_r * HD + d) = o;
          if (d == 0) *reinterpret_cast<f2_t*>(p.rec_ml + (long)at_r * 2) = f2_t{rec_max(M, L), L};
        }
      }
    }
    // ---- the last of a row tile's workgroups joins their records (the stores above have
    // completed when it is counted; a count goes back to zero with its last)
    if constexpr (JOIN) {
      if (!complete) {
        __shared__ int order;
        const int x0 = h * total + line.before(e), g0 = parts.of(x0), n = parts.of(x0 + units - 1) - g0 + 1;
        int* count = p.counts + (line.base + e) * p.num_kv + h;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) order = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (order == n - 1) {
          const int r0 = 2 * g0 + (parts.begin(g0) == x0 ? 0 : 1);
          // (a step's loads of all records and elements are under way at once: one element a thread in
          // a decode step, else two)
          auto join = [&](auto wide) {
            constexpr int kJoinWide = decltype(wide)::value;
            for (int x0 = tid * 4; x0 < rows * HD; x0 += kJoinWide * THREADS * 4) {
              float M[kJoinWide], L[kJoinWide];
              f4_t o[kJoinWide];
#pragma unroll
              for (int b = 0; b < kJoinWide; b++) {
                M[b] = -INFINITY;
                L[b] = 0.f;
                o[b] = f4_t{0.f, 0.f, 0.f, 0.f};
              }
              for (int i0 = 0; i0 < n; i0 += kJoinStep) {
                f2_t ml_r[kJoinWide][kJoinStep];
                f4_t ov[kJoinWide][kJoinStep];
#pragma unroll
                for (int b = 0; b < kJoinWide; b++)
#pragma unroll
                  for (int i = 0; i < kJoinStep; i++) {
                    const int x = min(x0 + b * THREADS * 4, rows * HD - 4), k = min(i0 + i, n - 1);
                    const int at_r = (k == 0 ? r0 : 2 * (g0 + k)) * p.rec_rows + x / HD;
                    ml_r[b][i] = __builtin_amdgcn_raw_buffer_load_b64(rec_ml, (uint32_t)at_r * 8, 0, kCoherent);
                    ov[b][i] = __builtin_amdgcn_raw_buffer_load_b128(rec_o, (uint32_t)(at_r * HD + x % HD) * 4, 0, kCoherent);
                  }
#pragma unroll
                for (int b = 0; b < kJoinWide; b++) {
                  float mn = M[b];
#pragma unroll
                  for (int i = 0; i < kJoinStep; i++) {
                    if (i0 + i >= n) ml_r[b][i][1] = 0.f;
                    if (ml_r[b][i][1] != 0.f) mn = fmaxf(mn, ml_r[b][i][0]);
                  }
                  if (mn == -INFINITY) continue;   // no key so far
                  const float f = __builtin_amdgcn_exp2f(M[b] - mn);
                  M[b] = mn;
                  L[b] *= f;
                  o[b] *= f;
#pragma unroll
                  for (int i = 0; i < kJoinStep; i++)
                    if (ml_r[b][i][1] != 0.f) {
                      const float w = __builtin_amdgcn_exp2f(ml_r[b][i][0] - mn);
                      L[b] += w * ml_r[b][i][1];
                      o[b] += w * ov[b][i];
                    }
                }
              }
#pragma unroll
              for (int b = 0; b < kJoinWide; b++) {
                const int x = x0 + b * THREADS * 4;
                if (x >= rows * HD) break;
                const int r = x / HD, d = x - r * HD, t = token_of(p, r);
                const f4_t y = o[b] * (L[b] > 0.f ? 1.f / L[b] : 0.f);
                *reinterpret_cast<u2_t*>(p.out + ((long)(sl.t0 + t) * p.num_q + h * gqa + (r - t * gqa)) * HD + d) =
                    u2_t{f2h(y[0]) | (f2h(y[1]) << 16), f2h(y[2]) | (f2h(y[3]) << 16)};
              }
            }
          };
          if (rows * HD <= THREADS * 4) join(std::integral_constant<int, 1>{});
          else join(std::integral_constant<int, 2>{});
          if (tid == 0) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
      }
    }
    u += n_u;
    if (u >= u_end) break;
    __syncthreads();   // (the next segment's waves write the same LDS)
    first_seg = false;
    at = 0;
    bool wrapped;
    e = line.next(e, wrapped);
    if (wrapped) h++;
  }
}

// 17 to 64 rows: waves of 32 rows on the 32x32 matrix instruction, RG of them side by
// side on the same keys (the second's loads meet the first's lines in the caches), 4 / RG
// key streams.  Otherwise as above: lane l%32 is the key of K's operand and takes 16 of
// every 32 dims; V comes by runs of HD/32 dims, and output block d has dims HD/32 * m + d.
// At head_dim 256 one wave a SIMD holds the sums, so the codes of two tiles ahead wait in LDS,
// loaded there past the registers (32 KB a wave; with one tile ahead in registers 93 against 83 us)
// and past the caches (RG = 1: every byte is used once).  At 128 two workgroups fit a CU (9 tokens, GQA
// 4, at 131,072 keys: 49 against 60 us with one).  K's 16-byte chunks are permuted within a row by
// the row's number, which keeps its reads on distinct banks.  Up to 32 rows bound by HBM: four slots of
// 5 to 8 tokens, GQA 4, at 32K to 64K keys, 403 MB in 80 us (5.0 TB/s).  Beyond, by one wave's chain
// of scores, softmax and values: 16 tokens at 131,072 keys, 268 MB, 95 us (8 tokens 65; one wave with
// both row groups needs more registers than there are).
template <int HD, int RG>
__global__ __launch_bounds__(256, HD == 128 ? 2 : 1) void f8_mid_kernel(F8AttnArgs p) {
  constexpr int KT = 32, ROWS = 32 * RG, KG = 4 / RG, PER = KG, THREADS = 256;
  constexpr int KW = HD / 32;        // 16-byte key loads of a lane
  constexpr int DB = HD / 32;        // 32-dim blocks of the output, value bytes of a lane and key
  constexpr int VD = DB / 4;         // value dwords of a lane and key
  constexpr int PITCH = HD + 4;
  constexpr int TB = KT * HD;        // bytes of a tile's K or V codes
  constexpr int RL = 1024 / HD;      // rows of a 1 KB load
  __shared__ __align__(16) union {
    uint8_t ring[4][2][2][TB];       // wave, tile parity, K / V
    float red[4 * 32 * PITCH];       // (after the last tile)
  } sm;
  float* red = sm.red;
  __shared__ float ml[KG][ROWS][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hh = lane >> 5, rg = wave % RG, kg = wave / RG;
  const int gqa = p.gqa;

  SlotLine<ROWS, KT, PER> line(p, gqa);
  const int total = line.total();
  const Parts parts(total * p.num_kv, p.groups);
  const int grp = blockIdx.x;
  if (grp >= parts.n) return;
  int u = parts.begin(grp);
  const int u_end = parts.begin(grp + 1);
  int h = __builtin_amdgcn_readfirstlane(u / total), at;
  int e = line.find(u - h * total, at);
  bool first_seg = true;
  const uint32_t key_bytes = (uint32_t)p.num_kv * HD;
  // a load's lane: row lane / (HD/16), its chunk permuted by the row (K) or in place (V)
  const int ld_row = lane / (HD / 16), ld_chunk = lane % (HD / 16);
  const uint32_t v_off = ld_row * key_bytes + ld_chunk * 16;

  while (true) {
    const Slot sl = line.slot(e);
    const RowTile rt = row_tile<ROWS, KT>(p, sl, 0, gqa);
    const int units = (rt.tiles + PER - 1) / PER;
    const int n_u = min(units - at, u_end - u);
    const int rows = sl.n * gqa;
    if (rows <= 0 || n_u <= 0) return;   // (starts or positions that change under the call: no loop without end)
    // a wave without rows loads nothing (the others wait for nobody)
    const int v_end = 32 * rg < rows ? min((at + n_u) * PER, rt.tiles) : 0;
    const const_i32* table = (const const_i32*)(p.tables + (long)(line.base + e) * p.max_blocks);
    // for the merge: the parts that hold the tile, and its first record
    if (at == 0 && tid == 0) {
      const int n = parts.of(u + units - 1) - grp + 1;
      p.desc[(line.base + e) * p.num_kv + h] = make_int2(n, 2 * grp + (first_seg ? 0 : 1));
    }

    uint8_t (*ring)[2][TB] = sm.ring[wave];
    uint32_t ke[2][2], ve[2][2];     // exponents, by parity and half
    auto load = [&](const Tile& t, int par) {
#pragma unroll
      for (int hf = 0; hf < 2; hf++) {
        const long pg = max(t.pg[hf], 0), from = (pg * p.block_tokens + t.row[hf]) * key_bytes + (long)h * HD;
#pragma unroll
        for (int l = 0; l < 16 / RL; l++) {
          const int r0 = l * RL;     // first row of the load, in the half
          const uint32_t k_off = ld_row * key_bytes + ((ld_chunk ^ ((r0 + ld_row) & (HD / 16 - 1))) * 16);
          const int to = (16 * hf + r0) * HD;
          __builtin_amdgcn_global_load_lds((glb_void*)(p.k_pool + from + (long)r0 * key_bytes + k_off), (lds_void*)(ring[par][0] + to), 16, 0, RG == 1 ? 2 : 0);
          __builtin_amdgcn_global_load_lds((glb_void*)(p.v_pool + from + (long)r0 * key_bytes + v_off), (lds_void*)(ring[par][1] + to), 16, 0, RG == 1 ? 2 : 0);
        }
        ke[par][hf] = p.k_exp[pg * p.num_kv + h];
        ve[par][hf] = p.v_exp[pg * p.num_kv + h];
      }
    };

    int v = at * PER + kg;
    Tile cur{}, nxt{}, far{};        // tiles v, v + PER (both loaded) and v + 2 PER
    if (v < v_end) {
      cur = tile_at(p, table, rt.key0(v, KT), rt.end);
      load(cur, 0);
    }
    if (v + PER < v_end) {
      nxt = tile_at(p, table, rt.key0(v + PER, KT), rt.end);
      load(nxt, 1);
    }
    // ---- queries: row c of the wave, dims 32 i + 16 hh + 8 x ..
    h8_t qf[KW][2];
    const int rc = min(32 * rg + c, rows - 1), tok = token_of(p, rc);
    const int pos_r = sl.pos0 + tok;
    {
      const uint16_t* src = p.q + ((long)(sl.t0 + tok) * p.num_q + h * gqa + (rc - tok * gqa)) * HD + 16 * hh;
#pragma unroll
      for (int i = 0; i < KW; i++)
#pragma unroll
        for (int x = 0; x < 2; x++) qf[i][x] = *reinterpret_cast<const h8_t*>(src + 32 * i + 8 * x);
    }
    if (v + 2 * PER < v_end) far = tile_at(p, table, rt.key0(v + 2 * PER, KT), rt.end);

    f16x_t acc[DB];
    float mx = -INFINITY, ls = 0.f;
#pragma unroll
    for (int d = 0; d < DB; d++) acc[d] = f16x_t{};

    auto step = [&](auto parity) {
      constexpr int P = decltype(parity)::value;
      const bool more = v + PER < v_end;
      // this tile's codes have landed; the next one's (all newer) may be under way
      if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * 32 / RL + 4) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      const uint8_t* kt = ring[P][0] + c * HD;
      const uint8_t* vt = ring[P][1] + 4 * hh * HD + c * DB;
      // ---- scores: lane c's row, keys 8 (x / 4) + 4 hh + x % 4
      f16x_t sc = f16x_t{};
      const float f = pow2f(c < 16 ? ke[P][0] : ke[P][1]);
#pragma unroll
      for (int i = 0; i < KW; i++) {
        const u4_t kr = *reinterpret_cast<const u4_t*>(kt + (((2 * i + hh) ^ (c & (HD / 16 - 1))) * 16));
#pragma unroll
        for (int x = 0; x < 2; x++)
          sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(
              join8(cvt2(kr[2 * x], f, false), cvt2(kr[2 * x], f, true), cvt2(kr[2 * x + 1], f, false),
                    cvt2(kr[2 * x + 1], f, true)),
              qf[i][x], sc, 0, 0, 0);
      }
      uint32_t vr[16][VD];           // keys 16 hf + 8 a + 4 hh + i
#pragma unroll
      for (int x = 0; x < 16; x++) {
        const uint8_t* src = vt + (8 * (x >> 2) + (x & 3)) * HD;
        if constexpr (VD == 2) {
          const u2_t w = *reinterpret_cast<const u2_t*>(src);
          vr[x][0] = w[0];
          vr[x][1] = w[1];
        } else {
          vr[x][0] = *reinterpret_cast<const uint32_t*>(src);
        }
      }
      sc *= p.scale_log2;
      const bool whole = cur.pg[0] >= 0 && cur.pg[1] >= 0 && cur.key0 + KT - 1 <= rt.pos_lo && cur.key0 + KT <= rt.end &&
                         (p.window <= 0 || cur.key0 > rt.pos_hi - p.window || cur.key0 + KT <= p.sink);
      if (!whole) {
#pragma unroll
        for (int x = 0; x < 16; x++) {
          const int key = cur.key0 + 8 * (x >> 2) + 4 * hh + (x & 3);
          const bool there = cur.pg[x >> 3] >= 0 && key < rt.end;
          sc[x] = there && sees(key, pos_r, rt.end, p.window, p.sink) ? sc[x] : -INFINITY;
          // rows past the last key hold whatever the page held before
#pragma unroll
          for (int d = 0; d < VD; d++) vr[x][d] = there ? vr[x][d] : 0u;
        }
      }
      float t = sc[0];
#pragma unroll
      for (int x = 1; x < 16; x++) t = fmaxf(t, sc[x]);
      t = max32(t);
      if (__builtin_amdgcn_ballot_w64(t > mx + kSlack) != 0) {
        const float mn = fmaxf(mx, t);
        const float r = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - mn);
        ls *= r;
#pragma unroll
        for (int d = 0; d < DB; d++) acc[d] *= r;
        mx = mn;
      }
      const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int hf = 0; hf < 2; hf++) {
        h8_t pb;
#pragma unroll
        for (int i = 0; i < 8; i++) pb[i] = (_Float16)__builtin_amdgcn_exp2f(sc[8 * hf + i] - base);
        ls = add8(pb, ls);
        const float vf = pow2f(cur.pg[hf] < 0 ? 127 : ve[P][hf]);
#pragma unroll
        for (int d = 0; d < VD; d++) {
          uint32_t w[4][2];   // key pairs x byte pairs
#pragma unroll
          for (int k = 0; k < 4; k++) {
            w[k][0] = __builtin_amdgcn_perm(vr[8 * hf + 2 * k + 1][d], vr[8 * hf + 2 * k][d], 0x05010400u);
            w[k][1] = __builtin_amdgcn_perm(vr[8 * hf + 2 * k + 1][d], vr[8 * hf + 2 * k][d], 0x07030602u);
          }
#pragma unroll
          for (int j = 0; j < 4; j++)
            acc[4 * d + j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                join8(cvt2(w[0][j >> 1], vf, j & 1), cvt2(w[1][j >> 1], vf, j & 1), cvt2(w[2][j >> 1], vf, j & 1),
                      cvt2(w[3][j >> 1], vf, j & 1)),
                pb, acc[4 * d + j], 0, 0, 0);
        }
      }
      // (every read of this tile's codes is done: its registers have been used)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (v + 2 * PER < v_end) load(far, P);
      cur = nxt;
      nxt = far;
      if (v + 3 * PER < v_end) far = tile_at(p, table, rt.key0(v + 3 * PER, KT), rt.end);
      v += PER;
    };
    while (v < v_end) {
      step(std::integral_constant<int, 0>{});
      if (v < v_end) step(std::integral_constant<int, 1>{});
    }

    // ---- join the streams; lane c holds dims DB * (8 (x / 4) + 4 hh + x % 4) + d of row c
    const bool complete = n_u == units;
    const int rec = 2 * grp + (first_seg ? 0 : 1);
    ls = sum32(ls);
    __syncthreads();   // (the ring is done with)
    if (hh == 0) {
      ml[kg][32 * rg + c][0] = mx;
      ml[kg][32 * rg + c][1] = ls;
    }
    if (32 * rg + c < rows) {
      float* dst = red + (kg * ROWS + 32 * rg + c) * PITCH;
#pragma unroll
      for (int x = 0; x < 16; x++)
#pragma unroll
        for (int d = 0; d < DB; d += 4)
          *reinterpret_cast<f4_t*>(dst + DB * (8 * (x >> 2) + 4 * hh + (x & 3)) + d) =
              f4_t{acc[d][x], acc[d + 1][x], acc[d + 2][x], acc[d + 3][x]};
    }
    __syncthreads();
    for (int x = tid * 4; x < rows * HD; x += THREADS * 4) {
      const int r = x / HD, d = x - r * HD;
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < KG; w++) M = fmaxf(M, ml[w][r][0]);
      f4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < KG; w++) {
        const float fw = ml[w][r][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[w][r][0] - M);
        L += ml[w][r][1] * fw;
        o += fw * *reinterpret_cast<const f4_t*>(red + (w * ROWS + r) * PITCH + d);
      }
      if (complete) {
        o *= L > 0.f ? 1.f / L : 0.f;
        const int t = token_of(p, r);
        *reinterpret_cast<u2_t*>(p.out + ((long)(sl.t0 + t) * p.num_q + h * gqa + (r - t * gqa)) * HD + d) =
            u2_t{f2h(o[0]) | (f2h(o[1]) << 16), f2h(o[2]) | (f2h(o[3]) << 16)};
      } else {
        *reinterpret_cast<f4_t*>(p.rec_o + ((long)rec * p.rec_rows + r) * HD + d) = o;
        if (d == 0) *reinterpret_cast<f2_t*>(p.rec_ml + ((long)rec * p.rec_rows + r) * 2) = f2_t{rec_max(M, L), L};
      }
    }
    u += n_u;
    if (u >= u_end) break;
    __syncthreads();   // (the next segment's waves write the same LDS)
    first_seg = false;
    at = 0;
    bool wrapped;
    e = line.next(e, wrapped);
    if (wrapped) h++;
  }
}

// ---------------------------------------------------------------------------
// many rows: prompts and chunks
// ---------------------------------------------------------------------------
// Eight waves of 32 rows share fp16 K and V tiles in LDS.  The codes of the tile after
// next go from memory straight to LDS (no registers: the sums and queries of a wave fill
// three quarters of them); the workgroup converts the next tile's once for all rows, each
// wave the rows that it loaded itself, so only its own loads are waited for.  V is stored
// by dim, four keys to 8 bytes, in the order that the scores' lanes hold them.  Pads
// keep 16-byte reads of 16 lanes on distinct banks, at constant offsets of one address.
// At head_dim 128 a tile is two halves of 32 keys, both scored before the weights.  All waves convert
// ahead of a tile's scores: one of each SIMD behind its values was slower (1,112 against 1,070 us
// below), and so were two workgroups of four waves a CU.
// Weights are rounded once to fp16 (2^-11 of a weight; their sum is that of the rounded ones), which
// puts the output's error against 64 bits at 2.5e-4 to 2.9e-4, beside 2.1e-4 of its own rounding: two
// parts, as the kernel for few rows has, take 1,347 against 1,023 us below and 191 against 147.
// Bound by the matrix cores at 2,048 tokens over 32,000 keys, GQA 4, 4 KV heads of 256: 1,108 GFLOP in
// 1,008 to 1,110 us (boxes differ), 1.0 to 1.10 PFLOP/s (a library product of fp16 matrices: 1.19; the
// conversion of tiles takes about a quarter).  Short prompts pay 8 to 11 us a row tile before its first
// product and after its last: six of 150 to 4,000 tokens, GQA 8, 128, window 1,500: 88 GFLOP in 145 to
// 157 us.

// A row tile's cost beside its key tiles, in tiles (measured to its first product and from its last:
// 11 us against 2.1 a tile at head_dim 256, 8 against 2.6 at 128; and a part that begins inside a row
// tile pays it too).  Geometric mean over 44 batches of prompts of 300 to 8,000 tokens, the loop as
// it then was: 98.7 us at 4, 95.5 at 6, 93.9 at 8, 92.6 at 10 and 5; now 90.3 to 91.1 anywhere
// between 8 and 4 and 12 and 6.
template <int HD>
constexpr int kLead = HD == 256 ? 10 : 5;

template <int HD>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void f8_many_kernel(F8AttnArgs p) {
  constexpr int WAVES = 8, ROWS = 32 * WAVES, THREADS = 64 * WAVES, LEAD = kLead<HD>;
  constexpr int KT = 8192 / HD;              // 32 or 64 keys: 8 KB of codes
  constexpr int KH = KT / 32;                // 32-key halves
  constexpr int WK = KT / WAVES;             // keys that a wave loads and converts
  constexpr int LPR = HD / 16;               // lanes of a key row's load
  constexpr int VP = KT * 2;                 // bytes of a dim's values
  constexpr int VPAD = KT == 32 ? 4 : 2;     // dims per 16-byte pad
  constexpr int KP = HD * 2 + 16;            // bytes of a key's row
  constexpr int KB = KT * KP, VB = HD * VP + HD / VPAD * 16;
  // (see `late` below)
  constexpr bool SHIFT = HD == 128;
  constexpr int VBUFS = SHIFT ? 3 : 2;
  __shared__ __align__(16) uint8_t k_lds[2][KB], v_lds[VBUFS][VB];
  __shared__ __align__(16) uint8_t raw_lds[2][8192];
  __shared__ int lds[WAVES], upto[THREADS], found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hh = lane >> 5;
  const int gqa = p.gqa;

  // (the same in every lane: said to the compiler, what follows stays out of the vector registers)
  RowLine<ROWS, KT, LEAD, THREADS> line{p, gqa, lds, upto};
  const int total = __builtin_amdgcn_readfirstlane(line.units());
  const int all = __builtin_amdgcn_readfirstlane(total * p.num_kv);
  if (blockIdx.x == 0 && tid == 0) p.cuts[4 * p.groups] = all;
  // neighbouring parts (the same head's keys) on one XCD, whose L2 holds their tiles
  const Parts parts(all, p.groups);
  const int grp = p.groups % 8 ? (int)blockIdx.x : (int)(blockIdx.x % 8) * (p.groups / 8) + (int)blockIdx.x / 8;
  if (grp >= parts.n) return;
  int u = parts.begin(grp);
  const int u_end = parts.begin(grp + 1);
  int h = u / total;
  Part at = line.find(u - h * total, found);
  bool first_seg = true;
  const uint32_t key_bytes = (uint32_t)p.num_kv * HD;
  const uint32_t page_bytes = (uint32_t)p.block_tokens * key_bytes;
  const int kt_div = KT / p.block_tokens, kt_mod = KT % p.block_tokens;
  const int entries = p.n_slots * p.slot_tiles;

  auto next = [&](int n_u) {
    first_seg = false;
    u += n_u;
    at.at = 0;
    at.entry++;
    if (at.entry >= entries) {
      at.entry = 0;
      h++;
    }
  };
  while (u < u_end) {
    const int s = at.entry / p.slot_tiles, rti = at.entry - s * p.slot_tiles;
    const Slot sl = slot_at(p, s);
    if (rti * ROWS >= sl.n * gqa) {   // past this slot's rows: on to the next slot with any, 64 at a time
      uint64_t any = 0;
      int t = s + 1;
      while (true) {
        if (t >= p.n_slots) {
          t = 0;
          if (++h >= p.num_kv) return;   // (starts or positions that change under the call)
        }
        any = __builtin_amdgcn_ballot_w64(t + lane < p.n_slots && slot_of(p, min(t + lane, p.n_slots - 1)).n > 0);
        if (any) break;
        t += 64;
      }
      at.entry = (t + __builtin_ctzll(any)) * p.slot_tiles;
      continue;
    }
    const RowTile rt = row_tile<ROWS, KT>(p, sl, rti, gqa);
    const int n_u = min(LEAD + rt.tiles - at.at, u_end - u);
    if (n_u <= 0) return;
    const int v0 = max(at.at - LEAD, 0), v1 = at.at + n_u - LEAD;   // (v1 <= v0: the next part's)
    // where the part begins, for the merge: row tile (-1: not past its first key tile), head, tile,
    // tiles
    if (first_seg && tid == 0)
      *reinterpret_cast<int4*>(p.cuts + 4 * grp) = make_int4(v0 > 0 ? at.entry : -1, h, v0, rt.tiles);
    const bool complete = v0 == 0 && v1 == rt.tiles;
    if (v1 <= v0) {
      next(n_u);
      continue;
    }
    const int rows = sl.n * gqa;
    const int row_w = rti * ROWS + wave * 32;      // this wave's first row
    const int row = min(row_w + c, rows - 1), tok = token_of(p, row);
    const int pos = sl.pos0 + tok;
    const int pos_lo = sl.pos0 + token_of(p, min(row_w, rows - 1)), pos_hi = sl.pos0 + token_of(p, min(row_w + 31, rows - 1));
    const bool live = row_w < rows;
    const long out_row = ((long)(sl.t0 + tok) * p.num_q + h * gqa + (row - tok * gqa)) * HD;

    const const_i32* table = (const const_i32*)(p.tables + (long)s * p.max_blocks);
    auto page_of = [&](int key) {   // (key the same in the whole wave)
      const int b = block_row(p, key).b;
      const int pg = key < rt.end && b < p.max_blocks ? table[b] : -1;
      return pg >= 0 && pg < p.n_pages ? pg : -1;
    };
    // Where this wave's rows see tiles whole, in halves y of 32 keys (key 32 (y + y_off) past the
    // sinks): y < y_sink or y_lo <= y < y_hi.  Tiles that none of them sees: v >= v_hi, and
    // v_sink <= v < v_lo.
    const int off = rt.w0 - rt.n_sink, y_off = off * KH;
    const int seen = min(pos_lo + 1, rt.end) / 32;
    const int y_hi = seen - y_off;
    int y_lo = rt.n_sink * KH, y_sink = 0;
    int v_hi = live ? pos_hi / KT + 1 - off : 0, v_lo = 0, v_sink = 0;
    if (p.window > 0) {
      if (pos_hi >= p.window) y_lo = max(y_lo, (pos_hi - p.window) / 32 + 1 - y_off);
      y_sink = min(min(p.sink / 32, seen), rt.n_sink * KH);
      v_sink = max(rt.n_sink, (p.sink + KT - 1) / KT - off);
      v_lo = pos_lo >= p.window ? (pos_lo - p.window + 1) / KT - off : 0;
      if (!live) v_hi = 0;
    }
    // This wave's WK keys of a tile lie in one page (pages are whole sixteens).  The next tile to
    // fetch is at row w_row of block w_base + w_at; lane i holds the page of block w_base + i (-1 past the
    // last key's: a page that was never written holds anything, its exponent too).
    int w_base, w_at, w_row, pages;
    auto load_pages = [&](int b) {
      w_base = b;
      w_at = 0;
      const bool any = b + lane < p.max_blocks && (uint32_t)(b + lane) * (uint32_t)p.block_tokens < (uint32_t)rt.end;
      const int pg = any ? table[b + lane] : -1;
      pages = pg < p.n_pages ? pg : -1;
    };
    auto seek = [&](int v) {
      const BlockRow x = block_row(p, rt.key0(v, KT) + wave * WK);
      load_pages(x.b);
      w_row = x.row;
    };
    // the fetched tile's exponents: the aligned words around them, by scalar loads (a vector load's
    // first use would wait for the codes under way too), and the bits at which they lie
    uint32_t kx = 0, vx = 0, k_bit = 0, v_bit = 0;
    int loaded = -1;                 // and its page
    const uint32_t lane_off = (uint32_t)(lane / LPR) * key_bytes + (uint32_t)(lane % LPR) * 16;
    const uint8_t* k_head = p.k_pool + (long)h * HD;
    const uint8_t* v_head = p.v_pool + (long)h * HD;
    auto fetch = [&](int v) {
      loaded = __builtin_amdgcn_readlane(pages, w_at);
      const uint32_t pg = max(loaded, 0);
      const uint64_t from = (uint64_t)pg * page_bytes + (uint32_t)w_row * key_bytes;
      uint32_t lo = lane_off;
      asm volatile("" : "+v"(lo));   // (else both sums with the bases are kept in registers)
      __builtin_amdgcn_global_load_lds((glb_void*)(k_head + from + lo), (lds_void*)(raw_lds[0] + wave * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((glb_void*)(v_head + from + lo), (lds_void*)(raw_lds[1] + wave * 1024), 16, 0, 0);
      const uint32_t ex = pg * (uint32_t)p.num_kv + h;
      const uint64_t ka = (uint64_t)p.k_exp + ex, va = (uint64_t)p.v_exp + ex;
      kx = *(const const_i32*)(ka & ~3ull);
      vx = *(const const_i32*)(va & ~3ull);
      k_bit = 8 * (uint32_t)(ka & 3);
      v_bit = 8 * (uint32_t)(va & 3);
      // on to the next tile
      w_row += kt_mod;
      w_at += kt_div;
      if (w_row >= p.block_tokens) {
        w_row -= p.block_tokens;
        w_at++;
      }
      if (v + 1 == rt.n_sink) seek(v + 1);
      else if (w_at >= 64) load_pages(w_base + w_at);
    };
    const int vl = lane % (HD / 4), vq = lane / (HD / 4);   // value dims 4 vl .., keys 4 vq .. of the wave's
    auto stage = [&](int v, int k_buf, int v_buf) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the codes are in LDS
      u4_t kr = *reinterpret_cast<const u4_t*>(raw_lds[0] + wave * 1024 + lane * 16);
      uint32_t vr[4];
#pragma unroll
      for (int i = 0; i < 4; i++)
        vr[i] = *reinterpret_cast<const uint32_t*>(raw_lds[1] + wave * 1024 + (4 * vq + i) * HD + vl * 4);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // ... and out of it again: the next may land
      const int key0 = rt.key0(v, KT) + wave * WK;
      // keys that do not exist are zeros (a page past the last key holds anything)
      if (loaded < 0 || key0 + WK > rt.end) {
        if (loaded < 0 || key0 + lane / LPR >= rt.end) kr = u4_t{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (loaded < 0 || key0 + 4 * vq + i >= rt.end) vr[i] = 0;
      }
      // (an absent page's exponent is not one)
      const float ksc = pow2f((kx >> k_bit) & 255u), vsc = pow2f(loaded < 0 ? 127 : (vx >> v_bit) & 255u);
      uint8_t* kb = k_lds[k_buf];
      uint8_t* vb = v_lds[v_buf];
      const int key = wave * WK + lane / LPR, slot = lane % LPR;
#pragma unroll
      for (int e = 0; e < 2; e++)
        *reinterpret_cast<h8_t*>(kb + key * KP + slot * 32 + e * 16) =
            join8(cvt2(kr[2 * e], ksc, false), cvt2(kr[2 * e], ksc, true), cvt2(kr[2 * e + 1], ksc, false),
                  cvt2(kr[2 * e + 1], ksc, true));
      const int q = wave * (WK / 4) + vq;
      // quad q of 16 keys (q & 3 = 2 a + half): 16-byte slot 2 (q / 4) + half, its part a
      const int at8 = ((q >> 2) * 2 + (q & 1)) * 16 + ((q >> 1) & 1) * 8;
      uint32_t w[2][2];
#pragma unroll
      for (int k = 0; k < 2; k++) {
        w[k][0] = __builtin_amdgcn_perm(vr[2 * k + 1], vr[2 * k], 0x05010400u);
        w[k][1] = __builtin_amdgcn_perm(vr[2 * k + 1], vr[2 * k], 0x07030602u);
      }
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int dim = 4 * vl + j;
        *reinterpret_cast<u2_t*>(vb + dim * VP + dim / VPAD * 16 + at8) =
            u2_t{__builtin_bit_cast(uint32_t, cvt2(w[0][j >> 1], vsc, j & 1)),
                 __builtin_bit_cast(uint32_t, cvt2(w[1][j >> 1], vsc, j & 1))};
      }
    };
    seek(v0);
    fetch(v0);
    // (the queries and the page check arrive beside the first codes)
    h8_t qf[HD / 16];
    {
      const uint16_t* src = p.q + out_row + 8 * hh;
#pragma unroll
      for (int i = 0; i < HD / 16; i++) qf[i] = *reinterpret_cast<const h8_t*>(src + 16 * i);
    }
    // whether every key from the part's first tile to its last has a page (else: looked up by tile)
    bool paged = true;
    for (int b = block_row(p, rt.key0(v0, KT)).b + lane, e = block_row(p, min(rt.key0(v1 - 1, KT) + KT, rt.end) - 1).b; b <= e; b += 64) {
      const int pg = b < p.max_blocks ? table[b] : -1;
      paged = paged && pg >= 0 && pg < p.n_pages;
    }
    paged = __builtin_amdgcn_ballot_w64(!paged) == 0;
    f16x_t acc[HD / 32];
#pragma unroll
    for (int d = 0; d < HD / 32; d++) acc[d] = f16x_t{};
    float mx = -INFINITY, ls = 0.f;
    // a negative scale is carried by the query, so that raw maxima serve; masked scores are -inf
    // ahead of the scale
    const float sl2 = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(fmaxf(fabsf(p.scale_log2), 1e-30f))));
    if (p.scale_log2 < 0.f) {
#pragma unroll
      for (int i = 0; i < HD / 16; i++) qf[i] = -qf[i];
    }
    __syncthreads();   // (the last segment's tiles are done with)
    stage(v0, 0, 0);
    if (v0 + 1 < v1) fetch(v0 + 1);
    __syncthreads();
    // At head_dim 128, with twice the weights for the same products, one wave of each SIMD takes a tile's
    // values in its turn and the other with the next tile, ahead of converting: one's products run
    // beside the other's conversions and weights (a prompt of 8,000 tokens, GQA 8, 585 -> 570 us; at 256
    // slower, 1,120 against 1,068 us for 2,048 tokens over 32,000 keys).
    const bool late = SHIFT && wave >= 4;
    bool held = false;
    h8_t w[2 * KH];
    constexpr int ND = HD / 32, NV = 2 * KH * ND;   // 32-dim blocks; of each 16 keys in turn
    auto products = [&](int v_buf) {
      const uint8_t* vat = v_lds[v_buf] + c * VP + c / VPAD * 16 + hh * 16;
      auto v_operand = [&](int i) {
        return *reinterpret_cast<const h8_t*>(vat + i % ND * (32 * VP + 32 / VPAD * 16) + i / ND * 32);
      };
      if (SHIFT) __builtin_amdgcn_s_setprio(1);
      h8_t va[4];
#pragma unroll
      for (int i = 0; i < 4; i++) va[i] = v_operand(i);
#pragma unroll
      for (int i = 0; i < NV; i++) {
        acc[i % ND] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[i % 4], w[i / ND], acc[i % ND], 0, 0, 0);
        if (i + 4 < NV) va[i % 4] = v_operand(i + 4);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int i = 0; i < NV - 4; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
      if (SHIFT) __builtin_amdgcn_s_setprio(0);
    };
    int v_buf = 0;
    for (int v = v0;; v++) {
      const int k_buf = (v - v0) & 1, v_next = v_buf == VBUFS - 1 ? 0 : v_buf + 1;
      if (late && held) products(v_buf == 0 ? VBUFS - 1 : v_buf - 1);
      if (v == v1) break;
      if (v + 1 < v1) {
        stage(v + 1, k_buf ^ 1, v_next);
        if (v + 2 < v1) fetch(v + 2);
      }
      held = v < v_hi && !(v >= v_sink && v < v_lo);   // (a wave none of whose rows sees the tile sits it out)
      if (held) {
        const uint8_t* kb = k_lds[k_buf];
        // scores of the tile's halves in turn (two chains of products at head_dim 128)
        if (SHIFT) __builtin_amdgcn_s_setprio(1);
        const uint8_t* krow = kb + c * KP + hh * 16;
        auto k_operand = [&](int i) { return *reinterpret_cast<const h8_t*>(krow + i % KH * (32 * KP) + i / KH * 32); };
        constexpr int NK = KH * HD / 16;
        f16x_t sd[KH] = {};
        h8_t ka[4];
#pragma unroll
        for (int i = 0; i < 4; i++) ka[i] = k_operand(i);
#pragma unroll
        for (int i = 0; i < NK; i++) {
          sd[i % KH] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[i % 4], qf[i / KH], sd[i % KH], 0, 0, 0);
          if (i + 4 < NK) ka[i % 4] = k_operand(i + 4);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int i = 0; i < NK - 4; i++) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
#pragma unroll
        for (int kh = 0; kh < KH; kh++) {
          const int y = v * KH + kh, k0 = (y < rt.n_sink * KH ? y : y + y_off) * 32;
          if (!((y >= y_lo && y < y_hi) || y < y_sink) || !paged) {
            const bool pa = page_of(k0) >= 0, pb = page_of(k0 + 16) >= 0;
#pragma unroll
            for (int x = 0; x < 16; x++) {
              const int key = k0 + 8 * (x >> 2) + 4 * hh + (x & 3);
              sd[kh][x] = (x < 8 ? pa : pb) && sees(key, pos, rt.end, p.window, p.sink) ? sd[kh][x] : -INFINITY;
            }
          }
        }
        if (SHIFT) __builtin_amdgcn_s_setprio(0);
        float t = sd[0][0];
#pragma unroll
        for (int x = 1; x < 16 * KH; x++) t = fmaxf(t, sd[x / 16][x % 16]);
        t = max32(t) * sl2;
        if (__builtin_amdgcn_ballot_w64(t > mx + kSlack) != 0) {
          const float mn = fmaxf(mx, t);
          const float r = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - mn);
          ls *= r;
#pragma unroll
          for (int d = 0; d < HD / 32; d++) acc[d] *= r;
          mx = mn;
        }
        const float base = mx == -INFINITY ? 0.f : mx;
        auto weights = [&](int sg) {
          h8_t w;
#pragma unroll
          for (int i = 0; i < 8; i++)
            w[i] = (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(sd[sg / 2][8 * (sg % 2) + i], sl2, -base));
          ls = add8(w, ls);
          return w;
        };
#pragma unroll
        for (int g = 0; g < 2 * KH; g++) w[g] = weights(g);
        if (!late) products(v_buf);
      }
      v_buf = v_next;
      __syncthreads();
    }

    ls = sum32(ls);
    if (row_w + c < rows) {
      if (complete) {
        const float inv = ls > 0.f ? 1.f / ls : 0.f;
        uint16_t* o = p.out + out_row + 4 * hh;
#pragma unroll
        for (int d = 0; d < HD / 32; d++)
#pragma unroll
          for (int a = 0; a < 4; a++)
            *reinterpret_cast<u2_t*>(o + 32 * d + 8 * a) =
                u2_t{f2h(acc[d][4 * a] * inv) | (f2h(acc[d][4 * a + 1] * inv) << 16),
                     f2h(acc[d][4 * a + 2] * inv) | (f2h(acc[d][4 * a + 3] * inv) << 16)};
      } else {
        // (in the registers' order: 1 KB a store; the merge reads them so)
        const long rec = 2 * grp + (first_seg ? 0 : 1);
        f4_t* ro = reinterpret_cast<f4_t*>(p.rec_o + (rec * ROWS + 32 * wave) * HD) + lane;
#pragma unroll
        for (int d = 0; d < HD / 32; d++)
#pragma unroll
          for (int a = 0; a < 4; a++)
            ro[(4 * d + a) * 64] = f4_t{acc[d][4 * a], acc[d][4 * a + 1], acc[d][4 * a + 2], acc[d][4 * a + 3]};
        if (hh == 0) *reinterpret_cast<f2_t*>(p.rec_ml + (rec * ROWS + 32 * wave + c) * 2) = f2_t{rec_max(mx, ls), ls};
      }
    }
    next(n_u);
  }
}

// The row tiles that parts cut: a wave per 32 rows and 32 dims, in the registers' order of the
// kernel above; the workgroups of a part's cut only if the tile begins in the part before
// (each tile once).  Bound by HBM: the records of 256 parts of 256 rows of 256, 134 MB, in 25 us.
template <int HD>
__global__ __launch_bounds__(256) void f8_cut_merge_kernel(F8AttnArgs p) {
  constexpr int ROWS = 256, DB = HD / 32, WGS = 8 * DB / 4;
  const int lane = threadIdx.x & 63, c = lane & 31, hh = lane >> 5;
  const int cut_at = blockIdx.x / WGS, grp = cut_at + 1;
  const int unit = (blockIdx.x - cut_at * WGS) * 4 + (threadIdx.x >> 6), rw = unit / DB, d = unit - rw * DB;
  const int4 cut = *reinterpret_cast<const int4*>(p.cuts + 4 * grp);
  const Parts parts(p.cuts[4 * p.groups], p.groups);
  if (grp >= parts.n) return;
  const int entry = cut.x, h = cut.y, v0 = cut.z, tiles = cut.w;
  if (entry < 0) return;
  // units of the row tile's first key tile, and of its lead
  const int x1 = parts.begin(grp) - v0, x0 = x1 - kLead<HD>, before = parts.begin(grp - 1);
  if (before > x1) return;   // an earlier cut is in this tile
  const int n = parts.of(x1 + tiles - 1) - grp + 2;
  const long r0 = 2 * (grp - 1) + (before >= x0 ? 0 : 1);
  auto rec_of = [&](int i) { return i == 0 ? r0 : 2l * (grp - 1 + i); };
  const int s = entry / p.slot_tiles, gqa = p.gqa;
  const Slot sl = slot_of(p, s);
  const int r = (entry - s * p.slot_tiles) * ROWS + 32 * rw + c;
  if (r >= sl.n * gqa) return;
  float M = -INFINITY, L = 0.f;
  f4_t o[4] = {};
#pragma unroll 2
  for (int i = 0; i < n; i++) {
    const long rec = rec_of(i);
    const f2_t ml = *reinterpret_cast<const f2_t*>(p.rec_ml + (rec * ROWS + 32 * rw + c) * 2);
    const f4_t* src = reinterpret_cast<const f4_t*>(p.rec_o + (rec * ROWS + 32 * rw) * HD) + 4 * d * 64 + lane;
    f4_t x[4];
#pragma unroll
    for (int a = 0; a < 4; a++) x[a] = src[a * 64];
    const bool any = ml[1] != 0.f;
    const float mn = fmaxf(M, any ? ml[0] : -INFINITY);
    const float f = mn == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - mn);
    const float w = any ? __builtin_amdgcn_exp2f(ml[0] - mn) : 0.f;
    M = mn;
    L = L * f + w * ml[1];
#pragma unroll
    for (int a = 0; a < 4; a++) o[a] = o[a] * f + x[a] * w;
  }
  const float inv = L > 0.f ? 1.f / L : 0.f;
  const int t = token_of(p, r);
  uint16_t* dst = p.out + ((long)(sl.t0 + t) * p.num_q + h * gqa + (r - t * gqa)) * HD + 32 * d + 4 * hh;
#pragma unroll
  for (int a = 0; a < 4; a++) {
    const f4_t y = o[a] * inv;
    *reinterpret_cast<u2_t*>(dst + 8 * a) = u2_t{f2h(y[0]) | (f2h(y[1]) << 16), f2h(y[2]) | (f2h(y[3]) << 16)};
  }
}

// ---------------------------------------------------------------------------
// merge of the row tiles that were cut
// ---------------------------------------------------------------------------
// A workgroup per row, whose waves share its records; bound by latency (5 us: the row's place, then
// its records at once).
template <int HD>
__global__ __launch_bounds__(256) void f8_merge_kernel(F8AttnArgs p) {
  constexpr int E = HD / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t at = blockIdx.y * kGridX + blockIdx.x, tile = at / p.rec_rows;
  const int row = (int)(at - tile * p.rec_rows);
  if (tile >= (uint32_t)(p.n_slots * p.num_kv)) return;
  const int s = (int)tile / p.num_kv, h = (int)tile - s * p.num_kv, gqa = p.gqa;
  const int2 desc = p.desc[tile];
  const Slot sl = slot_of(p, s);
  const int n = desc.x, r0 = desc.y;
  if (row >= sl.n * gqa || n < 2) return;   // (one part: stored whole)
  auto rec_of = [&](int i) { return i == 0 ? r0 : 2 * (r0 / 2 + i); };

  // 64 records a round: lane i holds record i's {m, l}, the wave reads 16 records' sums (all
  // of a round's loads are under way before the first is used), weights by lane reads
  float M = -INFINITY, L = 0.f;
  float o[E] = {};
  for (int i0 = 0; i0 < n; i0 += 64) {
    float x[16][E];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float* src = p.rec_o + ((long)rec_of(min(i0 + 16 * wave + i, n - 1)) * p.rec_rows + row) * HD + lane * E;
      if constexpr (E == 4) {
        const f4_t v = *reinterpret_cast<const f4_t*>(src);
#pragma unroll
        for (int e = 0; e < 4; e++) x[i][e] = v[e];
      } else {
        const f2_t v = *reinterpret_cast<const f2_t*>(src);
        x[i][0] = v[0];
        x[i][1] = v[1];
      }
    }
    f2_t r = {-INFINITY, 0.f};
    if (i0 + lane < n) r = *reinterpret_cast<const f2_t*>(p.rec_ml + ((long)rec_of(i0 + lane) * p.rec_rows + row) * 2);
    const bool any = r[1] != 0.f;
    const float mn = fmaxf(M, wave_max(any ? r[0] : -INFINITY));
    if (mn == -INFINITY) continue;   // no key so far
    const float f = __builtin_amdgcn_exp2f(M - mn), w = any ? __builtin_amdgcn_exp2f(r[0] - mn) : 0.f;
    M = mn;
    L = L * f + wave_sum(w * r[1]);
#pragma unroll
    for (int e = 0; e < E; e++) o[e] *= f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float wi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), 16 * wave + i));
#pragma unroll
      for (int e = 0; e < E; e++) o[e] = __builtin_fmaf(wi, x[i][e], o[e]);
    }
  }
  __shared__ float part[4][64][E];
#pragma unroll
  for (int e = 0; e < E; e++) part[wave][lane][e] = o[e];
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < 4; w++)
#pragma unroll
    for (int e = 0; e < E; e++) o[e] += part[w][lane][e];
  const float inv = L > 0.f ? 1.f / L : 0.f;
  const int t = token_of(p, row);
  uint16_t* dst = p.out + ((long)(sl.t0 + t) * p.num_q + h * gqa + (row - t * gqa)) * HD + lane * E;
  if constexpr (E == 4)
    *reinterpret_cast<u2_t*>(dst) = u2_t{f2h(o[0] * inv) | (f2h(o[1] * inv) << 16), f2h(o[2] * inv) | (f2h(o[3] * inv) << 16)};
  else
    *reinterpret_cast<uint32_t*>(dst) = f2h(o[0] * inv) | (f2h(o[1] * inv) << 16);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
F8AttnPlan f8_attn_plan(int num_q, int num_kv, int head_dim, int n_slots, long q_rows, int max_tok, int max_ctx) {
  F8AttnPlan x{};
  const long rows = (long)max_tok * (num_q / num_kv);
  x.many = rows > 64;
  x.row_tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  long units;   // most units of all heads
  if (x.many) {
    const int tile_rows = 256, kt = 8192 / head_dim;
    x.slot_tiles = (int)((rows + tile_rows - 1) / tile_rows);
    x.rec_rows = tile_rows;
    // (a slot has at most one row tile that is not full)
    const long tiles = std::min<long>((long)n_slots * x.slot_tiles, q_rows * (num_q / num_kv) / tile_rows + n_slots);
    units = tiles * num_kv * ((max_ctx + kt - 1) / kt);   // (key tiles: a part for less would be all lead)
    x.groups = (int)std::min<long>(units, 256);
    x.merges = true;
  } else {
    x.slot_tiles = 1;
    x.rec_rows = (int)rows;
    // Short contexts: few records, joined in the launch where one workgroup takes no longer for them than
    // a second launch: up to 1,024 keys (16 slots of 16 rows of 256: 19.8 against 18.8 to 19.6 us, 16 rows
    // of 128 12.9 and 14.0 to 15.4), for rows of up to 2,048 elements up to 2,048 keys (one token of 2,000
    // keys 10.5 and 11.1 to 13.3 us, though two in eight slots 17.3 and 14.9 to 16.1; not 16 rows of 256,
    // 24.2 and 19.8, nor four slots of 4,000 keys, 19.3 and 17.4).
    const long row_elems = rows * head_dim;
    x.join = x.row_tiles == 1 && max_ctx <= (row_elems <= 2048 ? 2 : 1) * kJoinKeys && n_slots <= 64 && n_slots * num_kv <= kJoinCounts;
    const int unit_keys = x.row_tiles == 4 ? 64 : 128;
    units = (long)n_slots * num_kv * ((max_ctx + unit_keys - 1) / unit_keys);
    x.groups = (int)std::min<long>(units, x.row_tiles == 1 || head_dim == 128 ? 512 : 256);   // (what the CUs hold at once)
    x.merges = max_ctx > unit_keys;   // (else no slot has two units)
  }
  const size_t ints = x.many ? 4 * (size_t)x.groups + 4 : 2 * (size_t)n_slots * num_kv;
  const size_t pre = kJoinCounts * 4 + (ints * 4 + 255) / 256 * 256;
  const size_t recs = x.merges ? 2 * (size_t)x.groups * x.rec_rows : 0;
  x.ml_off = pre;
  x.o_off = pre + (recs * 8 + 255) / 256 * 256;
  x.total = x.o_off + recs * head_dim * 4;
  return x;
}

// A call may hold prompts and single tokens.  A one-token slot costs the kernel for many rows the
// conversion of whole tiles for a 64th of their rows (32 slots at 4,000 keys and a prompt of 2,048
// tokens: 184 to 190 us in one launch, 132 to 140 as two); a launch for nothing costs 7 us.  The numbers do not
// say how the rows spread: the fewest slots that can hold them all are taken to be prompts, and the
// others to have up to 16 rows, with whole contexts.
int f8_attn_apart(int num_q, int num_kv, int head_dim, int n_slots, long rows, int max_tok, int max_ctx) {
  const int gqa = num_q / num_kv;
  if ((long)max_tok * gqa <= 64) return 0;
  const double small = n_slots - (rows + max_tok - 1) / max_tok;
  return small * num_kv * max_ctx * head_dim >= (double)(1 << 25) ? 16 / gqa : 0;
}

template <int HD>
static void launch_f8(const F8AttnArgs& a, const F8AttnPlan& x, hipStream_t stream) {
  const dim3 grid((unsigned)x.groups);
  if (x.many)
    hipLaunchKernelGGL((f8_many_kernel<HD>), grid, dim3(512), 0, stream, a);
  else if (x.join)
    hipLaunchKernelGGL((f8_few_kernel<HD, true>), grid, dim3(256), 0, stream, a);
  else if (x.row_tiles == 1)
    hipLaunchKernelGGL((f8_few_kernel<HD, false>), grid, dim3(256), 0, stream, a);
  else if (x.row_tiles == 2)
    hipLaunchKernelGGL((f8_mid_kernel<HD, 1>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((f8_mid_kernel<HD, 2>), grid, dim3(256), 0, stream, a);
  if (!x.merges || x.join) return;
  if (x.many) {
    if (x.groups > 1)
      hipLaunchKernelGGL((f8_cut_merge_kernel<HD>), dim3((unsigned)(x.groups - 1) * (HD / 16)), dim3(256), 0, stream, a);
  } else {
    // (at most 2^22 row tiles of 64 rows)
    hipLaunchKernelGGL((f8_merge_kernel<HD>), grid_xy((long)a.n_slots * a.num_kv * x.rec_rows), dim3(256), 0, stream, a);
  }
}

hipError_t launch_f8_attn(const F8AttnArgs& a, const F8AttnPlan& plan, int head_dim, hipStream_t stream) {
  if (head_dim == 256) launch_f8<256>(a, plan, stream);
  else if (head_dim == 128) launch_f8<128>(a, plan, stream);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

}  // namespace qkv
