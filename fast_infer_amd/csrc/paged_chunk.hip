// Attention of a chunk of new tokens over a paged KV pool [num_blocks, block_size,
// num_kv_heads, head_dim], for gfx950: the form between causal prefill (no cache) and decode
// (one token): prompts prefilled in pieces or behind a cached beginning, drafted tokens, single
// tokens of models whose scores are capped, biased or windowed.
//
//   x[t, j] = sm_scale * q[t] . k[j]            position pos = start + t, key j < len
//   x       = cap * tanh(x / cap)               (with a cap)
//   x      -= slope[h] * |pos - j|              (with a distance bias)
//   o[t]    = sum_j softmax_j(x[t, j]) v[j]     over the keys token t sees:
//             j < prefix, or pos - window < j <= pos
//
// Layout for MI355X:
//   * The query rows of one kv head are the pairs (token, head of the group), token-major, one row
//     per MFMA column, so that any group size fills the columns.  Up to 32 rows (single tokens,
//     drafted ones) are bound by the stream of K and V: narrow_kernel, whose waves share the rows
//     and split the keys.  More rows are bound by the matrix cores and the softmax beside them:
//     chunk_kernel, whose waves share the key tiles and have 16 to 48 rows each.
//   * S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16: the lane that holds a query
//     column keeps its scores, P and O; the softmax (online, fp32, base 2) needs no shuffles.
//   * 64-key tiles are copied global -> LDS without registers, the next one while one is used; so
//     are the block table's entries.  Keys at or past the row's length, or behind an invalid
//     entry, are copied from a row of zeros, and never read.
//   * The tiles that need a mask (the diagonal, the ends of the window and of the prefix) come first, in
//     a loop of their own: the others run without any (233 -> 92 us for 512 tokens at 8192).
//   * Where the row tiles alone do not fill the device their lists of key tiles are cut into parts, by
//     the rows' own lengths, on the device; a second kernel adds the parts.
// Measured (24 query heads on 8 kv heads, 128 wide, MI355X): 2 x 2048 tokens, of 16384, 0.72-0.74 ms, 1.06
// PFLOP/s; 512 tokens at 8192 73 us, 0.69; 24 rows of 5 drafted tokens (300 to 4096 keys) 45 us, 4.5 TB/s.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "common.h"

namespace fi {
namespace chunk {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kKTile = 64;  // keys per tile
constexpr float kLazyLog2 = 8.f;  // the reference max may lag the true max by 2^8
constexpr int kNoWindow = 0x3fffffff;
constexpr int64_t kMaxTokens = (int64_t)1 << 22;
constexpr int kMinPart = 2;  // key tiles of the smallest part
// Calls of few query rows and up to this many tokens are not cut: adding the parts takes as long as
// the key tiles they save (one token of 256 11.8 against 8.6 us).
constexpr int64_t kWholeTokens = 512;
// Largest cap whose tanh is taken from exp2 alone: its absolute error, about 2e-7, times the
// cap is an error of the logit, here 1e-4.
constexpr float kExpCap = 500.f;

constexpr float kMaxScale = 1e7f;  // scale or cap; the start of the running max stays finite in log2 units
constexpr float kFlat = 1e-20f;    // scale or cap below which every score counts as zero

constexpr int kCap = 1;   // kMod bits: capped scores,
constexpr int kBias = 2;  // distance bias

// n / d for 0 <= n < 2^31 by a multiplication.
struct FastDiv {
  uint32_t mul;
  int shift;
};
static FastDiv fast_div(uint32_t d) {
  int l = 0;
  while (((uint64_t)1 << l) < d) ++l;
  return {(uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << l) - d)) / d + 1), l};
}
__device__ __forceinline__ int div_by(int n, FastDiv d) {
  return (int)((__umulhi((uint32_t)n, d.mul) + (uint32_t)n) >> d.shift);
}

struct Params {
  const half_t* q;
  int64_t q_sb, q_st, q_sh;
  const half_t* k_cache;
  const half_t* v_cache;
  int num_pool_blocks;
  int block_size;
  int whole;  // block_size % 16 == 0: the 16 keys that a wave copies lie in one block
  FastDiv block_div;
  int num_kv_heads;
  FastDiv kv_div;
  int64_t row_bytes;  // one pool slot, all kv heads
  const int32_t* block_table;
  int64_t bt_stride;
  int max_blocks_per_seq;
  const int32_t* start_positions;
  const int32_t* context_lens;
  int num_tokens;  // bound of the lengths, at most the table's width
  half_t* o;
  int64_t o_sb, o_st, o_sh;
  int batch, chunk;
  FastDiv batch_div;
  int num_q_heads;
  FastDiv head_div;
  int group;
  FastDiv group_div;
  int head_dim;
  int d_chunks;       // 16-byte chunks of a row; those past it are read as zeros
  float scale_log2;   // score unit -> log2 unit
  float lazy_raw;     // kLazyLog2 in score units
  float lazy_log2;    // lazy_raw * scale_log2
  uint32_t q_sign;    // 0x80008000: Q negated (negative sm_scale without a cap)
  int q_zero;         // sm_scale == 0 without a cap: Q read as zeros
  float cap_exp;      // sm_scale / cap * 2 log2(e)
  const float* slopes;
  float slope_mul;    // slope unit -> score unit
  int window;
  const int32_t* prefix_lens;
  int tile_rows;      // query rows of a row tile, 64 * NB
  FastDiv tile_div;
  int row_tiles;      // of each (batch row, kv head): ceil(chunk * group / tile_rows)
  int target;         // parts aimed at, all kv heads together: one round of workgroups
  int target2;        // or this many, where one round would be uneven (0: never)
  int part_rows;      // min(tile_rows, chunk * group): rows of a part's results
  float* part_o;      // [parts, num_kv_heads][part_rows][128]; null: no parts, write o
  float* part_ml;     // [...][2]: reference max (log2 units), sum
  int32_t* shares;    // [batch][2]: Share::before and parts, for the kernel that adds the parts
};

// What a batch row attends over.
struct Row {
  int start, len, prefix;
};
__device__ __forceinline__ Row row_of(const Params& p, int b) {
  Row r;
  int len = p.context_lens ? p.context_lens[b] : p.num_tokens;
  len = min(len, p.num_tokens);
  r.len = max(len, 0);
  int s = p.start_positions ? p.start_positions[b] : r.len - p.chunk;
  r.start = max(min(s, r.len), -p.chunk);
  int pre = p.prefix_lens ? p.prefix_lens[b] : 0;
  r.prefix = max(min(pre, r.len), 0);
  return r;
}

// Positions of the valid tokens among query rows r0 .. r1 (lo > hi: none).
__device__ __forceinline__ void row_positions(const Params& p, const Row& row, int r0, int r1, int& lo,
                                              int& hi) {
  lo = max(row.start + div_by(r0, p.group_div), 0);
  hi = min(row.start + min(div_by(r1, p.group_div), p.chunk - 1), row.len - 1);
}

// The key tiles a row tile visits: tiles 0 .. n_pre - 1 (prefix), then the causal ones from `from`
// on.  They are taken in an order that puts those first in which some row may not see some key
// (the ends of the window and of the prefix, the diagonal), so that the others run in a loop
// without masks: list places [tail, n), [full_pre, head), then [0, full_pre), [head, tail).
struct Span {
  int n_pre, from, n;
  int full_pre, head, tail;
  __device__ __forceinline__ int masked() const { return n - tail + head - full_pre; }
  __device__ __forceinline__ int tile(int i) const {  // of place i in the order
    int at = i + tail;
    if (i >= n - tail) at = full_pre + i - (n - tail);
    if (i >= masked()) at = i - masked();
    if (i >= masked() + full_pre) at = head + i - masked() - full_pre;
    return at < n_pre ? at : from + at - n_pre;
  }
};
__device__ __forceinline__ Span span_of(const Params& p, const Row& row, int lo, int hi) {
  Span s;
  s.n_pre = (row.prefix + kKTile - 1) / kKTile;
  s.from = max(max(lo - p.window + 1, 0) / kKTile, s.n_pre);
  const int end = max((hi + kKTile) / kKTile, s.from);
  s.n = s.n_pre + end - s.from;
  s.full_pre = row.prefix / kKTile;
  if (p.slopes) s.full_pre = min(s.full_pre, (lo + 1) / kKTile);  // the distance bias bends at the row
  // causal tiles that every row sees whole: behind hi - window, and up to lo
  const int a = min(max(hi >= p.window ? (hi - p.window) / kKTile + 1 : 0, s.from), end);
  const int e = max(min((lo + 1) / kKTile, end), a);
  s.head = s.n_pre + a - s.from;
  s.tail = s.n_pre + e - s.from;
  if (lo > hi) s.n = s.full_pre = s.head = s.tail = 0;
  return s;
}
// The row tiles of a batch row that hold tokens (first .. first + count - 1), and the key tiles
// of the last of them.
struct RowTiles {
  int first, count, n;
};
__device__ __forceinline__ RowTiles row_tiles_of(const Params& p, const Row& row) {
  const int t0 = max(-row.start, 0), t1 = min(row.len - row.start, p.chunk);
  RowTiles r = {0, 0, 0};
  if (t0 < t1) {
    r.first = div_by(t0 * p.group, p.tile_div);
    const int last = div_by(t1 * p.group - 1, p.tile_div);
    r.count = last - r.first + 1;
    int lo, hi;
    row_positions(p, row, last * p.tile_rows, (last + 1) * p.tile_rows - 1, lo, hi);
    r.n = span_of(p, row, lo, hi).n;
  }
  return r;
}

// Every workgroup finds its part by itself, from the lengths on the device: each row tile of batch
// row b is cut into parts(b) = ceil(its longest list / size) equal pieces; the work list is, for
// each b, its parts (row tile fastest, so that neighbours read the same keys), then its row
// tiles without tokens, one each.  The size is the one at which all parts fit one round of
// workgroups (a few steps from below; a few more than that take as long as a whole round); many
// query rows of uneven lengths may be better off with two rounds of smaller parts.  In key tiles
// of a CU: the workgroups that share one take as many times the longest part, all of them at
// least all tiles over the CUs, and a part costs about nine tiles (its results, written and
// read, and its start).  6 rows of up to 6000 tokens 173 -> 147 us with two rounds, 512 new
// tokens at 8192 77 against 95.  Returns the batch row of list place `item` (-1 past the list), the
// places before it and its parts.  For the whole workgroup; s_tiles: an int of LDS per batch row (fewer
// than 2^10, a call of more workgroups than that is not cut).
struct Share {
  int b, before, parts;
};
// A barrier for LDS: copies stay on their way.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
// Inclusive sums over the lanes (row shifts, then row broadcasts: no LDS round trips).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);   // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);   // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);   // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1, 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2, 3
  return v;
}
__device__ __forceinline__ int wave_sum(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }
__device__ __forceinline__ int wave_max(int v) {  // of values >= 0
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(v, 63);
}
// ceil(n / size) for n, size <= 2^17 (1 for n = 0), from 1 / size to the last bit or two: n - 1/2 over
// size is further from a whole number than any rounding here.  Larger n: within one part in 2^22.
__device__ __forceinline__ float inverse(int x) { return __builtin_amdgcn_rcpf((float)x); }
__device__ __forceinline__ int parts_of(int n, float inv_size) {
  return n > 0 ? (int)(((float)n - 0.5f) * inv_size) + 1 : 1;
}
// floor(n / d) in the same range
__device__ __forceinline__ int whole_of(int n, int d) { return (int)(((float)n + 0.5f) * inverse(d)); }

__device__ __forceinline__ Share find_share(const Params& p, int item, int tid, int* s_tiles) {
  if (p.batch == 1) {
    const RowTiles t = row_tiles_of(p, row_of(p, 0));
    const int most = whole_of(p.target, max(t.count * p.num_kv_heads, 1));  // parts in one round
    const int parts = max(min(most, (t.n + kMinPart - 1) / kMinPart), 1);
    return {item < t.count * parts + p.row_tiles - t.count ? 0 : -1, 0, parts};
  }
  // row tiles (fewer than 2^10) and key tiles (at most 2^16 + 1) of every batch row, into LDS
  constexpr int kShift = 17, kMask = (1 << kShift) - 1;
  for (int i = tid; i < p.batch; i += kThreads) {
    const RowTiles t = row_tiles_of(p, row_of(p, i));
    s_tiles[i] = t.count << kShift | t.n;
  }
  lds_barrier();
  const int lane = tid & 63;
  auto tiles_at = [&](int i) { return i + lane < p.batch ? s_tiles[i + lane] : 0; };
  const int v0 = tiles_at(0);
  int total = (v0 >> kShift) * (v0 & kMask), rows = v0 >> kShift;
  for (int i = 64; i < p.batch; i += 64) {
    const int v = tiles_at(i);
    total += (v >> kShift) * (v & kMask);
    rows += v >> kShift;
  }
  total = wave_sum(total) * p.num_kv_heads;
  rows = wave_sum(rows) * p.num_kv_heads;
  float inv = 0.f;
  int best = INT_MAX;
  for (int round = 0; round < 2; ++round) {
    const int target = round ? p.target2 : p.target;
    if (target == 0) break;
    // no smaller than all tiles over the target (the list's bound); each row tile's last part is
    // half full on average
    const int least = max(parts_of(total, inverse(target)), kMinPart);
    int size = max(parts_of(total, inverse(max(target - rows / 2, 1))), least), wgs = 0, longest = 0;
    if (2 * rows > target) size = least;
    float inv_size = inverse(size);
    for (int step = 0; step < 5; ++step) {
      const int parts0 = parts_of(v0 & kMask, inv_size);
      wgs = (v0 >> kShift) * parts0;
      longest = parts_of(v0 & kMask, inverse(parts0));
      for (int i = 64; i < p.batch; i += 64) {
        const int v = tiles_at(i);
        const int parts = parts_of(v & kMask, inv_size);
        wgs += (v >> kShift) * parts;
        longest = max(longest, parts_of(v & kMask, inverse(parts)));
      }
      wgs = wave_sum(wgs) * p.num_kv_heads;
      if (wgs <= target || step == 4) break;
      size = max((int)((float)size * (float)wgs * inverse(target)), size + 1);
      inv_size = inverse(size);
    }
    if (p.target2 == 0) {
      inv = inv_size;
      break;
    }
    const int cost = max((wgs + 255) / 256 * 256 * wave_max(longest), total) + 9 * wgs;
    if (cost < best) {
      best = cost;
      inv = inv_size;
    }
  }
  Share s = {-1, 0, 1};
  int before = 0;
  for (int i = 0; i < p.batch; i += 64) {
    const int v = i == 0 ? v0 : tiles_at(i);
    const int parts = parts_of(v & kMask, inv);
    const int items = i + lane < p.batch ? (v >> kShift) * (parts - 1) + p.row_tiles : 0;
    const int upto = before + wave_scan(items);
    if (const uint64_t hit = __builtin_amdgcn_ballot_w64(upto > item)) {
      const int l = __builtin_ctzll(hit);
      s.b = i + l;
      s.before = __builtin_amdgcn_readlane(upto - items, l);
      s.parts = __builtin_amdgcn_readlane(parts, l);
      break;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  lds_barrier();  // the tiles that follow take this place
  return s;
}

// LDS layout of a tile of kD-wide rows (64 or 128; a smaller head_dim leaves zeros).  Whole rows
// of 2 kD bytes, as they lie in the pool, so that a copy instruction reads 1 KiB in full rows:
// with 64- and 32-byte pieces of many rows (as the prefill kernel copies) long contexts streamed
// at 3 TB/s.  The 16-byte chunks of a row are XOR-permuted: K fragment reads (16 rows, one chunk
// per 16-lane group; the LDS serves 8 rows of two such groups at a time) and V transpose reads (8
// rows, 32 bytes) are free of bank conflicts, and the fragments of a row differ by an XOR of the
// address with a constant.
template <int kD>
struct Tile {
  static constexpr int kRow = 2 * kD;           // bytes
  static constexpr int kChunks = kD / 8;
  static constexpr int kBytes = kKTile * kRow;  // of K or V
  static constexpr int kStage = 2 * kBytes;
  static constexpr int kCopyRows = 1024 / kRow;                // rows of one copy instruction
  static constexpr int kCopies = kKTile / kWaves / kCopyRows;  // of a wave, each of K and V
  static __device__ __forceinline__ int xk(int r) {
    return (kD == 128 ? (r & 3) << 2 : (r & 2) << 1) | ((r >> 1) & 2);
  }
  static __device__ __forceinline__ int xv(int r) { return kD == 128 ? (r & 7) << 1 : r & 6; }
};

// The row that masked keys and the columns past head_dim are copied from.
__device__ __attribute__((aligned(256))) const char g_zeros[2 * kHeadDim] = {0};
// The table entry of keys that are not to be read.
__device__ const int32_t g_no_block = -1;

// Values that are the same in every lane, where the compiler has them in vector registers.
__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint32_t scalar(uint32_t x) { return (uint32_t)scalar((int)x); }
__device__ __forceinline__ uint64_t scalar(uint64_t x) {
  return (uint64_t)scalar((uint32_t)(x >> 32)) << 32 | scalar((uint32_t)x);
}

// One direct-to-LDS copy from a 64-bit address per lane: 16 bytes to LDS byte lds + 16 * lane.
// Through inline asm for the reasons given at lds_copy16; the callers wait for the copies
// themselves.  M0 takes one idle slot before a global load reads it.
__device__ __forceinline__ void lds_copy16_global(const char* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(scalar(lds)), "v"(src)
               : "memory");
}

// The same with the non-temporal policy, for keys that one workgroup reads.
__device__ __forceinline__ void lds_copy16_global_nt(const char* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt"
               :
               : "s"(scalar(lds)), "v"(src)
               : "memory");
}
// The same from a common base and 32-bit offsets.
template <bool kOnce>
__device__ __forceinline__ void lds_copy16_base(const char* base, uint32_t offset, uint32_t lds) {
  if (kOnce)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt"
                 :
                 : "s"(scalar(lds)), "v"(offset), "s"(scalar((uint64_t)base))
                 : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(scalar(lds)), "v"(offset), "s"(scalar((uint64_t)base))
                 : "memory");
}
// The same with 4 bytes a lane.
__device__ __forceinline__ void lds_copy4_global(const int32_t* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
               :
               : "s"(scalar(lds)), "v"(src)
               : "memory");
}
// All but the last N of this wave's copies have landed (they do in order).
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// This wave's copies have landed, its LDS reads are done, and every other wave says the same.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// 16 bits of each wave, as one scalar.
__device__ __forceinline__ uint64_t uniform64(const uint16_t* x) {
  return scalar(*(const uint64_t*)x);
}

// This wave's copies of a tile: K and V of keys 16w .. 16w + 15, whose pool rows (-1: zeros) lanes
// lane0 .. lane0 + 15 hold in `row`.
template <int kD, bool kOnce>
__device__ __forceinline__ void issue_tile(const Params& p, const char* kbase, const char* vbase,
                                           char* stage, int row, int lane0, int w, int lane) {
  typedef Tile<kD> T;
  const int slot = lane % T::kChunks;
  const uint32_t dst = lds_addr(stage) + 16 * w * T::kRow;
#pragma unroll
  for (int q = 0; q < T::kCopies; ++q) {
    const int r = q * T::kCopyRows + lane / T::kChunks;
    const int from = __shfl(row, lane0 + r);
    const int64_t at = from * p.row_bytes;
    const int kc = slot ^ T::xk(r), vc = slot ^ T::xv(r);
    const char* ks = (from >= 0 && kc < p.d_chunks ? kbase + at : g_zeros) + 16 * kc;
    const char* vs = (from >= 0 && vc < p.d_chunks ? vbase + at : g_zeros) + 16 * vc;
    if (kOnce) {
      lds_copy16_global_nt(ks, dst + 1024 * q);
      lds_copy16_global_nt(vs, dst + T::kBytes + 1024 * q);
    } else {
      lds_copy16_global(ks, dst + 1024 * q);
      lds_copy16_global(vs, dst + T::kBytes + 1024 * q);
    }
  }
}

// The copies of one wave: keys 16w .. 16w + 15 of the part's tiles, and the table entries they need.
// Entries come through LDS (s_ent, 256 of the wave): an ordinary load in the loop would make the
// compiler wait for every copy.  Blocks of a multiple of 16 tokens: one entry a tile, those of 64
// tiles a copy; then the copies of a tile of 16 valid keys take a scalar base and constant
// offsets (with an address per lane the wide kernel spends a third of its vector instructions on
// them).  Other sizes: an entry per key, lane l's for key l % 16, copied two tiles ahead of the keys'.
template <int kD, bool kOnce>
struct Copier {
  typedef Tile<kD> T;
  const Params& p;
  const Span& span;
  int first, n, len, w, lane;
  const int32_t* table;
  const char *kbase, *vbase;
  char* stages;
  int* s_ent;
  uint32_t k_off, v_off;

  __device__ __forceinline__ Copier(const Params& p_, const Span& span_, int first_, int n_, int len_, int b,
                                    int kvh, int w_, int lane_, char* stages_, int* s_ent_)
      : p(p_), span(span_), first(first_), n(n_), len(len_), w(w_), lane(lane_),
        table(p_.block_table + (int64_t)b * p_.bt_stride),
        kbase((const char*)(p_.k_cache + (int64_t)kvh * p_.head_dim)),
        vbase((const char*)(p_.v_cache + (int64_t)kvh * p_.head_dim)), stages(stages_), s_ent(s_ent_) {
    const int r = lane / T::kChunks;
    const uint32_t row = (uint32_t)(r * (int)p.row_bytes);
    k_off = row + 16 * ((lane % T::kChunks) ^ T::xk(r));
    v_off = row + 16 * ((lane % T::kChunks) ^ T::xv(r));
  }
  __device__ __forceinline__ int key_of(int i) const { return span.tile(first + i) * kKTile + 16 * w; }
  __device__ __forceinline__ void entry(int i, int more, int slot) const {  // of key key_of(i) + more
    const int key = key_of(i) + more;
    const int blk = div_by(key, p.block_div);
    lds_copy4_global(i < n && key < len && blk < p.max_blocks_per_seq ? table + blk : &g_no_block,
                     lds_addr(s_ent + slot));
  }
  // The entries before the first tile, and with tile i (then those of tile i + 4 or of the next 64).
  __device__ __forceinline__ void first_entries() const {
    if (p.whole) {
      entry(lane, 0, 0);
      if (n > 64) entry(64 + lane, 0, 64);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) entry(i, lane & 15, 64 * i);
    }
  }
  __device__ __forceinline__ void more_entries(int i) const {
    if (!p.whole)
      entry(i + 4, lane & 15, 64 * (i & 3));
    else if (i > 0 && (i & 63) == 0)
      entry(i + 64 + lane, 0, (i + 64) & 64);
  }
  // The copies of tile i; returns its keys in the pool, one bit each.
  __device__ __forceinline__ uint32_t tile(int i) const {
    char* stage = stages + (i & 1) * T::kStage;
    const int key = key_of(i);
    int at;
    if (p.whole) {
      const int e = scalar(s_ent[i & 127]);
      const int slot = key - div_by(key, p.block_div) * p.block_size;
      const int valid = e >= 0 && e < p.num_pool_blocks ? min(len - key, 16) : 0;
      const int64_t row = (int64_t)e * p.block_size + slot;
      if (valid == 16 && p.d_chunks == T::kChunks) {
        const char* kb = kbase + row * p.row_bytes;
        const char* vb = vbase + row * p.row_bytes;
        const uint32_t dst = lds_addr(stage) + 16 * w * T::kRow;
#pragma unroll
        for (int q = 0; q < T::kCopies; ++q) {
          // rows 4 on of every 8: the other half of the permutation (head_dim is kD: a row is a
          // multiple of 256 bytes)
          const bool odd = kD == 128 && (q & 1);
          lds_copy16_base<kOnce>(kb, odd ? k_off ^ 32 : k_off, dst + 1024 * q);
          lds_copy16_base<kOnce>(vb, odd ? v_off ^ 128 : v_off, dst + T::kBytes + 1024 * q);
          kb += T::kCopyRows * p.row_bytes;
          vb += T::kCopyRows * p.row_bytes;
        }
        return 0xffffu;
      }
      at = (lane & 15) < valid ? (int)row + (lane & 15) : -1;
    } else {
      const int mine = key + (lane & 15);
      const int slot = mine - div_by(mine, p.block_div) * p.block_size;
      const int e = s_ent[64 * (i & 3) + lane];
      at = e >= 0 && e < p.num_pool_blocks ? e * p.block_size + slot : -1;
    }
    issue_tile<kD, kOnce>(p, kbase, vbase, stage, at, 0, w, lane);
    return (uint32_t)__builtin_amdgcn_ballot_w64(at >= 0) & 0xffffu;
  }
};

// A slice of 16 kT keys (kT = 4, 2 or 1) is what one step of the softmax covers.  P and V^T fragments
// hold 4 kT keys a lane: keys 16 t + 4g + j (j = 0..3) in slots 4 t + j.
typedef _Float16 half16 __attribute__((ext_vector_type(16)));
template <int kT>
struct Slice;
template <>
struct Slice<4> {
  typedef half16 frag;
  static __device__ __forceinline__ floatx4 mfma(half16 a, half16 b, floatx4 c) {
    return mfma16x16x32(__builtin_shufflevector(a, a, 8, 9, 10, 11, 12, 13, 14, 15),
                        __builtin_shufflevector(b, b, 8, 9, 10, 11, 12, 13, 14, 15),
                        mfma16x16x32(__builtin_shufflevector(a, a, 0, 1, 2, 3, 4, 5, 6, 7),
                                     __builtin_shufflevector(b, b, 0, 1, 2, 3, 4, 5, 6, 7), c));
  }
};
template <>
struct Slice<2> {
  typedef half8 frag;
  static __device__ __forceinline__ floatx4 mfma(half8 a, half8 b, floatx4 c) { return mfma16x16x32(a, b, c); }
};
template <>
struct Slice<1> {
  typedef half4 frag;
  static __device__ __forceinline__ floatx4 mfma(half4 a, half4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
  }
};
template <int kT>
__device__ __forceinline__ typename Slice<kT>::frag splat(float x) {
  typename Slice<kT>::frag f;
#pragma unroll
  for (int e = 0; e < 4 * kT; ++e) f[e] = (half_t)x;
  return f;
}

// V^T fragment of slice c: lane (col, g) receives its keys of column 16 dt + col.  vs: LDS address
// of the V tile at this lane's place for dt = 0 (v_lane).
template <int kD>
__device__ __forceinline__ int v_lane(int col, int g) {
  const int r = 4 * g + (col >> 2);
  return r * Tile<kD>::kRow + ((((col & 3) >> 1) ^ Tile<kD>::xv(r)) << 4) + ((col & 1) << 3);
}
template <int kD, int kT>
__device__ __forceinline__ typename Slice<kT>::frag vt_frag(uint32_t vs, int c, int dt) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  typedef s4 __attribute__((address_space(3))) * lds_s4;
  if constexpr (kT == 1) {
    const uint32_t at = (vs ^ (dt << 5)) + 16 * c * Tile<kD>::kRow;
    return __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)at));
  } else if constexpr (kT == 2) {
    return __builtin_shufflevector(vt_frag<kD, 1>(vs, 2 * c, dt), vt_frag<kD, 1>(vs, 2 * c + 1, dt), 0, 1, 2, 3, 4,
                                   5, 6, 7);
  } else {
    return __builtin_shufflevector(vt_frag<kD, 2>(vs, 2 * c, dt), vt_frag<kD, 2>(vs, 2 * c + 1, dt), 0, 1, 2, 3, 4,
                                   5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15);
  }
}

// K fragment: lane (col, g) receives columns 32 i + 8 g .. + 7 of key 16 kt + col.
template <int kD>
__device__ __forceinline__ int k_lane(int col, int g) {
  return col * Tile<kD>::kRow + ((g ^ Tile<kD>::xk(col)) << 4);
}
template <int kD>
__device__ __forceinline__ half8 k_frag(uint32_t ks, int kt, int i) {
  typedef u32x4 __attribute__((address_space(3))) * lds_u4;
  return as_half8(*(lds_u4)((ks ^ (i << 6)) + 16 * kt * Tile<kD>::kRow));
}

// S^T = K Q^T + init for slice c: s[j][t] holds keys 16 (kT c + t) + 4g + r of row block j.  With one
// row block a fragment feeds one product only, and waiting for each read in turn is what a slice
// takes: all reads go first.  With more, one step ahead.
template <int NB, int kD, int kT>
__device__ __forceinline__ void qk_slice(uint32_t ks, int c, const half8 (&qf)[NB][kD / 32],
                                         floatx4 (&s)[NB][kT]) {
  constexpr int kI = kD / 32, kN = kT * kI;
  if constexpr (NB == 1) {
    half8 f[kN];
#pragma unroll
    for (int u = 0; u < kN; ++u) f[u] = k_frag<kD>(ks, kT * c + u / kI, u % kI);
#pragma unroll
    for (int u = 0; u < kN; ++u) s[0][u / kI] = mfma16x16x32(f[u], qf[0][u % kI], s[0][u / kI]);
  } else {
    half8 cur = k_frag<kD>(ks, kT * c, 0);
#pragma unroll
    for (int u = 0; u < kN; ++u) {
      half8 nxt;
      if (u + 1 < kN) nxt = k_frag<kD>(ks, kT * c + (u + 1) / kI, (u + 1) % kI);
#pragma unroll
      for (int j = 0; j < NB; ++j) s[j][u / kI] = mfma16x16x32(cur, qf[j][u % kI], s[j][u / kI]);
      if (u + 1 < kN) cur = nxt;
    }
  }
}

// O^T += V^T P^T of slice c, and the sums of P (last accumulator tile, all-ones A).
template <int NB, int kD, int kT>
__device__ __forceinline__ void pv_slice(uint32_t vs, int c, const typename Slice<kT>::frag (&pf)[NB],
                                         floatx4 (&acc)[NB][kD / 16 + 1]) {
  constexpr int kN = kD / 16;
  typename Slice<kT>::frag vf = vt_frag<kD, kT>(vs, c, 0);
#pragma unroll
  for (int dt = 0; dt < kN; ++dt) {
    typename Slice<kT>::frag vn;
    if (dt + 1 < kN) vn = vt_frag<kD, kT>(vs, c, dt + 1);
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[j][dt] = Slice<kT>::mfma(vf, pf[j], acc[j][dt]);
    if (dt + 1 < kN) vf = vn;
  }
#pragma unroll
  for (int j = 0; j < NB; ++j) acc[j][kN] = Slice<kT>::mfma(splat<kT>(1.f), pf[j], acc[j][kN]);
}
// The same for one row block, from fragments read before the softmax.
template <int kD, int kT>
__device__ __forceinline__ void pv_read(const typename Slice<kT>::frag (&vf)[kD / 16],
                                        typename Slice<kT>::frag pf, floatx4 (&acc)[kD / 16 + 1]) {
#pragma unroll
  for (int dt = 0; dt < kD / 16; ++dt) acc[dt] = Slice<kT>::mfma(vf[dt], pf, acc[dt]);
  acc[kD / 16] = Slice<kT>::mfma(splat<kT>(1.f), pf, acc[kD / 16]);
}

// Infinities and NaN in V.  In the matrix product a value that a row does not see has weight 0, and
// 0 * inf would reach that row.  Tiles that some row may not see whole are therefore looked over
// first: each wave those 16 keys of V that it copied (bad_keys, a bit per key).  Where there are
// any, scrub() replaces such values by zeros and notes them, a bit per column, as +inf (or NaN)
// and -inf (or NaN); note_row() collects those that a row sees, and mark4() / mark8() put them
// into its output at the end (both: NaN).  (Put into the accumulators at once they cost the loops
// their registers.)
template <int kD>
struct Notes {
  uint8_t bit[2][kD / 8];  // of one key or row: +inf or NaN, -inf or NaN
};
template <int kD>
__device__ __forceinline__ uint32_t bad_keys(uint32_t v, int lane) {  // v: V of the wave's keys in LDS
  typedef u32x4 __attribute__((address_space(3))) * lds_u4;
  typedef Tile<kD> T;
  u32x4 x[T::kCopies];
#pragma unroll
  for (int q = 0; q < T::kCopies; ++q) x[q] = *(lds_u4)(v + 1024 * q + 16 * lane);
  uint32_t bad[T::kCopies], any = 0;
#pragma unroll
  for (int q = 0; q < T::kCopies; ++q) {
    bad[q] = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) bad[q] |= (x[q][e] & 0x7c007c00u) + 0x04000400u;  // carries where all ones
    bad[q] &= 0x80008000u;
    any |= bad[q];
  }
  if (__builtin_amdgcn_ballot_w64(any != 0) == 0) return 0;
  uint32_t keys = 0;
#pragma unroll
  for (int q = 0; q < T::kCopies; ++q) {
    const uint64_t m = __builtin_amdgcn_ballot_w64(bad[q] != 0);
    for (int r = 0; r < T::kCopyRows; ++r)
      if ((m >> (r * T::kChunks)) & ((1u << T::kChunks) - 1)) keys |= 1u << (q * T::kCopyRows + r);
  }
  return keys;
}
template <int kD>
__device__ __forceinline__ void scrub(uint32_t v, Notes<kD>* notes, int lane) {  // notes: of the wave's keys
  typedef unsigned short us8 __attribute__((ext_vector_type(8)));
  typedef us8 __attribute__((address_space(3))) * lds_us8;
  typedef Tile<kD> T;
  for (int q = 0; q < T::kCopies; ++q) {
    const lds_us8 at = (lds_us8)(v + 1024 * q + 16 * lane);
    us8 x = *at;
    uint32_t up = 0, down = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned short m = x[e] & 0x7fff;
      if (m > 0x7c00 || x[e] == 0x7c00) up |= 1u << e;
      if (m > 0x7c00 || x[e] == 0xfc00) down |= 1u << e;
      if (m >= 0x7c00) x[e] = 0;
    }
    *at = x;
    const int r = q * T::kCopyRows + lane / T::kChunks, c = (lane % T::kChunks) ^ T::xv(r);
    notes[r].bit[0][c] = (uint8_t)up;
    notes[r].bit[1][c] = (uint8_t)down;
  }
}
// Of the keys in `bad` (bit k: key k0 + k), those that a row at `pos` (-1: no token) sees.
__device__ __forceinline__ uint64_t bad_seen(const Params& p, uint64_t bad, int k0, int prefix, int pos) {
  uint64_t seen = 0;
  if (pos < 0) return 0;
  for (; bad; bad &= bad - 1) {
    const int k = __builtin_ctzll(bad), key = k0 + k;
    if (key < prefix || (key <= pos && key > pos - p.window)) seen |= 1ull << k;
  }
  return seen;
}
template <int kD>
__device__ __forceinline__ void note_row(const Notes<kD>* keys, uint64_t seen, Notes<kD>* row) {
  for (; seen; seen &= seen - 1) {
    const uint32_t* from = (const uint32_t*)&keys[__builtin_ctzll(seen)];
    for (int i = 0; i < (int)sizeof(Notes<kD>) / 4; ++i) atomicOr((uint32_t*)row + i, from[i]);
  }
}
__device__ __forceinline__ float mark(float x, uint32_t up, uint32_t down) {
  float a = up ? __builtin_inff() : 0.f, b = down ? -__builtin_inff() : 0.f;
  // the file is compiled for NaN-free arithmetic: these sums have to be taken, not folded
  asm volatile("" : "+v"(a), "+v"(b));
  return (x + a) + b;
}
template <int kD>
__device__ __forceinline__ floatx4 mark4(const Notes<kD>& row, int d, floatx4 v) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
    v[r] = mark(v[r], (row.bit[0][(d + r) >> 3] >> ((d + r) & 7)) & 1, (row.bit[1][(d + r) >> 3] >> ((d + r) & 7)) & 1);
  return v;
}
template <int kD>
__device__ __forceinline__ u32x4 mark8(const Notes<kD>& row, int chunk, u32x4 v) {
  half8 h = as_half8(v);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    h[e] = (half_t)mark((float)h[e], (row.bit[0][chunk] >> e) & 1, (row.bit[1][chunk] >> e) & 1);
  return as_u32x4(h);
}

// Capped scores in units of 2 cap: cap tanh(y) = cap - 2 cap / (1 + e^2y), and the softmax does not
// change by a constant, so -1 / (1 + e^2y) will do (y = s * sm_scale / cap).
__device__ __forceinline__ float capped(const Params& p, float s) {
  return -__builtin_amdgcn_rcpf(1.f + fast_exp2(s * p.cap_exp));
}
// The same for large caps, where the absolute error of that form would show: tanh(y) / 2, below 1/4
// from its series (the next term is under 2e-8).
__device__ __forceinline__ float capped_series(const Params& p, float s) {
  const float y = s * (p.cap_exp * (0.5f / kLog2e)), z = y * y;
  float t = __builtin_fmaf(z, 62.f / 2835.f, -17.f / 315.f);
  t = __builtin_fmaf(z, t, 2.f / 15.f);
  t = __builtin_fmaf(z, t, -1.f / 3.f);
  t = __builtin_fmaf(z * y, t, y);
  return __builtin_fabsf(y) < 0.25f ? 0.5f * t : 0.5f + capped(p, s);
}

// kSlices slices of 16 kT resident keys (k0 on) for this wave's rows.  s_pos, s_slope: of the wave's
// rows; keys: bit k is set when key k0 + k is before the row's length and in the pool; kMasked:
// some row may not see some key.
template <int NB, int kD, int kMod, int kT, int kSlices, bool kMasked>
__device__ __forceinline__ void consume(const Params& p, uint32_t ks, uint32_t vs, int k0, uint64_t keys,
                                        int prefix, const int* s_pos, const float* s_slope, int col,
                                        int g, const half8 (&qf)[NB][kD / 32], float (&t_run)[NB],
                                        floatx4 (&acc)[NB][kD / 16 + 1]) {
  typedef typename Slice<kT>::frag frag;
  constexpr uint64_t kAll = ~0ull >> (64 - 16 * kT * kSlices);
  constexpr int kE = 4 * kT;  // scores of a lane and row block
#pragma unroll
  for (int c = 0; c < kSlices; ++c) {
    // a uniform branch, never taken, between the slices: without it the compiler overlaps the
    // unrolled slices beyond the register file
    if (p.chunk < 0) break;
    const int key0 = k0 + 16 * kT * c + 4 * g;  // lane's key of score e: key0 + 16 (e / 4) + e % 4
    floatx4 s[NB][kT];
    // -slope |pos - key|; where every key is before its row (!kMasked) the difference is linear
    float slope[NB], back0[NB];
    if (kMod & kBias) {
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        slope[j] = s_slope[16 * j + col];
        back0[j] = (float)(s_pos[16 * j + col] - key0) * (kMasked ? 1.f : -slope[j]);
      }
    }
    auto bias = [&](int j, int e) {
      const float at = (float)(16 * (e >> 2) + (e & 3));
      return kMasked ? -slope[j] * __builtin_fabsf(back0[j] - at) : __builtin_fmaf(slope[j], at, back0[j]);
    };
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int e = 0; e < kE; ++e) s[j][e >> 2][e & 3] = kMod == kBias ? bias(j, e) : 0.f;
    qk_slice<NB, kD, kT>(ks, c, qf, s);
    frag vf[kD / 16];
    if constexpr (NB == 1) {
#pragma unroll
      for (int dt = 0; dt < kD / 16; ++dt) vf[dt] = vt_frag<kD, kT>(vs, c, dt);
    }
    if (kMod & kCap) {
      const bool series = p.scale_log2 > kExpCap * (2.f * kLog2e);
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        if (series) {
#pragma unroll
          for (int e = 0; e < kE; ++e) s[j][e >> 2][e & 3] = capped_series(p, s[j][e >> 2][e & 3]);
        } else {
#pragma unroll
          for (int e = 0; e < kE; ++e) s[j][e >> 2][e & 3] = capped(p, s[j][e >> 2][e & 3]);
        }
        if (kMod & kBias) {
#pragma unroll
          for (int e = 0; e < kE; ++e) s[j][e >> 2][e & 3] += bias(j, e);
        }
      }
    }
    if (kMasked) {
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        // without branches: as conditions they took three times a full tile's time
        const int back = s_pos[16 * j + col] - key0, ahead = prefix - key0;
        const uint64_t here = keys >> (16 * kT * c) >> (4 * g);
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const int at = 16 * (e >> 2) + (e & 3);
          const bool see = (((uint32_t)(back - at) < (uint32_t)p.window) | (ahead > at)) &
                           (((uint32_t)(here >> (at & 32)) >> (at & 31) & 1) != 0);
          s[j][e >> 2][e & 3] = see ? s[j][e >> 2][e & 3] : -__builtin_inff();
        }
      }
    } else if (keys != kAll) {  // missing table entries
      const uint64_t here = keys >> (16 * kT * c) >> (4 * g);
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int e = 0; e < kE; ++e)
          if (!((here >> (16 * (e >> 2) + (e & 3))) & 1)) s[j][e >> 2][e & 3] = -__builtin_inff();
    }
    // Online softmax with a lazily moved reference max, kept as the threshold t = max + slack in
    // score units: it moves only when a score exceeds it (p <= 2^8, exact in fp16; sums in fp32).
    bool move = false;
    float lmax[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      lmax[j] = fmaxf(fmaxf(s[j][0][0], s[j][0][1]), fmaxf(s[j][0][2], s[j][0][3]));
#pragma unroll
      for (int t = 1; t < kT; ++t)
        lmax[j] = fmaxf(fmaxf(fmaxf(s[j][t][0], s[j][t][1]), fmaxf(s[j][t][2], s[j][t][3])), lmax[j]);
      move |= lmax[j] > t_run[j];
    }
    if (__builtin_amdgcn_ballot_w64(move)) {
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const float t_old = t_run[j];
        const float rmax = row4_max(lmax[j]);
        const float t_new = rmax > t_old ? rmax + p.lazy_raw : t_old;
        const float alpha = fast_exp2((t_old - t_new) * p.scale_log2);
        t_run[j] = t_new;
#pragma unroll
        for (int dt = 0; dt <= kD / 16; ++dt) acc[j][dt] *= alpha;
      }
    }
    // P is rounded to fp16 for the matrix cores; the sums take the rounded values too.
    frag pf[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const float mc = __builtin_fmaf(t_run[j], p.scale_log2, -p.lazy_log2);
#pragma unroll
      for (int e = 0; e < kE; ++e)
        pf[j][e] = (half_t)fast_exp2(__builtin_fmaf(s[j][e >> 2][e & 3], p.scale_log2, -mc));
    }
    if constexpr (NB == 1)
      pv_read<kD, kT>(vf, pf[0], acc[0]);
    else
      pv_slice<NB, kD, kT>(vs, c, pf, acc);
  }
}

// Q^T fragments of the wave's row blocks, rows r0 on (MFMA i takes d = 32 i + 8 g + s in reduction
// slot 8 g + s), and their positions and biases into LDS.
template <int NB, int kD, int kMod>
__device__ __forceinline__ void load_rows(const Params& p, const Row& row, int b, int kvh, int r0, int col,
                                          int g, half8 (&qf)[NB][kD / 32], int* s_pos, float* s_slope) {
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int r = r0 + 16 * j + col;
    const int t = div_by(r, p.group_div);
    const int h = kvh * p.group + r - t * p.group;
    const int pos = row.start + t;
    const bool ok = t < p.chunk && pos >= 0 && pos < row.len;
    const half_t* src = p.q + (int64_t)b * p.q_sb + (int64_t)(ok ? t : 0) * p.q_st + (int64_t)h * p.q_sh;
#pragma unroll
    for (int i = 0; i < kD / 32; ++i) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (ok && !p.q_zero && 32 * i + 8 * g < p.head_dim) v = *(const u32x4*)(src + 32 * i + 8 * g);
      qf[j][i] = as_half8(v ^ p.q_sign);
    }
    if (g == 0) {
      s_pos[16 * j + col] = ok ? pos : -1;
      if (kMod & kBias) s_slope[16 * j + col] = p.slopes[h] * p.slope_mul;
    }
  }
}

// The part of the work of a workgroup: its batch row, row tile and key tiles first .. first + n - 1 of
// the span's order.  False where there is nothing to do.
struct Job {
  int b, kvh, r0, parts, first, n;
  Row row;
  Span span;
};
__device__ __forceinline__ bool find_job(const Params& p, int tid, int tile_rows, int* s_tiles, Job& job) {
  const int item = div_by(blockIdx.x, p.kv_div);
  job.kvh = blockIdx.x - item * p.num_kv_heads;
  int tile, part = 0;
  job.parts = 1;
  if (p.part_o) {
    const Share s = find_share(p, item, tid, s_tiles);
    if (s.b < 0) return false;  // past the list
    job.b = s.b;
    const RowTiles rt = row_tiles_of(p, row_of(p, job.b));
    int at = item - s.before;
    if (at == 0 && job.kvh == 0 && tid < 2) p.shares[2 * job.b + tid] = tid ? s.parts : s.before;
    if (at < rt.count * s.parts) {
      part = scalar(whole_of(at, rt.count));
      job.parts = s.parts;
      tile = rt.first + rt.count - 1 - (at - part * rt.count);
    } else {  // a row tile without tokens
      at -= rt.count * s.parts;
      tile = at < rt.first ? at : at + rt.count;
    }
  } else {  // the last row tiles see the most keys: first
    const int back = div_by(item, p.batch_div);
    job.b = item - back * p.batch;
    tile = p.row_tiles - 1 - back;
  }
  job.b = scalar(job.b);
  job.parts = scalar(job.parts);
  part = scalar(part);
  job.r0 = scalar(tile) * tile_rows;
  job.row = row_of(p, job.b);
  int lo, hi;
  row_positions(p, job.row, job.r0, job.r0 + tile_rows - 1, lo, hi);
  job.span = span_of(p, job.row, lo, hi);
  const int size =
      job.parts == 1 ? job.span.n
                     : scalar(parts_of(job.span.n, inverse(job.parts)));
  job.first = min(part * size, job.span.n);
  job.n = min(size, job.span.n - job.first);
  // a short list in few pieces: the other kernel reads no more
  return job.parts == 1 || job.n > 0;
}

// Many rows: the waves share the tiles, each with 16 NB rows of its own, so that a tile read once
// from memory and a fragment read once from LDS serve many.  Bound by the matrix cores and the
// softmax, which the two workgroups of a CU overlap in part: a tile of three blocks takes 2780
// cycles, 1632 of them MFMA (16384 keys; the two together 1.06 PFLOP/s, the library's largest fp16
// products 1.2 to 1.45).  A cap adds an exp2 and a reciprocal a score, about a third.
template <int NB, int kD, int kMod>
__global__ __launch_bounds__(kThreads, kD == 64 ? 3 : 2) void chunk_kernel(Params p) {
  typedef Tile<kD> T;
  constexpr int kRowsPerWave = 16 * NB;
  constexpr int kRows = kWaves * kRowsPerWave;
  // Two slices a tile, or one where the registers allow it, whose steps wait for one another half as
  // often: one row block, 777 tokens of 3 rows, 64 wide, 23 -> 20.7 us, a prompt of 2000 51 -> 49; two blocks,
  // 128 wide, 4096 tokens 129 -> 122, 4 x 1000 at 5000 with biases 349 -> 324 (64 wide 60.4 -> 61.6).  With a
  // cap 27 -> 39 for 250 tokens at 1500 and 68 -> 77 for 2 x 1000.
  constexpr bool kOne = (NB == 1 || (NB == 2 && kD == 128)) && !(kMod & kCap);
  constexpr int kT = kOne ? 4 : 2;
  __shared__ __attribute__((aligned(16))) char stages[2 * T::kStage];
  __shared__ int s_pos[kRows];  // position of each query row, -1 for rows without a token
  __shared__ float s_slope[kMod & kBias ? kRows : 1];  // its distance bias in score units
  __shared__ int s_ent[kWaves][256];
  __shared__ __attribute__((aligned(8))) uint16_t s_keys[2][kWaves], s_bad[kWaves];
  __shared__ Notes<kD> s_notes[kKTile];    // of the keys of a tile,
  __shared__ Notes<kD> s_rows[kRows];      // of the rows, where `noted`

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15;
  const int g = lane >> 4;
  Job job;
  if (!find_job(p, tid, kRows, (int*)stages, job)) return;
  const int b = job.b, kvh = job.kvh, r0 = job.r0, first = job.first, n = job.n;
  const Row& row = job.row;
  const Span& span = job.span;

  const Copier<kD, false> copies(p, span, first, n, row.len, b, kvh, w, lane, stages, s_ent[w]);
  auto copy_tile = [&](int i) {
    const uint32_t there = copies.tile(i);
    if (lane == 0) s_keys[i & 1][w] = (uint16_t)there;
  };
  copies.first_entries();
  int wlo, whi;  // positions of this wave's tokens
  row_positions(p, row, r0 + kRowsPerWave * w, r0 + kRowsPerWave * (w + 1) - 1, wlo, whi);

  float t_run[NB];
  floatx4 acc[NB][kD / 16 + 1];  // O^T columns 16dt .. 16dt + 15, then the sum of P
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    t_run[j] = kNegBig;
#pragma unroll
    for (int dt = 0; dt <= kD / 16; ++dt) acc[j][dt] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  wait_copies<0>();
  copy_tile(0);
  copy_tile(1);
  half8 qf[NB][kD / 32];
  int* w_pos = s_pos + kRowsPerWave * w;
  float* w_slope = s_slope + (kMod & kBias ? kRowsPerWave * w : 0);
  load_rows<NB, kD, kMod>(p, row, b, kvh, r0 + kRowsPerWave * w, col, g, qf, w_pos, w_slope);
  stage_barrier();

  // Tile i lies in stage i % 2.  While it is consumed, tile i + 1 is copied into the other stage
  // (whose readers have passed the last barrier).
  auto copy_next = [&](int i) -> uint64_t {  // the keys of tile i
    const uint64_t keys = uniform64(s_keys[i & 1]);
    copies.more_entries(i);
    if (i > 0) copy_tile(i + 1);  // the first two are on their way
    return keys;
  };
  const uint32_t ks = lds_addr(stages) + k_lane<kD>(col, g);
  const uint32_t vs = lds_addr(stages) + T::kBytes + v_lane<kD>(col, g);
  int i = 0;
  const uint32_t v_own = lds_addr(stages) + T::kBytes + 16 * w * T::kRow;  // V of the keys it copies
  bool noted = false;
  for (const int end = min(max(span.masked() - first, 0), n); i < end; ++i) {
    const uint64_t keys = copy_next(i);
    const int at = (i & 1) * T::kStage;
    const uint32_t mine = bad_keys<kD>(v_own + at, lane);
    if (lane == 0) s_bad[w] = (uint16_t)mine;
    lds_barrier();
    const uint64_t bad = uniform64(s_bad);
    const int k0 = span.tile(first + i) * kKTile;
    if (bad) {
      scrub<kD>(v_own + at, s_notes + 16 * w, lane);
      lds_barrier();
      if (lane < kRowsPerWave) {
        Notes<kD>& r = s_rows[kRowsPerWave * w + lane];
        if (!noted) r = Notes<kD>{};
        note_row<kD>(s_notes, bad_seen(p, bad & keys, k0, row.prefix, w_pos[lane]), &r);
      }
      noted = true;
    }
    if (wlo <= whi && (k0 < row.prefix || (k0 <= whi && k0 + kKTile > wlo - p.window + 1)))
      consume<NB, kD, kMod, kT, 4 / kT, true>(p, ks + at, vs + at, k0, keys, row.prefix, w_pos, w_slope, col, g, qf,
                                        t_run, acc);
    stage_barrier();
  }
  for (; i < n; ++i) {
    const uint64_t keys = copy_next(i);
    if (wlo <= whi)
      consume<NB, kD, kMod, kT, 4 / kT, false>(p, ks + (i & 1) * T::kStage, vs + (i & 1) * T::kStage,
                                         span.tile(first + i) * kKTile, keys, row.prefix, w_pos, w_slope,
                                         col, g, qf, t_run, acc);
    stage_barrier();
  }

  if (job.parts > 1) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int rl = kRowsPerWave * w + 16 * j + col;
      if (w_pos[16 * j + col] < 0) continue;
      const int64_t slot = (int64_t)blockIdx.x * p.part_rows + rl;
#pragma unroll
      for (int dt = 0; dt < kD / 16; ++dt) {
        floatx4 v = acc[j][dt];
        if (noted) v = mark4<kD>(s_rows[rl], 16 * dt + 4 * g, v);
        *(floatx4*)(p.part_o + slot * kD + 16 * dt + 4 * g) = v;
      }
      if (g == 0) {
        p.part_ml[slot * 2] = __builtin_fmaf(t_run[j], p.scale_log2, -p.lazy_log2);
        p.part_ml[slot * 2 + 1] = acc[j][kD / 16][0];
      }
    }
    return;
  }

  // Normalise; the rows go through this wave's part of the stages (idle since the last barrier)
  // so that each store instruction writes whole rows.  Rows are padded by 16 bytes: the 16 rows of
  // one write land in distinct banks.
  constexpr int kORow = T::kRow + 16;
  static_assert(kWaves * kRowsPerWave * kORow <= 2 * T::kStage, "output rows fit the stages");
  char* ostage = stages + w * kRowsPerWave * kORow;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const float l = acc[j][kD / 16][0];
    const float inv = w_pos[16 * j + col] >= 0 && __builtin_bit_cast(uint32_t, l) != 0 ? 1.f / l : 0.f;
    char* orow = ostage + (16 * j + col) * kORow + 8 * g;
#pragma unroll
    for (int dt = 0; dt < kD / 16; ++dt) *(half4*)(orow + 32 * dt) = to_half4(acc[j][dt] * inv);
  }
  wave_lds_sync();
  const int orl = lane / T::kChunks, oc = lane % T::kChunks;
#pragma unroll
  for (int rr = 0; rr < kRowsPerWave / T::kCopyRows; ++rr) {
    const int rl = T::kCopyRows * rr + orl;
    const int r = r0 + kRowsPerWave * w + rl;
    const int t = div_by(r, p.group_div);
    const int h = kvh * p.group + r - t * p.group;
    u32x4 v = *(const u32x4*)(ostage + rl * kORow + 16 * oc);
    if (noted) v = mark8<kD>(s_rows[kRowsPerWave * w + rl], oc, v);
    if (t < p.chunk && oc < p.d_chunks)
      *(u32x4*)(p.o + (int64_t)b * p.o_sb + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + 8 * oc) = v;
  }
}

// Few rows (at most 16 NB): every wave has all of them and takes 16 keys of each tile, those that it
// copies itself, so the waves run without barriers, each waiting for its own copies only, and
// are added up through LDS at the end.  Bound by the stream of K and V, which a kv head reads in
// slices of 256 bytes (5.2 to 5.8 TB/s for such a read alone): 24 rows of 5 drafted tokens, 203 MB, 39 us
// of which about 6 pass before the first tile (the work list, the table, the first copies), 32 single
// capped tokens, 335 MB, 62; 2.9 TB/s when the waves shared the tiles as in chunk_kernel.
template <int NB, int kD, int kMod>
__global__ __launch_bounds__(kThreads, kD == 64 ? 4 : 2) void narrow_kernel(Params p) {
  typedef Tile<kD> T;
  constexpr int kRows = 16 * NB;
  __shared__ __attribute__((aligned(16))) char stages[2 * T::kStage];
  __shared__ int s_ent[kWaves][256];
  __shared__ int s_pos[kWaves][kRows];
  __shared__ float s_slope[kWaves][kMod & kBias ? kRows : 1];
  __shared__ float s_ml[kWaves][kRows][2];
  __shared__ Notes<kD> s_notes[kWaves][16];  // of the keys of a wave's tile,
  __shared__ Notes<kD> s_rows[kRows];        // of the rows, where s_noted
  __shared__ int s_noted;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15;
  const int g = lane >> 4;
  Job job;
  if (!find_job(p, tid, kRows, (int*)stages, job)) return;
  const int b = job.b, kvh = job.kvh, r0 = job.r0, first = job.first, n = job.n;
  const Row& row = job.row;
  const Span& span = job.span;

  const Copier<kD, true> copies(p, span, first, n, row.len, b, kvh, w, lane, stages, s_ent[w]);
  copies.first_entries();
  wait_copies<0>();
  uint32_t keys = 0, keys_next = 0;
  if (n > 0) keys = copies.tile(0);
  if (n > 1) keys_next = copies.tile(1);
  half8 qf[NB][kD / 32];
  load_rows<NB, kD, kMod>(p, row, b, kvh, r0, col, g, qf, s_pos[w], s_slope[w]);
  if (tid < kRows) s_rows[tid] = Notes<kD>{};
  if (tid == 0) s_noted = 0;
  // Q and the first tiles have landed, also for the compiler, which would otherwise wait for every
  // copy at the first use of Q
  wait_vmcnt<0>();
  lds_barrier();

  float t_run[NB];
  floatx4 acc[NB][kD / 16 + 1];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    t_run[j] = kNegBig;
#pragma unroll
    for (int dt = 0; dt <= kD / 16; ++dt) acc[j][dt] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t ks = lds_addr(stages) + 16 * w * T::kRow + k_lane<kD>(col, g);
  const uint32_t vs = lds_addr(stages) + T::kBytes + 16 * w * T::kRow + v_lane<kD>(col, g);
  auto arrive = [&](int i) {  // tile i; tile i + 1 is on its way
    if (i + 1 < n)
      wait_copies<2 * T::kCopies>();
    else
      wait_copies<0>();
  };
  auto advance = [&](int i) {
    keys = keys_next;
    if (i + 2 < n) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the reads of this stage are done
      copies.more_entries(i);
      keys_next = copies.tile(i + 2);
    }
  };
  int i = 0;
  const uint32_t v_own = lds_addr(stages) + T::kBytes + 16 * w * T::kRow;
  for (const int end = min(max(span.masked() - first, 0), n); i < end; ++i) {
    arrive(i);
    const int at = (i & 1) * T::kStage;
    const int k0 = span.tile(first + i) * kKTile + 16 * w;
    const uint32_t bad = bad_keys<kD>(v_own + at, lane);
    if (bad) {
      scrub<kD>(v_own + at, s_notes[w], lane);
      wave_lds_sync();
      if (lane < kRows)
        note_row<kD>(s_notes[w], bad_seen(p, bad & keys, k0, row.prefix, s_pos[w][lane]), &s_rows[lane]);
      if (lane == 0) s_noted = 1;
      wave_lds_sync();
    }
    consume<NB, kD, kMod, 1, 1, true>(p, ks + at, vs + at, k0, keys, row.prefix, s_pos[w], s_slope[w], col, g,
                                      qf, t_run, acc);
    advance(i);
  }
  for (; i < n; ++i) {
    arrive(i);
    consume<NB, kD, kMod, 1, 1, false>(p, ks + (i & 1) * T::kStage, vs + (i & 1) * T::kStage,
                                       span.tile(first + i) * kKTile + 16 * w, keys, row.prefix, s_pos[w],
                                       s_slope[w], col, g, qf, t_run, acc);
    advance(i);
  }

  // Add the waves up, one row block at a time: O and the sums relative to the waves' own maxima.
  // (Rows padded by 16 bytes: the 16 rows of one write would share a bank.)
  constexpr int kPad = kD + 4;
  float* cmb = (float*)stages;  // [wave][16][kPad]
  static_assert(kWaves * 16 * kPad * 4 <= 2 * T::kStage, "a row block of every wave fits the stages");
  if (g == 0) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      s_ml[w][16 * j + col][0] = __builtin_fmaf(t_run[j], p.scale_log2, -p.lazy_log2);
      s_ml[w][16 * j + col][1] = acc[j][kD / 16][0];
    }
  }
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    if (r0 + 16 * j >= p.chunk * p.group) break;
    __syncthreads();
#pragma unroll
    for (int dt = 0; dt < kD / 16; ++dt)
      *(floatx4*)(cmb + (w * 16 + col) * kPad + 16 * dt + 4 * g) = acc[j][dt];
    __syncthreads();
    for (int x = tid; x < 16 * kD / 4; x += kThreads) {
      const int c = x / (kD / 4), d = x % (kD / 4) * 4;
      const int rl = 16 * j + c, r = r0 + rl;
      const int t = div_by(r, p.group_div);
      if (t >= p.chunk) continue;
      float m = kNegBig;
#pragma unroll
      for (int ww = 0; ww < kWaves; ++ww)
        if (__builtin_bit_cast(uint32_t, s_ml[ww][rl][1]) != 0) m = fmaxf(m, s_ml[ww][rl][0]);
      float l = 0.f;
      floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ww = 0; ww < kWaves; ++ww) {
        const float lw = s_ml[ww][rl][1];
        if (__builtin_bit_cast(uint32_t, lw) == 0) continue;  // saw no key (a NaN is not 0)
        const float e = fast_exp2(s_ml[ww][rl][0] - m);
        l += lw * e;
        o += *(const floatx4*)(cmb + (ww * 16 + c) * kPad + d) * e;
      }
      if (s_noted) o = mark4<kD>(s_rows[rl], d, o);
      const bool there = s_pos[0][rl] >= 0;
      if (job.parts > 1) {
        if (!there) continue;
        const int64_t slot = (int64_t)blockIdx.x * p.part_rows + rl;
        *(floatx4*)(p.part_o + slot * kD + d) = o;
        if (d == 0) {
          p.part_ml[slot * 2] = m;
          p.part_ml[slot * 2 + 1] = l;
        }
      } else if (d < p.head_dim) {
        const float inv = there && __builtin_bit_cast(uint32_t, l) != 0 ? 1.f / l : 0.f;
        const int h = kvh * p.group + r - t * p.group;
        *(half4*)(p.o + (int64_t)b * p.o_sb + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + d) =
            to_half4(o * inv);
      }
    }
  }
}

// Adds the parts of each query row: o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s.  Four
// columns a lane; grid (rows of a batch row, batch).  Batch rows that were not cut, and row tiles
// without a token, were written by the kernels above.  All loads of a few parts are issued at once;
// with kSpread (few rows in many parts) the workgroup has one row and each kD / 4 lanes every
// 1024 / kD-th part, added up through LDS.  4.0 to 4.7 us for few rows, most of it the launch; 512
// tokens in 8 parts, 50 MB, 10.8 us (4.7 TB/s).
constexpr int kMergeThreads = 256;
struct Sum {
  float m = kNegBig, l = 0.f;
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  // (a part without a visible key has l = 0; a NaN is not)
  __device__ __forceinline__ void add(bool use, float ms, float ls, floatx4 os) {
    use = use && __builtin_bit_cast(uint32_t, ls) != 0;
    const float mn = fmaxf(m, use ? ms : kNegBig);
    const float a = fast_exp2(m - mn), e = use ? fast_exp2(ms - mn) : 0.f;
    l = l * a + (use ? ls : 0.f) * e;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = o[c] * a + (use ? os[c] : 0.f) * e;
    m = mn;
  }
};
template <int kD, bool kSpread>
__global__ __launch_bounds__(kMergeThreads) void merge_kernel(Params p) {
  constexpr int kLanes = kD / 4;  // of a row
  constexpr int kGroups = kMergeThreads / kLanes;
  const int b = blockIdx.y;
  const int before = p.shares[2 * b], parts = p.shares[2 * b + 1];
  if (parts <= 1) return;
  const int group = threadIdx.x / kLanes;
  const int r = kSpread ? blockIdx.x : blockIdx.x * kGroups + group;  // (token, query head)
  const int d = 4 * (threadIdx.x % kLanes);
  if (r >= p.chunk * p.num_q_heads) return;
  const int t = div_by(r, p.head_div);
  const int h = r - t * p.num_q_heads;
  const Row row = row_of(p, b);
  const int pos = row.start + t;
  const RowTiles rt = row_tiles_of(p, row);
  const int kvh = div_by(h, p.group_div);
  const int kr = t * p.group + h - kvh * p.group;
  const int tile = div_by(kr, p.tile_div);
  if (tile < rt.first || tile >= rt.first + rt.count) return;
  Sum sum;
  if (pos >= 0 && pos < row.len) {
    int lo, hi;
    row_positions(p, row, tile * p.tile_rows, (tile + 1) * p.tile_rows - 1, lo, hi);
    const int n = span_of(p, row, lo, hi).n;
    const int size = parts_of(n, inverse(parts));
    const int used = parts_of(n, inverse(size));  // parts with key tiles
    const int64_t step = (int64_t)rt.count * p.num_kv_heads * p.part_rows;
    const int64_t slot0 = ((int64_t)(before + rt.first + rt.count - 1 - tile) * p.num_kv_heads + kvh) *
                              p.part_rows + kr - tile * p.tile_rows;
    auto add = [&](auto most) {
      constexpr int kParts = decltype(most)::value, kStep = kSpread ? kGroups : 1;
      for (int s0 = kSpread ? group : 0; s0 < used; s0 += kParts * kStep) {
        float ms[kParts], ls[kParts];
        floatx4 os[kParts];
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
          const int64_t slot = slot0 + min(s0 + k * kStep, used - 1) * step;
          ms[k] = p.part_ml[slot * 2];
          ls[k] = p.part_ml[slot * 2 + 1];
          os[k] = *(const floatx4*)(p.part_o + slot * kD + d);
        }
#pragma unroll
        for (int k = 0; k < kParts; ++k) sum.add(s0 + k * kStep < used, ms[k], ls[k], os[k]);
      }
    };
    if (used <= 3 * (kSpread ? kGroups : 1))
      add(std::integral_constant<int, 3>());
    else
      add(std::integral_constant<int, 8>());
  }
  if constexpr (kSpread) {  // the row's groups, in order
    __shared__ floatx4 s_o[kMergeThreads];
    __shared__ float s_m[kMergeThreads], s_l[kMergeThreads];
    s_o[threadIdx.x] = sum.o;
    s_m[threadIdx.x] = sum.m;
    s_l[threadIdx.x] = sum.l;
    __syncthreads();
    if (group > 0) return;
    sum = Sum();
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const int x = k * kLanes + threadIdx.x;
      sum.add(true, s_m[x], s_l[x], s_o[x]);
    }
  }
  const float inv = __builtin_bit_cast(uint32_t, sum.l) != 0 ? 1.f / sum.l : 0.f;
  if (d < p.head_dim)
    *(half4*)(p.o + (int64_t)b * p.o_sb + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + d) =
        to_half4(sum.o * inv);
}

// How a call is cut: row blocks per wave, row tiles per (batch row, kv head), parts aimed at (0: not
// cut) and rows of a part's results.
constexpr int64_t kMaxWgs = (1 << 24) - 1;  // a launch takes fewer than 2^32 threads along x
struct Plan {
  bool narrow;
  int nb;
  int64_t rows, row_lists;  // query rows of each (batch row, kv head), and how many of those
  int64_t row_tiles, wgs, target, target2, part_rows, width;
  int64_t tile_rows() const { return narrow ? 16 * nb : 64 * nb; }
  int64_t parts() const { return std::max(target, target2); }
  void shape(int blocks) {
    nb = blocks;
    row_tiles = (rows + tile_rows() - 1) / tile_rows();
    wgs = row_lists * row_tiles;
    part_rows = std::min(rows, tile_rows());
  }
  size_t bytes(int64_t batch) const {
    return (size_t)((parts() + wgs) * part_rows * (width + 2) + 2 * batch) * sizeof(float);
  }
};

// Up to 32 rows per kv head: the narrow form, cut into one round of workgroups (two per CU, four
// of the 64-wide form); with 48 rows it takes four blocks, too many registers, 59 us against 35
// for 8 x 12 tokens at 4000.  More rows: 1, 2 or 3 row blocks per wave, cut or not, by
// the estimate that fits what was measured.  A key tile takes a workgroup alone on its CU
// `alone` us and costs the CU `shared` us where more of them run there: 1.17, 1.74, 2.08 and 0.72,
// 1.1, 1.5 for 1, 2, 3 blocks (128 wide; chunks of 512 tokens at 8192, 2 x 1000 at 5000, 2 x 2048
// at 16384).  A call costs 6 us besides, one that is cut 6 more, and a round of parts 6 us per
// block for results written and read.  Rows of one call that have their own lengths are taken to
// have two thirds of the bound on average, the longest the whole; the row tiles of one row the mean
// of its first and last token's keys (a prompt of 2000 tokens 75 -> 49 us, of 4096 152 -> 134, against all
// the last token's).  The 64-wide form takes 0.6 of that time, and has room for three workgroups per CU
// (two: 2 x 1000 tokens at 8000 102 us against 92, 1500 at 20000 173 against 149).  The choice is
// within 5% of the best of the six but for single cases (8 x 300 tokens at 3000: 85 against 77).
// Against three blocks, uncut: 4 x 128 tokens at 300 20 -> 13 us, a prompt of 512 25 -> 15.5, 2 x
// 1000 at 5000 201 -> 169.
static Plan plan(int64_t batch, int64_t chunk, int64_t num_q_heads, int64_t num_kv_heads,
                 int64_t num_tokens, int64_t head_dim, int64_t window, bool lens,
                 bool may_cut) {
  constexpr int64_t kCus = 256;
  Plan pl = {};
  pl.rows = chunk * (num_q_heads / num_kv_heads);
  pl.row_lists = batch * num_kv_heads;
  pl.width = head_dim <= 64 ? 64 : 128;
  pl.narrow = pl.rows <= 32;
  if (pl.narrow) {
    pl.shape((int)((pl.rows + 15) / 16));
    const int64_t slots = pl.width == 64 ? 4 * kCus : 2 * kCus;
    pl.target = may_cut && pl.wgs < slots && num_tokens > kWholeTokens ? slots : 0;
  } else {
    static constexpr double kAlone[3] = {1.17, 1.74, 2.08}, kShared[3] = {0.72, 1.1, 1.5};
    const int64_t per_slot = pl.width == 64 ? 3 : 2;  // workgroups of a CU
    const int64_t slots = per_slot * kCus;
    const double wide = pl.width == 64 ? 0.6 : 1.0;
    const bool ragged = lens && batch > 1;
    double best = 0;
    int nb = 0;
    bool cut = false;
    for (int i = 1; i <= 3; ++i) {
      pl.shape(i);
      const int64_t span = window + pl.tile_rows() / (num_q_heads / num_kv_heads) + kKTile;
      const double n = (double)((std::min(num_tokens, span) + kKTile - 1) / kKTile);
      // the first tokens of the chunk see fewer keys
      const double mean = num_tokens <= span ? n - (double)std::min(chunk, num_tokens) / (2 * kKTile) : n;
      const double alone = wide * kAlone[i - 1], shared = wide * kShared[i - 1];
      const int64_t per_cu = (pl.wgs + kCus - 1) / kCus;
      const double whole = 6 + (per_cu == 1 ? n * alone : std::max(n * alone, (double)per_cu * mean * shared));
      if (nb == 0 || whole < best) best = whole, nb = i, cut = false;
      const int64_t parts = std::min<int64_t>(slots / pl.wgs, (int64_t)n / kMinPart);
      if (may_cut && pl.wgs < slots && (parts >= 2 || (ragged && n > 2 * kMinPart))) {
        const double round = std::min(1.0, (double)(pl.wgs * std::max<int64_t>(parts, 1)) / slots);
        double chain = ceil(n / (double)std::max<int64_t>(parts, 1));
        if (ragged) chain = (0.65 + 0.7 / (double)batch) * n * (double)pl.wgs / slots;
        const double step = round * per_slot <= 1 && !ragged ? alone : per_slot * shared;
        const double pieces = 12 + chain * step + 6 * wide * i * (ragged ? 1.0 : round);
        if (pieces < best) best = pieces, nb = i, cut = true;
      }
    }
    pl.shape(nb);
    pl.target = cut ? slots : 0;
    pl.target2 = cut && ragged ? 2 * slots : 0;
  }
  return pl;
}

// |x| <= limit, false for NaN, by the bits: this file is compiled for NaN-free arithmetic.
static bool within(float x, float limit) {
  uint32_t a, b;
  memcpy(&a, &x, 4);
  memcpy(&b, &limit, 4);
  return (a & 0x7fffffffu) <= b;
}

static bool sizes_ok(int64_t batch, int64_t chunk, int64_t num_q_heads, int64_t num_kv_heads) {
  return batch >= 0 && chunk >= 0 && num_q_heads > 0 && num_kv_heads > 0 &&
         num_q_heads % num_kv_heads == 0;
}

template <int kD, int kMod>
static void launch(const Plan& pl, dim3 grid, hipStream_t st, const Params& p) {
  const dim3 block(kThreads);
  if (pl.narrow && pl.nb == 1)
    hipLaunchKernelGGL((narrow_kernel<1, kD, kMod>), grid, block, 0, st, p);
  else if (pl.narrow)
    hipLaunchKernelGGL((narrow_kernel<2, kD, kMod>), grid, block, 0, st, p);
  else if (pl.nb == 1)
    hipLaunchKernelGGL((chunk_kernel<1, kD, kMod>), grid, block, 0, st, p);
  else if (pl.nb == 2)
    hipLaunchKernelGGL((chunk_kernel<2, kD, kMod>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((chunk_kernel<3, kD, kMod>), grid, block, 0, st, p);
}
template <int kD>
static void launch(int mod, const Plan& pl, dim3 grid, hipStream_t st, const Params& p) {
  switch (mod) {
    case 0: launch<kD, 0>(pl, grid, st, p); break;
    case kCap: launch<kD, kCap>(pl, grid, st, p); break;
    case kBias: launch<kD, kBias>(pl, grid, st, p); break;
    default: launch<kD, kCap | kBias>(pl, grid, st, p); break;
  }
}

}  // namespace chunk
}  // namespace fi

extern "C" size_t fi_paged_chunk_attention_workspace_size(int64_t batch, int64_t num_new,
                                                          int64_t num_q_heads, int64_t num_kv_heads,
                                                          int64_t max_num_tokens, int64_t head_dim) {
  using namespace fi::chunk;
  if (!sizes_ok(batch, num_new, num_q_heads, num_kv_heads) || batch == 0 || num_new == 0 ||
      max_num_tokens <= 0 || max_num_tokens > kMaxTokens || !fi::head_dim_ok(head_dim) ||
      batch > 0x7fffffff || num_new > 0x7fffffff / num_q_heads)
    return 0;
  // whether the call will have lengths of its own, or a window (which may choose other row blocks),
  // is not known here: the most of these
  size_t bytes = 0;
  for (const bool lens : {false, true}) {
    Plan pl =
        plan(batch, num_new, num_q_heads, num_kv_heads, max_num_tokens, head_dim, kNoWindow, lens, true);
    if (!pl.target) continue;
    bytes = std::max(bytes, pl.bytes(batch));
    for (int nb = 1; nb <= 3 && !pl.narrow; ++nb) {
      pl.shape(nb);
      if (pl.wgs < pl.target) bytes = std::max(bytes, pl.bytes(batch));
    }
  }
  return bytes;
}

extern "C" int fi_paged_chunk_attention_fwd(
    const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k_cache, const void* v_cache,
    int64_t num_pool_blocks, int64_t block_size, int64_t num_kv_heads, const int32_t* block_table,
    int64_t bt_stride, int64_t max_blocks_per_seq, const int32_t* start_positions,
    const int32_t* context_lens, int64_t num_tokens, void* o, int64_t o_sb, int64_t o_st, int64_t o_sh,
    int64_t batch, int64_t num_new, int64_t num_q_heads, int64_t head_dim, float sm_scale, float softcap,
    const float* alibi_slopes, int64_t window, const int32_t* prefix_lens, void* workspace,
    size_t workspace_bytes, void* stream) {
  using namespace fi;
  using namespace fi::chunk;
  static const char* fn = "fi_paged_chunk_attention_fwd";
  clear_error();
  if (!head_dim_ok(head_dim)) {
    set_error("%s: head_dim %lld not supported (a multiple of 8 up to %d)", fn, (long long)head_dim,
              kHeadDim);
    return FI_ERR_UNSUPPORTED;
  }
  if (!sizes_ok(batch, num_new, num_q_heads, num_kv_heads) || num_tokens < 0 || num_pool_blocks < 0 ||
      max_blocks_per_seq < 0) {
    set_error("%s: invalid sizes (batch %lld, new tokens %lld, heads %lld/%lld, tokens %lld)", fn,
              (long long)batch, (long long)num_new, (long long)num_q_heads, (long long)num_kv_heads,
              (long long)num_tokens);
    return FI_ERR_INVALID;
  }
  if (block_size <= 0 || block_size > 0x7fffffff) {
    set_error("%s: block_size %lld must be positive, below 2^31", fn, (long long)block_size);
    return FI_ERR_INVALID;
  }
  if (window < 0) {
    set_error("%s: window %lld must be positive, or 0 for none", fn, (long long)window);
    return FI_ERR_INVALID;
  }
  if (!within(sm_scale, kMaxScale) || !within(softcap, kMaxScale) || softcap < 0.f) {
    set_error("%s: sm_scale %g and softcap %g must be at most %g, the cap positive (0 for none)", fn,
              (double)sm_scale, (double)softcap, (double)kMaxScale);
    return FI_ERR_INVALID;
  }
  if (batch == 0 || num_new == 0) return FI_OK;
  if (num_tokens > kMaxTokens || num_pool_blocks > 0x7fffffff / block_size ||
      max_blocks_per_seq > 0x7fffffff || batch > 0x7fffffff / num_kv_heads || num_kv_heads > (1 << 19) ||
      num_new > 0x7fffffff / num_q_heads / 2) {
    set_error("%s: sizes too large (at most %lld tokens a row, 2^31 pool slots)", fn,
              (long long)kMaxTokens);
    return FI_ERR_UNSUPPORTED;
  }
  // an empty bound reads no table and no pool
  if (!q || !o || (num_tokens > 0 && (!k_cache || !v_cache || !block_table))) {
    set_error("%s: null pointer", fn);
    return FI_ERR_INVALID;
  }
  if ((((uintptr_t)q | (uintptr_t)o | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15u) ||
      (q_sb | q_st | q_sh | o_sb | o_st | o_sh) % 8 != 0) {
    set_error("%s: rows must be 16-byte aligned (strides multiple of 8)", fn);
    return FI_ERR_INVALID;
  }

  Params p = {};
  p.q = (const half_t*)q;
  p.q_sb = q_sb; p.q_st = q_st; p.q_sh = q_sh;
  p.k_cache = (const half_t*)k_cache;
  p.v_cache = (const half_t*)v_cache;
  p.num_pool_blocks = (int)num_pool_blocks;
  p.block_size = (int)block_size;
  p.whole = block_size % 16 == 0;
  p.block_div = fast_div((uint32_t)block_size);
  p.num_kv_heads = (int)num_kv_heads;
  p.kv_div = fast_div((uint32_t)num_kv_heads);
  p.row_bytes = num_kv_heads * head_dim * 2;
  p.block_table = block_table;
  p.bt_stride = bt_stride;
  p.max_blocks_per_seq = (int)max_blocks_per_seq;
  p.start_positions = start_positions;
  p.context_lens = context_lens;
  p.num_tokens = (int)(max_blocks_per_seq < num_tokens / block_size + 1
                           ? std::min(num_tokens, max_blocks_per_seq * block_size) : num_tokens);
  p.o = (half_t*)o;
  p.o_sb = o_sb; p.o_st = o_st; p.o_sh = o_sh;
  p.batch = (int)batch;
  p.batch_div = fast_div((uint32_t)batch);
  p.chunk = (int)num_new;
  p.num_q_heads = (int)num_q_heads;
  p.head_div = fast_div((uint32_t)num_q_heads);
  p.group = (int)(num_q_heads / num_kv_heads);
  p.group_div = fast_div((uint32_t)p.group);
  p.head_dim = (int)head_dim;
  p.d_chunks = (int)(head_dim / 8);
  // Scores of a smaller scale or cap than kFlat differ by less than fp32 resolves in a weight: all
  // zero, as with a scale of zero (scores are masked before they are scaled, and -inf * 0 is NaN).
  const bool flat = std::fabs(sm_scale) < kFlat || (softcap > 0.f && softcap < kFlat);
  const bool cap = softcap > 0.f && !flat;
  if (cap) {
    p.scale_log2 = softcap * (2.f * kLog2e);  // see capped()
    p.cap_exp = sm_scale / softcap * (2.f * kLog2e);
  } else {
    // a zero scale runs as unit scale on a Q of zeros, a negative one on a negated Q
    p.q_zero = flat;
    p.q_sign = sm_scale < 0.f ? 0x80008000u : 0u;
    p.scale_log2 = flat ? kLog2e : std::fabs(sm_scale) * kLog2e;
  }
  p.lazy_raw = kLazyLog2 / p.scale_log2;
  p.lazy_log2 = p.lazy_raw * p.scale_log2;
  p.slopes = alibi_slopes;
  p.slope_mul = kLog2e / p.scale_log2;
  p.window = window == 0 || window > kNoWindow ? kNoWindow : (int)window;
  p.prefix_lens = prefix_lens;

  Plan pl =
      plan(batch, num_new, num_q_heads, num_kv_heads, num_tokens, head_dim, p.window, context_lens, true);
  if (pl.target && (!workspace || workspace_bytes < pl.bytes(batch)))
    pl = plan(batch, num_new, num_q_heads, num_kv_heads, num_tokens, head_dim, p.window, context_lens, false);
  if (pl.wgs > kMaxWgs) {
    set_error("%s: too many new tokens (%lld rows of %lld)", fn, (long long)batch, (long long)num_new);
    return FI_ERR_UNSUPPORTED;
  }
  p.tile_rows = (int)pl.tile_rows();
  p.tile_div = fast_div((uint32_t)p.tile_rows);
  p.row_tiles = (int)pl.row_tiles;
  if (pl.target) {
    if ((uintptr_t)workspace & 15u) {
      set_error("%s: workspace must be 16-byte aligned", fn);
      return FI_ERR_INVALID;
    }
    p.target = (int)pl.target;
    p.target2 = (int)pl.target2;
    p.part_rows = (int)pl.part_rows;
    p.part_o = (float*)workspace;
    p.part_ml = p.part_o + (pl.parts() + pl.wgs) * pl.part_rows * pl.width;
    p.shares = (int32_t*)(p.part_ml + (pl.parts() + pl.wgs) * pl.part_rows * 2);
  }
  // list entries: at most parts() / num_kv_heads and one per row tile, nor more than the smallest
  // parts of the longest list
  const int64_t most = (num_tokens + kKTile * kMinPart - 1) / (kKTile * kMinPart);
  int64_t items = batch * pl.row_tiles;
  if (pl.target) items = std::min(items + pl.parts() / num_kv_heads, items * std::max<int64_t>(most, 1));
  const dim3 grid((unsigned)(items * num_kv_heads));
  const hipStream_t st = (hipStream_t)stream;
  const int mod = (cap ? kCap : 0) | (alibi_slopes ? kBias : 0);
  if (pl.width == 64)
    launch<64>(mod, pl, grid, st, p);
  else
    launch<128>(mod, pl, grid, st, p);
  const int rc = check_launch(fn);
  if (rc != FI_OK || !pl.target) return rc;
  // a workgroup per row where the parts per row are many (4 drafted tokens at 1024: eight)
  const bool spread = pl.target >= 4 * pl.wgs && pl.narrow;
  const int64_t merge_rows = spread ? 1 : kMergeThreads / (pl.width / 4);
  const dim3 mgrid((unsigned)((num_new * num_q_heads + merge_rows - 1) / merge_rows), (unsigned)batch);
  const dim3 mblock(kMergeThreads);
  if (pl.width == 64 && spread)
    hipLaunchKernelGGL((merge_kernel<64, true>), mgrid, mblock, 0, st, p);
  else if (pl.width == 64)
    hipLaunchKernelGGL((merge_kernel<64, false>), mgrid, mblock, 0, st, p);
  else if (spread)
    hipLaunchKernelGGL((merge_kernel<128, true>), mgrid, mblock, 0, st, p);
  else
    hipLaunchKernelGGL((merge_kernel<128, false>), mgrid, mblock, 0, st, p);
  return check_launch(fn);
}
