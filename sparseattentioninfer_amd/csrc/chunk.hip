// Causal attention of a chunk of new tokens over a paged cache, gfx950 (CDNA4): sequences of different lengths,
// whole caches or the pages that a selection lists for each 64-query block.
//
//   o[row] = sum_j softmax_j(q . k_j * scale) v_j over the keys j <= position of the row (and listed pages),
//
// position = kv_len - new tokens + index of the row's token.  fp32 statistics and accumulators; probabilities are
// rounded to the element type for the second product, which is matrix-core work, and the sum that divides is of
// the unrounded ones.  A row that sees no key is 0.
//
// Rows of an item are (token, query head of one KV head) pairs, flattened with the head fastest, so a tile of 32
// rows is full whatever the group size, and every K/V tile read serves the whole group.  Keys are read in tiles
// of 64, each four chunks of 16 keys; a page is a whole number of chunks, so a chunk lies in one page and each of
// its wave-wide direct loads has one uniform address.  A wave looks its chunks' pages up 64 at a time, one a
// lane, and takes them lane by lane.
#include <algorithm>
#include <type_traits>

#include "lds_tile.h"
#include "ragged.h"

namespace sa {

constexpr int CK_ROWS = 32;        // rows of a wave
constexpr int CK_KT = 64;          // keys of a tile
constexpr int CK_BLOCK = 64;       // new tokens that share one selection
constexpr int64_t CK_PART_ROWS = 1 << 17;  // rows of partials (68 MB at head dim 128) that a planned division uses at most
constexpr int CK_NO_KEY = 0x60000000;  // key position of a chunk that is not there: past every row
// Largest token stride (elements) of the pools: per-lane offsets within a chunk are 32-bit.
constexpr int64_t CK_MAX_STRIDE = (int64_t)1 << 24;

// 16 readable zero bytes: what lanes of keys that are not there load, so masked keys add 0 * 0.
__device__ __attribute__((aligned(16))) const uint32_t c_zero16[4] = {0u, 0u, 0u, 0u};

// Where a sequence's partial results are (splits > 1).
struct SeqPart {
  int first, splits, n;
  int any;           // whether any sequence is split
};

struct ChunkArgs {
  const elem_t* q;
  int64_t q_st, q_sh;
  const elem_t *k, *v;
  int64_t kv_sp, kv_sh, kv_st;
  const int32_t* table;
  int64_t table_stride;
  int max_blocks, num_pages, page;
  uint32_t mul_page;
  Ragged seqs;
  // selection (sel_off NULL: every page): row of query block i, KV head g: sel[i * sel_sr + g * sel_sh + e]; sel is NULL
  // where its rows have no entry
  const int32_t* sel;
  int64_t sel_sr, sel_sh;
  const int32_t* sel_off;
  int64_t off_sr, off_sh;
  int sel_rows, sel_width;
  uint32_t mul_ppc;                // fast_div multiplier of the chunks of a page
  elem_t* o;
  int64_t o_st, o_sh;
  int Hq, Hkv, G;
  uint32_t mul_G, mul_heads, mul_Hq, mul_tpb;
  float scale_log2;
  int tiles_per_block;             // with a selection: wide row tiles of a 64-token block
  int key_tiles;                   // key tiles that a row may see at most: the table's, or the longest list's
  int cus;
  int splits;                      // of every sequence; 0: planned, 1: none
  // Partial results of sequences whose keys are split: row (split, token, head) of sequence b at part[b].first +
  // (split * tokens + token) * Hq + head.
  SeqPart* part;                   // [B], written by the launch's first workgroup
  float* part_acc;                 // [part_rows, D]
  float* part_ml;                  // [part_rows, 2]: row reference (base 2) and row sum
  int64_t part_rows;
};

// ---- which workgroup does what ----------------------------------------------------------------
//
// A sequence of few rows (CK_NARROW or less: one token, a few drafts) is read by narrow items, 32 rows whose keys
// four waves divide; others by wide items, 256 rows that share every key tile.  Where there are fewer items than
// CUs, or one sequence is much longer than the rest, each item's keys are divided over `splits` workgroups.  The
// lengths are device memory, so the launch is as large as any lengths need and every workgroup works out the
// division for itself, the same in all of them: `limit` key tiles to a workgroup, from the total.
//
// Key tiles are what is balanced.  With the chip full a wide item takes 1.75 us for one (256 rows on its matrix
// cores), a narrow one 1.45 us where narrow items are most of the work (32 KB at a CU's share of HBM) and about half of
// a wide one's beside wide ones.  A workgroup costs CK_START of them besides its own: 9.6 us, of which finding its item
// takes 2.5, the pages of its first tiles 2.6, the tiles 1.5 and the end 3.
constexpr float CK_START = 5.5f;
// A division costs the merge, 4 us after narrow and 6.5 after wide items, and for each row of partials its write and
// read: 1,040 bytes at D = 128, 0.2 ns at the rate of a copy.
constexpr float CK_MERGE_WIDE = 4.f, CK_MERGE_NARROW = 2.5f, CK_MERGE_ROW = 1.3e-4f;
constexpr int CK_NARROW = 64;
constexpr int CK_WIDE_ROWS = 256;

// Sum or maximum over the lanes that differ in bits 3..5 only, in every lane.
enum : int { SUM = 0, MAX = 1 };
template <int OP>
__device__ __forceinline__ float over_eights(float x) {
  auto op = [](float a, float b) { return OP == MAX ? fmaxf(a, b) : a + b; };
  x = op(x, dpp<0x128>(x));   // row_ror:8
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = op(__uint_as_float(s[0]), __uint_as_float(s[1]));
  return OP == MAX ? halves_max(x) : halves_sum(x);
}

struct SeqShape {
  int n, end;       // new tokens; tokens in all
  int row;          // packed row of the first new token
  int tiles;        // row tiles
  int nt, nt0;      // key tiles of the last row tile; of the first
};

__device__ __forceinline__ bool is_narrow(const ChunkArgs& a, int n) { return (int64_t)n * a.G <= CK_NARROW; }

__device__ __forceinline__ SeqShape seq_shape(const ChunkArgs& a, int b) {
  SeqShape s;
  s.n = a.seqs.rows(b, s.row);
  s.end = a.seqs.kv_len(b);
  const int64_t rows = (int64_t)s.n * a.G;
  if (is_narrow(a, s.n))
    s.tiles = ((int)rows + CK_ROWS - 1) / CK_ROWS;
  else
    s.tiles = a.sel_off ? (s.n + CK_BLOCK - 1) / CK_BLOCK * a.tiles_per_block : (int)((rows + CK_WIDE_ROWS - 1) / CK_WIDE_ROWS);
  s.nt = min((s.end + CK_KT - 1) / CK_KT, a.key_tiles);
  s.nt0 = min((max(s.end - s.n, 0) + CK_KT) / CK_KT, s.nt);
  return s;
}

// Workgroups that share a row tile's keys when one takes at most `limit` key tiles.  At least
// 4: one for each wave of a narrow one; of a wide one, whose 256 rows leave 133 KB of partials, fewer do not pay (64 new
// tokens over 1,024 keys, 32/8 heads, bf16, D = 128: 28.7 us in one, 24.7 in 2, 20.7 in 4, 20.6 in 8, 25.1 in 16).
constexpr int CK_MAX_SPLITS = 64;
constexpr int CK_NO_LIMIT = 0x40000000;   // at or past this: no division
struct SplitRule {
  int limit;
  int most_wide, most_narrow;    // key tiles of a workgroup
  float rcp_wide, rcp_narrow;
  // half: a narrow item's key tile counts half of a wide one's.
  __device__ __forceinline__ SplitRule(int l, int half) {
    limit = l;
    most_wide = max(l, 4);
    most_narrow = max(l >= CK_NO_LIMIT ? l : l << half, 4);
    rcp_wide = __builtin_amdgcn_rcpf((float)most_wide);
    rcp_narrow = __builtin_amdgcn_rcpf((float)most_narrow);
  }
  __device__ __forceinline__ int splits(int fixed, int narrow, int nt) const {
    if (limit >= CK_NO_LIMIT) return 1;
    if (fixed) return max(1, min(fixed, nt));
    // ceil(nt / m): nt < 2^24, so the rounded product is off by one at most.
    const int m = narrow ? most_narrow : most_wide, x = nt + m - 1;
    int q = (int)((float)x * (narrow ? rcp_narrow : rcp_wide));
    q += (q + 1) * m <= x ? 1 : 0;
    q -= q * m > x ? 1 : 0;
    return min(max(1, q), CK_MAX_SPLITS);
  }
};

// The division of the keys (a.splits: any limit below CK_NO_LIMIT stands for that division).  Every workgroup comes
// through here before its first load, so eight choices are weighed side by side: lane 8 y + x adds up choice x over
// the sequences y, y + 8, ...  The sums are fp32: exact where they decide between neighbouring choices (below 2^24),
// and the room for partials is kept with a margin above their rounding; a fixed division, which fills its room
// exactly, is summed in 64 bits.
__device__ __forceinline__ SplitRule plan_splits(const ChunkArgs& a, const SeqShape& first64) {
  const int lane = threadIdx.x & 63;
  if (a.splits) {
    int64_t x = 0;
    for (int b = lane; b < a.seqs.B; b += 64) {
      const SeqShape s = b < 64 ? first64 : seq_shape(a, b);
      const int k = SplitRule(1, 0).splits(a.splits, is_narrow(a, s.n), s.nt);
      x += k > 1 ? (int64_t)s.n * k * a.Hq : 0;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
    return SplitRule(x > a.part_rows ? CK_NO_LIMIT : 1, 0);
  }
  const float heads = (float)a.Hkv, cus = (float)a.cus;
  float wide = 0.f, narrow = 0.f, longest = 0.f, tiles = 0.f;
  for (int b0 = 0; b0 < a.seqs.B; b0 += 64)
    if (b0 + lane < a.seqs.B) {
      const SeqShape s = b0 ? seq_shape(a, b0 + lane) : first64;
      const float w = (float)s.tiles * (float)(s.nt + s.nt0);
      (is_narrow(a, s.n) ? narrow : wide) += w;
      tiles += (float)s.tiles;
      longest = fmaxf(longest, (float)s.nt);
    }
  wide = wave_sum(wide) * (0.5f * heads);
  narrow = wave_sum(narrow) * (0.5f * heads);
  tiles = wave_sum(tiles);
  longest = wave_max(longest);
  const int half = narrow > wide ? 0 : 1;
  const float nw = half ? 0.5f : 1.f, work = wide + nw * narrow;
  const float even = fminf(ceilf(work / cus), (float)(CK_NO_LIMIT / 16));
  if (longest <= 0.5f * even) return SplitRule(CK_NO_LIMIT, half);   // there are row tiles enough
  // Choices: 1/2, 3/4, 1, 5/4, 3/2, 2 and 3 even shares, and no division.
  const int quarters = (0x0C865432u >> (4 * (lane & 7))) & 15;
  const SplitRule r(quarters ? max(1, (int)ceilf(even * (float)quarters * 0.25f)) : CK_NO_LIMIT, half);
  auto each = [&](auto f) {   // f(sequence's row tiles, splits, longest, shortest key tiles, new tokens, weight)
    for (int b0 = 0; b0 < a.seqs.B; b0 += 64) {
      SeqShape s = first64;
      if (b0) {
        s = SeqShape{};
        if (b0 + lane < a.seqs.B) s = seq_shape(a, b0 + lane);
      }
      const int nar = is_narrow(a, s.n);
      for (int y = 0; y < min(64, a.seqs.B - b0); y += 8) {
        const int from = y + (lane >> 3);   // sequences past the last have no tiles
        const int st = __shfl(s.tiles, from, 64), nt = __shfl(2 * s.nt + nar, from, 64);
        const int nt0 = __shfl(s.nt0, from, 64), n = __shfl(s.n, from, 64);
        const int k = r.splits(0, nt & 1, nt >> 1);
        f((float)st, (float)k, (float)(nt >> 1), (float)nt0, (float)n, nt & 1 ? nw : 1.f);
      }
    }
  };
  float groups = 0.f, rows = 0.f;
  each([&](float st, float k, float, float, float n, float) {
    groups += st * k;
    rows += k > 1.f ? n * k : 0.f;
  });
  groups = over_eights<SUM>(groups) * heads;
  rows = over_eights<SUM>(rows) * (float)a.Hq;
  // When it ends.  In one round: with the longest workgroup.  Else, handed out longest first: the mean load, or
  // two of those longer than half of it where they outnumber the CUs (their lengths taken as spread evenly).
  const float mean = (work + groups * CK_START) / cus;
  // Narrow items that do not fill the chip are not bound by HBM: 0.5 us for a tile instead of 1.45.
  const float alone = half ? 1.f : fminf(fmaxf(0.35f, groups / cus), 1.f);
  float one = 0.f, many = 0.f, lo = __builtin_inff(), hi = 0.f;
  each([&](float st, float k, float nt, float nt0, float, float w) {
    if (st == 0.f) return;
    const float x = w * alone * __builtin_amdgcn_rcpf(k), h = nt * x + CK_START, l = nt0 * x + CK_START;
    one = fmaxf(one, h);
    if (h <= 0.5f * mean) return;
    const float from = fmaxf(l, 0.5f * mean);
    many += st * k * (l >= 0.5f * mean ? 1.f : (h - from) * __builtin_amdgcn_rcpf(h - l));
    lo = fminf(lo, from);
    hi = fmaxf(hi, h);
  });
  one = over_eights<MAX>(one);
  many = over_eights<SUM>(many) * heads;
  lo = -over_eights<MAX>(-lo);
  hi = over_eights<MAX>(hi);
  float time = one;
  if (groups > cus) time = fmaxf(one, 1.08f * mean);
  if (groups > cus && many > cus) time = fmaxf(time, 2.f * (lo + (hi - lo) * (many - cus) / many));
  if (rows > 0.f) time += (half ? CK_MERGE_WIDE : CK_MERGE_NARROW) + CK_MERGE_ROW * rows;
  // The partials must fit, and no more workgroups are added than there are CUs (chunk_items: the launch has that
  // many to spare, and idle ones cost time too).  No division always does.
  if (rows * 1.001f > (float)a.part_rows || groups > tiles * heads + cus) time = __builtin_inff();
  int limit = CK_NO_LIMIT;
  float best = __builtin_inff();
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    const float t = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(time), x));
    const int l = __builtin_amdgcn_readlane(r.limit, x);
    if (t < best) {
      best = t;
      limit = l;
    }
  }
  return SplitRule(limit, half);
}

// The rows and keys of one work item.
struct ChunkItem {
  int b, kvh, split, splits;
  bool narrow;
  int row0, row_end;               // flattened rows of the sequence
  int n, tok0;                     // its new tokens, and the packed row of the first
  int start;                       // position of its first new token
  int end;                         // its tokens in all
  int pos_max;                     // position of the last row
  int c0, c1;                      // chunks of the item: [c0, c1)
  const int32_t* list;             // selected pages, or NULL
  int list_chunks;
  int64_t part;                    // first row of the sequence's partials

  // Row of the partials of flattened row r.
  __device__ __forceinline__ int64_t part_row(const ChunkArgs& a, int token, int head) const {
    return part + ((int64_t)split * n + token) * a.Hq + head;
  }
};

// Work item of workgroup `id`, or false.  Heads go fastest (one XCD's workgroups then read one KV head where there
// are eight of them).  Longest first, so that the launch ends evenly: up to 64 sequences in the order of their
// workgroups' key tiles (a narrow one's take half as long while the matrix cores bound the rest), more as they come;
// within a sequence later row tiles, which see more keys, first.
__device__ __forceinline__ bool find_chunk_item(const ChunkArgs& a, int id, ChunkItem& it) {
  const int lane = threadIdx.x & 63;
  const int t = (int)fast_div((uint32_t)id, (uint32_t)a.Hkv, a.mul_heads);
  it.kvh = id - t * a.Hkv;
  SeqShape s64 = {};
  if (lane < a.seqs.B) s64 = seq_shape(a, lane);
  const bool split = a.part != nullptr;
  const SplitRule rule = split ? plan_splits(a, s64) : SplitRule(CK_NO_LIMIT, 0);
  const bool first = id == 0 && split && __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) == 0;
  const bool ranked = a.seqs.B > 1 && a.seqs.B <= 64;
  int base = 0, block0 = 0, part0 = 0, local = 0;
  bool found = false;
  for (int b0 = 0; b0 < a.seqs.B && (first || !found); b0 += 64) {
    SeqShape s = s64;
    if (b0) {
      s = SeqShape{};
      if (b0 + lane < a.seqs.B) s = seq_shape(a, b0 + lane);
    }
    const int narrow = is_narrow(a, s.n), k = rule.splits(a.splits, narrow, s.nt);
    const int c = s.tiles * k, blocks = a.sel_off ? (s.n + CK_BLOCK - 1) / CK_BLOCK : 0;
    const int rows = k > 1 ? s.n * k * a.Hq : 0;   // all of them fit 31 bits: part_rows does
    const int ib = a.sel_off ? scan_lanes(blocks) : 0, ir = split ? scan_lanes(rows) : 0;
    if (first && b0 + lane < a.seqs.B) a.part[b0 + lane] = SeqPart{part0 + ir - rows, k, s.n, rule.limit < CK_NO_LIMIT};
    // The sequences in their order: lane i then holds the item count and the lane of the i-th.
    int co = c, from = lane;
    if (ranked) {
      const float len = (float)((s.nt + s.nt0) << (1 - narrow)) * __builtin_amdgcn_rcpf((float)k);
      int rank = 0;
      for (int j = 0; j < a.seqs.B; ++j) {
        const float lj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(len), j));
        rank += lj > len || (lj == len && j < lane) ? 1 : 0;
      }
      rank = lane < a.seqs.B ? rank : lane;
      co = __builtin_amdgcn_ds_permute(4 * rank, c);
      from = __builtin_amdgcn_ds_permute(4 * rank, lane);
    }
    const int io = scan_lanes(co);
    const uint64_t past = __builtin_amdgcn_ballot_w64(base + io > t);
    if (past && !found) {
      found = true;
      const int lo = __builtin_ctzll(past), l = __builtin_amdgcn_readlane(from, lo);
      auto lane_of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      local = base + __builtin_amdgcn_readlane(io, lo) - 1 - t;   // from the sequence's last item back
      it.b = b0 + l;
      it.n = lane_of(s.n);
      it.tok0 = lane_of(s.row);
      it.end = lane_of(s.end);
      it.splits = lane_of(k);
      it.narrow = is_narrow(a, it.n);
      it.start = it.end - it.n;
      it.part = part0 + lane_of(ir - rows);
      block0 += lane_of(ib - blocks);
    }
    if (!found) block0 += __builtin_amdgcn_readlane(ib, 63);
    base += __builtin_amdgcn_readlane(io, 63);
    part0 += __builtin_amdgcn_readlane(ir, 63);
  }
  if (!found) return false;
  const uint32_t mul_k = it.splits > 1 ? 0xFFFFFFFFu / (uint32_t)it.splits : 0xFFFFFFFFu;
  const int tile = (int)fast_div((uint32_t)local, (uint32_t)it.splits, mul_k);
  it.split = local - tile * it.splits;
  const int rows = it.narrow ? CK_ROWS : CK_WIDE_ROWS;
  it.list = nullptr;
  it.list_chunks = 0;
  if (a.sel_off) {
    const int blk = it.narrow ? 0 : (int)fast_div((uint32_t)tile, (uint32_t)a.tiles_per_block, a.mul_tpb);
    const int sub = it.narrow ? tile : tile - blk * a.tiles_per_block;
    it.row_end = min(it.n, (blk + 1) * CK_BLOCK) * a.G;
    it.row0 = blk * CK_BLOCK * a.G + sub * rows;
    if (it.row0 >= it.row_end) return false;
    it.row_end = min(it.row_end, it.row0 + rows);
    const int sr = block0 + blk;
    if (sr >= a.sel_rows) return false;
    const int32_t* off = a.sel_off + sr * a.off_sr + it.kvh * a.off_sh;
    const int e0 = min(max(off[0], 0), a.sel_width), e1 = min(max(off[1], e0), a.sel_width);
    it.list = a.sel + sr * a.sel_sr + it.kvh * a.sel_sh + e0;
    it.list_chunks = a.max_blocks > 0 ? (e1 - e0) * (a.page / 16) : 0;
  } else {
    it.row0 = tile * rows;
    it.row_end = (int)min((int64_t)it.n * a.G, (int64_t)it.row0 + rows);
  }
  it.pos_max = it.start + (int)fast_div((uint32_t)(it.row_end - 1), (uint32_t)a.G, a.mul_G);
  // Lengths past the table end with it.
  const int last = (int)min((int64_t)it.pos_max, (int64_t)a.max_blocks * a.page - 1);
  const int chunks = a.sel_off ? it.list_chunks : last < 0 ? 0 : last / 16 + 1;
  const int nt = (chunks + 3) / 4;   // at most 2^24, and 64 splits
  it.c0 = 4 * (int)fast_div((uint32_t)(nt * it.split), (uint32_t)it.splits, mul_k);
  it.c1 = min(chunks, 4 * (int)fast_div((uint32_t)(nt * (it.split + 1)), (uint32_t)it.splits, mul_k));
  return true;
}

// 64 chunks looked up at once: lane i holds where chunk base + i of the item lies in the pools (elements from
// the KV head's start) and its first key position, CK_NO_KEY if no row of the item sees it.
struct ChunkWindow {
  int base;
  int64_t off;
  int key;

  __device__ __forceinline__ void fill(const ChunkArgs& a, const ChunkItem& it, int first) {
    base = first;
    const int x = first + (int)(threadIdx.x & 63);
    key = CK_NO_KEY;
    off = 0;
    if (x < it.c1) {
      int lb, slot;
      if (it.list) {
        const int e = (int)fast_div((uint32_t)x, (uint32_t)(a.page / 16), a.mul_ppc);
        lb = it.list[e];
        slot = (x - e * (a.page / 16)) * 16;
      } else {
        lb = (int)fast_div((uint32_t)(16 * x), (uint32_t)a.page, a.mul_page);
        slot = 16 * x - lb * a.page;
      }
      if (lb >= 0 && lb < a.max_blocks && (int64_t)lb * a.page + slot <= it.pos_max) {
        const int pg = a.table[it.b * a.table_stride + lb];
        if (pg >= 0 && pg < a.num_pages) {
          off = (int64_t)pg * a.kv_sp + (int64_t)slot * a.kv_st;
          key = lb * a.page + slot;
        }
      }
    }
  }
  __device__ __forceinline__ int key_of(int c) const { return __builtin_amdgcn_readlane(key, c - base); }
  __device__ __forceinline__ int64_t off_of(int c) const {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(uint64_t)off, c - base);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)off >> 32), c - base);
    return (int64_t)(((uint64_t)hi << 32) | lo);
  }
};

// 32 rows to a workgroup: its first four waves hold the same rows and divide the keys, each with tiles of its own in
// LDS and no barrier before they merge.  Bound by the keys' bytes: a wave keeps 32 KB of loads in flight.  8 sequences of
// 4 new tokens over 4,001 to 4,096 keys, 32/8 heads, bf16, D = 128: 34 us for 132 MB, and 4 to 5 for the merge.
template <bool BF16, int D>
struct ChunkNarrow : StagedTile {
  using E = Elem<BF16>;
  static constexpr int NW = 4;
  static constexpr int NCG = D / 32;               // column groups of a staged tile
  static constexpr int NI = 4 * NCG;               // 1 KiB direct loads of a tile
  static constexpr int TILE_BYTES = CK_KT * D * 2;
  static constexpr int LDS_BYTES = NW * 2 * TILE_BYTES;
  static_assert(LDS_BYTES >= NW * CK_ROWS * D * 4, "the accumulators are merged in the staging buffers");
  // The row reference is raised when a lane's probabilities of a tile sum past this: no probability then
  // exceeds 2^16 in bf16 (2^15 in fp16, whose largest is 65,504).
  static constexpr float REFIT_SUM = BF16 ? 65536.f : 32768.f;

  static __device__ __forceinline__ void wait_reads() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  template <int LEFT>
  static __device__ __forceinline__ void wait_loads() {  // until at most LEFT of the wave's loads are in flight
    asm volatile("s_waitcnt vmcnt(%0)" ::"i"(LEFT) : "memory");
  }

  // Direct loads of the 64 keys of chunks c .. c + 3 into `tile`.
  template <bool PERMUTE>
  static __device__ __forceinline__ void load_tile(const ChunkArgs& a, const ChunkItem& it, const ChunkWindow& w,
                                                   const elem_t* head, char* tile, int c, int lane, uint32_t lane_off) {
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      const int key = w.key_of(c + rb);
      const elem_t* src = head + w.off_of(c + rb);
      const uint32_t lds = lds_addr(tile + rb * 1024);
      if (key + 16 <= it.end) {
#pragma unroll
        for (int cg = 0; cg < NCG; ++cg) load_lds16(src + 32 * cg, lane_off, lds + cg * 4096);
      } else {
        const int r = PERMUTE ? krow(lane >> 2) : lane >> 2;
        const bool live = key + r < it.end;
#pragma unroll
        for (int cg = 0; cg < NCG; ++cg) {
          const void* p = live ? (const void*)(src + r * a.kv_st + 32 * cg + dma_col(lane)) : (const void*)c_zero16;
          load_lds16(p, lds + cg * 4096);
        }
      }
    }
  }

  // s_ml: 2 * CK_ROWS floats a wave.
  static __device__ void run(const ChunkArgs& a, const ChunkItem& it, char* s_kv, float* s_ml) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 5, l32 = lane & 31;
    if (wave >= NW) {   // the barriers of the merge below
      __syncthreads();
      __syncthreads();
      return;
    }
    const int row = min(it.row0 + l32, it.row_end - 1);
    const int token = (int)fast_div((uint32_t)row, (uint32_t)a.G, a.mul_G);
    const int pos = it.start + token;
    const int pos_min = it.start + (int)fast_div((uint32_t)it.row0, (uint32_t)a.G, a.mul_G);
    u32x4 qf[D / 16];
    {
      const elem_t* qs = a.q + (int64_t)(it.tok0 + token) * a.q_st + (it.kvh * a.G + row - token * a.G) * a.q_sh + 8 * g;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) qf[c] = *reinterpret_cast<const u32x4*>(qs + 16 * c);
    }
    const Frag f(lane);
    char* sK = s_kv + wave * 2 * TILE_BYTES;
    char* sV = sK + TILE_BYTES;
    const elem_t* kh = a.k + it.kvh * a.kv_sh;
    const elem_t* vh = a.v + it.kvh * a.kv_sh;
    const uint32_t koff = (uint32_t)((krow(lane >> 2) * a.kv_st + dma_col(lane)) * 2);
    const uint32_t voff = (uint32_t)(((lane >> 2) * a.kv_st + dma_col(lane)) * 2);

    f32x16 O[NCG];
#pragma unroll
    for (int dt = 0; dt < NCG; ++dt) O[dt] = f32x16{};
    float m_ref = -__builtin_inff(), neg_m = 0.f, l_run = 0.f;
    bool ref_ok = false;
    const float c = a.scale_log2;

    // This wave's share of the item's tiles.
    const int nt = (it.c1 - it.c0 + 3) / 4;
    const int t0 = nt * wave / NW, t1 = nt * (wave + 1) / NW;
    ChunkWindow w;
    w.base = 0;
    auto look = [&](int ch) {
      if (ch - w.base >= 64) w.fill(a, it, ch);
    };
    auto raise = [&](const f32x16 (&S)[2]) {
      float mx = S[0][0];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, S[j][r]);
      const float m_new = fmaxf(m_ref, halves_max(mx) * c);  // -inf stays -inf (c > 0)
      const float alpha = m_ref == -__builtin_inff() ? 1.f : fast_exp2(m_ref - m_new);
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < NCG; ++dt) O[dt] *= alpha;
      m_ref = m_new;
      neg_m = m_ref == -__builtin_inff() ? 0.f : -m_ref;
      ref_ok = !__any(m_ref == -__builtin_inff());
    };
    u32x4 P[2][2];
    auto probs = [&](const f32x16 (&S)[2]) {
      float ls = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p0 = fast_exp2(fmaf(S[j][8 * h + 2 * e], c, neg_m));
            const float p1 = fast_exp2(fmaf(S[j][8 * h + 2 * e + 1], c, neg_m));
            ls += p0 + p1;
            P[j][h][e] = E::pack2f(p0, p1);
          }
      return ls;
    };

    if (t0 < t1) {
      int ch = it.c0 + 4 * t0;
      w.fill(a, it, ch);
      load_tile<true>(a, it, w, kh, sK, ch, lane, koff);
      load_tile<false>(a, it, w, vh, sV, ch, lane, voff);
      for (int t = t0; t < t1; ++t, ch += 4) {
        int key[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) key[x] = w.key_of(ch + x);
        wait_loads<NI>();  // K is in LDS, V may be in flight
        f32x16 S[2] = {f32x16{}, f32x16{}};
#pragma unroll
        for (int cc = 0; cc < D / 16; ++cc)
#pragma unroll
          for (int j = 0; j < 2; ++j) S[j] = E::mfma32(kfrag(sK, f, j, cc), qf[cc], S[j]);
        const bool more = t + 1 < t1;
        if (more) {
          look(ch + 4);
          wait_reads();
          load_tile<true>(a, it, w, kh, sK, ch + 4, lane, koff);
        }
        // Keys past a row's position, in the tiles that hold any.
        if (max(max(key[0], key[1]), max(key[2], key[3])) + 15 > pos_min) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int lim = pos - key[2 * j + h] - 8 * g;
#pragma unroll
              for (int e = 0; e < 8; ++e) S[j][8 * h + e] = e > lim ? -__builtin_inff() : S[j][8 * h + e];
            }
        }
        if (!ref_ok) raise(S);
        float ls = probs(S);
        if (__any(!(ls <= REFIT_SUM))) {
          raise(S);
          ls = probs(S);
        }
        l_run += ls;
        if (more)
          wait_loads<NI>();  // V is in LDS, the next K may be in flight
        else
          wait_loads<0>();
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int dt = 0; dt < NCG; ++dt) O[dt] = E::mfma32(vfrag(sV, f, j, h, dt), P[j][h], O[dt]);
        if (more) {
          wait_reads();
          load_tile<false>(a, it, w, vh, sV, ch + 4, lane, voff);
        }
      }
    }

    // Merge of the waves' shares through LDS, in fp32: accumulator row r is D floats at r * 4 D, its 16-byte
    // chunk x at position x ^ (r % (D / 4)).
    constexpr int NC4 = D / 4, OC = D / 8 / NW, ACC = CK_ROWS * D * 4;
    const float lt = halves_sum(l_run);
    __syncthreads();
    char* acc = s_kv + wave * ACC;
#pragma unroll
    for (int dt = 0; dt < NCG; ++dt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {  // d = 32 dt + 8 rq + 4 g + 0..3
        const int x = 8 * dt + 2 * rq + g;
        *reinterpret_cast<f32x4*>(acc + l32 * 4 * D + 16 * (x ^ (l32 & (NC4 - 1)))) =
            f32x4{O[dt][4 * rq], O[dt][4 * rq + 1], O[dt][4 * rq + 2], O[dt][4 * rq + 3]};
      }
    if (g == 0) {
      s_ml[wave * 2 * CK_ROWS + l32] = m_ref;
      s_ml[wave * 2 * CK_ROWS + CK_ROWS + l32] = lt;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < CK_ROWS * OC / 64; ++k) {
      const int x = 64 * k + lane;
      const int r = x / OC, oc = wave * OC + x % OC;
      float m[NW], l = 0.f, M = -__builtin_inff();
#pragma unroll
      for (int s = 0; s < NW; ++s) {
        m[s] = s_ml[s * 2 * CK_ROWS + r];
        M = fmaxf(M, m[s]);
      }
      const float Mu = M == -__builtin_inff() ? 0.f : M;
      f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll
      for (int s = 0; s < NW; ++s) {
        const float fs = fast_exp2(m[s] - Mu);
        l += fs * s_ml[s * 2 * CK_ROWS + CK_ROWS + r];
        const char* p = s_kv + s * ACC + r * 4 * D;
        lo += fs * *reinterpret_cast<const f32x4*>(p + 16 * ((2 * oc) ^ (r & (NC4 - 1))));
        hi += fs * *reinterpret_cast<const f32x4*>(p + 16 * ((2 * oc + 1) ^ (r & (NC4 - 1))));
      }
      if (it.row0 + r < it.row_end) {
        const int tk = (int)fast_div((uint32_t)(it.row0 + r), (uint32_t)a.G, a.mul_G);
        const int h = it.kvh * a.G + it.row0 + r - tk * a.G;
        if (it.splits > 1) {
          const int64_t at = it.part_row(a, tk, h);
          f32x4* d = reinterpret_cast<f32x4*>(a.part_acc + at * D + 8 * oc);
          d[0] = lo;
          d[1] = hi;
          if (oc == 0) {
            a.part_ml[2 * at] = M;
            a.part_ml[2 * at + 1] = l;
          }
        } else {
          const float inv = l > 0.f ? 1.f / l : 1.f;
          *reinterpret_cast<u32x4*>(a.o + (int64_t)(it.tok0 + tk) * a.o_st + h * a.o_sh + 8 * oc) =
              u32x4{E::pack2f(lo[0] * inv, lo[1] * inv), E::pack2f(lo[2] * inv, lo[3] * inv),
                    E::pack2f(hi[0] * inv, hi[1] * inv), E::pack2f(hi[2] * inv, hi[3] * inv)};
        }
      }
    }
  }
};

// 256 rows to a workgroup: eight waves of 32 rows share every K/V tile, which direct loads bring into LDS while the
// tile before is worked on.  One step per tile and one barrier per step.  Block A of a step runs S^T = K Q^T of the
// next tile on the matrix cores under the exponentials of this one, block B O^T += V^T P^T.  Waves 0..3 run A(i),
// B(i) in step i and waves 4..7, one on each SIMD beside them, B(i - 1), A(i), so that the two waves of a SIMD run the
// vector-heavy A and the matrix-only B at the same time.  Step i issues the loads of K(i + 3) and V(i + 2) and ends
// with a wait for those of the step before, so a tile has two steps to arrive; the waves read K(i + 1), V(i) and
// V(i - 1) meanwhile, hence three K and four V buffers.
// A row's reference is the maximum of its first tile and is raised only when its probabilities would pass the
// element type's range (REFIT_SUM), so the common step never touches O with vector instructions.
// Bound by the step: 1.75 us of it per tile at D = 128 with the chip full, 1.35 at D = 64 (exponentials).  8K new tokens
// over 32K keys, 32/8 heads, bf16, take 3.1 to 3.3 ms on different cards, 1.16 to 1.24 PFLOP/s
// where a large matrix product reaches 1.44.  Over a selection an item holds rows of one block of 64 tokens only: all 256
// are in use for groups of 4 and 8, 64 for groups of one, 128 for 2, 320 of 512 for 5.
template <bool BF16, int D>
struct ChunkWide : StagedTile {
  using E = Elem<BF16>;
  static constexpr int NW = 8;
  static_assert(NW * CK_ROWS == CK_WIDE_ROWS, "rows of a wide item");
  static constexpr int NCG = D / 32;
  static constexpr int NIW = 4 * NCG / NW;         // direct loads of a tile per wave: one row block each
  static constexpr int TILE_BYTES = CK_KT * D * 2;
  static constexpr int NBK = 3, NBV = 4;
  static constexpr int STAGE = CK_ROWS * D * 2;    // a wave's share of O
  static constexpr int LDS_BYTES = (NBK + NBV) * TILE_BYTES;
  static constexpr int KEYS = NW * 4 * 64;         // ints of LDS for the tiles' first keys
  static_assert(NW * STAGE <= LDS_BYTES, "O is staged in the K/V buffers");
  static constexpr float REFIT_SUM = BF16 ? 65536.f : 32768.f;

  // 64 tiles looked up at once: lane i holds, for tile base + i, the place and first key of the chunk that this
  // wave loads, and the tile's largest key; the first keys of its four chunks go to LDS, for the tiles that need
  // a mask.  Tiles are loaded two ahead of the one whose mask is due, so a window starts two tiles back.
  struct Window {
    int base;
    int64_t off;
    int key, last;

    // Four 32-bit reads that have completed when it returns: one opaque block, so that the compiler has no pending
    // load whose wait would cover the direct loads in the tile loop.
    static __device__ __forceinline__ void read4(const int32_t* const (&p)[4], int (&x)[4]) {
      asm volatile(
          "global_load_dword %0, %4, off\n\t"
          "global_load_dword %1, %5, off\n\t"
          "global_load_dword %2, %6, off\n\t"
          "global_load_dword %3, %7, off\n\t"
          "s_waitcnt vmcnt(0)"
          : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
          : "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3])
          : "memory");
    }
    __device__ __forceinline__ void fill(const ChunkArgs& a, const ChunkItem& it, int first, int rb, int* s_keys) {
      base = first;
      const int lane = threadIdx.x & 63;
      int lb[4], slot[4], page[4], keys[4];
      const int32_t* p[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int c = it.c0 + 4 * (first + lane) + x;
        keys[x] = c < it.c1 ? 0 : CK_NO_KEY;
        if (it.list) {
          const int e = (int)fast_div((uint32_t)c, (uint32_t)(a.page / 16), a.mul_ppc);
          p[x] = it.list + (c < it.c1 ? e : 0);   // there is an entry: the item has a chunk
          slot[x] = (c - e * (a.page / 16)) * 16;
        } else {
          lb[x] = (int)fast_div((uint32_t)(16 * c), (uint32_t)a.page, a.mul_page);
          slot[x] = 16 * c - lb[x] * a.page;
        }
      }
      if (it.list) read4(p, lb);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        // (a page whose first key no row sees is not looked up; neither are ids that are no column)
        if (lb[x] < 0 || lb[x] >= a.max_blocks || (int64_t)lb[x] * a.page + slot[x] > it.pos_max) keys[x] = CK_NO_KEY;
        p[x] = a.table + it.b * a.table_stride + (keys[x] ? 0 : lb[x]);
      }
      read4(p, page);
      key = CK_NO_KEY;
      off = 0;
      last = -1;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (page[x] < 0 || page[x] >= a.num_pages) keys[x] = CK_NO_KEY;
        if (!keys[x]) keys[x] = lb[x] * a.page + slot[x];
        else keys[x] = CK_NO_KEY;
        if (x == rb && keys[x] != CK_NO_KEY) {
          off = (int64_t)page[x] * a.kv_sp + (int64_t)slot[x] * a.kv_st;
          key = keys[x];
        }
        last = max(last, keys[x] + 15);
      }
      *reinterpret_cast<int4*>(s_keys + 4 * lane) = int4{keys[0], keys[1], keys[2], keys[3]};
    }
    __device__ __forceinline__ int key_of(int t) const { return __builtin_amdgcn_readlane(key, t - base); }
    __device__ __forceinline__ int last_of(int t) const { return __builtin_amdgcn_readlane(last, t - base); }
    __device__ __forceinline__ int64_t off_of(int t) const {
      const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(uint64_t)off, t - base);
      const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)off >> 32), t - base);
      return (int64_t)(((uint64_t)hi << 32) | lo);
    }
  };

  static __device__ void run(const ChunkArgs& a, const ChunkItem& it, char* s_kv, int* s_all_keys) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 5, l32 = lane & 31;
    int* s_keys = s_all_keys + 4 * 64 * wave;
    char* sK = s_kv;
    char* sV = s_kv + NBK * TILE_BYTES;

    const int row0 = min(it.row0 + CK_ROWS * wave, it.row_end - 1);   // a wave past the rows repeats the last one
    const int row = min(row0 + l32, it.row_end - 1);
    const int token = (int)fast_div((uint32_t)row, (uint32_t)a.G, a.mul_G);
    const int pos_min = it.start + (int)fast_div((uint32_t)row0, (uint32_t)a.G, a.mul_G);
    const int pos8 = it.start + token - 8 * g;   // a key at offset e of a chunk's lane half is seen if e <= pos8 - key
    u32x4 Qr[D / 16];
    {
      const elem_t* qs = a.q + (int64_t)(it.tok0 + token) * a.q_st + (it.kvh * a.G + row - token * a.G) * a.q_sh + 8 * g;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) Qr[c] = *reinterpret_cast<const u32x4*>(qs + 16 * c);
    }
    const Frag f(lane);
    const float c = a.scale_log2;

    // This wave's direct loads of a tile: NIW column groups of row block rb.
    const int rb = wave * NIW / NCG, cg0 = wave * NIW % NCG;
    const char* kh = reinterpret_cast<const char*>(a.k + it.kvh * a.kv_sh + 32 * cg0);
    const char* vh = reinterpret_cast<const char*>(a.v + it.kvh * a.kv_sh + 32 * cg0);
    const uint32_t koff = (uint32_t)((krow(lane >> 2) * a.kv_st + dma_col(lane)) * 2);
    const uint32_t voff = (uint32_t)(((lane >> 2) * a.kv_st + dma_col(lane)) * 2);
    const uint32_t lds_k = lds_addr(sK + cg0 * 4096 + rb * 1024);
    const uint32_t lds_v = lds_addr(sV + cg0 * 4096 + rb * 1024);
    const int nt = (it.c1 - it.c0 + 3) / 4;
    Window w;
    auto load = [&](const char* head, uint32_t lane_off, int r, uint32_t lds, int t) {
      const char* src = head + 2 * w.off_of(t);
      const int key = w.key_of(t);
      if (key + 16 <= it.end) {
        load_lds16_at<0>(src, lane_off, lds);
        if constexpr (NIW > 1) load_lds16_at<64>(src, lane_off, lds + 4096);
      } else {   // keys that are not there are zeros
        const bool live = key + r < it.end;
#pragma unroll
        for (int u = 0; u < NIW; ++u)
          load_lds16(live ? (const void*)(src + lane_off + 64 * u) : (const void*)c_zero16, lds + u * 4096);
      }
    };
    auto load_k = [&](int t, int kb) {
      if (t - w.base >= 64) w.fill(a, it, t - 2, rb, s_keys);
      load(kh, koff, krow(lane >> 2), lds_k + kb * TILE_BYTES, t);
    };
    auto load_v = [&](int t, int vb) { load(vh, voff, lane >> 2, lds_v + vb * TILE_BYTES, t); };
    // Scores of tile t past a row's position become -inf.
    auto mask = [&](f32x16 (&S)[2], int t) {
      if (w.last_of(t) <= pos_min) return;
      const int4 keys = *reinterpret_cast<const int4*>(&s_keys[4 * (t - w.base)]);
      const int lim[4] = {pos8 - keys.x, pos8 - keys.y, pos8 - keys.z, pos8 - keys.w};
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            S[j][8 * h + e] = e > lim[2 * j + h] ? -__builtin_inff() : S[j][8 * h + e];
    };

    f32x16 O[NCG];
#pragma unroll
    for (int dt = 0; dt < NCG; ++dt) O[dt] = f32x16{};
    float m_ref = -__builtin_inff(), l_run = 0.f;
    f32x16 S[2] = {f32x16{}, f32x16{}};
    if (nt > 0) {
      w.fill(a, it, 0, rb, s_keys);
      load_k(0, 0);
      load_v(0, 0);
      if (nt > 1) {
        load_k(1, 1);
        load_v(1, 1);
      }
      if (nt > 2) load_k(2, 2);
      wait_dma();
      __syncthreads();
#pragma unroll
      for (int cc = 0; cc < D / 16; ++cc)
#pragma unroll
        for (int j = 0; j < 2; ++j) S[j] = E::mfma32(kfrag(sK, f, j, cc), Qr[cc], S[j]);
      mask(S, 0);
      float mx = S[0][0];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, S[j][r]);
      m_ref = halves_max(mx) * c;   // -inf stays -inf (c > 0)
      __syncthreads();              // K of tile 0 has been read
    }
    float neg_m = m_ref == -__builtin_inff() ? 0.f : -m_ref;
    bool ref_ok = !__any(m_ref == -__builtin_inff());

    const bool lag = wave >= NW / 2;
    int vb_cur = 0, kb_cur = 0;   // buffers of the current tile
    bool pending = false;
    auto ring = [](int x, int n) { return x >= n ? x - n : x; };
    u32x4 P[2][2];
    constexpr int NQ = D / 8;    // QK MFMAs of a tile: i -> (key half i % 2, cc = i / 2)
    constexpr int PE = 32 / NQ;  // probabilities per QK MFMA
    constexpr int NP = D / 8;    // PV MFMAs: i -> (dt = i % NCG, h, j)

    auto block_b = [&](const char* cV) {
      auto vfr = [&](int i) { return vfrag(cV, f, i / (2 * NCG), (i / NCG) & 1, i % NCG); };
      u32x4 vf[2] = {vfr(0), vfr(1)};
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        O[i % NCG] = E::mfma32(vf[i & 1], P[i / (2 * NCG)][(i / NCG) & 1], O[i % NCG]);
        if (i + 2 < NP) vf[i & 1] = vfr(i + 2);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto probs = [&](const f32x16 (&Sc)[2], float& ls) {
      ls = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p0 = fast_exp2(fmaf(Sc[j][8 * h + 2 * e], c, neg_m));
            const float p1 = fast_exp2(fmaf(Sc[j][8 * h + 2 * e + 1], c, neg_m));
            ls += p0 + p1;
            P[j][h][e] = E::pack2f(p0, p1);
          }
    };
    // Rare: a row without a reference yet, or probabilities past REFIT_SUM.
    auto raise = [&](const f32x16 (&Sc)[2], float& ls) {
      float mx = Sc[0][0];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, Sc[j][r]);
      const float m_new = fmaxf(m_ref, halves_max(mx) * c);
      const float alpha = m_ref == -__builtin_inff() ? 1.f : fast_exp2(m_ref - m_new);
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < NCG; ++dt) O[dt] *= alpha;
      m_ref = m_new;
      neg_m = m_ref == -__builtin_inff() ? 0.f : -m_ref;
      ref_ok = !__any(m_ref == -__builtin_inff());
      probs(Sc, ls);
    };

    // One step on tile t, whose scores are in Sc; fills Sx with the next tile's.
    auto step = [&](int t, f32x16 (&Sc)[2], f32x16 (&Sx)[2]) {
      const bool ahead = t + 3 < nt;
      if (ahead) load_k(t + 3, kb_cur);
      if (t + 2 < nt) load_v(t + 2, ring(vb_cur + 2, NBV));
      if (lag && pending) block_b(sV + ring(vb_cur + NBV - 1, NBV) * TILE_BYTES);
      const char* cK = sK + ring(kb_cur + 1, NBK) * TILE_BYTES;
      auto kfr = [&](int i) { return kfrag(cK, f, i & 1, i >> 1); };
      u32x4 kf[3] = {kfr(0), kfr(1), kfr(2)};
      Sx[0] = f32x16{};
      Sx[1] = f32x16{};
      float ls = 0.f;
      uint32_t pw[2][2][4];
      __builtin_amdgcn_s_setprio(1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        Sx[i & 1] = E::mfma32(kf[i % 3], Qr[i >> 1], Sx[i & 1]);
        if (i + 3 < NQ) kf[i % 3] = kfr(i + 3);
#pragma unroll
        for (int u = 0; u < PE; u += 2) {
          const int x = PE * i + u, j = x >> 4, rr = x & 15;
          const float p0 = fast_exp2(fmaf(Sc[j][rr], c, neg_m));
          const float p1 = fast_exp2(fmaf(Sc[j][rr + 1], c, neg_m));
          ls += p0 + p1;
          uint32_t pk = E::pack2f(p0, p1);
          asm volatile("" : "+v"(pk), "+v"(ls));   // computed here, not sunk to its use in block B
          pw[j][rr >> 3][(rr & 7) >> 1] = pk;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) P[j][h] = u32x4{pw[j][h][0], pw[j][h][1], pw[j][h][2], pw[j][h][3]};
      if (!ref_ok || __any(!(ls <= REFIT_SUM))) raise(Sc, ls);
      l_run += ls;
      mask(Sx, t + 1);
      if (!lag) block_b(sV + vb_cur * TILE_BYTES);
      pending = true;
      if (ahead)
        __builtin_amdgcn_s_waitcnt(0x0F70 | (2 * NIW));   // vmcnt: this step's loads may be in flight
      else
        wait_dma();
      __syncthreads();
      vb_cur = ring(vb_cur + 1, NBV);
      kb_cur = ring(kb_cur + 1, NBK);
    };
    if (nt > 0) {
      f32x16 Sn[2];
      int t = 0;
      while (t + 2 < nt) {
        step(t, S, Sn);
        step(t + 1, Sn, S);
        t += 2;
      }
      if (t + 1 < nt) {
        step(t, S, Sn);
        S[0] = Sn[0];
        S[1] = Sn[1];
      }
      // The last tile: no next one, nothing to load.
      if (lag && pending) block_b(sV + ring(vb_cur + NBV - 1, NBV) * TILE_BYTES);
      float ls;
      probs(S, ls);
      if (!ref_ok || __any(!(ls <= REFIT_SUM))) raise(S, ls);
      l_run += ls;
      block_b(sV + vb_cur * TILE_BYTES);
    }
    __syncthreads();   // the K/V buffers are free
    const float lt = halves_sum(l_run);
    if (it.splits > 1) {
      if (it.row0 + CK_ROWS * wave + l32 < it.row_end) {
        const int64_t at = it.part_row(a, token, it.kvh * a.G + row - token * a.G);
#pragma unroll
        for (int dt = 0; dt < NCG; ++dt)
#pragma unroll
          for (int rq = 0; rq < 4; ++rq)
            *reinterpret_cast<f32x4*>(a.part_acc + at * D + 32 * dt + 8 * rq + 4 * g) =
                f32x4{O[dt][4 * rq], O[dt][4 * rq + 1], O[dt][4 * rq + 2], O[dt][4 * rq + 3]};
        if (g == 0) {
          a.part_ml[2 * at] = m_ref;
          a.part_ml[2 * at + 1] = lt;
        }
      }
      return;
    }
    // O / l through this wave's 32 x D staging area: 16-byte chunk x of row r at position x ^ (r % (D / 8)); each
    // store instruction then writes whole rows.
    constexpr int NCH = D / 8, RPI = 64 / NCH;
    const float inv = lt > 0.f ? 1.f / lt : 1.f;
    char* stage = s_kv + wave * STAGE;
#pragma unroll
    for (int dt = 0; dt < NCG; ++dt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const int x = 4 * dt + rq;
        *reinterpret_cast<u32x2*>(stage + l32 * 2 * D + 16 * (x ^ (l32 & (NCH - 1))) + 8 * g) =
            u32x2{E::pack2f(O[dt][4 * rq] * inv, O[dt][4 * rq + 1] * inv),
                  E::pack2f(O[dt][4 * rq + 2] * inv, O[dt][4 * rq + 3] * inv)};
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the wave reads back what its own lanes wrote
    const int p = lane % NCH;
#pragma unroll
    for (int k = 0; k < CK_ROWS / RPI; ++k) {
      const int r = RPI * k + lane / NCH;
      const u32x4 v = *reinterpret_cast<const u32x4*>(stage + r * 2 * D + 16 * p);
      const int fr = it.row0 + CK_ROWS * wave + r;
      if (fr < it.row_end) {
        const int tk = (int)fast_div((uint32_t)fr, (uint32_t)a.G, a.mul_G);
        __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(a.o + (int64_t)(it.tok0 + tk) * a.o_st +
                                                                 (it.kvh * a.G + fr - tk * a.G) * a.o_sh +
                                                                 8 * (p ^ (r & (NCH - 1)))));
      }
    }
  }
};

template <bool BF16, int D>
__global__ __launch_bounds__(512, 2) void chunk_kernel(const ChunkArgs a) {
  using W = ChunkWide<BF16, D>;
  using S = ChunkNarrow<BF16, D>;
  __shared__ __attribute__((aligned(16))) char s_kv[W::LDS_BYTES > S::LDS_BYTES ? W::LDS_BYTES : S::LDS_BYTES];
  __shared__ __attribute__((aligned(16))) int s_aux[W::KEYS];
  ChunkItem it;
  if (!find_chunk_item(a, blockIdx.x, it)) return;
  if (it.narrow)
    S::run(a, it, s_kv, reinterpret_cast<float*>(s_aux));
  else
    W::run(a, it, s_kv, s_aux);
}

// Merges the partials of the rows (token, head), D / 8 lanes a row, after the workgroups of the launch before have left
// them; rows of sequences that were not split are done.  Each lane of a wave holds one sequence's range of
// rows and place, so a row finds its own without a chain of reads.
template <bool BF16, int D>
__global__ __launch_bounds__(256) void chunk_combine_kernel(const ChunkArgs a) {
  using E = Elem<BF16>;
  constexpr int LPR = D / 8, U = 4;
  const int lane = threadIdx.x & 63, oc = threadIdx.x % LPR;
  const int64_t rows = a.seqs.N * a.Hq;
  for (int b0 = 0; b0 < a.seqs.B; b0 += 64) {
    SeqPart sp = {0, 1, 0, 0};
    int r0 = 0, n_of = 0;
    if (b0 + lane < a.seqs.B) {
      sp = a.part[b0 + lane];
      n_of = a.seqs.rows(b0 + lane, r0);
    }
    if (!__any(sp.any != 0)) return;
    if (sp.n != n_of) sp.splits = 1;   // lengths that changed under the launch
    const uint64_t split = __builtin_amdgcn_ballot_w64(sp.splits > 1 && n_of > 0);
    for (int64_t w0 = ((int64_t)blockIdx.x * 256 + threadIdx.x - lane) / LPR; w0 < rows && split;
         w0 += (int64_t)gridDim.x * (256 / LPR)) {
      const int64_t row = w0 + lane / LPR;
      const int n = row < rows ? (int)fast_div((uint32_t)row, (uint32_t)a.Hq, a.mul_Hq) : -1;
      int first = 0, k = 0, tokens = 0, at0 = 0;
      for (uint64_t m = split; m; m &= m - 1) {
        const int l = __builtin_ctzll(m);
        const int s0 = __builtin_amdgcn_readlane(r0, l), sn = __builtin_amdgcn_readlane(n_of, l);
        if (n >= s0 && n < s0 + sn) {
          first = __builtin_amdgcn_readlane(sp.first, l);
          k = __builtin_amdgcn_readlane(sp.splits, l);
          tokens = sn;
          at0 = s0;
        }
      }
      if (k <= 1) continue;
      const int h = (int)(row - (int64_t)n * a.Hq);
      const int64_t step = (int64_t)tokens * a.Hq, at = first + (int64_t)(n - at0) * a.Hq + h;
      float M = -__builtin_inff(), L = 0.f;
      f32x4 acc[2] = {f32x4{}, f32x4{}};
      for (int s0 = 0; s0 < k; s0 += U) {
        float m[U], l[U];
        f32x4 v[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t p = at + min(s0 + u, k - 1) * step;   // past the last: a repeat, not used
          m[u] = a.part_ml[2 * p];
          l[u] = a.part_ml[2 * p + 1];
          v[u][0] = reinterpret_cast<const f32x4*>(a.part_acc + p * D + 8 * oc)[0];
          v[u][1] = reinterpret_cast<const f32x4*>(a.part_acc + p * D + 8 * oc)[1];
        }
        float Mc = M;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (s0 + u < k) Mc = fmaxf(Mc, m[u]);
        // A share without a key of the row has a reference of -inf and sums of 0.  One whose scores are all NaN has a
        // reference of -inf or NaN, which the maximum passes over, and sums of NaN, which reach the row from here.
        const float Mu = Mc == -__builtin_inff() ? 0.f : Mc;
        const float f0 = fast_exp2(M - Mu);
        L *= f0;
        acc[0] *= f0;
        acc[1] *= f0;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (s0 + u < k) {
            const float fs = fast_exp2(m[u] - Mu);
            L += fs * l[u];
            acc[0] += fs * v[u][0];
            acc[1] += fs * v[u][1];
          }
        M = Mc;
      }
      const float inv = L > 0.f ? 1.f / L : 1.f;
      *reinterpret_cast<u32x4*>(a.o + (int64_t)n * a.o_st + h * a.o_sh + 8 * oc) =
          u32x4{E::pack2f(acc[0][0] * inv, acc[0][1] * inv), E::pack2f(acc[0][2] * inv, acc[0][3] * inv),
                E::pack2f(acc[1][0] * inv, acc[1][1] * inv), E::pack2f(acc[1][2] * inv, acc[1][3] * inv)};
    }
  }
}

template <bool BF16, int D>
static int launch_chunk(const ChunkArgs& a, int64_t groups, hipStream_t s) {
  hipLaunchKernelGGL((chunk_kernel<BF16, D>), dim3((unsigned)groups), dim3(512), 0, s, a);
  if (a.part) {
    const int64_t rows = a.seqs.N * a.Hq, per = 256 / (D / 8);
    hipLaunchKernelGGL((chunk_combine_kernel<BF16, D>), 
                       dim3((unsigned)std::min<int64_t>((rows + per - 1) / per, 2048)), dim3(256), 0, s, a);
  }
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : set_error((int)err, "sa_paged_chunk_attn: launch failed: %s", hipGetErrorString(err));
}

static int chunk_cus() {
  static int cached[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (!cached[dev]) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1) n = 256;
    cached[dev] = n;
  }
  return cached[dev];
}

// Row tiles that any division of N tokens over B sequences may have: a narrow sequence has at most two, a wide one
// its rows over 256 rounded up (or, with a selection, those of its blocks).
static int64_t chunk_tiles(int64_t N, int64_t B, int64_t G, bool blocks) {
  B = std::min(B, N);
  const int64_t per_block = (CK_BLOCK * G + CK_WIDE_ROWS - 1) / CK_WIDE_ROWS;
  if (blocks) return (N / CK_BLOCK + B) * std::max<int64_t>(per_block, CK_NARROW / CK_ROWS);
  return N * G / CK_WIDE_ROWS + std::min(B * (CK_NARROW / CK_ROWS), N * G / CK_ROWS + B);
}

// Row tiles and splits: a planned division has at most a workgroup per CU more than the row tiles need.
static int64_t chunk_items(int64_t N, int64_t B, int64_t G, int64_t Hkv, bool blocks, int splits) {
  const int64_t tiles = chunk_tiles(N, B, G, blocks);
  return splits ? tiles * splits : tiles + chunk_cus() / Hkv;
}

static int64_t chunk_part_header(int64_t B) { return (B * (int64_t)sizeof(SeqPart) + 255) / 256 * 256; }

static bool bad_ptr(const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; }

}  // namespace sa

using namespace sa;

extern "C" int64_t sa_paged_chunk_workspace_bytes(int N, int B, int Hq, int Hkv, int D, int max_keys, int num_splits) {
  if (N < 1 || B < 1 || Hkv < 1 || Hq < Hkv || D < 1 || max_keys < 1 || num_splits == 1 || num_splits < 0) return 0;
  const int64_t key_tiles = (max_keys + CK_KT - 1) / CK_KT;
  const int64_t all = (int64_t)N * Hq;
  if (num_splits > 1) return chunk_part_header(B) + all * std::min<int64_t>(num_splits, key_tiles) * (D + 2) * 4;
  // Nothing is gained where the row tiles fill the chip several times over, twice for those of one sequence, nor by
  // dividing few keys.  bf16, D = 128, 32/8 heads, divided against not: 8 sequences of 4 new tokens 13.6 us against 9.8 at
  // 512 keys, 18.6 against 15.2 at 1,024; 4 of 128 (wide) 22.1 against 19.0 at 512, but one of 64 21.9 against 28.8 at
  // 1,024.  One sequence of one token takes 11.7 against 12.9 at 1,024: less than the 3.5 us of host time that the
  // workspace and the second launch cost, so narrow items are not divided there either.
  const bool narrow = (int64_t)N * (Hq / Hkv) <= CK_NARROW * (int64_t)B;
  if (key_tiles <= (narrow ? 16 : 8) ||
      (int64_t)N * (Hq / Hkv) / CK_WIDE_ROWS * Hkv >= (B == 1 ? 2 : 8) * (int64_t)chunk_cus())
    return 0;
  return chunk_part_header(B) + std::min(all * std::min<int64_t>(key_tiles / 4 + 1, 64), CK_PART_ROWS) * (D + 2) * 4;
}

extern "C" int sa_paged_chunk_attn(int dtype, const void* q, int64_t q_st, int64_t q_sh, const void* k_pages,
                                   const void* v_pages, int64_t pages_sp, int64_t pages_sh, int64_t pages_st,
                                   int num_pages, const int32_t* block_table, int64_t block_table_stride,
                                   int max_blocks, const int32_t* cu_seqlens, const int32_t* kv_lens,
                                   const int32_t* sel, int64_t sel_sr, int64_t sel_sh, int sel_rows, int sel_width,
                                   const int32_t* sel_off, int64_t off_sr, int64_t off_sh, void* o, int64_t o_st,
                                   int64_t o_sh, int N, int B, int Hq, int Hkv, int D, int page, float sm_scale,
                                   int num_splits, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  const char* name = "sa_paged_chunk_attn";
  if (dtype != SA_DTYPE_BF16 && dtype != SA_DTYPE_F16)
    return set_error(SA_E_DTYPE, "%s: dtype %d is not bf16 (0) or f16 (1)", name, dtype);
  if (D != 64 && D != 128) return set_error(SA_E_HEADDIM, "%s: head dim %d not supported (64, 128)", name, D);
  if (page < 16 || page > 128 || page % 16)
    return set_error(SA_E_BLOCK, "%s: page %d is not a multiple of 16 in [16, 128]", name, page);
  if (N < 0 || B < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || Hq > (1 << 15) || max_blocks < 0 || num_pages < 0 ||
      block_table_stride < max_blocks || num_splits < 0 || num_splits > CK_MAX_SPLITS)
    return set_error(SA_E_SHAPE, "%s: bad sizes N=%d B=%d Hq=%d Hkv=%d, table of %d columns (stride %lld), %d pages, "
                     "%d splits (0..64)", name, N, B, Hq, Hkv, max_blocks, (long long)block_table_stride, num_pages,
                     num_splits);
  if (!(sm_scale >= 1e-30f && sm_scale <= 1e30f))
    return set_error(SA_E_SHAPE, "%s: scale %g is not in [1e-30, 1e30]", name, sm_scale);
  if ((int64_t)N * Hq > 0x7fffffff) return set_error(SA_E_SHAPE, "%s: N=%d x Hq=%d rows are too many", name, N, Hq);
  const bool selected = sel || sel_off;
  if (selected && (!sel_off || sel_width < 0 || sel_rows < (int64_t)N / CK_BLOCK + B))
    return set_error(SA_E_SHAPE, "%s: a selection needs offsets and %lld rows, got %d", name,
                     (long long)N / CK_BLOCK + B, sel_rows);
  if (N == 0 || B == 0) return 0;
  // A table without columns and pools without pages are never read.
  if (!q || (num_pages && (!k_pages || !v_pages)) || (max_blocks && !block_table) || !cu_seqlens || !kv_lens || !o ||
      (selected && sel_width && !sel))
    return set_error(SA_E_NULL, "%s: NULL pointer", name);
  if (bad_ptr(q) || bad_ptr(k_pages) || bad_ptr(v_pages) || bad_ptr(o) || bad_ptr(workspace) ||
      (q_st | q_sh | pages_sp | pages_sh | pages_st | o_st | o_sh) % 8)
    return set_error(SA_E_ALIGN, "%s: head rows must be 16-byte aligned", name);
  if (pages_st < 0 || pages_st > CK_MAX_STRIDE)
    return set_error(SA_E_SHAPE, "%s: token stride %lld of the pools", name, (long long)pages_st);
  if (num_splits > 1 && (int64_t)N * Hq * num_splits > 0x7fffffff)
    return set_error(SA_E_SHAPE, "%s: N=%d x Hq=%d x %d splits are too many partial rows", name, N, Hq, num_splits);
  const int64_t max_keys = std::min<int64_t>((int64_t)(selected ? std::min(max_blocks, sel_width) : max_blocks) * page, 1 << 30);
  const int64_t need = sa_paged_chunk_workspace_bytes(N, B, Hq, Hkv, D, (int)max_keys, num_splits);
  if (num_splits > 1 && need && (!workspace || workspace_bytes < need))
    return set_error(SA_E_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", name, (long long)workspace_bytes,
                     (long long)need);
  ChunkArgs a = {};
  a.q = static_cast<const elem_t*>(q);
  a.q_st = q_st, a.q_sh = q_sh;
  a.k = static_cast<const elem_t*>(k_pages);
  a.v = static_cast<const elem_t*>(v_pages);
  a.kv_sp = pages_sp, a.kv_sh = pages_sh, a.kv_st = pages_st;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.max_blocks = max_blocks, a.num_pages = num_pages, a.page = page;
  a.mul_page = div_mul((uint32_t)page);
  a.seqs = Ragged{cu_seqlens, kv_lens, B, N};
  a.sel = sel;
  a.sel_sr = sel_sr, a.sel_sh = sel_sh, a.sel_rows = sel_rows, a.sel_width = sel_width;
  a.sel_off = sel_off;
  a.off_sr = off_sr, a.off_sh = off_sh;
  a.mul_ppc = div_mul((uint32_t)(page / 16));
  a.o = static_cast<elem_t*>(o);
  a.o_st = o_st, a.o_sh = o_sh;
  a.Hq = Hq, a.Hkv = Hkv, a.G = Hq / Hkv;
  a.mul_G = div_mul((uint32_t)a.G);
  a.mul_heads = div_mul((uint32_t)Hkv);
  a.mul_Hq = div_mul((uint32_t)Hq);
  a.scale_log2 = sm_scale * 1.44269504088896340736f;
  a.tiles_per_block = (int)((CK_BLOCK * (int64_t)a.G + CK_WIDE_ROWS - 1) / CK_WIDE_ROWS);
  a.mul_tpb = div_mul((uint32_t)a.tiles_per_block);
  a.key_tiles = (int)((max_keys + CK_KT - 1) / CK_KT);
  a.cus = chunk_cus();
  // Without room for partials nothing is split.
  const int64_t room = std::min<int64_t>((workspace_bytes - chunk_part_header(B)) / ((int64_t)(D + 2) * 4), 0x7fffffff);
  a.splits = need && workspace && room > 0 ? num_splits : 1;
  if (a.splits != 1) {
    a.part = static_cast<SeqPart*>(workspace);
    a.part_rows = room;
    a.part_acc = reinterpret_cast<float*>(static_cast<char*>(workspace) + chunk_part_header(B));
    a.part_ml = a.part_acc + room * D;
  }
  // As many workgroups as any lengths need; those past the last item exit.
  const int64_t groups = chunk_items(N, B, a.G, Hkv, selected, a.splits) * Hkv;
  if (groups > MAX_WORKGROUPS / 2)
    return set_error(SA_E_SHAPE, "%s: %lld workgroups are too many for one launch", name, (long long)groups);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == SA_DTYPE_BF16) return D == 128 ? launch_chunk<true, 128>(a, groups, s) : launch_chunk<true, 64>(a, groups, s);
  return D == 128 ? launch_chunk<false, 128>(a, groups, s) : launch_chunk<false, 64>(a, groups, s);
}
