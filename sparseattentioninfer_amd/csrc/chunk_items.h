// Division of a ragged batch's rows and keys over the workgroups of a chunk attention launch, the merge of the partial
// results where keys are divided, and the launch's sizes: the same for caches of every form.
#pragma once

#include <algorithm>

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
// the waves of a workgroup divide (four over 16 bits, eight over 4); others by wide items, 256 rows that share every key tile.  Where there are fewer items than
// CUs, or one sequence is much longer than the rest, each item's keys are divided over `splits` workgroups.  The
// lengths are device memory, so the launch is as large as any lengths need and every workgroup works out the
// division for itself, the same in all of them: `limit` key tiles to a workgroup, from the total.
//
// Key tiles are what is balanced.  With the chip full a wide item takes 1.75 us for one (256 rows on its matrix
// cores), a narrow one 1.45 us where narrow items are most of the work (32 KB at a CU's share of HBM) and about half of
// a wide one's beside wide ones.  A workgroup costs `start` of them (5.5) besides its own: 9.6 us, of which finding its item
// takes 2.5, the pages of its first tiles 2.6, the tiles 1.5 and the end 3.
// A division costs the merge, 4 us after narrow and 6.5 after wide items, and for each row of partials its write and
// read: 1,040 bytes at D = 128, 0.2 ns at the rate of a copy.
struct ChunkCost {
  static constexpr float MERGE_WIDE = 4.f, MERGE_NARROW = 2.5f, MERGE_ROW = 1.3e-4f;
  static __device__ __forceinline__ float start(int) { return 5.5f; }
  // Narrow items that do not fill the chip are not bound by HBM: 0.5 us for a tile instead of 1.45.
  static __device__ __forceinline__ float alone(float groups, float cus) { return fminf(fmaxf(0.35f, groups / cus), 1.f); }
};
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
template <class Cost>
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
  const float start = Cost::start(half);
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
  const float mean = (work + groups * start) / cus;
  const float alone = half ? 1.f : Cost::alone(groups, cus);
  float one = 0.f, many = 0.f, lo = __builtin_inff(), hi = 0.f;
  each([&](float st, float k, float nt, float nt0, float, float w) {
    if (st == 0.f) return;
    const float x = w * alone * __builtin_amdgcn_rcpf(k), h = nt * x + start, l = nt0 * x + start;
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
  if (rows > 0.f) time += (half ? Cost::MERGE_WIDE : Cost::MERGE_NARROW) + Cost::MERGE_ROW * rows;
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
template <class Cost = ChunkCost>
__device__ __forceinline__ bool find_chunk_item(const ChunkArgs& a, int id, ChunkItem& it) {
  const int lane = threadIdx.x & 63;
  const int t = (int)fast_div((uint32_t)id, (uint32_t)a.Hkv, a.mul_heads);
  it.kvh = id - t * a.Hkv;
  SeqShape s64 = {};
  if (lane < a.seqs.B) s64 = seq_shape(a, lane);
  const bool split = a.part != nullptr;
  const SplitRule rule = split ? plan_splits<Cost>(a, s64) : SplitRule(CK_NO_LIMIT, 0);
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

// Merges the partials of the rows (token, head), D / 8 lanes a row, after the workgroups of the launch before have left
// them; rows of sequences that were not split are done.  Each lane of a wave holds one sequence's range of
// rows and place, so a row finds its own without a chain of reads.
template <bool BF16, int D>
static __global__ __launch_bounds__(256) void chunk_combine_kernel(const ChunkArgs a) {
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
