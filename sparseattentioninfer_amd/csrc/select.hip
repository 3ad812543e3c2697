// Pages of a paged cache that a cheap score picks for each query, gfx950.
//
// Every page keeps the minimum lo and the maximum hi of its keys in each dim (sa_paged_append).  The largest q . k
// that any key of the page can reach is sum_d max(q_d lo_d, q_d hi_d).  Summed over the queries that share a list (the
// heads of a KV group, of one token or of a block of 64) it is linear in the queries' positive and negative parts:
//
//   score(page) = hi . P + lo . N,   P = sum of max(q, 0),   N = sum of min(q, 0)
//
// with 0 times an infinite bound counted as 0, so a list costs 2 D multiply-adds a page however many queries share
// it.  Kept are the first `sink` pages, the last `recent` (from the page of the list's first query back, and all up to
// that of its last), and the top_k best of those between, ties to the lowest page.  Pages between are full and wholly
// visible to every query of the list.
//
// P, N and the scores are fp64: which page is the last one in depends on the order of near-equal scores, and in fp32
// that order would follow the order of summation.  It costs little: a page's 4 D bytes take 2 D fp64 multiply-adds.
//
// One workgroup makes a list: scores of all its pages as order-preserving 64-bit keys in LDS, the top_k-th key by
// radix selection (8 bits a pass, from the highest bit in which the keys differ), then the kept pages in ascending
// order by ballots.  All of it runs once or a few times, so its time is latency and instruction fetch: loops are kept
// rolled.  Few lists of many pages, and those of more pages than fit LDS, are scored by workgroups of their own first,
// into the workspace.
#include <algorithm>

#include "ragged.h"

namespace sa {

constexpr int SEL_BLOCK = 64;          // new tokens that share one list
constexpr int SEL_LDS_PAGES = 4096;    // keys of a list held in LDS
// Few lists of many pages leave most CUs idle, so their pages are scored by workgroups of their own first.  One token a
// sequence, D = 128, bf16, us in one workgroup a list against apart: 8 lists of 512 pages 17.2 / 10.7, of 4,096 70.6 / 22;
// 64 of 512 17.5 / 14.7, of 4,096 77.4 / 49.5; but 128 of 512 20.2 / 20.7, 256 of 1,024 31 / 42.  Of 256 pages, 12.7 / 10.1 for
// 8 lists, it is less than the host time of the second launch and the workspace (3.5).
constexpr int SEL_APART_LISTS = 64, SEL_APART_PAGES = 256;
// Pages of such a workgroup: as many as make SEL_SCORE_GROUPS of them within these limits.  Each sums the queries again,
// so more cost time (32 lists of 2,048 pages: 32 a workgroup 30 us, 64 23.7, 128 23.0; 512 lists of 4,096: 128 284, 4,096
// 355), and fewer leave CUs idle (8 lists of 512 pages: 64 a workgroup 11.7, 32 10.6).
constexpr int SEL_SCORE_GROUPS = 512, SEL_SCORE_MIN = 32, SEL_SCORE_MAX = 128;
// Threads of a workgroup that scores its own list: 1,024 up to one workgroup per CU, if its pages are many, else 512 (256
// lists of 1,024 pages: 31 us with 1,024, 34 with 512; of 128: 14.0, 10.9; 264 lists of 1,024: 55, 43).
constexpr int SEL_FEW_LISTS = 256, SEL_FEW_PAGES = 512;

struct SelectArgs {
  const elem_t* q;
  int64_t q_st, q_sh;
  const elem_t* bounds;                // [pages, Hkv, 2, D]
  int64_t bd_sp, bd_sh;
  const int32_t* table;
  int64_t table_stride;
  int max_blocks, num_pages, page;
  Ragged seqs;                         // cu == NULL: one token per sequence, row b
  int rows, Hkv, G;
  uint32_t mul_G;
  int top_k, sink, recent;
  int32_t* sel;
  int64_t sel_sr, sel_sh;
  int width;
  int32_t* off;                        // [rows, Hkv, 2]
  int score_pages;                     // pages scored by a workgroup of its own
  unsigned long long* keys;            // workspace [rows, Hkv, max_blocks], or NULL: a list's workgroup scores its pages
};

// The queries of one list and the pages it may keep.
struct SelectItem {
  int row, g, b;
  int64_t tok0;      // first query's packed row
  int n;             // queries (tokens)
  int pages;         // pages up to the last query's
  int head;          // pages [0, head) and [lo, pages) are kept; [head, lo) are ranked
  int lo;
};

__device__ __forceinline__ bool find_list(const SelectArgs& a, int id, SelectItem& it) {
  it.g = id % a.Hkv;
  it.row = id / a.Hkv;
  int first, last;
  if (!a.seqs.cu) {
    it.b = it.row;
    it.tok0 = it.row;
    it.n = 1;
    first = last = a.seqs.kv_len(it.b) - 1;
  } else {
    auto blocks = [&](int s) {
      int r0;
      return (a.seqs.rows(s, r0) + SEL_BLOCK - 1) / SEL_BLOCK;
    };
    int local;
    if (!find_item(a.seqs.B, it.row, blocks, it.b, local)) return false;
    int r0;
    const int n = a.seqs.rows(it.b, r0), start = a.seqs.kv_len(it.b) - n;
    it.tok0 = r0 + local * SEL_BLOCK;
    it.n = min(SEL_BLOCK, n - local * SEL_BLOCK);
    first = start + local * SEL_BLOCK;
    last = first + it.n - 1;
  }
  if (last < 0) return false;
  it.pages = min(last / a.page + 1, a.max_blocks);
  it.lo = min(max(0, max(first, 0) / a.page - a.recent + 1), it.pages);
  it.head = min(a.sink, it.lo);
  return true;
}

// Larger scores have larger keys; -0 and 0 share one, and a NaN ranks last.
__device__ __forceinline__ unsigned long long key_of(double s) {
  if (!(s == s)) return 0ull;
  const unsigned long long u = (unsigned long long)__double_as_longlong(s + 0.0);
  return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}

template <bool BF16, int D, int T>
struct Select {
  static constexpr int WAVES = T / 64;
  static constexpr int LPR = D / 8;     // lanes of one page's (or query's) row
  static constexpr int RPP = T / LPR;   // rows of a pass
  static constexpr int U = 4;           // rows of queries whose loads are in flight together
  static constexpr int POOL_ROWS = 256 / LPR;   // rows of lanes that sum the queries: a single token's heads are few
  struct Shared {
    double share[POOL_ROWS][2 * D];
    double pool[2 * D];   // P, N
    int hist[256];
    int sums[2][WAVES];
    unsigned long long hi[WAVES], lo[WAVES];
    unsigned long long cut;
    int need, ties;
  };

  static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = Elem<BF16>::to_f32((elem_t)(v[e] & 0xffffu));
      f[2 * e + 1] = Elem<BF16>::to_f32((elem_t)(v[e] >> 16));
    }
  }

  // P and N of the list's queries, into sh.pool.  Each row of lanes sums its share of the (query, head) rows; one
  // thread per dim then adds the shares.
  static __device__ __forceinline__ void pool(const SelectArgs& a, const SelectItem& it, Shared& sh) {
    const int c = threadIdx.x % LPR, r = threadIdx.x / LPR, rows = it.n * a.G;
    if (r < POOL_ROWS) {
      double p[8] = {}, n[8] = {};
      for (int x0 = r; x0 < rows; x0 += U * POOL_ROWS) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int x = x0 + u * POOL_ROWS;
          v[u] = u32x4{0u, 0u, 0u, 0u};
          if (x < rows) {
            const int t = (int)fast_div((uint32_t)x, (uint32_t)a.G, a.mul_G);
            v[u] = *reinterpret_cast<const u32x4*>(a.q + (it.tok0 + t) * a.q_st + (it.g * a.G + x - t * a.G) * a.q_sh + 8 * c);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float f[8];
          unpack(v[u], f);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            p[e] += f[e] < 0.f ? 0. : (double)f[e];   // a NaN too: its list's scores are NaN
            n[e] += f[e] < 0.f ? (double)f[e] : 0.;
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sh.share[r][8 * c + e] = p[e];
        sh.share[r][D + 8 * c + e] = n[e];
      }
    }
    __syncthreads();
    if (threadIdx.x < 2 * D) {
      double s = 0.;
#pragma unroll 4
      for (int x = 0; x < POOL_ROWS; ++x) s += sh.share[x][threadIdx.x];
      sh.pool[threadIdx.x] = s;
    }
    __syncthreads();
  }

  // Keys of pages [p0, p1) into keys[page].  The bounds of the pages after these are on their way meanwhile.
  static __device__ __forceinline__ void score(const SelectArgs& a, const SelectItem& it, const Shared& sh, int p0, int p1,
                                               unsigned long long* keys) {
    const int c = threadIdx.x % LPR, r = threadIdx.x / LPR;
    const int32_t* table = a.table + it.b * a.table_stride;
    const elem_t* bounds = a.bounds + it.g * a.bd_sh + 8 * c;
    double P[8], N[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      P[e] = sh.pool[8 * c + e];
      N[e] = sh.pool[D + 8 * c + e];
    }
    auto page_of = [&](int x) {
      const int pg = x < p1 ? table[x] : -1;
      return pg < a.num_pages ? pg : -1;
    };
    u32x4 lo = {0u, 0u, 0u, 0u}, hi = lo;
    auto load = [&](int pg) {
      if (pg >= 0) {
        lo = *reinterpret_cast<const u32x4*>(bounds + pg * a.bd_sp);
        hi = *reinterpret_cast<const u32x4*>(bounds + pg * a.bd_sp + D);
      }
    };
    int pg = page_of(p0 + r), pg1 = page_of(p0 + r + RPP);
    load(pg);
    for (int x = p0 + r; x < p1; x += RPP) {
      const u32x4 l4 = lo, h4 = hi;
      const bool live = pg >= 0;
      const int pg2 = page_of(x + 2 * RPP);
      load(pg1);
      float l[8], h[8];
      double s = 0.;
      unpack(l4, l);
      unpack(h4, h);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += (double)h[e] * P[e] + (double)l[e] * N[e];
      if (!(s == s)) {   // rare: a bound may be infinite, and a sign that no query has takes nothing of it
        s = 0.;
#pragma unroll
        for (int e = 0; e < 8; ++e) s += (P[e] != 0. ? (double)h[e] * P[e] : 0.) + (N[e] != 0. ? (double)l[e] * N[e] : 0.);
      }
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) s += __shfl_xor(s, o, 64);
      if (c == 0) keys[x] = live ? key_of(s) : 0ull;
      pg = pg1;
      pg1 = pg2;
    }
  }

  // Radix selection: sh.cut and sh.ties such that the best `need` of the keys [p0, p1) are those above cut and the
  // first `ties` equal to it.
  static __device__ __forceinline__ void find_cut(const unsigned long long* keys, int p0, int p1, int need, Shared& sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    unsigned long long hi = 0, lo = ~0ull;
    for (int x = p0 + tid; x < p1; x += T) {
      const unsigned long long k = keys[x];
      hi = k > hi ? k : hi;
      lo = k < lo ? k : lo;
    }
#pragma unroll 1
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned long long h = __shfl_xor(hi, o, 64), l = __shfl_xor(lo, o, 64);
      hi = h > hi ? h : hi;
      lo = l < lo ? l : lo;
    }
    if (lane == 0) {
      sh.hi[wave] = hi;
      sh.lo[wave] = lo;
    }
    if (tid < 256) sh.hist[tid] = 0;
    __syncthreads();
#pragma unroll 1
    for (int w = 0; w < WAVES; ++w) {
      hi = sh.hi[w] > hi ? sh.hi[w] : hi;
      lo = sh.lo[w] < lo ? sh.lo[w] : lo;
    }
    // `left` bits are undecided; the keys that may hold the cut are those whose bits above are `prefix`.
    int left = hi == lo ? 0 : 64 - __builtin_clzll(hi ^ lo);
    unsigned long long prefix = left == 64 ? 0ull : hi >> left;
    int count = p1 - p0;
    while (left > 0 && count != need) {
      const int bits = min(8, left), shift = left - bits;
      for (int x = p0 + tid; x < p1; x += T) {
        const unsigned long long k = keys[x];
        if (left == 64 || (k >> left) == prefix) atomicAdd(&sh.hist[(int)(k >> shift) & ((1 << bits) - 1)], 1);
      }
      __syncthreads();
      if (tid < 64) {   // lane l: digits 255 - 4 l down to 252 - 4 l
        int h[4], mine = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          mine += h[e] = sh.hist[255 - 4 * tid - e];
          sh.hist[255 - 4 * tid - e] = 0;
        }
        int above = scan_lanes(mine) - mine;
        if (above < need && above + mine >= need) {
          int e = 0;
          while (above + h[e] < need) above += h[e++];
          sh.cut = (prefix << bits) | (unsigned long long)(255 - 4 * tid - e);
          sh.need = need - above;
          sh.ties = h[e];
        }
      }
      __syncthreads();
      prefix = sh.cut;
      need = sh.need;
      count = sh.ties;
      left = shift;
    }
    __syncthreads();
    if (tid == 0) {
      // All `count` keys with the prefix are in (those above prefix << left, less one), or, all bits decided,
      // `need` of the equal ones.  A prefix of zeros with all of its keys in would mean that every key is.
      sh.cut = count == need ? (prefix << left) - 1ull : prefix;
      sh.ties = count == need ? 0 : need;
    }
    __syncthreads();
  }

  // Exclusive rank of this thread's flag among the workgroup's, and their number.
  static __device__ __forceinline__ int rank(bool flag, int (&sums)[WAVES], int& total) {
    const int wave = threadIdx.x >> 6;
    const uint64_t m = __builtin_amdgcn_ballot_w64(flag);
    if ((threadIdx.x & 63) == 0) sums[wave] = __popcll(m);
    __syncthreads();
    int before = __popcll(m & ((1ull << (threadIdx.x & 63)) - 1ull));
    total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) before += sums[w];
      total += sums[w];
    }
    return before;
  }

  // The kept pages in ascending order; `ranked`: [head, lo) holds more than top_k pages.
  static __device__ __forceinline__ void write_list(const SelectArgs& a, const SelectItem& it, bool ranked,
                                                    const unsigned long long* keys, Shared& sh) {
    int32_t* out = a.sel + it.row * a.sel_sr + it.g * a.sel_sh;
    int count = 0, tied = 0;
    for (int p0 = 0; p0 < it.pages; p0 += T) {
      const int p = p0 + threadIdx.x;
      bool keep = p < it.pages && (p < it.head || p >= it.lo);
      bool tie = false;
      if (p >= it.head && p < it.lo && a.top_k > 0) {
        if (!ranked) {
          keep = true;
        } else {
          keep = keys[p] > sh.cut;
          tie = keys[p] == sh.cut;
        }
      }
      int n;
      if (ranked) {
        const int r = rank(tie, sh.sums[0], n) + tied;
        keep |= tie && r < sh.ties;
        tied += n;
      }
      const int at = count + rank(keep, sh.sums[1], n);
      if (keep && at < a.width) out[at] = p;
      count += n;
      __syncthreads();
    }
    count = min(count, a.width);
    for (int x = count + threadIdx.x; x < a.width; x += T) out[x] = 0;
    if (threadIdx.x < 2) a.off[((int64_t)it.row * a.Hkv + it.g) * 2 + threadIdx.x] = threadIdx.x ? count : 0;
  }

  static __device__ void empty_list(const SelectArgs& a, const SelectItem& it) {
    int32_t* out = a.sel + it.row * a.sel_sr + it.g * a.sel_sh;
    for (int x = threadIdx.x; x < a.width; x += T) out[x] = 0;
    if (threadIdx.x < 2) a.off[((int64_t)it.row * a.Hkv + it.g) * 2 + threadIdx.x] = 0;
  }
};

// Scores of a.score_pages pages of a list, into the workspace.
template <bool BF16, int D>
__global__ __launch_bounds__(256) void select_score_kernel(const SelectArgs a) {
  using S = Select<BF16, D, 256>;
  __shared__ typename S::Shared sh;
  SelectItem it;
  if (!find_list(a, blockIdx.x, it) || it.lo - it.head <= a.top_k || a.top_k == 0) return;
  const int p0 = it.head + (int)blockIdx.y * a.score_pages, p1 = min(it.lo, p0 + a.score_pages);
  if (p0 >= p1) return;
  S::pool(a, it, sh);
  S::score(a, it, sh, p0, p1, a.keys + (int64_t)blockIdx.x * a.max_blocks);
}

// A list, of the workspace's scores or its own.  LDS: it has the keys there.
template <bool BF16, int D, int T, bool LDS>
__global__ __launch_bounds__(T) void select_kernel(const SelectArgs a) {
  using S = Select<BF16, D, T>;
  __shared__ typename S::Shared sh;
  extern __shared__ unsigned long long s_keys[];   // max_blocks
  SelectItem it;
  if (!find_list(a, blockIdx.x, it)) {
    S::empty_list(a, it);
    return;
  }
  const bool ranked = it.lo - it.head > a.top_k && a.top_k > 0;
  unsigned long long* keys = LDS ? s_keys : a.keys + (int64_t)blockIdx.x * a.max_blocks;
  if (ranked) {
    if constexpr (LDS) {
      if (a.keys) {
        const unsigned long long* from = a.keys + (int64_t)blockIdx.x * a.max_blocks;
        for (int x = it.head + threadIdx.x; x < it.lo; x += T) keys[x] = from[x];
      } else {
        S::pool(a, it, sh);
        S::score(a, it, sh, it.head, it.lo, keys);
      }
      __syncthreads();
    }
    S::find_cut(keys, it.head, it.lo, a.top_k, sh);
  }
  S::write_list(a, it, ranked, keys, sh);
}

template <bool BF16, int D>
static int launch_select(const SelectArgs& a, hipStream_t s) {
  const int64_t lists = (int64_t)a.rows * a.Hkv;
  const dim3 grid((unsigned)lists);
  const bool in_lds = a.max_blocks <= SEL_LDS_PAGES;
  const size_t lds = in_lds ? (size_t)a.max_blocks * 8 : 0;
  if (a.keys)
    hipLaunchKernelGGL((select_score_kernel<BF16, D>),
                       dim3((unsigned)lists, (a.max_blocks + a.score_pages - 1) / a.score_pages), dim3(256), 0, s, a);
  if (!in_lds)
    hipLaunchKernelGGL((select_kernel<BF16, D, 1024, false>), grid, dim3(1024), lds, s, a);
  else if (!a.keys && lists <= SEL_FEW_LISTS && a.max_blocks > SEL_FEW_PAGES)
    hipLaunchKernelGGL((select_kernel<BF16, D, 1024, true>), grid, dim3(1024), lds, s, a);
  else
    hipLaunchKernelGGL((select_kernel<BF16, D, 512, true>), grid, dim3(512), lds, s, a);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : set_error((int)err, "sa_paged_block_select: launch failed: %s", hipGetErrorString(err));
}

}  // namespace sa

using namespace sa;

extern "C" int64_t sa_paged_block_select_workspace_bytes(int rows, int Hkv, int max_blocks) {
  if (rows < 1 || Hkv < 1 || max_blocks < 1) return 0;
  const int64_t lists = (int64_t)rows * Hkv;
  const bool apart = max_blocks > SEL_LDS_PAGES || (lists <= SEL_APART_LISTS && max_blocks > SEL_APART_PAGES);
  return apart ? lists * max_blocks * 8 : 0;
}

extern "C" int sa_paged_block_select(int dtype, const void* q, int64_t q_st, int64_t q_sh, const void* k_bounds,
                                     int64_t bounds_sp, int64_t bounds_sh, int num_pages, const int32_t* block_table,
                                     int64_t block_table_stride, int max_blocks, const int32_t* cu_seqlens,
                                     const int32_t* kv_lens, int N, int B, int Hq, int Hkv, int D, int page, int top_k,
                                     int sink, int recent, int32_t* sel, int64_t sel_sr, int64_t sel_sh, int rows,
                                     int width, int32_t* sel_off, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
  clear_error();
  const char* name = "sa_paged_block_select";
  if (dtype != SA_DTYPE_BF16 && dtype != SA_DTYPE_F16)
    return set_error(SA_E_DTYPE, "%s: dtype %d is not bf16 (0) or f16 (1)", name, dtype);
  if (D != 64 && D != 128) return set_error(SA_E_HEADDIM, "%s: head dim %d not supported (64, 128)", name, D);
  if (page < 16 || page > 128 || page % 16)
    return set_error(SA_E_BLOCK, "%s: page %d is not a multiple of 16 in [16, 128]", name, page);
  if (N < 0 || B < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || Hq > (1 << 15) || max_blocks < 0 || num_pages < 0 ||
      block_table_stride < max_blocks || max_blocks > (1 << 21))
    return set_error(SA_E_SHAPE, "%s: bad sizes N=%d B=%d Hq=%d Hkv=%d, table of %d columns (stride %lld), %d pages", name,
                     N, B, Hq, Hkv, max_blocks, (long long)block_table_stride, num_pages);
  if (top_k < 0 || sink < 0 || recent < 1 || top_k > (1 << 22) || sink > (1 << 22) || recent > (1 << 22))
    return set_error(SA_E_SHAPE, "%s: top_k=%d, sink=%d (not negative), recent=%d (at least 1)", name, top_k, sink, recent);
  const int span = cu_seqlens ? (SEL_BLOCK + page - 2) / page + 1 : 1;   // pages that the queries of a list lie in
  const int64_t need_rows = cu_seqlens ? (int64_t)N / SEL_BLOCK + B : B;
  if (!cu_seqlens && N != B) return set_error(SA_E_SHAPE, "%s: one token per sequence, but N=%d for B=%d", name, N, B);
  if (rows != need_rows || width < sink + top_k + recent - 1 + span)
    return set_error(SA_E_SHAPE, "%s: lists [%d, Hkv, %d], needed [%lld, Hkv, %d]", name, rows, width, (long long)need_rows,
                     sink + top_k + recent - 1 + span);
  if (rows == 0) return 0;
  // A table without columns and bounds of no page are never read.
  if ((N && !q) || (num_pages && !k_bounds) || (max_blocks && !block_table) || !kv_lens || !sel || !sel_off) return set_error(SA_E_NULL, "%s: NULL pointer", name);
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_bounds) | reinterpret_cast<uintptr_t>(workspace)) & 15) ||
      (q_st | q_sh | bounds_sp | bounds_sh) % 8)
    return set_error(SA_E_ALIGN, "%s: rows must be 16-byte aligned", name);
  const int64_t need = sa_paged_block_select_workspace_bytes(rows, Hkv, max_blocks);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(SA_E_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", name, (long long)workspace_bytes,
                     (long long)need);
  if ((int64_t)rows * Hkv > MAX_WORKGROUPS / 4)   // of up to 1,024 threads
    return set_error(SA_E_SHAPE, "%s: %d rows of %d heads are too many", name, rows, Hkv);
  SelectArgs a = {};
  a.q = static_cast<const elem_t*>(q);
  a.q_st = q_st, a.q_sh = q_sh;
  a.bounds = static_cast<const elem_t*>(k_bounds);
  a.bd_sp = bounds_sp, a.bd_sh = bounds_sh;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.max_blocks = max_blocks, a.num_pages = num_pages, a.page = page;
  a.seqs = Ragged{cu_seqlens, kv_lens, B, N};
  a.rows = rows, a.Hkv = Hkv, a.G = Hq / Hkv;
  a.mul_G = div_mul((uint32_t)a.G);
  a.top_k = top_k, a.sink = sink, a.recent = recent;
  a.sel = sel;
  a.sel_sr = sel_sr, a.sel_sh = sel_sh, a.width = width;
  a.off = sel_off;
  a.keys = need ? static_cast<unsigned long long*>(workspace) : nullptr;
  const int64_t pages = (int64_t)rows * Hkv * max_blocks;
  a.score_pages = (int)std::min<int64_t>(std::max<int64_t>(pages / SEL_SCORE_GROUPS, SEL_SCORE_MIN), SEL_SCORE_MAX);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == SA_DTYPE_BF16) return D == 128 ? launch_select<true, 128>(a, s) : launch_select<true, 64>(a, s);
  return D == 128 ? launch_select<false, 128>(a, s) : launch_select<false, 64>(a, s);
}
