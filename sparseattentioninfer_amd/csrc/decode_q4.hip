// One new token per sequence over a paged cache held in 4 bits (gfx950): the whole cache, or the blocks that a list keeps
// for each (sequence, KV head) or (sequence, query head).
//
//   o = sum_j softmax_j(q . k_j * scale) v_j over the kept keys below kv_len; fp32 statistics and accumulators
//
// A workgroup has the query heads of one list (up to 8 at D = 128, 16 at 64) and `unit` steps of 32 keys of it, which its
// four waves take in turn; a longer list is shared by workgroups whose fp32 partials a second kernel merges.  The unit is
// the same for all lists, so the workgroups' loads are even whatever the lengths.  Over whole caches every workgroup works
// it out for itself and finds its list by a scan of the lengths: the launch is as large as any lengths need, and what is past
// the last list leaves at once.
//
// Up to 4 heads of a KV head at D = 128 are bound by HBM (64 sequences of 4,096 tokens, 8 KV heads, 335 MB: 67 to 72 us,
// 4.7 to 5.0 TB/s; over 16 bits 170), up to 8 by vector issue (81 to 83 us; fp16, with two products for p s, 89 to 91),
// few short lists by latency.
#include <algorithm>

#include "attn_q4.h"

namespace sa {

constexpr int DQ_WAVES = 4;
constexpr int DQ_DEPTH = 2;        // steps of a wave's ring
constexpr int DQ_TARGET = 512;     // workgroups that run at once, two to a CU
constexpr int DQ_MIN_UNIT = 8;     // steps of a workgroup of a planned division, two for each wave
constexpr int DQ_MOST = 1344;      // workgroups that a planned division adds to one for each list: DQ_TARGET / 0.381
constexpr float DQ_START = 8.f;    // what a workgroup costs besides its steps, in steps: 4 us of 0.5

struct DecodeQ4Args {
  const elem_t* q;
  int64_t q_sb, q_sh;
  const uint8_t *k, *v;
  int64_t sp, sh;
  const int32_t* table;
  int64_t table_stride;
  int max_blocks, num_pages, page;
  uint32_t mul_page, mul_ppc;
  const int32_t* kv_lens;
  const int32_t* sel;              // lists (sel_off NULL: every block)
  int64_t sel_sb, sel_sr;
  const int32_t* sel_off;
  int64_t off_sb, off_sr;
  int sel_width;
  int rows, heads, tiles;          // lists of a sequence; query heads of a list; workgroups that share those
  int group;                       // lists that read one KV head
  elem_t* o;
  int64_t o_sb, o_sh;
  int B, Hq;
  int unit;                        // steps of a workgroup; 0: planned
  int splits;                      // with lists: workgroups of each
  float* part;                     // NULL: no list is shared; else of workgroup x and its head r [x, r, D], ...
  float* part_ml;                  // ... and row reference and sum [x, r, 2]
  int* planned;                    // the planned unit, written by the launch's first workgroup for the merge
  float scale_log2;

  __device__ __forceinline__ int length(int b) const { return min(max(kv_lens[b], 0), MAX_KV_LEN); }
  // Steps of a whole cache of `len` tokens, as far as the table goes.
  __device__ __forceinline__ int steps(int len) const {
    return ((int)min((int64_t)len, (int64_t)max_blocks * page) + 31) / 32;
  }
};

// Which list a workgroup has, and which share of it.
struct DecodeQ4Item {
  int b, row, tile, len;
  int split, splits;
  int unit;
  int first;                       // workgroup of the list's and tile's first share

  // Workgroup x.  False if there is none.
  __device__ __forceinline__ bool find(const DecodeQ4Args& a, int x) {
    const int of_seq = a.rows * a.tiles;
    if (a.sel_off) {
      unit = a.unit;
      splits = a.splits;
      const int per = of_seq * splits;
      b = x / per;
      if (b >= a.B) return false;
      set(a, x - b * per, x);
      len = a.length(b);
      return true;
    }
    const int lane = threadIdx.x & 63;
    const int len64 = lane < a.B ? a.length(lane) : 0;
    plan(a, len64, of_seq);
    auto count = [&](int s) { return shares(a.steps(s < 64 ? len64 : a.length(s))) * of_seq; };
    int local;
    if (!find_item(a.B, x, count, b, local)) return false;
    len = a.length(b);
    splits = shares(a.steps(len));
    set(a, local, x);
    return true;
  }
  // The shares of list `row`'s tile `t` of sequence s (whole caches): splits and first.
  __device__ __forceinline__ void of_list(const DecodeQ4Args& a, int s, int r, int t) {
    const int of_seq = a.rows * a.tiles;
    b = s, row = r, tile = t;
    if (a.sel_off) {
      splits = a.splits;
      first = ((s * a.rows + r) * a.tiles + t) * splits;
      return;
    }
    const int lane = threadIdx.x & 63;
    const int len64 = lane < a.B ? a.length(lane) : 0;
    unit = a.unit ? a.unit : *a.planned;
    first = 0;
    for (int b0 = 0; b0 <= s; b0 += 64) {
      const int l = b0 ? (b0 + lane < a.B ? a.length(b0 + lane) : 0) : len64;
      const int k = b0 + lane < a.B ? shares(a.steps(l)) : 0, incl = scan_lanes(k);
      if (s < b0 + 64) {
        splits = __builtin_amdgcn_readlane(k, s - b0);
        first += __builtin_amdgcn_readlane(incl, s - b0) - splits;
      } else {
        first += __builtin_amdgcn_readlane(incl, 63);
      }
    }
    first = first * of_seq + (r * a.tiles + t) * splits;
  }

 private:
  __device__ __forceinline__ int shares(int steps) const { return max(1, (steps + unit - 1) / unit); }
  __device__ __forceinline__ void set(const DecodeQ4Args& a, int local, int x) {
    split = local % splits;
    const int l = local / splits;
    tile = l % a.tiles;
    row = l / a.tiles;
    first = x - split;
  }
  // The unit of a planned division: of no division, an even share of all steps and 0.76, 0.5 and 0.381 of it the one that
  // ends first.  While the shares run at once that is when the longest ends; else the mean load and half the longest.
  // (Equal lists are best left whole or cut evenly, uneven ones finely.  Replayed, whole / even / 0.76 / 0.5 / 0.381 of it / as
  // planned: 28 sequences of 64 to 30,000 tokens, 40 heads, 319 / 131 / 117 / 114 / 111 / 114 us; 48 of 500 to 16,010, 32
  // heads, 162 / 129 / 125 / 122 / 116 / 117; 64 of 4,096 71 / 71 / 92 / 76 / 80 / 72; one of 32,001 275 / 18.8 / 20.2 / 22.3 /
  // 22.2 / 19.9.)  Sums are fp32; the margin above their rounding keeps the shares within DQ_MOST, and a unit of no division
  // is one step more where fp32 may have rounded the longest list down (past 2^24 steps, of at most 2^25).
  __device__ __forceinline__ void plan(const DecodeQ4Args& a, int len64, int of_seq) {
    unit = a.unit;
    if (unit) return;
    const int lane = threadIdx.x & 63;
    const float of = (float)of_seq;
    const int n64 = a.steps(len64);
    float sum = (float)n64, longest = (float)n64;
    for (int s = 64 + lane; s < a.B; s += 64) {
      const float n = (float)a.steps(a.length(s));
      sum += n;
      longest = fmaxf(longest, n);
    }
    sum = wave_sum(sum) * of;
    longest = wave_max(longest);
    const float even = sum * (1.001f / DQ_TARGET);
    int u[5];
    float rcp[5], groups[5], share[5];
    // Shares as shares() counts them, up to 2^20 steps (past that a rest of a step may go uncounted).  The reciprocal is off by
    // a step for some units (of 1,535, times 1,535 it passes 1): with 2^-21 less than it the product stays below a whole
    // number that it should be (2^-23 and three roundings of 2^-24), and above one that n passes by a step.
    auto weigh = [&](int c, float n) {
      const float k = fmaxf(1.f, ceilf(n * rcp[c]));
      groups[c] += n > 0.f ? k : 0.f;
      share[c] = fmaxf(share[c], n * __builtin_amdgcn_rcpf(k));
    };
#pragma unroll
    for (int c = 0; c < 5; ++c) {
      const float f = c == 1 ? 1.f : c == 2 ? 0.76f : c == 3 ? 0.5f : 0.381f;
      u[c] = c ? max(DQ_MIN_UNIT, (int)fminf(ceilf(even * f), 33554432.f))
             : max(1, (int)longest + (longest >= 16777216.f ? 1 : 0));
      rcp[c] = __builtin_amdgcn_rcpf((float)u[c]) * 0.9999995231628418f;
      groups[c] = share[c] = 0.f;
      weigh(c, (float)n64);
    }
    for (int s = 64 + lane; s < a.B; s += 64) {
      const float n = (float)a.steps(a.length(s));
#pragma unroll
      for (int c = 0; c < 5; ++c) weigh(c, n);
    }
    float best = __builtin_inff();
#pragma unroll
    for (int c = 0; c < 5; ++c) {
      const float g = wave_sum(groups[c]) * of, h = wave_max(share[c]) + DQ_START;
      const float time = g <= DQ_TARGET ? h : (sum + g * DQ_START) * (1.f / DQ_TARGET) + 0.5f * h;
      unit = time < best ? u[c] : unit;
      best = fminf(time, best);
    }
    unit = __builtin_amdgcn_readfirstlane(unit);
  }
};

template <bool BF16, int D, int NQ>
struct DecodeQ4 {
  using E = Elem<BF16>;
  using Rows = Q4Fold<BF16, D, NQ, DQ_DEPTH>;
  static constexpr int ROWS = Rows::ROWS;
  static constexpr int ACC = ROWS * D * 4;
  static constexpr int LDS_BYTES = DQ_WAVES * (ACC > Q4Ring<D, DQ_DEPTH>::BYTES ? ACC : Q4Ring<D, DQ_DEPTH>::BYTES);

  static __device__ void run(const DecodeQ4Args& a, char* s_lds, float* s_ml) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    DecodeQ4Item it;
    if (!it.find(a, blockIdx.x)) return;
    if (a.planned && blockIdx.x == 0 && threadIdx.x == 0) *a.planned = it.unit;
    const int b = it.b, row = it.row, len = it.len;
    // Chunks of 16 keys of the list.
    const int last = (int)min((int64_t)len, (int64_t)a.max_blocks * a.page);
    int chunks = (last + 15) / 16;
    const int32_t* list = nullptr;
    if (a.sel_off) {
      const int32_t* off = a.sel_off + b * a.off_sb + row * a.off_sr;
      const int e0 = min(max(off[0], 0), a.sel_width), e1 = min(max(off[1], e0), a.sel_width);
      list = a.sel + b * a.sel_sb + row * a.sel_sr + e0;
      chunks = last > 0 ? (e1 - e0) * (a.page / 16) : 0;
    }
    const int head0 = row * a.heads + it.tile * ROWS, live = min(ROWS, a.heads - it.tile * ROWS);
    Rows w;
#pragma unroll
    for (int x = 0; x < NQ; ++x)
      w.set_query(x, a.q + b * a.q_sb + (head0 + min(x * Rows::RPS + Rows::row_of(lane), live - 1)) * a.q_sh, len - 1);
    w.pos_min = len - 1;
    w.start();
    w.ring.lds = s_lds + wave * Q4Ring<D, DQ_DEPTH>::BYTES;
    Q4Keys ks;
    const int kvh = row / a.group;
    ks.k = a.k + kvh * a.sh;
    ks.v = a.v + kvh * a.sh;
    ks.sp = a.sp;
    ks.table = a.table + b * a.table_stride;
    ks.list = list;
    ks.max_blocks = a.max_blocks, ks.num_pages = a.num_pages, ks.page = a.page;
    ks.mul_page = a.mul_page, ks.mul_ppc = a.mul_ppc;
    ks.c0 = min(chunks, 2 * it.unit * it.split);
    ks.c1 = min(chunks, ks.c0 + 2 * it.unit);
    ks.end = len, ks.pos_max = len - 1;
    ks.wave = wave, ks.waves = DQ_WAVES;
    q4_run(w, ks, a.scale_log2);
    __syncthreads();               // the rings lie where the accumulators go
    // Merge in fp32: row r is D floats at r * 4 D, its 16-byte chunk x at position x ^ (r % (D / 4)).
    constexpr int NC4 = D / 4, OC = D / 8;
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      const int r = x * Rows::RPS + Rows::row_of(lane), g = Rows::group_of(lane);
      f32x4 out[2];
      w.result(x, out);
#pragma unroll
      for (int half = 0; half < 2; ++half)
        *reinterpret_cast<f32x4*>(s_lds + wave * ACC + r * 4 * D + 16 * ((8 * g + 4 * half + (lane >> 4)) ^ (r & (NC4 - 1)))) = out[half];
      const float l = quarters_sum(w.l_run[x]);
      if (lane < Rows::RPS) {
        s_ml[2 * (wave * ROWS + r)] = w.m_ref[x];
        s_ml[2 * (wave * ROWS + r) + 1] = l;
      }
    }
    __syncthreads();
    for (int y = threadIdx.x; y < live * OC; y += 64 * DQ_WAVES) {
      const int r = y / OC, oc = y % OC;
      float m[DQ_WAVES], l = 0.f, M = -__builtin_inff();
#pragma unroll
      for (int s = 0; s < DQ_WAVES; ++s) {
        m[s] = s_ml[2 * (s * ROWS + r)];
        M = fmaxf(M, m[s]);
      }
      const float Mu = M == -__builtin_inff() ? 0.f : M;
      f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll
      for (int s = 0; s < DQ_WAVES; ++s) {
        const float fs = fast_exp2(m[s] - Mu);
        l += fs * s_ml[2 * (s * ROWS + r) + 1];
        const char* p = s_lds + s * ACC + r * 4 * D;
        lo += fs * *reinterpret_cast<const f32x4*>(p + 16 * ((2 * oc) ^ (r & (NC4 - 1))));
        hi += fs * *reinterpret_cast<const f32x4*>(p + 16 * ((2 * oc + 1) ^ (r & (NC4 - 1))));
      }
      const int h = head0 + r;
      if (it.splits > 1) {
        const int64_t at = (int64_t)blockIdx.x * ROWS + r;
        f32x4* d = reinterpret_cast<f32x4*>(a.part + at * D + 8 * oc);
        d[0] = lo;
        d[1] = hi;
        if (oc == 0) {
          a.part_ml[2 * at] = M;
          a.part_ml[2 * at + 1] = l;
        }
      } else {
        const float inv = l > 0.f ? 1.f / l : 1.f;
        *reinterpret_cast<u32x4*>(a.o + b * a.o_sb + h * a.o_sh + 8 * oc) =
            u32x4{E::pack2f(lo[0] * inv, lo[1] * inv), E::pack2f(lo[2] * inv, lo[3] * inv),
                  E::pack2f(hi[0] * inv, hi[1] * inv), E::pack2f(hi[2] * inv, hi[3] * inv)};
      }
    }
  }
};

template <bool BF16, int D, int NQ>
static __global__ __launch_bounds__(64 * DQ_WAVES, 2) void decode_q4_kernel(const DecodeQ4Args a) {
  using K = DecodeQ4<BF16, D, NQ>;
  __shared__ __attribute__((aligned(16))) char s_lds[K::LDS_BYTES];
  __shared__ float s_ml[2 * DQ_WAVES * K::ROWS];
  K::run(a, s_lds, s_ml);
}

// Merges the partials of a query head whose list was shared: a workgroup a head, D / 8 lanes a share, 2048 / D shares at a
// time.
template <bool BF16, int D>
static __global__ __launch_bounds__(256) void decode_q4_combine_kernel(const DecodeQ4Args a, int per_tile) {
  using E = Elem<BF16>;
  constexpr int LPR = D / 8, SH = 256 / LPR;
  __shared__ __attribute__((aligned(16))) float s_acc[4][D + 4];
  const int x = blockIdx.x, b = x / a.Hq, h = x - b * a.Hq;
  const int oc = threadIdx.x % LPR, sh = threadIdx.x / LPR, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  DecodeQ4Item it;
  const int row = h / a.heads, r = h - row * a.heads;
  it.of_list(a, b, row, r / per_tile);
  if (it.splits <= 1) return;
  const int64_t at = (int64_t)it.first * per_tile + r % per_tile;
  float M = -__builtin_inff(), L = 0.f;
  f32x4 acc[2] = {f32x4{}, f32x4{}};
  for (int s = sh; s < it.splits; s += SH) {
    const int64_t p = at + (int64_t)s * per_tile;
    const float m = a.part_ml[2 * p], l = a.part_ml[2 * p + 1];
    const f32x4* v = reinterpret_cast<const f32x4*>(a.part + p * D + 8 * oc);
    const f32x4 v0 = v[0], v1 = v[1];
    // As in chunk_items.h: a share of NaN scores has sums of NaN, which reach the row.
    const float Mc = fmaxf(M, m), Mu = Mc == -__builtin_inff() ? 0.f : Mc;
    const float f0 = fast_exp2(M - Mu), f1 = fast_exp2(m - Mu);
    L = L * f0 + l * f1;
    acc[0] = acc[0] * f0 + v0 * f1;
    acc[1] = acc[1] * f0 + v1 * f1;
    M = Mc;
  }
  // Over the shares of a wave, then of the four waves, in a fixed order.
#pragma unroll
  for (int o = LPR; o < 64; o <<= 1) {
    const float m = __shfl_xor(M, o, 64), l = __shfl_xor(L, o, 64);
    const float Mc = fmaxf(M, m), Mu = Mc == -__builtin_inff() ? 0.f : Mc;
    const float f0 = fast_exp2(M - Mu), f1 = fast_exp2(m - Mu);
    L = L * f0 + l * f1;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[k][e] = acc[k][e] * f0 + __shfl_xor(acc[k][e], o, 64) * f1;
    M = Mc;
  }
  if (lane < LPR) {
    f32x4* d = reinterpret_cast<f32x4*>(&s_acc[wave][8 * oc]);
    d[0] = acc[0];
    d[1] = acc[1];
    if (lane == 0) s_acc[wave][D] = M, s_acc[wave][D + 1] = L;
  }
  __syncthreads();
  if (threadIdx.x >= LPR) return;
  M = fmaxf(fmaxf(s_acc[0][D], s_acc[1][D]), fmaxf(s_acc[2][D], s_acc[3][D]));
  const float Mu = M == -__builtin_inff() ? 0.f : M;
  L = 0.f;
  acc[0] = acc[1] = f32x4{};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = fast_exp2(s_acc[w][D] - Mu);
    const f32x4* d = reinterpret_cast<const f32x4*>(&s_acc[w][8 * oc]);
    L += f * s_acc[w][D + 1];
    acc[0] += f * d[0];
    acc[1] += f * d[1];
  }
  const float inv = L > 0.f ? 1.f / L : 1.f;
  *reinterpret_cast<u32x4*>(a.o + b * a.o_sb + h * a.o_sh + 8 * oc) =
      u32x4{E::pack2f(acc[0][0] * inv, acc[0][1] * inv), E::pack2f(acc[0][2] * inv, acc[0][3] * inv),
            E::pack2f(acc[1][0] * inv, acc[1][1] * inv), E::pack2f(acc[1][2] * inv, acc[1][3] * inv)};
}

template <bool BF16, int D>
static int launch_decode_q4(const DecodeQ4Args& a, int64_t groups, int sets, hipStream_t s) {
  if (sets == 1)
    hipLaunchKernelGGL((decode_q4_kernel<BF16, D, 1>), dim3((unsigned)groups), dim3(64 * DQ_WAVES), 0, s, a);
  else
    hipLaunchKernelGGL((decode_q4_kernel<BF16, D, 2>), dim3((unsigned)groups), dim3(64 * DQ_WAVES), 0, s, a);
  if (a.part)
    hipLaunchKernelGGL((decode_q4_combine_kernel<BF16, D>), dim3((unsigned)(a.B * a.Hq)), dim3(256), 0, s, a, sets * 16 / (D / 32));
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : set_error((int)err, "sa_decode_q4: launch failed: %s", hipGetErrorString(err));
}

// Sizes of a launch.
struct DecodeQ4Plan {
  int sets, tiles;                 // column sets of a workgroup; workgroups that share the query heads of a list
  int unit, splits;                // as in DecodeQ4Args; splits 1: nothing is shared
  int64_t groups, bytes;           // workgroups; bytes of the planned unit and the partials
  static constexpr int HEADER = 64;

  DecodeQ4Plan(int B, int Hq, int rows, int D, int64_t keys, bool lists, int num_splits) {
    const int per_set = 16 / (D / 32), heads = Hq / rows;
    sets = heads > per_set ? 2 : 1;
    tiles = (heads + sets * per_set - 1) / (sets * per_set);
    const int64_t of = (int64_t)B * rows * tiles;
    const int64_t steps = std::max<int64_t>(1, (std::min<int64_t>(keys, MAX_KV_LEN) + 31) / 32);
    unit = (int)steps;
    groups = of;
    // Sharing up to 16 steps costs more than it saves: the merge is 3 us, and four waves have 4 steps each.  (16 lists of 16
    // steps, D = 64: 6.9 us in one, 7.7 in two; 8 of 32, D = 128: 11.6 in one, 8.5 in 4.)
    if (num_splits == 0 && steps > 16) {
      if (lists) {
        // Their lengths are taken to be about those of the longest.
        num_splits = (int)std::max<int64_t>(1, std::min<int64_t>({64, DQ_TARGET / of, steps / DQ_MIN_UNIT}));
      } else {
        unit = 0;
        groups = std::min(of + DQ_MOST, of * ((steps + DQ_MIN_UNIT - 1) / DQ_MIN_UNIT));
      }
    }
    if (num_splits > 1) {
      unit = (int)((steps + num_splits - 1) / num_splits);
      groups = of * ((steps + unit - 1) / unit);
    }
    splits = unit ? (int)((steps + unit - 1) / unit) : 2;
    bytes = splits > 1 ? HEADER + groups * sets * per_set * (D + 2) * 4 : 0;
  }
};

}  // namespace sa

using namespace sa;

extern "C" int64_t sa_decode_q4_workspace_bytes(int B, int Hq, int rows, int D, int max_keys, int selected, int num_splits) {
  if (B < 1 || Hq < 1 || rows < 1 || Hq % rows || (D != 64 && D != 128) || num_splits < 0) return 0;
  return DecodeQ4Plan(B, Hq, rows, D, max_keys, selected != 0, num_splits).bytes;
}

extern "C" int sa_decode_q4(int dtype, const void* q, int64_t q_sb, int64_t q_sh, const void* k_pages, const void* v_pages,
                            int64_t pages_sp, int64_t pages_sh, int num_pages, const int32_t* block_table,
                            int64_t block_table_stride, int max_blocks, const int32_t* kv_lens, const int32_t* sel,
                            int64_t sel_sb, int64_t sel_sr, int sel_width, const int32_t* sel_off, int64_t off_sb,
                            int64_t off_sr, int sel_rows, void* o, int64_t o_sb, int64_t o_sh, int B, int Hq, int Hkv, int D,
                            int page, float sm_scale, int num_splits, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  clear_error();
  const char* name = "sa_decode_q4";
  if (dtype != SA_DTYPE_BF16 && dtype != SA_DTYPE_F16)
    return set_error(SA_E_DTYPE, "%s: dtype %d is not bf16 (0) or f16 (1)", name, dtype);
  if (D != 64 && D != 128) return set_error(SA_E_HEADDIM, "%s: head dim %d not supported (64, 128)", name, D);
  if (page < 16 || page > 128 || page % 16)
    return set_error(SA_E_BLOCK, "%s: page %d is not a multiple of 16 in [16, 128]", name, page);
  if (B < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || Hq > (1 << 15) || max_blocks < 0 || num_pages < 0 ||
      block_table_stride < max_blocks || num_splits < 0 || num_splits > 64)
    return set_error(SA_E_SHAPE, "%s: bad sizes B=%d Hq=%d Hkv=%d, table of %d columns (stride %lld), %d pages, "
                     "%d splits (0..64)", name, B, Hq, Hkv, max_blocks, (long long)block_table_stride, num_pages, num_splits);
  if (!(sm_scale >= 1e-30f && sm_scale <= 1e30f))
    return set_error(SA_E_SHAPE, "%s: scale %g is not in [1e-30, 1e30]", name, sm_scale);
  if (sel_off && sel_rows != Hq && sel_rows != Hkv)
    return set_error(SA_E_CSR, "%s: sel_rows=%d is not Hq=%d or Hkv=%d", name, sel_rows, Hq, Hkv);
  if (sel_off ? sel_width < 0 || (int64_t)sel_width * (page / 16) > (1 << 26) : sel != nullptr)
    return set_error(SA_E_SHAPE, "%s: a selection needs offsets and a width that is not negative or past 2^26 chunks of 16 keys, "
                     "got %d", name, sel_width);
  if (B == 0) return 0;
  // A table without columns and pools without pages are never read.
  if (!q || (num_pages && (!k_pages || !v_pages)) || (max_blocks && !block_table) || !kv_lens || !o || (sel_off && sel_width && !sel))
    return set_error(SA_E_NULL, "%s: NULL pointer", name);
  if (bad_ptr(q) || bad_ptr(k_pages) || bad_ptr(v_pages) || bad_ptr(o) || bad_ptr(workspace) || (q_sb | q_sh | o_sb | o_sh) % 8 ||
      (pages_sp | pages_sh) % 16)
    return set_error(SA_E_ALIGN, "%s: head rows and blocks must be 16-byte aligned", name);
  DecodeQ4Args a = {};
  a.max_blocks = num_pages ? max_blocks : 0;      // without pages no key is there, and none is loaded
  a.rows = sel_off ? sel_rows : Hkv;
  const int64_t keys = std::min<int64_t>((int64_t)(sel_off ? sel_width : max_blocks) * page, MAX_KV_LEN);
  const DecodeQ4Plan plan(B, Hq, a.rows, D, keys, sel_off != nullptr, num_splits);
  if (plan.bytes && (!workspace || workspace_bytes < plan.bytes))
    return set_error(SA_E_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", name, (long long)workspace_bytes,
                     (long long)plan.bytes);
  a.q = static_cast<const elem_t*>(q);
  a.q_sb = q_sb, a.q_sh = q_sh;
  a.k = static_cast<const uint8_t*>(k_pages);
  a.v = static_cast<const uint8_t*>(v_pages);
  a.sp = pages_sp, a.sh = pages_sh;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.num_pages = num_pages, a.page = page;
  a.mul_page = div_mul((uint32_t)page);
  a.mul_ppc = div_mul((uint32_t)(page / 16));
  a.kv_lens = kv_lens;
  a.sel = sel;
  a.sel_sb = sel_sb, a.sel_sr = sel_sr, a.sel_width = sel_width;
  a.sel_off = sel_off;
  a.off_sb = off_sb, a.off_sr = off_sr;
  a.heads = Hq / a.rows;
  a.group = a.rows / Hkv;
  a.tiles = plan.tiles;
  a.unit = plan.unit, a.splits = plan.splits;
  a.o = static_cast<elem_t*>(o);
  a.o_sb = o_sb, a.o_sh = o_sh;
  a.B = B, a.Hq = Hq;
  const int per_tile = plan.sets * 16 / (D / 32);
  if (plan.bytes) {
    a.planned = plan.unit ? nullptr : static_cast<int*>(workspace);
    a.part = static_cast<float*>(workspace) + DecodeQ4Plan::HEADER / 4;
    a.part_ml = a.part + plan.groups * per_tile * D;
  }
  a.scale_log2 = sm_scale * 1.44269504088896340736f;
  const int64_t groups = plan.groups;
  const int sets = plan.sets;
  if (groups > MAX_WORKGROUPS || (int64_t)B * Hq > MAX_WORKGROUPS)
    return set_error(SA_E_SHAPE, "%s: %lld workgroups are too many for one launch", name, (long long)groups);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == SA_DTYPE_BF16)
    return D == 128 ? launch_decode_q4<true, 128>(a, groups, sets, s) : launch_decode_q4<true, 64>(a, groups, sets, s);
  return D == 128 ? launch_decode_q4<false, 128>(a, groups, sets, s) : launch_decode_q4<false, 64>(a, groups, sets, s);
}
