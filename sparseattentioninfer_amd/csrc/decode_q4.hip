// One new token per sequence over a paged cache held in 4 bits (gfx950): the whole cache, or the blocks that a list keeps
// for each (sequence, KV head) or (sequence, query head).
//
//   o = sum_j softmax_j(q . k_j * scale) v_j over the kept keys below kv_len; fp32 statistics and accumulators
//
// A workgroup has the query heads of one list (up to 8 at D = 128, 16 at 64) and `unit` steps of 32 keys of it, which its four waves take in
// turn; a longer list is shared by workgroups whose fp32 partials a second kernel merges.  The unit is the same for every
// sequence, so the workgroups' loads are even whatever the lengths, and those past a sequence's end leave at once.
#include <algorithm>

#include "attn_q4.h"

namespace sa {

constexpr int DQ_WAVES = 4;

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
  int unit, splits;                // steps of a workgroup; most workgroups of a list
  float* part;                     // [splits, B, Hq, D], then [splits, B, Hq, 2] (splits > 1)
  float scale_log2;

  // Chunks of 16 keys of list `row` of sequence b.
  __device__ __forceinline__ int chunks(int b, int row, const int32_t*& list, int& len) const {
    len = min(max(kv_lens[b], 0), MAX_KV_LEN);
    const int last = (int)min((int64_t)len, (int64_t)max_blocks * page);
    list = nullptr;
    if (!sel_off) return (last + 15) / 16;
    const int32_t* off = sel_off + b * off_sb + row * off_sr;
    const int e0 = min(max(off[0], 0), sel_width), e1 = min(max(off[1], e0), sel_width);
    list = sel + b * sel_sb + row * sel_sr + e0;
    return last > 0 ? (e1 - e0) * (page / 16) : 0;
  }
  // Workgroups that share `chunks` chunks.
  __device__ __forceinline__ int splits_of(int chunks) const {
    return max(1, ((chunks + 1) / 2 + unit - 1) / unit);
  }
};

template <bool BF16, int D, int NQ>
struct DecodeQ4 {
  using E = Elem<BF16>;
  using Rows = Q4Fold<BF16, D, NQ>;
  static constexpr int ROWS = Rows::ROWS;
  static constexpr int ACC = ROWS * D * 4;

  static __device__ void run(const DecodeQ4Args& a, char* s_acc, float* s_ml) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int x = blockIdx.x;
    const int tile = x % a.tiles;
    x /= a.tiles;
    const int row = x % a.rows;
    x /= a.rows;
    const int b = x % a.B, split = x / a.B;
    int len;
    const int32_t* list;
    const int chunks = a.chunks(b, row, list, len);
    const int n = a.splits_of(chunks);
    if (split >= n) return;
    const int head0 = row * a.heads + tile * ROWS, live = min(ROWS, a.heads - tile * ROWS);
    Rows w;
#pragma unroll
    for (int x = 0; x < NQ; ++x)
      w.set_query(x, a.q + b * a.q_sb + (head0 + min(x * Rows::RPS + Rows::row_of(lane), live - 1)) * a.q_sh, len - 1);
    w.pos_min = len - 1;
    w.start();
    Q4Keys ks;
    const int kvh = row / a.group;
    ks.k = a.k + kvh * a.sh;
    ks.v = a.v + kvh * a.sh;
    ks.sp = a.sp;
    ks.table = a.table + b * a.table_stride;
    ks.list = list;
    ks.max_blocks = a.max_blocks, ks.num_pages = a.num_pages, ks.page = a.page;
    ks.mul_page = a.mul_page, ks.mul_ppc = a.mul_ppc;
    ks.c0 = 2 * a.unit * split;
    ks.c1 = min(chunks, ks.c0 + 2 * a.unit);
    ks.end = len, ks.pos_max = len - 1;
    ks.wave = wave, ks.waves = DQ_WAVES;
    q4_run(w, ks, a.scale_log2);
    // Merge in fp32: row r is D floats at r * 4 D, its 16-byte chunk x at position x ^ (r % (D / 4)).
    constexpr int NC4 = D / 4, OC = D / 8;
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      const int r = x * Rows::RPS + Rows::row_of(lane), g = Rows::group_of(lane);
      f32x4 out[2];
      w.result(x, out);
#pragma unroll
      for (int half = 0; half < 2; ++half)
        *reinterpret_cast<f32x4*>(s_acc + wave * ACC + r * 4 * D + 16 * ((8 * g + 4 * half + (lane >> 4)) ^ (r & (NC4 - 1)))) = out[half];
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
        const char* p = s_acc + s * ACC + r * 4 * D;
        lo += fs * *reinterpret_cast<const f32x4*>(p + 16 * ((2 * oc) ^ (r & (NC4 - 1))));
        hi += fs * *reinterpret_cast<const f32x4*>(p + 16 * ((2 * oc + 1) ^ (r & (NC4 - 1))));
      }
      const int h = head0 + r;
      if (n > 1) {
        const int64_t at = ((int64_t)split * a.B + b) * a.Hq + h;
        f32x4* d = reinterpret_cast<f32x4*>(a.part + at * D + 8 * oc);
        d[0] = lo;
        d[1] = hi;
        if (oc == 0) {
          float* ml = a.part + (int64_t)a.splits * a.B * a.Hq * D + 2 * at;
          ml[0] = M;
          ml[1] = l;
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
static __global__ __launch_bounds__(64 * DQ_WAVES, NQ == 1 ? 3 : 2) void decode_q4_kernel(const DecodeQ4Args a) {
  using K = DecodeQ4<BF16, D, NQ>;
  __shared__ __attribute__((aligned(16))) char s_acc[DQ_WAVES * K::ACC];
  __shared__ float s_ml[2 * DQ_WAVES * K::ROWS];
  K::run(a, s_acc, s_ml);
}

// Merges the partials of the query heads of lists that were shared, D / 8 lanes a head.
template <bool BF16, int D>
static __global__ __launch_bounds__(256) void decode_q4_combine_kernel(const DecodeQ4Args a) {
  using E = Elem<BF16>;
  constexpr int LPR = D / 8, U = 4;
  const int x = (int)blockIdx.x * (256 / LPR) + (int)threadIdx.x / LPR, oc = threadIdx.x % LPR;
  if (x >= a.B * a.Hq) return;
  const int b = x / a.Hq, h = x - b * a.Hq;
  int len;
  const int32_t* list;
  const int n = a.splits_of(a.chunks(b, h / a.heads, list, len));
  if (n <= 1) return;
  const int64_t step = (int64_t)a.B * a.Hq;
  const float* ml = a.part + (int64_t)a.splits * step * D;
  float M = -__builtin_inff(), L = 0.f;
  f32x4 acc[2] = {f32x4{}, f32x4{}};
  for (int s0 = 0; s0 < n; s0 += U) {
    float m[U], l[U];
    f32x4 v[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t p = x + min(s0 + u, n - 1) * step;   // past the last: a repeat, not used
      m[u] = ml[2 * p];
      l[u] = ml[2 * p + 1];
      v[u][0] = reinterpret_cast<const f32x4*>(a.part + p * D + 8 * oc)[0];
      v[u][1] = reinterpret_cast<const f32x4*>(a.part + p * D + 8 * oc)[1];
    }
    float Mc = M;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u < n) Mc = fmaxf(Mc, m[u]);
    // As in chunk_items.h: a share of NaN scores has sums of NaN, which reach the row.
    const float Mu = Mc == -__builtin_inff() ? 0.f : Mc;
    const float f0 = fast_exp2(M - Mu);
    L *= f0;
    acc[0] *= f0;
    acc[1] *= f0;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u < n) {
        const float fs = fast_exp2(m[u] - Mu);
        L += fs * l[u];
        acc[0] += fs * v[u][0];
        acc[1] += fs * v[u][1];
      }
    M = Mc;
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
  if (a.splits > 1) {
    const int per = 256 / (D / 8);
    hipLaunchKernelGGL((decode_q4_combine_kernel<BF16, D>), dim3((unsigned)((a.B * a.Hq + per - 1) / per)), dim3(256), 0, s, a);
  }
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : set_error((int)err, "sa_decode_q4: launch failed: %s", hipGetErrorString(err));
}

// Steps of 32 keys of the longest list.
static int64_t decode_q4_steps(int64_t blocks, int page) { return std::max<int64_t>(1, (std::min<int64_t>(blocks * page, MAX_KV_LEN) + 31) / 32); }

}  // namespace sa

using namespace sa;

extern "C" int64_t sa_decode_q4_workspace_bytes(int B, int Hq, int D, int num_splits) {
  return num_splits > 1 && B > 0 && Hq > 0 && D > 0 ? (int64_t)num_splits * B * Hq * (D + 2) * 4 : 0;
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
      block_table_stride < max_blocks || num_splits < 1 || num_splits > 64)
    return set_error(SA_E_SHAPE, "%s: bad sizes B=%d Hq=%d Hkv=%d, table of %d columns (stride %lld), %d pages, "
                     "%d splits (1..64)", name, B, Hq, Hkv, max_blocks, (long long)block_table_stride, num_pages, num_splits);
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
  const int64_t steps = decode_q4_steps(sel_off ? sel_width : a.max_blocks, page);
  a.unit = (int)((steps + num_splits - 1) / num_splits);
  a.splits = (int)((steps + a.unit - 1) / a.unit);
  const int64_t need = sa_decode_q4_workspace_bytes(B, Hq, D, a.splits);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(SA_E_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", name, (long long)workspace_bytes,
                     (long long)need);
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
  a.rows = sel_off ? sel_rows : Hkv;
  a.heads = Hq / a.rows;
  a.group = a.rows / Hkv;
  // Query heads of a workgroup: one column set, or two.
  const int per_set = 16 / (D / 32), sets = a.heads > per_set ? 2 : 1;
  a.tiles = (a.heads + sets * per_set - 1) / (sets * per_set);
  a.o = static_cast<elem_t*>(o);
  a.o_sb = o_sb, a.o_sh = o_sh;
  a.B = B, a.Hq = Hq;
  a.part = static_cast<float*>(workspace);
  a.scale_log2 = sm_scale * 1.44269504088896340736f;
  const int64_t groups = (int64_t)B * a.rows * a.tiles * a.splits;
  if (groups > MAX_WORKGROUPS || (int64_t)B * Hq > 0x7fffffff / 2)
    return set_error(SA_E_SHAPE, "%s: %lld workgroups are too many for one launch", name, (long long)groups);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == SA_DTYPE_BF16)
    return D == 128 ? launch_decode_q4<true, 128>(a, groups, sets, s) : launch_decode_q4<true, 64>(a, groups, sets, s);
  return D == 128 ? launch_decode_q4<false, 128>(a, groups, sets, s) : launch_decode_q4<false, 64>(a, groups, sets, s);
}
