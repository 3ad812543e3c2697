// Causal attention of a chunk of new tokens over a paged cache held in 4 bits (gfx950): sequences of different lengths, whole
// caches or the pages that a selection lists for each 64-query block.  Rows, items, the division of keys and the merge
// are those of the 16-bit cache (chunk_items.h).
#include "attn_q4.h"

namespace sa {

struct ChunkQ4Args {
  ChunkArgs c;
  const uint8_t *k, *v;
  int64_t sp, sh;                  // bytes of a page and of a head's block
};

template <bool BF16, int D>
struct ChunkQ4 {
  using E = Elem<BF16>;
  static constexpr int NW = 8;
  static constexpr int ACC = CK_ROWS * D * 4;
  static constexpr int LDS_BYTES = NW * ACC;
  using Rows32 = Q4Dequant<BF16, D, 2>;

  static __device__ __forceinline__ Q4Keys keys_of(const ChunkQ4Args& a, const ChunkItem& it) {
    Q4Keys ks;
    ks.k = a.k + it.kvh * a.sh;
    ks.v = a.v + it.kvh * a.sh;
    ks.sp = a.sp;
    ks.table = a.c.table + it.b * a.c.table_stride;
    ks.list = it.list;
    ks.max_blocks = a.c.max_blocks, ks.num_pages = a.c.num_pages, ks.page = a.c.page;
    ks.mul_page = a.c.mul_page, ks.mul_ppc = a.c.mul_ppc;
    ks.c0 = it.c0, ks.c1 = it.c1;
    ks.end = it.end, ks.pos_max = it.pos_max;
    ks.wave = 0, ks.waves = 1;
    return ks;
  }

  // Flattened rows row0 .. row0 + 31 of the item's sequence, those at or past `row_end` repeats of the last.
  static __device__ __forceinline__ void queries(const ChunkQ4Args& a, const ChunkItem& it, Rows32& w, int row0) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int row = min(row0 + 16 * c + (lane & 15), it.row_end - 1);
      const int token = (int)fast_div((uint32_t)row, (uint32_t)a.c.G, a.c.mul_G);
      w.pos[c] = it.start + token;
      const elem_t* qs = a.c.q + (int64_t)(it.tok0 + token) * a.c.q_st + (it.kvh * a.c.G + row - token * a.c.G) * a.c.q_sh +
                         8 * (lane >> 4);
#pragma unroll
      for (int g = 0; g < Rows32::NG; ++g) w.qf[c][g] = *reinterpret_cast<const u32x4*>(qs + 32 * g);
    }
    w.pos_min = it.start + (int)fast_div((uint32_t)min(row0, it.row_end - 1), (uint32_t)a.c.G, a.c.mul_G);
  }

  // 32 rows whose keys the waves divide.
  static __device__ void narrow(const ChunkQ4Args& a, const ChunkItem& it, char* s_acc, float* s_ml) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Rows32 w;
    queries(a, it, w, it.row0);
    w.start();
    Q4Keys ks = keys_of(a, it);
    ks.wave = wave, ks.waves = NW;
    q4_run(w, ks, a.c.scale_log2);
    // Merge in fp32: accumulator row r is D floats at r * 4 D, its 16-byte chunk x at position x ^ (r % (D / 4)).
    constexpr int NC4 = D / 4;
    char* acc = s_acc + wave * ACC;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = 16 * c + (lane & 15);
#pragma unroll
      for (int e = 0; e < D / 16; ++e)
        *reinterpret_cast<f32x4*>(acc + r * 4 * D + 16 * ((4 * e + (lane >> 4)) ^ (r & (NC4 - 1)))) = w.O[c][e];
      const float l = quarters_sum(w.l_run[c]);
      if (lane < 16) {
        s_ml[2 * (wave * CK_ROWS + r)] = w.m_ref[c];
        s_ml[2 * (wave * CK_ROWS + r) + 1] = l;
      }
    }
    __syncthreads();
    constexpr int OC = D / 8;
    for (int x = threadIdx.x; x < CK_ROWS * OC; x += 64 * NW) {
      const int r = x / OC, oc = x % OC;
      if (it.row0 + r >= it.row_end) continue;
      float m[NW], l = 0.f, M = -__builtin_inff();
#pragma unroll
      for (int s = 0; s < NW; ++s) {
        m[s] = s_ml[2 * (s * CK_ROWS + r)];
        M = fmaxf(M, m[s]);
      }
      const float Mu = M == -__builtin_inff() ? 0.f : M;
      f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll
      for (int s = 0; s < NW; ++s) {
        const float fs = fast_exp2(m[s] - Mu);
        l += fs * s_ml[2 * (s * CK_ROWS + r) + 1];
        const char* p = s_acc + s * ACC + r * 4 * D;
        lo += fs * *reinterpret_cast<const f32x4*>(p + 16 * ((2 * oc) ^ (r & (NC4 - 1))));
        hi += fs * *reinterpret_cast<const f32x4*>(p + 16 * ((2 * oc + 1) ^ (r & (NC4 - 1))));
      }
      const int tk = (int)fast_div((uint32_t)(it.row0 + r), (uint32_t)a.c.G, a.c.mul_G);
      const int h = it.kvh * a.c.G + it.row0 + r - tk * a.c.G;
      if (it.splits > 1) {
        const int64_t at = it.part_row(a.c, tk, h);
        f32x4* d = reinterpret_cast<f32x4*>(a.c.part_acc + at * D + 8 * oc);
        d[0] = lo;
        d[1] = hi;
        if (oc == 0) {
          a.c.part_ml[2 * at] = M;
          a.c.part_ml[2 * at + 1] = l;
        }
      } else {
        const float inv = l > 0.f ? 1.f / l : 1.f;
        *reinterpret_cast<u32x4*>(a.c.o + (int64_t)(it.tok0 + tk) * a.c.o_st + h * a.c.o_sh + 8 * oc) =
            u32x4{E::pack2f(lo[0] * inv, lo[1] * inv), E::pack2f(lo[2] * inv, lo[3] * inv),
                  E::pack2f(hi[0] * inv, hi[1] * inv), E::pack2f(hi[2] * inv, hi[3] * inv)};
      }
    }
  }

  // 256 rows, 32 to a wave.
  static __device__ void wide(const ChunkQ4Args& a, const ChunkItem& it) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row0 = it.row0 + CK_ROWS * wave;
    if (row0 >= it.row_end) return;
    Rows32 w;
    queries(a, it, w, row0);
    w.start();
    q4_run(w, keys_of(a, it), a.c.scale_log2);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int row = row0 + 16 * c + (lane & 15);
      const float l = quarters_sum(w.l_run[c]);
      if (row >= it.row_end) continue;
      const int tk = (int)fast_div((uint32_t)row, (uint32_t)a.c.G, a.c.mul_G);
      const int h = it.kvh * a.c.G + row - tk * a.c.G, q = lane >> 4;
      if (it.splits > 1) {
        const int64_t at = it.part_row(a.c, tk, h);
#pragma unroll
        for (int e = 0; e < D / 16; ++e)
          *reinterpret_cast<f32x4*>(a.c.part_acc + at * D + 16 * e + 4 * q) = w.O[c][e];
        if (q == 0) {
          a.c.part_ml[2 * at] = w.m_ref[c];
          a.c.part_ml[2 * at + 1] = l;
        }
      } else {
        const float inv = l > 0.f ? 1.f / l : 1.f;
        elem_t* o = a.c.o + (int64_t)(it.tok0 + tk) * a.c.o_st + h * a.c.o_sh + 4 * q;
#pragma unroll
        for (int e = 0; e < D / 16; ++e)
          *reinterpret_cast<u32x2*>(o + 16 * e) = u32x2{E::pack2f(w.O[c][e][0] * inv, w.O[c][e][1] * inv),
                                                         E::pack2f(w.O[c][e][2] * inv, w.O[c][e][3] * inv)};
      }
    }
  }
};

template <bool BF16, int D>
static __global__ __launch_bounds__(512, 2) void chunk_q4_kernel(const ChunkQ4Args a) {
  using K = ChunkQ4<BF16, D>;
  __shared__ __attribute__((aligned(16))) char s_acc[K::LDS_BYTES];
  __shared__ float s_ml[2 * K::NW * CK_ROWS];
  ChunkItem it;
  if (!find_chunk_item(a.c, blockIdx.x, it)) return;
  if (it.narrow)
    K::narrow(a, it, s_acc, s_ml);
  else
    K::wide(a, it);
}

template <bool BF16, int D>
static int launch_chunk_q4(const ChunkQ4Args& a, int64_t groups, hipStream_t s) {
  hipLaunchKernelGGL((chunk_q4_kernel<BF16, D>), dim3((unsigned)groups), dim3(512), 0, s, a);
  if (a.c.part) {
    const int64_t rows = a.c.seqs.N * a.c.Hq, per = 256 / (D / 8);
    hipLaunchKernelGGL((chunk_combine_kernel<BF16, D>),
                       dim3((unsigned)std::min<int64_t>((rows + per - 1) / per, 2048)), dim3(256), 0, s, a.c);
  }
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : set_error((int)err, "sa_paged_chunk_attn_q4: launch failed: %s", hipGetErrorString(err));
}

}  // namespace sa

using namespace sa;

extern "C" int sa_paged_chunk_attn_q4(int dtype, const void* q, int64_t q_st, int64_t q_sh, const void* k_pages,
                                      const void* v_pages, int64_t pages_sp, int64_t pages_sh, int num_pages,
                                      const int32_t* block_table, int64_t block_table_stride, int max_blocks,
                                      const int32_t* cu_seqlens, const int32_t* kv_lens, const int32_t* sel,
                                      int64_t sel_sr, int64_t sel_sh, int sel_rows, int sel_width,
                                      const int32_t* sel_off, int64_t off_sr, int64_t off_sh, void* o, int64_t o_st,
                                      int64_t o_sh, int N, int B, int Hq, int Hkv, int D, int page, float sm_scale,
                                      int num_splits, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  const char* name = "sa_paged_chunk_attn_q4";
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
  if (bad_ptr(q) || bad_ptr(k_pages) || bad_ptr(v_pages) || bad_ptr(o) || bad_ptr(workspace) || (q_st | q_sh | o_st | o_sh) % 8 ||
      (pages_sp | pages_sh) % 16)
    return set_error(SA_E_ALIGN, "%s: head rows and blocks must be 16-byte aligned", name);
  if (num_splits > 1 && (int64_t)N * Hq * num_splits > 0x7fffffff)
    return set_error(SA_E_SHAPE, "%s: N=%d x Hq=%d x %d splits are too many partial rows", name, N, Hq, num_splits);
  const int64_t max_keys = std::min<int64_t>((int64_t)(selected ? std::min(max_blocks, sel_width) : max_blocks) * page, 1 << 30);
  const int64_t need = sa_paged_chunk_workspace_bytes(N, B, Hq, Hkv, D, (int)max_keys, num_splits);
  if (num_splits > 1 && need && (!workspace || workspace_bytes < need))
    return set_error(SA_E_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", name, (long long)workspace_bytes,
                     (long long)need);
  ChunkQ4Args x = {};
  x.k = static_cast<const uint8_t*>(k_pages);
  x.v = static_cast<const uint8_t*>(v_pages);
  x.sp = pages_sp, x.sh = pages_sh;
  ChunkArgs& a = x.c;
  a.q = static_cast<const elem_t*>(q);
  a.q_st = q_st, a.q_sh = q_sh;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.max_blocks = num_pages ? max_blocks : 0;      // without pages no key is there, and none is loaded
  a.num_pages = num_pages, a.page = page;
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
  if (dtype == SA_DTYPE_BF16)
    return D == 128 ? launch_chunk_q4<true, 128>(x, groups, s) : launch_chunk_q4<true, 64>(x, groups, s);
  return D == 128 ? launch_chunk_q4<false, 128>(x, groups, s) : launch_chunk_q4<false, 64>(x, groups, s);
}
