// Reads a 4-bit paged cache back into rows (gfx950): the last tokens of each sequence as contiguous keys and values.
//
//   x = m + s c   in fp32, rounded once, to the element type
//
// Bound by what it writes: 2 D bytes of a token's head for 5/8 D read.  A workgroup takes the 16 positions of a chunk,
// which lie in one page, and its waves take heads in turn.  Keys: four lanes to a token, each the 8 dims of a word of
// every group, 16 bytes of output a word.  Values: a lane has 4 tokens of the dims i, i + 16 of every group; two
// exchanges with the lanes of dims i ^ 1 and i ^ 2 leave it 4 neighbouring dims, so that a store instruction writes 128
// consecutive bytes of 4 tokens (D = 128) instead of 2-byte pieces.
#include <algorithm>

#include "kv4.h"
#include "lds_tile.h"
#include "ragged.h"

namespace sa {

constexpr int RD_THREADS = 256;
constexpr int RD_CHUNK = 16;
// Outputs that the Infinity Cache would not hold are written past the caches: 289 MB in 76 us instead of 85 (4.9 TB/s, a
// copy reaches 5.2), but 66 MB in 20.1 instead of 17.7, and 131 MB and what reads it next in 82 instead of 80.
constexpr int64_t STREAM_BYTES = 1 << 28;

struct ReadArgs {
  const uint8_t *k, *v;
  int64_t sp, sh;
  elem_t *ko, *vo;
  int64_t ko_st, ko_sh, vo_st, vo_sh;
  const int32_t* table;
  int64_t table_stride;
  int max_blocks, num_pages, page;
  uint32_t mul_page;
  Ragged seqs;
  int Hkv, heads_per_part;
};

// STREAM: past the caches.
template <bool BF16, int D, bool STREAM>
struct ReadBack {
  using E = Elem<BF16>;
  using F = Kv4<D>;
  static constexpr int NG = F::NG;

  // The 8 values of a word of keys.
  static __device__ __forceinline__ u32x4 key_word(uint32_t w, uint32_t st) {
    const float s = q4_scale<BF16>(st), m = q4_min<BF16>(st);
    const uint32_t lo = q4_low(w), hi = q4_high(w);
    return u32x4{q4_scaled<BF16, false>(lo, s, m), q4_scaled<BF16, true>(lo, s, m), q4_scaled<BF16, false>(hi, s, m),
                 q4_scaled<BF16, true>(hi, s, m)};
  }
  // The two values (dims i and i + 16) of each of the four tokens of a word of values.
  static __device__ __forceinline__ u32x4 value_pairs(uint32_t w, u32x4 st) {
    const f32x2 l[2] = {q4_pair_f32<false>(q4_low(w)), q4_pair_f32<true>(q4_low(w))};
    const f32x2 h[2] = {q4_pair_f32<false>(q4_high(w)), q4_pair_f32<true>(q4_high(w))};
    u32x4 x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float s = q4_scale<BF16>(st[j]), m = q4_min<BF16>(st[j]);
      x[j] = E::pack2f(fmaf(l[j >> 1][j & 1], s, m), fmaf(h[j >> 1][j & 1], s, m));
    }
    return x;
  }
  template <int CTRL>
  static __device__ __forceinline__ uint32_t from(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
  }

  template <class T>
  static __device__ __forceinline__ void store(T* p, T x) {
    if constexpr (STREAM)
      __builtin_nontemporal_store(x, p);
    else
      *p = x;
  }

  static __device__ void run(const ReadArgs& a) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // The chunk's sequence: positions base .. base + 15, of which lo .. hi - 1 are new.
    auto chunk_of = [](int p) { return p >> 4; };   // rounded down
    auto chunks = [&](int s) {
      int r0;
      const int n = a.seqs.rows(s, r0), end = a.seqs.kv_len(s);
      return n ? chunk_of(end - 1) - chunk_of(end - n) + 1 : 0;
    };
    int b, local;
    if (!find_item(a.seqs.B, (int)blockIdx.x, chunks, b, local)) return;
    int r0;
    const int n = a.seqs.rows(b, r0), end = a.seqs.kv_len(b), start = end - n;
    const int base = (chunk_of(start) + local) * RD_CHUNK;
    const int lo = max(start, base) - base, hi = min(end - base, RD_CHUNK);
    const int64_t row0 = (int64_t)r0 + base - start;
    int pg = -1, slot = 0;
    if (base >= 0) {
      const int lb = (int)fast_div((uint32_t)base, (uint32_t)a.page, a.mul_page);
      if (lb < a.max_blocks) pg = a.table[b * a.table_stride + lb];
      if (pg >= a.num_pages) pg = -1;
      slot = base - lb * a.page;
    }
    const int64_t at = (int64_t)max(pg, 0) * a.sp;
    const int h_end = min(a.Hkv, (int)(blockIdx.y + 1) * a.heads_per_part);
    const int t = lane >> 2, q = lane & 3;        // keys: token, word of each group
    const int i = lane & 15, t4 = lane >> 4;      // values: dim of each group, four tokens
    const bool odd = i & 1, high = i & 2;
#pragma unroll 1
    for (int h = (int)blockIdx.y * a.heads_per_part + wave; h < h_end; h += RD_THREADS / 64) {
      Words<NG> kw, vw;
      uint32_t ks[NG];
      u32x4 vs[NG];
      if (pg >= 0) {
        const uint8_t* kb = a.k + at + h * a.sh;
        const uint8_t* vb = a.v + at + h * a.sh;
        kw.load(kb + (slot + t) * F::ROW + 4 * NG * q);
        vw.load(vb + slot * F::ROW + t4 * F::QUAD + 4 * NG * i);
        const int st = F::stats_at(a.page) + 4 * slot;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          ks[g] = *reinterpret_cast<const uint32_t*>(kb + st + 4 * (g * a.page + t));
          vs[g] = *reinterpret_cast<const u32x4*>(vb + st + 4 * (g * a.page) + 16 * t4);
        }
      } else {                                    // positions without a page are zeros
#pragma unroll
        for (int g = 0; g < NG; ++g) kw.w[g] = vw.w[g] = ks[g] = 0u, vs[g] = u32x4{0u, 0u, 0u, 0u};
      }
      if (t >= lo && t < hi) {
        elem_t* d = a.ko + (row0 + t) * a.ko_st + h * a.ko_sh + 8 * q;
#pragma unroll
        for (int g = 0; g < NG; ++g) store(reinterpret_cast<u32x4*>(d + 32 * g), key_word(kw.w[g], ks[g]));
      }
      // Values: x[g][j] = dims i, i + 16 of group g, token 4 t4 + j.  From lane i ^ 1: dims i & ~1 and the next, of the
      // group's lower half in even lanes, upper half in odd ones.  From lane i ^ 2: four dims, of an even group in
      // lanes i < 2 of four, of the odd group after it in the others.
      u32x4 x[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) x[g] = value_pairs(vw.w[g], vs[g]);
      const uint32_t sel = odd ? 0x03020706u : 0x05040100u;   // (neighbour's, own) upper halves; (own, neighbour's) lower
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int tok = 4 * t4 + j;
        const bool live = tok >= lo && tok < hi;
        elem_t* d = a.vo + (row0 + tok) * a.vo_st + h * a.vo_sh + (odd ? 16 : 0) + (i & 12) + (high ? 32 : 0);
#pragma unroll
        for (int g = 0; g < NG; g += 2) {
          const uint32_t y0 = __builtin_amdgcn_perm(from<0xB1>(x[g][j]), x[g][j], sel);
          const uint32_t y1 = __builtin_amdgcn_perm(from<0xB1>(x[g + 1][j]), x[g + 1][j], sel);
          const uint32_t z = from<0x4E>(high ? y0 : y1);
          if (live) store(reinterpret_cast<u32x2*>(d + 32 * g), high ? u32x2{z, y1} : u32x2{y0, z});
        }
      }
    }
  }
};

template <bool BF16, int D, bool STREAM>
static __global__ __launch_bounds__(RD_THREADS) void read_q4_kernel(const ReadArgs a) {
  ReadBack<BF16, D, STREAM>::run(a);
}

template <bool BF16, int D>
static void launch_read_q4(const ReadArgs& a, bool stream, dim3 grid, hipStream_t s) {
  if (stream)
    hipLaunchKernelGGL((read_q4_kernel<BF16, D, true>), grid, dim3(RD_THREADS), 0, s, a);
  else
    hipLaunchKernelGGL((read_q4_kernel<BF16, D, false>), grid, dim3(RD_THREADS), 0, s, a);
}

}  // namespace sa

using namespace sa;

extern "C" int sa_paged_read_q4(int dtype, const void* k_pages, const void* v_pages, int64_t pages_sp, int64_t pages_sh,
                                int num_pages, const int32_t* block_table, int64_t block_table_stride, int max_blocks,
                                const int32_t* cu_seqlens, const int32_t* kv_lens, void* k_out, int64_t ko_st,
                                int64_t ko_sh, void* v_out, int64_t vo_st, int64_t vo_sh, int N, int B, int Hkv, int D,
                                int page, void* stream) {
  clear_error();
  const char* name = "sa_paged_read_q4";
  if (dtype != SA_DTYPE_BF16 && dtype != SA_DTYPE_F16)
    return set_error(SA_E_DTYPE, "%s: dtype %d is not bf16 (0) or f16 (1)", name, dtype);
  if (D != 64 && D != 128) return set_error(SA_E_HEADDIM, "%s: head dim %d not supported (64, 128)", name, D);
  if (page < 16 || page > 128 || page % 16)
    return set_error(SA_E_BLOCK, "%s: page %d is not a multiple of 16 in [16, 128]", name, page);
  if (N < 0 || B < 0 || Hkv < 1 || Hkv > (1 << 20) || max_blocks < 0 || num_pages < 0 || block_table_stride < max_blocks)
    return set_error(SA_E_SHAPE, "%s: bad sizes N=%d B=%d Hkv=%d, table of %d columns (stride %lld), %d pages", name, N, B,
                     Hkv, max_blocks, (long long)block_table_stride, num_pages);
  if (N == 0 || B == 0) return 0;
  // A table without columns and pools without pages are not read.
  if ((num_pages && (!k_pages || !v_pages)) || (max_blocks && !block_table) || !cu_seqlens || !kv_lens || !k_out || !v_out)
    return set_error(SA_E_NULL, "%s: NULL pointer", name);
  auto misaligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  if (misaligned(k_pages) || misaligned(v_pages) || misaligned(k_out) || misaligned(v_out) || (pages_sp | pages_sh) % 16 ||
      (ko_st | ko_sh | vo_st | vo_sh) % 8)
    return set_error(SA_E_ALIGN, "%s: blocks and head rows must be 16-byte aligned", name);
  ReadArgs a = {};
  a.k = static_cast<const uint8_t*>(k_pages);
  a.v = static_cast<const uint8_t*>(v_pages);
  a.sp = pages_sp, a.sh = pages_sh;
  a.ko = static_cast<elem_t*>(k_out);
  a.vo = static_cast<elem_t*>(v_out);
  a.ko_st = ko_st, a.ko_sh = ko_sh, a.vo_st = vo_st, a.vo_sh = vo_sh;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.max_blocks = max_blocks, a.num_pages = num_pages, a.page = page;
  a.mul_page = div_mul((uint32_t)page);
  a.seqs = Ragged{cu_seqlens, kv_lens, B, N};
  a.Hkv = Hkv;
  // n tokens touch at most (n - 1) / 16 + 2 chunks, and at most n
  const int64_t chunks = std::min<int64_t>(N, (int64_t)N / RD_CHUNK + 2 * (int64_t)std::min(B, N));
  if (chunks > MAX_WORKGROUPS) return set_error(SA_E_SHAPE, "%s: N=%d B=%d are too many", name, N, B);
  // Heads are dealt over workgroups, one to a wave, unless there are workgroups for many rounds.
  const int64_t most = (Hkv + RD_THREADS / 64 - 1) / (RD_THREADS / 64);
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(most, 16384 / std::max<int64_t>(1, chunks)));
  a.heads_per_part = (int)((Hkv + parts - 1) / parts);
  const dim3 grid((unsigned)chunks, (unsigned)((Hkv + a.heads_per_part - 1) / a.heads_per_part));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool past = (int64_t)N * Hkv * D * 4 > STREAM_BYTES;
  if (dtype == SA_DTYPE_BF16) {
    if (D == 128) launch_read_q4<true, 128>(a, past, grid, s);
    else launch_read_q4<true, 64>(a, past, grid, s);
  } else {
    if (D == 128) launch_read_q4<false, 128>(a, past, grid, s);
    else launch_read_q4<false, 64>(a, past, grid, s);
  }
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : set_error((int)err, "%s: launch failed: %s", name, hipGetErrorString(err));
}
