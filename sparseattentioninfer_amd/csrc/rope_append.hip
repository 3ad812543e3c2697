// Per-head RMS norms and rotary embedding of queries and keys, and the paged write of a chunk's keys and values
// with the key bounds of the pages (gfx950).
//
//   n = x * rsqrt(mean(x^2) + eps) * w                                   (w given; else n = x)
//   y[i] = n[i] c - n[i + D/2] s,  y[i + D/2] = n[i + D/2] c + n[i] s,   c, s = cos, sin(inv_freq[i] * position)
//
// Everything is fp32 and rounded once, to the element type, on the way out.  The angle is the exception: an
// fp32 product inv_freq * position is off by up to 2^-24 of itself, 0.006 rad at position 100,000, more than the
// output's rounding.  It is formed in fp64, in turns, reduced to half a turn and only then taken to fp32.
//
// Memory bound: each element is read once and written once.  A workgroup takes a window of consecutive tokens and
// a share of the heads.  It computes the window's cos and sin once, into LDS (one sincos per token and pair
// whatever the number of heads), then each wave takes whole heads: D/16 lanes hold one token's head, each the two
// 16-byte chunks that the rotation mixes, so a wave moves 1024 / D tokens of a head per pass and the norm is a
// reduction over D/16 neighbouring lanes.  One pass's loads run under the pass before (loops are kept rolled: short
// calls are bound by latency and instruction fetch).
//
// Pages: with bounds a window is the positions of one page, else 16, so the tokens that a chunk adds to one page
// belong to one window where bounds need it, and one wave sees all of them for a head.  It keeps their minimum and maximum in
// registers and updates the page's bounds with plain stores: merged with the stored bounds when the page held
// tokens before, else written fresh.  Min and max are exact and have no order, so the result has none either.
//
// Measured, bf16, D = 128, 32 + 8 heads: 32K tokens unpaged 136 us, 4.9 TB/s (a copy reaches 5.4); 8K tokens in 8
// sequences into pages of 16 with bounds 51 us, 3.9 TB/s, of which the kernel takes 45 to 47; 64 single tokens 7.3 to 7.6 us,
// the latency of four dependent reads (lengths, table, rows, bounds).  Angles of given positions, one 8-byte read a token,
// cost 1 % of the former (41.1 against 40.7, replayed) and nothing of the latter.
#include <algorithm>

#include "lds_tile.h"
#include "ragged.h"

namespace sa {

constexpr int RA_THREADS = 256;
constexpr int RA_WAVES = RA_THREADS / 64;
constexpr int RA_MAX_WINDOW = 128;              // tokens of a window
constexpr int RA_CHUNK = 16;                    // positions that share a page for every page size

struct RopeArgs {
  const elem_t *q, *k, *v;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_st, v_sh;
  elem_t *qo, *ko;
  int64_t qo_sb, qo_st, qo_sh, ko_sb, ko_st, ko_sh;
  const elem_t *qw, *kw;                        // norm weights, or NULL
  const float* inv_freq;                        // or NULL: no rotation
  int Hq, Hkv, heads_per_part, window;
  float eps;
  // What the angles follow.  Unpaged: token n is row n % T of batch n / T.  Paged: of packed row n, or NULL, where they
  // follow the tokens' places in their sequences.
  const int64_t* positions;
  int64_t pos_sb, pos_st;
  int64_t N;
  int T;
  uint32_t mul_T;
  uint32_t mul_window, mul_page;
  // paged
  Ragged seqs;
  elem_t *k_pages, *v_pages;
  int64_t pg_sp, pg_sh, pg_st;
  elem_t* bounds;                               // [pages, Hkv, 2, D], or NULL
  int64_t bd_sp, bd_sh;
  const int32_t* table;
  int64_t table_stride;
  int max_blocks, num_pages, page;
};

template <bool BF16>
__device__ __forceinline__ void unpack8(u32x4 v, float* f) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = Elem<BF16>::to_f32((elem_t)(v[e] & 0xffffu));
    f[2 * e + 1] = Elem<BF16>::to_f32((elem_t)(v[e] >> 16));
  }
}
template <bool BF16>
__device__ __forceinline__ u32x4 pack8(const float* f) {
  u32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = Elem<BF16>::pack2f(f[2 * e], f[2 * e + 1]);
  return v;
}

template <bool BF16, int D, bool PAGED>
struct RopeAppend {
  static constexpr int LPR = D / 16;            // lanes of one token's head
  static constexpr int RPI = 64 / LPR;          // tokens of a wave's pass
  static constexpr int HALF = D / 2;
  static constexpr int CS_STRIDE = D + 4;       // floats of a token's cos | sin row; the pad spreads tokens over banks

  // A window: `lo` .. `hi` - 1 are the slots (token index within the window) that hold tokens.
  struct Window {
    int lo, hi, base;   // base: position of slot 0 (paged), or 0
    int64_t row0;       // packed row of slot 0 (may lie before the tensor; slots below lo are not touched)
  };

  // Batch and token of row n of an unpaged tensor.
  static __device__ __forceinline__ void batch_of(const RopeArgs& a, int64_t n, int& b, int& t) {
    b = (int)fast_div((uint32_t)n, (uint32_t)a.T, a.mul_T);
    t = (int)((uint32_t)n - (uint32_t)b * (uint32_t)a.T);
  }

  // Norm weights of a lane's 16 dims.
  struct Weights {
    u32x4 l, h;
  };

  // Where a head comes from and goes to: rows of src, then rows of dst or (paged keys and values) pages of it.
  struct Head {
    int kind, hh;                 // query, key, value; head among its kind
    const elem_t* src;
    elem_t* dst;
    int64_t s_sb, s_st, d_sb, d_st;
  };
  static __device__ __forceinline__ Head head_of(const RopeArgs& a, int h) {
    Head x;
    if (h < a.Hq) {
      x.kind = 0, x.hh = h;
      x.src = a.q + x.hh * a.q_sh, x.s_st = a.q_st, x.s_sb = a.q_sb;
      x.dst = a.qo + x.hh * a.qo_sh, x.d_st = a.qo_st, x.d_sb = a.qo_sb;
    } else if (h < a.Hq + a.Hkv) {
      x.kind = 1, x.hh = h - a.Hq;
      x.src = a.k + x.hh * a.k_sh, x.s_st = a.k_st, x.s_sb = a.k_sb;
      x.dst = PAGED ? a.k_pages + x.hh * a.pg_sh : a.ko + x.hh * a.ko_sh;
      x.d_st = PAGED ? a.pg_st : a.ko_st, x.d_sb = a.ko_sb;
    } else {
      x.kind = 2, x.hh = h - a.Hq - a.Hkv;
      x.src = a.v + x.hh * a.v_sh, x.s_st = a.v_st, x.s_sb = 0;
      x.dst = a.v_pages + x.hh * a.pg_sh, x.d_st = a.pg_st, x.d_sb = 0;
    }
    return x;
  }

  // Offset of packed row n (paged), or of token n % T of batch n / T.
  static __device__ __forceinline__ int64_t row_at(const RopeArgs& a, int64_t n, int64_t sb, int64_t st) {
    if constexpr (PAGED) return n * st;
    int bt, t;
    batch_of(a, n, bt, t);
    return bt * sb + t * st;
  }

  // Window of position p, rounded down; a position may be negative where a sequence has fewer tokens than new ones.
  static __device__ __forceinline__ int window_of(const RopeArgs& a, int p) {
    const uint32_t m = (uint32_t)(p < 0 ? a.window - 1 - p : p);
    const int q = (int)fast_div(m, (uint32_t)a.window, a.mul_window);
    return p < 0 ? -q : q;
  }

  static __device__ __forceinline__ bool find_window(const RopeArgs& a, int x, Window& w, int& b) {
    b = 0;
    if constexpr (!PAGED) {
      w.base = 0;
      w.row0 = (int64_t)x * a.window;
      w.lo = 0;
      w.hi = (int)(a.N - w.row0 < a.window ? a.N - w.row0 : a.window);
      return true;
    } else {
      auto windows = [&](int s) {
        int r0;
        const int n = a.seqs.rows(s, r0), end = a.seqs.kv_len(s);
        return n ? window_of(a, end - 1) - window_of(a, end - n) + 1 : 0;
      };
      int local;
      if (!find_item(a.seqs.B, x, windows, b, local)) return false;
      int r0;
      const int n = a.seqs.rows(b, r0), end = a.seqs.kv_len(b), start = end - n;
      w.base = (window_of(a, start) + local) * a.window;
      w.lo = max(0, start - w.base);
      w.hi = min(a.window, end - w.base);
      w.row0 = (int64_t)r0 + w.base - start;
      return true;
    }
  }

  static __device__ void run(const RopeArgs& a) {
    extern __shared__ float s_cs[];   // window x CS_STRIDE
    __shared__ int s_page[RA_MAX_WINDOW / RA_CHUNK], s_slot[RA_MAX_WINDOW / RA_CHUNK];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Window w;
    int b;
    if (!find_window(a, blockIdx.x, w, b)) return;

    // The norm weights of this lane's dims, and cos and sin of the window's tokens: one pair to a thread.
    const int c = lane % LPR;
    Weights qw = {}, kw = {};
    if (a.qw) qw = {*reinterpret_cast<const u32x4*>(a.qw + 8 * c), *reinterpret_cast<const u32x4*>(a.qw + HALF + 8 * c)};
    if (a.kw) kw = {*reinterpret_cast<const u32x4*>(a.kw + 8 * c), *reinterpret_cast<const u32x4*>(a.kw + HALF + 8 * c)};
    if (a.inv_freq) {
      const int i = tid % HALF;
      const double freq = (double)a.inv_freq[i] * 0.15915494309189533577;   // / 2 pi: turns
      for (int slot = w.lo + tid / HALF; slot < w.hi; slot += RA_THREADS / HALF) {
        double p;
        if constexpr (PAGED) {
          p = a.positions ? (double)a.positions[(w.row0 + slot) * a.pos_st] : (double)(w.base + slot);
        } else {
          int bt, t;
          batch_of(a, w.row0 + slot, bt, t);
          p = (double)a.positions[bt * a.pos_sb + t];
        }
        const double turns = p * freq;
        float si, co;
        sincospif(2.f * (float)(turns - rint(turns)), &si, &co);
        s_cs[slot * CS_STRIDE + i] = co;
        s_cs[slot * CS_STRIDE + HALF + i] = si;
      }
    }
    if (PAGED && tid < a.window / RA_CHUNK) {
      const int p = w.base + tid * RA_CHUNK;
      int pg = -1, slot = 0;
      const int lb = p < 0 ? -1 : (int)fast_div((uint32_t)p, (uint32_t)a.page, a.mul_page);
      if (lb >= 0 && lb < a.max_blocks) {
        pg = a.table[b * a.table_stride + lb];
        slot = p - lb * a.page;
        if (pg < 0 || pg >= a.num_pages) pg = -1;
      }
      s_page[tid] = pg;
      s_slot[tid] = slot;
    }
    __syncthreads();

    // Passes of RPI tokens of a head, head by head; the loads of the next pass are in flight meanwhile.
    const int heads = a.Hq + a.Hkv + (PAGED ? a.Hkv : 0);
    const int h_end = min(heads, (int)(blockIdx.y + 1) * a.heads_per_part);
    const int g = lane / LPR, t_first = w.lo / RPI * RPI;
    u32x4 nl = {0u, 0u, 0u, 0u}, nh = nl;
    auto load = [&](const Head& hd, int slot) {
      if (slot >= w.lo && slot < w.hi) {
        const elem_t* p = hd.src + row_at(a, w.row0 + slot, hd.s_sb, hd.s_st) + 8 * c;
        nl = *reinterpret_cast<const u32x4*>(p);
        nh = *reinterpret_cast<const u32x4*>(p + HALF);
      }
    };
    int h = (int)blockIdx.y * a.heads_per_part + wave, t0 = t_first;
    if (h >= h_end) return;
    Head hd = head_of(a, h);
    load(hd, t0 + g);
    float mn[16], mx[16];
    int from = w.lo;              // first slot of the page at hand (bounds)
#pragma unroll 1
    while (true) {
      const Head cur = hd;
      const int slot = t0 + g;
      const bool live = slot >= w.lo && slot < w.hi;
      u32x4 vl = nl, vh = nh;
      t0 += RPI;
      const bool head_done = t0 >= w.hi;
      if (head_done) {
        h += RA_WAVES;
        t0 = t_first;
        if (h < h_end) hd = head_of(a, h);
      }
      if (h < h_end) load(hd, t0 + g);
      if (cur.kind < 2) {
        float l[8], r[8];
        unpack8<BF16>(vl, l);
        unpack8<BF16>(vh, r);
        if (cur.kind ? a.kw != nullptr : a.qw != nullptr) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss += l[e] * l[e] + r[e] * r[e];
          ss = row_total(ss);
          const float inv = rsqrtf(ss * (1.f / D) + a.eps);
          float wl[8], wh[8];
          unpack8<BF16>(cur.kind ? kw.l : qw.l, wl);
          unpack8<BF16>(cur.kind ? kw.h : qw.h, wh);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            l[e] *= inv * wl[e];
            r[e] *= inv * wh[e];
          }
        }
        if (a.inv_freq && live) {
          const float* cs = s_cs + slot * CS_STRIDE + 8 * c;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float co = cs[e], si = cs[HALF + e];
            const float y = l[e] * co - r[e] * si;
            r[e] = r[e] * co + l[e] * si;
            l[e] = y;
          }
        }
        vl = pack8<BF16>(l);
        vh = pack8<BF16>(r);
      }
      if (live) {
        elem_t* d = nullptr;
        if (!PAGED || cur.kind == 0) {
          d = cur.dst + row_at(a, w.row0 + slot, cur.d_sb, cur.d_st) + 8 * c;
        } else {
          const int pg = s_page[slot / RA_CHUNK];
          if (pg >= 0)
            d = cur.dst + pg * a.pg_sp + (int64_t)(s_slot[slot / RA_CHUNK] + slot % RA_CHUNK) * cur.d_st + 8 * c;
        }
        if (d) {
          *reinterpret_cast<u32x4*>(d) = vl;
          *reinterpret_cast<u32x4*>(d + HALF) = vh;
        }
      }
      if (PAGED && cur.kind == 1 && a.bounds) {   // bounds of the stored (rounded) keys
        float y[16];
        unpack8<BF16>(vl, y);
        unpack8<BF16>(vh, y + 8);
        const int first_slot = slot - g;          // of the pass
        const bool first = first_slot <= from;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          mn[e] = fminf(first ? __builtin_inff() : mn[e], live ? y[e] : __builtin_inff());
          mx[e] = fmaxf(first ? -__builtin_inff() : mx[e], live ? y[e] : -__builtin_inff());
        }
        const int page_end = min(w.hi, from + a.page - (s_slot[from / RA_CHUNK] + from % RA_CHUNK));
        if (first_slot + RPI >= page_end) {
          bound_page(a, mn, mx, s_page[from / RA_CHUNK], s_slot[from / RA_CHUNK] + from % RA_CHUNK == 0, cur.hh, c, g);
          from = head_done ? w.lo : page_end;
        }
      }
      if (h >= h_end) break;
    }
  }

  // Sum over the LPR (4 or 8) lanes of a token's head, in every one.
  static __device__ __forceinline__ float row_total(float x) {
    x += dpp<0xB1>(x);    // lane pairs
    x += dpp<0x4E>(x);    // quads
    if constexpr (LPR == 8) x += dpp<0x141>(x);   // the two quads of 8 lanes
    return x;
  }

  // Brings a page's bounds up to date with the minimum and maximum of new keys of head hh that the lanes hold.
  static __device__ __forceinline__ void bound_page(const RopeArgs& a, float (&mn)[16], float (&mx)[16], int pg, bool fresh,
                                                    int hh, int c, int g) {
    if (pg < 0) return;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      // Over the lanes that differ in the bits of the token.
      if constexpr (LPR == 4) {
        mn[e] = fminf(mn[e], __shfl_xor(mn[e], 4, 64));
        mx[e] = fmaxf(mx[e], __shfl_xor(mx[e], 4, 64));
      }
      mn[e] = fminf(mn[e], dpp<0x128>(mn[e]));   // row_ror:8
      mx[e] = fmaxf(mx[e], dpp<0x128>(mx[e]));
      auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(mn[e]), __float_as_uint(mn[e]), false, false);
      mn[e] = -halves_max(-fminf(__uint_as_float(s[0]), __uint_as_float(s[1])));
      s = __builtin_amdgcn_permlane16_swap(__float_as_uint(mx[e]), __float_as_uint(mx[e]), false, false);
      mx[e] = halves_max(fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1])));
    }
    if (g < 2) {   // lanes of token group 0 write the minima, of group 1 the maxima
      elem_t* d = a.bounds + pg * a.bd_sp + hh * a.bd_sh + g * D + 8 * c;
      float y[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e] = g ? mx[e] : mn[e];
      if (!fresh) {
        float old[16];
        unpack8<BF16>(*reinterpret_cast<const u32x4*>(d), old);
        unpack8<BF16>(*reinterpret_cast<const u32x4*>(d + HALF), old + 8);
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] = g ? fmaxf(y[e], old[e]) : fminf(y[e], old[e]);
      }
      *reinterpret_cast<u32x4*>(d) = pack8<BF16>(y);
      *reinterpret_cast<u32x4*>(d + HALF) = pack8<BF16>(y + 8);
    }
  }
};

template <bool BF16, int D, bool PAGED>
__global__ __launch_bounds__(RA_THREADS) void rope_append_kernel(const RopeArgs a) {
  RopeAppend<BF16, D, PAGED>::run(a);
}

template <bool PAGED>
static int launch_rope(const char* name, int dtype, int D, const RopeArgs& a, dim3 grid, hipStream_t s) {
  const dim3 block(RA_THREADS);
  const size_t lds = a.inv_freq ? (size_t)a.window * (D + 4) * sizeof(float) : 0;
  if (dtype == SA_DTYPE_BF16 && D == 128)
    hipLaunchKernelGGL((rope_append_kernel<true, 128, PAGED>), grid, block, lds, s, a);
  else if (dtype == SA_DTYPE_BF16)
    hipLaunchKernelGGL((rope_append_kernel<true, 64, PAGED>), grid, block, lds, s, a);
  else if (D == 128)
    hipLaunchKernelGGL((rope_append_kernel<false, 128, PAGED>), grid, block, lds, s, a);
  else
    hipLaunchKernelGGL((rope_append_kernel<false, 64, PAGED>), grid, block, lds, s, a);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : set_error((int)err, "%s: launch failed: %s", name, hipGetErrorString(err));
}

// Heads per workgroup: the heads of a window are dealt over up to target / windows workgroups, each of which computes
// the window's cos and sin again.  Paged, four workgroups fit a CU and one round of them is best (8K tokens in 8
// sequences, 521 windows: 46.6 us with one workgroup each, 53.8 with 4, 50.0 with 7; 64 single tokens 9.1 us with 12,
// 10.3 with 7).  Unpaged, seven fit, and a round and a bit is worse than several (32K tokens, 2,048 windows: 146 us with
// one workgroup each, 139 with two).
constexpr int64_t RA_TARGET_PAGED = 1024, RA_TARGET = 4096;
static int heads_per_part(int64_t windows, int heads, int64_t target) {
  const int64_t most = (heads + RA_WAVES - 1) / RA_WAVES;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(most, target / std::max<int64_t>(1, windows)));
  return (int)((heads + parts - 1) / parts);
}

static bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; }

}  // namespace sa

using namespace sa;

extern "C" int sa_qk_norm_rope(int dtype, const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k,
                               int64_t k_sb, int64_t k_st, int64_t k_sh, void* q_out, int64_t qo_sb, int64_t qo_st,
                               int64_t qo_sh, void* k_out, int64_t ko_sb, int64_t ko_st, int64_t ko_sh,
                               const void* q_weight, const void* k_weight, const float* inv_freq,
                               const int64_t* positions, int64_t pos_sb, int B, int T, int Hq, int Hkv, int D,
                               float eps, void* stream) {
  clear_error();
  const char* name = "sa_qk_norm_rope";
  if (dtype != SA_DTYPE_BF16 && dtype != SA_DTYPE_F16)
    return set_error(SA_E_DTYPE, "%s: dtype %d is not bf16 (0) or f16 (1)", name, dtype);
  if (D != 64 && D != 128) return set_error(SA_E_HEADDIM, "%s: head dim %d not supported (64, 128)", name, D);
  if (B < 0 || T < 0 || Hq < 0 || Hkv < 0 || Hq > (1 << 20) || Hkv > (1 << 20))
    return set_error(SA_E_SHAPE, "%s: bad sizes B=%d T=%d Hq=%d Hkv=%d", name, B, T, Hq, Hkv);
  if (B == 0 || T == 0 || Hq + Hkv == 0) return 0;
  if ((Hq && (!q || !q_out)) || (Hkv && (!k || !k_out)) || !inv_freq || !positions)
    return set_error(SA_E_NULL, "%s: NULL pointer", name);
  if (misaligned(q) || misaligned(k) || misaligned(q_out) || misaligned(k_out) || misaligned(q_weight) ||
      misaligned(k_weight) || (q_sb | q_st | q_sh | k_sb | k_st | k_sh | qo_sb | qo_st | qo_sh | ko_sb | ko_st | ko_sh) % 8)
    return set_error(SA_E_ALIGN, "%s: head rows must be 16-byte aligned", name);
  RopeArgs a = {};
  a.q = static_cast<const elem_t*>(q);
  a.k = static_cast<const elem_t*>(k);
  a.qo = static_cast<elem_t*>(q_out);
  a.ko = static_cast<elem_t*>(k_out);
  a.q_sb = q_sb, a.q_st = q_st, a.q_sh = q_sh, a.k_sb = k_sb, a.k_st = k_st, a.k_sh = k_sh;
  a.qo_sb = qo_sb, a.qo_st = qo_st, a.qo_sh = qo_sh, a.ko_sb = ko_sb, a.ko_st = ko_st, a.ko_sh = ko_sh;
  a.qw = static_cast<const elem_t*>(q_weight);
  a.kw = static_cast<const elem_t*>(k_weight);
  a.inv_freq = inv_freq;
  a.positions = positions;
  a.pos_sb = pos_sb;
  a.N = (int64_t)B * T;
  a.T = T;
  a.mul_T = div_mul((uint32_t)T);
  a.Hq = Hq, a.Hkv = Hkv, a.eps = eps;
  a.window = 16;
  const int64_t windows = (a.N + a.window - 1) / a.window;
  if (windows > MAX_WORKGROUPS) return set_error(SA_E_SHAPE, "%s: %lld tokens are too many", name, (long long)a.N);
  a.heads_per_part = heads_per_part(windows, Hq + Hkv, RA_TARGET);
  const int parts = (Hq + Hkv + a.heads_per_part - 1) / a.heads_per_part;
  return launch_rope<false>(name, dtype, D, a, dim3((unsigned)windows, parts), static_cast<hipStream_t>(stream));
}

static int append(const char* name, int dtype, const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st,
                  int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, void* q_out, int64_t qo_st, int64_t qo_sh,
                  const void* q_weight, const void* k_weight, const float* inv_freq, const int64_t* positions,
                  int64_t pos_st, void* k_pages, void* v_pages, int64_t pages_sp, int64_t pages_sh, int64_t pages_st,
                  int num_pages, void* k_bounds, int64_t bounds_sp, int64_t bounds_sh, const int32_t* block_table,
                  int64_t block_table_stride, int max_blocks, const int32_t* cu_seqlens, const int32_t* kv_lens, int N,
                  int B, int Hq, int Hkv, int D, int page, float eps, void* stream) {
  if (dtype != SA_DTYPE_BF16 && dtype != SA_DTYPE_F16)
    return set_error(SA_E_DTYPE, "%s: dtype %d is not bf16 (0) or f16 (1)", name, dtype);
  if (D != 64 && D != 128) return set_error(SA_E_HEADDIM, "%s: head dim %d not supported (64, 128)", name, D);
  if (page < 16 || page > 128 || page % 16)
    return set_error(SA_E_BLOCK, "%s: page %d is not a multiple of 16 in [16, 128]", name, page);
  if (N < 0 || B < 0 || Hkv < 1 || Hq < 0 || Hq > (1 << 20) || Hkv > (1 << 20) || max_blocks < 0 || num_pages < 0 ||
      block_table_stride < max_blocks)
    return set_error(SA_E_SHAPE, "%s: bad sizes N=%d B=%d Hq=%d Hkv=%d, table of %d columns (stride %lld), %d pages",
                     name, N, B, Hq, Hkv, max_blocks, (long long)block_table_stride, num_pages);
  if (N == 0 || B == 0) return 0;
  // A table without columns and pools without pages are neither read nor written.
  if (!k || !v || (num_pages && (!k_pages || !v_pages)) || (max_blocks && !block_table) || !cu_seqlens || !kv_lens ||
      (Hq && (!q || !q_out)))
    return set_error(SA_E_NULL, "%s: NULL pointer", name);
  if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(q_out) || misaligned(q_weight) ||
      misaligned(k_weight) || misaligned(k_pages) || misaligned(v_pages) || misaligned(k_bounds) ||
      (q_st | q_sh | k_st | k_sh | v_st | v_sh | qo_st | qo_sh | pages_sp | pages_sh | pages_st | bounds_sp | bounds_sh) % 8)
    return set_error(SA_E_ALIGN, "%s: head rows must be 16-byte aligned", name);
  RopeArgs a = {};
  a.q = static_cast<const elem_t*>(q);
  a.k = static_cast<const elem_t*>(k);
  a.v = static_cast<const elem_t*>(v);
  a.qo = static_cast<elem_t*>(q_out);
  a.q_st = q_st, a.q_sh = q_sh, a.k_st = k_st, a.k_sh = k_sh, a.v_st = v_st, a.v_sh = v_sh;
  a.qo_st = qo_st, a.qo_sh = qo_sh;
  a.qw = static_cast<const elem_t*>(q_weight);
  a.kw = static_cast<const elem_t*>(k_weight);
  a.inv_freq = inv_freq;
  a.positions = positions;
  a.pos_st = pos_st;
  a.N = N;
  a.Hq = Hq, a.Hkv = Hkv, a.eps = eps;
  a.seqs = Ragged{cu_seqlens, kv_lens, B, N};
  a.k_pages = static_cast<elem_t*>(k_pages);
  a.v_pages = static_cast<elem_t*>(v_pages);
  a.pg_sp = pages_sp, a.pg_sh = pages_sh, a.pg_st = pages_st;
  a.bounds = static_cast<elem_t*>(k_bounds);
  a.bd_sp = bounds_sp, a.bd_sh = bounds_sh;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.max_blocks = max_blocks, a.num_pages = num_pages, a.page = page;
  // Bounds want whole pages; else the shortest window, whose cos and sin are soonest done.
  a.window = k_bounds ? page : RA_CHUNK;
  a.mul_window = div_mul((uint32_t)a.window);
  a.mul_page = div_mul((uint32_t)page);
  // n new tokens touch at most (n - 1) / window + 2 windows, and at most n
  const int64_t windows = std::min<int64_t>(N, (int64_t)N / a.window + 2 * (int64_t)std::min(B, N));
  if (windows > MAX_WORKGROUPS) return set_error(SA_E_SHAPE, "%s: N=%d B=%d are too many", name, N, B);
  const int heads = Hq + 2 * Hkv;
  a.heads_per_part = heads_per_part(windows, heads, RA_TARGET_PAGED);
  const int parts = (heads + a.heads_per_part - 1) / a.heads_per_part;
  return launch_rope<true>(name, dtype, D, a, dim3((unsigned)windows, parts), static_cast<hipStream_t>(stream));
}

extern "C" int sa_paged_append(int dtype, const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st,
                               int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, void* q_out, int64_t qo_st,
                               int64_t qo_sh, const void* q_weight, const void* k_weight, const float* inv_freq,
                               void* k_pages, void* v_pages, int64_t pages_sp, int64_t pages_sh, int64_t pages_st,
                               int num_pages, void* k_bounds, int64_t bounds_sp, int64_t bounds_sh,
                               const int32_t* block_table, int64_t block_table_stride, int max_blocks,
                               const int32_t* cu_seqlens, const int32_t* kv_lens, int N, int B, int Hq, int Hkv,
                               int D, int page, float eps, void* stream) {
  clear_error();
  return append("sa_paged_append", dtype, q, q_st, q_sh, k, k_st, k_sh, v, v_st, v_sh, q_out, qo_st, qo_sh, q_weight,
                k_weight, inv_freq, nullptr, 0, k_pages, v_pages, pages_sp, pages_sh, pages_st, num_pages, k_bounds,
                bounds_sp, bounds_sh, block_table, block_table_stride, max_blocks, cu_seqlens, kv_lens, N, B, Hq, Hkv, D,
                page, eps, stream);
}

extern "C" int sa_paged_append_at(int dtype, const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st,
                                  int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, void* q_out, int64_t qo_st,
                                  int64_t qo_sh, const void* q_weight, const void* k_weight, const float* inv_freq,
                                  const int64_t* positions, int64_t pos_st, void* k_pages, void* v_pages,
                                  int64_t pages_sp, int64_t pages_sh, int64_t pages_st, int num_pages, void* k_bounds,
                                  int64_t bounds_sp, int64_t bounds_sh, const int32_t* block_table,
                                  int64_t block_table_stride, int max_blocks, const int32_t* cu_seqlens,
                                  const int32_t* kv_lens, int N, int B, int Hq, int Hkv, int D, int page, float eps,
                                  void* stream) {
  clear_error();
  const char* name = "sa_paged_append_at";
  if (N > 0 && B > 0 && (!inv_freq || !positions)) return set_error(SA_E_NULL, "%s: NULL inv_freq or positions", name);
  if (pos_st < 0) return set_error(SA_E_SHAPE, "%s: positions of stride %lld", name, (long long)pos_st);
  return append(name, dtype, q, q_st, q_sh, k, k_st, k_sh, v, v_st, v_sh, q_out, qo_st, qo_sh, q_weight, k_weight,
                inv_freq, positions, pos_st, k_pages, v_pages, pages_sp, pages_sh, pages_st, num_pages, k_bounds,
                bounds_sp, bounds_sh, block_table, block_table_stride, max_blocks, cu_seqlens, kv_lens, N, B, Hq, Hkv, D,
                page, eps, stream);
}
