// Causal attention of a chunk of new tokens over a paged cache held in 4 bits (gfx950): sequences of different lengths, whole
// caches or the pages that a selection lists for each 64-query block.  Rows, items, the division of keys and the merge
// are those of the 16-bit cache (chunk_items.h).
//
// Few rows are bound by latency (8 sequences of 4 tokens over 4K, 32 + 8 heads: 23 to 24 us and 4 to 5 for the merge, for
// 42 MB; 31 to 38 in all over a 16-bit cache), many by vector and matrix issue (8K tokens over 32K: 3.65 to 4.0 ms on four cards,
// 0.96 to 1.05 PFLOP/s; a 16-bit cache reaches 1.16 to 1.24).
#include "attn_q4.h"

namespace sa {

// What the division of keys weighs (chunk_items.h), in key tiles: 2.07 us for a wide item's, 0.77 for a narrow one's
// with the chip full and 0.37 where it is not.  With the 16-bit cache's weights 8 sequences of 4 tokens over 4K take 31.3 us
// instead of 28.0 (replayed), 1,000 tokens beside 8 single ones over 8K 53.4 instead of 47.4, nine other batches within 3 %.
// MERGE_ROW is in wide tiles, 0.27 ns a row; where all items are narrow it stands for 0.1 ns, and twice the number there
// divides those eleven batches no differently.
struct ChunkQ4Cost {
  static constexpr float MERGE_WIDE = 3.f, MERGE_NARROW = 5.f, MERGE_ROW = 1.3e-4f;
  static __device__ __forceinline__ float start(int half) { return half ? 4.6f : 12.f; }   // 9.6 us
  static __device__ __forceinline__ float alone(float groups, float cus) { return groups <= cus ? 0.5f : 1.f; }
};

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
  static constexpr int DEPTH = 3;
  static_assert(ACC >= Q4Ring<D, DEPTH>::BYTES, "the waves' rings lie in the accumulators' LDS");

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

  // Query row r of the item (a repeat of its last past the end), its position.
  static __device__ __forceinline__ const elem_t* query(const ChunkQ4Args& a, const ChunkItem& it, int r, int& pos) {
    const int row = min(it.row0 + r, it.row_end - 1);
    const int token = (int)fast_div((uint32_t)row, (uint32_t)a.c.G, a.c.mul_G);
    pos = it.start + token;
    return a.c.q + (int64_t)(it.tok0 + token) * a.c.q_st + (it.kvh * a.c.G + row - token * a.c.G) * a.c.q_sh;
  }

  // Accumulator row r of a wave is D floats at r * 4 D, its 16-byte chunk x at position x ^ (r % (D / 4)).
  static __device__ __forceinline__ f32x4* acc_at(char* acc, int r, int x) {
    return reinterpret_cast<f32x4*>(acc + r * 4 * D + 16 * (x ^ (r & (D / 4 - 1))));
  }

  // Up to 16 NC rows, by scaled keys and values.
  template <int NC>
  static __device__ __forceinline__ void scaled(const ChunkQ4Args& a, const ChunkItem& it, const Q4Keys& ks, int pos_min,
                                                char* acc, float* ml, char* ring) {
    using W = Q4Dequant<BF16, D, NC, DEPTH>;
    const int lane = threadIdx.x & 63;
    W w;
    w.ring.lds = ring;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const elem_t* qs = query(a, it, 16 * c + (lane & 15), w.pos[c]) + 8 * (lane >> 4);
#pragma unroll
      for (int g = 0; g < W::NG; ++g) w.qf[c][g] = *reinterpret_cast<const u32x4*>(qs + 32 * g);
    }
    w.pos_min = pos_min;
    w.start();
    q4_run(w, ks, a.c.scale_log2);
    __syncthreads();               // the rings lie where the accumulators go
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int r = 16 * c + (lane & 15);
#pragma unroll
      for (int e = 0; e < D / 16; ++e) *acc_at(acc, r, 4 * e + (lane >> 4)) = w.O[c][e];
      const float l = quarters_sum(w.l_run[c]);
      if (lane < 16) {
        ml[2 * r] = w.m_ref[c];
        ml[2 * r + 1] = l;
      }
    }
  }

  // Up to Q4Fold::ROWS rows, by codes.
  template <int NQ>
  static __device__ __forceinline__ void folded(const ChunkQ4Args& a, const ChunkItem& it, const Q4Keys& ks, int pos_min,
                                                char* acc, float* ml, char* ring) {
    using W = Q4Fold<BF16, D, NQ, DEPTH>;
    const int lane = threadIdx.x & 63;
    W w;
    w.ring.lds = ring;
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      int pos;
      const elem_t* qs = query(a, it, x * W::RPS + W::row_of(lane), pos);
      w.set_query(x, qs, pos);
    }
    w.pos_min = pos_min;
    w.start();
    q4_run(w, ks, a.c.scale_log2);
    __syncthreads();               // the rings lie where the accumulators go
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      const int r = x * W::RPS + W::row_of(lane);
      f32x4 out[2];
      w.result(x, out);
#pragma unroll
      for (int half = 0; half < 2; ++half) *acc_at(acc, r, 8 * W::group_of(lane) + 4 * half + (lane >> 4)) = out[half];
      const float l = quarters_sum(w.l_run[x]);
      if (lane < W::RPS) {
        ml[2 * r] = w.m_ref[x];
        ml[2 * r + 1] = l;
      }
    }
  }

  // 32 rows whose keys the waves divide.  Codes are multiplied as they are for up to two column sets of rows (8 at D = 128, 16
  // at 64); more rows share the work of scaling them.
  static __device__ void narrow(const ChunkQ4Args& a, const ChunkItem& it, char* s_acc, float* s_ml) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Q4Keys ks = keys_of(a, it);
    ks.wave = wave, ks.waves = NW;
    const int pos_min = it.start + (int)fast_div((uint32_t)it.row0, (uint32_t)a.c.G, a.c.mul_G);
    const int rows = it.row_end - it.row0;
    char* acc = s_acc + wave * ACC;
    float* ml = s_ml + 2 * CK_ROWS * wave;
    char* ring = s_acc + wave * Q4Ring<D, DEPTH>::BYTES;
    constexpr int SET = Q4Fold<BF16, D, 1, DEPTH>::RPS;
    if (rows <= SET) {
      folded<1>(a, it, ks, pos_min, acc, ml, ring);
    } else if (rows <= 2 * SET) {
      folded<2>(a, it, ks, pos_min, acc, ml, ring);
    } else if (2 * SET < 16 && rows <= 16) {
      scaled<1>(a, it, ks, pos_min, acc, ml, ring);
    } else {
      scaled<2>(a, it, ks, pos_min, acc, ml, ring);
    }
    // Merge in fp32.
    __syncthreads();
    constexpr int OC = D / 8;
    for (int x = threadIdx.x; x < rows * OC; x += 64 * NW) {
      const int r = x / OC, oc = x % OC;
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
        lo += fs * *acc_at(s_acc + s * ACC, r, 2 * oc);
        hi += fs * *acc_at(s_acc + s * ACC, r, 2 * oc + 1);
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
};

// 256 rows to a workgroup: eight waves of 32 rows share every key tile.  Each wave brings an eighth of a tile's codes into
// registers a step ahead, scales them to the element type and writes them to LDS: keys as rows (lds_tile.h), values
// transposed, [D][64], so that both products read their fragments with 16-byte reads.  One step per tile and one barrier per
// step.  Block A of a step runs S^T = K Q^T of the next tile on the matrix cores under the exponentials of this one, block
// B O^T += V^T P^T.  Waves 0..3 run A(i), B(i) in step i and waves 4..7, one on each SIMD beside them, B(i - 1), A(i), so
// that the two waves of a SIMD run the vector-heavy A and the matrix-only B at the same time.  In step i the waves
// read K(i + 1), V(i) and V(i - 1) and write K(i + 2) and V(i + 1): two K and three V buffers.
// A row's reference is the maximum of its first tile and is raised only when its probabilities would pass the
// element type's range (REFIT_SUM), so the common step never touches O with vector instructions.
// Scaling is some 88 of about 225 vector instructions of a wave's step.  256 rows are what the registers hold, and so what a
// tile's scaling is shared by; each row tile of a KV head scales its key tiles again.  Roundings are those of Q4Dequant.
template <bool BF16, int D>
struct ChunkQ4Wide : StagedTile {
  using E = Elem<BF16>;
  using F = Kv4<D>;
  static constexpr int NW = 8;
  static_assert(NW * CK_ROWS == CK_WIDE_ROWS, "rows of a wide item");
  static constexpr int NCG = D / 32;
  static constexpr int NWD = D / 64;               // words of a tile's keys (and of its values) that a lane scales
  static constexpr int TILE_BYTES = CK_KT * D * 2;
  static constexpr int NBK = 2, NBV = 3;
  static constexpr int STAGE = CK_ROWS * D * 2;    // a wave's share of O
  static constexpr int LDS_BYTES = (NBK + NBV) * TILE_BYTES;
  static constexpr int KEYS = NW * 4 * 64;         // ints of LDS for the tiles' first keys
  static_assert(NW * STAGE <= LDS_BYTES, "O is staged in the K/V buffers");
  static constexpr float REFIT_SUM = BF16 ? 65536.f : 32768.f;

  // 64 tiles looked up at once: lane i holds, for tile base + i, the page and first key of the chunk of which this wave
  // scales half (a multiple of 16, and its 16 keys' place in the page in the low bits), and the tile's largest key; the
  // first keys of its four chunks go to LDS, for the tiles that need a mask.  Tiles are looked up three ahead of the one
  // whose mask is due, so a window starts three tiles back.
  static constexpr int AHEAD = 3;
  struct Window {
    int base, page, key, last;

    __device__ __forceinline__ void fill(const ChunkArgs& a, const ChunkItem& it, int first, int rb, int* s_keys) {
      base = first;
      const int lane = threadIdx.x & 63;
      key = CK_NO_KEY;
      page = 0;
      last = -1;
      int keys[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int c = it.c0 + 4 * (first + lane) + x;
        keys[x] = CK_NO_KEY;
        if (c < it.c1) {
          int lb, s;
          if (it.list) {
            const int e = (int)fast_div((uint32_t)c, (uint32_t)(a.page / 16), a.mul_ppc);
            lb = it.list[e];
            s = (c - e * (a.page / 16)) * 16;
          } else {
            lb = (int)fast_div((uint32_t)(16 * c), (uint32_t)a.page, a.mul_page);
            s = 16 * c - lb * a.page;
          }
          // (a page whose first key no row sees is not looked up; neither are ids that are no column)
          if (lb >= 0 && lb < a.max_blocks && (int64_t)lb * a.page + s <= it.pos_max) {
            const int pg = a.table[it.b * a.table_stride + lb];
            if (pg >= 0 && pg < a.num_pages) {
              keys[x] = lb * a.page + s;
              if (x == rb) {
                page = pg;
                key = keys[x] | (s >> 4);
              }
            }
          }
        }
        last = max(last, keys[x] + 15);
      }
      *reinterpret_cast<int4*>(s_keys + 4 * lane) = int4{keys[0], keys[1], keys[2], keys[3]};
    }
    __device__ __forceinline__ int key_of(int t) const { return __builtin_amdgcn_readlane(key, t - base); }
    __device__ __forceinline__ int page_of(int t) const { return __builtin_amdgcn_readlane(page, t - base); }
    __device__ __forceinline__ int last_of(int t) const { return __builtin_amdgcn_readlane(last, t - base); }
  };

  // A lane's words of a tile and their pairs.
  struct KeyWords {
    uint32_t w[NWD], st[NWD];
  };
  struct ValueWords {
    uint32_t w[NWD];
    u32x4 st;
  };

  // A operand of O^T = V^T P^T: lane l holds d = 32 dt + l % 32 of keys 32 j + 16 h + 8 (l / 32) + 0..7.
  static __device__ __forceinline__ u32x4 vtfrag(const char* cV, int v0, int swz, int j, int h, int dt) {
    return *reinterpret_cast<const u32x4*>(cV + 4096 * dt + v0 + ((16 * (4 * j + 2 * h)) ^ swz));
  }

  static __device__ void run(const ChunkQ4Args& x, const ChunkItem& it, char* s_kv, int* s_all_keys) {
    const ChunkArgs& a = x.c;
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
    const int v0 = l32 * 128, vswz = 16 * (g ^ (l32 & 7));
    const float c = a.scale_log2;
    const int nt = (it.c1 - it.c0 + 3) / 4;

    // This wave's eighth of a tile: half of chunk rb.
    const int rb = wave >> 1;
    const uint8_t* kh = x.k + it.kvh * x.sh;
    const uint8_t* vh = x.v + it.kvh * x.sh;
    // Keys: words NWD p + u of quarter kq of a token.
    const int ktok = 8 * (wave & 1) + ((lane >> 2) & 7), kq = lane & 3, p = lane >> 5;
    // Values: four tokens of one group vg; at D = 128 its dims vi and vi + 8 of both halves, at 64 dim vi.
    const int vtok = 8 * (wave & 1) + 4 * (lane & 1);
    const int vi = NWD == 2 ? (lane >> 1) & 7 : (lane >> 1) & 15, vg = NWD == 2 ? lane >> 4 : lane >> 5;
    const int k_at = ktok * F::ROW + 4 * F::NG * kq + 4 * NWD * p;
    const int v_at = (vtok >> 2) * F::QUAD + 4 * F::NG * vi + 4 * vg;
    const int stats = F::stats_at(a.page);
    const int krow16 = krow(ktok);
    char* const lds_k = sK + rb * 1024 + krow16 * 64 + 16 * (kq ^ ((krow16 >> 2) & 3)) + 4096 * NWD * p;
    char* const lds_v = sV + (32 * vg + vi) * 128 + 16 * (wave ^ (vi & 7)) + 8 * (lane & 1);
    Window w;
    KeyWords kw;
    ValueWords vw;
    auto load_k = [&](int t) {
      if (t - w.base >= 64) w.fill(a, it, t - AHEAD, rb, s_keys);
      const uint8_t* b = kh + w.page_of(t) * x.sp;
      const int packed = w.key_of(t), slot = 16 * (packed & 15), key = packed & ~15;
      if constexpr (NWD == 2) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(b + slot * F::ROW + k_at);
        kw.w[0] = v[0], kw.w[1] = v[1];
      } else {
        kw.w[0] = *reinterpret_cast<const uint32_t*>(b + slot * F::ROW + k_at);
      }
#pragma unroll
      for (int u = 0; u < NWD; ++u)
        kw.st[u] = *reinterpret_cast<const uint32_t*>(b + stats + 4 * slot + 4 * ((NWD * p + u) * a.page + ktok));
      if (key + 16 > it.end) {       // keys that are not there are zeros
#pragma unroll
        for (int u = 0; u < NWD; ++u) kw.st[u] = key + ktok < it.end ? kw.st[u] : 0u;
      }
    };
    auto load_v = [&](int t) {
      const uint8_t* b = vh + w.page_of(t) * x.sp;
      const int packed = w.key_of(t), slot = 16 * (packed & 15), key = packed & ~15;
#pragma unroll
      for (int u = 0; u < NWD; ++u)
        vw.w[u] = *reinterpret_cast<const uint32_t*>(b + slot * F::ROW + v_at + 8 * u * 4 * F::NG);
      vw.st = *reinterpret_cast<const u32x4*>(b + stats + 4 * slot + 4 * (vg * a.page + vtok));
      if (key + 16 > it.end) {
#pragma unroll
        for (int j = 0; j < 4; ++j) vw.st[j] = key + vtok + j < it.end ? vw.st[j] : 0u;
      }
    };
    // Scales the loaded words into buffers kb and vb, in 4 NWD pieces: halves of words of keys, then of values.
    constexpr int PIECES = 4 * NWD;
    uint32_t half[2];
    auto put = [&](int piece, int kb, int vb) {
      const int u = (piece >> 1) % NWD;
      if (piece < 2 * NWD) {
        const float s = q4_scale<BF16>(kw.st[u]), m = q4_min<BF16>(kw.st[u]);
        const uint32_t cs = piece & 1 ? q4_high(kw.w[u]) : q4_low(kw.w[u]);
        const uint32_t d0 = q4_scaled<BF16, false>(cs, s, m), d1 = q4_scaled<BF16, true>(cs, s, m);
        if (piece & 1)
          *reinterpret_cast<u32x4*>(lds_k + kb * TILE_BYTES + 4096 * u) = u32x4{half[0], half[1], d0, d1};
        else
          half[0] = d0, half[1] = d1;
      } else {
        const uint32_t cs = piece & 1 ? q4_high(vw.w[u]) : q4_low(vw.w[u]);
        *reinterpret_cast<u32x2*>(lds_v + vb * TILE_BYTES + 1024 * u + 2048 * (piece & 1)) =
            u32x2{q4_scaled<BF16, false>(cs, q4_scale<BF16>(vw.st[0]), q4_min<BF16>(vw.st[0]), q4_scale<BF16>(vw.st[1]),
                                         q4_min<BF16>(vw.st[1])),
                  q4_scaled<BF16, true>(cs, q4_scale<BF16>(vw.st[2]), q4_min<BF16>(vw.st[2]), q4_scale<BF16>(vw.st[3]),
                                        q4_min<BF16>(vw.st[3]))};
      }
    };
    auto put_k = [&](int kb) {
#pragma unroll
      for (int y = 0; y < 2 * NWD; ++y) put(y, kb, 0);
    };
    auto put_v = [&](int vb) {
#pragma unroll
      for (int y = 2 * NWD; y < PIECES; ++y) put(y, 0, vb);
    };
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
      load_k(0);
      load_v(0);
      put_k(0);
      put_v(0);
      if (nt > 1) {
        load_k(1);
        put_k(1);
      }
      if (nt > 2) load_k(2);
      if (nt > 1) load_v(1);
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
    auto ring = [](int y, int n) { return y >= n ? y - n : y; };
    u32x4 P[2][2];
    constexpr int NQ = D / 8;    // QK MFMAs of a tile: i -> (key half i % 2, cc = i / 2)
    constexpr int PE = 32 / NQ;  // probabilities per QK MFMA
    constexpr int NP = D / 8;    // PV MFMAs: i -> (dt = i % NCG, h, j)
    static_assert(NP == 2 * PIECES, "a piece of the scaling to every other one");

    // Block B; work(i) after its i-th product.
    auto block_b = [&](const char* cV, auto work) {
      auto vfr = [&](int i) { return vtfrag(cV, v0, vswz, i / (2 * NCG), (i / NCG) & 1, i % NCG); };
      u32x4 vf[2] = {vfr(0), vfr(1)};
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        O[i % NCG] = E::mfma32(vf[i & 1], P[i / (2 * NCG)][(i / NCG) & 1], O[i % NCG]);
        if (i + 2 < NP) vf[i & 1] = vfr(i + 2);
        work(i);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto nothing = [](int) {};
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
      put_k(kb_cur);                            // of tile t + 2 (a repeat where there is none, to a buffer that no one reads)
      put_v(ring(vb_cur + 1, NBV));             // of tile t + 1
      if (t + 3 < nt) load_k(t + 3);
      if (t + 2 < nt) load_v(t + 2);
      if (lag && pending) block_b(sV + ring(vb_cur + NBV - 1, NBV) * TILE_BYTES, nothing);
      const char* cK = sK + (kb_cur ^ 1) * TILE_BYTES;
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
          const int y = PE * i + u, j = y >> 4, rr = y & 15;
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
      if (!lag) block_b(sV + vb_cur * TILE_BYTES, nothing);
      pending = true;
      __syncthreads();
      vb_cur = ring(vb_cur + 1, NBV);
      kb_cur ^= 1;
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
      if (lag && pending) block_b(sV + ring(vb_cur + NBV - 1, NBV) * TILE_BYTES, nothing);
      float ls;
      probs(S, ls);
      if (!ref_ok || __any(!(ls <= REFIT_SUM))) raise(S, ls);
      l_run += ls;
      block_b(sV + vb_cur * TILE_BYTES, nothing);
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
        const int y = 4 * dt + rq;
        *reinterpret_cast<u32x2*>(stage + l32 * 2 * D + 16 * (y ^ (l32 & (NCH - 1))) + 8 * g) =
            u32x2{E::pack2f(O[dt][4 * rq] * inv, O[dt][4 * rq + 1] * inv),
                  E::pack2f(O[dt][4 * rq + 2] * inv, O[dt][4 * rq + 3] * inv)};
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the wave reads back what its own lanes wrote
    const int pc = lane % NCH;
#pragma unroll
    for (int k = 0; k < CK_ROWS / RPI; ++k) {
      const int r = RPI * k + lane / NCH;
      const u32x4 v = *reinterpret_cast<const u32x4*>(stage + r * 2 * D + 16 * pc);
      const int fr = it.row0 + CK_ROWS * wave + r;
      if (fr < it.row_end) {
        const int tk = (int)fast_div((uint32_t)fr, (uint32_t)a.G, a.mul_G);
        __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(a.o + (int64_t)(it.tok0 + tk) * a.o_st +
                                                                 (it.kvh * a.G + fr - tk * a.G) * a.o_sh +
                                                                 8 * (pc ^ (r & (NCH - 1)))));
      }
    }
  }
};

template <bool BF16, int D>
static __global__ __launch_bounds__(512, 2) void chunk_q4_kernel(const ChunkQ4Args a) {
  using N = ChunkQ4<BF16, D>;
  using W = ChunkQ4Wide<BF16, D>;
  __shared__ __attribute__((aligned(16))) char s_kv[W::LDS_BYTES > N::LDS_BYTES ? W::LDS_BYTES : N::LDS_BYTES];
  __shared__ __attribute__((aligned(16))) int s_aux[W::KEYS];
  static_assert(W::KEYS >= 2 * N::NW * CK_ROWS, "row references and sums of the narrow items' waves");
  ChunkItem it;
  if (!find_chunk_item<ChunkQ4Cost>(a.c, blockIdx.x, it)) return;
  if (it.narrow)
    N::narrow(a, it, s_kv, reinterpret_cast<float*>(s_aux));
  else
    W::run(a, it, s_kv, s_aux);
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
