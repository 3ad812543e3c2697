// Attention of one wave over keys held in 4 bits (gfx950): codes go from memory to the operands of v_mfma 16x16x32 by way
// of LDS of the wave's own, without a barrier and without a change of lanes.
//
// A step is 32 keys, two chunks of 16 that each lie in one page.  S^T = K Q^T: keys are the rows of the product, so a lane
// of column n holds scores of row n of the queries for four keys of each chunk, and those of both chunks are, as they lie,
// the B operand of O^T = V^T P^T.  The order of the codes in a page (kv4.h) makes each operand whole bytes of the lane.
#pragma once

#include "chunk_items.h"
#include "kv4.h"

namespace sa {

// Sum / max over lanes that differ in bits 4 and 5 only, in every lane.
__device__ __forceinline__ float quarters_sum(float x) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return halves_sum(__uint_as_float(s[0]) + __uint_as_float(s[1]));
}
__device__ __forceinline__ float quarters_max(float x) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return halves_max(fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1])));
}

// The keys of an item: chunks [c0, c1) of one sequence and KV head, of which this wave takes every `waves`-th step of two,
// from step `wave` on.
struct Q4Keys {
  const uint8_t *k, *v;            // pools, from the KV head on
  int64_t sp;                      // bytes of a page
  const int32_t* table;            // of the sequence
  const int32_t* list;             // selected pages, or NULL
  int max_blocks, num_pages, page;
  uint32_t mul_page, mul_ppc;
  int c0, c1;
  int end, pos_max;                // tokens of the sequence; the last position that a row of the item sees
  int wave, waves;

  __device__ __forceinline__ int steps() const {
    const int all = (c1 - c0 + 1) / 2;
    return max(0, (all - wave + waves - 1) / waves);
  }
};

// The chunks of 32 steps, looked up at once: lane 2 i + h holds chunk h of step base + i.
struct Q4Window {
  int base;
  int64_t off;                     // its page's byte
  int key, slot;                   // its first key, CK_NO_KEY if no row of the item sees it; that key's slot

  __device__ __forceinline__ void fill(const Q4Keys& ks, int first) {
    base = first;
    const int lane = threadIdx.x & 63;
    const int x = ks.c0 + 2 * (ks.wave + (first + (lane >> 1)) * ks.waves) + (lane & 1);
    key = CK_NO_KEY;
    off = 0;
    slot = 0;
    if (x < ks.c1) {
      int lb, s;
      if (ks.list) {
        const int e = (int)fast_div((uint32_t)x, (uint32_t)(ks.page / 16), ks.mul_ppc);
        lb = ks.list[e];
        s = (x - e * (ks.page / 16)) * 16;
      } else {
        lb = (int)fast_div((uint32_t)(16 * x), (uint32_t)ks.page, ks.mul_page);
        s = 16 * x - lb * ks.page;
      }
      if (lb >= 0 && lb < ks.max_blocks && (int64_t)lb * ks.page + s <= ks.pos_max) {
        const int pg = ks.table[lb];
        if (pg >= 0 && pg < ks.num_pages) {
          off = (int64_t)pg * ks.sp;
          key = lb * ks.page + s;
          slot = s;
        }
      }
    }
  }
  __device__ __forceinline__ int key_of(int step, int h) const {
    return __builtin_amdgcn_readlane(key, 2 * (step - base) + h);
  }
  __device__ __forceinline__ int slot_of(int step, int h) const {
    return __builtin_amdgcn_readlane(slot, 2 * (step - base) + h);
  }
  __device__ __forceinline__ int64_t off_of(int step, int h) const {
    const int l = 2 * (step - base) + h;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(uint64_t)off, l);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)off >> 32), l);
    return (int64_t)(((uint64_t)hi << 32) | lo);
  }
};

// What a wave's 32-key steps leave: fp32 accumulators of rows of queries against row references (base 2), and the sums of
// their probabilities.  Row references are raised when a lane's probabilities of a step sum past this: no probability then exceeds 2^16 in
// bf16 (2^15 in fp16, whose largest is 65,504).
template <bool BF16>
constexpr float Q4_REFIT = BF16 ? 65536.f : 32768.f;

// A wave's steps on their way: a ring of DEPTH steps of codes and pairs in LDS of its own, filled by direct loads.  The
// loads of the DEPTH - 1 steps ahead are in flight while one is worked on, without registers of their own.
template <int D, int DEPTH>
struct Q4Ring {
  using F = Kv4<D>;
  static constexpr int NG = F::NG;
  static constexpr int CODES = 16 * F::ROW, PAIRS = 64 * NG;       // bytes of a chunk's keys (or values)
  static constexpr int STEP = 4 * (CODES + PAIRS);                 // [keys, values][chunk] codes, then so the pairs
  static constexpr int BYTES = DEPTH * STEP;
  static constexpr int LOADS = NG == 4 ? 8 : 4;                    // direct loads of a step
  char* lds;

  __device__ __forceinline__ void issue(const Q4Keys& keys, const Q4Window& w, int step, int slot) const {
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
    const uint32_t at = lds_addr(lds + slot * STEP), pairs_at = at + 4 * CODES;
    if constexpr (NG == 4) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int s = w.slot_of(step, h);
        const int64_t off = w.off_of(step, h) + s * F::ROW;
        const uint8_t *kb = keys.k + off, *vb = keys.v + off;
        const int st = F::stats_at(keys.page) + s * (4 - F::ROW);
        load_lds16(kb, i * F::ROW + 16 * q, at + h * CODES);
        load_lds16(vb, q * F::QUAD + 16 * i, at + (2 + h) * CODES);
        load_lds4(kb + st, 4 * (q * keys.page + i), pairs_at + h * PAIRS);
        load_lds4(vb + st, 4 * (q * keys.page + i), pairs_at + (2 + h) * PAIRS);
      }
    } else {
      // Half a wave holds a chunk: both chunks in one load.
      const int h = lane >> 5, s0 = w.slot_of(step, 0), s1 = w.slot_of(step, 1);
      const int64_t o0 = w.off_of(step, 0), o1 = w.off_of(step, 1);
      const int s = h ? s1 : s0;
      const int64_t off = (h ? o1 : o0) + s * F::ROW + 16 * (lane & 31);
      const int64_t st = (h ? o1 : o0) + F::stats_at(keys.page) + 4 * (s + (q & 1) * keys.page + i);
      load_lds16(keys.k + off, at);
      load_lds16(keys.v + off, at + 2 * CODES);
      load_lds4(keys.k + st, pairs_at);
      load_lds4(keys.v + st, pairs_at + 2 * PAIRS);
    }
  }
  // The lane's words of chunk h.
  __device__ __forceinline__ Words<NG> keys(int slot, int h) const {
    const int lane = threadIdx.x & 63;
    Words<NG> x;
    x.load(reinterpret_cast<const uint8_t*>(lds) + slot * STEP + h * CODES +
           (NG == 4 ? 16 * lane : (lane & 15) * F::ROW + 8 * (lane >> 4)));
    return x;
  }
  __device__ __forceinline__ Words<NG> values(int slot, int h) const {
    const int lane = threadIdx.x & 63;
    Words<NG> x;
    x.load(reinterpret_cast<const uint8_t*>(lds) + slot * STEP + (2 + h) * CODES +
           (NG == 4 ? 16 * lane : (lane >> 4) * F::QUAD + 8 * (lane & 15)));
    return x;
  }
  // Pairs of group g: of key i of the chunk, and of keys 4 q .. + 3.
  __device__ __forceinline__ uint32_t key_pair(int slot, int h, int g, int i) const {
    return reinterpret_cast<const uint32_t*>(lds + slot * STEP + 4 * CODES + h * PAIRS)[16 * g + i];
  }
  __device__ __forceinline__ u32x4 key_pairs(int slot, int h, int g, int q) const {
    return *reinterpret_cast<const u32x4*>(lds + slot * STEP + 4 * CODES + h * PAIRS + 64 * g + 16 * q);
  }
  // (0 times what a slot without a token holds is 0)
  __device__ __forceinline__ u32x4 value_pairs(int slot, int h, int g, int q, int key, int end) const {
    u32x4 x = *reinterpret_cast<const u32x4*>(lds + slot * STEP + 4 * CODES + (2 + h) * PAIRS + 64 * g + 16 * q);
    if (key + 16 > end) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = key + 4 * q + j < end ? x[j] : 0u;
    }
    return x;
  }
};

// 16 NC rows of queries.  Keys and values are brought to the element type in registers, m + s c in fp32 and one rounding, and
// probabilities are rounded to it as well, since both products are 16-bit matrix instructions (fp32 ones have a sixteenth of
// their rate); the sums that divide are of the unrounded ones.  Outputs are off by 0.0032 of their size in bf16 and 0.00036 in
// fp16, their own rounding included; fp32 arithmetic on m + s c leaves 0.0017 and 0.0002, nearly all of it that rounding.
template <bool BF16, int D, int NC, int DEPTH>
struct Q4Dequant {
  using E = Elem<BF16>;
  using F = Kv4<D>;
  static constexpr int NG = F::NG, NE = D / 16;

  static constexpr int STEPS = DEPTH;

  Q4Ring<D, DEPTH> ring;
  u32x4 qf[NC][NG];
  int pos[NC];                     // position of the lane's row
  int pos_min;                     // of all rows
  f32x4 O[NC][NE];
  float m_ref[NC], l_run[NC];      // base-2 reference; sum of the lane's probabilities
  bool ref_ok;

  __device__ __forceinline__ void start() {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int e = 0; e < NE; ++e) O[c][e] = f32x4{};
      m_ref[c] = -__builtin_inff();
      l_run[c] = 0.f;
    }
    ref_ok = false;
  }

  __device__ __forceinline__ void raise(const f32x4 (&S)[NC][2], float scale) {
    ref_ok = true;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float mx = S[c][0][0];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, S[c][h][j]);
      const float m_new = fmaxf(m_ref[c], quarters_max(mx) * scale);   // -inf stays -inf (scale > 0)
      const float alpha = m_ref[c] == -__builtin_inff() ? 1.f : fast_exp2(m_ref[c] - m_new);
      l_run[c] *= alpha;
#pragma unroll
      for (int e = 0; e < NE; ++e) O[c][e] *= alpha;
      m_ref[c] = m_new;
      ref_ok = ref_ok && !__any(m_new == -__builtin_inff());
    }
  }

  // A step whose codes and pairs are in `slot` of the ring, of two chunks from keys key0 and key1 on.
  __device__ __forceinline__ void step(int slot, int key0, int key1, int end, float scale) {
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
    const int key[2] = {key0, key1};
    f32x4 S[NC][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Words<NG> kw = ring.keys(slot, h);
#pragma unroll
      for (int c = 0; c < NC; ++c) S[c][h] = f32x4{};
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t st = ring.key_pair(slot, h, g, i);
        const float s = q4_scale<BF16>(st), m = q4_min<BF16>(st);
        const uint32_t lo = q4_low(kw.w[g]), hi = q4_high(kw.w[g]);
        const u32x4 kf = {q4_scaled<BF16, false>(lo, s, m), q4_scaled<BF16, true>(lo, s, m),
                          q4_scaled<BF16, false>(hi, s, m), q4_scaled<BF16, true>(hi, s, m)};
#pragma unroll
        for (int c = 0; c < NC; ++c) S[c][h] = E::mfma16(kf, qf[c][g], S[c][h]);
      }
      if (key[h] + 15 > pos_min) {              // keys past a row's position
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int lim = pos[c] - key[h] - 4 * q;
#pragma unroll
          for (int j = 0; j < 4; ++j) S[c][h][j] = j > lim ? -__builtin_inff() : S[c][h][j];
        }
      }
    }
    u32x4 P[NC];
    auto probs = [&](int c) {
      const float neg = m_ref[c] == -__builtin_inff() ? 0.f : -m_ref[c];
      float ls = 0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float p0 = fast_exp2(fmaf(S[c][x >> 1][2 * (x & 1)], scale, neg));
        const float p1 = fast_exp2(fmaf(S[c][x >> 1][2 * (x & 1) + 1], scale, neg));
        ls += p0 + p1;
        P[c][x] = E::pack2f(p0, p1);
      }
      return ls;
    };
    if (!ref_ok) raise(S, scale);
    float ls[NC];
    bool over = false;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      ls[c] = probs(c);
      over = over || !(ls[c] <= Q4_REFIT<BF16>);
    }
    if (__any(over)) {
      raise(S, scale);
#pragma unroll
      for (int c = 0; c < NC; ++c) ls[c] = probs(c);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) l_run[c] += ls[c];
    const Words<NG> vw[2] = {ring.values(slot, 0), ring.values(slot, 1)};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float s[2][4], m[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 st = ring.value_pairs(slot, h, g, q, key[h], end);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[h][j] = q4_scale<BF16>(st[j]), m[h][j] = q4_min<BF16>(st[j]);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {       // dims 32 g + 16 half + 0..15
        u32x4 vf;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t x = half ? q4_high(vw[h].w[g]) : q4_low(vw[h].w[g]);
          vf[2 * h] = q4_scaled<BF16, false>(x, s[h][0], m[h][0], s[h][1], m[h][1]);
          vf[2 * h + 1] = q4_scaled<BF16, true>(x, s[h][2], m[h][2], s[h][3], m[h][3]);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) O[c][2 * g + half] = E::mfma16(vf, P[c], O[c][2 * g + half]);
      }
    }
  }
};

// Few rows, codes multiplied as they are: with the groups g of the dims and c the codes,
//   q . k_t = sum_g s[t,g] (sum_{d in g} q_d c[t,d]) + m[t,g] sum_{d in g} q_d
//   o_d     = sum_t (p_t s[t,g]) c[t,d] + sum_t p_t m[t,g]              (d in g)
// so neither keys nor values are scaled one by one, and q c is exact.  The columns of the products are (group, row) pairs:
// the operand of column (g, r) is row r of the queries in group g and 0 in the others, so that one accumulator holds the
// partial scores of all groups, each lane needs the pairs of one group only, and a rotation over 16 lanes adds them up.  In
// the second product column (g, r) is p s[., g], of use in the dims of g.
// What rounds: p s, once, to bf16, for the 16-bit product; outputs are off by 0.0023 of their size in bf16, their own rounding
// of 0.0017 included.  Codes lie in 0 .. 15, so that would weigh with up to 15 s where half of it is the
// values' own; sum_t (p s) 7.5, of the rounded products (a row of ones more in the matrix product), is taken out
// and put back from the unrounded ones.  For fp16 the product is split in two bf16 parts instead, 16 bits in all.
template <bool BF16, int D, int NQ, int DEPTH>
struct Q4Fold {
  using E = Elem<BF16>;
  using F = Kv4<D>;
  static constexpr int NG = F::NG, NE = D / 16;
  static constexpr int RPS = 16 / NG;              // rows of a column set
  static constexpr int ROWS = RPS * NQ;
  static constexpr float REFIT = 65536.f;

  static constexpr int STEPS = DEPTH;

  Q4Ring<D, DEPTH> ring;
  u32x4 qz[NQ][NG];
  float qsum[NQ];                                  // of the lane's group and row
  int pos[NQ];                                     // position of the lane's row
  int pos_min;                                     // of all rows
  f32x4 O[NQ][NE], ones[NQ];
  float base[NQ];                                  // sum p m (+ 7.5 p s in bf16) of the lane's keys
  float m_ref[NQ], l_run[NQ];
  bool ref_ok;

  static __device__ __forceinline__ int group_of(int lane) { return (lane & 15) / RPS; }
  static __device__ __forceinline__ int row_of(int lane) { return (lane & 15) % RPS; }

  // The lane's row of set x: its query from element 0 on, and its position.
  __device__ __forceinline__ void set_query(int x, const elem_t* row, int position) {
    const int lane = threadIdx.x & 63, g = group_of(lane);
    const u32x4 v = *reinterpret_cast<const u32x4*>(row + 32 * g + 8 * (lane >> 4));
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += E::to_f32((elem_t)(v[e] & 0xffffu)) + E::to_f32((elem_t)(v[e] >> 16));
    qsum[x] = quarters_sum(sum);
    pos[x] = position;
#pragma unroll
    for (int y = 0; y < NG; ++y) qz[x][y] = y == g ? v : u32x4{0u, 0u, 0u, 0u};
  }

  __device__ __forceinline__ void start() {
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
#pragma unroll
      for (int e = 0; e < NE; ++e) O[x][e] = f32x4{};
      ones[x] = f32x4{};
      base[x] = l_run[x] = 0.f;
      m_ref[x] = -__builtin_inff();
    }
    ref_ok = false;
  }

  __device__ __forceinline__ void raise(const f32x4 (&S)[NQ][2], float scale) {
    ref_ok = true;
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      float mx = S[x][0][0];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, S[x][h][j]);
      // The lanes of a row's groups have its scores from sums in different orders: one reference for all of them.
      mx = over_groups<MAX>(mx);
      const float m_new = fmaxf(m_ref[x], quarters_max(mx) * scale);   // -inf stays -inf (scale > 0)
      const float alpha = m_ref[x] == -__builtin_inff() ? 1.f : fast_exp2(m_ref[x] - m_new);
      l_run[x] *= alpha;
      base[x] *= alpha;
      ones[x] *= alpha;
#pragma unroll
      for (int e = 0; e < NE; ++e) O[x][e] *= alpha;
      m_ref[x] = m_new;
      ref_ok = ref_ok && !__any(m_new == -__builtin_inff());
    }
  }

  // Sum or maximum over the lanes of a row's groups, in every one.
  template <int OP>
  static __device__ __forceinline__ float over_groups(float x) {
    auto op = [](float a, float b) { return OP == MAX ? fmaxf(a, b) : a + b; };
    if constexpr (NG == 4) x = op(x, dpp<0x124>(x));   // row_ror:4
    return op(x, dpp<0x128>(x));                       // row_ror:8
  }

  __device__ __forceinline__ void step(int slot, int key0, int key1, int end, float scale) {
    const int lane = threadIdx.x & 63, q = lane >> 4, group = group_of(lane);
    const int key[2] = {key0, key1};
    f32x4 S[NQ][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Words<NG> kw = ring.keys(slot, h);
#pragma unroll
      for (int x = 0; x < NQ; ++x) S[x][h] = f32x4{};
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t lo = q4_low(kw.w[g]), hi = q4_high(kw.w[g]);
        const u32x4 kf = BF16 ? u32x4{q4_pair_bf16<false>(lo), q4_pair_bf16<true>(lo), q4_pair_bf16<false>(hi), q4_pair_bf16<true>(hi)}
                              : u32x4{q4_pair_f16<false>(lo), q4_pair_f16<true>(lo), q4_pair_f16<false>(hi), q4_pair_f16<true>(hi)};
#pragma unroll
        for (int x = 0; x < NQ; ++x) S[x][h] = E::mfma16(kf, qz[x][g], S[x][h]);
      }
      const u32x4 ks = ring.key_pairs(slot, h, group, q);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float s = q4_scale<BF16>(ks[j]), m = q4_min<BF16>(ks[j]);
#pragma unroll
        for (int x = 0; x < NQ; ++x) S[x][h][j] = over_groups<SUM>(fmaf(s, S[x][h][j], m * qsum[x]));
      }
      if (key[h] + 15 > pos_min) {              // keys past a row's position
#pragma unroll
        for (int x = 0; x < NQ; ++x) {
          const int lim = pos[x] - key[h] - 4 * q;
#pragma unroll
          for (int j = 0; j < 4; ++j) S[x][h][j] = j > lim ? -__builtin_inff() : S[x][h][j];
        }
      }
    }
    float p[NQ][8];
    auto probs = [&](int x) {
      const float neg = m_ref[x] == -__builtin_inff() ? 0.f : -m_ref[x];
      float ls = 0.f;
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        p[x][y] = fast_exp2(fmaf(S[x][y >> 2][y & 3], scale, neg));
        ls += p[x][y];
      }
      return ls;
    };
    if (!ref_ok) raise(S, scale);
    float ls[NQ];
    bool over = false;
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      ls[x] = probs(x);
      over = over || !(ls[x] <= REFIT);
    }
    if (__any(over)) {
      raise(S, scale);
#pragma unroll
      for (int x = 0; x < NQ; ++x) ls[x] = probs(x);
    }
#pragma unroll
    for (int x = 0; x < NQ; ++x) l_run[x] += ls[x];
    // p s of the lane's group in the order of the operand, and p m.
    u32x4 P[NQ], R[NQ];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4 vs = ring.value_pairs(slot, h, group, q, key[h], end);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const float s0 = q4_scale<BF16>(vs[j]), s1 = q4_scale<BF16>(vs[j + 1]);
        const float m0 = q4_min<BF16>(vs[j]), m1 = q4_min<BF16>(vs[j + 1]);
#pragma unroll
        for (int x = 0; x < NQ; ++x) {
          const float p0 = p[x][4 * h + j], p1 = p[x][4 * h + j + 1];
          const float y0 = p0 * s0, y1 = p1 * s1;
          base[x] = fmaf(p0, m0, fmaf(p1, m1, base[x]));
          const uint32_t w = Elem<true>::pack2f(y0, y1);
          P[x][2 * h + (j >> 1)] = w;
          if constexpr (BF16)
            base[x] = fmaf(y0, 7.5f, fmaf(y1, 7.5f, base[x]));
          else
            R[x][2 * h + (j >> 1)] = Elem<true>::pack2f(y0 - __uint_as_float(w << 16), y1 - __uint_as_float(w & 0xffff0000u));
        }
      }
    }
    const Words<NG> vw[2] = {ring.values(slot, 0), ring.values(slot, 1)};
    constexpr uint32_t ONE2 = 0x3f803f80u;
#pragma unroll
    for (int x = 0; x < NQ; ++x)
      if constexpr (BF16) ones[x] = Elem<true>::mfma16(u32x4{ONE2, ONE2, ONE2, ONE2}, P[x], ones[x]);
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int half = 0; half < 2; ++half) {       // dims 32 g + 16 half + 0..15
        u32x4 vf;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t c = half ? q4_high(vw[h].w[g]) : q4_low(vw[h].w[g]);
          vf[2 * h] = q4_pair_bf16<false>(c);
          vf[2 * h + 1] = q4_pair_bf16<true>(c);
        }
#pragma unroll
        for (int x = 0; x < NQ; ++x) {
          O[x][2 * g + half] = Elem<true>::mfma16(vf, P[x], O[x][2 * g + half]);
          if constexpr (!BF16) O[x][2 * g + half] = Elem<true>::mfma16(vf, R[x], O[x][2 * g + half]);
        }
      }
  }

  // Dims 32 g + 16 half + 4 q .. + 3 of the lane's group g and row of set x.
  __device__ __forceinline__ void result(int x, f32x4 (&out)[2]) const {
    const int g = group_of(threadIdx.x & 63);
    const float b = quarters_sum(base[x]);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      out[half] = O[x][half];
#pragma unroll
      for (int y = 1; y < NG; ++y) out[half] = y == g ? O[x][2 * y + half] : out[half];
      if constexpr (BF16) out[half] = out[half] - 7.5f * ones[x] + b;
      else out[half] = out[half] + b;
    }
  }
};

// All steps of the wave.
template <class W>
__device__ __forceinline__ void q4_run(W& wave, const Q4Keys& ks, float scale) {
  constexpr int DEPTH = W::STEPS, LOADS = decltype(wave.ring)::LOADS;
  const int ns = ks.steps();
  if (ns == 0) return;
  Q4Window w;
  w.fill(ks, 0);
  for (int s = 0; s < min(ns, DEPTH - 1); ++s) wave.ring.issue(ks, w, s, s);
  int slot = 0;
#pragma unroll 1
  for (int s = 0; s < ns; ++s) {
    const int ahead = s + DEPTH - 1;
    if (ahead < ns) {
      if (ahead - w.base >= 32) w.fill(ks, s);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the slot's last step has been read
      wave.ring.issue(ks, w, ahead, slot == 0 ? DEPTH - 1 : slot - 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"i"((DEPTH - 1) * LOADS) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    wave.step(slot, w.key_of(s, 0), w.key_of(s, 1), ks.end, scale);
    slot = slot == DEPTH - 1 ? 0 : slot + 1;
  }
}

}  // namespace sa
