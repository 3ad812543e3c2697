// Attention of one wave over keys held in 4 bits (gfx950): keys and values go from memory to the operands of
// v_mfma 16x16x32 in registers, without LDS.
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

// Row references are raised when a lane's probabilities of a step sum past this: no probability then exceeds 2^16 in
// bf16 (2^15 in fp16, whose largest is 65,504).
template <bool BF16>
constexpr float Q4_REFIT = BF16 ? 65536.f : 32768.f;

// 16 NC rows of queries.  Keys and values are brought to the element type in registers: m + s c in fp32, one rounding.
template <bool BF16, int D, int NC>
struct Q4Dequant {
  using E = Elem<BF16>;
  using F = Kv4<D>;
  static constexpr int NG = F::NG, NE = D / 16;

  struct Chunk {
    Words<NG> k, v;
    uint32_t ks[NG];
    u32x4 vs[NG];
    int key;
  };

  u32x4 qf[NC][NG];
  int pos[NC];                     // position of the lane's row
  int pos_min;                     // of all rows
  f32x4 O[NC][NE];
  float m_ref[NC], l_run[NC];      // base-2 reference; sum of the lane's probabilities
  bool ref_ok;

  static __device__ __forceinline__ void load(Chunk& c, const Q4Keys& ks, const Q4Window& w, int step, int h) {
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
    const int slot = w.slot_of(step, h);
    const int64_t off = w.off_of(step, h);
    c.key = w.key_of(step, h);
    const uint8_t *kb = ks.k + off, *vb = ks.v + off;
    c.k.load(kb + slot * F::ROW + (i * F::ROW + 4 * NG * q));
    c.v.load(vb + slot * F::ROW + (q * F::QUAD + 4 * NG * i));
    const int st = F::stats_at(ks.page) + 4 * slot;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      c.ks[g] = *reinterpret_cast<const uint32_t*>(kb + st + 4 * g * ks.page + 4 * i);
      c.vs[g] = *reinterpret_cast<const u32x4*>(vb + st + 4 * g * ks.page + 16 * q);
    }
  }

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

  __device__ __forceinline__ void step(const Chunk (&ch)[2], int end, float scale) {
    const int lane = threadIdx.x & 63, q = lane >> 4;
    f32x4 S[NC][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int c = 0; c < NC; ++c) S[c][h] = f32x4{};
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float s = q4_scale<BF16>(ch[h].ks[g]), m = q4_min<BF16>(ch[h].ks[g]);
        const uint32_t lo = q4_low(ch[h].k.w[g]), hi = q4_high(ch[h].k.w[g]);
        const u32x4 kf = {E::pack2f(fmaf(q4_code<0>(lo), s, m), fmaf(q4_code<1>(lo), s, m)),
                          E::pack2f(fmaf(q4_code<2>(lo), s, m), fmaf(q4_code<3>(lo), s, m)),
                          E::pack2f(fmaf(q4_code<0>(hi), s, m), fmaf(q4_code<1>(hi), s, m)),
                          E::pack2f(fmaf(q4_code<2>(hi), s, m), fmaf(q4_code<3>(hi), s, m))};
#pragma unroll
        for (int c = 0; c < NC; ++c) S[c][h] = E::mfma16(kf, qf[c][g], S[c][h]);
      }
      if (ch[h].key + 15 > pos_min) {              // keys past a row's position
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int lim = pos[c] - ch[h].key - 4 * q;
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
    u32x4 vs[2][NG];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int live = end - ch[h].key - 4 * q;    // of the lane's four keys, those that are there
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        vs[h][g] = ch[h].vs[g];
        if (ch[h].key + 16 > end) {                // 0 times what a slot without a token holds is 0
#pragma unroll
          for (int j = 0; j < 4; ++j) vs[h][g][j] = j < live ? vs[h][g][j] : 0u;
        }
      }
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float s[2][4], m[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[h][j] = q4_scale<BF16>(vs[h][g][j]), m[h][j] = q4_min<BF16>(vs[h][g][j]);
#pragma unroll
      for (int half = 0; half < 2; ++half) {       // dims 32 g + 16 half + 0..15
        u32x4 vf;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t x = half ? q4_high(ch[h].v.w[g]) : q4_low(ch[h].v.w[g]);
          vf[2 * h] = E::pack2f(fmaf(q4_code<0>(x), s[h][0], m[h][0]), fmaf(q4_code<1>(x), s[h][1], m[h][1]));
          vf[2 * h + 1] = E::pack2f(fmaf(q4_code<2>(x), s[h][2], m[h][2]), fmaf(q4_code<3>(x), s[h][3], m[h][3]));
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) O[c][2 * g + half] = E::mfma16(vf, P[c], O[c][2 * g + half]);
      }
    }
  }

  // All steps of the wave; the loads of the next are in flight during one.
  __device__ __forceinline__ void run(const Q4Keys& ks, float scale) {
    const int ns = ks.steps();
    if (ns == 0) return;
    Q4Window w;
    w.fill(ks, 0);
    Chunk a[2], b[2];
    auto fetch = [&](Chunk (&ch)[2], int s) {
      if (s - w.base >= 32) w.fill(ks, s);
      load(ch[0], ks, w, s, 0);
      load(ch[1], ks, w, s, 1);
    };
    fetch(a, 0);
#pragma unroll 1
    for (int s = 0; s < ns; s += 2) {
      if (s + 1 < ns) fetch(b, s + 1);
      step(a, ks.end, scale);
      if (s + 1 >= ns) break;
      if (s + 2 < ns) fetch(a, s + 2);
      step(b, ks.end, scale);
    }
  }
};

}  // namespace sa
