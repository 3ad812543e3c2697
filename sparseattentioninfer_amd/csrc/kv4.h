// A page of a cache held in 4 bits, for one KV head: a block of page * D * 5 / 8 bytes.
//
// 32 dims of one token's head are a group, held as m + s c with codes c of 4 bits:
//   m = min x,   s = (max x - min x) / 15, toward zero to the element type,   c = min(floor((x - m) / s + 1/2), 15).
// x is of the element type (what a 16-bit cache would hold), so m is exact.  s is cut and not rounded, so that no value
// is read back past the group's largest.  A value is off by at most s / 2 or, past the code 15, by what the cut leaves of the
// range, max x - min x - 15 s: less than 15 s 2^-7 (bf16) and 15 s 2^-10 (fp16), which is less than s / 2, but 15 2^-24 where
// s is one of fp16's subnormal multiples of 2^-24.  A scale below 2^-126 (bf16) is taken for 0, and c for 0 with it: off by
// less than 15 2^-126.  Ranges and quotients are formed in fp32: one less than 2^-20 of itself below the border to the next s
// or c may be taken for the border, which moves the bound by that much.  A group with a NaN or an infinity has s = m = NaN.
//
// First the codes, page * D / 2 bytes; then (s, m) pairs of the element type, [D / 32][page].  The order of the codes is
// that of the matrix instructions' operands, so that attention takes them from memory to registers with 16-byte loads
// and no transposition, while every byte belongs to one token, so that single tokens can be written.
//   Keys (S^T = K Q^T: a lane holds 8 dims of a token): D / 2 bytes a token; the 32-bit word (D / 32) q + g holds dims
//     32 g + 8 q + e at bit 8 (e % 4) + 4 (e / 4), e < 8.  A lane's words of all groups are consecutive.
//   Values (O^T = V^T P^T: a lane holds tokens of one dim): four tokens share 2 D bytes; byte t % 4 of word
//     (D / 32) i + g of these holds dims 32 g + i (low) and 32 g + 16 + i (high) of token t, i < 16.
#pragma once

#include "sa_common.h"

namespace sa {

template <int D>
struct Kv4 {
  static constexpr int NG = D / 32;        // groups of a token's head
  static constexpr int ROW = D / 2;        // bytes of codes of a token
  static constexpr int QUAD = 2 * D;       // bytes of codes of four tokens
  static __device__ __host__ constexpr int stats_at(int page) { return page * ROW; }   // byte of the first pair
};

// Loads and words of a lane: NG of them, 8 or 16 bytes.
template <int NG>
struct Words {
  uint32_t w[NG];
  __device__ __forceinline__ void load(const uint8_t* p) {
    static_assert(NG == 2 || NG == 4, "head dim 64 or 128");
    if constexpr (NG == 4) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = v[i];
    } else {
      const u32x2 v = *reinterpret_cast<const u32x2*>(p);
      w[0] = v[0], w[1] = v[1];
    }
  }
};

// Scale and minimum of a pair.
template <bool BF16>
__device__ __forceinline__ float q4_scale(uint32_t st) {
  if constexpr (BF16) return __uint_as_float(st << 16);
  return Elem<false>::to_f32((elem_t)(st & 0xffffu));
}
template <bool BF16>
__device__ __forceinline__ float q4_min(uint32_t st) {
  if constexpr (BF16) return __uint_as_float(st & 0xffff0000u);
  return Elem<false>::to_f32((elem_t)(st >> 16));
}

// The codes in the low and in the high halves of a word's bytes.
__device__ __forceinline__ uint32_t q4_low(uint32_t w) { return w & 0x0f0f0f0fu; }
__device__ __forceinline__ uint32_t q4_high(uint32_t w) { return (w >> 4) & 0x0f0f0f0fu; }
// Byte e of codes as a number (v_cvt_f32_ubyte).
template <int E>
__device__ __forceinline__ float q4_code(uint32_t codes) { return (float)((codes >> (8 * E)) & 0xffu); }

// Two of four codes as fp32 and as 16-bit numbers, exact: a code in a byte is an e4m3 number of that many 2^-9, subnormals and the
// first binade together, so the conversion scales by 2^9.
template <bool HIGH>
__device__ __forceinline__ f32x2 q4_pair_f32(uint32_t codes) {
  return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8((int)codes, 512.f, HIGH);
}
// m + s c of two codes, rounded to the element type.
template <bool BF16, bool HIGH>
__device__ __forceinline__ uint32_t q4_scaled(uint32_t codes, float s, float m) {
  const f32x2 c = q4_pair_f32<HIGH>(codes);
  return Elem<BF16>::pack2f(fmaf(c[0], s, m), fmaf(c[1], s, m));
}
template <bool BF16, bool HIGH>      // the same with a scale and a minimum of its own for each
__device__ __forceinline__ uint32_t q4_scaled(uint32_t codes, float s0, float m0, float s1, float m1) {
  const f32x2 c = q4_pair_f32<HIGH>(codes);
  return Elem<BF16>::pack2f(fmaf(c[0], s0, m0), fmaf(c[1], s1, m1));
}
template <bool HIGH>
__device__ __forceinline__ uint32_t q4_pair_bf16(uint32_t codes) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)codes, 512.f, HIGH));
}
template <bool HIGH>
__device__ __forceinline__ uint32_t q4_pair_f16(uint32_t codes) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)codes, 512.f, HIGH));
}

}  // namespace sa
