// Staged K/V tiles of the matrix-core attention kernels: direct global -> LDS loads, the layout of a tile in
// LDS and its fragment reads, and reductions over the lanes of a wave.
#pragma once

#include "sa_common.h"

namespace sa {

// Sum / max of a value over lanes l and l ^ 32, in every lane: one v_permlane32_swap of the
// value with itself puts the lower half's values in one result and the upper half's in the other.
__device__ __forceinline__ float halves_sum(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ float halves_max(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

// Lane l's value from lane l ^ 1, l ^ 2, and the mirror images of l in its 8 and 16 lanes.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, true));
}

// Sum / max of a value over the wave, in every lane, without LDS.
__device__ __forceinline__ float wave_sum(float x) {
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  x += dpp<0x141>(x);
  x += dpp<0x140>(x);
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return halves_sum(__uint_as_float(s[0]) + __uint_as_float(s[1]));
}
__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, dpp<0xB1>(x));
  x = fmaxf(x, dpp<0x4E>(x));
  x = fmaxf(x, dpp<0x141>(x));
  x = fmaxf(x, dpp<0x140>(x));
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return halves_max(fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1])));
}

__device__ __forceinline__ __attribute__((address_space(3))) void* lds_ptr(const void* p) {
  return (__attribute__((address_space(3))) void*)(p);
}

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)lds_ptr(p);
}

// Direct global -> LDS loads of 16 bytes per lane (global_load_lds_dwordx4: lane l's bytes
// land at the LDS address in M0 plus 16 l).  They are issued from assembly so that the
// compiler does not make every later LDS read wait for them (it cannot tell the staging
// buffers apart); callers wait with wait_dma() before the barrier that publishes the data.
// M0 is written one instruction ahead of its use by the load, as the hardware requires.
//
// Uniform base address `sbase` plus a per-lane 32-bit byte offset.
__device__ __forceinline__ void load_lds16(const void* sbase, uint32_t voff, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, %1"
      :
      : "v"(voff), "s"(sbase), "s"(lds)
      : "memory", "m0");
}

// Uniform base plus per-lane offset plus the immediate IMM (a signed 13-bit field of the
// instruction), so consecutive loads from one base need no address arithmetic.  The
// instruction adds IMM to the LDS address as well (M0 + IMM + 16 l), so M0 is lds - IMM.
template <int IMM>
__device__ __forceinline__ void load_lds16_at(const void* sbase, uint32_t voff, uint32_t lds) {
  static_assert(IMM >= -4096 && IMM < 4096, "global instruction offsets are 13-bit signed");
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, %1 offset:%3"
      :
      : "v"(voff), "s"(sbase), "s"(lds - (uint32_t)IMM), "i"(IMM)
      : "memory", "m0");
}

// Per-lane 64-bit address.
__device__ __forceinline__ void load_lds16(const void* vaddr, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, off"
      :
      : "v"(vaddr), "s"(lds)
      : "memory", "m0");
}

// Waits for the calling wave's direct loads (and any other vector memory access).
__device__ __forceinline__ void wait_dma() { __builtin_amdgcn_s_waitcnt(0x0F70); }  // vmcnt(0)

// Layout of a staged tile of 64 key rows and its fragment reads, the same for every head dim and type.
struct StagedTile {
  // LDS row of key k within a staged K tile: bits 2 and 3 swapped.  With this order the S^T
  // accumulator gives each lane half 8 consecutive keys per 16-key chunk, the k-order of the
  // V^T operand.
  static __device__ __forceinline__ int krow(int k) {
    return (k & ~12) | ((k & 4) << 1) | ((k & 8) >> 1);
  }

  // Column of lane l's 16 bytes within its 32-column group in one wave-wide direct load.
  static __device__ __forceinline__ int dma_col(int lane) { return 8 * ((lane & 3) ^ ((lane >> 4) & 3)); }

  // Per-lane byte offsets of the fragment reads (tile-invariant).  The K offset of odd
  // chunk pairs is k0 ^ 32 and the V^T offset of the upper key quad is (v0 + 256) ^ 16.
  struct Frag {
    int k0, v0;
    __device__ __forceinline__ Frag(int lane) {
      const int l32 = lane & 31, g = lane >> 5;
      k0 = l32 * 64 + 16 * (g ^ ((l32 >> 2) & 3));
      const int i = lane & 15, G = lane >> 4;
      const int c4 = 2 * (G & 1) + ((i >> 1) & 1);
      v0 = (8 * g + (i >> 2)) * 64 + 16 * (c4 ^ (2 * g)) + 8 * (i & 1);
    }
  };

  // A operand of S^T = K Q^T: row 32j + l32 of the staged K tile (key krow of it),
  // columns 16cc + 8g .. +7.
  static __device__ __forceinline__ u32x4 kfrag(const char* cK, const Frag& f, int j, int cc) {
    const int off = (cc & 1) ? (f.k0 ^ 32) : f.k0;
    return *reinterpret_cast<const u32x4*>(cK + 4096 * (cc >> 1) + 2048 * j + off);
  }

  static __device__ __forceinline__ u32x2 ds_tr16(const char* p) {
    typedef short v4i16 __attribute__((ext_vector_type(4)));
    const v4i16 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)(p));
    return __builtin_bit_cast(u32x2, r);
  }

  // A operand of O^T = V^T P^T: lane l holds d = 32dt + l32 of keys 32j + 16h + 8g + 0..7.
  // ds_read_b64_tr_b16 gives lane i of each 16-lane group element e = the (i & 3)-th value
  // at the address of lane 4e + (i >> 2); each lane addresses key (i >> 2) of a 4-key quad
  // at columns 4(i & 3) of its 16-column group, so lane i receives column i of 4 keys.
  static __device__ __forceinline__ u32x4 vfrag(const char* cV, const Frag& f, int j, int h, int dt) {
    const char* p = cV + 4096 * dt + 2048 * j + 1024 * h;
    const u32x2 lo = ds_tr16(p + f.v0);
    const u32x2 hi = ds_tr16(p + ((f.v0 + 256) ^ 16));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  }
};

}  // namespace sa
