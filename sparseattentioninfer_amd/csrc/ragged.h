// Sequences of different lengths packed into one launch: new tokens of sequence b are rows cu[b] .. cu[b + 1] - 1
// of a packed tensor of N rows, and end its first kv_lens[b] cached tokens.  All of it is device memory, so a
// launch has as many workgroups as any lengths may need and each finds its own share.
#pragma once

#include "sa_common.h"

namespace sa {

// Lengths past this are taken for it, so positions stay well inside 32 bits.
constexpr int MAX_KV_LEN = 1 << 30;

// A launch of one workgroup per item has at most this many (2^32 threads of 256).
constexpr int64_t MAX_WORKGROUPS = (1 << 24) - 1;

struct Ragged {
  const int32_t* cu;
  const int32_t* kv_lens;
  int B;
  int64_t N;          // rows of the packed tensor

  // Rows [r0, r0 + n) of sequence b; offsets outside the tensor are clamped to it.
  __device__ __forceinline__ int rows(int b, int& r0) const {
    const int64_t lo = cu[b], hi = cu[b + 1];
    r0 = (int)(lo < 0 ? 0 : lo > N ? N : lo);
    const int r1 = (int)(hi < 0 ? 0 : hi > N ? N : hi);
    return r1 > r0 ? r1 - r0 : 0;
  }
  __device__ __forceinline__ int kv_len(int b) const { return min(max(kv_lens[b], 0), MAX_KV_LEN); }
};

// Sum of x over this lane and those before it, without LDS: four shifts within rows of 16 lanes, then the last
// lane of a row to the next and of the lower half to the upper.
__device__ __forceinline__ int scan_lanes(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return x;
}

// Sequence b and index `local` within it of item x, where sequence b has count(b) items.  Called by whole
// waves; 64 sequences are counted at a time.  False if x is past the last item.
template <class Count>
__device__ __forceinline__ bool find_item(int B, int x, Count count, int& b, int& local) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    const int c = b0 + lane < B ? count(b0 + lane) : 0;
    const int incl = scan_lanes(c);
    const uint64_t past = __builtin_amdgcn_ballot_w64(base + incl > x);
    if (past) {
      const int l = __builtin_ctzll(past);
      b = b0 + l;
      local = x - base - (__builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(c, l));
      return true;
    }
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

}  // namespace sa
