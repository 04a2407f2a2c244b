// The 4-bit KV cache: format, layout and the small device helpers that its kernels share.
//
// Format.  A row (one token, one KV head, D channels) is cut into groups of G channels.  A group has a `low` (its
// smallest value) and a `scale`, both in the cache's 16-bit type, and a code 0 .. 15 per channel:
//     scale = r16((max - low) / 15)        code = rint((x - low) / scale)   (0 where scale is 0)
//     value = scale * code + low
// in fp32 with IEEE division, ties to even.  `low` is one of the row's own values, so it needs no rounding.  A group
// that holds an infinity or a NaN gets NaN as its scale: all of it reads back as NaN instead of as plausible numbers.
//
// Layout.  Everything of one (page, KV head) is contiguous, tokens in order, so that a wave that walks tokens of one
// head reads whole kilobytes (16 tokens x D / 2 bytes = 1 KiB per load instruction at D = 128):
//   k_codes  [pages, Hkv, page, D / 2]       A row is D / 8 dwords; dword lg * (D / 32) + s (lg < 4, s < D / 32) holds
//            channels 32 s + 8 lg .. + 7 - the eight that lane group lg feeds to step s of a 16x16x32 MFMA over the
//            head dim - so a lane's share of a row is one run.  Channel 2 n sits at bits 4 n, channel 2 n + 1 at
//            bits 16 + 4 n: one shift and one mask give a register with two neighbouring channels.
//   v_codes  [pages, Hkv, page / 4, 16, D / 64, 4]  16-bit units.  Unit (c, h, t) of four tokens holds channels
//            16 (4 h + n) + c at bits 4 n: lane c of the MFMA that multiplies V^T finds its channel of every
//            16-channel tile, for four tokens, in one run; neighbouring tokens are the two halves of a dword.
//   k_params, v_params  [pages, Hkv, D / G, page]   dwords: scale in the low half, low in the high half.
#pragma once
#include "tdist/common.hpp"

namespace tdist {
namespace kv4 {

struct Cache {
  uint8_t* k_codes;
  uint8_t* v_codes;
  uint32_t* k_params;
  uint32_t* v_params;
  int pages, kv_heads, page_size;
};

template <bool IS_BF16>
__device__ __forceinline__ float from16(uint32_t low16) {
  if constexpr (IS_BF16) {
    return __builtin_bit_cast(float, low16 << 16);
  } else {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)low16);
  }
}
template <bool IS_BF16>
__device__ __forceinline__ uint32_t to16(float f) {
  if constexpr (IS_BF16) {
    return __builtin_bit_cast(uint16_t, (__bf16)f);
  } else {
    return __builtin_bit_cast(uint16_t, (_Float16)f);
  }
}
template <bool IS_BF16>
__device__ __forceinline__ float scale_of(uint32_t param) { return from16<IS_BF16>(param & 0xffffu); }
template <bool IS_BF16>
__device__ __forceinline__ float low_of(uint32_t param) {
  if constexpr (IS_BF16) {
    return __builtin_bit_cast(float, param & 0xffff0000u);
  } else {
    return from16<false>(param >> 16);
  }
}

// Token `pos` of a sequence: its page, and its place in the page; page -1 for a position that the table has no page of
// the cache for (behind its end, or an entry that is not one of the `pages`).
struct Place {
  int page, off;
};
__device__ __forceinline__ Place place_of(const Cache& c, const int* table_row, long long pos, int max_pages) {
  if (pos < 0 || pos >= (long long)max_pages * c.page_size) return Place{-1, 0};
  const uint32_t i = (uint32_t)pos / (uint32_t)c.page_size;      // (an int32 offset plus an int32 count)
  const int page = table_row[i];
  return Place{page >= 0 && page < c.pages ? page : -1, (int)((uint32_t)pos - i * (uint32_t)c.page_size)};
}

// Between one lane's writes to LDS and another lane's reads of them, and between those and the next writes to the same place, in one
// wave.  A wave's LDS accesses are carried out in the order in which they are issued, so there is nothing to wait for and this is no
// instruction; what it does is to keep the compiler from issuing them in another order, which it may where it can tell that no lane
// meets its own address again.
__device__ __forceinline__ void lanes_meet() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

}  // namespace kv4
}  // namespace tdist
