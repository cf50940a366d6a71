// Internal: the 4-bit key/value cache (its layout and conversions).  Not part of the C ABI.
//
// Per layer, for keys and for values, with D = head_dim and P = block_size:
//   data   uint8 [num_blocks][num_kv_heads][P][D / 2]    two e2m1 codes a byte, lower nibble first
//   scale  f16   [num_blocks][num_kv_heads][D / 32][P]
// A (page, head) is one block of memory: what the attention of a kv head streams is contiguous,
// which the [slot][head] order of the 16-bit caches would break into pieces of D / 2 bytes.
//
// e2m1: sign, then 0, 0.5, 1, 1.5, 2, 3, 4, 6: what gfx950 converts to bf16 and f16, two
// codes per instruction and exactly.  The scale of 32 dimensions is f16(min(max|x| / 6, 65504)):
// 16 bits of it cost 0.5 bit per value, and keep the grid's top at the largest value, where a power
// of two (one byte) would leave up to half of the grid unused (rms error of N(0, 1) values: 0.094
// with this scale, 0.125 with powers of two).  f16 rather than bf16: v_fma_mix takes it as it is.
//
// A row of values holds its dimensions in order.  A row of keys holds them in units of 8
// (4 bytes): unit 32 s + 8 g .. + 7 at place (D / 32) g + s, so that the 16 (D = 64: 8) bytes that
// lane group g of a 16x16x32 MFMA loads are its operands of the D / 32 steps, step s being group s.
#pragma once

#include "nvk_common.h"

constexpr int kFp4Group = 32;  // dimensions per scale

// The 8 codes of a word as 8 elements of T (bf16 or f16), in order.
template <bool F16>
NVK_DEVICE typename NvkElt<F16>::vec8 fp4_unpack(uint32_t w) {
  nvk_u32x4 v;
  if constexpr (F16) {
    v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 0));
    v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 1));
    v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 2));
    v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 3));
  } else {
    v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 0));
    v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 1));
    v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 2));
    v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 3));
  }
  return __builtin_bit_cast(typename NvkElt<F16>::vec8, v);
}

// Place of the 8-dimension unit u of a row of HD dimensions.
template <int HD, bool KEYS>
NVK_DEVICE int fp4_place(int u) {
  return KEYS ? (HD / 32) * (u & 3) + (u >> 2) : u;
}
