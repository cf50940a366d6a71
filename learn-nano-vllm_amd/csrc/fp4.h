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
// of two (one byte) would leave up to half of the grid unused (rms error of N(0, 1) values: 0.101
// with this scale, 0.115 with the best rule for powers of two).  f16 rather than bf16: v_fma_mix takes it as it is.
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

// ---- long query ranges: the pages in f16, and the prefill kernel over them --------------------------
// A tile of 128 query rows reads every key 8 times less often than one of 16, and its matrix
// instructions leave no time to convert the codes once per wave.  So a pass converts a step's
// keys and values once, into pages of 256 tokens in the workspace, sequence after sequence.
constexpr int kFp4Page = 256;
// f16 pages of a bf16 model hold keys and values times 2^-3: 6 * 65504, the format's largest, fits.
// (An f16 model's own are held as they are, the largest cut to 65504.)
constexpr int kFp4KeyShift = 3;

struct Fp4Expand {
  const uint8_t *k_data, *v_data;
  const uint16_t *k_scale, *v_scale;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* cu_k;          // prefix sums of the keys; or, where lens is given:
  const int32_t* lens;          // the keys of every sequence of the batch, this part's from `first` on,
  int first, total_batch, n_query;
  int32_t *cu_q_out, *cu_k_out;  // whose prefix sums are written here (null: they are already)
  int batch, pages_per_seq, max_blocks, block_size, bs_shift, num_blocks, num_kv_heads;
  uint16_t *k_pages, *v_pages;  // [batch * pages_per_seq][kFp4Page][num_kv_heads][128]
  int32_t* tables;              // [batch][pages_per_seq]: the pages' numbers
  bool f16;                     // of an f16 model
};
int fp4_expand_launch(const Fp4Expand& p, hipStream_t stream);

// Varlen attention over such pages (varlen_prefill.hip); q and out are f16 or bf16.
struct Fp4Prefill {
  const void* q;
  int64_t q_stride_tok, q_stride_head, total_q;
  const void *k_pages, *v_pages;
  const int32_t *cu_q, *cu_k, *tables;
  int batch, max_seqlen_q, max_seqlen_k, pages_per_seq, num_q_heads, num_kv_heads;
  float scale;
  void* out;
  int64_t out_stride_tok, out_stride_head;
  void* workspace;
  size_t workspace_bytes;
  bool f16;
};
int fp4_prefill_launch(const Fp4Prefill& p, hipStream_t stream);
