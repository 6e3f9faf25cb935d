// K/V caches held in 4 bits: the format of a token's row, and the conversions every kernel of such caches uses
// (fp4_rows.hip writes and reads back rows, fp4_attention.hip attends over them).
//
// A row (K or V of one token, bytes) is
//     num_kv_heads x 64 bytes of values, two to a byte, the lower dimension in the low four bits;
//     num_kv_heads x 4 scale bytes, one per 32 dimensions;
//     0 to 15 bytes up to a multiple of 16, never read or written.
// A value is a sign, two bits of exponent and one of mantissa -- 0, 0.5, 1, 1.5, 2, 3, 4 or 6 -- times
// 2^(scale byte - 127); scale byte 255 makes its 32 values NaN, 0, 253 and 254 do not occur. Every value is exact in
// bf16 (v_cvt_scalef32_pk_bf16_fp4 applies the scale's exponent as it converts).
// Token-major rows keep a page one run of bytes whose first n tokens are its first n rows, which is what the page
// operators (kv_pages.hip) copy.
#pragma once

#include "common.h"

namespace pk {

constexpr int kFp4HeadBytes = kHeadDim / 2;   // values of one kv head
constexpr int kFp4HeadScales = kHeadDim / 32;  // its scale bytes
constexpr int kFp4MaxScale = 252;              // the largest scale byte of finite values
constexpr int kFp4ScaleNaN = 255;
constexpr int kFp4MaxHeads = 255;

// Bytes of a token's row.
inline int32_t fp4_row_bytes(int32_t num_kv_heads) {
  return (num_kv_heads * (kFp4HeadBytes + kFp4HeadScales) + 15) / 16 * 16;
}

// Scale byte of 32 values whose largest magnitude has the bf16 bits `top` (sign cleared): the smallest power of
// two s with top <= 7 s. Up to 7 s the largest value rounds to 6 s with an error of at most s, which is what the
// step of 2 s between 4 s and 6 s costs anyway; with the next smaller s it would lose more than a rounding does.
// 2^-126 .. 2^125: the smallest normal scale, and the largest one whose 6 s is finite. Infinities and NaN: 255.
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t top) {
  const int e = (int)(top >> 7) - 2 + ((top & 0x7f) > 0x60 ? 1 : 0);  // 0x60: a mantissa of 1.75
  return top >= 0x7f80 ? kFp4ScaleNaN : (uint32_t)min(max(e, 1), kFp4MaxScale);
}

typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 fp4_bf16x2;

// Two fp32 values to a packed bf16 pair, rounded to nearest even in one instruction.
__device__ __forceinline__ uint32_t fp4_pack_bf16(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, fp4_bf16x2));
}

// The scale of a scale byte as v_cvt_scalef32_* take it: they use its exponent alone, and an exponent of all
// ones gives NaN.
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// 8 bf16 values (four packed pairs) to 8 four-bit values: divided by the scale, rounded to nearest with ties to
// even, at most 6.
__device__ __forceinline__ uint32_t fp4_pack8(const uint4 w, uint32_t scale_byte) {
  const float s = fp4_scale(scale_byte);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(fp4_bf16x2, w.x), s, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(fp4_bf16x2, w.y), s, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(fp4_bf16x2, w.z), s, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(fp4_bf16x2, w.w), s, 3);
  return scale_byte == kFp4ScaleNaN ? 0 : r;
}

// Byte kByte of w, two four-bit values, to a packed pair of bf16.
template <int kByte>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, kByte));
}

__device__ __forceinline__ uint4 fp4_unpack8(uint32_t w, float scale) {
  return make_uint4(fp4_pair<0>(w, scale), fp4_pair<1>(w, scale), fp4_pair<2>(w, scale), fp4_pair<3>(w, scale));
}

// Rows of a step's tokens into 4-bit caches.
struct Fp4StoreArgs {
  const uint16_t* key;           // (N, Hkv, D) bf16, row strides in elements
  int64_t key_stride;
  const uint16_t* value;
  int64_t value_stride;
  uint8_t* k_cache;              // slot s at s * row_bytes
  uint8_t* v_cache;
  const int32_t* slot_mapping;
  int32_t num_tokens, num_kv_heads, row_bytes;
  int64_t num_slots;             // slots outside [0, num_slots) are passed over
};
struct Fp4AppendArgs {
  const uint16_t* qkv;           // (N, (Hq + 2 Hkv) * D) bf16
  int64_t qkv_stride;
  const int64_t* positions;
  const float* cos_sin;          // (max_position, D): cos in [0, D/2), sin in [D/2, D)
  int64_t max_position;
  const uint16_t* q_weight;      // (D,) bf16 or nullptr (no norm)
  const uint16_t* k_weight;
  float eps;
  int32_t num_tokens, num_heads, num_kv_heads, row_bytes;
  uint16_t* q_out;               // (N, Hq, D)
  int64_t q_out_stride;
  uint16_t* k_out;               // (N, Hkv, D) the stored rows' values, or nullptr
  int64_t k_out_stride;
  uint16_t* v_out;
  int64_t v_out_stride;
  uint8_t* k_cache;
  uint8_t* v_cache;
  const int32_t* slot_mapping;
  int64_t num_slots;
};
struct Fp4GatherArgs {
  const uint8_t* cache;
  int64_t block_stride;          // bytes
  int32_t num_blocks, block_size, num_kv_heads, row_bytes;
  const int32_t* block_table;
  int32_t bt_stride;
  const int32_t* cu_k;
  int32_t num_seqs, max_seqlen_k;
  int64_t num_rows;              // of dst
  uint16_t* dst;                 // (num_rows, Hkv, D) bf16
};
hipError_t launch_store_fp4(const Fp4StoreArgs& a, hipStream_t stream);
hipError_t launch_append_fp4(const Fp4AppendArgs& a, hipStream_t stream);
hipError_t launch_gather_fp4(const Fp4GatherArgs& a, hipStream_t stream);

// Attention over 4-bit caches (fp4_attention.hip).
struct Fp4AttnArgs {
  const uint16_t* q;             // (N, Hq, D) bf16
  int64_t q_stride;
  const uint8_t* k;
  const uint8_t* v;
  int64_t k_block, v_block;      // bytes from block to block
  int32_t row_bytes, block_size, num_blocks;
  const int32_t* block_table;
  int32_t bt_stride;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int32_t num_seqs, max_seqlen_q, max_seqlen_k;
  int64_t num_rows;              // of q and out: rows past them are not computed
  int32_t num_heads, num_kv_heads;
  int32_t group_shift;           // log2(num_heads / num_kv_heads)
  float scale_log2;              // softmax_scale * log2(e)
  int32_t causal;
  uint16_t* out;                 // (N, Hq, D) bf16
  int64_t out_stride;
  void* workspace;
};
// Launch shapes of a call, a function of its bounds; runs and columns of the partial results.
struct Fp4AttnPlan {
  int32_t few_runs;              // work-groups over the sequences of few rows (per group of kv heads)
  int32_t few_heads;             // kv heads of one of them
  int32_t few_slots;             // the next power of two
  int32_t few_cols;              // columns (rows x query heads) of a kv head's partial result
  int32_t many_runs;             // work-groups over the sequences of more rows, 0: there can be none
  int64_t many_tiles;            // about as many tiles of rows (of all kv heads) as they have
  size_t few_bytes, many_bytes;  // partial results
  int64_t steps;                 // of a line at most, by the call's bounds: those of the sequences of few rows, or of
  int32_t step_keys;             // more rows on one kv head, whichever are more; keys of one of them
};
Fp4AttnPlan fp4_attention_plan(int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads, int32_t max_seqlen_q,
                               int32_t max_seqlen_k, int64_t num_rows);
hipError_t launch_fp4_attention(const Fp4AttnArgs& a, const Fp4AttnPlan& p, hipStream_t stream);

}  // namespace pk
