// The 8-bit KV cache: e4m3 codes with one power-of-two scale a (token, head)
// row of head_dim codes.  The scale travels as its e8m0 byte b (2^(b - 127), 255
// NaN).  Scales that are powers of two make every step but one exact: dividing a
// row by its scale, and multiplying a code by it, only move exponents, so a
// cached value carries the single rounding to 4 significant bits.  (An arbitrary
// fp32 scale would round twice more and gain nothing: a floating code has the
// same relative step at every magnitude.)
#pragma once

#include "common.hpp"

namespace rlt {

typedef float f32x2v __attribute__((ext_vector_type(2)));

// The byte of the smallest scale with amax <= 448 * 2^(b - 127), 448 = 1.75 * 2^8
// the largest code: amax = m * 2^k, m in [1, 2), needs 2^(k - 8), or twice that
// when m > 1.75.  amax is finite; 0 and subnormal rows get the smallest scale.
__device__ __forceinline__ uint32_t scale_byte(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int b = static_cast<int>(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(b < 0 ? 0 : b);
}
// 1 / scale of a byte that scale_byte() gives (at most 247).
__device__ __forceinline__ float inverse_scale(uint32_t b) { return __uint_as_float((254u - b) << 23); }

// The scale of any byte: 2^-127 of byte 0 is subnormal, 255 is NaN.
__device__ __forceinline__ float scale_value(uint32_t b) {
  const uint32_t u = max(b << 23, 0x00400000u);
  return __uint_as_float(b == 255u ? 0x7fc00000u : u);
}

// Sums of p V are kept kLift times as large, so that products with the smallest scales are
// normal numbers (in bf16, too).  What a key whose V scale has byte b adds to its candidate for
// the running maximum (log2 units): with p at most 2^8, p V stays below 2^96 a key, lifted, and
// its sum over 2^30 keys inside fp32.  0 up to kFreeScale, 2^55; no more than that, for beside a
// bias of x weights of 2^(x - 126) become 0.
constexpr float kLift = 0x1p24f;
constexpr uint32_t kFreeScale = 182;
__device__ __forceinline__ float value_bias(uint32_t b) {
  return static_cast<float>(max(static_cast<int>(b) - static_cast<int>(kFreeScale), 0));
}

// |x| where x is finite, 0 elsewhere: what a row's scale is taken over.
__device__ __forceinline__ float finite_abs(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return __uint_as_float(u < 0x7f800000u ? u : 0u);
}

// Two codes (low and high byte of the result's low half) of x, y times inv:
// rounded to nearest even; what is not finite becomes NaN, the type has no
// infinity.
__device__ __forceinline__ uint32_t codes2(float x, float y, float inv) {
  const float nan = __uint_as_float(0x7fc00000u);
  const float a = (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? nan : x * inv;
  const float b = (__float_as_uint(y) & 0x7f800000u) == 0x7f800000u ? nan : y * inv;
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false)) & 0xffffu;
}

__device__ __forceinline__ float code_value(uint8_t c) { return __builtin_amdgcn_cvt_f32_fp8(c, 0); }

// Largest over aligned groups of W lanes (group_sum's butterfly).
template <int W>
__device__ __forceinline__ float group_max(float x) {
  if constexpr (W >= 2) x = fmaxf(x, dpp<kDppXor1>(x));
  if constexpr (W >= 4) x = fmaxf(x, dpp<kDppXor2>(x));
  if constexpr (W >= 8) x = fmaxf(x, dpp<kDppHalfMirror>(x));
  if constexpr (W >= 16) x = fmaxf(x, dpp<kDppMirror>(x));
  if constexpr (W >= 32) x = fmaxf(x, xor_lane(x, 16));
  if constexpr (W >= 64) x = fmaxf(x, xor_lane(x, 32));
  return x;
}

// Limits of the attention calls: token counts and what is added to them stay inside 31
// bits, and the threads of a launch (blocks of up to 512) inside 32.
constexpr int64_t kMaxKeys = int64_t(1) << 30;
constexpr int64_t kMaxBlocks = (int64_t(1) << 24) - 1;
constexpr int64_t kMaxRows = (int64_t(1) << 23) - 1;

// Arguments of the attention kernels over an 8-bit cache (strides in elements).
struct Attn8Args {
  const void* q;
  int64_t q_row, q_head, q_dim;
  const uint8_t* k;
  const uint8_t* v;
  int64_t kv_block, kv_token, kv_head, kv_dim;
  const uint8_t* ks;
  const uint8_t* vs;
  int64_t s_block, s_token, s_head;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lens;
  const int32_t* cu;  // packed rows of several sequences; null: row r is sequence r's only one
  void* out;
  int64_t o_row, o_head, o_dim;
  int64_t rows;  // packed query rows
  int num_seqs, hq, hkv, d, page;
  int64_t num_blocks, max_len;  // max_len: table width * page, lengths are clamped to it
  float qscale;                 // softmax scale * log2(e)
};

// The block of table entry id: one outside the pool reads block 0, in bounds.
__device__ __forceinline__ int64_t block_of(const Attn8Args& a, int32_t id) {
  return id >= 0 && id < a.num_blocks ? id : 0;
}

// A sequence's key count, never past what its table covers.
__device__ __forceinline__ int sequence_length(const Attn8Args& a, int s) {
  const int64_t n = a.lens[s];
  return static_cast<int>(n < 0 ? 0 : n < a.max_len ? n : a.max_len);
}

// Attention of every row by the kernel for any shape (attention_fp8.hip).
int launch_attn8_generic(const Attn8Args& a, int dtype, hipStream_t stream, const char* name);

}  // namespace rlt
