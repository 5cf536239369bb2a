// The block-scaled 8-bit KV cache: signed codes, -127 to 127, with one fp32 scale
// for each block (a page of tokens) and KV head.  A cached value is code * scale.
// It is off by at most half a step, 1/254 of its block's largest magnitude, where the
// block was written in one call; by half a step more of each scale that it was rounded to
// since, where appends made the block's grow.  Rms of normal values in pages of 16 / 128,
// of theirs: 0.0083 / 0.0094 in one call, 0.0104 / 0.0122 token by token (up to five half
// steps), where e4m3 codes at the same bytes, with a scale for each token, lose 0.0265.  But
// a block's scale is its largest channel's: with four channels of 128 times 4 and
// tokens of different size it is 0.0230 / 0.0318 and 0.0268 / 0.0386.
// A scale that is not finite makes its whole block NaN.
#pragma once

#include <type_traits>

#include "attn8.hpp"

namespace rlt {

constexpr float kInverseLargest = 1.f / 127.f;  // of the largest code
constexpr float kSmallestScale = 0x1p-126f;  // the smallest normal number, whose inverse is finite as well

// The attention calls' arguments: a.s_block and a.s_head are the scales' strides, a.ks and a.vs unused.
struct AttnI8Args {
  Attn8Args a;
  const float* ks;
  const float* vs;
};

// Online softmax over values whose scales differ from block to block.  With x_j the
// scores in log2 units, a row keeps m, a whole number not much below its largest x, and
// sums l = sum 2^(x_j - m); and e, a whole number not much below the largest log2 of
// 2^(x_j - m) vs_j, and sums acc = sum w_j code_j with weights w_j = 2^(x_j - m) vs_j 2^-e.
// The result is acc / l * 2^e.  So a weight that goes into a product in 16 bits is near 1
// for the keys that matter, whatever their blocks' scales, and every change of m and e
// scales the sums by a power of two, exactly.  e is kept relative to m: m itself may be
// large, and their sum would then lose e.

// A block's scale, NaN where it is not finite.
__device__ __forceinline__ float block_scale(float scale) { return fmaf(scale, 0.f, scale); }

// The smallest whole number b with |scale| < 2^b, for any scale down to 0.
__device__ __forceinline__ float scale_exponent(float scale) {
  return static_cast<float>(static_cast<int>(__float_as_uint(scale) >> 23 & 255u) - 126);
}

// scale * 2^-e, NaN if that is.  Past fp32's largest number that number: a weight it multiplies is 0 there.
__device__ __forceinline__ float weight_scale(float scale, float e) {
  const float g = ldexpf(scale, -static_cast<int>(e));
  return __builtin_elementwise_minimum(g, 3.4028234664e38f);
}

constexpr float kNoExponent = -1024.f;  // e before any key

// Of weights in fp16: e puts the largest between 2^5 and 2^7 when it moves, and moves when one
// could pass 2^15.  So weights down to 2^-19 of the largest are normal numbers of the type.
constexpr float kUsualExponent = 7.f, kMostExponent = 15.f;

typedef _Float16 half2v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float f16_value(uint32_t bits) {
  return static_cast<float>(__builtin_bit_cast(f16, static_cast<uint16_t>(bits)));
}

// The four codes of a word as two words of bf16 or fp16 pairs, exact.  For fp16 a code plus 128 becomes
// the low bits of 1024 plus that, of which 1152 is taken away.
template <typename S>
__device__ __forceinline__ uint2 code_pairs(uint32_t word) {
  if constexpr (std::is_same_v<S, f16>) {
    const uint32_t x = word ^ 0x80808080u;
    const half2v shift = {static_cast<_Float16>(-1152.f), static_cast<_Float16>(-1152.f)};
    const half2v lo = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) + shift;
    const half2v hi = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) + shift;
    return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
  } else {
    uint32_t f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __float_as_uint(static_cast<float>(static_cast<int8_t>(word >> (8 * i))));
    // Their upper halves: the lower ones are 0.
    return make_uint2(__builtin_amdgcn_perm(f[1], f[0], 0x07060302u), __builtin_amdgcn_perm(f[3], f[2], 0x07060302u));
  }
}

// Bytes of a partial's state: m, l and e, and a place that keeps them on 16 bytes.
struct __align__(16) PartState {
  float m, l, e, unused;
};

int launch_attn_i8_generic(const AttnI8Args& p, int dtype, hipStream_t stream, const char* name);

}  // namespace rlt
