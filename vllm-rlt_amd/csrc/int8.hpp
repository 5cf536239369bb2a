// The block-scaled 8-bit KV cache: signed codes, -127 to 127, with one fp32 scale
// for each block (a page of tokens) and KV head.  A cached value is code * scale,
// so it is off by at most half a step, 1/254 of its block's largest magnitude: a
// third of what e4m3 codes lose at the same bytes (rms, normal values), with a
// sixteenth of the scales.  A scale that is not finite makes its whole block NaN.
#pragma once

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

// scale * 2^-e.  Past fp32's largest number that number: a weight it multiplies is 0 there.
__device__ __forceinline__ float weight_scale(float scale, float e) {
  const float g = ldexpf(scale, -static_cast<int>(e));
  return g > 3.4028234664e38f ? 3.4028234664e38f : g;
}

constexpr float kNoExponent = -1024.f;  // e before any key

// Bytes of a partial's state: m, l and e, and a place that keeps them on 16 bytes.
struct __align__(16) PartState {
  float m, l, e, unused;
};

int launch_attn_i8_generic(const AttnI8Args& p, int dtype, hipStream_t stream, const char* name);

}  // namespace rlt
