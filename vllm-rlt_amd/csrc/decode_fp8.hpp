// Decode over the 8-bit cache, shared between its entry point (attention_fp8.hip)
// and its kernels (decode_fp8.hip).
#pragma once

#include <algorithm>

#include "fp8.hpp"

namespace rlt {

// Whether the split kernels cover the shape, and the layout of a call of it.
bool decode8_shape(int64_t hq, int64_t hkv, int64_t d, int64_t page);
bool decode8_layout(const Attn8Args& a);
// Bytes of the partials of rows of up to max_len tokens.
int64_t decode8_workspace(int64_t rows, int64_t max_len, int64_t hq, int64_t d);
int launch_decode8(const Attn8Args& a, int dtype, void* ws, hipStream_t stream, const char* name);

}  // namespace rlt
