// Decode over the block-scaled cache, shared between its entry point (attention_int8.hip)
// and its kernels (decode_int8.hip), which cover head sizes up to 256 that are multiples of 16, pages
// of a multiple of 16 tokens and decode8_strides' layouts.
#pragma once

#include "decode_fp8.hpp"
#include "int8.hpp"

namespace rlt {

bool decode_i8_shape(int64_t hq, int64_t hkv, int64_t d, int64_t page);
// Bytes of the partials of rows of up to max_len tokens.
int64_t decode_i8_workspace(int64_t rows, int64_t max_len, int64_t hq, int64_t d);
int launch_decode_i8(const AttnI8Args& s, int dtype, void* ws, hipStream_t stream, const char* name);

}  // namespace rlt
