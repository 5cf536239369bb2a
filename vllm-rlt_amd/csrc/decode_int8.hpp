// Decode over the block-scaled cache, shared between its entry point (attention_int8.hip)
// and its kernels (decode_int8.hip).  Shapes and layouts are decode8_shape's and decode8_layout's.
#pragma once

#include "decode_fp8.hpp"
#include "int8.hpp"

namespace rlt {

// Bytes of the partials of rows of up to max_len tokens.
int64_t decode_i8_workspace(int64_t rows, int64_t max_len, int64_t hq, int64_t d);
int launch_decode_i8(const AttnI8Args& s, int dtype, void* ws, hipStream_t stream, const char* name);

}  // namespace rlt
