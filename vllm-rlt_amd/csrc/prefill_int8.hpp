// Prefill over the block-scaled cache, shared between its entry point (attention_int8.hip)
// and its kernels (prefill_int8.hip), which cover head sizes up to 256 that are multiples of 16, pages
// of a power of two from 16 tokens on and prefill8_strides' layouts.
#pragma once

#include "int8.hpp"
#include "prefill_fp8.hpp"

namespace rlt {

bool prefill_i8_shape(int64_t d, int64_t page);
// Bytes of the partials of cut sequences; ws null cuts none.
int64_t prefill_i8_workspace(int64_t rows, int64_t num_seqs, int64_t max_len, int64_t hq, int64_t d);
int launch_prefill_i8(const AttnI8Args& s, int dtype, void* ws, hipStream_t stream, const char* name);

}  // namespace rlt
