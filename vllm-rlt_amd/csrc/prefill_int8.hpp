// Prefill over the block-scaled cache, shared between its entry point (attention_int8.hip)
// and its kernels (prefill_int8.hip).  Shapes and layouts are prefill8_shape's and prefill8_layout's.
#pragma once

#include "int8.hpp"
#include "prefill_fp8.hpp"

namespace rlt {

// Bytes of the partials of cut sequences; ws null cuts none.
int64_t prefill_i8_workspace(int64_t rows, int64_t num_seqs, int64_t max_len, int64_t hq, int64_t d);
int launch_prefill_i8(const AttnI8Args& s, int dtype, void* ws, hipStream_t stream, const char* name);

}  // namespace rlt
