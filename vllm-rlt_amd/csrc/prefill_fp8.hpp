// Prefill over the 8-bit cache, shared between its entry point (attention_fp8.hip)
// and its kernel (prefill_fp8.hip).
#pragma once

#include <algorithm>

#include "fp8.hpp"

namespace rlt {

bool prefill8_shape(int64_t d, int64_t page);
bool prefill8_layout(const Attn8Args& a);
// Bytes of the partials of cut sequences; ws null cuts none.
int64_t prefill8_workspace(int64_t rows, int64_t num_seqs, int64_t max_len, int64_t hq, int64_t d);
int launch_prefill8(const Attn8Args& a, int dtype, void* ws, hipStream_t stream, const char* name);

}  // namespace rlt
