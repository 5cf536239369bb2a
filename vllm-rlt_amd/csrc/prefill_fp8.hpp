// Prefill over the 8-bit cache, shared between its entry point (attention_fp8.hip)
// and its kernel (prefill_fp8.hip).
#pragma once

#include <algorithm>

#include "fp8.hpp"

namespace rlt {

bool prefill8_shape(int64_t d, int64_t page);
bool prefill8_layout(const Attn8Args& a);
int launch_prefill8(const Attn8Args& a, int dtype, hipStream_t stream, const char* name);

}  // namespace rlt
