// Decode over the 8-bit cache, shared between its entry point (attention_fp8.hip)
// and its kernels (decode_fp8.hip: head_dim 64 with one query head a KV head on the vector
// units, and the merge; decode_mfma_fp8.hip: the others on the matrix cores).
#pragma once

#include <algorithm>

#include "fp8.hpp"

namespace rlt {

constexpr int kDecode8MaxSplits = 64;

// The splits of a row of len keys: `base` tokens each, doubled until kDecode8MaxSplits
// cover the row.
__host__ __device__ inline void decode8_split_plan(int64_t len, int base, int* split_len, int* nsplit) {
  int64_t per = base;
  while (per * kDecode8MaxSplits < len) per <<= 1;
  *split_len = static_cast<int>(per);
  *nsplit = static_cast<int>(len > 0 ? (len + per - 1) / per : 1);
}
// The most splits that a row of up to max_len keys has: not those of max_len itself, whose
// splits may be twice as long as a shorter row's.
inline int decode8_most_splits(int64_t max_len, int base) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kDecode8MaxSplits, (max_len + base - 1) / base)));
}

struct Decode8Args {
  Attn8Args a;
  float* ws_acc;   // [rows][hkv][splits][G][D]
  float2* ws_ml;   // [rows][hkv][splits][G], max in log2 units and sum
  int base;        // tokens of a split (decode8_split_plan)
  int splits;      // most splits of a row inside the tables' width
  int split_slots; // split-dimension workgroups launched; each walks every split_slots-th split
  int hpw;         // heads a wave
  int xcd;         // the heads of a (split, row) share an XCD
  int q_vec;       // q rows are 16-byte aligned, dims together
};

// Whether the split kernels cover the shape, and the layout of a call of it.
bool decode8_shape(int64_t hq, int64_t hkv, int64_t d, int64_t page);
bool decode8_layout(const Attn8Args& a);
// Bytes of the partials of rows of up to max_len tokens.
int64_t decode8_workspace(int64_t rows, int64_t max_len, int64_t hq, int64_t hkv, int64_t d);
int launch_decode8(const Attn8Args& a, int dtype, void* ws, hipStream_t stream, const char* name);

// The split pass on the matrix cores: workgroups are (row, KV head, 16 of its query
// heads, split).
constexpr int kMfmaSplit = 512;
void launch_decode8_mfma(const Decode8Args& p, int dtype, hipStream_t stream);

}  // namespace rlt
