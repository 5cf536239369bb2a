// What the attention calls over 8-bit caches share, whatever the form of their
// scales: limits, arguments, and how a row finds its keys.
#pragma once

#include "common.hpp"

namespace rlt {

// Largest over aligned groups of W lanes (group_sum's butterfly).
template <int W>
__device__ __forceinline__ float group_max(float x) {
  if constexpr (W >= 2) x = fmaxf(x, dpp<kDppXor1>(x));
  if constexpr (W >= 4) x = fmaxf(x, dpp<kDppXor2>(x));
  if constexpr (W >= 8) x = fmaxf(x, dpp<kDppHalfMirror>(x));
  if constexpr (W >= 16) x = fmaxf(x, dpp<kDppMirror>(x));
  if constexpr (W >= 32) x = fmaxf(x, xor_lane(x, 16));
  if constexpr (W >= 64) x = fmaxf(x, xor_lane(x, 32));
  return x;
}

// x y, rounded also where the product is added to something.
__device__ __forceinline__ float rounded_product(float x, float y) {
#pragma clang fp contract(off)
  return x * y;
}

// Limits of the attention calls: token counts and what is added to them stay inside 31
// bits, and the threads of a launch (blocks of up to 512) inside 32.
constexpr int64_t kMaxKeys = int64_t(1) << 30;
constexpr int64_t kMaxBlocks = (int64_t(1) << 24) - 1;
constexpr int64_t kMaxRows = (int64_t(1) << 23) - 1;

// The kernels for any shape: elements of a head a lane, and waves a (row, query head).
constexpr int kPerLane = 8;
constexpr int kGenericWaves = 8;

// Arguments of the attention kernels over an 8-bit cache (strides in elements).
struct Attn8Args {
  const void* q;
  int64_t q_row, q_head, q_dim;
  const uint8_t* k;
  const uint8_t* v;
  int64_t kv_block, kv_token, kv_head, kv_dim;
  const uint8_t* ks;
  const uint8_t* vs;
  int64_t s_block, s_token, s_head;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lens;
  const int32_t* cu;  // packed rows of several sequences; null: row r is sequence r's only one
  void* out;
  int64_t o_row, o_head, o_dim;
  int64_t rows;  // packed query rows
  int num_seqs, hq, hkv, d, page;
  int64_t num_blocks, max_len;  // max_len: table width * page, lengths are clamped to it
  float qscale;                 // softmax scale * log2(e)
};

// The block of table entry id: one outside the pool reads block 0, in bounds.
__device__ __forceinline__ int64_t block_of(const Attn8Args& a, int32_t id) {
  return id >= 0 && id < a.num_blocks ? id : 0;
}

// A sequence's key count, never past what its table covers.
__device__ __forceinline__ int sequence_length(const Attn8Args& a, int s) {
  const int64_t n = a.lens[s];
  return static_cast<int>(n < 0 ? 0 : n < a.max_len ? n : a.max_len);
}

// Packed row `row` of a prefill (a.cu), or row `row` of a decode: its sequence and how many
// of its keys it sees.  False for a row of no sequence, which is left as it was.
__device__ __forceinline__ bool row_keys(const Attn8Args& a, int64_t row, int* seq, int* len) {
  if (!a.cu) {
    *seq = static_cast<int>(row);
    *len = sequence_length(a, *seq);
    return true;
  }
  int lo = 0, hi = a.num_seqs;  // the last sequence that begins at or before row
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid] <= row) lo = mid;
    else hi = mid;
  }
  if (row < a.cu[lo] || row >= a.cu[lo + 1]) return false;
  *seq = lo;
  const int64_t n = sequence_length(a, lo) - (a.cu[lo + 1] - 1 - row);
  *len = static_cast<int>(n < 0 ? 0 : n);
  return true;
}

// Checks what the attention calls share and fills the arguments (attention_fp8.hip).
int attn8_args(const char* name, const void* q, const int64_t* q_strides, const void* key_cache, const void* value_cache,
               const int64_t* kv_strides, const void* key_scales, const void* value_scales, const int64_t* scale_strides,
               const int32_t* tables, int64_t table_stride, int64_t width, const int32_t* lens, int64_t num_seqs, void* out,
               const int64_t* out_strides, int64_t rows, int64_t hq, int64_t hkv, int64_t d, int64_t page,
               int64_t num_blocks, float scale, int dtype, Attn8Args* a);

}  // namespace rlt
