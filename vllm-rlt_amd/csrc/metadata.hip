// GPU-resident routing metadata: per-row write addresses, context lengths and
// depth-resolved block tables built on the device from compact
// (slot, depth, position) descriptors, plus the packed-prefill staging and
// expansion.  All integer work; results are bit-exact by construction.
#include <algorithm>

#include "common.hpp"

namespace rlt {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kRound = 1024;  // workgroups that run at once, four a CU

struct DecodeMetaArgs {
  const int64_t* desc;
  const int32_t* tables;
  int64_t num_slots, table_width, planes, page;
  int64_t count;
  int64_t* slots;
  int64_t* positions;
  int32_t* lengths;
  int64_t* blocks;
  int64_t* offsets;
  int32_t* out_tables;
  int64_t out_stride, out_width;
};

// grid (size): one workgroup per output row; padding rows (row >= count)
// get slot = pos = length = 0, no write address, and an all-zero table row.
// A descriptor that points outside the tables is treated as padding after its
// slot and position are recorded, so no table read leaves the tables.
__global__ __launch_bounds__(kThreads) void decode_metadata_kernel(DecodeMetaArgs a) {
  const int64_t row = blockIdx.x;
  const bool real = row < a.count;
  const int64_t slot = real ? a.desc[3 * row] : 0;
  const int64_t depth = real ? a.desc[3 * row + 1] : 0;
  const int64_t pos = real ? a.desc[3 * row + 2] : 0;
  const int64_t plane = a.planes > 1 ? depth : 0;
  const bool valid = real && slot >= 0 && slot < a.num_slots && plane >= 0 && plane < a.planes && pos >= 0 &&
                     pos / a.page < a.table_width;
  const int32_t* src = a.tables + (valid ? (slot * a.planes + plane) * a.table_width : 0);
  if (threadIdx.x == 0) {
    a.slots[row] = slot;
    a.positions[row] = pos;
    a.lengths[row] = valid ? static_cast<int32_t>(pos + 1) : 0;
    if (valid) {
      a.blocks[row] = src[pos / a.page];
      a.offsets[row] = pos % a.page;
    }
  }
  int32_t* dst = a.out_tables + row * a.out_stride;
  for (int64_t c = threadIdx.x; c < a.out_width; c += kThreads) dst[c] = valid ? src[c] : 0;
}

__global__ __launch_bounds__(kThreads) void stage_prefill_kernel(const int64_t* src, int64_t* dst, int32_t* dst32,
                                                               int64_t n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= n) return;
  const int64_t x = src[i];
  dst[i] = x;
  dst32[i] = static_cast<int32_t>(x);
}

// Entries whose (sequence, page) fall outside the tables get block -1.
__global__ __launch_bounds__(kThreads) void expand_prefill_kernel(const int64_t* positions, const int64_t* sequences,
                                                                const int32_t* tables, int64_t num_seqs, int64_t width,
                                                                int64_t page, int64_t* blocks, int64_t* offsets,
                                                                int64_t n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= n) return;
  const int64_t pos = positions[i];
  const int64_t seq = sequences[i];
  const bool ok = seq >= 0 && seq < num_seqs && pos >= 0 && pos / page < width;
  blocks[i] = ok ? tables[seq * width + pos / page] : -1;
  offsets[i] = pos % page;
}

// Packed chunks from (slot, depth, start, tokens) descriptors: sequence i takes
// `tokens` new tokens at positions start, start + 1, ... of its request's table.
struct ChunkMetaArgs {
  const int64_t* desc;
  const int32_t* tables;
  int64_t num_slots, table_width, planes, page;
  int64_t count, size, capacity;
  int32_t* cu;
  int32_t* lengths;
  int64_t* positions;
  int64_t* sequences;
  int64_t* blocks;
  int64_t* offsets;
  int32_t* out_tables;
  int64_t out_stride, out_width;
};

__device__ __forceinline__ int64_t chunk_tokens(const int64_t* desc, int64_t i, int64_t capacity) {
  const int64_t n = desc[4 * i + 3];
  return n < 0 ? 0 : n < capacity ? n : capacity;  // sums of up to 2^31 of them stay inside 64 bits
}

// Latency bounds it (2 MB for 256 sequences): descriptors, then the table, then the
// stores.  Grid (size + 1, parts): the workgroups of x < size write sequence x (its table
// row, lengths and cu entry, its tokens in `parts` strides), those of x == size the
// tokens behind the last sequence.  Every workgroup sums the token counts before
// its sequence itself: one launch, no scratch.
__global__ __launch_bounds__(kThreads) void chunk_metadata_kernel(ChunkMetaArgs a) {
  const int64_t seq = blockIdx.x, part = blockIdx.y, parts = gridDim.y;
  const int tid = threadIdx.x;
  const int64_t before = seq < a.count ? seq : a.count;
  int64_t sum = 0;
  for (int64_t i = tid; i < before; i += kThreads) sum += chunk_tokens(a.desc, i, a.capacity);
  __shared__ int64_t sums[kThreads / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((tid & 63) == 0) sums[tid >> 6] = sum;
  __syncthreads();
  int64_t first = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) first += sums[w];
  if (first > a.capacity) first = a.capacity;
  if (seq == a.size) {
    if (part == 0 && tid == 0) a.cu[a.size] = static_cast<int32_t>(first);
    for (int64_t t = first + part * kThreads + tid; t < a.capacity; t += parts * kThreads) {
      a.positions[t] = 0;
      a.sequences[t] = -1;
      a.blocks[t] = -1;
      a.offsets[t] = 0;
    }
    return;
  }
  const bool real = seq < a.count;
  const int64_t slot = real ? a.desc[4 * seq] : 0;
  const int64_t depth = real ? a.desc[4 * seq + 1] : 0;
  const int64_t start = real ? a.desc[4 * seq + 2] : 0;
  const int64_t asked = real ? a.desc[4 * seq + 3] : 0;
  const int64_t plane = a.planes > 1 ? depth : 0;
  const int64_t covered = a.table_width * a.page;
  const bool valid = real && slot >= 0 && slot < a.num_slots && plane >= 0 && plane < a.planes && start >= 0 &&
                     asked >= 0 && start <= covered && asked <= covered - start;
  int64_t tokens = real ? chunk_tokens(a.desc, seq, a.capacity) : 0;
  if (tokens > a.capacity - first) tokens = a.capacity - first;
  const int32_t* src = a.tables + (valid ? (slot * a.planes + plane) * a.table_width : 0);
  if (part == 0 && tid == 0) {
    a.cu[seq] = static_cast<int32_t>(first);
    a.lengths[seq] = valid ? static_cast<int32_t>(start + tokens) : 0;
  }
  int32_t* dst = a.out_tables + seq * a.out_stride;
  for (int64_t c = part * kThreads + tid; c < a.out_width; c += parts * kThreads) dst[c] = valid ? src[c] : 0;
  for (int64_t i = part * kThreads + tid; i < tokens; i += parts * kThreads) {
    const int64_t t = first + i, pos = valid ? start + i : 0;
    const int64_t page = pos / a.page;
    a.positions[t] = pos;
    a.sequences[t] = seq;
    a.blocks[t] = valid ? src[page] : -1;
    a.offsets[t] = pos - page * a.page;
  }
}

unsigned blocks_for(int64_t n) { return static_cast<unsigned>((n + kThreads - 1) / kThreads); }

}  // namespace
}  // namespace rlt

using namespace rlt;

extern "C" int rlt_build_decode_metadata(const int64_t* descriptors, int64_t count, int64_t size,
                                         const int32_t* tables, int64_t num_slots, int64_t table_width, int64_t planes,
                                         int64_t page_size, int64_t* slots, int64_t* positions, int32_t* lengths,
                                         int64_t* blocks, int64_t* offsets, int32_t* out_tables,
                                         int64_t out_table_stride, int64_t out_width, void* stream) {
  if (count < 0 || size < count) return fail(RLT_EINVAL, "rlt_build_decode_metadata: need 0 <= count <= size");
  if (num_slots <= 0 || table_width <= 0 || planes <= 0 || page_size <= 0)
    return fail(RLT_EINVAL, "rlt_build_decode_metadata: table shape and page_size must be positive");
  if (out_width < 0 || out_width > table_width || out_table_stride < out_width)
    return fail(RLT_EINVAL, "rlt_build_decode_metadata: need out_width <= table_width and <= out_table_stride");
  if (size == 0) return RLT_OK;
  if (!tables || !slots || !positions || !lengths || !out_tables || (count && (!descriptors || !blocks || !offsets)))
    return fail(RLT_EINVAL, "rlt_build_decode_metadata: NULL pointer argument");
  if (size > 0x7fffffff) return fail(RLT_EUNSUPPORTED, "rlt_build_decode_metadata: too many rows");
  DecodeMetaArgs a{descriptors, tables,  num_slots, table_width, planes,     page_size,        count,    slots,
                   positions,   lengths, blocks,    offsets,     out_tables, out_table_stride, out_width};
  hipLaunchKernelGGL(decode_metadata_kernel, dim3(static_cast<unsigned>(size)), dim3(kThreads), 0, as_stream(stream), a);
  return check_launch("rlt_build_decode_metadata");
}

extern "C" int rlt_stage_prefill(const int64_t* source, int64_t* target, int32_t* target32, int64_t n, void* stream) {
  if (n < 0) return fail(RLT_EINVAL, "rlt_stage_prefill: n is negative");
  if (n == 0) return RLT_OK;
  if (!source || !target || !target32) return fail(RLT_EINVAL, "rlt_stage_prefill: NULL pointer argument");
  hipLaunchKernelGGL(stage_prefill_kernel, dim3(blocks_for(n)), dim3(kThreads), 0, as_stream(stream), source, target,
                     target32, n);
  return check_launch("rlt_stage_prefill");
}

extern "C" int rlt_expand_prefill(const int64_t* positions, const int64_t* sequences, const int32_t* tables,
                                  int64_t num_sequences, int64_t table_width, int64_t page_size, int64_t* blocks,
                                  int64_t* offsets, int64_t n, void* stream) {
  if (n < 0) return fail(RLT_EINVAL, "rlt_expand_prefill: n is negative");
  if (num_sequences <= 0 || table_width <= 0 || page_size <= 0)
    return fail(RLT_EINVAL, "rlt_expand_prefill: bad table shape");
  if (n == 0) return RLT_OK;
  if (!positions || !sequences || !tables || !blocks || !offsets)
    return fail(RLT_EINVAL, "rlt_expand_prefill: NULL pointer argument");
  hipLaunchKernelGGL(expand_prefill_kernel, dim3(blocks_for(n)), dim3(kThreads), 0, as_stream(stream), positions,
                     sequences, tables, num_sequences, table_width, page_size, blocks, offsets, n);
  return check_launch("rlt_expand_prefill");
}

extern "C" int rlt_build_chunk_metadata(const int64_t* descriptors, int64_t count, int64_t size, const int32_t* tables,
                                        int64_t num_slots, int64_t table_width, int64_t planes, int64_t page_size,
                                        int32_t* cu_seqlens, int32_t* lengths, int64_t* positions, int64_t* sequences,
                                        int64_t* blocks, int64_t* offsets, int64_t capacity, int32_t* out_tables,
                                        int64_t out_table_stride, int64_t out_width, void* stream) {
  if (count < 0 || size < count) return fail(RLT_EINVAL, "rlt_build_chunk_metadata: need 0 <= count <= size");
  if (num_slots <= 0 || table_width <= 0 || planes <= 0 || page_size <= 0)
    return fail(RLT_EINVAL, "rlt_build_chunk_metadata: table shape and page_size must be positive");
  if (out_width < 0 || out_width > table_width || out_table_stride < out_width)
    return fail(RLT_EINVAL, "rlt_build_chunk_metadata: need out_width <= table_width and <= out_table_stride");
  if (capacity < 0 || capacity > 0x7fffffff || table_width > 0x7fffffff / page_size)
    return fail(RLT_EUNSUPPORTED, "rlt_build_chunk_metadata: token counts must fit 31 bits");
  if (size >= (1 << 24) - 1) return fail(RLT_EUNSUPPORTED, "rlt_build_chunk_metadata: too many sequences");
  if (!tables || !cu_seqlens || (size && (!lengths || (out_width && !out_tables))) || (count && !descriptors) ||
      (capacity && (!positions || !sequences || !blocks || !offsets)))
    return fail(RLT_EINVAL, "rlt_build_chunk_metadata: NULL pointer argument");
  ChunkMetaArgs a{descriptors, tables,  num_slots, table_width, planes,    page_size, count,
                  size,        capacity, cu_seqlens, lengths,   positions, sequences, blocks,
                  offsets,     out_tables, out_table_stride, out_width};
  // A part for 1024 tokens (one sequence may hold all), within one round of workgroups:
  // 256 sequences of 25 thousand tokens 3.8 us (6.6 in 16 parts), 1024 of up to 40 4.5 (18.8).
  const unsigned parts = static_cast<unsigned>(std::max<int64_t>(1, std::min({1 + capacity / (4 * kThreads), int64_t(16), kRound / (size + 1)})));
  hipLaunchKernelGGL(chunk_metadata_kernel, dim3(static_cast<unsigned>(size + 1), parts), dim3(kThreads), 0,
                     as_stream(stream), a);
  return check_launch("rlt_build_chunk_metadata");
}
