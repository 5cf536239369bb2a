// Appends to the block-scaled 8-bit KV cache, and reading it back (int8.hpp).
//
// Append.  The rows of a call that go to one block stand together in it; a wave takes them
// as one, for a head:
//   s0 = the block's scale, 0 where the call writes its offset 0 (which begins the block)
//   s  = max(s0, largest |x| of the new rows / 127, 2^-126)
//   codes the block holds: rint(code * (s0 / s)), where s is not s0
//   new codes: rint(x * (1 / s))
// each operation rounded to fp32 on its own, ties to even.  A code that is kept is rounded
// again each time s grows, by at most half a step of the new scale.  New rows with a value that
// is not finite make s NaN and their codes 0; s0 NaN stays.
#include <algorithm>

#include "int8.hpp"

namespace rlt {
namespace {

constexpr int kWaves = 4;

struct AppendI8Args {
  const void* x[2];  // k, v
  int64_t x_row[2], x_head[2], x_dim[2];
  uint8_t* codes[2];
  int64_t c_block, c_layer, c_token, c_head, c_dim;
  float* scales[2];
  int64_t s_block, s_layer, s_head;
  const int64_t* blocks;
  const int64_t* offsets;
  int64_t rows, layer, num_blocks, page;
  int hkv, d;
};

__device__ __forceinline__ bool valid_block(const AppendI8Args& a, int64_t b) { return b >= 0 && b < a.num_blocks; }
__device__ __forceinline__ bool valid_offset(const AppendI8Args& a, int64_t o) { return o >= 0 && o < a.page; }

// Rows from row on that go to the same block.
__device__ __forceinline__ int64_t run_length(const AppendI8Args& a, int64_t row, int64_t block, int lane) {
  for (int64_t n = 1;; n += 64) {
    const int64_t at = row + n + lane;
    const uint64_t other = __builtin_amdgcn_ballot_w64(!(at < a.rows && a.blocks[at] == block));
    if (other) return n + __builtin_ctzll(other);
  }
}

// The new scale, from the old one (0 for a block that begins) and the bits of the largest |x|.
__device__ __forceinline__ float grown_scale(float before, uint32_t top) {
  if (top >= 0x7f800000u || before != before) return __uint_as_float(0x7fc00000u);
  return fmaxf(fmaxf(before, __uint_as_float(top) / kLargestCode), kSmallestScale);
}

// The low byte of the result is x rounded to a whole number, ties to even, for |x| below 2^22: added to
// 1.5 * 2^23 it moves to the last bits of the sum.  (0 for NaN.)
__device__ __forceinline__ uint32_t code_of(float x, float inv) {
#pragma clang fp contract(off)
  return __float_as_uint(x * inv + 12582912.f);
}
// Four of them, the first in the lowest byte.
__device__ __forceinline__ uint32_t codes4(const float* x, float inv) {
  const uint32_t lo = __builtin_amdgcn_perm(code_of(x[1], inv), code_of(x[0], inv), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(code_of(x[3], inv), code_of(x[2], inv), 0x04000c0cu);
  return lo | hi;
}
// A code's value, rounded to fp32 also where it is rounded to 16 bits next (the compiler would
// join both into one instruction for fp16, and not for bf16).
__device__ __forceinline__ float code_value(int code, float scale) {
  float x = static_cast<float>(code) * scale;
  asm("" : "+v"(x));
  return x;
}

// Any strides and head size: a wave a (row, K or V, head); the first row of a block works.
template <typename T>
__global__ __launch_bounds__(64) void append_i8_generic_kernel(AppendI8Args a) {
  const int lane = threadIdx.x, which = blockIdx.y / a.hkv, head = blockIdx.y % a.hkv;
  const int64_t row = blockIdx.x, block = a.blocks[row];
  if (!valid_block(a, block) || (row > 0 && a.blocks[row - 1] == block)) return;
  const int64_t n = run_length(a, row, block, lane);
  const T* x = static_cast<const T*>(a.x[which]) + row * a.x_row[which] + head * a.x_head[which];
  uint8_t* codes = a.codes[which] + block * a.c_block + a.layer * a.c_layer + head * a.c_head;
  float* scale = a.scales[which] + block * a.s_block + a.layer * a.s_layer + head * a.s_head;
  uint32_t top = 0;
  bool begins = false, any = false;
  for (int64_t r = 0; r < n; ++r) {
    const int64_t offset = a.offsets[row + r];
    if (!valid_offset(a, offset)) continue;
    any = true;
    begins |= offset == 0;
    for (int d = lane; d < a.d; d += 64)
      top = max(top, __float_as_uint(load_elem(x + r * a.x_row[which] + d * a.x_dim[which])) & 0x7fffffffu);
  }
  if (!any) return;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), i, 64)));
  const float before = begins ? 0.f : *scale, s = grown_scale(before, top);
  if (lane == 0) *scale = s;
  if (!begins && s != before && s == s) {
    const float ratio = before / s;
    for (int64_t o = 0; o < a.page; ++o)
      for (int d = lane; d < a.d; d += 64) {
        uint8_t* c = codes + o * a.c_token + d * a.c_dim;
        *c = static_cast<uint8_t>(code_of(static_cast<float>(static_cast<int8_t>(*c)), ratio));
      }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // before the new rows' codes
  }
  const float inv = s == s ? 1.f / s : s;
  for (int64_t r = 0; r < n; ++r) {
    const int64_t offset = a.offsets[row + r];
    if (!valid_offset(a, offset)) continue;
    for (int d = lane; d < a.d; d += 64)
      codes[offset * a.c_token + d * a.c_dim] =
          static_cast<uint8_t>(code_of(load_elem(x + r * a.x_row[which] + d * a.x_dim[which]), inv));
  }
}

struct GatherI8Args {
  const uint8_t* codes[2];
  int64_t c_block, c_layer, c_token, c_head, c_dim;
  const float* scales[2];
  int64_t s_block, s_layer, s_head;
  const int64_t* blocks;
  const int64_t* offsets;
  void* out[2];  // [rows, hkv, d]
  int64_t rows, layer, num_blocks, page;
  int hkv, d;
};

// Any strides and head size: a wave a (row, K or V, head).
template <typename T>
__global__ __launch_bounds__(64) void gather_i8_generic_kernel(GatherI8Args a) {
  const int lane = threadIdx.x, which = blockIdx.y / a.hkv, head = blockIdx.y % a.hkv;
  const int64_t row = blockIdx.x, block = a.blocks[row], offset = a.offsets[row];
  const bool in = block >= 0 && block < a.num_blocks && offset >= 0 && offset < a.page;
  const uint8_t* codes = a.codes[which] + block * a.c_block + a.layer * a.c_layer + offset * a.c_token + head * a.c_head;
  T* out = static_cast<T*>(a.out[which]) + (row * a.hkv + head) * a.d;
  const float s = in ? a.scales[which][block * a.s_block + a.layer * a.s_layer + head * a.s_head] : 0.f;
  for (int d = lane; d < a.d; d += 64)
    store_elem(out + d, in ? code_value(static_cast<int8_t>(codes[d * a.c_dim]), s) : 0.f);
}

// What both entry points check.
int cache_args(const char* name, const void* key_cache, const void* value_cache, const int64_t* cache_strides,
               const void* key_scales, const void* value_scales, const int64_t* scale_strides, const int64_t* blocks,
               const int64_t* offsets, int64_t n_rows, int64_t layer, int64_t num_layers, int64_t num_blocks, int64_t page_size,
               int64_t hkv, int64_t d, int dtype) {
  if (!dtype_size(dtype)) return fail(RLT_EINVAL, "%s: unknown dtype %d", name, dtype);
  if (n_rows < 0) return fail(RLT_EINVAL, "%s: n_rows is negative", name);
  if (hkv <= 0 || d <= 0) return fail(RLT_EINVAL, "%s: num_kv_heads and head_dim must be positive", name);
  if (num_blocks <= 0 || num_layers <= 0 || page_size <= 0) return fail(RLT_EINVAL, "%s: pool dimensions must be positive", name);
  if (layer < 0 || layer >= num_layers) return fail(RLT_EINVAL, "%s: layer %lld out of range", name, (long long)layer);
  if (d > 64 * kPerLane) return fail(RLT_EUNSUPPORTED, "%s: head_dim above %d", name, 64 * kPerLane);
  if (n_rows > kMaxBlocks || hkv > 16384) return fail(RLT_EUNSUPPORTED, "%s: too many rows or heads", name);
  if (n_rows == 0) return RLT_OK;
  if (!key_cache || !value_cache || !cache_strides || !key_scales || !value_scales || !scale_strides || !blocks || !offsets)
    return fail(RLT_EINVAL, "%s: NULL pointer argument", name);
  for (int i = 0; i < 5; ++i)
    if (cache_strides[i] < 0 || (i < 3 && scale_strides[i] < 0)) return fail(RLT_EINVAL, "%s: negative cache stride", name);
  if (reinterpret_cast<uintptr_t>(key_scales) % 4 || reinterpret_cast<uintptr_t>(value_scales) % 4)
    return fail(RLT_EINVAL, "%s: scales must be on 4 bytes", name);
  return RLT_OK;
}

template <typename T>
void launch_append(const AppendI8Args& a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.rows), static_cast<unsigned>(2 * a.hkv));
  hipLaunchKernelGGL((append_i8_generic_kernel<T>), grid, dim3(64), 0, stream, a);
}

template <typename T>
void launch_gather(const GatherI8Args& a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.rows), static_cast<unsigned>(2 * a.hkv));
  hipLaunchKernelGGL((gather_i8_generic_kernel<T>), grid, dim3(64), 0, stream, a);
}

}  // namespace
}  // namespace rlt

using namespace rlt;

extern "C" int rlt_kv_append_int8(void* key_cache, void* value_cache, const int64_t* cache_strides, void* key_scales,
                                  void* value_scales, const int64_t* scale_strides, const void* k,
                                  const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                  const int64_t* write_blocks, const int64_t* write_offsets, int64_t n_rows,
                                  int64_t layer, int64_t num_layers, int64_t num_blocks, int64_t page_size,
                                  int64_t num_kv_heads, int64_t head_dim, int dtype, void* stream) {
  const char* name = "rlt_kv_append_int8";
  if (int rc = cache_args(name, key_cache, value_cache, cache_strides, key_scales, value_scales, scale_strides, write_blocks,
                          write_offsets, n_rows, layer, num_layers, num_blocks, page_size, num_kv_heads, head_dim, dtype))
    return rc;
  if (n_rows == 0) return RLT_OK;
  if (!k || !k_strides || !v || !v_strides) return fail(RLT_EINVAL, "%s: NULL pointer argument", name);
  AppendI8Args a{};
  a.x[0] = k, a.x_row[0] = k_strides[0], a.x_head[0] = k_strides[1], a.x_dim[0] = k_strides[2];
  a.x[1] = v, a.x_row[1] = v_strides[0], a.x_head[1] = v_strides[1], a.x_dim[1] = v_strides[2];
  a.codes[0] = static_cast<uint8_t*>(key_cache), a.codes[1] = static_cast<uint8_t*>(value_cache);
  a.c_block = cache_strides[0], a.c_layer = cache_strides[1], a.c_token = cache_strides[2];
  a.c_head = cache_strides[3], a.c_dim = cache_strides[4];
  a.scales[0] = static_cast<float*>(key_scales), a.scales[1] = static_cast<float*>(value_scales);
  a.s_block = scale_strides[0], a.s_layer = scale_strides[1], a.s_head = scale_strides[2];
  a.blocks = write_blocks, a.offsets = write_offsets;
  a.rows = n_rows, a.layer = layer, a.num_blocks = num_blocks, a.page = page_size;
  a.hkv = static_cast<int>(num_kv_heads), a.d = static_cast<int>(head_dim);
  switch (dtype) {
    case RLT_BFLOAT16: launch_append<bf16>(a, as_stream(stream)); break;
    case RLT_FLOAT16: launch_append<f16>(a, as_stream(stream)); break;
    default: launch_append<float>(a, as_stream(stream)); break;
  }
  return check_launch(name);
}

extern "C" int rlt_kv_gather_int8(const void* key_cache, const void* value_cache, const int64_t* cache_strides,
                                  const void* key_scales, const void* value_scales, const int64_t* scale_strides,
                                  const int64_t* blocks, const int64_t* offsets, int64_t n_rows, void* out_k, void* out_v,
                                  int64_t layer, int64_t num_layers, int64_t num_blocks, int64_t page_size,
                                  int64_t num_kv_heads, int64_t head_dim, int dtype, void* stream) {
  const char* name = "rlt_kv_gather_int8";
  if (int rc = cache_args(name, key_cache, value_cache, cache_strides, key_scales, value_scales, scale_strides, blocks, offsets,
                          n_rows, layer, num_layers, num_blocks, page_size, num_kv_heads, head_dim, dtype))
    return rc;
  if (n_rows == 0) return RLT_OK;
  if (!out_k || !out_v) return fail(RLT_EINVAL, "%s: NULL pointer argument", name);
  GatherI8Args a{};
  a.codes[0] = static_cast<const uint8_t*>(key_cache), a.codes[1] = static_cast<const uint8_t*>(value_cache);
  a.c_block = cache_strides[0], a.c_layer = cache_strides[1], a.c_token = cache_strides[2];
  a.c_head = cache_strides[3], a.c_dim = cache_strides[4];
  a.scales[0] = static_cast<const float*>(key_scales), a.scales[1] = static_cast<const float*>(value_scales);
  a.s_block = scale_strides[0], a.s_layer = scale_strides[1], a.s_head = scale_strides[2];
  a.blocks = blocks, a.offsets = offsets;
  a.out[0] = out_k, a.out[1] = out_v;
  a.rows = n_rows, a.layer = layer, a.num_blocks = num_blocks, a.page = page_size;
  a.hkv = static_cast<int>(num_kv_heads), a.d = static_cast<int>(head_dim);
  switch (dtype) {
    case RLT_BFLOAT16: launch_gather<bf16>(a, as_stream(stream)); break;
    case RLT_FLOAT16: launch_gather<f16>(a, as_stream(stream)); break;
    default: launch_gather<float>(a, as_stream(stream)); break;
  }
  return check_launch(name);
}
