// Appends to the 8-bit KV cache (codes and scales: fp8.hpp), and the rotary
// embedding by positions of several axes fused with an append to a cache of
// either kind.
//
// Rotation.  Frequency j of a head (dims j and j + half) turns by the position of
// axis axis_of[j]: (c, s) = table[position[axis_of[j]]][j], a table of fp32 pairs the
// caller computes once (a table rather than angles in the kernel: sine and cosine
// of a far position need its angle in 64 bits).
//   out[j] = x[j] c - x[j + half] s,   out[j + half] = x[j + half] c + x[j] s
// each product and the sum rounded to fp32 on its own, the result rounded once to
// the type it is stored in.  Dims past 2 * half pass through.
#include "fp8.hpp"

namespace rlt {
namespace {

constexpr int kMaxAxes = 4;
constexpr int kMaxHalf = 256;  // frequencies of a head

struct AppendRow {
  const void* x;
  int64_t row, head, dim;
};

// One row's work: rotate q (all rows), rotate and store k, store v.
struct RopeAxesArgs {
  AppendRow in[3];  // q (absent: hq 0), k, v
  void* q_out;
  int64_t qo_row, qo_head, qo_dim;
  void* cache[2];
  int64_t c_block, c_layer, c_token, c_head, c_dim;
  uint8_t* scales[2];  // null: a cache of the activations' type
  int64_t s_block, s_layer, s_token, s_head;
  const int64_t* positions;
  int64_t p_row, p_axis;
  const float* table;  // [max_position, half, 2]
  int64_t max_position;
  const int64_t* blocks;
  const int64_t* offsets;
  int64_t n_write, layer, num_blocks, page;
  int axes, half, hq, hkv, d;
  uint32_t axis_of[kMaxHalf / 16];  // 2 bits a frequency
};

__device__ __forceinline__ int axis_of(const RopeAxesArgs& a, int j) { return (a.axis_of[j >> 4] >> (2 * (j & 15))) & 3; }

__device__ __forceinline__ void turn(float lo, float hi, float c, float s, float* out_lo, float* out_hi) {
#pragma clang fp contract(off)
  *out_lo = lo * c - hi * s;
  *out_hi = hi * c + lo * s;
}

// Whether every axis of the row has its position inside the table.
__device__ __forceinline__ bool positions_inside(const RopeAxesArgs& a, int64_t row) {
  bool ok = true;
  for (int x = 0; x < a.axes; ++x) {
    const int64_t p = a.positions[row * a.p_row + x * a.p_axis];
    ok &= p >= 0 && p < a.max_position;
  }
  return ok;
}

// Any strides and head size up to 2 * kMaxHalf: one wave a (row, head of q, k or v).
// A lane owns both dims of its pairs, so q_out may be q.
template <typename T>
__global__ __launch_bounds__(64) void rope_axes_generic_kernel(RopeAxesArgs a) {
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  int which = 0, head = blockIdx.y;
  if (head >= a.hq) which = 1, head -= a.hq;
  if (which && head >= a.hkv) which = 2, head -= a.hkv;
  int64_t block = -1, offset = 0;
  if (which) {
    if (row >= a.n_write) return;
    block = a.blocks[row];
    offset = a.offsets[row];
    if (block < 0 || block >= a.num_blocks || offset < 0 || offset >= a.page) return;
  }
  const bool turned = a.half > 0 && which < 2;
  const bool inside = a.half == 0 || positions_inside(a, row);
  if (which && !inside) return;
  const AppendRow in = a.in[which];
  const T* x = static_cast<const T*>(in.x) + row * in.row + head * in.head;
  const int half = turned ? a.half : 0;
  constexpr int kPairs = kMaxHalf / 64, kRest = 2 * kPairs;
  float lo[kPairs], hi[kPairs], rest[kRest];
  float amax = 0.f;
#pragma unroll
  for (int c = 0; c < kPairs; ++c) {
    const int j = lane + 64 * c;
    lo[c] = hi[c] = 0.f;
    if (j >= half || !inside) continue;
    const int64_t p = a.positions[row * a.p_row + axis_of(a, j) * a.p_axis];
    const float* t = a.table + (p * half + j) * 2;
    turn(load_elem(x + j * in.dim), load_elem(x + (half + j) * in.dim), t[0], t[1], &lo[c], &hi[c]);
    amax = fmaxf(amax, fmaxf(finite_abs(lo[c]), finite_abs(hi[c])));
  }
#pragma unroll
  for (int c = 0; c < kRest; ++c) {
    const int j = 2 * half + lane + 64 * c;
    rest[c] = 0.f;
    if (j >= a.d || !inside) continue;
    rest[c] = load_elem(x + j * in.dim);
    amax = fmaxf(amax, finite_abs(rest[c]));
  }
  if (which && a.scales[which - 1]) {
    const uint32_t b = scale_byte(group_max<64>(amax));
    const float inv = inverse_scale(b);
    uint8_t* codes = static_cast<uint8_t*>(a.cache[which - 1]) + block * a.c_block + a.layer * a.c_layer +
                     offset * a.c_token + head * a.c_head;
    if (lane == 0)
      a.scales[which - 1][block * a.s_block + a.layer * a.s_layer + offset * a.s_token + head * a.s_head] =
          static_cast<uint8_t>(b);
#pragma unroll
    for (int c = 0; c < kPairs; ++c) {
      const int j = lane + 64 * c;
      if (j >= half) continue;
      const uint32_t w = codes2(lo[c], hi[c], inv);
      codes[j * a.c_dim] = static_cast<uint8_t>(w);
      codes[(half + j) * a.c_dim] = static_cast<uint8_t>(w >> 8);
    }
#pragma unroll
    for (int c = 0; c < kRest; ++c) {
      const int j = 2 * half + lane + 64 * c;
      if (j < a.d) codes[j * a.c_dim] = static_cast<uint8_t>(codes2(rest[c], 0.f, inv));
    }
    return;
  }
  T* dst;
  int64_t dim;
  if (which) {
    dst = static_cast<T*>(a.cache[which - 1]) + block * a.c_block + a.layer * a.c_layer + offset * a.c_token + head * a.c_head;
    dim = a.c_dim;
  } else {
    dst = static_cast<T*>(a.q_out) + row * a.qo_row + head * a.qo_head;
    dim = a.qo_dim;
  }
#pragma unroll
  for (int c = 0; c < kPairs; ++c) {
    const int j = lane + 64 * c;
    if (j >= half) continue;
    store_elem(dst + j * dim, lo[c]);
    store_elem(dst + (half + j) * dim, hi[c]);
  }
#pragma unroll
  for (int c = 0; c < kRest; ++c) {
    const int j = 2 * half + lane + 64 * c;
    if (j < a.d) store_elem(dst + j * dim, rest[c]);
  }
}

// Checks of both entry points; fills everything but q, the rotation and the rows.
int append_args(const char* name, void* key_cache, void* value_cache, const int64_t* cache_strides, void* key_scales,
                void* value_scales, const int64_t* scale_strides, const void* k, const int64_t* k_strides,
                const void* v, const int64_t* v_strides, const int64_t* write_blocks, const int64_t* write_offsets,
                int64_t n_rows, int64_t n_write, int64_t layer, int64_t num_layers, int64_t num_blocks,
                int64_t page_size, int64_t hkv, int64_t d, int dtype, RopeAxesArgs* a) {
  if (!dtype_size(dtype)) return fail(RLT_EINVAL, "%s: unknown dtype %d", name, dtype);
  if (n_rows < 0 || n_write < 0 || n_write > n_rows) return fail(RLT_EINVAL, "%s: need 0 <= n_write <= n_rows", name);
  if (hkv <= 0 || d <= 0) return fail(RLT_EINVAL, "%s: num_kv_heads and head_dim must be positive", name);
  if (d > 2 * kMaxHalf) return fail(RLT_EUNSUPPORTED, "%s: head_dim above %d", name, 2 * kMaxHalf);
  if (num_blocks <= 0 || num_layers <= 0 || page_size <= 0) return fail(RLT_EINVAL, "%s: pool dimensions must be positive", name);
  if (layer < 0 || layer >= num_layers) return fail(RLT_EINVAL, "%s: layer %lld out of range", name, (long long)layer);
  if (n_rows > 0x7fffffff || hkv > 16384) return fail(RLT_EUNSUPPORTED, "%s: too many rows or heads", name);
  if (n_rows == 0) return RLT_OK;
  if (!key_cache || !value_cache || !cache_strides || !k || !k_strides || !v || !v_strides ||
      (n_write > 0 && (!write_blocks || !write_offsets)) || !key_scales != !value_scales || (key_scales && !scale_strides))
    return fail(RLT_EINVAL, "%s: NULL pointer argument", name);
  for (int i = 0; i < 5; ++i)
    if (cache_strides[i] < 0 || (key_scales && i < 4 && scale_strides[i] < 0))
      return fail(RLT_EINVAL, "%s: negative cache stride", name);
  *a = RopeAxesArgs{};
  a->in[1] = AppendRow{k, k_strides[0], k_strides[1], k_strides[2]};
  a->in[2] = AppendRow{v, v_strides[0], v_strides[1], v_strides[2]};
  a->cache[0] = key_cache;
  a->cache[1] = value_cache;
  a->c_block = cache_strides[0], a->c_layer = cache_strides[1], a->c_token = cache_strides[2];
  a->c_head = cache_strides[3], a->c_dim = cache_strides[4];
  if (key_scales) {
    a->scales[0] = static_cast<uint8_t*>(key_scales);
    a->scales[1] = static_cast<uint8_t*>(value_scales);
    a->s_block = scale_strides[0], a->s_layer = scale_strides[1];
    a->s_token = scale_strides[2], a->s_head = scale_strides[3];
  }
  a->blocks = write_blocks;
  a->offsets = write_offsets;
  a->n_write = n_write;
  a->layer = layer;
  a->num_blocks = num_blocks;
  a->page = page_size;
  a->hkv = static_cast<int>(hkv);
  a->d = static_cast<int>(d);
  return RLT_OK;
}

int launch(const RopeAxesArgs& a, int64_t n_rows, int dtype, hipStream_t stream, const char* name) {
  const dim3 grid(static_cast<unsigned>(n_rows), static_cast<unsigned>(a.hq + 2 * a.hkv));
  switch (dtype) {
    case RLT_BFLOAT16: hipLaunchKernelGGL((rope_axes_generic_kernel<bf16>), grid, dim3(64), 0, stream, a); break;
    case RLT_FLOAT16: hipLaunchKernelGGL((rope_axes_generic_kernel<f16>), grid, dim3(64), 0, stream, a); break;
    default: hipLaunchKernelGGL((rope_axes_generic_kernel<float>), grid, dim3(64), 0, stream, a); break;
  }
  return check_launch(name);
}

}  // namespace
}  // namespace rlt

using namespace rlt;

extern "C" int rlt_kv_append_fp8(void* key_cache, void* value_cache, const int64_t* cache_strides, void* key_scales,
                                 void* value_scales, const int64_t* scale_strides, const void* k,
                                 const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                 const int64_t* write_blocks, const int64_t* write_offsets, int64_t n_rows,
                                 int64_t layer, int64_t num_layers, int64_t num_blocks, int64_t page_size,
                                 int64_t num_kv_heads, int64_t head_dim, int dtype, void* stream) {
  RopeAxesArgs a;
  if (int rc = append_args("rlt_kv_append_fp8", key_cache, value_cache, cache_strides, key_scales, value_scales,
                           scale_strides, k, k_strides, v, v_strides, write_blocks, write_offsets, n_rows, n_rows,
                           layer, num_layers, num_blocks, page_size, num_kv_heads, head_dim, dtype, &a))
    return rc;
  if (n_rows == 0) return RLT_OK;
  if (!key_scales) return fail(RLT_EINVAL, "rlt_kv_append_fp8: NULL pointer argument");
  return launch(a, n_rows, dtype, as_stream(stream), "rlt_kv_append_fp8");
}

extern "C" int rlt_rope_axes_kv_append(void* key_cache, void* value_cache, const int64_t* cache_strides,
                                       void* key_scales, void* value_scales, const int64_t* scale_strides,
                                       const void* q, const int64_t* q_strides, const void* k,
                                       const int64_t* k_strides, const void* v, const int64_t* v_strides, void* q_out,
                                       const int64_t* q_out_strides, const int64_t* positions,
                                       const int64_t* position_strides, int64_t axes, const float* table,
                                       int64_t max_position, const uint8_t* axis_of, int64_t half,
                                       const int64_t* write_blocks, const int64_t* write_offsets, int64_t n_rows,
                                       int64_t n_write, int64_t layer, int64_t num_layers, int64_t num_blocks,
                                       int64_t page_size, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                       int dtype, void* stream) {
  const char* name = "rlt_rope_axes_kv_append";
  RopeAxesArgs a;
  if (int rc = append_args(name, key_cache, value_cache, cache_strides, key_scales, value_scales, scale_strides, k,
                           k_strides, v, v_strides, write_blocks, write_offsets, n_rows, n_write, layer, num_layers,
                           num_blocks, page_size, num_kv_heads, head_dim, dtype, &a))
    return rc;
  if (num_q_heads <= 0 || num_q_heads > 16384) return fail(RLT_EINVAL, "%s: bad num_q_heads", name);
  if (axes < 1 || axes > kMaxAxes) return fail(RLT_EINVAL, "%s: 1 to %d axes", name, kMaxAxes);
  if (half < 1 || 2 * half > head_dim) return fail(RLT_EINVAL, "%s: the table turns more dims than a head has", name);
  if (max_position <= 0) return fail(RLT_EINVAL, "%s: the table has no positions", name);
  if (n_rows == 0) return RLT_OK;
  if (!q || !q_strides || !q_out || !q_out_strides || !positions || !position_strides || !table || !axis_of)
    return fail(RLT_EINVAL, "%s: NULL pointer argument", name);
  for (int64_t j = 0; j < half; ++j) {
    if (axis_of[j] >= axes) return fail(RLT_EINVAL, "%s: frequency %lld turns by an axis past the last", name, (long long)j);
    a.axis_of[j >> 4] |= static_cast<uint32_t>(axis_of[j]) << (2 * (j & 15));
  }
  a.in[0] = AppendRow{q, q_strides[0], q_strides[1], q_strides[2]};
  a.q_out = q_out;
  a.qo_row = q_out_strides[0], a.qo_head = q_out_strides[1], a.qo_dim = q_out_strides[2];
  a.positions = positions;
  a.p_row = position_strides[0], a.p_axis = position_strides[1];
  a.table = table;
  a.max_position = max_position;
  a.axes = static_cast<int>(axes);
  a.half = static_cast<int>(half);
  a.hq = static_cast<int>(num_q_heads);
  return launch(a, n_rows, dtype, as_stream(stream), name);
}
