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
#include <algorithm>

#include "fp8.hpp"

namespace rlt {
namespace {

constexpr int kMaxAxes = 4;
constexpr int kMaxHalf = 256;  // frequencies of a head
constexpr int kFewWaves = 4096;

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

// Aligned rows of 16-bit or fp32 heads that turn as a whole (2 half == d, or half 0: no
// rotation): a wave takes a row, LPH lanes a head.  Lane i of a head holds the 16-byte packets
// i of its two halves, so both dims of its pairs, and its cosines and sines serve all
// heads of the row.  Bytes bound it: 4096 rows of 16 + 16 + 16 heads x 128, bf16 to 8 bits, move
// 86 MB in 18.9 us, 4.6 TB/s; the append alone 51 MB in 12.2.
template <typename T, bool ROT, bool FP8, int LPH, int U>
__global__ __launch_bounds__(256) void rope_axes_kernel(RopeAxesArgs a, int64_t n_rows, int parts) {
  using PK = Packet<T>;
  constexpr int N = PK::N, HALF = LPH * N, NG = 64 / LPH;  // dims of a half, heads at a time (U times, of q, k and v each)
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + uniform(threadIdx.x >> 6);
  const int64_t row = parts == 1 ? item : item / parts;
  if (row >= n_rows) return;
  const int lane = threadIdx.x & 63, i = lane % LPH, g = lane / LPH;
  const int first = static_cast<int>(item - row * parts) * NG + g, stride = parts * NG;
  const bool listed = row < a.n_write;
  auto load = [&](int which, int head, u32x4 (&x)[2]) __attribute__((always_inline)) {
    const T* src = static_cast<const T*>(a.in[which].x) + row * a.in[which].row + head * a.in[which].head + i * N;
    x[0] = *reinterpret_cast<const u32x4*>(src);
    x[1] = *reinterpret_cast<const u32x4*>(src + HALF);
  };
  u32x4 q[U][2] = {}, k[U][2] = {}, v[U][2] = {};
  auto load_heads = [&](int h0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * stride;
      if (ROT && h < a.hq) load(0, h, q[u]);
      if (listed && h < a.hkv) {
        load(1, h, k[u]);
        load(2, h, v[u]);
      }
    }
  };
  load_heads(first);
  int64_t block = -1, offset = -1;
  if (listed) {
    block = a.blocks[row];
    offset = a.offsets[row];
  }
  bool write = block >= 0 && block < a.num_blocks && offset >= 0 && offset < a.page;
  bool inside = true;
  float cs[N], sn[N];
  if constexpr (ROT) {
    const int64_t* pos = a.positions + row * a.p_row;
    const int64_t p0 = pos[0], p1 = a.axes > 1 ? pos[a.p_axis] : 0, p2 = a.axes > 2 ? pos[2 * a.p_axis] : 0;
    const int64_t p3 = a.axes > 3 ? pos[3 * a.p_axis] : 0;
    const uint64_t most = static_cast<uint64_t>(a.max_position);
    inside = static_cast<uint64_t>(p0) < most && static_cast<uint64_t>(p1) < most && static_cast<uint64_t>(p2) < most &&
             static_cast<uint64_t>(p3) < most;
    write &= inside;
    uint32_t words = 0;  // the axes of this lane's frequencies, 2 bits each
#pragma unroll
    for (int w = 0; w < (HALF + 15) / 16; ++w)
      if (i * N / 16 == w) words = a.axis_of[w] >> (2 * (i * N % 16));
    // 32-bit byte offsets into the table (the host checks its size).
    const uint32_t r0 = static_cast<uint32_t>(p0), r1 = static_cast<uint32_t>(p1), r2 = static_cast<uint32_t>(p2), r3 = static_cast<uint32_t>(p3);
    const char* base = reinterpret_cast<const char*>(a.table);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const uint32_t x = words >> (2 * e) & 3;
      const uint32_t at = x & 2 ? (x & 1 ? r3 : r2) : (x & 1 ? r1 : r0);
      const float2 t = *reinterpret_cast<const float2*>(base + (inside ? at * (8u * HALF) : 0u) + 8u * (i * N + e));
      cs[e] = t.x, sn[e] = t.y;
    }
  }
  auto turned = [&](const u32x4 (&x)[2], bool rotate, float (&lo)[N], float (&hi)[N]) __attribute__((always_inline)) {
    PK::unpack(x[0], lo);
    PK::unpack(x[1], hi);
    if (rotate) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float l = lo[e], h = hi[e];
        turn(l, h, cs[e], sn[e], &lo[e], &hi[e]);
      }
    }
  };
  auto store = [&](int which, int head, const u32x4 (&x)[2], bool rotate) __attribute__((always_inline)) {
    float lo[N], hi[N];
    turned(x, rotate, lo, hi);
    const int64_t slot = block * a.c_block + a.layer * a.c_layer + offset * a.c_token + head * a.c_head;
    if constexpr (FP8) {
      float amax = 0.f;
#pragma unroll
      for (int e = 0; e < N; ++e) amax = fmaxf(amax, fmaxf(finite_abs(lo[e]), finite_abs(hi[e])));
      const uint32_t b = scale_byte(group_max<LPH>(amax));
      const float inv = inverse_scale(b);
      uint8_t* codes = static_cast<uint8_t*>(a.cache[which]) + slot + i * N;
      uint32_t w[2][N / 4];
#pragma unroll
      for (int e = 0; e < N / 4; ++e) {
        w[0][e] = codes2(lo[4 * e], lo[4 * e + 1], inv) | codes2(lo[4 * e + 2], lo[4 * e + 3], inv) << 16;
        w[1][e] = codes2(hi[4 * e], hi[4 * e + 1], inv) | codes2(hi[4 * e + 2], hi[4 * e + 3], inv) << 16;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if constexpr (N == 8) *reinterpret_cast<uint2*>(codes + u * HALF) = make_uint2(w[u][0], w[u][1]);
        else *reinterpret_cast<uint32_t*>(codes + u * HALF) = w[u][0];
      }
      if (i == 0)
        a.scales[which][block * a.s_block + a.layer * a.s_layer + offset * a.s_token + head * a.s_head] = static_cast<uint8_t>(b);
    } else {
      T* dst = static_cast<T*>(a.cache[which]) + slot + i * N;
      *reinterpret_cast<u32x4*>(dst) = rotate ? PK::pack(lo) : x[0];
      *reinterpret_cast<u32x4*>(dst + HALF) = rotate ? PK::pack(hi) : x[1];
    }
  };
  for (int h0 = first; h0 < max(a.hq, write ? a.hkv : 0); h0 += U * stride) {
    if (h0 != first) load_heads(h0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * stride;
      if (ROT && h < a.hq) {
        float lo[N], hi[N];
        turned(q[u], true, lo, hi);
        T* dst = static_cast<T*>(a.q_out) + row * a.qo_row + h * a.qo_head + i * N;
        *reinterpret_cast<u32x4*>(dst) = inside ? PK::pack(lo) : u32x4{0u, 0u, 0u, 0u};
        *reinterpret_cast<u32x4*>(dst + HALF) = inside ? PK::pack(hi) : u32x4{0u, 0u, 0u, 0u};
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * stride;
      if (write && h < a.hkv) {
        store(0, h, k[u], ROT);
        store(1, h, v[u], false);
      }
    }
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
  // (A wave a row in workgroups of four, and one a row and head: threads of a launch inside 32 bits.)
  if (n_rows > 4 * kMaxBlocks || hkv > 16384) return fail(RLT_EUNSUPPORTED, "%s: too many rows or heads", name);
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

// Whether rope_axes_kernel covers the call.
bool rows16(const RopeAxesArgs& a, int es) {
  auto packets = [&](const void* x, int64_t s0, int64_t s1, int64_t dim) {
    return dim == 1 && aligned16(x) && s0 * es % 16 == 0 && s1 * es % 16 == 0;
  };
  if (a.half && 2 * a.half != a.d) return false;
  for (int w = a.half ? 0 : 1; w < 3; ++w)
    if (!packets(a.in[w].x, a.in[w].row, a.in[w].head, a.in[w].dim)) return false;
  if (a.half && !packets(a.q_out, a.qo_row, a.qo_head, a.qo_dim)) return false;
  if (a.half && ((reinterpret_cast<uintptr_t>(a.table) & 7u) || a.max_position > (int64_t(1) << 32) / (8 * a.half))) return false;
  const int ce = a.scales[0] ? 1 : es, unit = a.scales[0] ? 16 / es : 16;  // bytes a lane stores at once
  for (int w = 0; w < 2; ++w)
    if (reinterpret_cast<uintptr_t>(a.cache[w]) % unit) return false;
  return a.c_dim == 1 && a.c_block * ce % unit == 0 && a.c_layer * ce % unit == 0 && a.c_token * ce % unit == 0 &&
         a.c_head * ce % unit == 0;
}

template <typename T, bool ROT, bool FP8>
bool launch_rows(const RopeAxesArgs& a, int64_t n_rows, hipStream_t stream) {
  const int lanes = a.d % (2 * Packet<T>::N) == 0 ? a.d / 2 / Packet<T>::N : 0;  // of a head
  // A wave a row, or a few waves where rows are few (us, one against several): 8 rows of 16 +
  // 16 heads x 128 into a bf16 cache 5.5 / 4.0, 512 of 32 + 8 into an 8-bit one 8.2 / 6.1, 1500
  // of 16 + 16 12.4 / 11.1.
  int parts = 1;
  while (lanes && n_rows * parts < kFewWaves && parts * (64 / lanes) < std::max(a.hq, a.hkv)) parts *= 2;
  const bool once = lanes && parts * (64 / lanes) >= std::max(a.hq, a.hkv);  // a wave has all its heads at once
  const int64_t waves = n_rows * parts;
  const dim3 grid(static_cast<unsigned>((waves + 3) / 4)), block(256);
#define LAUNCH(L)                                                                                                      \
  do {                                                                                                                 \
    if (once) hipLaunchKernelGGL((rope_axes_kernel<T, ROT, FP8, L, 1>), grid, block, 0, stream, a, n_rows, parts);     \
    else hipLaunchKernelGGL((rope_axes_kernel<T, ROT, FP8, L, 2>), grid, block, 0, stream, a, n_rows, parts);          \
  } while (0)
  switch (lanes) {
    case 4: LAUNCH(4); return true;
    case 8: LAUNCH(8); return true;
    case 16: LAUNCH(16); return true;
    case 32: LAUNCH(32); return true;
    default: return false;
  }
#undef LAUNCH
}

template <typename T>
void launch_type(const RopeAxesArgs& a, int64_t n_rows, hipStream_t stream) {
  if (rows16(a, sizeof(T))) {
    if (a.half ? (a.scales[0] ? launch_rows<T, true, true>(a, n_rows, stream) : launch_rows<T, true, false>(a, n_rows, stream))
               : launch_rows<T, false, true>(a, n_rows, stream))
      return;
  }
  const dim3 grid(static_cast<unsigned>(n_rows), static_cast<unsigned>(a.hq + 2 * a.hkv));
  hipLaunchKernelGGL((rope_axes_generic_kernel<T>), grid, dim3(64), 0, stream, a);
}

int launch(const RopeAxesArgs& a, int64_t n_rows, int dtype, hipStream_t stream, const char* name) {
  switch (dtype) {
    case RLT_BFLOAT16: launch_type<bf16>(a, n_rows, stream); break;
    case RLT_FLOAT16: launch_type<f16>(a, n_rows, stream); break;
    default: launch_type<float>(a, n_rows, stream); break;
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
