// Attention over the block-scaled 8-bit paged KV cache (int8.hpp):
//   s_j = scale * ks_b(j) (q . K_j),  out = sum_j softmax(s)_j vs_b(j) V_j
// over a sequence's keys, K_j and V_j codes and b(j) the block of key j; for one new
// token a sequence (decode) and for packed chunks, bottom-right causal (prefill).
// Scores, softmax sums and the sums of weighted values are fp32, outputs of q's type.
#include "decode_int8.hpp"
#include "int8.hpp"
#include "prefill_int8.hpp"

namespace rlt {
namespace {

// Any head size up to 64 * kPerLane, page size, grouping and strides: one workgroup a
// (row, query head), wave w takes tokens w, w + kGenericWaves, ... with the head's dims over
// its lanes; the waves are joined through LDS in wave order.  Latency bounds it, a byte a
// lane and token: 24 rows of 512-4096 tokens, 16 heads x 72, 808 us (16 heads x 80, which the kernels on the
// matrix cores take, 56).
template <typename T>
__global__ __launch_bounds__(64 * kGenericWaves) void attn_i8_generic_kernel(AttnI8Args p) {
  const Attn8Args& a = p.a;
  const int64_t row = blockIdx.x;
  const int h = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  int seq, len;
  if (!row_keys(a, row, &seq, &len)) return;
  T* orow = static_cast<T*>(a.out) + row * a.o_row + h * a.o_head;
  const T* qrow = static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head;
  const int kvh = h / (a.hq / a.hkv);
  float qv[kPerLane], acc[kPerLane];
#pragma unroll
  for (int c = 0; c < kPerLane; ++c) {
    const int d = lane + 64 * c;
    qv[c] = d < a.d ? load_elem(qrow + d * a.q_dim) * a.qscale : 0.f;
    acc[c] = 0.f;
  }
  float m = -INFINITY, l = 0.f, e = kNoExponent;
  const int32_t* trow = a.tables + seq * a.table_stride;
  for (int t = wave; t < len; t += kGenericWaves) {
    const int64_t block = block_of(a, trow[t / a.page]);
    const int64_t base = block * a.kv_block + (t % a.page) * a.kv_token + kvh * a.kv_head;
    const int64_t at = block * a.s_block + kvh * a.s_head;
    const float sk = block_scale(p.ks[at]), sv = block_scale(p.vs[at]);
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < kPerLane; ++c) {
      const int d = lane + 64 * c;
      if (d < a.d) dot = fmaf(qv[c], static_cast<float>(static_cast<int8_t>(a.k[base + d * a.kv_dim])), dot);
    }
    const float x = rounded_product(group_sum<64>(dot), sk);  // as its maximum is: a large one's last bits are whole numbers
    const float mn = fmaxf(m, ceilf(x));
    const float off = mn == -INFINITY ? 0.f : mn;  // only -inf scores so far: they weigh 0
    const float w = fast_exp2(x - off);
    const float down = off - m;  // +inf at the first key
    const float en = fmaxf(e - down, ceilf(x - off) + scale_exponent(sv));
    const float corr = mn == -INFINITY ? 0.f : fast_exp2(e - down - en);
    l = l * fast_exp2(m - off) + w;
    const float wv = w * weight_scale(sv, fmaxf(en, kNoExponent));
#pragma unroll
    for (int c = 0; c < kPerLane; ++c) {
      const int d = lane + 64 * c;
      if (d < a.d) acc[c] = fmaf(wv, static_cast<float>(static_cast<int8_t>(a.v[base + d * a.kv_dim])), acc[c] * corr);
    }
    m = mn;
    e = fmaxf(en, kNoExponent);
  }
  __shared__ float ms[kGenericWaves], ls[kGenericWaves], es[kGenericWaves], accs[kGenericWaves][64 * kPerLane];
  if (lane == 0) ms[wave] = m, ls[wave] = l, es[wave] = e;
#pragma unroll
  for (int c = 0; c < kPerLane; ++c) accs[wave][lane + 64 * c] = acc[c];
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kGenericWaves; ++w) top = fmaxf(top, ms[w]);
  const float off = top == -INFINITY ? 0.f : top;
  float sum = 0.f, exponent = kNoExponent;
#pragma unroll
  for (int w = 0; w < kGenericWaves; ++w) {
    sum += ls[w] * fast_exp2(ms[w] - off);
    exponent = fmaxf(exponent, es[w] + (ms[w] - off));
  }
  const float inv = 1.f / sum;
  for (int d = threadIdx.x; d < a.d; d += 64 * kGenericWaves) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kGenericWaves; ++w) x = fmaf(accs[w][d], fast_exp2(es[w] + (ms[w] - off) - exponent), x);
    store_elem(orow + d * a.o_dim, len > 0 ? ldexpf(x * inv, static_cast<int>(exponent)) : 0.f);
  }
}

}  // namespace

int launch_attn_i8_generic(const AttnI8Args& p, int dtype, hipStream_t stream, const char* name) {
  const dim3 grid(static_cast<unsigned>(p.a.rows), static_cast<unsigned>(p.a.hq)), block(64 * kGenericWaves);
  switch (dtype) {
    case RLT_BFLOAT16: hipLaunchKernelGGL((attn_i8_generic_kernel<bf16>), grid, block, 0, stream, p); break;
    case RLT_FLOAT16: hipLaunchKernelGGL((attn_i8_generic_kernel<f16>), grid, block, 0, stream, p); break;
    default: hipLaunchKernelGGL((attn_i8_generic_kernel<float>), grid, block, 0, stream, p); break;
  }
  return check_launch(name);
}

namespace {

// The arguments of either call; RLT_OK with a.rows 0 where there is nothing to do.
int attention_args(const char* name, const void* q, const int64_t* q_strides, const void* key_cache, const void* value_cache,
                   const int64_t* kv_strides, const void* key_scales, const void* value_scales, const int64_t* scale_strides,
                   const int32_t* tables, int64_t table_stride, int64_t width, const int32_t* lens, int64_t num_seqs, void* out,
                   const int64_t* out_strides, int64_t rows, int64_t hq, int64_t hkv, int64_t d, int64_t page,
                   int64_t num_blocks, float scale, int dtype, AttnI8Args* p) {
  *p = AttnI8Args{};
  const int64_t strides[3] = {scale_strides ? scale_strides[0] : 0, 0, scale_strides ? scale_strides[1] : 0};
  if (int rc = attn8_args(name, q, q_strides, key_cache, value_cache, kv_strides, key_scales, value_scales,
                          scale_strides ? strides : nullptr, tables, table_stride, width, lens, num_seqs, out, out_strides, rows, hq,
                          hkv, d, page, num_blocks, scale, dtype, &p->a))
    return rc;
  if (reinterpret_cast<uintptr_t>(key_scales) % 4 || reinterpret_cast<uintptr_t>(value_scales) % 4)
    return fail(RLT_EINVAL, "%s: scales must be on 4 bytes", name);
  p->ks = static_cast<const float*>(key_scales);
  p->vs = static_cast<const float*>(value_scales);
  return RLT_OK;
}

}  // namespace
}  // namespace rlt

using namespace rlt;

extern "C" int64_t rlt_paged_decode_int8_workspace_bytes(int64_t n_rows, int64_t max_table_width, int64_t num_q_heads,
                                                         int64_t num_kv_heads, int64_t head_dim, int64_t page_size) {
  if (n_rows <= 0 || max_table_width <= 0 || !decode_i8_shape(num_q_heads, num_kv_heads, head_dim, page_size) ||
      max_table_width > kMaxKeys / page_size)
    return 0;
  return decode_i8_workspace(n_rows, max_table_width * page_size, num_q_heads, head_dim);
}

extern "C" int rlt_paged_decode_int8(const void* q, const int64_t* q_strides, const void* key_cache,
                                     const void* value_cache, const int64_t* kv_strides, const void* key_scales,
                                     const void* value_scales, const int64_t* scale_strides, const int32_t* block_tables,
                                     int64_t table_row_stride, int64_t max_table_width, const int32_t* context_lengths,
                                     void* out, const int64_t* out_strides, int64_t n_rows, int64_t num_q_heads,
                                     int64_t num_kv_heads, int64_t head_dim, int64_t page_size, int64_t num_blocks,
                                     float scale, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* name = "rlt_paged_decode_int8";
  AttnI8Args p;
  if (int rc = attention_args(name, q, q_strides, key_cache, value_cache, kv_strides, key_scales, value_scales,
                              scale_strides, block_tables, table_row_stride, max_table_width, context_lengths, n_rows, out,
                              out_strides, n_rows, num_q_heads, num_kv_heads, head_dim, page_size, num_blocks, scale, dtype, &p))
    return rc;
  if (n_rows == 0) return RLT_OK;
  const int64_t need = rlt_paged_decode_int8_workspace_bytes(n_rows, max_table_width, num_q_heads, num_kv_heads, head_dim, page_size);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(RLT_EWORKSPACE, "%s: workspace must be %lld bytes on 16", name, (long long)need);
  if (decode_i8_shape(p.a.hq, p.a.hkv, p.a.d, p.a.page) && decode8_strides(p.a)) return launch_decode_i8(p, dtype, workspace, as_stream(stream), name);
  return launch_attn_i8_generic(p, dtype, as_stream(stream), name);
}

extern "C" int64_t rlt_paged_prefill_int8_workspace_bytes(int64_t total_q, int64_t num_seqs, int64_t max_table_width,
                                                          int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                                          int64_t page_size) {
  if (total_q <= 0 || num_seqs <= 0 || max_table_width <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      !prefill_i8_shape(head_dim, page_size) || max_table_width > kMaxKeys / page_size)
    return 0;
  return prefill_i8_workspace(total_q, num_seqs, max_table_width * page_size, num_q_heads, head_dim);
}

extern "C" int rlt_paged_prefill_int8(const void* q, const int64_t* q_strides, const void* key_cache,
                                      const void* value_cache, const int64_t* kv_strides, const void* key_scales,
                                      const void* value_scales, const int64_t* scale_strides,
                                      const int32_t* block_tables, int64_t table_row_stride, int64_t max_table_width,
                                      const int32_t* context_lengths, const int32_t* cu_seqlens_q, int64_t num_seqs,
                                      int64_t total_q, int64_t max_seqlen_q, void* out, const int64_t* out_strides,
                                      int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
                                      int64_t num_blocks, float scale, int dtype, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  const char* name = "rlt_paged_prefill_int8";
  AttnI8Args p;
  if (int rc = attention_args(name, q, q_strides, key_cache, value_cache, kv_strides, key_scales, value_scales,
                              scale_strides, block_tables, table_row_stride, max_table_width, context_lengths, num_seqs, out,
                              out_strides, total_q, num_q_heads, num_kv_heads, head_dim, page_size, num_blocks, scale, dtype, &p))
    return rc;
  if (max_seqlen_q < 0) return fail(RLT_EINVAL, "%s: max_seqlen_q is negative", name);
  if (total_q == 0 || num_seqs == 0) return RLT_OK;
  if (!cu_seqlens_q) return fail(RLT_EINVAL, "%s: NULL pointer argument", name);
  p.a.cu = cu_seqlens_q;
  const int64_t need = rlt_paged_prefill_int8_workspace_bytes(total_q, num_seqs, max_table_width, num_q_heads, num_kv_heads,
                                                              head_dim, page_size);
  if (workspace && need > 0 && (workspace_bytes < need || !aligned16(workspace)))
    return fail(RLT_EWORKSPACE, "%s: workspace must be %lld bytes on 16", name, (long long)need);
  if (prefill_i8_shape(p.a.d, p.a.page) && prefill8_strides(p.a)) return launch_prefill_i8(p, dtype, workspace, as_stream(stream), name);
  return launch_attn_i8_generic(p, dtype, as_stream(stream), name);
}
