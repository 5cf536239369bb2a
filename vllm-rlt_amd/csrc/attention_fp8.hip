// Attention over the 8-bit paged KV cache (codes and scales: fp8.hpp):
//   s_j = scale * q . (K_j 2^ek_j),  out = sum_j softmax(s)_j (V_j 2^ev_j)
// over a sequence's keys, for one new token a sequence (decode) and for packed
// chunks, bottom-right causal (prefill).  Scores, softmax sums and the sums of p V are
// fp32, outputs of q's type; the scales multiply the score and the probability of their
// token, or become part of a bf16 that holds their code exactly.
#include "decode_fp8.hpp"
#include "fp8.hpp"
#include "prefill_fp8.hpp"

namespace rlt {
namespace {

// Any head size up to 64 * kPerLane, page size, grouping and strides: one
// workgroup a (row, query head), wave w takes tokens w, w + kGenericWaves, ...
// with the head's dims over its lanes and a running maximum and sum of its own;
// the waves are joined through LDS in wave order.  Every query head reads its keys itself, a
// byte a lane: latency bounds it (64 rows of 512-4096 tokens, 16 heads x 80: 1112 us).
constexpr int kPerLane = 8;
constexpr int kGenericWaves = 8;

template <typename T>
__global__ __launch_bounds__(64 * kGenericWaves) void attn8_generic_kernel(Attn8Args a) {
  const int64_t row = blockIdx.x;
  const int h = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  int seq = static_cast<int>(row), len;
  if (a.cu) {
    int lo = 0, hi = a.num_seqs;  // the last sequence that begins at or before row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu[mid] <= row) lo = mid;
      else hi = mid;
    }
    if (row < a.cu[lo] || row >= a.cu[lo + 1]) return;  // a row of no sequence is left as it was
    seq = lo;
    const int64_t n = sequence_length(a, seq) - (a.cu[lo + 1] - 1 - row);
    len = static_cast<int>(n < 0 ? 0 : n);
  } else {
    len = sequence_length(a, seq);
  }
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
  const int32_t* trow = a.tables + seq * a.table_stride;
  float m = -INFINITY, l = 0.f;
  for (int t = wave; t < len; t += kGenericWaves) {
    const int64_t blk = block_of(a, trow[t / a.page]);
    const int64_t slot = t % a.page;
    const int64_t base = blk * a.kv_block + slot * a.kv_token + kvh * a.kv_head;
    const int64_t sbase = blk * a.s_block + slot * a.s_token + kvh * a.s_head;
    const uint32_t vb = a.vs[sbase];
    const float sk = scale_value(a.ks[sbase]), sv = scale_value(vb);
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < kPerLane; ++c) {
      const int d = lane + 64 * c;
      if (d < a.d) dot = fmaf(qv[c], code_value(a.k[base + d * a.kv_dim]), dot);
    }
    dot = group_sum<64>(dot) * sk;
    const float mn = fmaxf(m, dot + value_bias(vb));
    const float off = mn == -INFINITY ? 0.f : mn;  // only -inf scores so far: they weigh 0
    const float corr = fast_exp2(m - off);
    const float p = fast_exp2(dot - off);
    l = l * corr + p;
    const float pv = p * kLift * sv;
#pragma unroll
    for (int c = 0; c < kPerLane; ++c) {
      const int d = lane + 64 * c;
      if (d < a.d) acc[c] = fmaf(pv, code_value(a.v[base + d * a.kv_dim]), acc[c] * corr);
    }
    m = mn;
  }
  __shared__ float ms[kGenericWaves], ls[kGenericWaves], accs[kGenericWaves][64 * kPerLane];
  if (lane == 0) {
    ms[wave] = m;
    ls[wave] = l;
  }
#pragma unroll
  for (int c = 0; c < kPerLane; ++c) accs[wave][lane + 64 * c] = acc[c];
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kGenericWaves; ++w) top = fmaxf(top, ms[w]);
  const float off = top == -INFINITY ? 0.f : top;
  float sum = 0.f, weight[kGenericWaves];
#pragma unroll
  for (int w = 0; w < kGenericWaves; ++w) {
    weight[w] = fast_exp2(ms[w] - off);
    sum += ls[w] * weight[w];
  }
  const float inv = 1.f / kLift / sum;
  for (int d = threadIdx.x; d < a.d; d += 64 * kGenericWaves) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kGenericWaves; ++w) x = fmaf(accs[w][d], weight[w], x);
    store_elem(orow + d * a.o_dim, len > 0 ? x * inv : 0.f);
  }
}

// Checks what both calls share and fills the arguments.
int attention_args(const char* name, const void* q, const int64_t* q_strides, const void* key_cache,
                   const void* value_cache, const int64_t* kv_strides, const void* key_scales,
                   const void* value_scales, const int64_t* scale_strides, const int32_t* tables,
                   int64_t table_stride, int64_t width, const int32_t* lens, int64_t num_seqs, void* out,
                   const int64_t* out_strides, int64_t rows, int64_t hq, int64_t hkv, int64_t d, int64_t page,
                   int64_t num_blocks, float scale, int dtype, Attn8Args* a) {
  if (!dtype_size(dtype)) return fail(RLT_EINVAL, "%s: unknown dtype %d", name, dtype);
  if (rows < 0 || num_seqs < 0) return fail(RLT_EINVAL, "%s: negative row count", name);
  if (hkv <= 0 || hq <= 0 || hq % hkv) return fail(RLT_EINVAL, "%s: query heads must be a positive multiple of KV heads", name);
  if (d <= 0 || page <= 0 || num_blocks <= 0 || width <= 0 || table_stride < 0)
    return fail(RLT_EINVAL, "%s: head_dim, page_size, num_blocks and the table width must be positive", name);
  if (d > 64 * kPerLane) return fail(RLT_EUNSUPPORTED, "%s: head_dim above %d", name, 64 * kPerLane);
  if (rows > kMaxRows || num_seqs > 0x7fffffff || hq > 65535 || page > 0x7fffffff || num_blocks > 0x7fffffff)
    return fail(RLT_EUNSUPPORTED, "%s: too many rows, heads, tokens a page or blocks", name);
  if (width > kMaxKeys / page) return fail(RLT_EUNSUPPORTED, "%s: the tables cover more than 2^30 tokens", name);
  if (rows == 0 || num_seqs == 0) return RLT_OK;
  if (!q || !q_strides || !key_cache || !value_cache || !kv_strides || !key_scales || !value_scales ||
      !scale_strides || !tables || !lens || !out || !out_strides)
    return fail(RLT_EINVAL, "%s: NULL pointer argument", name);
  *a = Attn8Args{};
  a->q = q;
  a->q_row = q_strides[0], a->q_head = q_strides[1], a->q_dim = q_strides[2];
  a->k = static_cast<const uint8_t*>(key_cache);
  a->v = static_cast<const uint8_t*>(value_cache);
  a->kv_block = kv_strides[0], a->kv_token = kv_strides[1], a->kv_head = kv_strides[2], a->kv_dim = kv_strides[3];
  a->ks = static_cast<const uint8_t*>(key_scales);
  a->vs = static_cast<const uint8_t*>(value_scales);
  a->s_block = scale_strides[0], a->s_token = scale_strides[1], a->s_head = scale_strides[2];
  a->tables = tables;
  a->table_stride = table_stride;
  a->lens = lens;
  a->num_seqs = static_cast<int>(num_seqs);
  a->out = out;
  a->o_row = out_strides[0], a->o_head = out_strides[1], a->o_dim = out_strides[2];
  a->rows = rows;
  a->hq = static_cast<int>(hq), a->hkv = static_cast<int>(hkv), a->d = static_cast<int>(d);
  a->page = static_cast<int>(page);
  a->num_blocks = num_blocks;
  a->max_len = width * page;
  a->qscale = scale * 1.4426950408889634f;
  return RLT_OK;
}

}  // namespace

int launch_attn8_generic(const Attn8Args& a, int dtype, hipStream_t stream, const char* name) {
  const dim3 grid(static_cast<unsigned>(a.rows), static_cast<unsigned>(a.hq)), block(64 * kGenericWaves);
  switch (dtype) {
    case RLT_BFLOAT16: hipLaunchKernelGGL((attn8_generic_kernel<bf16>), grid, block, 0, stream, a); break;
    case RLT_FLOAT16: hipLaunchKernelGGL((attn8_generic_kernel<f16>), grid, block, 0, stream, a); break;
    default: hipLaunchKernelGGL((attn8_generic_kernel<float>), grid, block, 0, stream, a); break;
  }
  return check_launch(name);
}

}  // namespace rlt

using namespace rlt;

extern "C" int64_t rlt_paged_decode_fp8_workspace_bytes(int64_t n_rows, int64_t max_table_width, int64_t num_q_heads,
                                                        int64_t num_kv_heads, int64_t head_dim, int64_t page_size) {
  if (n_rows <= 0 || max_table_width <= 0 || !decode8_shape(num_q_heads, num_kv_heads, head_dim, page_size) ||
      max_table_width > kMaxKeys / page_size)
    return 0;
  return decode8_workspace(n_rows, max_table_width * page_size, num_q_heads, num_kv_heads, head_dim);
}

extern "C" int rlt_paged_decode_fp8(const void* q, const int64_t* q_strides, const void* key_cache,
                                    const void* value_cache, const int64_t* kv_strides, const void* key_scales,
                                    const void* value_scales, const int64_t* scale_strides, const int32_t* block_tables,
                                    int64_t table_row_stride, int64_t max_table_width, const int32_t* context_lengths,
                                    void* out, const int64_t* out_strides, int64_t n_rows, int64_t num_q_heads,
                                    int64_t num_kv_heads, int64_t head_dim, int64_t page_size, int64_t num_blocks,
                                    float scale, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  Attn8Args a;
  if (int rc = attention_args("rlt_paged_decode_fp8", q, q_strides, key_cache, value_cache, kv_strides, key_scales,
                              value_scales, scale_strides, block_tables, table_row_stride, max_table_width,
                              context_lengths, n_rows, out, out_strides, n_rows, num_q_heads, num_kv_heads, head_dim,
                              page_size, num_blocks, scale, dtype, &a))
    return rc;
  if (n_rows == 0) return RLT_OK;
  const int64_t need = rlt_paged_decode_fp8_workspace_bytes(n_rows, max_table_width, num_q_heads, num_kv_heads, head_dim, page_size);
  if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 8))
    return fail(RLT_EWORKSPACE, "rlt_paged_decode_fp8: workspace must be %lld bytes on 8", (long long)need);
  if (!decode8_layout(a)) return launch_attn8_generic(a, dtype, as_stream(stream), "rlt_paged_decode_fp8");
  return launch_decode8(a, dtype, workspace, as_stream(stream), "rlt_paged_decode_fp8");
}

extern "C" int64_t rlt_paged_prefill_fp8_workspace_bytes(int64_t total_q, int64_t num_seqs, int64_t max_table_width,
                                                         int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                                         int64_t page_size) {
  if (total_q <= 0 || num_seqs <= 0 || max_table_width <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      !prefill8_shape(head_dim, page_size) || max_table_width > kMaxKeys / page_size)
    return 0;
  return prefill8_workspace(total_q, num_seqs, max_table_width * page_size, num_q_heads, head_dim);
}

extern "C" int rlt_paged_prefill_fp8(const void* q, const int64_t* q_strides, const void* key_cache,
                                     const void* value_cache, const int64_t* kv_strides, const void* key_scales,
                                     const void* value_scales, const int64_t* scale_strides,
                                     const int32_t* block_tables, int64_t table_row_stride, int64_t max_table_width,
                                     const int32_t* context_lengths, const int32_t* cu_seqlens_q, int64_t num_seqs,
                                     int64_t total_q, int64_t max_seqlen_q, void* out, const int64_t* out_strides,
                                     int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
                                     int64_t num_blocks, float scale, int dtype, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
  Attn8Args a;
  if (int rc = attention_args("rlt_paged_prefill_fp8", q, q_strides, key_cache, value_cache, kv_strides, key_scales,
                              value_scales, scale_strides, block_tables, table_row_stride, max_table_width,
                              context_lengths, num_seqs, out, out_strides, total_q, num_q_heads, num_kv_heads,
                              head_dim, page_size, num_blocks, scale, dtype, &a))
    return rc;
  if (max_seqlen_q < 0) return fail(RLT_EINVAL, "rlt_paged_prefill_fp8: max_seqlen_q is negative");
  if (total_q == 0 || num_seqs == 0) return RLT_OK;
  if (!cu_seqlens_q) return fail(RLT_EINVAL, "rlt_paged_prefill_fp8: NULL pointer argument");
  a.cu = cu_seqlens_q;
  const int64_t need = rlt_paged_prefill_fp8_workspace_bytes(total_q, num_seqs, max_table_width, num_q_heads, num_kv_heads,
                                                             head_dim, page_size);
  if (workspace && need > 0 && (workspace_bytes < need || !aligned16(workspace)))
    return fail(RLT_EWORKSPACE, "rlt_paged_prefill_fp8: workspace must be %lld bytes on 16", (long long)need);
  if (prefill8_layout(a)) return launch_prefill8(a, dtype, workspace, as_stream(stream), "rlt_paged_prefill_fp8");
  return launch_attn8_generic(a, dtype, as_stream(stream), "rlt_paged_prefill_fp8");
}
