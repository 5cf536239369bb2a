// Decode over the 8-bit KV cache: one new token a sequence, split over the
// cache's length and joined.
//
// A row's keys are cut into splits of kSplit tokens (longer ones, doubled, where
// kMaxSplits would not cover the row), a function of the row's length alone, so a
// row's bits never depend on its batch.  One workgroup of four waves takes one (row,
// KV head, split): wave w the w-th quarter of its tokens, so a short row's keys are
// all in flight at once.  Rows of one split are written at once; the others leave
// (max, sum, acc) in the workspace for a merge kernel.
//
// Bytes bound it: 2 (D + 1) of them a (token, KV head) against 4 D G flops.  D
// 64/128/256 on the vector units (one or two query heads a KV head): a lane owns 16
// dims of a token (one 16-byte load) and D/16 lanes a token, so one load instruction
// moves 1 KiB of 64 D/16 tokens; codes become fp32 two an instruction.
#include "decode_fp8.hpp"

namespace rlt {
namespace {

constexpr int kWaves = 4;
constexpr int kSplit = 512;
constexpr int kMaxSplits = 64;
constexpr int kXcds = 8;
constexpr int64_t kMaxGrid = 32768;

__host__ __device__ inline void split_plan(int64_t len, int* split_len, int* nsplit) {
  int64_t per = kSplit;
  while (per * kMaxSplits < len) per <<= 1;
  *split_len = static_cast<int>(per);
  *nsplit = static_cast<int>(len > 0 ? (len + per - 1) / per : 1);
}

struct Decode8Args {
  Attn8Args a;
  float* ws_acc;   // [rows][hkv][splits][G][D]
  float2* ws_ml;   // [rows][hkv][splits][G], max in log2 units and sum
  int splits;      // splits a row of the tables' width has
  int split_slots; // split-dimension workgroups launched; each walks every split_slots-th split
  int xcd;         // workgroups of one (split, head) of all rows share an XCD
  int q_vec;       // q rows are 16-byte aligned, dims together
};

__device__ __forceinline__ u32x4 load_codes(const uint8_t* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
}

// 16 codes as fp32.
__device__ __forceinline__ void unpack_codes(const u32x4 w, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2v lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[i]), false);
    const f32x2v hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[i]), true);
    x[4 * i] = lo[0], x[4 * i + 1] = lo[1], x[4 * i + 2] = hi[0], x[4 * i + 3] = hi[1];
  }
}

__device__ __forceinline__ int64_t readlane64(int64_t x, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(x)), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint64_t>(x) >> 32), lane);
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

#ifndef WPE
#define WPE 2
#endif
template <typename T, int D, int G>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(WPE))) void decode8_split_kernel(Decode8Args p) {
  constexpr int LPT = D / 16;      // lanes a token
  constexpr int TPI = 64 / LPT;    // tokens a load instruction
  constexpr int IPU = 16 / TPI;    // load instructions a unit of 16 tokens
  constexpr int TILE = D == 256 ? 32 : 64;
  constexpr int NI = TILE / TPI;   // loads a tile
  constexpr int UPT = TILE / 16;   // units a tile
  constexpr int PARTS = kWaves * TPI;
  __shared__ __align__(16) float part[PARTS][D];
  __shared__ float2 part_ml[G][PARTS];

  const Attn8Args& a = p.a;
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  const uint32_t groups = static_cast<uint32_t>(a.hkv) * p.split_slots;
  uint32_t gi, r;
  if (p.xcd) {  // workgroup b runs on XCD b % 8: the rows of one (split, head) on one XCD, back to back
    const uint32_t t = blockIdx.x / kXcds, rows = static_cast<uint32_t>(a.rows);
    gi = t / rows * kXcds + blockIdx.x % kXcds;
    r = t % rows;
  } else {
    gi = blockIdx.x % groups;
    r = blockIdx.x / groups;
  }
  gi = uniform(gi), r = uniform(r);
  const int h = gi % a.hkv;
  const int len = sequence_length(a, r);
  int split_len, ns;
  split_plan(len, &split_len, &ns);
  const int g = lane / LPT, s = lane % LPT;

  T* orow = static_cast<T*>(a.out) + r * a.o_row;
  const int32_t* trow = a.tables + r * a.table_stride;
  const uint8_t* kh = a.k + h * a.kv_head + 16 * s;
  const uint8_t* vh = a.v + h * a.kv_head + 16 * s;
  const uint8_t* ksh = a.ks + h * a.s_head;
  const uint8_t* vsh = a.vs + h * a.s_head;

  for (int sp = gi / a.hkv; sp < ns; sp += p.split_slots) {
    // The wave's tokens [t0, t0 + n).
    const int quarter = split_len / kWaves;
    const int t0 = sp * split_len + wave * quarter;
    const int n = min(max(len - t0, 0), quarter);
    float q[G][16], acc[G][16], m[G], l[G];
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const T* qrow = static_cast<const T*>(a.q) + r * a.q_row + (h * G + j) * a.q_head;
      if (p.q_vec) {
        constexpr int N = Packet<T>::N;
#pragma unroll
        for (int c = 0; c < 16 / N; ++c) Packet<T>::unpack(*reinterpret_cast<const u32x4*>(qrow + 16 * s + c * N), &q[j][c * N]);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) q[j][e] = load_elem(qrow + (16 * s + e) * a.q_dim);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) q[j][e] *= a.qscale, acc[j][e] = 0.f;
      m[j] = -INFINITY, l[j] = 0.f;
    }
    for (int c0 = 0; c0 < n; c0 += 1024) {  // 64 units, one a lane
      const int left = min(n - c0, 1024);
      const int units = (left + 15) / 16;
      // This lane's unit: where its 16 tokens begin (pages hold whole units).
      const int tok = t0 + c0 + 16 * min(lane, units - 1);
      const int page = tok / a.page, slot = tok - page * a.page;
      const int64_t blk = block_of(a, trow[page]);
      const int64_t unit_kv = blk * a.kv_block + slot * a.kv_token;
      const int64_t unit_s = blk * a.s_block + slot * a.s_token;
      const int last_unit = units - 1, last_tok = left - 1 - 16 * last_unit;
      u32x4 k[NI], v[NI];
      uint32_t kb = 0, vb = 0;
      // Tokens past the end re-read the last one: in bounds, and masked below.
      auto issue = [&](int tile, const uint8_t* base, u32x4 (&x)[NI]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int u = min(tile * UPT + i / IPU, last_unit);
          const int t = min((i % IPU) * TPI + g, u == last_unit ? last_tok : 15);
          x[i] = load_codes(base + readlane64(unit_kv, u) + static_cast<int32_t>(t * static_cast<int32_t>(a.kv_token)));
        }
      };
      auto issue_scales = [&](int tile) __attribute__((always_inline)) {
        const int t = min(tile * TILE + (lane & (TILE - 1)), left - 1);
        const int64_t at = __shfl(unit_s, t >> 4, 64) + (t & 15) * a.s_token;
        kb = ksh[at];
        vb = vsh[at];
      };
      const int tiles = (left + TILE - 1) / TILE;
      issue_scales(0);
      issue(0, kh, k);
      issue(0, vh, v);
      for (int tile = 0; tile < tiles; ++tile) {
        const float sk = scale_value(kb), sv = scale_value(vb), bias = value_bias(vb);
        if (tile + 1 < tiles) issue_scales(tile + 1);
        float score[G][NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          float x[16];
          unpack_codes(k[i], x);
          const float scale = __shfl(sk, i * TPI + g, 64);
          const bool in = tile * TILE + i * TPI + g < left;
#pragma unroll
          for (int j = 0; j < G; ++j) {
            float dot = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) dot = fmaf(q[j][e], x[e], dot);
            dot = group_sum<LPT>(dot) * scale;
            score[j][i] = in ? dot : -INFINITY;
          }
        }
        if (tile + 1 < tiles) issue(tile + 1, kh, k);
        float w[NI], b[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          w[i] = __shfl(sv, i * TPI + g, 64);
          b[i] = __shfl(bias, i * TPI + g, 64);
        }
#pragma unroll
        for (int j = 0; j < G; ++j) {
          float top = m[j];
#pragma unroll
          for (int i = 0; i < NI; ++i) top = fmaxf(top, score[j][i] + b[i]);
          const float off = top == -INFINITY ? 0.f : top;  // only -inf scores so far: they weigh 0
          const float corr = fast_exp2(m[j] - off);
          m[j] = top;
          l[j] *= corr;
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[j][e] *= corr;
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            score[j][i] = fast_exp2(score[j][i] - off);
            l[j] += score[j][i];
            score[j][i] *= w[i];
          }
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          float x[16];
          unpack_codes(v[i], x);
#pragma unroll
          for (int j = 0; j < G; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][e] = fmaf(score[j][i], x[e], acc[j][e]);
        }
        if (tile + 1 < tiles) issue(tile + 1, vh, v);
      }
    }
    // Join the waves' token groups, in a fixed order.
#pragma unroll
    for (int j = 0; j < G; ++j)
      if (s == 0) part_ml[j][wave * TPI + g] = make_float2(m[j], l[j]);
#pragma unroll
    for (int j = 0; j < G; ++j) {
      if (j) __syncthreads();
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        u32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __float_as_uint(acc[j][4 * c + e]);
        *reinterpret_cast<u32x4*>(&part[wave * TPI + g][16 * s + 4 * c]) = x;
      }
      __syncthreads();
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < PARTS; ++i) top = fmaxf(top, part_ml[j][i].x);
      const float off = top == -INFINITY ? 0.f : top;
      const int d = threadIdx.x;
      if (d < D) {
        float sum = 0.f, x = 0.f;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          const float2 ml = part_ml[j][i];
          const float w = fast_exp2(ml.x - off);
          sum = fmaf(ml.y, w, sum);
          x = fmaf(part[i][d], w, x);
        }
        if (ns == 1) {
          store_elem(orow + (h * G + j) * a.o_head + d * a.o_dim, len > 0 ? x * (1.f / sum) : 0.f);
        } else {
          const int64_t at = ((static_cast<int64_t>(r) * a.hkv + h) * p.splits + sp) * G + j;
          p.ws_acc[at * D + d] = x;
          if (d == 0) p.ws_ml[at] = make_float2(top, sum);
        }
      }
    }
    __syncthreads();
  }
}

// One wave a (row, query head) of more than one split: lane i holds split i's
// (max, sum), and the accumulators are added in split order.
template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) void decode8_merge_kernel(Decode8Args p) {
  const Attn8Args& a = p.a;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
  if (item >= a.rows * a.hq) return;
  const int lane = threadIdx.x & 63;
  const int r = static_cast<int>(item / a.hq), hq = static_cast<int>(item - static_cast<int64_t>(r) * a.hq);
  const int G = a.hq / a.hkv, h = hq / G, j = hq - h * G;
  int split_len, ns;
  split_plan(sequence_length(a, r), &split_len, &ns);
  if (ns < 2) return;
  const int64_t base = (static_cast<int64_t>(r) * a.hkv + h) * p.splits * G + j;
  const float2 ml = lane < ns ? p.ws_ml[base + static_cast<int64_t>(lane) * G] : make_float2(-INFINITY, 0.f);
  const float top = group_max<64>(ml.x);
  const float off = top == -INFINITY ? 0.f : top;
  const float w = lane < ns ? fast_exp2(ml.x - off) : 0.f;
  const float inv = 1.f / group_sum<64>(ml.y * w);
  constexpr int E = D / 64;
  float acc[E] = {};
  const float* src = p.ws_acc + base * D + lane;
  constexpr int BATCH = 8;
  for (int s0 = 0; s0 < ns; s0 += BATCH) {
    float x[BATCH][E];
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) x[i][e] = src[static_cast<int64_t>(min(s0 + i, ns - 1)) * G * D + 64 * e];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const float wi = s0 + i < ns ? __shfl(w, s0 + i, 64) : 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = s0 + i < ns ? fmaf(x[i][e], wi, acc[e]) : acc[e];
    }
  }
  T* orow = static_cast<T*>(a.out) + r * a.o_row + hq * a.o_head;
#pragma unroll
  for (int e = 0; e < E; ++e) store_elem(orow + (lane + 64 * e) * a.o_dim, acc[e] * inv);
}

template <typename T, int D>
void launch_shape(const Decode8Args& p, int G, unsigned grid, hipStream_t stream) {
  const dim3 block(64 * kWaves);
  switch (G) {
    case 1: hipLaunchKernelGGL((decode8_split_kernel<T, D, 1>), dim3(grid), block, 0, stream, p); break;
    default: hipLaunchKernelGGL((decode8_split_kernel<T, D, 2>), dim3(grid), block, 0, stream, p); break;
  }
  if (p.splits > 1) {
    const unsigned merge = static_cast<unsigned>((p.a.rows * p.a.hq + kWaves - 1) / kWaves);
    hipLaunchKernelGGL((decode8_merge_kernel<T, D>), dim3(merge), block, 0, stream, p);
  }
}

template <typename T>
void launch_type(const Decode8Args& p, int G, unsigned grid, hipStream_t stream) {
  switch (p.a.d) {
    case 64: launch_shape<T, 64>(p, G, grid, stream); break;
    case 128: launch_shape<T, 128>(p, G, grid, stream); break;
    default: launch_shape<T, 256>(p, G, grid, stream); break;
  }
}

}  // namespace

bool decode8_shape(int64_t hq, int64_t hkv, int64_t d, int64_t page) {
  const int64_t G = hkv > 0 ? hq / hkv : 0;
  return (d == 64 || d == 128 || d == 256) && page % 16 == 0 && (G == 1 || G == 2);
}

int64_t decode8_workspace(int64_t rows, int64_t max_len, int64_t hq, int64_t d) {
  int per, ns;
  split_plan(max_len, &per, &ns);
  return ns > 1 ? rows * ns * hq * (d + 2) * 4 : 0;
}

bool decode8_layout(const Attn8Args& a) {
  auto rows16 = [](const void* x) { return aligned16(x); };
  return decode8_shape(a.hq, a.hkv, a.d, a.page) && a.kv_dim == 1 && rows16(a.k) && rows16(a.v) && a.kv_head % 16 == 0 &&
         a.kv_token % 16 == 0 && a.kv_block % 16 == 0 && a.kv_token < (int64_t(1) << 27);
}

int launch_decode8(const Attn8Args& a, int dtype, void* ws, hipStream_t stream, const char* name) {
  Decode8Args p{};
  p.a = a;
  int per;
  split_plan(a.max_len, &per, &p.splits);
  const int64_t items = a.rows * a.hkv;
  p.split_slots = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(p.splits, kMaxGrid / items)));
  p.xcd = a.hkv * p.split_slots % kXcds == 0;
  const int es = dtype_size(dtype);
  p.q_vec = a.q_dim == 1 && aligned16(a.q) && a.q_row * es % 16 == 0 && a.q_head * es % 16 == 0;
  p.ws_acc = static_cast<float*>(ws);
  p.ws_ml = reinterpret_cast<float2*>(p.ws_acc + a.rows * p.splits * a.hq * a.d);
  const unsigned grid = static_cast<unsigned>(items * p.split_slots);
  const int G = a.hq / a.hkv;
  switch (dtype) {
    case RLT_BFLOAT16: launch_type<bf16>(p, G, grid, stream); break;
    case RLT_FLOAT16: launch_type<f16>(p, G, grid, stream); break;
    default: launch_type<float>(p, G, grid, stream); break;
  }
  return check_launch(name);
}

}  // namespace rlt
