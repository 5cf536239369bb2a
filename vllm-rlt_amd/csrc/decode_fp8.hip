// Decode over the 8-bit KV cache: one new token a sequence, split over the cache's
// length and joined.  Here: which kernel a call takes, the merge of the splits, and the
// split pass of head_dim 64 with one query head a KV head, on the vector units.
//
// A row's keys are cut into splits (decode8_split_plan), a function of the row's length
// alone; a split's parts and then the splits are joined in order.  So a row's bits depend
// neither on its batch nor on how the parts are spread over waves.
//
// The split pass here.  A split is kParts parts of consecutive tokens, each worked by 4
// lanes a head in order, with a running maximum and sum of its own.  Bytes bound it: 2 (D +
// 1) of them a (token, head) against 4 D flops.  A lane owns 16 dims of a (token, head).  A
// wave works on HPW neighbouring heads of PPI parts at once: a load instruction moves HPW *
// 64 contiguous bytes of PPI tokens.  After 4 instructions (a tile, 64 (token, head) rows) a
// reduce-scatter leaves one row's score in every lane, which does one row's softmax.  Wide
// waves read the longest runs of memory; narrow ones, of more parts, give a small launch
// more waves.  Measured (16 heads, bf16): 256 rows of 1024-8192 tokens 434 us, 5.65 TB/s.
#include <type_traits>

#include "decode_fp8.hpp"

namespace rlt {
namespace {

constexpr int kWaves = 4;
constexpr int kParts = 16;
constexpr int kUnit = 16;  // tokens of a page looked up at once (pages hold whole units), and of the shortest part
constexpr int kXcds = 8;
constexpr int kCus = 256;
constexpr int64_t kMaxGrid = 32768;

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

// Sum over the 4 lanes of a group of 4 values at once: lane s of the group ends with the
// sum of value s.  Every step halves the values a lane still carries.
__device__ __forceinline__ float reduce_scatter(float (&x)[4], int s) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool up = s & 2;
    const float keep = up ? x[i + 2] : x[i], send = up ? x[i] : x[i + 2];
    x[i] = keep + dpp<kDppXor2>(send);
  }
  const bool up = s & 1;
  const float keep = up ? x[1] : x[0], send = up ? x[0] : x[1];
  return keep + dpp<kDppXor1>(send);
}

template <typename T, int HPW, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2))) void decode8_split_kernel(Decode8Args p) {
  constexpr int D = 64, LPT = D / 16;      // lanes a (token, head), and tokens (load instructions) a tile
  constexpr int PPI = 64 / (LPT * HPW);    // parts a wave works on at once
  constexpr int PPW = kParts / (W * PPI);  // parts a group of lanes works through
  constexpr int TPU = kUnit / LPT;         // tiles a unit
  static_assert(LPT * HPW * PPI == 64 && PPW * W * PPI == kParts && TPU * LPT == kUnit, "whole groups, parts and tiles");
  __shared__ __align__(16) float part[kParts][HPW][D];
  __shared__ float2 part_ml[kParts][HPW];

  const Attn8Args& a = p.a;
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  const uint32_t rows = static_cast<uint32_t>(a.rows), x = blockIdx.x % kXcds, t = blockIdx.x / kXcds;
  const uint32_t blocks = a.hkv / HPW;
  uint32_t gi, r;
  if (p.xcd) {  // workgroup b runs on XCD b % 8: the heads of a (split, row) on one XCD, back to back
    const uint32_t item = t / blocks * kXcds + x;
    gi = item / rows * blocks + t % blocks;
    r = (item + item / rows) % rows;  // a row's splits on different ones
  } else {
    gi = blockIdx.x / rows;
    r = blockIdx.x % rows;
  }
  gi = uniform(gi), r = uniform(r);
  const int h0 = gi % blocks * HPW;
  const int len = sequence_length(a, r);
  int split_len, ns;
  decode8_split_plan(len, kParts * kUnit, &split_len, &ns);
  const int s = lane % LPT, gh = lane / LPT % HPW, gp = lane / (LPT * HPW), group0 = lane & ~(LPT - 1);
  const int part_len = split_len / kParts;
  const uint32_t units = static_cast<uint32_t>(part_len) / kUnit;  // a part, a power of two
  const int unit_shift = 31 - __builtin_clz(units);

  T* orow = static_cast<T*>(a.out) + r * a.o_row;
  const int32_t* trow = a.tables + r * a.table_stride;
  const uint8_t* kh = a.k + h0 * a.kv_head;
  const uint8_t* vh = a.v + h0 * a.kv_head;
  const uint8_t* ksh = a.ks + (h0 + gh) * a.s_head;
  const uint8_t* vsh = a.vs + (h0 + gh) * a.s_head;
  const uint32_t token_bytes = static_cast<uint32_t>(a.kv_token);
  const int64_t lane_off = gh * a.kv_head + 16 * s;

  for (int sp = gi / blocks; sp < ns; sp += p.split_slots) {
    const int n_split = min(len - sp * split_len, split_len);
    // Steps of this wave: unit u of its k-th parts, as far as its first group has tokens.
    const int wave_tok = wave * (PPW * PPI) * part_len;
    const int rel = n_split - wave_tok;
    uint32_t tiles = 0;
    if (rel > 0) {
      const int round = PPI * part_len;  // tokens from one part of a group to its next
      const int k = min(rel / round, PPW), rem = k < PPW ? rel - k * round : 0;
      tiles = k * (units * TPU) + (min(rem, part_len) + LPT - 1) / LPT;
    }
    // The first token of a step's unit in this lane's group.
    auto unit_token = [&](uint32_t step) __attribute__((always_inline)) {
      return sp * split_len + wave_tok + static_cast<int>((step >> unit_shift) * PPI + gp) * part_len +
             static_cast<int>(step & (units - 1)) * kUnit;
    };
    float q[16], acc[16], m = -INFINITY, l = 0.f;
    if (!p.q_vec) {  // any strides: through LDS, a few elements a thread
#pragma unroll 1
      for (int o = threadIdx.x; o < HPW * D; o += 64 * W)
        (&part[0][0][0])[o] = load_elem(static_cast<const T*>(a.q) + r * a.q_row + (h0 + o / D) * a.q_head + o % D * a.q_dim);
      __syncthreads();
    }
    if (p.q_vec) {
      const T* qrow = static_cast<const T*>(a.q) + r * a.q_row + (h0 + gh) * a.q_head + 16 * s;
      constexpr int N = Packet<T>::N;
#pragma unroll
      for (int c = 0; c < 16 / N; ++c) Packet<T>::unpack(*reinterpret_cast<const u32x4*>(qrow + c * N), &q[c * N]);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) q[e] = part[0][0][gh * D + 16 * s + e];
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) q[e] *= a.qscale, acc[e] = 0.f;
    if (!p.q_vec) __syncthreads();

    if (tiles > 0) {
      const int last_unit = (len - 1) / kUnit * kUnit;
      int64_t entry_kv, entry_s;  // lane s of a group: where the group's unit of step chunk * LPT + s begins
      int64_t off, off_s;         // where this lane's unit of the tile being loaded begins
      int lim;                    // its last token
      uint32_t kb, vb;
      u32x4 k[LPT], v[LPT];
      // A unit past the row's end is replaced by the row's last, and a token past it by
      // its last token: in bounds, and masked below.
      auto load_entries = [&](uint32_t chunk) __attribute__((always_inline)) {
        const int tok = min(unit_token(chunk * LPT + s), last_unit);
        const int page = tok / a.page, slot = tok - page * a.page;
        const int64_t blk = block_of(a, trow[page]);
        entry_kv = blk * a.kv_block + slot * a.kv_token;
        entry_s = blk * a.s_block + slot * a.s_token;
      };
      auto find_unit = [&](uint32_t step) __attribute__((always_inline)) {
        if (step % LPT == 0) load_entries(step / LPT);
        const int from = group0 + static_cast<int>(step % LPT);
        off = __shfl(entry_kv, from, 64) + lane_off;
        off_s = __shfl(entry_s, from, 64);
        lim = min(len - 1 - min(unit_token(step), last_unit), kUnit - 1);
      };
      auto issue = [&](uint32_t tile, const uint8_t* base, u32x4 (&y)[LPT]) __attribute__((always_inline)) {
        const uint32_t first = tile % TPU * LPT;
#pragma unroll
        for (uint32_t i = 0; i < LPT; ++i)
          y[i] = load_codes(base + (off + __umul24(min(first + i, static_cast<uint32_t>(lim)), token_bytes)));
      };
      // This lane's row of a tile: token s, head gh.
      auto issue_scales = [&](uint32_t tile) __attribute__((always_inline)) {
        const int64_t at = off_s + min(static_cast<int>(tile % TPU * LPT) + s, lim) * a.s_token;
        kb = ksh[at];
        vb = vsh[at];
      };
      auto step = [&](uint32_t tile, auto more) __attribute__((always_inline)) {
        constexpr bool MORE = decltype(more)::value;  // another tile follows
        float score[LPT];
#pragma unroll
        for (int i = 0; i < LPT; ++i) {
          float y[16];
          unpack_codes(k[i], y);
          score[i] = q[0] * y[0];
#pragma unroll
          for (int e = 1; e < 16; ++e) score[i] = fmaf(q[e], y[e], score[i]);
          __builtin_amdgcn_sched_barrier(0);
        }
        const float sk = scale_value(kb), sv = scale_value(vb), bias = value_bias(vb);
        const bool in = unit_token(tile / TPU) + static_cast<int>(tile % TPU * LPT) + s < len;
        if constexpr (MORE) {
          if ((tile + 1) % TPU == 0) find_unit((tile + 1) / TPU);
          issue_scales(tile + 1);
          issue(tile + 1, kh, k);
          __builtin_amdgcn_sched_barrier(0);
        }
        const float sum = reduce_scatter(score, s) * sk;
        const float dot = in ? sum : -INFINITY;
        const float top = fmaxf(m, group_max<LPT>(dot + bias));
        const float base = top == -INFINITY ? 0.f : top;  // only -inf scores so far: they weigh 0
        const float corr = fast_exp2(m - base);
        const float w = fast_exp2(dot - base);
        m = top;
        l = fmaf(l, corr, w);
        const float pv = w * kLift * sv;  // this lane's row: its probability times its V scale
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] *= corr;
#pragma unroll
        for (int i = 0; i < LPT; ++i) {
          float y[16];
          unpack_codes(v[i], y);
          const float wi = __shfl(pv, group0 + i, 64);
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[e] = fmaf(wi, y[e], acc[e]);
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (MORE) {
          issue(tile + 1, vh, v);
          __builtin_amdgcn_sched_barrier(0);
        }
        // The end of a part: its state to LDS.
        if (!MORE || (tile + 1) % (units * TPU) == 0) {
          const int pt = (wave * PPW + static_cast<int>(tile / TPU >> unit_shift)) * PPI + gp;
          const float sum = group_sum<LPT>(l);
          if (s == 0) part_ml[pt][gh] = make_float2(m, sum);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            u32x4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = __float_as_uint(acc[4 * c + e]), acc[4 * c + e] = 0.f;
            *reinterpret_cast<u32x4*>(&part[pt][gh][16 * s + 4 * c]) = y;
          }
          m = -INFINITY, l = 0.f;
        }
      };
      find_unit(0);
      issue_scales(0);
      issue(0, kh, k);
      issue(0, vh, v);
#pragma unroll 1
      for (uint32_t tile = 0; tile + 1 < tiles; ++tile) step(tile, std::true_type{});
      step(tiles - 1, std::false_type{});
    }
    __syncthreads();
    // Join the parts that have tokens, in order.
    const int live = (n_split + part_len - 1) / part_len;
#pragma unroll 1
    for (int o = threadIdx.x; o < HPW * D; o += 64 * W) {
      const int hd = o / D, d = o % D, h = h0 + hd;
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < kParts; ++i)
        if (i < live) top = fmaxf(top, part_ml[i][hd].x);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f, y = 0.f;
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        if (i >= live) break;
        const float2 ml = part_ml[i][hd];
        const float w = fast_exp2(ml.x - base);
        sum = fmaf(ml.y, w, sum);
        y = fmaf(part[i][hd][d], w, y);
      }
      if (ns == 1) {
        store_elem(orow + h * a.o_head + d * a.o_dim, len > 0 ? y * (1.f / kLift / sum) : 0.f);
      } else {
        const int64_t at = (static_cast<int64_t>(r) * a.hkv + h) * p.splits + sp;
        p.ws_acc[at * D + d] = y;
        if (d == 0) p.ws_ml[at] = make_float2(top, sum);
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
  decode8_split_plan(sequence_length(a, r), p.base, &split_len, &ns);
  if (ns < 2) return;
  const int64_t base = (static_cast<int64_t>(r) * a.hkv + h) * p.splits * G + j;
  constexpr int E = D / 64;
  constexpr int BATCH = 8;
  const float* src = p.ws_acc + base * D + lane;
  float x[BATCH][E], acc[E] = {};
  auto load = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) x[i][e] = src[static_cast<int64_t>(min(s0 + i, ns - 1)) * G * D + 64 * e];
  };
  const float2 ml = lane < ns ? p.ws_ml[base + static_cast<int64_t>(lane) * G] : make_float2(-INFINITY, 0.f);
  load(0);  // on its way while the weights are worked out
  const float top = group_max<64>(ml.x);
  const float off = top == -INFINITY ? 0.f : top;
  const float w = lane < ns ? fast_exp2(ml.x - off) : 0.f;
  const float inv = 1.f / kLift / group_sum<64>(ml.y * w);
  for (int s0 = 0; s0 < ns; s0 += BATCH) {
    if (s0) load(s0);
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

template <typename T>
void launch_split(const Decode8Args& p, unsigned grid, hipStream_t stream) {
  switch (p.hpw) {
    case 8: hipLaunchKernelGGL((decode8_split_kernel<T, 8, 4>), dim3(grid), dim3(256), 0, stream, p); break;
    case 4: hipLaunchKernelGGL((decode8_split_kernel<T, 4, 4>), dim3(grid), dim3(256), 0, stream, p); break;
    case 2: hipLaunchKernelGGL((decode8_split_kernel<T, 2, 2>), dim3(grid), dim3(128), 0, stream, p); break;
    default: hipLaunchKernelGGL((decode8_split_kernel<T, 1, 1>), dim3(grid), dim3(64), 0, stream, p); break;
  }
}

template <typename T>
void launch_merge(const Decode8Args& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.a.rows * p.a.hq + kWaves - 1) / kWaves)), block(64 * kWaves);
  switch (p.a.d) {
    case 64: hipLaunchKernelGGL((decode8_merge_kernel<T, 64>), grid, block, 0, stream, p); break;
    case 128: hipLaunchKernelGGL((decode8_merge_kernel<T, 128>), grid, block, 0, stream, p); break;
    default: hipLaunchKernelGGL((decode8_merge_kernel<T, 256>), grid, block, 0, stream, p); break;
  }
}

// Heads a wave: as many neighbours as divide the heads and leave a workgroup for three CUs
// in four.  Measured, us (16 heads x 64, bf16, 1 / 2 / 4 / 8 heads a wave): 4 rows of up to
// 256 tokens 6.3 / 6.8 / 7.0 / 11.2, 16 of up to 512 10.9 / 10.8 / 11.0 / 15.4, 1 of 8000
// 12.6 / 12.5 / 12.7 / 16.6, 256 of up to 256 32.0 / 23.7 / 22.3 / 21.8, 64 of 512-4096 93.9
// / 63.3 / 61.6 / 62.7, 256 of 1024-8192 751 / 474 / 450 / 434.
int heads_a_wave(const Attn8Args& a, int64_t splits) {
  int hpw = 1;
  while (hpw < 8 && a.hkv % (2 * hpw) == 0 &&
         a.rows * (a.hkv / (2 * hpw)) * splits >= kCus * 3 / 4)
    hpw *= 2;
  return hpw;
}

}  // namespace

bool decode8_shape(int64_t hq, int64_t hkv, int64_t d, int64_t page) {
  return (d == 64 || d == 128 || d == 256) && page > 0 && page % kUnit == 0 && hkv > 0 && hq > 0;
}

// Which kernel.  The matrix cores leave 15 columns of 16 empty for one query head a KV head,
// and pay there only from head_dim 128 on, where all but the smallest launches gain and a
// single row loses.  Measured, us, vector units / matrix cores: 16 heads x 64, 64 rows of
// 512-4096 tokens 64 / 90; 16 x 128 121 / 116, 256 rows of 1024-8192 850 / 821, 16 of up to 512
// 11.9 / 10.3, 4 of up to 256 6.5 / 6.9, 1 of 1000 10.3 / 12.4; 16 + 8 heads x 64, 64 rows of
// 512-4096 54 / 48.
bool on_matrix_cores(int64_t hq, int64_t hkv, int64_t d) { return hq > hkv || d > 64; }
int split_base(int64_t hq, int64_t hkv, int64_t d) { return on_matrix_cores(hq, hkv, d) ? kMfmaSplit : kParts * kUnit; }

int64_t decode8_workspace(int64_t rows, int64_t max_len, int64_t hq, int64_t hkv, int64_t d) {
  const int64_t ns = decode8_most_splits(max_len, split_base(hq, hkv, d));
  return ns > 1 ? rows * ns * hq * (d + 2) * 4 : 0;
}

bool decode8_layout(const Attn8Args& a) { return decode8_shape(a.hq, a.hkv, a.d, a.page) && decode8_strides(a); }
bool decode8_strides(const Attn8Args& a) {
  auto near = [](int64_t x) { return x >= 0 && x < (int64_t(1) << 24) && x % 16 == 0; };
  return a.kv_dim == 1 && aligned16(a.k) && aligned16(a.v) && near(a.kv_head) &&
         near(a.kv_token) && a.kv_block % 16 == 0;
}

int launch_decode8(const Attn8Args& a, int dtype, void* ws, hipStream_t stream, const char* name) {
  Decode8Args p{};
  p.a = a;
  p.base = split_base(a.hq, a.hkv, a.d);
  const bool mfma = on_matrix_cores(a.hq, a.hkv, a.d);
  p.splits = decode8_most_splits(a.max_len, p.base);
  p.hpw = mfma ? 1 : heads_a_wave(a, p.splits);
  const int64_t columns = mfma ? (a.hq / a.hkv + 15) / 16 : 1;
  const int64_t items = a.rows * (a.hkv / p.hpw) * columns;
  p.split_slots = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(p.splits, kMaxGrid / items)));
  p.xcd = a.rows * p.split_slots % kXcds == 0;
  const int es = dtype_size(dtype);
  p.q_vec = a.q_dim == 1 && aligned16(a.q) && a.q_row * es % 16 == 0 && a.q_head * es % 16 == 0;
  p.ws_acc = static_cast<float*>(ws);
  p.ws_ml = reinterpret_cast<float2*>(p.ws_acc + a.rows * p.splits * a.hq * a.d);
  if (items * p.split_slots > kMaxBlocks || a.rows * a.hq > kMaxBlocks * kWaves) return fail(RLT_EUNSUPPORTED, "%s: too many rows", name);
  const unsigned grid = static_cast<unsigned>(items * p.split_slots);
  if (mfma) {
    launch_decode8_mfma(p, dtype, stream);
  } else {
    switch (dtype) {
      case RLT_BFLOAT16: launch_split<bf16>(p, grid, stream); break;
      case RLT_FLOAT16: launch_split<f16>(p, grid, stream); break;
      default: launch_split<float>(p, grid, stream); break;
    }
  }
  if (p.splits > 1) {
    switch (dtype) {
      case RLT_BFLOAT16: launch_merge<bf16>(p, stream); break;
      case RLT_FLOAT16: launch_merge<f16>(p, stream); break;
      default: launch_merge<float>(p, stream); break;
    }
  }
  return check_launch(name);
}

}  // namespace rlt
