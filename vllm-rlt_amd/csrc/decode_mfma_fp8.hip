// Decode over the 8-bit KV cache on the matrix cores: three or more query heads a KV
// head.  A key is then used by G heads, which on the vector units costs 4 D G flops a
// token in fp32 and G accumulators; here up to 16 heads are the columns of one tile.
//
// A workgroup takes one (row, KV head, 16 query heads, split), its four waves a quarter of
// the split's tokens each, 32 tokens a tile, through rows of LDS of its own (no barrier):
// - S^T = K Q^T on the scaled 8-bit MFMA (16x16x128), codes and scales as they are, q in
//   parts of 4 significant bits (two hold a bf16, three an fp16); an fp32 q in three bf16
//   parts on the bf16 MFMA against K converted with its scale (prefill_fp8.hip has the
//   reasons).
// - O^T += V^T P^T on the bf16 MFMA (16x16x32): P stays in the registers S^T left it in,
//   times its token's V scale, in one, two or three bf16 parts for bf16, fp16 and fp32; V's
//   codes come from transposing 8-bit LDS reads and become bf16 exactly.
// Bytes bound it, as for one head; the loads of the next tile go out before this one is
// worked on.
#include <type_traits>

#include "decode_fp8.hpp"
#include "mfma.hpp"

namespace rlt {
namespace {

constexpr int kWaves = 4;
constexpr int kXcds = 8;
constexpr int kTile = 32;
constexpr float kRescale = 8.f;  // the running maximum moves when a tile's exceeds it by 2^kRescale

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

template <typename T> struct Parts;
template <> struct Parts<bf16> { static constexpr int Q = 2, P = 1; };
template <> struct Parts<f16> { static constexpr int Q = 3, P = 2; };
template <> struct Parts<float> { static constexpr int Q = 3, P = 3; };

__device__ __forceinline__ uint32_t bf16_pair(float x, float y) { return MfmaOps<bf16>::pack2(x, y); }

// Two codes of a word (its low or high half) times a power of two, as bf16.
__device__ __forceinline__ uint32_t scaled_bf16(uint32_t word, float scale, bool high) {
  const bf16x2 r = high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(word), scale, true)
                        : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(word), scale, false);
  return __builtin_bit_cast(uint32_t, r);
}

__device__ __forceinline__ f32x4 mma16(u32x4 x, u32x4 y, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_v8<bf16x8>(x), as_v8<bf16x8>(y), c, 0, 0, 0);
}

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2))) void decode8_mfma_kernel(Decode8Args p) {
  constexpr bool WIDE = sizeof(T) == 4;
  constexpr int NQ = Parts<T>::Q, NP = Parts<T>::P;
  constexpr int KS = (D + 127) / 128;  // 8-bit MFMA steps over the dims
  constexpr int DT = D / 16;           // output tiles of 16 dims
  constexpr int CH = D / 16;           // 16-byte chunks of a code row
  constexpr int TPI = 64 / CH;         // tokens a load instruction
  constexpr int NI = kTile / TPI;      // loads a tile
  // Padded rows: an odd multiple of 16 bytes modulo 128 puts 8 rows' chunks, and the 8
  // rows of a transposing read, into distinct bank groups.
  constexpr int ROW = D + 16;
  constexpr int kTileBytes = 2 * kTile * ROW;
  constexpr int kJoinBytes = 16 * (D + 4) * 4;
  constexpr int kWaveBytes = kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes;
  __shared__ __align__(16) uint8_t lds[kWaves][kWaveBytes];
  __shared__ __align__(16) float sv_lds[kWaves][kTile];
  __shared__ uint8_t ks_lds[kWaves][kTile];
  __shared__ float2 ml_lds[kWaves][16];

  const Attn8Args& a = p.a;
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  const int G = a.hq / a.hkv;
  const uint32_t columns = (G + 15) / 16, rows = static_cast<uint32_t>(a.rows);
  const uint32_t heads = a.hkv * columns, groups = heads * p.split_slots;
  const uint32_t x = blockIdx.x % kXcds, t = blockIdx.x / kXcds;
  uint32_t gi, r;
  if (p.xcd) {  // workgroup b runs on XCD b % 8: all rows of a (split, head) on one XCD, back to back
    gi = t / rows * kXcds + x;
    r = t % rows;
  } else {
    gi = blockIdx.x % groups;
    r = blockIdx.x / groups;
  }
  gi = uniform(gi), r = uniform(r);
  const int h = gi % heads / columns, c0 = gi % heads % columns * 16;
  const int live = min(G - c0, 16);  // query heads of this tile
  const int len = sequence_length(a, r);
  int split_len, ns;
  decode8_split_plan(len, kMfmaSplit, &split_len, &ns);
  const int col = lane & 15, j = lane >> 4;
  const int st = lane / CH, sc = lane % CH;  // this lane's token and chunk of a load

  const int32_t* trow = a.tables + r * a.table_stride;
  const uint8_t* kh = a.k + h * a.kv_head + 16 * sc;
  const uint8_t* vh = a.v + h * a.kv_head + 16 * sc;
  const uint8_t* ksh = a.ks + h * a.s_head;
  const uint8_t* vsh = a.vs + h * a.s_head;
  const uint32_t token_bytes = static_cast<uint32_t>(a.kv_token);
  uint8_t* const k_lds = lds[wave];
  uint8_t* const v_lds = lds[wave] + kTile * ROW;
  static_assert(16 * (D + 4) * 4 <= sizeof(lds), "q as fp32 fits the tiles' rows");
  float(*const q_lds)[D + 4] = reinterpret_cast<float(*)[D + 4]>(lds[0]);

  for (int sp = gi / heads; sp < ns; sp += p.split_slots) {
    const int quarter = split_len / kWaves;
    const int t0 = sp * split_len + wave * quarter;
    const int n = min(max(len - t0, 0), quarter);
    f32x4 acc[DT];
#pragma unroll
    for (int c = 0; c < DT; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    int left = 0, last_unit = 0;  // of the chunk: 64 units of 16 tokens, one a lane
    int64_t unit_kv = 0, unit_s = 0;
    u32x4 k[NI], v[NI];
    uint32_t kb = 0, vb = 0;
    auto load_units = [&](int n0) __attribute__((always_inline)) {
      left = min(n - n0, 1024);
      last_unit = (left - 1) / 16;
      const int tok = t0 + n0 + 16 * min(lane, last_unit);
      const int page = tok / a.page, slot = tok - page * a.page;
      const int64_t blk = block_of(a, trow[page]);
      unit_kv = blk * a.kv_block + slot * a.kv_token;
      unit_s = blk * a.s_block + slot * a.s_token;
    };
    // Tokens past the end re-read the last one: in bounds, and masked below.
    auto load_tile = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int first = tile * kTile + i * TPI;  // the instruction's tokens lie in one unit
        const int at = min(first + st, left - 1);
        const int64_t off = __shfl(unit_kv, min(first / 16, last_unit), 64) +
                            __umul24(static_cast<uint32_t>(at - min(first / 16, last_unit) * 16), token_bytes);
        k[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kh + off));
        v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vh + off));
      }
      const int at = min(tile * kTile + (lane & (kTile - 1)), left - 1);
      const int64_t off = __shfl(unit_s, at / 16, 64) + at % 16 * a.s_token;
      kb = ksh[off];
      vb = vsh[off];
    };
    if (n > 0) {  // the first tile's loads go out before q is worked on
      load_units(0);
      load_tile(0);
    }
    // q's parts, B operands: lane (col, j) holds dims [128 c + 32 j, + 32) of query head c0 +
    // col; for bf16, 8 of them a k-step.
    i32x8 qb[NQ][KS];
    u32x4 qw[NQ][4 * KS];
    int q_scale[NQ];
    {
      // Through the tiles' LDS as fp32, whatever its strides.
#pragma unroll 1
      for (int o = threadIdx.x; o < live * D; o += 64 * kWaves)
        q_lds[o / D][o % D] = load_elem(static_cast<const T*>(a.q) + r * a.q_row + (h * G + c0 + o / D) * a.q_head + o % D * a.q_dim);
      __syncthreads();
      float y[KS][32];
      float amax = 0.f;
#pragma unroll
      for (int c = 0; c < KS; ++c) {
        const int d0 = 128 * c + 32 * j;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const f32x4 z = *reinterpret_cast<const f32x4*>(&q_lds[min(col, live - 1)][(d0 < D ? d0 : 0) + 4 * i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[c][4 * i + e] = d0 < D ? z[e] : 0.f;
            amax = fmaxf(amax, finite_abs(y[c][4 * i + e]));
          }
        }
      }
      __syncthreads();
      if constexpr (WIDE) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int c = 0; c < KS; ++c)
#pragma unroll
            for (int w = 0; w < 16; ++w) {
              const uint32_t lo = __float_as_uint(y[c][2 * w]), hi = __float_as_uint(y[c][2 * w + 1]);
              qw[n][4 * c + w / 4][w % 4] = lo >> 16 | (hi & 0xffff0000u);
              y[c][2 * w] -= __uint_as_float(lo & 0xffff0000u);
              y[c][2 * w + 1] -= __uint_as_float(hi & 0xffff0000u);
            }
      } else {
        amax = strided_max<16>(amax);
        const uint32_t b = max(scale_byte(amax), 4u * NQ);
        const float inv = inverse_scale(b);
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            y[c][i] = (__float_as_uint(y[c][i]) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fc00000u) : y[c][i] * inv;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          q_scale[n] = static_cast<int>(b) - 4 * n;
#pragma unroll
          for (int c = 0; c < KS; ++c)
#pragma unroll
            for (int w = 0; w < 8; ++w) {
              float* z = &y[c][4 * w];
              int word = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
              word = __builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], word, true);
              qb[n][c][w] = word;
              if (n + 1 < NQ) {
                const f32x2v lo = __builtin_amdgcn_cvt_pk_f32_fp8(word, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
                z[0] = (z[0] - lo[0]) * 16.f, z[1] = (z[1] - lo[1]) * 16.f;
                z[2] = (z[2] - hi[0]) * 16.f, z[3] = (z[3] - hi[1]) * 16.f;
              }
            }
        }
      }
    }

    for (int n0 = 0; n0 < n; n0 += 1024) {
      if (n0) {
        load_units(n0);
        load_tile(0);
      }
      const int tiles = (left + kTile - 1) / kTile;
#pragma unroll 1
      for (int tile = 0; tile < tiles; ++tile) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          *reinterpret_cast<u32x4*>(k_lds + (i * TPI + st) * ROW + 16 * sc) = k[i];
          *reinterpret_cast<u32x4*>(v_lds + (i * TPI + st) * ROW + 16 * sc) = v[i];
        }
        if (lane < kTile) {
          sv_lds[wave][lane] = scale_value(vb);
          ks_lds[wave][lane] = static_cast<uint8_t>(kb);
        }
        float bias = 0.f;
        if (__builtin_amdgcn_ballot_w64(vb > 191u)) bias = group_max<64>(value_bias(vb == 255u ? 0u : vb));
        if (tile + 1 < tiles) load_tile(tile + 1);
        __builtin_amdgcn_wave_barrier();
        // S^T: element r of half u is token 16 u + 4 j + r of the tile.
        f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint8_t* row = k_lds + (16 * u + col) * ROW;
          const uint32_t ksc = ks_lds[wave][16 * u + col];
#pragma unroll
          for (int c = 0; c < KS; ++c) {
            const bool in = D >= 128 || j < 2;  // head_dim 64: the upper half of the step is 0
            const u32x4 lo = in ? *reinterpret_cast<const u32x4*>(row + 128 * c + 32 * j) : u32x4{0u, 0u, 0u, 0u};
            const u32x4 hi = in ? *reinterpret_cast<const u32x4*>(row + 128 * c + 32 * j + 16) : u32x4{0u, 0u, 0u, 0u};
            if constexpr (WIDE) {
              const float scale = scale_value(ksc);
#pragma unroll
              for (int q4 = 0; q4 < 4; ++q4) {
                u32x4 ka;
#pragma unroll
                for (int e = 0; e < 4; ++e) ka[e] = scaled_bf16((q4 < 2 ? lo : hi)[q4 % 2 * 2 + e / 2], scale, e % 2);
#pragma unroll
                for (int i = 0; i < NQ; ++i) s[u] = mma16(ka, qw[i][4 * c + q4], s[u]);
              }
            } else {
              i32x8 ka;
#pragma unroll
              for (int e = 0; e < 4; ++e) ka[e] = static_cast<int>(lo[e]), ka[4 + e] = static_cast<int>(hi[e]);
#pragma unroll
              for (int i = 0; i < NQ; ++i)
                s[u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(ka, qb[i][c], s[u], 0, 0, 0, static_cast<int>(ksc), 0,
                                                                        q_scale[i]);
            }
          }
        }
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[u][e] = tile * kTile + 16 * u + 4 * j + e < left ? s[u][e] * a.qscale : -INFINITY;
            top = fmaxf(top, s[u][e]);
          }
        top = strided_max<16>(top) + bias;
        if (__builtin_amdgcn_ballot_w64(top > m + kRescale) != 0) {
          const float mn = fmaxf(m, top);
          const float corr = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
          m = mn;
          l *= corr;
#pragma unroll
          for (int c = 0; c < DT; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[c][e] *= corr;
        }
        const float off = m == -INFINITY ? 0.f : m;  // only -inf scores so far: they weigh 0
        // P^T, element e of the k-step is token 16 (e / 4) + 4 j + e % 4, times its V scale.
        u32x4 pb[NP];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const f32x4 sv = *reinterpret_cast<const f32x4*>(&sv_lds[wave][16 * u + 4 * j]);
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[e] = fast_exp2(s[u][e] - off);
            l += w[e];
            w[e] *= sv[e];
          }
#pragma unroll
          for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              pb[i][2 * u + e] = bf16_pair(w[2 * e], w[2 * e + 1]);
              w[2 * e] -= bf16_lo(pb[i][2 * u + e]), w[2 * e + 1] -= bf16_hi(pb[i][2 * u + e]);
            }
        }
        // V^T, 16 dims a tile: in each 16-lane group lane L addresses 8 bytes of token row L / 2 of
        // its 8, and gets one dim of all 8.
        const int vt = lane & 15, vr = vt / 2;
        const uint8_t* vrow = v_lds + (4 * j + vr % 4 + 16 * (vr / 4)) * ROW + 8 * (vt & 1);
#pragma unroll
        for (int c = 0; c < DT; ++c) {
          const i32x2 codes = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(vrow + 16 * c));
          u32x4 va;
#pragma unroll
          for (int e = 0; e < 4; ++e) va[e] = scaled_bf16(static_cast<uint32_t>(codes[e / 2]), 1.f, e % 2);
#pragma unroll
          for (int i = 0; i < NP; ++i) acc[c] = mma16(va, pb[i], acc[c]);
        }
      }
    }
    // Join the waves, in order.
    l = strided_sum<16>(l);
    __syncthreads();
    float* const join = reinterpret_cast<float*>(lds[wave]);  // [16 columns][D + 4]
#pragma unroll
    for (int c = 0; c < DT; ++c) *reinterpret_cast<f32x4*>(join + col * (D + 4) + 16 * c + 4 * j) = acc[c];
    if (j == 0) ml_lds[wave][col] = make_float2(m, l);
    __syncthreads();
    for (int o = threadIdx.x; o < live * D; o += 64 * kWaves) {
      const int hd = o / D, d = o % D;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml_lds[w][hd].x);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float2 ml = ml_lds[w][hd];
        const float c = fast_exp2(ml.x - base);
        sum = fmaf(ml.y, c, sum);
        y = fmaf(reinterpret_cast<const float*>(lds[w])[hd * (D + 4) + d], c, y);
      }
      const int q = c0 + hd;  // of the KV head's
      if (ns == 1) {
        store_elem(static_cast<T*>(a.out) + r * a.o_row + (h * G + q) * a.o_head + d * a.o_dim, len > 0 ? y * (1.f / sum) : 0.f);
      } else {
        const int64_t at = ((static_cast<int64_t>(r) * a.hkv + h) * p.splits + sp) * G + q;
        p.ws_acc[at * D + d] = y;
        if (d == 0) p.ws_ml[at] = make_float2(top, sum);
      }
    }
    __syncthreads();
  }
}

template <typename T>
void launch_type(const Decode8Args& p, hipStream_t stream) {
  const int64_t columns = (p.a.hq / p.a.hkv + 15) / 16;
  const dim3 grid(static_cast<unsigned>(p.a.rows * p.a.hkv * columns * p.split_slots)), block(64 * kWaves);
  switch (p.a.d) {
    case 64: hipLaunchKernelGGL((decode8_mfma_kernel<T, 64>), grid, block, 0, stream, p); break;
    case 128: hipLaunchKernelGGL((decode8_mfma_kernel<T, 128>), grid, block, 0, stream, p); break;
    default: hipLaunchKernelGGL((decode8_mfma_kernel<T, 256>), grid, block, 0, stream, p); break;
  }
}

}  // namespace

void launch_decode8_mfma(const Decode8Args& p, int dtype, hipStream_t stream) {
  switch (dtype) {
    case RLT_BFLOAT16: launch_type<bf16>(p, stream); break;
    case RLT_FLOAT16: launch_type<f16>(p, stream); break;
    default: launch_type<float>(p, stream); break;
  }
}

}  // namespace rlt
