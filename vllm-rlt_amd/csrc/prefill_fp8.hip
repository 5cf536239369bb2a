// Packed chunked prefill over the 8-bit KV cache, bottom-right causal, on the
// matrix cores (head_dim 64 / 128, pages of a power of two of at least 16 tokens).
//
// A workgroup of 4 waves takes 128 query rows of one (sequence, query head) over a
// segment of its keys, a wave 32 rows, 64 keys a tile:
// - S^T = K Q^T on the 16-bit MFMA (32x32x16).  K becomes bf16, its scale included (exact: a
//   code has 4 bits), once a workgroup, on its way into LDS, for q in bf16, or fp32 in three bf16
//   parts.  For an fp16 q codes become fp16, and their scales multiply the sums (two bf16 parts
//   of q instead: 980 us for 877 below).  (The scaled 8-bit MFMA would take K's codes and scales
//   as they are, but drops what lies 2^-11 below the largest product of its 64; the 16-bit
//   ones keep fp32's bits.)
// - O^T += V^T P^T likewise.  V becomes bf16 as K does, kLift times as large (keys whose scale
//   leaves no room for that get a larger weight instead, on a path of their own); V^T comes from
//   transposing LDS reads, P from the registers S^T left it in.  P is split in two or three bf16
//   parts for fp16 and fp32 outputs.  For bf16 ones it is rounded to bf16, as rlt_paged_prefill
//   does, and its sum taken over the rounded values: outputs are off by 0.0023 of their rms.
//   Their own rounding is 0.0017 of it, which two parts would come down to for 27% more time (835
//   us for 655 below).
// The running maximum moves only when a tile's exceeds it by 2^kRescale.
//
// The products' rate and the vector work beside them bound it (a tile of a wave is 1024 cycles of
// MFMA and some 1100 of vector work in bf16; two waves a SIMD).  Measured, 16 chunks of 512 rows at
// the end of 8192 keys, 16 heads x 128: bf16 655 us, 865 TFLOP/s, fp16 877 us, fp32 406 us for four
// chunks.
//
// prefill_plan.hpp has the launch's plan: key segments, and the merge that joins them.
#include "prefill_plan.hpp"

namespace rlt {
namespace {

constexpr uint32_t kLargestScale = 246;  // the largest scale byte whose codes are all finite in bf16
constexpr uint32_t kLiftExp = 24;        // kLift = 2^kLiftExp
static_assert(kLift == static_cast<float>(uint64_t(1) << kLiftExp) && kLargestScale - kLiftExp > kFreeScale);
template <typename T> struct Parts;
template <> struct Parts<bf16> { static constexpr int Q = 1, P = 1; using S = bf16; };
template <> struct Parts<f16> { static constexpr int Q = 1, P = 2; using S = f16; };
template <> struct Parts<float> { static constexpr int Q = 3, P = 3; using S = bf16; };

__device__ __forceinline__ uint32_t bf16_pair(float x, float y) { return MfmaOps<bf16>::pack2(x, y); }

// The top bit of every byte of a word of codes that is NaN (all bits of its magnitude set).
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Two codes of a word (its low or high half) times the scale of byte b, as bf16.
// The instruction takes the scale as an fp32's exponent, with the byte's meaning: 0
// is 2^-127, 255 NaN.
__device__ __forceinline__ uint32_t scaled_bf16(uint32_t word, uint32_t b, bool high) {
  const float s = __uint_as_float(b << 23);
  const bf16x2 r = high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(word), s, true)
                        : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(word), s, false);
  return __builtin_bit_cast(uint32_t, r);
}

// Two codes of a word (its low or high half) as fp16, exact.
__device__ __forceinline__ uint32_t f16_codes(uint32_t word, bool high) {
  const f16x2 r = high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(word), 1.f, true)
                       : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(word), 1.f, false);
  return __builtin_bit_cast(uint32_t, r);
}

template <typename T, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 ? 1 : 2))) void prefill8_kernel(Prefill8Args p) {
  using Ops = MfmaOps<bf16>;
  using S = typename Parts<T>::S;  // of the scores' operands
  constexpr bool LATE = std::is_same_v<S, f16>;  // K's scales multiply the sums
  constexpr int NQ = Parts<T>::Q, NP = Parts<T>::P;
  constexpr int KS = D / 16;       // MFMA steps over the dims
  constexpr int DT = D / 32;       // output tiles of 32 dims
  constexpr int CH = D / 16;       // 16-byte chunks of a code row
  constexpr int TPP = 256 / CH;    // tokens a staging pass
  constexpr int PASSES = kBN / TPP;
  // Padded rows: 8 lanes' 16-byte reads of 8 K rows fall into distinct bank groups
  // (the stride is an odd multiple of 16 bytes modulo 128), and so do the
  // transposing V reads (64 modulo 256).
  constexpr int KROW = D + 8, VROW = D + 32;
  __shared__ __align__(16) uint16_t k_lds[2][kBN * KROW];
  __shared__ __align__(16) uint16_t v_lds[2][kBN * VROW];
  __shared__ __align__(16) float ks_lds[2][LATE ? kBN : 4];  // K's scales times 2^q_exp
  __shared__ __align__(16) float bias_lds[2][4];  // of each wave's staged V scales (value_bias)
  __shared__ uint8_t vs_lds[2][kBN];              // and those scales' bytes, where that is not 0

  const Attn8Args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  Item it;
  if (!find_item<false>(p, &it)) return;
  const int seq = uniform(it.seq), h = uniform(it.head), row0 = uniform(it.row0), nq = uniform(it.nq);
  const int len = uniform(it.len);
  const int prefix = len - nq;  // query row i sees keys up to prefix + i
  const int qt0 = uniform(it.tile) * kBM;
  const int kvh = h / (a.hq / a.hkv);
  const int wg_keys = min(prefix + min(qt0 + kBM, nq), len);  // keys that some row of the workgroup sees
  const int first_tile = uniform(it.seg * it.seg_tiles);
  const int ntiles = min(first_tile + uniform(it.seg_tiles), (max(wg_keys, 0) + kBN - 1) / kBN);
  if (it.segs > 1 && it.seg > 0 && ntiles <= first_tile) return;  // the merge skips such a segment

  const int half = lane >> 5, col = lane & 31;
  const int wave_row0 = qt0 + wave * 32;
  const int my_row = wave_row0 + col;
  const bool row_valid = my_row < nq;
  const int limit = row_valid ? prefix + my_row : -1;  // last key this lane's query sees
  const int wave_last = prefix + min(wave_row0 + 31, nq - 1);
  const bool wave_live = wave_row0 < nq;

  // q's parts, B operands: lane (col, half) holds dims [16 c + 8 half, + 8) of row col for step c.
  u32x4 qw[NQ][KS];
  {
    const T* qrow = static_cast<const T*>(a.q) + (row0 + min(my_row, nq - 1)) * a.q_row + h * a.q_head;
    const float power = __uint_as_float(static_cast<uint32_t>(127 + (LATE ? 0 : p.q_exp)) << 23 | p.q_sign);
#pragma unroll
    for (int c = 0; c < KS; ++c) {
      const int d0 = 16 * c + 8 * half;
      float x[8];
      if (p.q_vec) {
        constexpr int N = Packet<T>::N;
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) Packet<T>::unpack(*reinterpret_cast<const u32x4*>(qrow + d0 + i * N), &x[i * N]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = load_elem(qrow + (d0 + i) * a.q_dim);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)  // infinities as NaN, which no other row's maximum takes up
        x[i] = (__float_as_uint(x[i]) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fc00000u) : x[i] * power;
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if constexpr (NQ > 1) {  // the top 16 bits: the rest is exact, and the last part holds all of it
            const uint32_t lo = __float_as_uint(x[2 * w]), hi = __float_as_uint(x[2 * w + 1]);
            qw[n][c][w] = lo >> 16 | (hi & 0xffff0000u);
            x[2 * w] -= __uint_as_float(lo & 0xffff0000u);
            x[2 * w + 1] -= __uint_as_float(hi & 0xffff0000u);
          } else {
            qw[n][c][w] = MfmaOps<S>::pack2(x[2 * w], x[2 * w + 1]);
          }
        }
    }
  }

  // Staging: thread (token, chunk), PASSES tokens TPP apart.  Tokens past the last key
  // re-read it (in bounds; they are masked).
  const int32_t* trow = a.tables + seq * a.table_stride;
  const int st = tid / CH, sc = tid % CH;
  const uint8_t* kbase = a.k + kvh * a.kv_head + sc * 16;
  const uint8_t* vbase = a.v + kvh * a.kv_head + sc * 16;
  const uint8_t* ksbase = a.ks + kvh * a.s_head;
  const uint8_t* vsbase = a.vs + kvh * a.s_head;
  const uint32_t block_bytes = static_cast<uint32_t>(a.kv_block), token_bytes = static_cast<uint32_t>(a.kv_token);
  const uint32_t s_block = static_cast<uint32_t>(a.s_block), s_token = static_cast<uint32_t>(a.s_token);
  const uint32_t page_mask = a.page - 1, last_key = max(wg_keys, 1) - 1, num_blocks = static_cast<uint32_t>(a.num_blocks);
  uint32_t ids[PASSES];  // of the tile loaded next
  u32x4 kreg[PASSES], vreg[PASSES];
  uint32_t ksreg[PASSES], vsreg[PASSES];
  auto token = [&](int tile, int t) { return min(static_cast<uint32_t>(tile * kBN + t), last_key); };
  auto load_ids = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) ids[i] = trow[token(tile, i * TPP + st) >> p.page_shift];
  };
  auto load_tile = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const uint32_t slot = token(tile, i * TPP + st) & page_mask;
      const uint64_t id = ids[i] < num_blocks ? ids[i] : 0;
      const uint64_t at = id * block_bytes + __umul24(slot, token_bytes), s_at = id * s_block + __umul24(slot, s_token);
      kreg[i] = *reinterpret_cast<const u32x4*>(kbase + at);
      ksreg[i] = ksbase[s_at];
      vreg[i] = *reinterpret_cast<const u32x4*>(vbase + at);
      vsreg[i] = vsbase[s_at];
    }
  };
  // Keys of 2^128 and more become the largest finite bf16: a score then is as large as fp32
  // holds, and not NaN where q is 0.
  auto store_k = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      u32x4 w[2];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e / 4][e % 4] = LATE ? f16_codes(kreg[i][e / 2], e % 2) : scaled_bf16(kreg[i][e / 2], ksreg[i], e % 2);
      if constexpr (LATE) {
        if (sc == 0) ks_lds[buf][i * TPP + st] = scale_value(ksreg[i]) * __uint_as_float(static_cast<uint32_t>(127 + p.q_exp) << 23);
      } else if (__builtin_amdgcn_ballot_w64(ksreg[i] > kLargestScale)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t x = w[e / 4][e % 4];
          w[e / 4][e % 4] = x - ((x & 0x7fffu) == 0x7f80u ? 1u : 0u) - ((x >> 16 & 0x7fffu) == 0x7f80u ? 0x10000u : 0u);
        }
      }
      uint16_t* dst = &k_lds[buf][(i * TPP + st) * KROW + sc * 16];
      *reinterpret_cast<u32x4*>(dst) = w[0];
      *reinterpret_cast<u32x4*>(dst + 8) = w[1];
    }
  };
  // A V that is NaN must not reach the rows that do not see it through a product with 0:
  // in tiles that some row sees part of, it is stored as 0, and noted (see the end).
  bool nan = false;
  auto store_v = [&](int buf, bool masked) __attribute__((always_inline)) {
    uint32_t top = 0;  // largest V scale
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int t = i * TPP + st;
      if (masked) {
        bool here = vsreg[i] == 255u;
#pragma unroll
        for (int e = 0; e < 4; ++e) here |= nan_codes(vreg[i][e]) != 0;
        if (here) {
          nan = true;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t bad = vsreg[i] == 255u ? 0x80808080u : nan_codes(vreg[i][e]);
            vreg[i][e] &= ~((bad >> 7) * 0xffu);
          }
          vsreg[i] = vsreg[i] == 255u ? 127u : vsreg[i];
        }
      }
      u32x4 w[2];
      const uint32_t lifted = vsreg[i] == 255u ? 255u : min(vsreg[i] + kLiftExp, kLargestScale);
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e / 4][e % 4] = scaled_bf16(vreg[i][e / 2], lifted, e % 2);
      uint16_t* dst = &v_lds[buf][t * VROW + sc * 16];
      *reinterpret_cast<u32x4*>(dst) = w[0];
      *reinterpret_cast<u32x4*>(dst + 8) = w[1];
      top = max(top, vsreg[i]);
    }
    float bias = 0.f;
    if (__builtin_amdgcn_ballot_w64(top > kFreeScale)) {
      bias = group_max<64>(value_bias(top == 255u ? 0u : top));
      if (sc == 0) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) vs_lds[buf][i * TPP + st] = static_cast<uint8_t>(vsreg[i]);
      }
    }
    if (lane == 0) bias_lds[buf][wave] = bias;
  };
  // Whether some row of the workgroup does not see all of a tile's keys.
  auto tile_masked = [&](int tile) { return tile * kBN + kBN - 1 > prefix + qt0; };

  f32x16 acc[DT];
#pragma unroll
  for (int c = 0; c < DT; ++c) acc[c] = f32x16{};
  float m = -INFINITY, lsum = 0.f;

  // V^T operands: in each 16-lane group lane L addresses key row L / 4 of its four and 4
  // dims; k-step ks, element e of half hf holds key 16 ks + 8 (e / 4) + 4 hf + e % 4.
  const int grp = lane >> 4, gl = lane & 15;
  const int tr_off = (4 * (grp >> 1) + (gl >> 2)) * VROW + 16 * (grp & 1) + 4 * (gl & 3);

  // S^T of tile j.
  auto scores = [&](int buf, f32x16 (&s)[2]) __attribute__((always_inline)) {
    s[0] = s[1] = f32x16{};
#pragma unroll
    for (int c = 0; c < KS; ++c)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const u32x4 ka = *reinterpret_cast<const u32x4*>(&k_lds[buf][(hh * 32 + col) * KROW + 16 * c + 8 * half]);
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[hh] = MfmaOps<S>::mma(as_v8<typename MfmaOps<S>::V8>(ka), as_v8<typename MfmaOps<S>::V8>(qw[n][c]), s[hh]);
      }
    if constexpr (LATE) {
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const f32x4 k4 = *reinterpret_cast<const f32x4*>(&ks_lds[buf][8 * g + 4 * half]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[g / 4][g % 4 * 4 + e] *= k4[e];
      }
    }
  };
  auto step = [&](int j) __attribute__((always_inline)) {
    const int buf = j & 1;
    if (j + 1 < ntiles) {
      load_tile(j + 1);
      load_ids(j + 2);
    }
    if (wave_live && j * kBN <= wave_last) {
      f32x16 s[2];
      scores(buf, s);
      // Element r of half hh is key key0 + 32 hh + 8 (r / 4) + 4 half + r % 4.
      const int key0 = j * kBN;
      const bool masked = uniform(key0 + kBN - 1 > prefix + wave_row0 || wave_row0 + 31 >= nq);
      if (masked) {
        const int lim = limit - key0 - 4 * half;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[hh][r] = hh * 32 + (r / 4) * 8 + r % 4 > lim ? -INFINITY : s[hh][r];
      }
      float tmax = -INFINITY;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int r = 0; r < 16; ++r) tmax = fmaxf(tmax, s[hh][r]);
      const f32x4 b4 = *reinterpret_cast<const f32x4*>(bias_lds[buf]);
      const float bias = fmaxf(fmaxf(b4[0], b4[1]), fmaxf(b4[2], b4[3]));
      tmax = max_across_halves(tmax) * p.qscale + bias;
      const bool rescale = __builtin_amdgcn_ballot_w64(tmax > m + kRescale) != 0;
      float corr = 1.f;
      if (rescale) {
        const float mn = fmaxf(m, tmax);
        corr = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
        m = mn;
        lsum *= corr;
      }
      const float mb = m == -INFINITY ? 0.f : m;  // only -inf scores so far: they weigh 0
      // exp2(s * qscale - m) in one rounding, unless m's own is no longer small.  Keys whose V is
      // stored less than kLift as large weigh the more; the sum of the weights is taken before that.
      float qs = p.qscale, whole = -1.f;  // that sum
      if (__builtin_amdgcn_ballot_w64(fabsf(mb) > 4096.f || bias > value_bias(kLargestScale - kLiftExp)) != 0) {
        qs = 1.f;
        whole = lsum;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[hh][r] = rounded_product(s[hh][r], p.qscale);  // the same in both sums
            const float x = fast_exp2(s[hh][r] - mb);
            whole += NP == 1 ? bf16_lo(bf16_pair(x, x)) : x;
            const int key = hh * 32 + r / 4 * 8 + 4 * half + r % 4;
            const uint32_t b = b4[key % TPP / (TPP / 4)] > 0.f ? vs_lds[buf][key] : 0u;  // (of the wave that staged it)
            s[hh][r] += static_cast<float>(max(b, kLargestScale - kLiftExp) - (kLargestScale - kLiftExp));
          }
      }
      // P of k-step ks, in parts; its sum is taken over what the products see.
      auto weights = [&](int ks, u32x4 (&pb)[NP]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = (ks % 2) * 8 + 2 * e;
          float x = fast_exp2(fmaf(s[ks / 2][r], qs, -mb)), y = fast_exp2(fmaf(s[ks / 2][r + 1], qs, -mb));
          if constexpr (NP > 1) lsum += x + y;
#pragma unroll
          for (int n = 0; n < NP; ++n) {
            pb[n][e] = bf16_pair(x, y);
            x -= bf16_lo(pb[n][e]), y -= bf16_hi(pb[n][e]);
          }
          if constexpr (NP == 1) lsum = Ops::sum2(pb[0][e], lsum);
        }
      };
      auto values = [&](int ks, int c) __attribute__((always_inline)) {
        const uint16_t* vlo = &v_lds[buf][tr_off + ks * 16 * VROW + c * 32];
        const u32x2 lo = lds_read_tr(vlo), hi = lds_read_tr(vlo + 8 * VROW);
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
      };
      // One site for all products: accumulators changed on two paths get two register sets.
      if (rescale) {
#pragma unroll
        for (int c = 0; c < DT; ++c)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[c][r] *= corr;
      }
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        u32x4 pb[NP];
        weights(ks, pb);
#pragma unroll
        for (int c = 0; c < DT; ++c) {
          const u32x4 va = values(ks, c);
#pragma unroll
          for (int n = 0; n < NP; ++n) acc[c] = Ops::mma(as_v8<bf16x8>(va), as_v8<bf16x8>(pb[n]), acc[c]);
        }
      }
      if (whole >= 0.f) lsum = whole;
    }
    if (j + 1 < ntiles) {
      store_k(buf ^ 1);
      store_v(buf ^ 1, tile_masked(j + 1));
    }
    __syncthreads();
  };

  if (ntiles > first_tile) {
    load_ids(first_tile);
    load_tile(first_tile);
    load_ids(first_tile + 1);
    store_k(first_tile & 1);
    store_v(first_tile & 1, tile_masked(first_tile));
    __syncthreads();
  }
  for (int j = first_tile; j < ntiles; ++j) step(j);

  // V that was NaN in tiles that some row sees part of: it is NaN in the rows that see it.
  if (__syncthreads_or(nan)) {
    for (int j = max(first_tile, max(prefix + qt0 + 1, 0) / kBN); j < ntiles; ++j) {
#pragma unroll 1
      for (int t = j * kBN; t < min(j * kBN + kBN, wg_keys); ++t) {
        const uint32_t id = trow[t >> p.page_shift], slot = t & page_mask;
        const uint64_t blk = id < num_blocks ? id : 0;
        const uint8_t* row = a.v + kvh * a.kv_head + blk * block_bytes + slot * token_bytes + 4 * half;
        const bool all = vsbase[blk * s_block + slot * s_token] == 255u;
#pragma unroll
        for (int c = 0; c < DT; ++c)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint32_t bad = all ? 0x80808080u : nan_codes(*reinterpret_cast<const uint32_t*>(row + 32 * c + 8 * g));
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (t <= limit && (bad >> (8 * e + 7) & 1)) acc[c][4 * g + e] = __uint_as_float(0x7fc00000u);
          }
      }
    }
  }
  lsum += __shfl_xor(lsum, 32, 64);
  if (!row_valid) return;
  if (uniform(it.segs) > 1) {
    const int64_t slot = (static_cast<int64_t>(it.slot0) + static_cast<int64_t>(it.seg) * nq + my_row) * a.hq + h;
    float* dst = p.part_acc + slot * D + 4 * half;
#pragma unroll
    for (int c = 0; c < DT; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(dst + 32 * c + 8 * g) = f32x4{acc[c][4 * g], acc[c][4 * g + 1], acc[c][4 * g + 2], acc[c][4 * g + 3]};
    if (half == 0) p.part_ml[slot] = make_float2(m, lsum);
    return;
  }
  // A row that sees no key is zeros.
  const float inv = limit < 0 ? 0.f : 1.f / kLift / lsum;
  T* orow = static_cast<T*>(a.out) + (row0 + my_row) * a.o_row + h * a.o_head;
#pragma unroll
  for (int c = 0; c < DT; ++c)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * c + 8 * g + 4 * half;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = limit < 0 ? 0.f : acc[c][4 * g + e] * inv;
      store4(orow, d, x, a.o_dim, p.out_vec);
    }
}

// Joins the segments of cut sequences: a workgroup takes 1024 neighbouring elements of a row
// at a time, 4 a thread, and adds the segments in order under a running maximum, BATCH of them
// on their way at once.  Bytes and latency bound it: eight chunks of 512 rows over 0-16384 keys
// x 16 heads 12.9 us.  The grid is one round at most and walks the rows of cut sequences only:
// 16 chunks of 512 rows, none of them cut, take 64 us, 67 with workgroups for every row.
template <typename T, int D>
__global__ __launch_bounds__(256) void prefill8_merge_kernel(Prefill8Args p, int parts) {
  constexpr int BATCH = 4;
  const Attn8Args& a = p.a;
  const int lane = threadIdx.x & 63;
  SeqPlan s{};
  if (lane < a.num_seqs) s = p.plan[lane];
  const int rows = s.segs > 1 ? s.nq : 0, last = scan_sum(rows), first = last - rows;
  const int64_t items = static_cast<int64_t>(__builtin_amdgcn_readlane(last, 63)) * parts;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int r = static_cast<int>(item / parts), e0 = (static_cast<int>(item % parts) * 256 + static_cast<int>(threadIdx.x)) * 4;
    const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(r >= first && r < last));
    const int nq = __builtin_amdgcn_readlane(s.nq, at), len = __builtin_amdgcn_readlane(s.len, at);
    const int segs = __builtin_amdgcn_readlane(s.segs, at), slot0 = __builtin_amdgcn_readlane(s.slot0, at);
    const int seg_keys = __builtin_amdgcn_readlane(s.seg_tiles, at) * kBN;
    const int i = r - __builtin_amdgcn_readlane(first, at), row = __builtin_amdgcn_readlane(s.row0, at) + i;
    const int h = e0 / D, d = e0 % D;
    if (h >= a.hq) continue;
    // Segments past the last key of the row's query tile were not computed.
    const int keys = max(len - nq + min(i / kBM * kBM + kBM, nq), 0);
    const int live = min(segs, max(1, (keys + seg_keys - 1) / seg_keys));
    const int64_t step = static_cast<int64_t>(nq) * a.hq;  // slots from one segment to the next
    const int64_t base = (static_cast<int64_t>(slot0) + i) * a.hq + h;
    float m = -INFINITY, sum = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int g0 = 0; g0 < live; g0 += BATCH) {
      float2 ml[BATCH];
      f32x4 x[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int64_t slot = base + min(g0 + u, live - 1) * step;
        ml[u] = p.part_ml[slot];
        x[u] = *reinterpret_cast<const f32x4*>(p.part_acc + slot * D + d);
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < BATCH; ++u) top = fmaxf(top, ml[u].x);
      const float off = top == -INFINITY ? 0.f : top;
      const float corr = fast_exp2(m - off);
      m = top;
      sum *= corr;
      acc *= corr;
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const float w = g0 + u < live ? fast_exp2(ml[u].x - off) : 0.f;
        sum = fmaf(ml[u].y, w, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = g0 + u < live ? fmaf(x[u][e], w, acc[e]) : acc[e];
      }
    }
    const bool blind = len - nq + i < 0;  // a row that sees no key
    const float inv = 1.f / kLift / sum;
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = blind ? 0.f : acc[e] * inv;
    store4(static_cast<T*>(a.out) + row * a.o_row + h * a.o_head, d, y, a.o_dim, p.out_vec);
  }
}

}  // namespace

bool prefill8_shape(int64_t d, int64_t page) { return (d == 64 || d == 128) && page >= 16 && (page & (page - 1)) == 0; }

bool prefill8_layout(const Attn8Args& a) { return prefill8_shape(a.d, a.page) && prefill8_strides(a); }
bool prefill8_strides(const Attn8Args& a) {
  auto near = [](int64_t x) { return x >= 0 && x < (int64_t(1) << 24); };
  auto small = [](int64_t x) { return x >= 0 && x < (int64_t(1) << 32); };
  return a.kv_dim == 1 && aligned16(a.k) && aligned16(a.v) && a.kv_head % 16 == 0 &&
         a.kv_token % 16 == 0 && a.kv_block % 16 == 0 && small(a.kv_block) && small(a.s_block) &&
         near(a.kv_token) && near(a.s_token) && near(a.page) && small(a.kv_token * a.page) && small(a.s_token * a.page);
}

int64_t prefill8_workspace(int64_t rows, int64_t num_seqs, int64_t max_len, int64_t hq, int64_t d) {
  const int64_t slots = partial_slots(rows, num_seqs, max_len, hq);
  return slots ? slots * hq * (d * 4 + 8) + kPlanSeqs * static_cast<int64_t>(sizeof(SeqPlan)) : 0;
}

int launch_prefill8(const Attn8Args& a, int dtype, void* ws, hipStream_t stream, const char* name) {
  Prefill8Args p{};
  p.a = a;
  const int64_t slots = ws ? partial_slots(a.rows, a.num_seqs, a.max_len, a.hq) : 0;
  if (slots > kMaxBlocks) return fail(RLT_EUNSUPPORTED, "%s: too many rows", name);  // 64 sequences' stay inside 31 bits
  p.slots = static_cast<int>(slots);
  p.group = 1;
  p.round = dtype == RLT_FLOAT32 && a.d == 128 ? kRound / 2 : kRound;
  if (slots) {
    p.part_acc = static_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float2*>(p.part_acc + slots * a.hq * a.d);
    p.plan = reinterpret_cast<SeqPlan*>(p.part_ml + slots * a.hq);
  }
  fill_prefill8(&p, dtype);
  const int64_t tiles = prefill8_tiles(p, kTargetItems);
  const int parts = static_cast<int>((static_cast<int64_t>(a.hq) * a.d + 1023) / 1024);
  if (tiles * a.hq > kMaxBlocks) return fail(RLT_EUNSUPPORTED, "%s: too many rows", name);
  const dim3 grid(static_cast<unsigned>(tiles * a.hq)), block(256);
  const dim3 merge(static_cast<unsigned>(std::min<int64_t>(a.rows * parts, kMergeRound)));
#define LAUNCH_D(T, D)                                                                                   \
  do {                                                                                                   \
    hipLaunchKernelGGL((prefill8_kernel<T, D>), grid, block, 0, stream, p);                              \
    if (slots) hipLaunchKernelGGL((prefill8_merge_kernel<T, D>), merge, block, 0, stream, p, parts);            \
  } while (0)
#define LAUNCH(T)                       \
  do {                                  \
    if (a.d == 64) LAUNCH_D(T, 64);     \
    else LAUNCH_D(T, 128);              \
  } while (0)
  switch (dtype) {
    case RLT_BFLOAT16: LAUNCH(bf16); break;
    case RLT_FLOAT16: LAUNCH(f16); break;
    default: LAUNCH(float); break;
  }
#undef LAUNCH
#undef LAUNCH_D
  return check_launch(name);
}

}  // namespace rlt
