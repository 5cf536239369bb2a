// Decode over the block-scaled 8-bit KV cache, on the matrix cores: one new token a
// sequence, split over the cache's length and joined (int8.hpp has the softmax).
//
// A workgroup takes one (row, KV head, 16 query heads, split); its four waves take every
// fourth 32 tokens of the split each, through LDS of their own (no barrier).  16 tokens lie in
// one block, so that a tile has two scales of K and two of V:
// - S^T = K Q^T on the 16-bit MFMA of q's type (16x16x32; an fp32 q in three bf16 parts): a
//   code is a bf16 or an fp16 exactly, and the block's scale multiplies the fp32 sum.
// - O^T += V^T W^T on the fp16 MFMA (16x16x32), W the probabilities times their block's V scale,
//   near 1 for the keys that matter, in two parts, 22 bits.  (One for bf16 would save 1%, and round
//   8% of the outputs the other way.)  The sum of the probabilities is taken before that.
// Bytes bound it: 256 rows of 1024-8192 tokens, 16 heads x 128, bf16, 4.84 GB, take 811 us, 6.0 TB/s; few rows
// the latency of length, table, first tile and join (24 rows of 512-4096, 32 + 8 heads, fp16, 114 MB: 31.6 us).
// Tiles go from memory into LDS directly: K of the next one as soon as this
// one's K is in registers, V likewise, one buffer each.  The heads of a row's split run on one XCD
// at the same time, which reads whole token rows of the cache.
//
// A row's keys are cut into splits (decode8_split_plan), a function of the row's length
// alone, which are joined in order: a row's bits do not depend on its batch.
#include "decode_int8.hpp"

#include "decode_mfma.hpp"

namespace rlt {
namespace {

constexpr int kWaves = kDecodeWaves;
constexpr int kXcds = kDecodeXcds;
constexpr int kTile = kDecodeTile;
constexpr int64_t kMaxGrid = 32768;
constexpr float kRescale = 8.f;  // the running maximum moves when a tile's exceeds it by 2^kRescale

struct DecodeI8Args {
  AttnI8Args s;
  float* ws_acc;        // [rows][hkv][splits][G][D]
  PartState* ws_state;  // [rows][hkv][splits][G]
  int splits;           // most splits of a row inside the tables' width
  int split_slots;      // split-dimension workgroups launched; each walks every split_slots-th split
  int xcd;              // the heads of a (split, row) share an XCD
};

// Parts of q and of the weights, and the type of the scores' operands.
template <typename T> struct Parts;
template <> struct Parts<bf16> { static constexpr int Q = 1, P = 2; using S = bf16; };
template <> struct Parts<f16> { static constexpr int Q = 1, P = 2; using S = f16; };
template <> struct Parts<float> { static constexpr int Q = 3, P = 2; using S = bf16; };

template <typename T, int D>
constexpr int kWavesPerEu = D == 256 ? (sizeof(T) == 4 ? 1 : 2) : sizeof(T) == 4 ? 3 : 4;  // as LDS holds

// PAD: heads of fewer than D dims, a multiple of 16.  q is 0 in the others, where K and V are codes of the
// head's last 16 dims (any codes: they are finite), and nothing of them is stored.
template <typename T, int D, bool PAD>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(kWavesPerEu<T, D>))) void decode_i8_kernel(DecodeI8Args p) {
  using S = typename Parts<T>::S;
  constexpr int NQ = Parts<T>::Q, NP = Parts<T>::P;
  constexpr int KD = D < 128 ? D : 128, KS = D / KD;  // dims of K at a time, of which a lane has LD: ST MFMA steps
  constexpr int LD = KD / 4, ST = LD / 8, KC = LD / 16;
  constexpr int DT = D / 16;           // output tiles of 16 dims
  constexpr int CH = D / 16;           // 16-byte chunks of a code row
  constexpr int TPI = 64 / CH;         // tokens a load instruction
  constexpr int NI = kTile / TPI;      // loads a tile, of K and of V
  constexpr int kScales = 2 * kTile * D, kWaveBytes = kScales + 512;  // K rows, V rows, two sets of K and V scales (one a token)
  constexpr int JROW = D + 4;
  constexpr int QE = D / 16, QROW = 2 * D;
  static_assert(16 * JROW * 4 <= kWaveBytes, "a wave's accumulators fit its tile");
  __shared__ __align__(16) uint8_t lds[kWaves][kWaveBytes];
  __shared__ __align__(16) uint8_t q_lds[NQ][16][QROW];
  PartState(*const state_lds)[16] = reinterpret_cast<PartState(*)[16]>(q_lds);

  const Attn8Args& a = p.s.a;
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  const int G = a.hq / a.hkv;
  const uint32_t columns = (G + 15) / 16, rows = static_cast<uint32_t>(a.rows);
  const uint32_t heads = a.hkv * columns;
  const uint32_t x = blockIdx.x % kXcds, t = blockIdx.x / kXcds;
  uint32_t gi, r;
  if (p.xcd) {  // workgroup b runs on XCD b % 8: the heads of a (split, row) on one XCD, back to back
    const uint32_t item = t / heads * kXcds + x;
    gi = item / rows * heads + t % heads;
    r = (item + item / rows) % rows;  // a row's splits on different ones
  } else {
    gi = blockIdx.x / rows;
    r = blockIdx.x % rows;
  }
  gi = uniform(gi), r = uniform(r);
  const int h = gi % heads / columns, c0 = gi % heads % columns * 16;
  const int live = min(G - c0, 16);  // query heads of this tile
  const int len = sequence_length(a, r);
  int split_len, ns;
  decode8_split_plan(len, kMfmaSplit, &split_len, &ns);
  const int col = lane & 15, j = lane >> 4;

  const int32_t* trow = a.tables + r * a.table_stride;
  const uint8_t* kh = a.k + h * a.kv_head;
  const uint8_t* vh = a.v + h * a.kv_head;
  const float* sh = (lane < kTile ? p.s.ks : p.s.vs) + h * a.s_head;
  const uint32_t token_bytes = static_cast<uint32_t>(a.kv_token);
  uint8_t* const k_lds = lds[wave];
  uint8_t* const v_lds = lds[wave] + kTile * D;
  // The swizzles are linear in the row's bits, so that a place is a base of the lane's xor a
  // constant; `opaque` keeps the compiler from holding one register for each in the tile loop.
  uint32_t k_read = col * D + 16 * (KC * j ^ k_swizzle<D>(col));
  const int vt = lane & 15, v_row = 4 * j + vt / 2 % 4 + 16 * (vt / 8);  // of a transposing read
  uint32_t v_read = v_row * D + 16 * v_swizzle<D>(v_row) + 8 * (vt & 1);
  uint32_t k_chunk = 16 * (lane % CH ^ k_swizzle<D>(lane / CH)), v_chunk = 16 * (lane % CH ^ v_swizzle<D>(lane / CH));
  uint32_t load_row = lane / CH;
  auto opaque = [](uint32_t& x) __attribute__((always_inline)) { asm volatile("" : "+v"(x)); };
  const uint32_t k_at = lds_address(k_lds), v_at = k_at + kTile * D, s_at = k_at + kScales;

  // Of q, 16 threads a head.
  float y[QE];
  auto load_q = [&]() __attribute__((always_inline)) {
    uint32_t thread = threadIdx.x;
    opaque(thread);
    const T* src = static_cast<const T*>(a.q) + r * a.q_row + (h * G + c0 + min(static_cast<int>(thread) / 16, live - 1)) * a.q_head +
                   static_cast<int>(thread) % 16 * QE * a.q_dim;
#pragma unroll
    for (int e = 0; e < QE; ++e) y[e] = !PAD || static_cast<int>(thread) % 16 * QE + e < a.d ? load_elem(src + e * a.q_dim) : 0.f;
  };
  // A wave's tile i of split sp is its (4 i + wave)-th 32 tokens.  Lane l holds where the 16 tokens
  // of half l % 2 of tile first + l / 2 begin (past the row's end anything inside the tables).
  int64_t unit_kv, unit_s;
  auto load_units = [&](int sp, int first) __attribute__((always_inline)) {
    uint32_t of = lane;
    opaque(of);
    const int64_t want = static_cast<int64_t>(sp) * split_len + ((first + static_cast<int>(of) / 2) * kWaves + wave) * kTile + of % 2 * 16;
    const int tok = static_cast<int>(min(want, a.max_len - 16));
    const int page = tok / a.page, slot = tok - page * a.page;
    const int64_t blk = block_of(a, trow[page]);
    unit_kv = blk * a.kv_block + slot * a.kv_token;
    unit_s = blk * a.s_block;
  };
  int sp = gi / heads;
  if (sp >= ns) return;
  load_q();
  load_units(sp, 0);
  for (;;) {
    const int t0 = sp * split_len + wave * kTile, end = min(len, (sp + 1) * split_len);  // this wave's first token
    const int tiles = end > t0 ? (end - t0 + kWaves * kTile - 1) / (kWaves * kTile) : 0;
    auto chunk_of = [&](uint32_t chunk) __attribute__((always_inline)) { return PAD ? min(chunk, static_cast<uint32_t>(a.d - 16)) : chunk; };
    // At head_dim 64 a token's row is half a line of the L2, where it stays for the next head (256 rows
    // of 1024-8192 tokens, 16 + 8 heads, 304 us as other loads, so 268).
    auto load16 = [](uint32_t lds_byte, uint32_t offset, const uint8_t* from) __attribute__((always_inline)) {
      if constexpr (D == 64) dma16_kept(lds_byte, offset, from);
      else dma16(lds_byte, offset, from);
    };
    // Tokens past the end re-read the last one: in bounds, and masked below.
    auto load_rows = [&](int tile, const uint8_t* base, uint32_t to, uint32_t chunk, auto swizzle) __attribute__((always_inline)) {
      const int last = min(end - 1 - t0 - tile * (kWaves * kTile), kTile - 1);  // row
      auto unit_at = [&](int half) __attribute__((always_inline)) {  // an instruction's tokens lie in one
        const int unit = tile % 32 * 2 + half;
        return static_cast<int64_t>(__builtin_amdgcn_readlane(static_cast<int>(unit_kv >> 32), unit)) << 32 |
               static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(unit_kv), unit));
      };
      if (last == kTile - 1) {
        const uint32_t row = __umul24(load_row, token_bytes);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint8_t* from = base + unit_at(half);
#pragma unroll
          for (int i = half * NI / 2; i < (half + 1) * NI / 2; ++i, from += TPI * token_bytes)
            load16(to + i * 1024, row + chunk_of(chunk ^ (16 * swizzle(i * TPI))), from);
        }
        return;
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int half = min(i * TPI, last) / 16;
        const uint32_t tok = min(i * TPI + static_cast<int>(load_row), last) - 16 * half;
        load16(to + i * 1024, __umul24(tok, token_bytes) + chunk_of(chunk ^ (16 * swizzle(i * TPI))), base + unit_at(half));
      }
    };
    auto load_k = [&](int tile) __attribute__((always_inline)) {
      const int at = min(lane & (kTile - 1), end - 1 - t0 - tile * (kWaves * kTile));
      dma_dword(s_at + tile % 2 * 256, sh + __shfl(unit_s, tile % 32 * 2 + at / 16, 64));
      load_rows(tile, kh, k_at, k_chunk, k_swizzle<D>);
    };
    auto load_v = [&](int tile) __attribute__((always_inline)) { load_rows(tile, vh, v_at, v_chunk, v_swizzle<D>); };
    if (tiles > 0) {  // the first tile's loads go out before q is worked on
      load_k(0);
      load_v(0);
    }
    // q's parts, B operands: lane (col, j) holds dims [KD c + LD j, + LD) of query head c0 +
    // col, 8 of them a step.
    u32x4 qw[NQ][ST * KS];
    {
      uint32_t thread = threadIdx.x;
      opaque(thread);
      const int qh = thread / 16, qd = thread % 16 * QE;
#pragma unroll
      for (int e = 0; e < QE; ++e)  // infinities as NaN, which no other head's maximum takes up
        if ((__float_as_uint(y[e]) & 0x7f800000u) == 0x7f800000u) y[e] = __uint_as_float(0x7fc00000u);
#pragma unroll
      for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int e = 0; e < QE; e += 2) {
          uint32_t word;
          if constexpr (NQ > 1) {  // the top 16 bits: the rest is exact, and the third part holds all of it
            const uint32_t lo = __float_as_uint(y[e]), hi = __float_as_uint(y[e + 1]);
            word = lo >> 16 | (hi & 0xffff0000u);
            y[e] -= __uint_as_float(lo & 0xffff0000u);
            y[e + 1] -= __uint_as_float(hi & 0xffff0000u);
          } else {
            word = MfmaOps<S>::pack2(y[e], y[e + 1]);
          }
          *reinterpret_cast<uint32_t*>(q_lds[i][qh] + 2 * (qd + e)) = word;
        }
      wait_lds();
      asm volatile("s_barrier" ::: "memory");  // (__syncthreads() would wait for the tile)
#pragma unroll
      for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
          for (int e = 0; e < ST; ++e)
            qw[i][ST * c + e] = *reinterpret_cast<const u32x4*>(q_lds[i][col] + 2 * (KD * c + LD * j + 8 * e));
      wait_lds();
      asm volatile("s_barrier" ::: "memory");
    }
    f32x4 acc[DT];
#pragma unroll
    for (int c = 0; c < DT; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f, e = kNoExponent;

#pragma unroll 1
    for (int tile = 0; tile < tiles; ++tile) {
      const bool more = tile + 1 < tiles;
      opaque(k_read), opaque(v_read), opaque(k_chunk), opaque(v_chunk), opaque(load_row);
      const float* scales = reinterpret_cast<const float*>(lds[wave] + kScales + tile % 2 * 256);  // K's, then V's
      wait_loads<NI>();  // V may still be on its way
      u32x4 ka[2][KS][KC];
      float kf[2], vf[2];  // of the two halves: 16 tokens lie in one block
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        kf[u] = scales[16 * u], vf[u] = scales[kTile + 16 * u];
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
          for (int e = 0; e < KC; ++e) ka[u][c][e] = *reinterpret_cast<const u32x4*>(k_lds + (k_read ^ (16 * (KD / 16 * c + e))) + 16 * u * D);
      }
      wait_lds();
      if (more) load_k(tile + 1);
      // S^T: element r of half u is token 16 u + 4 j + r of the tile.
      f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
          for (int q4 = 0; q4 < ST; ++q4) {
            u32x4 kw;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint2 pairs = code_pairs<S>(ka[u][c][q4 / 2][q4 % 2 * 2 + i]);
              kw[2 * i] = pairs.x, kw[2 * i + 1] = pairs.y;
            }
#pragma unroll
            for (int i = 0; i < NQ; ++i) s[u] = mma16<S>(kw, qw[i][ST * c + q4], s[u]);
          }
      }
      const int first = t0 + tile * (kWaves * kTile);
      float top = -INFINITY, highest = -INFINITY;  // of the scores, of the scales' exponents
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float f = block_scale(kf[u]) * a.qscale;
        vf[u] = block_scale(vf[u]);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][i] = rounded_product(s[u][i], f);  // as their maximum is
      }
      if (first + kTile > end) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (first + 16 * u >= end) vf[u] = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (first + 16 * u + 4 * j + i >= end) s[u][i] = -INFINITY;
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        highest = fmaxf(highest, scale_exponent(vf[u]));
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[u][i]);
      }
      top = strided_max<16>(top);
      // No weight is above 2^(top - m + highest - e); it may be 2^15.
      if (__builtin_amdgcn_ballot_w64(top > m + kRescale || top - m + highest > e + kMostExponent) != 0) {
        const float mn = fmaxf(m, ceilf(top));
        const float down = mn - m;  // +inf at the first key, NaN before it
        float en = e - down;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float x = s[u][0];
#pragma unroll
          for (int i = 1; i < 4; ++i) x = fmaxf(x, s[u][i]);
          en = fmaxf(en, ceilf(strided_max<16>(x) - mn) + scale_exponent(vf[u]) - kUsualExponent);
        }
        const bool none = mn == -INFINITY;
        const float corr = none ? 0.f : fast_exp2(e - down - en);
        l = none ? 0.f : l * fast_exp2(-down);
        m = mn;
        e = none ? kNoExponent : en;
#pragma unroll
        for (int c = 0; c < DT; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[c][i] *= corr;
      }
      const float off = m == -INFINITY ? 0.f : m;  // only -inf scores so far: they weigh 0
      // P^T, element i of the k-step is token 16 (i / 4) + 4 j + i % 4, times its V scale.
      u32x4 pb[NP];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float w[4];
        const float g = weight_scale(vf[u], e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = fast_exp2(s[u][i] - off);
          l += w[i];
          w[i] *= g;
          asm("" : "+v"(w[i]));  // the parts are of one product, rounded to fp32
        }
#pragma unroll
        for (int n = 0; n < NP; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t x = MfmaOps<f16>::pack2(w[2 * i], w[2 * i + 1]);
            pb[n][2 * u + i] = x;
            w[2 * i] -= f16_value(x), w[2 * i + 1] -= f16_value(x >> 16);
          }
      }
      if (more) wait_loads<NI + 1>();  // the next tile's K and scales may still be on their way
      else wait_loads<0>();
      // V^T, 16 dims a tile: in each 16-lane group lane L addresses 8 bytes of token row L / 2 of
      // its 8, and gets one dim of all 8.
      i32x2 codes[DT];
#pragma unroll
      for (int c = 0; c < DT; ++c)
        codes[c] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(v_lds + (v_read ^ (16 * c))));
      wait_lds();
      if (more) load_v(tile + 1);
      if (more && tile % 32 == 30) load_units(sp, tile + 2);  // the next tile's loads were the last of these
#pragma unroll
      for (int c = 0; c < DT; ++c) {
        u32x4 va;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint2 pairs = code_pairs<f16>(static_cast<uint32_t>(codes[c][i]));
          va[2 * i] = pairs.x, va[2 * i + 1] = pairs.y;
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) acc[c] = mma16<f16>(va, pb[i], acc[c]);
      }
    }
    // Join the waves, in order.
    l = strided_sum<16>(l);
    uint32_t thread = threadIdx.x;
    opaque(thread);
    float* const join = reinterpret_cast<float*>(lds[wave]) + thread % 16 * JROW + thread / 16 % 4 * 4;  // [16 columns][JROW]
#pragma unroll
    for (int c = 0; c < DT; ++c) *reinterpret_cast<f32x4*>(join + 16 * c) = acc[c];
    if (thread % 64 < 16) state_lds[wave][thread % 16] = PartState{m, l, e, 0.f};
    __syncthreads();
    for (int o = thread; o < live * D; o += 64 * kWaves) {
      const int hd = o / D, d = o % D;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, state_lds[w][hd].m);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f, y = 0.f, exponent = kNoExponent;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) exponent = fmaxf(exponent, state_lds[w][hd].e + (state_lds[w][hd].m - base));
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const PartState x = state_lds[w][hd];
        sum = fmaf(x.l, fast_exp2(x.m - base), sum);
        y = fmaf(reinterpret_cast<const float*>(lds[w])[hd * JROW + d], fast_exp2(x.e + (x.m - base) - exponent), y);
      }
      const int q = c0 + hd;  // of the KV head's
      if (PAD && ns == 1 && d >= a.d) continue;
      if (ns == 1) {
        store_elem(static_cast<T*>(a.out) + r * a.o_row + (h * G + q) * a.o_head + d * a.o_dim,
                   len > 0 ? ldexpf(y * (1.f / sum), static_cast<int>(exponent)) : 0.f);
      } else {
        const int64_t at = ((static_cast<int64_t>(r) * a.hkv + h) * p.splits + sp) * G + q;
        p.ws_acc[at * D + d] = y;
        if (d == 0) p.ws_state[at] = PartState{top, sum, exponent, 0.f};
      }
    }
    sp += p.split_slots;
    if (sp >= ns) return;
    __syncthreads();
    load_q();
    load_units(sp, 0);
  }
}

// A workgroup a (row, query head) of more than one split: lane i of every wave holds split i's
// state; wave w adds the accumulators of every fourth split from w on, all on their way at once, and
// the waves are added in order.  (One wave a (row, query head), eight splits at a time: two rows of
// 30000 tokens, 64 splits, 9.6 us.)
template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) void decode_i8_merge_kernel(DecodeI8Args p) {
  constexpr int E = D / 64, PER = kDecode8MaxSplits / kWaves;
  __shared__ float sums[kWaves][D];
  const Attn8Args& a = p.s.a;
  const int r = static_cast<int>(blockIdx.x / a.hq), hq = static_cast<int>(blockIdx.x % a.hq);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int G = a.hq / a.hkv, h = hq / G, j = hq - h * G;
  int split_len, ns;
  decode8_split_plan(sequence_length(a, r), kMfmaSplit, &split_len, &ns);
  if (ns < 2) return;
  const int64_t base = (static_cast<int64_t>(r) * a.hkv + h) * p.splits * G + j;
  const PartState part = lane < ns ? p.ws_state[base + static_cast<int64_t>(lane) * G] : PartState{-INFINITY, 0.f, kNoExponent, 0.f};
  const float* src = p.ws_acc + base * D + lane;
  float x[PER][E], acc[E] = {};
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (kWaves * i + wave < ns) x[i][e] = src[static_cast<int64_t>(kWaves * i + wave) * G * D + 64 * e];
  const float top = group_max<64>(part.m);
  const float off = top == -INFINITY ? 0.f : top;
  const float at = part.e + (part.m - off);
  const float exponent = fmaxf(group_max<64>(at), kNoExponent);
  const float w = fast_exp2(at - exponent);
  const float inv = 1.f / group_sum<64>(part.l * fast_exp2(part.m - off));
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (kWaves * i + wave < ns) {
      const float wi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), kWaves * i + wave));
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(x[i][e], wi, acc[e]);
    }
#pragma unroll
  for (int e = 0; e < E; ++e) sums[wave][lane + 64 * e] = acc[e];
  __syncthreads();
  T* orow = static_cast<T*>(a.out) + r * a.o_row + hq * a.o_head;
  for (int d = threadIdx.x; d < a.d; d += 64 * kWaves) {
    float y = 0.f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) y += sums[v][d];
    store_elem(orow + d * a.o_dim, ldexpf(y * inv, static_cast<int>(exponent)));
  }
}

// The kernel's head size.
int64_t padded_dims(int64_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

template <typename T, int D>
void launch_size(const DecodeI8Args& p, unsigned grid, hipStream_t stream) {
  const Attn8Args& a = p.s.a;
  if (a.d == D) hipLaunchKernelGGL((decode_i8_kernel<T, D, false>), dim3(grid), dim3(64 * kWaves), 0, stream, p);
  else hipLaunchKernelGGL((decode_i8_kernel<T, D, true>), dim3(grid), dim3(64 * kWaves), 0, stream, p);
  if (p.splits < 2) return;
  hipLaunchKernelGGL((decode_i8_merge_kernel<T, D>), dim3(static_cast<unsigned>(a.rows * a.hq)), dim3(64 * kWaves), 0, stream, p);
}

template <typename T>
void launch_type(const DecodeI8Args& p, unsigned grid, hipStream_t stream) {
  switch (padded_dims(p.s.a.d)) {
    case 64: launch_size<T, 64>(p, grid, stream); break;
    case 128: launch_size<T, 128>(p, grid, stream); break;
    default: launch_size<T, 256>(p, grid, stream); break;
  }
}

}  // namespace

bool decode_i8_shape(int64_t hq, int64_t hkv, int64_t d, int64_t page) {
  return d > 0 && d <= 256 && d % 16 == 0 && page > 0 && page % 16 == 0 && hkv > 0 && hq > 0;
}

int64_t decode_i8_workspace(int64_t rows, int64_t max_len, int64_t hq, int64_t d) {
  const int64_t ns = decode8_most_splits(max_len, kMfmaSplit);
  return ns > 1 ? rows * ns * hq * (padded_dims(d) * 4 + static_cast<int64_t>(sizeof(PartState))) : 0;
}

int launch_decode_i8(const AttnI8Args& s, int dtype, void* ws, hipStream_t stream, const char* name) {
  const Attn8Args& a = s.a;
  DecodeI8Args p{};
  p.s = s;
  p.splits = decode8_most_splits(a.max_len, kMfmaSplit);
  const int64_t items = a.rows * a.hkv * ((a.hq / a.hkv + 15) / 16);
  p.split_slots = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(p.splits, kMaxGrid / items)));
  p.xcd = a.rows * p.split_slots % kXcds == 0;
  p.ws_acc = static_cast<float*>(ws);
  p.ws_state = reinterpret_cast<PartState*>(p.ws_acc + a.rows * p.splits * a.hq * padded_dims(a.d));
  if (items * p.split_slots > kMaxBlocks || a.rows * a.hq > kMaxBlocks) return fail(RLT_EUNSUPPORTED, "%s: too many rows", name);
  const unsigned grid = static_cast<unsigned>(items * p.split_slots);
  switch (dtype) {
    case RLT_BFLOAT16: launch_type<bf16>(p, grid, stream); break;
    case RLT_FLOAT16: launch_type<f16>(p, grid, stream); break;
    default: launch_type<float>(p, grid, stream); break;
  }
  return check_launch(name);
}

}  // namespace rlt
