// Decode over the 8-bit KV cache on the matrix cores.  A key is used by the G query heads
// of its KV head, which on the vector units costs 4 D G flops a token in fp32 and G
// accumulators; here up to 16 heads are the columns of one tile.
//
// A workgroup takes one (row, KV head, 16 query heads, split); its four waves take every
// fourth 32 tokens of the split each, through LDS of their own (no barrier):
// - S^T = K Q^T on the 16-bit MFMA of q's type (16x16x32; an fp32 q in three bf16 parts): a
//   code is a bf16 or an fp16 exactly, and its token's scale multiplies the fp32 sum.  (The
//   scaled 8-bit MFMA would take codes and scales as they are, but drops what lies 2^-11
//   below the largest product of its 128; the 16-bit ones keep fp32's bits.)
// - O^T += V^T P^T on the bf16 MFMA (16x16x32): P stays in the registers S^T left it in,
//   times its token's V scale, in two bf16 parts (16 bits) for bf16 and fp16, three for fp32 (one
//   part for bf16 would save 1% of a large call and 4% of a small one, and lose half a step of
//   the output's type again); its sum is taken before that.  V's codes come from transposing
//   8-bit LDS reads and become bf16 exactly.
// Bytes bound it.  Tiles go from memory into LDS directly: K of the next one as soon as this
// one's K is in registers, V likewise, one buffer each, so that a wave needs 8 KiB of LDS and
// no registers for what is on its way, and sixteen waves a CU (twelve for fp32, eight at
// head_dim 256) keep 128 KiB in flight.  The heads of a row's split run on one XCD at the
// same time, which reads whole token rows of the cache: 256 rows of 1024-8192 tokens, 16 + 8
// heads x 128, take 468 us with a head an XCD, 440 (5.5 TB/s) so.  24 rows of 512-4096, 32 + 8
// heads, fp16, 114 MB, take 32 us, 4.6 of them the merge.
#include <type_traits>

#include "decode_fp8.hpp"
#include "mfma.hpp"

namespace rlt {
namespace {

constexpr int kWaves = 4;
constexpr int kXcds = 8;
constexpr int kTile = 32;
constexpr float kRescale = 8.f;  // the running maximum moves when a tile's exceeds it by 2^kRescale

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

// Parts of q and of P, and the type of the scores' operands.
template <typename T> struct Parts;
template <> struct Parts<bf16> { static constexpr int Q = 1, P = 2; using S = bf16; };
template <> struct Parts<f16> { static constexpr int Q = 1, P = 2; using S = f16; };
template <> struct Parts<float> { static constexpr int Q = 3, P = 3; using S = bf16; };

__device__ __forceinline__ uint32_t bf16_pair(float x, float y) { return MfmaOps<bf16>::pack2(x, y); }

// Two codes of a word (its low or high half) as bf16 or fp16, both exact.
template <typename S>
__device__ __forceinline__ uint32_t code_pair(uint32_t word, bool high) {
  const int w = static_cast<int>(word);
  if constexpr (std::is_same_v<S, f16>)
    return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
  else
    return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
}

template <typename S>
__device__ __forceinline__ f32x4 mma16(u32x4 x, u32x4 y, f32x4 c) {
  if constexpr (std::is_same_v<S, f16>) return __builtin_amdgcn_mfma_f32_16x16x32_f16(as_v8<f16x8>(x), as_v8<f16x8>(y), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_v8<bf16x8>(x), as_v8<bf16x8>(y), c, 0, 0, 0);
}

// Direct global -> LDS loads, as assembly so that the compiler's wait analysis, which cannot
// tell the tiles apart, does not wait for one still in flight: the kernel orders them with
// vmcnt waits of its own.  Lane l writes bytes [16 l, 16 l + 16) (dword l of the scales' byte)
// after the LDS byte address in M0.  Earlier LDS reads are complete first.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(uint32_t lds_byte, uint32_t offset, const uint8_t* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds_byte), "v"(offset), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void dma_byte(uint32_t lds_byte, const uint8_t* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off" ::"s"(lds_byte), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(uniform(static_cast<int>((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p)));
}
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Where chunk c of row r lies: at c ^ k_swizzle(r) in K, c ^ v_swizzle(r) in V.  Rows of D bytes:
// the 8 (16) rows that one pass of a K read over 128 (256) bytes of banks serves, rows r0..r2
// (r0..r3), and the 8 (16) of a transposing V read, r0 r1 r4 (r0 r1 r2 r4), fall into distinct ones.
template <int D>
__device__ __forceinline__ int k_swizzle(int r) {
  const int r0 = r & 1, r1 = r >> 1 & 1, r2 = r >> 2 & 1, r3 = r >> 3 & 1;
  return D == 64 ? (r1 ^ r3) | r2 << 1 : D == 128 ? (r0 ^ r3) | r1 << 1 | r2 << 2 : r & 15;
}
template <int D>
__device__ __forceinline__ int v_swizzle(int r) {
  const int r0 = r & 1, r1 = r >> 1 & 1, r2 = r >> 2 & 1, r4 = r >> 4 & 1;
  return D == 64 ? (r1 ^ r2) | r4 << 1 : D == 128 ? (r0 ^ r2) | r1 << 1 | r4 << 2 : r0 | r1 << 1 | r4 << 2 | r2 << 3;
}

template <typename T, int D>
constexpr int kWavesPerEu = D == 256 ? (sizeof(T) == 4 ? 1 : 2) : sizeof(T) == 4 ? 3 : 4;  // as LDS holds

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(kWavesPerEu<T, D>))) void decode8_mfma_kernel(Decode8Args p) {
  using S = typename Parts<T>::S;
  constexpr int NQ = Parts<T>::Q, NP = Parts<T>::P;
  constexpr int KS = (D + 127) / 128;  // 128 dims each: four MFMA steps
  constexpr int DT = D / 16;           // output tiles of 16 dims
  constexpr int CH = D / 16;           // 16-byte chunks of a code row
  constexpr int TPI = 64 / CH;         // tokens a load instruction
  constexpr int NI = kTile / TPI;      // loads a tile, of K and of V
  constexpr int kScales = 2 * kTile * D, kWaveBytes = kScales + 512;  // K rows, V rows, two sets of K and V scale bytes (a dword each)
  constexpr int JROW = D + 4;
  constexpr int QE = D / 16, QROW = 2 * D;
  static_assert(16 * JROW * 4 <= kWaveBytes, "a wave's accumulators fit its tile");
  __shared__ __align__(16) uint8_t lds[kWaves][kWaveBytes];
  __shared__ __align__(16) uint8_t q_lds[NQ][16][QROW];
  float2(*const ml_lds)[16] = reinterpret_cast<float2(*)[16]>(q_lds);

  const Attn8Args& a = p.a;
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
  const uint8_t* sh = (lane < kTile ? a.ks : a.vs) + h * a.s_head;
  const uint32_t token_bytes = static_cast<uint32_t>(a.kv_token);
  uint8_t* const k_lds = lds[wave];
  uint8_t* const v_lds = lds[wave] + kTile * D;
  // The swizzles are linear in the row's bits, so that a place is a base of the lane's xor a
  // constant; `opaque` keeps the compiler from holding one register for each in the tile loop.
  uint32_t k_read = col * D + 16 * ((D >= 128 || j < 2 ? 2 * j : 0) ^ k_swizzle<D>(col));
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
    for (int e = 0; e < QE; ++e) y[e] = load_elem(src + e * a.q_dim);
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
    unit_s = blk * a.s_block + slot * a.s_token;
  };
  int sp = gi / heads;
  if (sp >= ns) return;
  load_q();
  load_units(sp, 0);
  for (;;) {
    const int t0 = sp * split_len + wave * kTile, end = min(len, (sp + 1) * split_len);  // this wave's first token
    const int tiles = end > t0 ? (end - t0 + kWaves * kTile - 1) / (kWaves * kTile) : 0;
    // Tokens past the end re-read the last one: in bounds, and masked below.
    auto load_rows = [&](int tile, const uint8_t* base, uint32_t to, uint32_t chunk, auto swizzle) __attribute__((always_inline)) {
      const int last = min(end - 1 - t0 - tile * (kWaves * kTile), kTile - 1);  // row
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int half = min(i * TPI, last) / 16, unit = tile % 32 * 2 + half;  // the instruction's tokens lie in one
        const int64_t from = static_cast<int64_t>(__builtin_amdgcn_readlane(static_cast<int>(unit_kv >> 32), unit)) << 32 |
                             static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(unit_kv), unit));
        const uint32_t tok = min(i * TPI + static_cast<int>(load_row), last) - 16 * half;
        dma16(to + i * 1024, __umul24(tok, token_bytes) + (chunk ^ (16 * swizzle(i * TPI))), base + from);
      }
    };
    auto load_k = [&](int tile) __attribute__((always_inline)) {
      const int at = min(lane & (kTile - 1), end - 1 - t0 - tile * (kWaves * kTile));
      dma_byte(s_at + tile % 2 * 256, sh + (__shfl(unit_s, tile % 32 * 2 + at / 16, 64) + at % 16 * a.s_token));
      load_rows(tile, kh, k_at, k_chunk, k_swizzle<D>);
    };
    auto load_v = [&](int tile) __attribute__((always_inline)) { load_rows(tile, vh, v_at, v_chunk, v_swizzle<D>); };
    if (tiles > 0) {  // the first tile's loads go out before q is worked on
      load_k(0);
      load_v(0);
    }
    // q's parts, B operands: lane (col, j) holds dims [128 c + 32 j, + 32) of query head c0 +
    // col, 8 of them a step.
    u32x4 qw[NQ][4 * KS];
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
      const u32x4 zero = {0u, 0u, 0u, 0u};
      const bool in = D >= 128 || j < 2;  // head_dim 64: the upper half of the 128 is 0
#pragma unroll
      for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          const int d0 = in ? 128 * c + 32 * j : 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(q_lds[i][col] + 2 * (d0 + 8 * e));
            qw[i][4 * c + e] = in ? w : zero;
          }
        }
      wait_lds();
      asm volatile("s_barrier" ::: "memory");
    }
    f32x4 acc[DT];
#pragma unroll
    for (int c = 0; c < DT; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

#pragma unroll 1
    for (int tile = 0; tile < tiles; ++tile) {
      const bool more = tile + 1 < tiles;
      opaque(k_read), opaque(v_read), opaque(k_chunk), opaque(v_chunk), opaque(load_row);
      const uint32_t* scales = reinterpret_cast<const uint32_t*>(lds[wave] + kScales + tile % 2 * 256);  // K's, then V's
      wait_loads<NI>();  // V may still be on its way
      u32x4 ka[2][KS][2], kb[2];
      const bool in = D >= 128 || j < 2;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        kb[u] = *reinterpret_cast<const u32x4*>(scales + 16 * u + 4 * j);
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(k_lds + (k_read ^ (16 * (8 * c + e))) + 16 * u * D);
            ka[u][c][e] = in ? w : u32x4{0u, 0u, 0u, 0u};
          }
      }
      const uint32_t vb = scales[kTile + (lane & (kTile - 1))] & 255u;
      wait_lds();
      if (more) load_k(tile + 1);
      // S^T: element r of half u is token 16 u + 4 j + r of the tile.
      f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            u32x4 kw;
#pragma unroll
            for (int e = 0; e < 4; ++e) kw[e] = code_pair<S>(ka[u][c][q4 / 2][q4 % 2 * 2 + e / 2], e % 2);
#pragma unroll
            for (int i = 0; i < NQ; ++i) s[u] = mma16<S>(kw, qw[i][4 * c + q4], s[u]);
          }
      }
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = s[u][e] * scale_value(kb[u][e] & 255u) * a.qscale;
          s[u][e] = t0 + tile * (kWaves * kTile) + 16 * u + 4 * j + e < end ? x : -INFINITY;
          top = fmaxf(top, s[u][e]);
        }
      f32x4 sv[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const u32x4 b = *reinterpret_cast<const u32x4*>(scales + kTile + 16 * u + 4 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) sv[u][e] = scale_value(b[e] & 255u);
      }
      float bias = 0.f;
      if (__builtin_amdgcn_ballot_w64(vb > kFreeScale)) bias = group_max<64>(value_bias(vb == 255u ? 0u : vb));
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
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = fast_exp2(s[u][e] - off);
          l += w[e];
          w[e] = w[e] * kLift * sv[u][e];
        }
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            pb[i][2 * u + e] = bf16_pair(w[2 * e], w[2 * e + 1]);
            w[2 * e] -= bf16_lo(pb[i][2 * u + e]), w[2 * e + 1] -= bf16_hi(pb[i][2 * u + e]);
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
        for (int e = 0; e < 4; ++e) va[e] = code_pair<bf16>(static_cast<uint32_t>(codes[c][e / 2]), e % 2);
#pragma unroll
        for (int i = 0; i < NP; ++i) acc[c] = mma16<bf16>(va, pb[i], acc[c]);
      }
    }
    // Join the waves, in order.
    l = strided_sum<16>(l);
    uint32_t thread = threadIdx.x;
    opaque(thread);
    float* const join = reinterpret_cast<float*>(lds[wave]) + thread % 16 * JROW + thread / 16 % 4 * 4;  // [16 columns][JROW]
#pragma unroll
    for (int c = 0; c < DT; ++c) *reinterpret_cast<f32x4*>(join + 16 * c) = acc[c];
    if (thread % 64 < 16) ml_lds[wave][thread % 16] = make_float2(m, l);
    __syncthreads();
    for (int o = thread; o < live * D; o += 64 * kWaves) {
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
        y = fmaf(reinterpret_cast<const float*>(lds[w])[hd * JROW + d], c, y);
      }
      const int q = c0 + hd;  // of the KV head's
      if (ns == 1) {
        store_elem(static_cast<T*>(a.out) + r * a.o_row + (h * G + q) * a.o_head + d * a.o_dim, len > 0 ? y * (1.f / kLift / sum) : 0.f);
      } else {
        const int64_t at = ((static_cast<int64_t>(r) * a.hkv + h) * p.splits + sp) * G + q;
        p.ws_acc[at * D + d] = y;
        if (d == 0) p.ws_ml[at] = make_float2(top, sum);
      }
    }
    sp += p.split_slots;
    if (sp >= ns) return;
    __syncthreads();
    load_q();
    load_units(sp, 0);
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
