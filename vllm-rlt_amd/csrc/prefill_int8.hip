// Packed chunked prefill over the block-scaled 8-bit KV cache, bottom-right causal, on the
// matrix cores (head sizes of multiples of 16 up to 256, pages of a power of two of at least 16
// tokens; int8.hpp has the softmax, prefill_plan.hpp the launch's plan).
//
// A workgroup of 4 waves takes 128 (query row, query head) pairs of one (sequence, KV head), a
// row's heads together, over a segment of its keys, a wave 32 of them, 64 keys a tile, four units
// of 16 keys that have one scale of K and one of V each.  (A tile of one head's rows only: four
// chunks of 740-983 rows over up to 4400 keys, 16 + 4 heads, 125.8 us, so 118.2; sixteen of 8 rows
// over 4000, 32 + 8 heads, 123 and 44.)
// - S^T = K Q^T on the 16-bit MFMA of q's type (32x32x16; an fp32 q in three bf16 parts).  Codes
//   become bf16 or fp16, exactly, once a workgroup, on their way into LDS; their unit's scale
//   multiplies the sums, in the instruction that takes the running maximum off.
// - O^T += V^T W^T on the fp16 MFMA, codes as fp16 likewise; V^T comes from transposing LDS
//   reads, W, the probabilities times their unit's V scale, from the registers S^T left it
//   in: in one part, 11 bits, for bf16, in two for fp16 and fp32.  (An fp16 output is off by 2.1e-4 of the
//   rms so, its own rounding; with one part by 2.9e-4, for 10 to 21% less time, eight chunks as below 349 us
//   where two take 445.  A bf16 output is off by 0.00167 with one and 0.00166 with two, for 345 and 440.)
// Products (42% of a SIMD's cycles) and vector work (69%: conversions, exponentials, sums) bound it: eight
// 512-token chunks over 1024-15360 keys, 16 heads x 128, bf16, take 345 to 363 us by run with their
// merge, 780 to 820 TFLOP/s, where a large product of matrices reaches 1210.  Short launches are 6 us of plan and
// first loads, a tile 1.6 to 2.4 us, and 4 us of merge.
#include "prefill_int8.hpp"

#include "prefill_plan.hpp"

namespace rlt {
namespace {

struct PrefillI8Args {
  Prefill8Args p;  // (part_ml unused)
  const float* ks;
  const float* vs;
  PartState* part_state;  // [slots][hq]
};

constexpr int kUnits = kBN / 16;

// f(0), f(1), ..., f(N - 1) of constants.
template <typename F, int... I>
__device__ __forceinline__ void unrolled_of(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void unrolled(F f) {
  unrolled_of(f, std::make_integer_sequence<int, N>{});
}

// Parts of q and of the weights, and the type of the scores' operands.
template <typename T> struct Parts;
template <> struct Parts<bf16> { static constexpr int Q = 1, P = 1; using S = bf16; };
template <> struct Parts<f16> { static constexpr int Q = 1, P = 2; using S = f16; };
template <> struct Parts<float> { static constexpr int Q = 3, P = 2; using S = bf16; };

// Workgroups a CU, as LDS and registers hold.
template <typename T, int D>
constexpr int kWorkgroups = sizeof(T) == 4 || D == 256 ? 1 : 2;

// PAD: heads of fewer than D dims, a multiple of 16.  q is 0 in the others, where K and V are codes of the
// head's last 16 dims (any codes: they are finite), and nothing of them is stored.
template <typename T, int D, bool PAD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kWorkgroups<T, D>))) void prefill_i8_kernel(PrefillI8Args args) {
  using S = typename Parts<T>::S;
  using SOps = MfmaOps<S>;
  using Ops = MfmaOps<f16>;
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
  __shared__ __align__(16) float f_lds[2][2][kUnits];  // of the units: K's scale times the softmax scale, V's scale

  const Prefill8Args& p = args.p;
  const Attn8Args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  Item it;
  if (!find_item<true>(p, &it)) return;
  const int seq = uniform(it.seq), kvh = uniform(it.head), row0 = uniform(it.row0), nq = uniform(it.nq);
  const int group = p.group, rows = nq * group;  // row i of the tiles is row i / group of query head i % group
  const int len = uniform(it.len);
  const int prefix = len - nq;  // query row i sees keys up to prefix + i
  const int qt0 = uniform(it.tile) * kBM;
  const int wg_keys = min(prefix + min((qt0 + kBM - 1) / group + 1, nq), len);  // keys that some row of the workgroup sees
  const int first_tile = uniform(it.seg * it.seg_tiles);
  const int ntiles = min(first_tile + uniform(it.seg_tiles), (max(wg_keys, 0) + kBN - 1) / kBN);
  if (it.segs > 1 && it.seg > 0 && ntiles <= first_tile) return;  // the merge skips such a segment

  const int half = lane >> 5, col = lane & 31;
  const int wave_row0 = qt0 + wave * 32;
  const int my_row = wave_row0 + col;
  const bool row_valid = my_row < rows;
  const int at_row = min(my_row, rows - 1) / group, h = kvh * group + min(my_row, rows - 1) - at_row * group;
  const int limit = row_valid ? prefix + at_row : -1;  // last key this lane's query sees
  const int wave_first = prefix + wave_row0 / group, wave_last = prefix + min((wave_row0 + 31) / group, nq - 1);
  const bool wave_live = wave_row0 < rows;

  // q's parts, B operands: lane (col, half) holds dims [16 c + 8 half, + 8) of row col for step c.
  // An fp16 q goes in as it is, the others times 2^q_exp.
  constexpr bool LATE = std::is_same_v<S, f16>;
  u32x4 qw[NQ][KS];

  // Staging: thread (token, chunk), PASSES tokens TPP apart.  A wave's tokens of a pass are of one unit,
  // so of one block, and their addresses are the wave's but for an offset that stays.  Units past
  // the last key are read from its block (in bounds; they are masked).  Lane l looks up the
  // block of unit l % 4, and has its scale of K, or of V from lane l % 8 = 4 on.
  const int32_t* trow = a.tables + seq * a.table_stride;
  const int st = tid / CH, sc = tid % CH;
  const uint8_t* kbase = a.k + kvh * a.kv_head;
  const uint8_t* vbase = a.v + kvh * a.kv_head;
  const int unit = lane % kUnits;
  const bool of_k = lane % (2 * kUnits) < kUnits;
  const float* sbase = (of_k ? args.ks : args.vs) + kvh * a.s_head;
  const float f_scale = of_k ? p.qscale * __uint_as_float(static_cast<uint32_t>(127 + (LATE ? p.q_exp : 0)) << 23) : 1.f;
  const uint32_t block_bytes = static_cast<uint32_t>(a.kv_block), token_bytes = static_cast<uint32_t>(a.kv_token);
  const uint32_t s_block = static_cast<uint32_t>(a.s_block);
  const uint32_t page_mask = a.page - 1, last_key = max(wg_keys, 1) - 1, num_blocks = static_cast<uint32_t>(a.num_blocks);
  const int last_chunk = PAD ? a.d / 16 - 1 : CH - 1;
  uint32_t offset[PASSES];  // of this thread's codes in a block, but for the tile's first token in it
#pragma unroll
  for (int i = 0; i < PASSES; ++i) offset[i] = ((i * TPP + st) & page_mask) * token_bytes + min(sc, last_chunk) * 16;
  uint32_t id, v_id;  // the unit's block, of the tile whose K is loaded next and the one whose V is
  u32x4 kreg[PASSES], vreg[PASSES];
  float sreg;
  auto load_id = [&](int tile) __attribute__((always_inline)) {
    id = trow[min(static_cast<uint32_t>(tile * kBN + unit * 16), last_key) >> p.page_shift];
  };
  auto load_codes = [&](u32x4 (&reg)[PASSES], const uint8_t* base, uint32_t blocks, int tile) __attribute__((always_inline)) {
    blocks = blocks < num_blocks ? blocks : 0;
    const uint64_t first = static_cast<uint64_t>((static_cast<uint32_t>(tile) * kBN) & page_mask) * token_bytes;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const uint32_t of_pass = __builtin_amdgcn_readlane(blocks, (i * TPP + wave * (64 / CH)) / 16);
      reg[i] = *reinterpret_cast<const u32x4*>(base + (static_cast<uint64_t>(of_pass) * block_bytes + first) + offset[i]);
    }
  };
  auto load_k = [&](int tile) __attribute__((always_inline)) { load_codes(kreg, kbase, id, tile); };
  auto load_v = [&](int tile) __attribute__((always_inline)) {
    load_codes(vreg, vbase, v_id, tile);
    sreg = sbase[static_cast<uint64_t>(v_id < num_blocks ? v_id : 0) * s_block];
  };
  // Eight codes of one of this thread's rows, of K (the first 2 PASSES chunks) or V, to their place in LDS.
  constexpr int CHUNKS = 4 * PASSES;
  auto store_chunk = [&](int chunk, int k_buf, int v_buf) __attribute__((always_inline)) {
    const int i = chunk % (2 * PASSES) / 2, w = chunk % 2;
    const int at = i * TPP + st;
    uint32_t x = chunk < 2 * PASSES ? kreg[i][2 * w] : vreg[i][2 * w], y = chunk < 2 * PASSES ? kreg[i][2 * w + 1] : vreg[i][2 * w + 1];
    asm volatile("" : "+v"(x), "+v"(y));  // here: not all of them as soon as they have arrived
    if (chunk < 2 * PASSES) {
      const uint2 lo = code_pairs<S>(x), hi = code_pairs<S>(y);
      *reinterpret_cast<u32x4*>(&k_lds[k_buf][at * KROW + sc * 16 + 8 * w]) = u32x4{lo.x, lo.y, hi.x, hi.y};
    } else {
      const uint2 lo = code_pairs<f16>(x), hi = code_pairs<f16>(y);
      *reinterpret_cast<u32x4*>(&v_lds[v_buf][at * VROW + sc * 16 + 8 * w]) = u32x4{lo.x, lo.y, hi.x, hi.y};
    }
  };
  auto store_k = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < CHUNKS / 2; ++i) store_chunk(i, buf, 0);
  };
  auto store_v = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = CHUNKS / 2; i < CHUNKS; ++i) store_chunk(i, 0, buf);
  };
  auto store_scales = [&](int buf) __attribute__((always_inline)) {
    if (tid < 2 * kUnits) f_lds[buf][tid / kUnits][unit] = block_scale(sreg) * f_scale;
  };

  f32x16 acc[DT];
#pragma unroll
  for (int c = 0; c < DT; ++c) acc[c] = f32x16{};
  float m = -INFINITY, lsum = 0.f, e = kNoExponent;
  bool large = false;  // whether some row's maximum is so large that a scaled score's own rounding counts

  // V^T operands: in each 16-lane group lane L addresses key row L / 4 of its four and 4
  // dims; k-step ks, element e of half hf holds key 16 ks + 8 (e / 4) + 4 hf + e % 4.
  const int grp = lane >> 4, gl = lane & 15;
  const int tr_off = (4 * (grp >> 1) + (gl >> 2)) * VROW + 16 * (grp & 1) + 4 * (gl & 3);

  // S^T of half hh of a tile, step c of its products: element r is key key0 + 32 hh + 8 (r / 4) + 4 half +
  // r % 4, of unit 2 hh + r / 8.
  auto scores = [&](int buf, int c, int hh, f32x16& s) __attribute__((always_inline)) {
    const u32x4 ka = *reinterpret_cast<const u32x4*>(&k_lds[buf][(hh * 32 + col) * KROW + 16 * c + 8 * half]);
#pragma unroll
    for (int n = 0; n < NQ; ++n) s = SOps::mma(as_v8<typename SOps::V8>(ka), as_v8<typename SOps::V8>(qw[n][c]), s);
  };
  f32x16 s[2] = {f32x16{}, f32x16{}};
  // Loads of the tiles after those whose codes were just stored.  All of them go out, past the last
  // tile too (the last key again), and in this order: a wait for one is a wait for all before it.
  auto load_next = [&](int j) __attribute__((always_inline)) {
    load_v(j + 2);
    load_k(j + 3);
    v_id = id;
  };
  // Tile j, whose scores s holds.  Its weights and the codes of the tiles after it are worked out
  // between the products: of its own values, and of the next tile's scores, which take the
  // registers of its own as they are used up.
  auto step = [&](int j) __attribute__((always_inline)) {
    const int buf = j & 1;
    load_id(j + 3);
    {
      f32x4 f = *reinterpret_cast<const f32x4*>(f_lds[buf][0]);
      f32x4 vs = *reinterpret_cast<const f32x4*>(f_lds[buf][1]);
      const int key0 = j * kBN;
      // Scores are scaled ahead where some are masked (a scale of 0 or NaN times -inf would not be).
      const bool masked = uniform(key0 + kBN - 1 > wave_first || wave_row0 + 31 >= rows);
      if (masked) {
        const int lim = limit - key0 - 4 * half;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[hh][r] = rounded_product(s[hh][r], f[2 * hh + r / 8]);
            if (hh * 32 + (r / 4) * 8 + r % 4 > lim) s[hh][r] = -INFINITY;
          }
#pragma unroll
        for (int u = 0; u < kUnits; ++u)  // a unit that the row sees nothing of counts 0, whatever its scale
          if (16 * u > limit - key0) vs[u] = 0.f;
        f = f32x4{1.f, 1.f, 1.f, 1.f};
      }
      float x[kUnits];  // the largest score of a unit, of this lane's eight
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        x[u] = s[u / 2][u % 2 * 8];
#pragma unroll
        for (int r = 1; r < 8; ++r) x[u] = fmaxf(x[u], s[u / 2][u % 2 * 8 + r]);
        x[u] *= f[u];
      }
      const float top = max_across_halves(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
      const float highest = scale_exponent(fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3])));
      // No weight is above 2^(top - m + highest - e); it may be 2^15.
      if (__builtin_amdgcn_ballot_w64(top > m + kRescale || top - m + highest > e + kMostExponent) != 0) {
        const float mn = fmaxf(m, ceilf(top));
        const float down = mn - m;  // +inf at the first key, NaN before it
        float en = e - down;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) en = fmaxf(en, ceilf(max_across_halves(x[u]) - mn) + scale_exponent(vs[u]) - kUsualExponent);
        const bool none = mn == -INFINITY;
        const float corr = none ? 0.f : fast_exp2(e - down - en);
        lsum = none ? 0.f : lsum * fast_exp2(-down);
        m = mn;
        e = none ? kNoExponent : en;
        large = __builtin_amdgcn_ballot_w64(fabsf(m) > 4096.f && m != -INFINITY) != 0;
#pragma unroll
        for (int c = 0; c < DT; ++c)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[c][r] *= corr;
      }
      // m is a rounded score's bound.  One that is left unrounded may pass it by half a step of its own:
      // nothing for small ones, 2^7 at 2^31, whose weight would be infinite.
      if (large) {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[hh][r] = rounded_product(s[hh][r], f[2 * hh + r / 8]);
        f = f32x4{1.f, 1.f, 1.f, 1.f};
      }
      const float mb = m == -INFINITY ? 0.f : m;  // only -inf scores so far: they weigh 0
      u32x4 pb[kUnits][NP];
      float g[kUnits];
#pragma unroll
      for (int u = 0; u < kUnits; ++u) g[u] = weight_scale(vs[u], e);
      // Two weights, in parts: elements 2 i and 2 i + 1 of unit u.
      auto pair = [&](int k) __attribute__((always_inline)) {
        const int u = k / 4, i = k % 4, r = u % 2 * 8 + 2 * i;
        float y = fast_exp2(fmaf(s[u / 2][r], f[u], -mb)), z = fast_exp2(fmaf(s[u / 2][r + 1], f[u], -mb));
        lsum += y + z;
        asm volatile("" : "+v"(lsum));  // here: left to the end, the sums would keep 32 probabilities
        y *= g[u], z *= g[u];
        if constexpr (NP > 1) asm("" : "+v"(y), "+v"(z));  // the parts are of one product, rounded to fp32
#pragma unroll
        for (int n = 0; n < NP; ++n) {
          pb[u][n][i] = Ops::pack2(y, z);
          if (n + 1 < NP) y -= f16_value(pb[u][n][i]), z -= f16_value(pb[u][n][i] >> 16);
        }
      };
      // The products, in this order: values of unit 0, scores of half 0, values of units 1 and 2, scores of
      // half 1, values of unit 3.  `values` of slot i: whether, of which unit; the step or output tile.
      constexpr int SLOTS = 4 * DT + 2 * KS;
      auto unit_of = [](int i) { return i < DT ? 0 : i < DT + KS ? -1 : i < 2 * DT + KS ? 1 : i < 3 * DT + KS ? 2 : i < 3 * DT + 2 * KS ? -2 : 3; };
      auto part_of = [](int i) { return i < DT ? i : i < DT + KS ? i - DT : i < 3 * DT + KS ? (i - KS) % DT : i < 3 * DT + 2 * KS ? i - 3 * DT - KS : i - 3 * DT - 2 * KS; };
      auto operand = [&](int i) __attribute__((always_inline)) {
        const int u = unit_of(i), c = part_of(i);
        if (u < 0) return *reinterpret_cast<const u32x4*>(&k_lds[buf ^ 1][((-u - 1) * 32 + col) * KROW + 16 * c + 8 * half]);
        const uint16_t* vlo = &v_lds[buf][tr_off + u * 16 * VROW + c * 32];
        const u32x2 lo = lds_read_tr(vlo), hi = lds_read_tr(vlo + 8 * VROW);
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
      };
      auto product = [&](int i, const u32x4& x) __attribute__((always_inline)) {
        const int u = unit_of(i), c = part_of(i);
        if (u < 0) {
          const int hh = -u - 1;
          if (c == 0) s[hh] = f32x16{};
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[hh] = SOps::mma(as_v8<typename SOps::V8>(x), as_v8<typename SOps::V8>(qw[n][c]), s[hh]);
        } else {
#pragma unroll
          for (int n = 0; n < NP; ++n) acc[c] = Ops::mma(as_v8<f16x8>(x), as_v8<f16x8>(pb[u][n]), acc[c]);
        }
      };
      constexpr int AHEAD = 4;
      u32x4 ring[AHEAD];
      unrolled<AHEAD>([&](auto at) __attribute__((always_inline)) { ring[at] = operand(at); });
      unrolled<4>([&](auto k) __attribute__((always_inline)) { pair(k); });
      // A wave at its products goes before the others of its SIMD: two in the same phase would wait for
      // the matrix cores, and then for the vector ones, in turn (373 -> 364 us).
      __builtin_amdgcn_s_setprio(1);
      __builtin_amdgcn_sched_barrier(0);
      unrolled<SLOTS>([&](auto at) __attribute__((always_inline)) {
        constexpr int i = decltype(at)::value;
        product(i, ring[i % AHEAD]);
        if constexpr (i + AHEAD < SLOTS) ring[i % AHEAD] = operand(i + AHEAD);
        unrolled<12>([&](auto of) __attribute__((always_inline)) {
          constexpr int k = 4 + decltype(of)::value;
          if constexpr (i == (k < 8 ? (k - 4) * DT / 4 : k < 14 ? DT + (k - 8) * (KS + DT) / 6 : 2 * DT + KS + (k - 14) * DT / 2)) pair(k);
        });
        unrolled<CHUNKS>([&](auto of) __attribute__((always_inline)) {
          constexpr int k = decltype(of)::value;
          if constexpr (i == 3 * DT + KS + k * (KS + DT) / CHUNKS) store_chunk(k, buf, buf ^ 1);
        });
        __builtin_amdgcn_sched_barrier(0);
      });
    }
    store_scales(buf ^ 1);
    load_next(j);
    __builtin_amdgcn_s_setprio(0);
    __syncthreads();
  };

  if (ntiles > first_tile) {
    // What the first products wait for is on its way at once: the blocks of three tiles; then q and the
    // codes of two (each in turn: 6.9 us to the first step, so 6.2).
    load_id(first_tile);
    v_id = id;
    load_id(first_tile + 1);
    const uint32_t next_id = id;
    load_id(first_tile + 2);
    constexpr int N = Packet<T>::N;
    const T* const qrow = static_cast<const T*>(a.q) + (row0 + at_row) * a.q_row + h * a.q_head;
    u32x4 raw[KS][8 / N];
    if (p.q_vec) {
#pragma unroll
      for (int c = 0; c < KS; ++c)
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) raw[c][i] = *reinterpret_cast<const u32x4*>(qrow + 16 * min(c, last_chunk) + 8 * half + i * N);
    } else {
#pragma unroll
      for (int c = 0; c < KS; ++c)
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) {
          T x[N];
#pragma unroll
          for (int e = 0; e < N; ++e) x[e] = qrow[(16 * min(c, last_chunk) + 8 * half + i * N + e) * a.q_dim];
          raw[c][i] = __builtin_bit_cast(u32x4, x);
        }
    }
    u32x4 knext[PASSES];
    load_codes(kreg, kbase, v_id, first_tile);
    load_v(first_tile);
    load_codes(knext, kbase, next_id, first_tile + 1);
    const float power = __uint_as_float(static_cast<uint32_t>(127 + (LATE ? 0 : p.q_exp)) << 23 | p.q_sign);
#pragma unroll
    for (int c = 0; c < KS; ++c) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8 / N; ++i) Packet<T>::unpack(raw[c][i], &x[i * N]);
#pragma unroll
      for (int i = 0; i < 8; ++i)  // infinities as NaN, which no other row's maximum takes up
        x[i] = (__float_as_uint(x[i]) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fc00000u) : x[i] * power;
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if constexpr (NQ > 1) {  // the top 16 bits: the rest is exact, and the last part holds all of it
            const uint32_t lo = __float_as_uint(x[2 * w]), hi = __float_as_uint(x[2 * w + 1]);
            qw[n][c][w] = c > last_chunk ? 0u : lo >> 16 | (hi & 0xffff0000u);
            x[2 * w] -= __uint_as_float(lo & 0xffff0000u);
            x[2 * w + 1] -= __uint_as_float(hi & 0xffff0000u);
          } else {
            qw[n][c][w] = c > last_chunk ? 0u : SOps::pack2(x[2 * w], x[2 * w + 1]);
          }
        }
    }
    store_k(first_tile & 1);
    store_v(first_tile & 1);
    store_scales(first_tile & 1);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) kreg[i] = knext[i];
    store_k(first_tile & 1 ^ 1);
    v_id = next_id;
    load_v(first_tile + 1);
    load_k(first_tile + 2);
    v_id = id;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < KS; ++c)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) scores(first_tile & 1, c, hh, s[hh]);
    __syncthreads();
    // Tiles that some row of the wave sees, and those that it only helps to stage.
    const int seen = wave_live && wave_last >= 0 ? min(ntiles, wave_last / kBN + 1) : first_tile;
    int j = first_tile;
    for (; j < seen; ++j) step(j);
    for (; j < ntiles; ++j) {
      load_id(j + 3);
      store_k(j & 1);
      store_v(j & 1 ^ 1);
      store_scales(j & 1 ^ 1);
      load_next(j);
      __syncthreads();
    }
  }

  lsum += __shfl_xor(lsum, 32, 64);
  if (!row_valid) return;
  if (uniform(it.segs) > 1) {
    const int64_t slot = (static_cast<int64_t>(it.slot0) + static_cast<int64_t>(it.seg) * nq + at_row) * a.hq + h;
    float* dst = p.part_acc + slot * D + 4 * half;
#pragma unroll
    for (int c = 0; c < DT; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(dst + 32 * c + 8 * g) = f32x4{acc[c][4 * g], acc[c][4 * g + 1], acc[c][4 * g + 2], acc[c][4 * g + 3]};
    if (half == 0) args.part_state[slot] = PartState{m, lsum, e, 0.f};
    return;
  }
  // A row that sees no key is zeros.
  const float inv = 1.f / lsum;
  const int exponent = static_cast<int>(e);
  T* orow = static_cast<T*>(a.out) + (row0 + at_row) * a.o_row + h * a.o_head;
#pragma unroll
  for (int c = 0; c < DT; ++c)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * c + 8 * g + 4 * half;
      if (2 * c + g / 2 > last_chunk) continue;
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = limit < 0 ? 0.f : ldexpf(acc[c][4 * g + i] * inv, exponent);
      store4(orow, d, x, a.o_dim, p.out_vec);
    }
}

// Joins the segments of cut sequences: a workgroup takes 1024 neighbouring elements of a row
// at a time, 4 a thread, and adds the segments in order, BATCH of them on their way at once.  The
// grid is one round at most and walks the rows of cut sequences only.  (The eight chunks above: 12 us.)
template <typename T, int D>
__global__ __launch_bounds__(256) void prefill_i8_merge_kernel(PrefillI8Args args, int parts) {
  constexpr int BATCH = 4;
  const Prefill8Args& p = args.p;
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
    const int tile_end = (i * p.group + h % p.group) / kBM * kBM + kBM;
    const int keys = max(len - nq + min((tile_end - 1) / p.group + 1, nq), 0);
    const int live = min(segs, max(1, (keys + seg_keys - 1) / seg_keys));
    const int64_t step = static_cast<int64_t>(nq) * a.hq;  // slots from one segment to the next
    const int64_t base = (static_cast<int64_t>(slot0) + i) * a.hq + h;
    float m = -INFINITY, sum = 0.f, exponent = kNoExponent;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int g0 = 0; g0 < live; g0 += BATCH) {
      PartState part[BATCH];
      f32x4 x[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int64_t slot = base + min(g0 + u, live - 1) * step;
        part[u] = args.part_state[slot];
        x[u] = *reinterpret_cast<const f32x4*>(p.part_acc + slot * D + d);
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < BATCH; ++u) top = fmaxf(top, part[u].m);
      const float off = top == -INFINITY ? 0.f : top;
      const float before = exponent + (m - off);
      exponent = fmaxf(before, kNoExponent);
#pragma unroll
      for (int u = 0; u < BATCH; ++u) exponent = fmaxf(exponent, part[u].e + (part[u].m - off));
      sum *= fast_exp2(m - off);
      acc *= fast_exp2(before - exponent);
      m = top;
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const bool in = g0 + u < live;
        const float w = fast_exp2(part[u].e + (part[u].m - off) - exponent);
        sum = in ? fmaf(part[u].l, fast_exp2(part[u].m - off), sum) : sum;
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = in ? fmaf(x[u][k], w, acc[k]) : acc[k];
      }
    }
    const bool blind = len - nq + i < 0;  // a row that sees no key
    const float inv = 1.f / sum;
    float y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = blind ? 0.f : ldexpf(acc[k] * inv, static_cast<int>(exponent));
    if (d < a.d) store4(static_cast<T*>(a.out) + row * a.o_row + h * a.o_head, d, y, a.o_dim, p.out_vec);
  }
}

template <typename T, int D>
void launch_size(const PrefillI8Args& args, unsigned grid, hipStream_t stream) {
  const Attn8Args& a = args.p.a;
  if (a.d == D) hipLaunchKernelGGL((prefill_i8_kernel<T, D, false>), dim3(grid), dim3(256), 0, stream, args);
  else hipLaunchKernelGGL((prefill_i8_kernel<T, D, true>), dim3(grid), dim3(256), 0, stream, args);
  if (!args.p.slots) return;
  const int parts = static_cast<int>((static_cast<int64_t>(a.hq) * D + 1023) / 1024);
  const dim3 merge(static_cast<unsigned>(std::min<int64_t>(a.rows * parts, kMergeRound)));
  hipLaunchKernelGGL((prefill_i8_merge_kernel<T, D>), merge, dim3(256), 0, stream, args, parts);
}

// The kernel's head size.
int64_t padded_dims(int64_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

template <typename T>
void launch_type(const PrefillI8Args& args, unsigned grid, hipStream_t stream) {
  switch (padded_dims(args.p.a.d)) {
    case 64: launch_size<T, 64>(args, grid, stream); break;
    case 128: launch_size<T, 128>(args, grid, stream); break;
    default: launch_size<T, 256>(args, grid, stream); break;
  }
}

}  // namespace

bool prefill_i8_shape(int64_t d, int64_t page) {
  return d > 0 && d <= 256 && d % 16 == 0 && page >= 16 && (page & (page - 1)) == 0;
}

int64_t prefill_i8_workspace(int64_t rows, int64_t num_seqs, int64_t max_len, int64_t hq, int64_t d) {
  const int64_t slots = partial_slots(rows, num_seqs, max_len, hq);
  return slots ? slots * hq * (padded_dims(d) * 4 + static_cast<int64_t>(sizeof(PartState))) + kPlanSeqs * static_cast<int64_t>(sizeof(SeqPlan)) : 0;
}

int launch_prefill_i8(const AttnI8Args& s, int dtype, void* ws, hipStream_t stream, const char* name) {
  const Attn8Args& a = s.a;
  PrefillI8Args args{};
  Prefill8Args& p = args.p;
  p.a = a;
  args.ks = s.ks, args.vs = s.vs;
  const int64_t slots = ws ? partial_slots(a.rows, a.num_seqs, a.max_len, a.hq) : 0;
  if (slots > kMaxBlocks) return fail(RLT_EUNSUPPORTED, "%s: too many rows", name);  // 64 sequences' stay inside 31 bits
  p.slots = static_cast<int>(slots);
  p.group = a.hq / a.hkv;
  p.round = a.d > 128 || (dtype == RLT_FLOAT32 && a.d > 64) ? kRound / 2 : kRound;
  if (slots) {
    p.part_acc = static_cast<float*>(ws);
    args.part_state = reinterpret_cast<PartState*>(p.part_acc + slots * a.hq * padded_dims(a.d));
    p.plan = reinterpret_cast<SeqPlan*>(args.part_state + slots * a.hq);
  }
  fill_prefill8(&p, dtype);
  const int64_t tiles = prefill8_tiles(p, p.round);
  // (So that rows of a tile, a row and head each, stay inside 31 bits as well.)
  if (tiles * a.hkv > kMaxBlocks) return fail(RLT_EUNSUPPORTED, "%s: too many rows", name);
  const unsigned grid = static_cast<unsigned>(tiles * a.hkv);
  switch (dtype) {
    case RLT_BFLOAT16: launch_type<bf16>(args, grid, stream); break;
    case RLT_FLOAT16: launch_type<f16>(args, grid, stream); break;
    default: launch_type<float>(args, grid, stream); break;
  }
  return check_launch(name);
}

}  // namespace rlt
