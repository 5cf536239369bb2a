// Packed chunked prefill over the block-scaled 8-bit KV cache, bottom-right causal, on the
// matrix cores (head_dim 64 / 128, pages of a power of two of at least 16 tokens; int8.hpp has
// the softmax, prefill_plan.hpp the launch's plan).
//
// A workgroup of 4 waves takes 128 query rows of one (sequence, query head) over a
// segment of its keys, a wave 32 rows, 64 keys a tile, four units of 16 keys that have one
// scale of K and one of V each:
// - S^T = K Q^T on the 16-bit MFMA of q's type (32x32x16; an fp32 q in three bf16 parts).  Codes
//   become bf16 or fp16, exactly, once a workgroup, on their way into LDS; their unit's scale
//   multiplies the sums, in the instruction that takes the running maximum off.
// - O^T += V^T W^T on the fp16 MFMA, codes as fp16 likewise; V^T comes from transposing LDS
//   reads, W, the probabilities times their unit's V scale, from the registers S^T left it
//   in: in one part, 11 bits, for bf16 and fp16, in two for fp32.
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

// Parts of q and of the weights, and the type of the scores' operands.
template <typename T> struct Parts;
template <> struct Parts<bf16> { static constexpr int Q = 1, P = 1; using S = bf16; };
template <> struct Parts<f16> { static constexpr int Q = 1, P = 1; using S = f16; };
template <> struct Parts<float> { static constexpr int Q = 3, P = 2; using S = bf16; };

template <typename T, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 ? 1 : 2))) void prefill_i8_kernel(PrefillI8Args args) {
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
  if (!find_item(p, &it)) return;
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
  // An fp16 q goes in as it is, the others times 2^q_exp.
  constexpr bool LATE = std::is_same_v<S, f16>;
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
            qw[n][c][w] = SOps::pack2(x[2 * w], x[2 * w + 1]);
          }
        }
    }
  }

  // Staging: thread (token, chunk), PASSES tokens TPP apart.  Tokens past the last key
  // re-read it (in bounds; they are masked).  Thread u (kUnits + u) has unit u's scale of K (V).
  const int32_t* trow = a.tables + seq * a.table_stride;
  const int st = tid / CH, sc = tid % CH;
  const uint8_t* kbase = a.k + kvh * a.kv_head + sc * 16;
  const uint8_t* vbase = a.v + kvh * a.kv_head + sc * 16;
  const float* sbase = (tid < kUnits ? args.ks : args.vs) + kvh * a.s_head;
  const float f_scale = tid < kUnits ? p.qscale * __uint_as_float(static_cast<uint32_t>(127 + (LATE ? p.q_exp : 0)) << 23) : 1.f;
  const uint32_t block_bytes = static_cast<uint32_t>(a.kv_block), token_bytes = static_cast<uint32_t>(a.kv_token);
  const uint32_t s_block = static_cast<uint32_t>(a.s_block);
  const uint32_t page_mask = a.page - 1, last_key = max(wg_keys, 1) - 1, num_blocks = static_cast<uint32_t>(a.num_blocks);
  uint32_t ids[PASSES], unit_id = 0;  // of the tile loaded next
  u32x4 kreg[PASSES], vreg[PASSES];
  float sreg = 0.f;
  auto token = [&](int tile, int t) { return min(static_cast<uint32_t>(tile * kBN + t), last_key); };
  auto load_ids = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) ids[i] = trow[token(tile, i * TPP + st) >> p.page_shift];
    if (tid < 2 * kUnits) unit_id = trow[token(tile, tid % kUnits * 16) >> p.page_shift];
  };
  auto load_tile = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const uint32_t slot = token(tile, i * TPP + st) & page_mask;
      const uint64_t id = ids[i] < num_blocks ? ids[i] : 0;
      const uint64_t at = id * block_bytes + __umul24(slot, token_bytes);
      kreg[i] = *reinterpret_cast<const u32x4*>(kbase + at);
      vreg[i] = *reinterpret_cast<const u32x4*>(vbase + at);
    }
    if (tid < 2 * kUnits) sreg = sbase[static_cast<uint64_t>(unit_id < num_blocks ? unit_id : 0) * s_block];
  };
  auto store_codes = [&](auto type, const u32x4& codes, uint16_t* dst) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint2 lo = code_pairs<decltype(type)>(codes[2 * i]), hi = code_pairs<decltype(type)>(codes[2 * i + 1]);
      *reinterpret_cast<u32x4*>(dst + 8 * i) = u32x4{lo.x, lo.y, hi.x, hi.y};
    }
  };
  auto store_tile = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      store_codes(S{}, kreg[i], &k_lds[buf][(i * TPP + st) * KROW + sc * 16]);
      store_codes(f16{}, vreg[i], &v_lds[buf][(i * TPP + st) * VROW + sc * 16]);
    }
    if (tid < 2 * kUnits) f_lds[buf][tid / kUnits][tid % kUnits] = block_scale(sreg) * f_scale;
  };

  f32x16 acc[DT];
#pragma unroll
  for (int c = 0; c < DT; ++c) acc[c] = f32x16{};
  float m = -INFINITY, lsum = 0.f, e = kNoExponent;

  // V^T operands: in each 16-lane group lane L addresses key row L / 4 of its four and 4
  // dims; k-step ks, element e of half hf holds key 16 ks + 8 (e / 4) + 4 hf + e % 4.
  const int grp = lane >> 4, gl = lane & 15;
  const int tr_off = (4 * (grp >> 1) + (gl >> 2)) * VROW + 16 * (grp & 1) + 4 * (gl & 3);

  auto step = [&](int j) __attribute__((always_inline)) {
    const int buf = j & 1;
    if (j + 1 < ntiles) {
      load_tile(j + 1);
      load_ids(j + 2);
    }
    if (wave_live && j * kBN <= wave_last) {
      // S^T: element r of half hh is key key0 + 32 hh + 8 (r / 4) + 4 half + r % 4, of unit 2 hh + r / 8.
      f32x16 s[2] = {f32x16{}, f32x16{}};
#pragma unroll
      for (int c = 0; c < KS; ++c)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const u32x4 ka = *reinterpret_cast<const u32x4*>(&k_lds[buf][(hh * 32 + col) * KROW + 16 * c + 8 * half]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[hh] = SOps::mma(as_v8<typename SOps::V8>(ka), as_v8<typename SOps::V8>(qw[n][c]), s[hh]);
        }
      f32x4 f = *reinterpret_cast<const f32x4*>(f_lds[buf][0]);
      const f32x4 vs = *reinterpret_cast<const f32x4*>(f_lds[buf][1]);
      const int key0 = j * kBN;
      // Scores are scaled ahead where some are masked (a scale of 0 or NaN times -inf would not
      // be) and where they are so large that the scaled maximum's own rounding counts.
      const bool masked = uniform(key0 + kBN - 1 > prefix + wave_row0 || wave_row0 + 31 >= nq);
      if (masked || __builtin_amdgcn_ballot_w64(fabsf(m) > 4096.f && m != -INFINITY) != 0) {
        const int lim = limit - key0 - 4 * half;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[hh][r] = rounded_product(s[hh][r], f[2 * hh + r / 8]);
            if (hh * 32 + (r / 4) * 8 + r % 4 > lim) s[hh][r] = -INFINITY;
          }
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
      const bool rescale = __builtin_amdgcn_ballot_w64(top > m + kRescale || top - m + highest > e + kMostExponent) != 0;
      float corr = 1.f;
      if (rescale) {
        const float mn = fmaxf(m, ceilf(top));
        const float down = mn - m;  // +inf at the first key, NaN before it
        float en = e - down;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) en = fmaxf(en, ceilf(max_across_halves(x[u]) - mn) + scale_exponent(vs[u]) - kUsualExponent);
        const bool none = mn == -INFINITY;
        corr = none ? 0.f : fast_exp2(e - down - en);
        lsum = none ? 0.f : lsum * fast_exp2(-down);
        m = mn;
        e = none ? kNoExponent : en;
      }
      const float mb = m == -INFINITY ? 0.f : m;  // only -inf scores so far: they weigh 0
      // One site for all products: accumulators changed on two paths get two register sets.
      if (rescale) {
#pragma unroll
        for (int c = 0; c < DT; ++c)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[c][r] *= corr;
      }
#pragma unroll
      for (int ks = 0; ks < kUnits; ++ks) {
        // The weights of unit ks, in parts; one that this lane sees nothing of counts 0, whatever its scale.
        const float g = x[ks] == -INFINITY ? 0.f : weight_scale(vs[ks], e);
        u32x4 pb[NP];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = (ks % 2) * 8 + 2 * i;
          float y = fast_exp2(fmaf(s[ks / 2][r], f[ks], -mb)), z = fast_exp2(fmaf(s[ks / 2][r + 1], f[ks], -mb));
          lsum += y + z;
          y *= g, z *= g;
          if constexpr (NP > 1) asm("" : "+v"(y), "+v"(z));  // the parts are of one product, rounded to fp32
#pragma unroll
          for (int n = 0; n < NP; ++n) {
            pb[n][i] = Ops::pack2(y, z);
            if (n + 1 < NP) y -= f16_value(pb[n][i]), z -= f16_value(pb[n][i] >> 16);
          }
        }
#pragma unroll
        for (int c = 0; c < DT; ++c) {
          const uint16_t* vlo = &v_lds[buf][tr_off + ks * 16 * VROW + c * 32];
          const u32x2 lo = lds_read_tr(vlo), hi = lds_read_tr(vlo + 8 * VROW);
          const u32x4 va = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
          for (int n = 0; n < NP; ++n) acc[c] = Ops::mma(as_v8<f16x8>(va), as_v8<f16x8>(pb[n]), acc[c]);
        }
      }
    }
    if (j + 1 < ntiles) store_tile(buf ^ 1);
    __syncthreads();
  };

  if (ntiles > first_tile) {
    load_ids(first_tile);
    load_tile(first_tile);
    load_ids(first_tile + 1);
    store_tile(first_tile & 1);
    __syncthreads();
  }
  for (int j = first_tile; j < ntiles; ++j) step(j);

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
    if (half == 0) args.part_state[slot] = PartState{m, lsum, e, 0.f};
    return;
  }
  // A row that sees no key is zeros.
  const float inv = 1.f / lsum;
  const int exponent = static_cast<int>(e);
  T* orow = static_cast<T*>(a.out) + (row0 + my_row) * a.o_row + h * a.o_head;
#pragma unroll
  for (int c = 0; c < DT; ++c)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * c + 8 * g + 4 * half;
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = limit < 0 ? 0.f : ldexpf(acc[c][4 * g + i] * inv, exponent);
      store4(orow, d, x, a.o_dim, p.out_vec);
    }
}

// Joins the segments of cut sequences: a workgroup takes 1024 neighbouring elements of a row
// at a time, 4 a thread, and adds the segments in order, BATCH of them on their way at once.  The
// grid is one round at most and walks the rows of cut sequences only.
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
    const int keys = max(len - nq + min(i / kBM * kBM + kBM, nq), 0);
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
    store4(static_cast<T*>(a.out) + row * a.o_row + h * a.o_head, d, y, a.o_dim, p.out_vec);
  }
}

template <typename T, int D>
void launch_size(const PrefillI8Args& args, unsigned grid, hipStream_t stream) {
  const Attn8Args& a = args.p.a;
  hipLaunchKernelGGL((prefill_i8_kernel<T, D>), dim3(grid), dim3(256), 0, stream, args);
  if (!args.p.slots) return;
  const int parts = static_cast<int>((static_cast<int64_t>(a.hq) * D + 1023) / 1024);
  const dim3 merge(static_cast<unsigned>(std::min<int64_t>(a.rows * parts, kMergeRound)));
  hipLaunchKernelGGL((prefill_i8_merge_kernel<T, D>), merge, dim3(256), 0, stream, args, parts);
}

template <typename T>
void launch_type(const PrefillI8Args& args, unsigned grid, hipStream_t stream) {
  if (args.p.a.d == 64) launch_size<T, 64>(args, grid, stream);
  else launch_size<T, 128>(args, grid, stream);
}

}  // namespace

int64_t prefill_i8_workspace(int64_t rows, int64_t num_seqs, int64_t max_len, int64_t hq, int64_t d) {
  const int64_t slots = partial_slots(rows, num_seqs, max_len, hq);
  return slots ? slots * hq * (d * 4 + static_cast<int64_t>(sizeof(PartState))) + kPlanSeqs * static_cast<int64_t>(sizeof(SeqPlan)) : 0;
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
  p.round = dtype == RLT_FLOAT32 && a.d == 128 ? kRound / 2 : kRound;
  if (slots) {
    p.part_acc = static_cast<float*>(ws);
    args.part_state = reinterpret_cast<PartState*>(p.part_acc + slots * a.hq * a.d);
    p.plan = reinterpret_cast<SeqPlan*>(args.part_state + slots * a.hq);
  }
  fill_prefill8(&p, dtype);
  const int64_t tiles = prefill8_tiles(p);
  if (tiles * a.hq > kMaxBlocks) return fail(RLT_EUNSUPPORTED, "%s: too many rows", name);
  const unsigned grid = static_cast<unsigned>(tiles * a.hq);
  switch (dtype) {
    case RLT_BFLOAT16: launch_type<bf16>(args, grid, stream); break;
    case RLT_FLOAT16: launch_type<f16>(args, grid, stream); break;
    default: launch_type<float>(args, grid, stream); break;
  }
  return check_launch(name);
}

}  // namespace rlt
