// What prefill over an 8-bit cache does whatever the form of its scales: the launch's plan.
//
// Key segments.  Items of one launch differ by two orders of magnitude (a new prompt's
// 128 rows beside a chunk at the end of 16000 keys), and a launch of few rows has too
// few of them.  So the keys of long sequences are cut into segments of about the
// launch's work over kTargetItems, and a merge kernel joins them; the items go out
// longest first, the heads of a sequence over the XCDs so that its query tiles share an
// L2.  Every wave works the plan out for itself from the lengths.
#pragma once

#include <cmath>
#include <limits>
#include <type_traits>

#include "mfma.hpp"
#include "prefill_fp8.hpp"

namespace rlt {

constexpr int kBM = 128;  // query rows a workgroup
constexpr int kBN = 64;   // keys a tile
constexpr float kRescale = 8.f;
constexpr int kMaxQExp = 24;
constexpr int kRound = 512;  // workgroups that run at once: two a CU (fp32 at head_dim 128: one)
constexpr int kTargetItems = kRound * 3 / 2;
// Shorter segments are not worth an item (about 9 us of plan, first loads and merge beside
// 1.5 a tile).  Measured, us, in 4 / 3 / 2 / 1: one chunk of 40 rows over 340 keys 14.8 / 14.9 /
// 13.2 / 12.5, of 128 over 4128 30.3 / 28.0 / 28.1 / 28.0, two of 20-100 over 200-1200 17.9 /
// 17.8 / 17.2 / 21.0.
constexpr int kMinSegTiles = 2;
constexpr int64_t kMergeRound = 2048;  // workgroups of the merge that run at once
constexpr int kPlanSeqs = 64;  // sequences ranked and cut: one a lane

// One sequence a lane: its rows, keys and cut.
struct SeqPlan {
  int row0, nq, len;
  int tiles;      // query tiles
  int segs;       // key segments
  int seg_tiles;  // key tiles of a segment
  int slot0;      // first partial row of a cut sequence: row i of segment g is slot0 + g * nq + i
};
struct Prefill8Args {
  Attn8Args a;
  int page_shift;
  // |softmax scale| * log2(e) = qscale * 2^q_exp, q_exp in [-kMaxQExp, 0]: the power of two goes
  // into q, so that a score overflows only where the scaled one does.
  float qscale;
  int q_exp;
  uint32_t q_sign;  // 0x80000000 negates q (a negative scale), else 0
  // Key segments: partials of cut sequences, row slots x heads (null: none is cut).
  float* part_acc;    // [slots][hq][D]
  float2* part_ml;    // [slots][hq], max in log2 units and sum
  SeqPlan* plan;      // [kPlanSeqs], for the merge kernel
  int slots;
  int round;  // workgroups that run at once
  int group;  // query heads whose rows stand together in a query tile: row i of head g of them is its row i * group + g
  int out_vec;  // 4 elements of an out row can be stored at once
  int q_vec;    // q rows are 16-byte aligned, dims together
};

// Rows [row0, row0 + nq) of sequence s, inside [0, rows) whatever cu holds.
__device__ __forceinline__ void seq_rows(const Attn8Args& a, int s, int& row0, int& nq) {
  const int rows = static_cast<int>(a.rows);
  row0 = min(max(a.cu[s], 0), rows);
  nq = min(max(a.cu[s + 1], row0), rows) - row0;
}

// Inclusive scans over the wave's lanes by DPP (a shuffle each would cost 1.3 us an item):
// row_shr 1, 2, 4, 8 within 16 lanes, then the rows' last lanes into the rows after.
template <typename X, typename F>
__device__ __forceinline__ X wave_scan(X x, F join) {
  auto take = [&](auto ctrl, auto rows) {
    return __builtin_bit_cast(X, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value,
                                                             decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  x = join(x, take(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{}));
  x = join(x, take(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{}));
  x = join(x, take(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{}));
  x = join(x, take(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{}));
  x = join(x, take(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{}));
  x = join(x, take(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{}));
  return x;
}
__device__ __forceinline__ int scan_sum(int x) { return wave_scan(x, [](int a, int b) { return a + b; }); }

// TAILS: the sequences of launches of many items are cut into whole segments and a shorter last one,
// not into equal ones; *tails: whether they are.
template <bool TAILS>
__device__ __forceinline__ SeqPlan plan_of(const Prefill8Args& p, int lane, bool* tails) {
  SeqPlan s{};
  *tails = false;
  if (lane < p.a.num_seqs) {
    seq_rows(p.a, lane, s.row0, s.nq);
    s.len = sequence_length(p.a, lane);
  }
  s.tiles = (s.nq * p.group + kBM - 1) / kBM;
  const int heads = p.a.hq / p.group;
  const int keys = (s.len + kBN - 1) / kBN;
  s.segs = 1;
  s.seg_tiles = keys;
  if (p.part_acc) {
    // In (query tile, key tile) pairs.  The sum's rounding is inside the slack of
    // partial_slots() and of the grid.
    const float work = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_scan(
        static_cast<float>(s.tiles) * static_cast<float>(keys), [](float a, float b) { return a + b; })), 63)) * heads;
    const int longest = __builtin_amdgcn_readlane(wave_scan(s.tiles ? keys : 0, [](int a, int b) { return max(a, b); }), 63);
    // Cut where the longest item would outlast the others by half: 24 chunks of 100-170 rows
    // over up to 1000 keys (768 items of up to 18 tiles) take 55 us whole, 69 cut.
    if (longest * (2.f * p.round) > 3.f * work) {
      // Few items: cut into one round of workgroups.  Many, of different lengths: into half as
      // many again, so that the short ones fill the gaps (eight chunks 402 us in 512, 353
      // in 768, 369 in 1024; one chunk of 64 items 96, 119, 109).
      const bool few = __builtin_amdgcn_readlane(scan_sum(s.tiles), 63) * heads <= p.round / 2;
      // Or, with tails, into a round of whole segments, longest first, and the shorter last ones of
      // their sequences, which fill the gaps (four chunks of 740-983 rows over up to 4400 keys, 16 + 4
      // heads, 119.1 us in equal ones, 113.8).
      *tails = TAILS && !few;
      int target = max(kMinSegTiles, static_cast<int>(fminf(ceilf(work / (few || *tails ? p.round : p.round * 3 / 2)), 1e9f)));
      for (int i = 0; few && i < 4; ++i) {  // as rounding up makes more items, towards the round
        const int items = __builtin_amdgcn_readlane(scan_sum(s.tiles * max(1, (keys + target - 1) / target)), 63) * heads;
        // Segments of two tiles pay for one workgroup a CU (over the block-scaled cache, in 2 / 3, us: six of
        // 20-67 rows over up to 1526, 16 + 8 heads, 27.3 / 22.8, one of 306 over 757, 16 heads x 64, 21.5 /
        // 19.2, three of 6-20 over up to 573, fewer items, 14.3 / 15.4).
        if (items <= (TAILS && target < 3 ? min(p.round, kRound / 2) : p.round)) break;
        target = max(target + 1, static_cast<int>(static_cast<float>(target) * items / p.round));
      }
      s.segs = max(1, (keys + target - 1) / target);
      s.seg_tiles = *tails && s.segs > 1 ? target : (keys + s.segs - 1) / s.segs;
      // cu_seqlens that do not rise ask for more slots than there are: those stay whole.
      const int slots = s.segs > 1 ? static_cast<int>(min(static_cast<int64_t>(s.nq) * s.segs, static_cast<int64_t>(p.slots) + 1)) : 0;
      s.slot0 = scan_sum(slots) - slots;
      if (s.slot0 + slots > p.slots) s.segs = 1, s.seg_tiles = keys;
    }
  }
  return s;
}

struct Item {
  int seq, head, tile, seg;  // head: a group of them
  int row0, nq, len, segs, seg_tiles, slot0;
};

// Work item blockIdx.x, worked out by every wave alike; false past the last.
template <bool TAILS>
__device__ __forceinline__ bool find_item(const Prefill8Args& p, Item* it) {
  const Attn8Args& a = p.a;
  const int lane = threadIdx.x & 63;
  // Workgroup b runs on XCD b % 8, which serves the heads h == b (mod 8), or (mod 4) or (mod 2) where their number
  // divides by no more.  (With all heads in turn on every XCD instead, over the e4m3 cache, us: three prompts of 1500-2048,
  // 12 / 20 / 10 / 2 heads 77 / 124 / 77 / 35.0, so 72 / 113 / 71 / 35.7; eight 512-token chunks, 12 / 20 heads
  // 291 / 471, so 286 / 478.)
  const int all_heads = a.hq / p.group;
  const int groups = all_heads % 8 == 0 ? 8 : all_heads % 4 == 0 ? 4 : all_heads % 2 == 0 ? 2 : 1, heads = all_heads / groups;
  const int x = blockIdx.x % groups;
  int pos = blockIdx.x / groups;
  int unit;
  if (a.num_seqs <= kPlanSeqs) {
    bool tails;
    const SeqPlan s = plan_of<TAILS>(p, lane, &tails);
    if (p.part_acc && blockIdx.x == 0 && threadIdx.x < a.num_seqs) p.plan[lane] = s;
    // A sequence's items: those of its segments, a shorter last one (`tail`) apart.
    const int last = (s.len + kBN - 1) / kBN - (s.segs - 1) * s.seg_tiles;
    const int tail_units = tails && s.segs > 1 && last < s.seg_tiles ? s.tiles : 0, units = s.tiles * s.segs - tail_units;
    // Units of longer items than these: their keys are distinct, equal lengths in the sequences' order.
    const uint32_t key = static_cast<uint32_t>(s.seg_tiles) << 7 | (127 - lane), tail_key = static_cast<uint32_t>(last) << 7 | (63 - lane);
    int before = 0, tail_before = 0;
    auto count = [&](uint32_t of_key, int of_units) __attribute__((always_inline)) {
#pragma unroll 4
      for (int q = 0; q < a.num_seqs; ++q) {
        const uint32_t k = __builtin_amdgcn_readlane(of_key, q);
        const int u = __builtin_amdgcn_readlane(of_units, q);
        before += k > key ? u : 0;
        if (tails) tail_before += k > tail_key ? u : 0;
      }
    };
    count(key, units);
    if (tails) count(tail_key, tail_units);
    auto item_of = [&](int b, int n) __attribute__((always_inline)) {  // the lane whose items [b, b + n) hold this one
      const int64_t first = static_cast<int64_t>(b) * heads, end = first + static_cast<int64_t>(n) * heads;
      return __builtin_amdgcn_ballot_w64(lane < a.num_seqs && pos >= first && pos < end);
    };
    const uint64_t body = item_of(before, units), tail = tails ? item_of(tail_before, tail_units) : 0;
    if (!(body | tail)) return false;
    const int at = __builtin_ctzll(body ? body : tail);
    it->seq = at;
    pos -= __builtin_amdgcn_readlane(body ? before : tail_before, at) * heads;
    it->row0 = __builtin_amdgcn_readlane(s.row0, at), it->nq = __builtin_amdgcn_readlane(s.nq, at);
    it->len = __builtin_amdgcn_readlane(s.len, at), it->segs = __builtin_amdgcn_readlane(s.segs, at);
    it->seg_tiles = __builtin_amdgcn_readlane(s.seg_tiles, at), it->slot0 = __builtin_amdgcn_readlane(s.slot0, at);
    const int tiles = __builtin_amdgcn_readlane(s.tiles, at), of_head = __builtin_amdgcn_readlane(body ? units : tail_units, at);
    it->head = x + groups * (pos / of_head);
    unit = pos % of_head;
    it->seg = unit / tiles;
    unit -= it->seg * tiles;
    if (!body) it->seg = it->segs - 1;
    it->tile = tiles - 1 - unit;  // the last rows, which see most keys, first
    return true;
  }
  // More sequences: in order and uncut, found 64 at a time.
  it->head = x + groups * (pos % heads);
  unit = pos / heads;
  for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
    int row0 = 0, nq = 0;
    if (s0 + lane < a.num_seqs) seq_rows(a, s0 + lane, row0, nq);
    const int tiles = (nq * p.group + kBM - 1) / kBM, before = scan_sum(tiles) - tiles;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(unit >= before && unit < before + tiles);
    if (hit) {
      const int at = __builtin_ctzll(hit);
      it->seq = s0 + at;
      it->row0 = __builtin_amdgcn_readlane(row0, at), it->nq = __builtin_amdgcn_readlane(nq, at);
      it->len = uniform(sequence_length(a, it->seq));
      it->segs = 1, it->seg = 0, it->slot0 = 0;
      it->seg_tiles = (it->len + kBN - 1) / kBN;
      it->tile = __builtin_amdgcn_readlane(tiles, at) - 1 - (unit - __builtin_amdgcn_readlane(before, at));
      return true;
    }
    unit -= __builtin_amdgcn_readlane(before + tiles, 63);
  }
  return false;
}

// Elements d .. d + 3 of an out row.
template <typename T>
__device__ __forceinline__ void store4(T* orow, int d, const float (&x)[4], int64_t stride, bool vec) {
  if (vec) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(orow + d) = f32x4{x[0], x[1], x[2], x[3]};
    else *reinterpret_cast<u32x2*>(orow + d) = u32x2{MfmaOps<T>::pack2(x[0], x[1]), MfmaOps<T>::pack2(x[2], x[3])};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) store_elem(orow + (d + e) * stride, x[e]);
  }
}

// Partial rows that a launch can need: a cut sequence's rows once a segment.  It has more keys
// than a segment, which is at least (all work) / kTargetItems: so its segments are fewer than
// twice its keys over a segment's, and those of all sequences, times their query tiles, fewer
// than 2 kTargetItems / hq; those past each sequence's first, fewer than half as many.  No
// sequence has more segments than its table's keys allow.
inline int64_t partial_slots(int64_t rows, int64_t num_seqs, int64_t max_len, int64_t hq) {
  const int64_t most = ((max_len + kBN - 1) / kBN + kMinSegTiles - 1) / kMinSegTiles;
  if (num_seqs > kPlanSeqs || most < 2) return 0;
  constexpr int64_t cut = kBM * kTargetItems;
  return std::min({rows * most, rows + (cut + hq - 1) / hq + 64, (2 * cut + hq - 1) / hq + 64});
}

// Everything of p but its partials: how q and out are read and written, and the softmax scale.
inline void fill_prefill8(Prefill8Args* p, int dtype) {
  const Attn8Args& a = p->a;
  p->page_shift = __builtin_ctz(a.page);
  p->qscale = std::fabs(a.qscale);
  // A scale of 0 stands as 2^-126 2^-kMaxQExp: a finite score ends below 2^-22, a masked one stays -inf.
  const bool none = p->qscale == 0.f;
  p->q_exp = none ? -kMaxQExp : std::isfinite(p->qscale) ? std::min(std::max(std::ilogb(p->qscale), -kMaxQExp), 0) : 0;
  p->qscale = none ? std::numeric_limits<float>::min() : std::ldexp(p->qscale, -p->q_exp);
  p->q_sign = a.qscale < 0.f ? 0x80000000u : 0u;
  const int es = dtype_size(dtype);
  p->q_vec = a.q_dim == 1 && aligned16(a.q) && a.q_row * es % 16 == 0 && a.q_head * es % 16 == 0;
  p->out_vec = a.o_dim == 1 && aligned16(a.out) && a.o_row * es % 16 == 0 && a.o_head * es % 16 == 0;
}

// Query tiles, and the segments past the first: of all heads fewer than `more`, as a segment is at least
// all work / `more` (which is kTargetItems, or with tails the round).
inline int64_t prefill8_tiles(const Prefill8Args& p, int64_t more) {
  const int64_t heads = p.a.hq / p.group;
  return p.a.rows * p.group / kBM + std::min<int64_t>(p.a.num_seqs, p.a.rows) + (p.slots ? (more + heads - 1) / heads + 2 : 0);
}

}  // namespace rlt
