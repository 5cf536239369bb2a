// Appends to the block-scaled 8-bit KV cache, and reading it back (int8.hpp).
//
// Append.  The rows of a call that go to one block stand together in it, but for rows that are
// skipped; a wave takes them as one, for a head:
//   s0 = the block's scale, 0 where the call writes its offset 0 (which begins the block)
//   s  = max(s0, largest |x| of the new rows * (1 / 127), 2^-126)
//   codes the block holds: rint(code * (s0 / s)), where s is not s0
//   new codes: rint(x * (1 / s))
// each operation rounded to fp32 on its own, ties to even.  A code that is kept is rounded
// again each time s grows, by at most half a step of the new scale.  New rows with a value that
// is not finite make s NaN, and their codes say nothing then; s0 NaN stays.
#include <algorithm>
#include <type_traits>

#include "int8.hpp"

namespace rlt {
namespace {

constexpr int kWaves = 4;

struct AppendI8Args {
  const void* x[2];  // k, v
  int64_t x_row[2], x_head[2], x_dim[2];
  uint8_t* codes[2];
  int64_t c_block, c_layer, c_token, c_head, c_dim;
  float* scales[2];
  int64_t s_block, s_layer, s_head;
  const int64_t* blocks;
  const int64_t* offsets;
  int64_t rows, layer, num_blocks, page;
  int hkv, d;
};

__device__ __forceinline__ bool valid_block(const AppendI8Args& a, int64_t b) { return b >= 0 && b < a.num_blocks; }
__device__ __forceinline__ bool valid_offset(const AppendI8Args& a, int64_t o) { return o >= 0 && o < a.page; }

// The block of row `row`, -1 for one that is skipped: outside the pool, or of an offset outside its page.
__device__ __forceinline__ int block_of_row(const AppendI8Args& a, int64_t row) {
  const int64_t block = a.blocks[row], offset = a.offsets[row];
  return valid_block(a, block) && valid_offset(a, offset) ? static_cast<int>(block) : -1;
}

// Rows of one block are a run, with up to kGap skipped rows between two of them, or a page's tokens: so many
// as consecutive tokens of a block can have.  (Any number would have a padded batch searched to its end: 100
// rows of 4096 12.7 us, so 4.5.)
constexpr int64_t kGap = 32;

// The last row of the run of `block` that has row `last`, its last one up to row from - 1; *count grows by its
// rows from `from` on.
__device__ __forceinline__ int64_t run_last(const AppendI8Args& a, int block, int64_t last, int64_t from, int lane, int64_t* count) {
  const int64_t gap = std::max(kGap, a.page);
  for (; from < a.rows && from - last - 1 <= gap; from += 64) {
    const int64_t at = from + lane;
    const int b = at < a.rows ? block_of_row(a, at) : -1;
    const uint64_t mine = __builtin_amdgcn_ballot_w64(b == block), other = __builtin_amdgcn_ballot_w64(b >= 0 && b != block);
    const uint64_t run = other ? mine & ((other & -other) - 1) : mine;
    if (run) last = from + 63 - __builtin_clzll(run);
    *count += __builtin_popcountll(run);
    if (other) return last;
  }
  return last;
}

// The block of the last row before `row` that is not skipped; -1 where the rows that a run can have between two
// of its own are skipped.
__device__ __forceinline__ int block_before(const AppendI8Args& a, int64_t row, int lane) {
  const int64_t stop = row - std::max(kGap, a.page);
  for (; row > 0 && row > stop; row -= 64) {
    const int64_t at = row - 64 + lane;
    const int b = at >= 0 ? block_of_row(a, at) : -1;
    if (const uint64_t in = __builtin_amdgcn_ballot_w64(b >= 0)) return __builtin_amdgcn_readlane(b, 63 - __builtin_clzll(in));
  }
  return -1;
}

// The new scale, from the old one (0 for a block that begins) and the bits of the largest |x|.
__device__ __forceinline__ float grown_scale(float before, uint32_t top) {
  if (top >= 0x7f800000u || before != before) return __uint_as_float(0x7fc00000u);
  return fmaxf(fmaxf(before, __uint_as_float(top) * kInverseLargest), kSmallestScale);
}

// The low byte of the result is x rounded to a whole number, ties to even, for |x| below 2^22: added to
// 1.5 * 2^23 it moves to the last bits of the sum.  (0 for NaN.)
__device__ __forceinline__ uint32_t code_of(float x, float inv) {
#pragma clang fp contract(off)
  return __float_as_uint(x * inv + 12582912.f);
}
// Four of them, the first in the lowest byte.
__device__ __forceinline__ uint32_t codes4(const float* x, float inv) {
  const uint32_t lo = __builtin_amdgcn_perm(code_of(x[1], inv), code_of(x[0], inv), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(code_of(x[3], inv), code_of(x[2], inv), 0x04000c0cu);
  return lo | hi;
}
// A code's value, rounded to fp32 also where it is rounded to 16 bits next (the compiler would
// join both into one instruction for fp16, and not for bf16).
__device__ __forceinline__ float code_value(int code, float scale) {
  float x = static_cast<float>(code) * scale;
  asm("" : "+v"(x));
  return x;
}

// Any strides and head size: a wave a (row, K or V, head); the first row of a block works.  Latency bounds it:
// 4096 rows of 8 sequences, 16 heads x 65, 65 us.
template <typename T>
__global__ __launch_bounds__(64) void append_i8_generic_kernel(AppendI8Args a) {
  const int lane = threadIdx.x, which = blockIdx.y / a.hkv, head = blockIdx.y % a.hkv;
  const int64_t row = blockIdx.x;
  const int block_at = uniform(block_of_row(a, row));
  if (block_at < 0) return;
  if (row > 0) {
    int previous = uniform(block_of_row(a, row - 1));
    if (previous < 0) previous = block_before(a, row - 1, lane);
    if (previous == block_at) return;
  }
  int64_t count = 1;
  const int64_t block = block_at, n = run_last(a, block_at, row, row + 1, lane, &count) - row + 1;
  const bool dense = count == n;  // no skipped rows between them
  const T* x = static_cast<const T*>(a.x[which]) + row * a.x_row[which] + head * a.x_head[which];
  uint8_t* codes = a.codes[which] + block * a.c_block + a.layer * a.c_layer + head * a.c_head;
  float* scale = a.scales[which] + block * a.s_block + a.layer * a.s_layer + head * a.s_head;
  uint32_t top = 0;
  bool begins = false;
  for (int64_t r = 0; r < n; ++r) {
    const int64_t offset = a.offsets[row + r];
    if (!dense && (a.blocks[row + r] != block || !valid_offset(a, offset))) continue;
    begins |= offset == 0;
    for (int d = lane; d < a.d; d += 64)
      top = max(top, __float_as_uint(load_elem(x + r * a.x_row[which] + d * a.x_dim[which])) & 0x7fffffffu);
  }
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), i, 64)));
  const float before = begins ? 0.f : *scale, s = grown_scale(before, top);
  if (lane == 0) *scale = s;
  if (!begins && s != before && s == s) {
    const float ratio = before / s;
    for (int64_t o = 0; o < a.page; ++o)
      for (int d = lane; d < a.d; d += 64) {
        uint8_t* c = codes + o * a.c_token + d * a.c_dim;
        *c = static_cast<uint8_t>(code_of(static_cast<float>(static_cast<int8_t>(*c)), ratio));
      }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // before the new rows' codes
  }
  const float inv = s == s ? 1.f / s : s;
  for (int64_t r = 0; r < n; ++r) {
    const int64_t offset = a.offsets[row + r];
    if (!dense && (a.blocks[row + r] != block || !valid_offset(a, offset))) continue;
    for (int d = lane; d < a.d; d += 64)
      codes[offset * a.c_token + d * a.c_dim] =
          static_cast<uint8_t>(code_of(load_elem(x + r * a.x_row[which] + d * a.x_dim[which]), inv));
  }
}

// Largest over aligned groups of W lanes.
template <int W>
__device__ __forceinline__ uint32_t group_umax(uint32_t x) {
  auto step = [&](uint32_t y) { x = max(x, y); };
  auto by = [&](auto ctrl) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  if constexpr (W >= 2) step(by(std::integral_constant<int, kDppXor1>{}));
  if constexpr (W >= 4) step(by(std::integral_constant<int, kDppXor2>{}));
  if constexpr (W >= 8) step(by(std::integral_constant<int, kDppHalfMirror>{}));
  if constexpr (W >= 16) step(by(std::integral_constant<int, kDppMirror>{}));
  if constexpr (W >= 32) step(static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), 16, 64)));
  if constexpr (W >= 64) step(static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), 32, 64)));
  return x;
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// Largest |x| of packets so far, in the type's own bits (their order is the magnitudes': infinities
// above the finite ones, NaNs above those), two 16-bit values a word.
template <typename T>
__device__ __forceinline__ uint32_t packet_max(uint32_t top, const u32x4& x) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (sizeof(T) == 4) top = max(top, x[w] & 0x7fffffffu);
    else top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top), __builtin_bit_cast(u16x2, x[w] & 0x7fff7fffu)));
  }
  return top;
}
// Those bits as fp32's.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint32_t top) {
  if constexpr (sizeof(T) == 4) return top;
  const uint32_t x = max(top & 0xffffu, top >> 16);
  if constexpr (std::is_same_v<T, bf16>) return x << 16;
  else return __float_as_uint(static_cast<float>(__builtin_bit_cast(f16, static_cast<uint16_t>(x))));
}

// Codes of a lane's packet of N values: a word of four each.
template <int N> struct Codes {
  uint32_t w[N / 4];
};
template <int N>
__device__ __forceinline__ Codes<N> load_codes(const uint8_t* p) {
  Codes<N> c;
  if constexpr (N == 8) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    c.w[0] = x.x, c.w[1] = x.y;
  } else {
    c.w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
  return c;
}
template <int N>
__device__ __forceinline__ void store_codes(uint8_t* p, const Codes<N>& c) {
  if constexpr (N == 8) *reinterpret_cast<uint2*>(p) = make_uint2(c.w[0], c.w[1]);
  else *reinterpret_cast<uint32_t*>(p) = c.w[0];
}
__device__ __forceinline__ int code_at(uint32_t word, int byte) { return static_cast<int8_t>(word >> (8 * byte)); }

// Codes that a block holds, rounded anew: this lane's packets of tokens first, first + step, ...; none where own is false.
template <int N, int BATCH>
__device__ __forceinline__ void requantise(uint8_t* codes, int64_t c_token, int page, int first, int step, float ratio, bool own) {
  for (int t0 = first; t0 < page; t0 += BATCH * step) {
    Codes<N> c[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) c[u] = load_codes<N>(codes + min(t0 + u * step, page - 1) * c_token);
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
#pragma unroll
      for (int w = 0; w < N / 4; ++w) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = static_cast<float>(code_at(c[u].w[w], e));
        c[u].w[w] = codes4(y, ratio);
      }
      if (own && t0 + u * step < page) store_codes<N>(codes + (t0 + u * step) * c_token, c[u]);
    }
  }
}

template <typename T>
__device__ __forceinline__ void store_packet(uint8_t* to, const u32x4& x, float inv) {
  constexpr int N = Packet<T>::N;
  float y[N];
  Packet<T>::unpack(x, y);
  Codes<N> c;
#pragma unroll
  for (int w = 0; w < N / 4; ++w) c.w[w] = codes4(y + 4 * w, inv);
  store_codes<N>(to, c);
}

// Aligned heads of LPH 16-byte packets, or (PAD) of fewer: lanes past the last have it again and store
// nothing.  A wave has K or V of a head of up to kHeld rows, `tile`: it looks
// for the blocks that begin there.  Those that get one row (a decode batch's) it takes all at once,
// LPH lanes a row; the others one after another, 64 / LPH tokens at once, so that a block's
// largest |x| is over the wave, and its scale is the wave's.  kHeld tokens of a block stay in
// registers between finding its scale and using it; more are read twice.  Bytes bound it: 4096 rows
// of 8 sequences, 16 heads x 128, bf16, move 50 MB in 12.1 us, 4.2 TB/s.  (With the heads, not the
// tokens, of a wave side by side 15.6: 16 registers a lane for every token, and few waves.)
// Blocks whose scales grow have their codes read, rounded and written, one after another in a wave: 64 rows of a
// block each, 8 heads, fp16, 3.6 us where none grows, 4.4 where one in six does, as when blocks of like values
// fill, 5.4 where all do; 4096 of them, 16 heads, bf16, 12.8, 26.5 and 103, those bytes' time (all: 537 MB).
constexpr int kHeld = 16;
template <typename T, int LPH, bool PAD>
__global__ __launch_bounds__(64 * kWaves) void append_i8_kernel(AppendI8Args a, int tile) {
  constexpr int N = Packet<T>::N, TPI = 64 / LPH, H = TPI < kHeld ? kHeld / TPI : 1;  // packets a lane holds
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kWaves + uniform(threadIdx.x >> 6);
  const int64_t row0 = item / (2 * a.hkv) * tile;
  if (row0 >= a.rows) return;
  const int of_tile = uniform(static_cast<int>(item % (2 * a.hkv)));
  const int which = of_tile >= a.hkv, head = of_tile - which * a.hkv;
  const int lane = threadIdx.x & 63, i = lane % LPH, sub = lane / LPH, page = static_cast<int>(a.page);
  const int packets = PAD ? a.d / N : LPH, at_dim = min(i, packets - 1) * N;
  const bool own = i < packets;
  // Lane l has the block and the offset of row row0 - 1 + l, -1 for a row that is skipped.
  const int64_t at = row0 - 1 + lane;
  const bool there = at >= 0 && at < a.rows;
  const int64_t block_at = there ? a.blocks[at] : -1, offset_at = there ? a.offsets[at] : -1;
  const int64_t x_row = a.x_row[which];
  const T* const x0 = static_cast<const T*>(a.x[which]) + row0 * x_row + head * a.x_head[which] + at_dim;
  u32x4 held[H];
  const bool early = tile <= TPI;  // few rows, mostly blocks of one: on their way with the block's number
  const int last = static_cast<int>(min(static_cast<int64_t>(tile), a.rows - row0)) - 1;  // (of the tile; rows past it: it again, of no use)
  if (early) held[0] = *reinterpret_cast<const u32x4*>(x0 + min(sub, last) * x_row);
  const bool used = valid_block(a, block_at) && valid_offset(a, offset_at);
  const int block = used ? static_cast<int>(block_at) : -1, offset = used ? static_cast<int>(offset_at) : -1;
  const uint64_t rows = __builtin_amdgcn_ballot_w64(used), below = rows & ((uint64_t(1) << lane) - 1);
  const int previous = __shfl(block, below ? 63 - __builtin_clzll(below) : lane, 64);
  uint64_t same = __builtin_amdgcn_ballot_w64(used && below && block == previous);  // as the row before that is not skipped
  const uint64_t tile_rows = ((uint64_t(1) << tile) - 1) << 1;
  if (row0 > 1 && rows & tile_rows && !(rows & 1)) {  // that of the tile's first row is further away
    const int first = __builtin_ctzll(rows);
    if (block_before(a, row0 - 1, lane) == __builtin_amdgcn_readlane(block, first)) same |= uint64_t(1) << first;
  }
  const uint64_t begins_at = rows & ~same, begin = begins_at & tile_rows;
  // Runs of more than one row: `same` moved down to the row before, over skipped ones, as a carry is.
  const uint64_t gaps = __builtin_bitreverse64(~rows);
  uint64_t followed = __builtin_bitreverse64((gaps + (__builtin_bitreverse64(same) << 1)) & ~gaps);
  // The last run in sight may go on behind it.
  int64_t end = -1, behind = 0;
  const int64_t in_sight = row0 - 1 + 63 - __builtin_clzll(rows | 1);
  if (begin && row0 + 63 < a.rows && row0 + 62 - in_sight <= std::max(kGap, a.page)) {
    const int first = 63 - __builtin_clzll(begins_at);
    if (begin >> first & 1) {
      end = run_last(a, __builtin_amdgcn_readlane(block, first), in_sight, row0 + 63, lane, &behind);
      if (end > in_sight) followed |= uint64_t(1) << first;
    }
  }
  const uint64_t single = begin & ~followed;
  uint8_t* const codes0 = a.codes[which] + a.layer * a.c_layer + head * a.c_head + at_dim;
  float* const scale0 = a.scales[which] + a.layer * a.s_layer + head * a.s_head;
  if (single) {
    float old[H], inv[H], ratio = 1.f;  // ratio: lane t's is row t's
    int blk[H], slot[H];
#pragma unroll
    for (int u = 0; u < H; ++u) {
      const int t = u * TPI + sub;
      blk[u] = __shfl(block, 1 + t, 64);
      slot[u] = __shfl(offset, 1 + t, 64);
      if (!(single >> (1 + t) & 1)) slot[u] = -1;
      if (!(early && u == 0)) held[u] = *reinterpret_cast<const u32x4*>(x0 + min(t, last) * x_row);
      old[u] = scale0[max(blk[u], 0) * a.s_block];
    }
#pragma unroll
    for (int u = 0; u < H; ++u) {
      const float before = slot[u] == 0 ? 0.f : old[u], s = grown_scale(before, group_umax<LPH>(top_bits<T>(packet_max<T>(0, held[u]))));
      inv[u] = s == s ? 1.f / s : s;
      const float of_row = slot[u] > 0 && s == s && s != before ? before / s : 1.f;  // (an infinite one stays)
      if (slot[u] >= 0 && i == 0) scale0[blk[u] * a.s_block] = s;
      const float of_lane = __shfl(of_row, lane % TPI * LPH, 64);
      ratio = lane / TPI == u ? of_lane : ratio;
    }
    uint64_t grown = __builtin_amdgcn_ballot_w64(lane < H * TPI && ratio != 1.f);
    for (; grown; grown &= grown - 1) {
      const int t = __builtin_ctzll(grown);
      const float r = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ratio), t));
      requantise<N, (H < 8 ? H : 8)>(codes0 + __builtin_amdgcn_readlane(block, 1 + t) * a.c_block, a.c_token, page, sub, TPI, r, own);
      if (!(grown & (grown - 1))) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // before the new rows' codes
    }
#pragma unroll
    for (int u = 0; u < H; ++u)
      if (own && slot[u] >= 0) store_packet<T>(codes0 + blk[u] * a.c_block + slot[u] * a.c_token, held[u], inv[u]);
  }
  for (uint64_t first = begin & ~single; first; first &= first - 1) {
    const int l0 = __builtin_ctzll(first);
    const int64_t row = row0 - 1 + l0, blk = __builtin_amdgcn_readlane(block, l0);
    const uint64_t after = ~((uint64_t(2) << l0) - 1), next = begins_at & after;
    const uint64_t run = same & after & (next ? (next & -next) - 1 : ~uint64_t(0));
    // Rows to the block's last, skipped ones among them.
    const int n = next || end < 0 ? 64 - __builtin_clzll(run) - l0 : static_cast<int>(end - row + 1);
    const bool dense = 1 + __builtin_popcountll(run) + (next ? 0 : behind) == n;
    float* const scale = scale0 + blk * a.s_block;
    uint8_t* const codes = codes0 + blk * a.c_block;
    const float old = *scale;
    const T* const x = x0 + (l0 - 1) * x_row;
    int o[H];  // the offset of this lane's token, -1 for none
    auto load = [&](int from) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < H; ++u) {
        const int t = from + u * TPI + sub;
        held[u] = *reinterpret_cast<const u32x4*>(x + min(t, n - 1) * x_row);
        o[u] = __shfl(offset, min(l0 + t, 63), 64);
        if (t < n && l0 + t > 63) {
          // (Without branches: the compiler of ROCm 7.2 lost the offset where the condition was one.)
          int64_t wide = a.offsets[row + t], of_block = blk;
          if (!dense) of_block = a.blocks[row + t];
          o[u] = static_cast<int>(wide) | -static_cast<int>((of_block != blk) | (wide < 0) | (wide >= a.page));
        }
        if (t >= n) o[u] = -1;
      }
    };
    uint32_t top = 0;
    bool begins = false;
    for (int from = 0; from < n; from += H * TPI) {
      load(from);
#pragma unroll
      for (int u = 0; u < H; ++u) {
        begins |= o[u] == 0;
        if (o[u] >= 0) top = packet_max<T>(top, held[u]);
      }
    }
    const bool fresh = __builtin_amdgcn_ballot_w64(begins) != 0;
    const float before = fresh ? 0.f : old, s = grown_scale(before, group_umax<64>(top_bits<T>(top)));
    if (lane == 0) *scale = s;
    if (__builtin_amdgcn_ballot_w64(!fresh && s != before && s == s)) {
      requantise<N, (H < 8 ? H : 8)>(codes, a.c_token, page, sub, TPI, before / s, own);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // before the new rows' codes
    }
    const float inv = s == s ? 1.f / s : s;
    for (int from = 0; from < n; from += H * TPI) {
      if (n > H * TPI) load(from);
#pragma unroll
      for (int u = 0; u < H; ++u)
        if (own && o[u] >= 0) store_packet<T>(codes + o[u] * a.c_token, held[u], inv);
    }
  }
}

struct GatherI8Args {
  const uint8_t* codes[2];
  int64_t c_block, c_layer, c_token, c_head, c_dim;
  const float* scales[2];
  int64_t s_block, s_layer, s_head;
  const int64_t* blocks;
  const int64_t* offsets;
  void* out[2];  // [rows, hkv, d]
  int64_t rows, layer, num_blocks, page;
  int hkv, d;
};

// Any strides and head size: a wave a (row, K or V, head); 8192 rows of 16 heads x 65 take 66 us.
template <typename T>
__global__ __launch_bounds__(64) void gather_i8_generic_kernel(GatherI8Args a) {
  const int lane = threadIdx.x, which = blockIdx.y / a.hkv, head = blockIdx.y % a.hkv;
  const int64_t row = blockIdx.x, block = a.blocks[row], offset = a.offsets[row];
  const bool in = block >= 0 && block < a.num_blocks && offset >= 0 && offset < a.page;
  const uint8_t* codes = a.codes[which] + block * a.c_block + a.layer * a.c_layer + offset * a.c_token + head * a.c_head;
  T* out = static_cast<T*>(a.out[which]) + (row * a.hkv + head) * a.d;
  const float s = in ? a.scales[which][block * a.s_block + a.layer * a.s_layer + head * a.s_head] : 0.f;
  for (int d = lane; d < a.d; d += 64)
    store_elem(out + d, in ? code_value(static_cast<int8_t>(codes[d * a.c_dim]), s) : 0.f);
}

// Aligned heads of up to LPH packets of N codes, 16 bytes of the result: a wave takes K and V of a row.
// Bytes bound it: 8192 rows of 16 heads x 128 to bf16, 101 MB, take 17 to 19 us.
template <typename T, int LPH>
__global__ __launch_bounds__(64 * kWaves) void gather_i8_kernel(GatherI8Args a) {
  constexpr int N = Packet<T>::N, HPW = 64 / LPH, U = 4;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + uniform(threadIdx.x >> 6);
  if (row >= a.rows) return;
  const int lane = threadIdx.x & 63, i = lane % LPH;
  if (i >= a.d / N) return;
  const int64_t block = a.blocks[row], offset = a.offsets[row];
  const bool in = block >= 0 && block < a.num_blocks && offset >= 0 && offset < a.page;
  const int64_t at = in ? block * a.c_block + a.layer * a.c_layer + offset * a.c_token + i * N : 0;
  const int64_t s_at = in ? block * a.s_block + a.layer * a.s_layer : 0;
  for (int h0 = lane / LPH; h0 < a.hkv; h0 += U * HPW) {
    Codes<N> c[2][U];
    float s[2][U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int h = h0 + u * HPW;
        if (!in || h >= a.hkv) continue;
        c[w][u] = load_codes<N>(a.codes[w] + at + h * a.c_head);
        s[w][u] = a.scales[w][s_at + h * a.s_head];
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int h = h0 + u * HPW;
        if (h >= a.hkv) continue;
        float y[N];
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = in ? code_value(code_at(c[w][u].w[e / 4], e % 4), s[w][u]) : 0.f;
        *reinterpret_cast<u32x4*>(static_cast<T*>(a.out[w]) + (row * a.hkv + h) * a.d + i * N) = Packet<T>::pack(y);
      }
  }
}

// What both entry points check.
int cache_args(const char* name, const void* key_cache, const void* value_cache, const int64_t* cache_strides,
               const void* key_scales, const void* value_scales, const int64_t* scale_strides, const int64_t* blocks,
               const int64_t* offsets, int64_t n_rows, int64_t layer, int64_t num_layers, int64_t num_blocks, int64_t page_size,
               int64_t hkv, int64_t d, int dtype) {
  if (!dtype_size(dtype)) return fail(RLT_EINVAL, "%s: unknown dtype %d", name, dtype);
  if (n_rows < 0) return fail(RLT_EINVAL, "%s: n_rows is negative", name);
  if (hkv <= 0 || d <= 0) return fail(RLT_EINVAL, "%s: num_kv_heads and head_dim must be positive", name);
  if (num_blocks <= 0 || num_layers <= 0 || page_size <= 0) return fail(RLT_EINVAL, "%s: pool dimensions must be positive", name);
  if (layer < 0 || layer >= num_layers) return fail(RLT_EINVAL, "%s: layer %lld out of range", name, (long long)layer);
  if (d > 64 * kPerLane) return fail(RLT_EUNSUPPORTED, "%s: head_dim above %d", name, 64 * kPerLane);
  // (A wave a row, K or V and head at worst, four a workgroup: threads of a launch inside 32 bits.  A
  // page's tokens and what a wave's steps add to them stay inside 31.)
  if (n_rows > kMaxBlocks || hkv > 16384 || n_rows * hkv > 2 * kMaxBlocks || num_blocks > 0x7fffffff || page_size > kMaxKeys)
    return fail(RLT_EUNSUPPORTED, "%s: too many rows, heads, blocks or tokens a page", name);
  if (n_rows == 0) return RLT_OK;
  if (!key_cache || !value_cache || !cache_strides || !key_scales || !value_scales || !scale_strides || !blocks || !offsets)
    return fail(RLT_EINVAL, "%s: NULL pointer argument", name);
  for (int i = 0; i < 5; ++i)
    if (cache_strides[i] < 0 || (i < 3 && scale_strides[i] < 0)) return fail(RLT_EINVAL, "%s: negative cache stride", name);
  if (reinterpret_cast<uintptr_t>(key_scales) % 4 || reinterpret_cast<uintptr_t>(value_scales) % 4)
    return fail(RLT_EINVAL, "%s: scales must be on 4 bytes", name);
  return RLT_OK;
}

// Whether codes of N at once are aligned, in both caches.
template <typename A>
bool code_packets(const A& a, int n) {
  for (int w = 0; w < 2; ++w)
    if (reinterpret_cast<uintptr_t>(a.codes[w]) % n) return false;
  return a.c_dim == 1 && a.c_block % n == 0 && a.c_layer % n == 0 && a.c_token % n == 0 && a.c_head % n == 0;
}

// Lanes of a head, one a 16-byte packet of T, a power of two of them; 0 where the packet kernels do not
// cover the head size.
template <typename T>
int lanes_of(int d) {
  constexpr int N = Packet<T>::N;
  if (d % N || d > 64 * N) return 0;
  int lanes = 4;
  while (lanes * N < d) lanes *= 2;
  return lanes;
}

#define BY_LANES(LAUNCH)   \
  switch (lanes) {         \
    case 4: LAUNCH(4);     \
    case 8: LAUNCH(8);     \
    case 16: LAUNCH(16);   \
    case 32: LAUNCH(32);   \
    case 64: LAUNCH(64);   \
  }

template <typename T>
void launch_append(const AppendI8Args& a, hipStream_t stream) {
  constexpr int64_t es = sizeof(T);
  bool packets = code_packets(a, Packet<T>::N);
  for (int w = 0; w < 2; ++w)
    packets = packets && a.x_dim[w] == 1 && aligned16(a.x[w]) && a.x_row[w] * es % 16 == 0 && a.x_head[w] * es % 16 == 0;
  const int lanes = packets ? lanes_of<T>(a.d) : 0;
  if (lanes) {
    // As many rows a wave as leave it 4096 waves, down to as many as it loads at once.  Measured, us, 4
    // / 8 / 16 rows: 4096 rows of 8 sequences, 16 heads x 128 21.6 / 12.9 / 12.4, 512 of two 5.4 / 6.1 /
    // 6.2, 4096 of 4096, 8 heads 13.0 / 9.3 / 8.6 (with one row a wave 51, 9 and 37).
    int tile = kHeld;
    while (tile > std::max(1, 64 / lanes) && (a.rows + tile - 1) / tile * 2 * a.hkv < 4096) tile /= 2;
    const int64_t waves = (a.rows + tile - 1) / tile * 2 * a.hkv;
    const dim3 grid(static_cast<unsigned>((waves + kWaves - 1) / kWaves)), block(64 * kWaves);
#define LAUNCH(L)                                                                                                    \
  if (a.d == L * Packet<T>::N) hipLaunchKernelGGL((append_i8_kernel<T, L, false>), grid, block, 0, stream, a, tile); \
  else hipLaunchKernelGGL((append_i8_kernel<T, L, true>), grid, block, 0, stream, a, tile);                          \
  return
    BY_LANES(LAUNCH)
#undef LAUNCH
  }
  const dim3 grid(static_cast<unsigned>(a.rows), static_cast<unsigned>(2 * a.hkv));
  hipLaunchKernelGGL((append_i8_generic_kernel<T>), grid, dim3(64), 0, stream, a);
}

template <typename T>
void launch_gather(const GatherI8Args& a, hipStream_t stream) {
  const bool packets = code_packets(a, Packet<T>::N) && aligned16(a.out[0]) && aligned16(a.out[1]);
  const int lanes = packets ? lanes_of<T>(a.d) : 0;
  if (lanes) {
    const int64_t waves = a.rows;
    const dim3 grid(static_cast<unsigned>((waves + kWaves - 1) / kWaves)), block(64 * kWaves);
#define LAUNCH(L) hipLaunchKernelGGL((gather_i8_kernel<T, L>), grid, block, 0, stream, a); return
    BY_LANES(LAUNCH)
#undef LAUNCH
  }
  const dim3 grid(static_cast<unsigned>(a.rows), static_cast<unsigned>(2 * a.hkv));
  hipLaunchKernelGGL((gather_i8_generic_kernel<T>), grid, dim3(64), 0, stream, a);
}
#undef BY_LANES

}  // namespace
}  // namespace rlt

using namespace rlt;

extern "C" int rlt_kv_append_int8(void* key_cache, void* value_cache, const int64_t* cache_strides, void* key_scales,
                                  void* value_scales, const int64_t* scale_strides, const void* k,
                                  const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                  const int64_t* write_blocks, const int64_t* write_offsets, int64_t n_rows,
                                  int64_t layer, int64_t num_layers, int64_t num_blocks, int64_t page_size,
                                  int64_t num_kv_heads, int64_t head_dim, int dtype, void* stream) {
  const char* name = "rlt_kv_append_int8";
  if (int rc = cache_args(name, key_cache, value_cache, cache_strides, key_scales, value_scales, scale_strides, write_blocks,
                          write_offsets, n_rows, layer, num_layers, num_blocks, page_size, num_kv_heads, head_dim, dtype))
    return rc;
  if (n_rows == 0) return RLT_OK;
  if (!k || !k_strides || !v || !v_strides) return fail(RLT_EINVAL, "%s: NULL pointer argument", name);
  AppendI8Args a{};
  a.x[0] = k, a.x_row[0] = k_strides[0], a.x_head[0] = k_strides[1], a.x_dim[0] = k_strides[2];
  a.x[1] = v, a.x_row[1] = v_strides[0], a.x_head[1] = v_strides[1], a.x_dim[1] = v_strides[2];
  a.codes[0] = static_cast<uint8_t*>(key_cache), a.codes[1] = static_cast<uint8_t*>(value_cache);
  a.c_block = cache_strides[0], a.c_layer = cache_strides[1], a.c_token = cache_strides[2];
  a.c_head = cache_strides[3], a.c_dim = cache_strides[4];
  a.scales[0] = static_cast<float*>(key_scales), a.scales[1] = static_cast<float*>(value_scales);
  a.s_block = scale_strides[0], a.s_layer = scale_strides[1], a.s_head = scale_strides[2];
  a.blocks = write_blocks, a.offsets = write_offsets;
  a.rows = n_rows, a.layer = layer, a.num_blocks = num_blocks, a.page = page_size;
  a.hkv = static_cast<int>(num_kv_heads), a.d = static_cast<int>(head_dim);
  switch (dtype) {
    case RLT_BFLOAT16: launch_append<bf16>(a, as_stream(stream)); break;
    case RLT_FLOAT16: launch_append<f16>(a, as_stream(stream)); break;
    default: launch_append<float>(a, as_stream(stream)); break;
  }
  return check_launch(name);
}

extern "C" int rlt_kv_gather_int8(const void* key_cache, const void* value_cache, const int64_t* cache_strides,
                                  const void* key_scales, const void* value_scales, const int64_t* scale_strides,
                                  const int64_t* blocks, const int64_t* offsets, int64_t n_rows, void* out_k, void* out_v,
                                  int64_t layer, int64_t num_layers, int64_t num_blocks, int64_t page_size,
                                  int64_t num_kv_heads, int64_t head_dim, int dtype, void* stream) {
  const char* name = "rlt_kv_gather_int8";
  if (int rc = cache_args(name, key_cache, value_cache, cache_strides, key_scales, value_scales, scale_strides, blocks, offsets,
                          n_rows, layer, num_layers, num_blocks, page_size, num_kv_heads, head_dim, dtype))
    return rc;
  if (n_rows == 0) return RLT_OK;
  if (!out_k || !out_v) return fail(RLT_EINVAL, "%s: NULL pointer argument", name);
  GatherI8Args a{};
  a.codes[0] = static_cast<const uint8_t*>(key_cache), a.codes[1] = static_cast<const uint8_t*>(value_cache);
  a.c_block = cache_strides[0], a.c_layer = cache_strides[1], a.c_token = cache_strides[2];
  a.c_head = cache_strides[3], a.c_dim = cache_strides[4];
  a.scales[0] = static_cast<const float*>(key_scales), a.scales[1] = static_cast<const float*>(value_scales);
  a.s_block = scale_strides[0], a.s_layer = scale_strides[1], a.s_head = scale_strides[2];
  a.blocks = blocks, a.offsets = offsets;
  a.out[0] = out_k, a.out[1] = out_v;
  a.rows = n_rows, a.layer = layer, a.num_blocks = num_blocks, a.page = page_size;
  a.hkv = static_cast<int>(num_kv_heads), a.d = static_cast<int>(head_dim);
  switch (dtype) {
    case RLT_BFLOAT16: launch_gather<bf16>(a, as_stream(stream)); break;
    case RLT_FLOAT16: launch_gather<f16>(a, as_stream(stream)); break;
    default: launch_gather<float>(a, as_stream(stream)); break;
  }
  return check_launch(name);
}
