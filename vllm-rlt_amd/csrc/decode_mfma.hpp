// Building blocks of decode over an 8-bit cache on the matrix cores, whatever the form of
// its scales: the split pass's workgroups, its direct loads into LDS and their places there.
#pragma once

#include <type_traits>

#include "decode_fp8.hpp"
#include "mfma.hpp"

namespace rlt {

constexpr int kDecodeWaves = 4;
constexpr int kDecodeXcds = 8;
constexpr int kDecodeTile = 32;

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

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
// The same, of bytes that stay in the L2: others read the rest of their lines.
__device__ __forceinline__ void dma16_kept(uint32_t lds_byte, uint32_t offset, const uint8_t* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_byte), "v"(offset), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void dma_byte(uint32_t lds_byte, const uint8_t* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off" ::"s"(lds_byte), "v"(from) : "memory", "m0");
}
__device__ __forceinline__ void dma_dword(uint32_t lds_byte, const float* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds_byte), "v"(from) : "memory", "m0");
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

}  // namespace rlt
