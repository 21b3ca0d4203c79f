// Key tiles in LDS for attention on 32x32 MFMAs: copies, swizzles and operand
// reads, shared by the prefill attention (prefill.hip) and the decode over shared
// prefixes (paged_shared.hip).
#pragma once

#include "common.h"

namespace lfs {
namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;

constexpr int KT = 64;               // keys per tile
constexpr int NW = 4;                // waves per workgroup
constexpr int RW = 32;               // rows (query token, head) per wave
// N copies of 16 bytes per lane, from base + off[c] (per lane) to LDS address
// lds + 1024 c + 16 * lane.  The kernel waits for them before its barrier
// (the compiler does not see that they write LDS).  m0 is kept for the
// compiler; an LDS copy may not be the instruction after a write of m0.
template <int N>
__device__ __forceinline__ void copy_rows(const uint8_t* base, const unsigned (&off)[N], unsigned lds) {
  const uint64_t b = (uint64_t)(uintptr_t)base;
  i32x4 rsrc;
  rsrc[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)b);
  rsrc[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32)) & 0xFFFF;
  rsrc[2] = -1;
  rsrc[3] = 0x00020000;
  const unsigned dst = __builtin_amdgcn_readfirstlane(lds);
  unsigned keep;
  if constexpr (N == 2) {
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %4, 0 offen lds\n\t"
                 "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %4, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "s"(dst), "v"(off[0]), "v"(off[1]), "s"(rsrc) : "memory", "scc");
  } else {
    static_assert(N == 4, "2 or 4 copies per wave");
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %6, 0 offen lds\n\t"
                 "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %6, 0 offen lds\n\t"
                 "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tbuffer_load_dwordx4 %4, %6, 0 offen lds\n\t"
                 "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tbuffer_load_dwordx4 %5, %6, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "s"(dst), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(rsrc)
                 : "memory", "scc");
  }
}
__device__ __forceinline__ u32x4 lds_read16(unsigned a) {
  return *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)a;
}
__device__ __forceinline__ void lds_write8(unsigned a, uint2 v) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  *(__attribute__((address_space(3))) u32x2*)(uintptr_t)a = u32x2{v.x, v.y};
}
__device__ __forceinline__ uint2 lds_read_tr(unsigned a) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) v4s*)(uintptr_t)a));
}

// 16-byte chunk c of key row r of a tile sits in chunk slot c ^ f(r).  K: the
// sixteen rows of an operand read (one chunk index) touch every bank once.
// V: the four rows of a transposed read (64 bytes each for 32 lanes) do.
template <int D>
__device__ __forceinline__ int kswz(int r) {
  return D == 64 ? (((r >> 1) & 7) ^ ((r & 1) << 2)) : (r & 15);
}
template <int D>
__device__ __forceinline__ int vswz(int r) {
  return D == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2;
}

// x / v.d for x < 2^31, by the reciprocal that div_by() rounded up: the product's
// high word is the quotient or one more.
struct Div {
  unsigned d, inv;
};
inline Div div_by(unsigned d) { return Div{d, d == 1 ? 0u : (unsigned)((0xFFFFFFFFull + d) / d)}; }
__device__ __forceinline__ unsigned operator/(unsigned x, Div v) {
  const unsigned q = v.inv != 0 ? __umulhi(x, v.inv) : x;
  return q * v.d > x ? q - 1 : q;
}

}  // namespace
}  // namespace lfs
