// Writes to and reads from a KV pool in 8 bits.
//
// The pool holds e4m3fn codes [NB, BS, Hkv, D] and a fp32 scale per token and
// kv head: s = max(amax, 1e-4) / 448 over the head's D values (act_quant's
// formula with a group of D), code = e4m3(x / s).  The scales lie as
// [NB, Hkv, BS]: a head's scales of a block's tokens follow each other, so a
// decode tile reads its tokens' scales as one run.
//
//  store  D / 8 lanes per (token, K or V, kv head): one 16-byte load, the row's
//         amax by an xor butterfly, one 8-byte store.  A workgroup takes tok
//         tokens and writes their scales last, through LDS, a run of tokens a
//         head.  Bound: HBM, 2 D bytes in and D + 4 out a row: 16383 tokens of 8
//         heads of 128 in 22.6 us, 4.5 TB/s.
//  load   8 values a thread and piece of the same rows back as bf16(code * s).  A
//         workgroup takes 16 rows of the result, whose slots its first threads
//         find (the sequence by a binary search, its block by the table).  Bound: HBM, D + 4
//         bytes in and 2 D out a row: 8 sequences of 4000 to 16384 tokens, 8 heads
//         of 128, blocks of 16 in 93 us, 5.4 TB/s (with 16 values a thread, whose
//         stores are half lines, 116).
#include <algorithm>

#include "tile32.h"

namespace lfs {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
constexpr int SU = 4;  // rows in flight per thread of a store
constexpr int MAX_ROWS = 1024;  // (K or V, head) rows of a workgroup
constexpr int64_t MAX_WGS = (1 << 24) - 1;  // of 256 threads: a launch takes less than 2^32

template <int D, bool VEC>
__global__ __launch_bounds__(256) void store_kvcache_fp8_kernel(
    const uint16_t* __restrict__ key, int64_t ks, const uint16_t* __restrict__ value, int64_t vs,
    uint8_t* __restrict__ kc, uint8_t* __restrict__ vc, float* __restrict__ ksc, float* __restrict__ vsc,
    const int64_t* __restrict__ slots, int64_t T, int tok, int Hkv, Div rows_tok, Div dBS, int64_t num_slots) {
  constexpr int LPR = D / 8;
  __shared__ float sc[MAX_ROWS];  // [token][K or V, head]
  const int64_t t0 = (int64_t)blockIdx.x * tok;
  const int nt = (int)min((int64_t)tok, T - t0), rows = nt * (int)rows_tok.d;
  const int c = threadIdx.x % LPR;
  for (int i0 = threadIdx.x / LPR; i0 < rows; i0 += SU * 256 / LPR) {
    uint4 w[SU];
    int64_t slot[SU];
    int hd[SU];
#pragma unroll
    for (int u = 0; u < SU; ++u) {
      const int i = i0 + u * (256 / LPR);
      if (i >= rows) break;
      const int t = (unsigned)i / rows_tok, r = i - t * (int)rows_tok.d;  // K's heads, then V's
      hd[u] = r;
      slot[u] = slots[t0 + t];
      const uint16_t* src = (r < Hkv ? key + (t0 + t) * ks + r * D : value + (t0 + t) * vs + (r - Hkv) * D) + c * 8;
      if constexpr (VEC) {
        const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src));
        w[u] = make_uint4(x[0], x[1], x[2], x[3]);
      } else {
        __builtin_memcpy(&w[u], src, 16);
      }
    }
#pragma unroll
    for (int u = 0; u < SU; ++u) {
      const int i = i0 + u * (256 / LPR);
      if (i >= rows) break;  // a row's lanes all in or all out
      float f[8], amax = 0.f;
      unpack8(w[u], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(f[e]));
      amax = group_max<LPR>(amax);
      const float s = scale_from_amax(amax, false);
      if (c == 0) sc[i] = s;
      if (slot[u] >= 0 && slot[u] < num_slots) {
        const int h = hd[u] < Hkv ? hd[u] : hd[u] - Hkv;
        const uint2 q = quant8(f, s);
        __builtin_nontemporal_store(
            u32x2{q.x, q.y}, reinterpret_cast<u32x2*>((hd[u] < Hkv ? kc : vc) + (slot[u] * Hkv + h) * D + c * 8));
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows; i += 256) {
    const int r = i / nt, t = i - r * nt;
    const int64_t slot = slots[t0 + t];
    if (slot < 0 || slot >= num_slots) continue;
    const int h = r < Hkv ? r : r - Hkv;
    const int64_t blk = slot >> 31 ? slot / (int64_t)dBS.d : (int64_t)((unsigned)slot / dBS);
    (r < Hkv ? ksc : vsc)[(blk * Hkv + h) * (int)dBS.d + (slot - blk * dBS.d)] = sc[t * (int)rows_tok.d + r];
  }
}

constexpr int LT = 16;  // rows of the result a workgroup of a load takes
constexpr int LU = 8;   // pieces in flight per thread

__device__ __forceinline__ u32x4 values8(const u32x2& w, float s) {
  float f[8];
  e4m3x4_to_f32(w[0], f), e4m3x4_to_f32(w[1], f + 4);
  return u32x4{pack_bf16x2(f[0] * s, f[1] * s), pack_bf16x2(f[2] * s, f[3] * s), pack_bf16x2(f[4] * s, f[5] * s),
               pack_bf16x2(f[6] * s, f[7] * s)};
}

template <int D>
__global__ __launch_bounds__(256) void load_kvcache_fp8_kernel(
    const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc, const float* __restrict__ ksc,
    const float* __restrict__ vsc, const int32_t* __restrict__ bt, int64_t bt_stride, int max_blocks,
    const int32_t* __restrict__ cu, int B, int64_t total, uint16_t* __restrict__ k, uint16_t* __restrict__ v, int Hkv,
    Div pieces, int BS, int64_t NB) {
  constexpr int LPR = D / 8;
  __shared__ int64_t block[LT];  // of a row, -1: none
  __shared__ int offset[LT];
  const int64_t t0 = (int64_t)blockIdx.x * LT;
  const int nt = (int)min((int64_t)LT, total - t0);
  if (threadIdx.x < nt) {
    const int64_t t = t0 + threadIdx.x;
    int lo = 0, hi = B;  // the last sequence that begins at or before row t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid] <= t) lo = mid;
      else hi = mid;
    }
    int64_t blk = -1;
    int off = 0;
    if (B > 0 && t >= cu[lo] && t < cu[lo + 1]) {
      const unsigned pos = (unsigned)(t - cu[lo]), col = pos / (unsigned)BS;
      off = (int)(pos - col * BS);
      if (col < (unsigned)max_blocks) blk = bt[lo * bt_stride + col];
    }
    block[threadIdx.x] = blk >= 0 && blk < NB ? blk : -1;
    offset[threadIdx.x] = off;
  }
  __syncthreads();
  const int n = nt * (int)pieces.d;  // pieces: 8 values each, Hkv * D / 8 a row
  for (int i0 = threadIdx.x; i0 < n; i0 += LU * 256) {
    u32x2 kw[LU], vw[LU];
    float a[LU], b[LU];
#pragma unroll
    for (int u = 0; u < LU; ++u) {
      const int i = i0 + u * 256;
      if (i >= n) break;
      const int t = (unsigned)i / pieces, c = i - t * (int)pieces.d, h = c / LPR;
      const int64_t blk = block[t];
      a[u] = b[u] = 0.f;
      kw[u] = vw[u] = u32x2{0, 0};
      if (blk >= 0) {
        const int64_t at = (blk * BS + offset[t]) * Hkv * D + c * 8, sat = (blk * Hkv + h) * BS + offset[t];
        kw[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(kc + at));
        vw[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(vc + at));
        a[u] = ksc[sat], b[u] = vsc[sat];
      }
    }
#pragma unroll
    for (int u = 0; u < LU; ++u) {
      const int i = i0 + u * 256;
      if (i >= n) break;
      const int64_t to = (t0 * (int)pieces.d + i) * 8;
      __builtin_nontemporal_store(values8(kw[u], a[u]), reinterpret_cast<u32x4*>(k + to));
      __builtin_nontemporal_store(values8(vw[u], b[u]), reinterpret_cast<u32x4*>(v + to));
    }
  }
}

}  // namespace
}  // namespace lfs

using namespace lfs;

extern "C" int lfs_store_kvcache_fp8(const void* key, int64_t k_stride_t, const void* value, int64_t v_stride_t,
                                     void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                                     const int64_t* slot_mapping, int64_t T, int32_t num_kv_heads, int32_t head_dim,
                                     int32_t block_size, int64_t num_blocks, void* stream) {
  const int Hkv = num_kv_heads, D = head_dim, BS = block_size;
  LFS_REQUIRE(T >= 0 && Hkv > 0 && BS > 0 && num_blocks >= 0, "store_kvcache_fp8: bad shape T=%lld Hkv=%d BS=%d",
              (long long)T, Hkv, BS);
  LFS_REQUIRE(D == 64 || D == 128, "store_kvcache_fp8: head_dim must be 64 or 128 (got %d)", D);
  if (T == 0) return 0;
  LFS_REQUIRE(key && value && slot_mapping, "store_kvcache_fp8: null pointer");
  LFS_REQUIRE(num_blocks == 0 || (k_cache && v_cache && k_scale && v_scale), "store_kvcache_fp8: null pointer");
  LFS_REQUIRE(((((uintptr_t)k_cache) | ((uintptr_t)v_cache)) & 7u) == 0,
              "store_kvcache_fp8: the caches must be 8-byte aligned");
  LFS_REQUIRE(T < (1ll << 31) / Hkv / 2, "store_kvcache_fp8: too many tokens");
  const bool vec = k_stride_t % 8 == 0 && v_stride_t % 8 == 0 && ((((uintptr_t)key) | ((uintptr_t)value)) & 15u) == 0;
  LFS_REQUIRE(Hkv <= MAX_ROWS / 2, "store_kvcache_fp8: at most %d kv heads (got %d)", MAX_ROWS / 2, Hkv);
  // Tokens a workgroup: as many as give its threads four pieces each where that
  // makes some hundreds of workgroups, else one each: one piece / four, us a call in
  // a graph: 4 heads of 64, 16 tokens 2.7 / 3.7, 4096 3.9 / 4.5, 16383 8.7 / 7.6; 8
  // of 128, 16 2.7 / 3.8, 2048 5.0 / 5.3, 4096 8.4 / 7.3, 16383 27.0 / 22.8.
  const int pieces = 2 * Hkv * (D / 8);
  int tok = std::max(1, std::min(16, 1024 / pieces));
  if (T < (int64_t)640 * tok) tok = std::max(1, std::min(16, 256 / pieces));
  const int64_t wgs = (T + tok - 1) / tok;
  LFS_REQUIRE(wgs <= MAX_WGS, "store_kvcache_fp8: too many tokens");
#define LFS_STORE(DD, VEC)                                                                                            \
  hipLaunchKernelGGL((store_kvcache_fp8_kernel<DD, VEC>), dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream,     \
                     (const uint16_t*)key, k_stride_t, (const uint16_t*)value, v_stride_t, (uint8_t*)k_cache,         \
                     (uint8_t*)v_cache, k_scale, v_scale, slot_mapping, T, tok, Hkv, div_by(2 * Hkv), div_by(BS),     \
                     num_blocks * BS)
  if (D == 64 && vec) LFS_STORE(64, true);
  else if (D == 64) LFS_STORE(64, false);
  else if (vec) LFS_STORE(128, true);
  else LFS_STORE(128, false);
#undef LFS_STORE
  return check_launch("store_kvcache_fp8");
}

extern "C" int lfs_load_kvcache_fp8(const void* k_cache, const void* v_cache, const float* k_scale,
                                    const float* v_scale, const int32_t* block_tables, int64_t bt_stride,
                                    int32_t max_blocks, const int32_t* cu_seqlens, int64_t B, int64_t total, void* k,
                                    void* v, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                    int64_t num_blocks, void* stream) {
  const int Hkv = num_kv_heads, D = head_dim, BS = block_size;
  LFS_REQUIRE(B >= 0 && B < (1ll << 31) && total >= 0 && Hkv > 0 && BS > 0 && num_blocks >= 0 && max_blocks >= 0,
              "load_kvcache_fp8: bad shape");
  LFS_REQUIRE(D == 64 || D == 128, "load_kvcache_fp8: head_dim must be 64 or 128 (got %d)", D);
  LFS_REQUIRE(bt_stride >= max_blocks, "load_kvcache_fp8: block table stride < max_blocks");
  LFS_REQUIRE(total < (1ll << 31) / Hkv, "load_kvcache_fp8: too many rows");
  if (total == 0) return 0;
  LFS_REQUIRE(cu_seqlens && k && v, "load_kvcache_fp8: null pointer");
  LFS_REQUIRE(B == 0 || max_blocks == 0 || block_tables, "load_kvcache_fp8: null block table");
  LFS_REQUIRE(num_blocks == 0 || (k_cache && v_cache && k_scale && v_scale), "load_kvcache_fp8: null pointer");
  LFS_REQUIRE(((((uintptr_t)k_cache) | ((uintptr_t)v_cache) | ((uintptr_t)k) | ((uintptr_t)v)) & 15u) == 0,
              "load_kvcache_fp8: caches, k and v must be 16-byte aligned");
  LFS_REQUIRE(Hkv <= 65536, "load_kvcache_fp8: too many kv heads (%d)", Hkv);
  const int64_t wgs = (total + LT - 1) / LT;
  LFS_REQUIRE(wgs <= MAX_WGS, "load_kvcache_fp8: too many rows");
#define LFS_LOAD(DD)                                                                                                  \
  hipLaunchKernelGGL((load_kvcache_fp8_kernel<DD>), dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream,           \
                     (const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, block_tables, bt_stride,     \
                     max_blocks, cu_seqlens, (int)B, total, (uint16_t*)k, (uint16_t*)v, Hkv, div_by(Hkv * DD / 8),   \
                     BS, num_blocks)
  if (D == 64) LFS_LOAD(64);
  else LFS_LOAD(128);
#undef LFS_LOAD
  return check_launch("load_kvcache_fp8");
}
