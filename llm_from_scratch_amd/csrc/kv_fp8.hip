// Writes to and reads from a KV pool in 8 bits.
//
// The pool holds e4m3fn codes [NB, BS, Hkv, D] and a fp32 scale per token and
// kv head: s = max(amax, 1e-4) / 448 over the head's D values (act_quant's
// formula with a group of D), code = e4m3(x / s).  The scales lie as
// [NB, Hkv, BS]: a head's scales of a block's tokens follow each other, so a
// decode tile reads its tokens' scales as one run.
//
//  store  D / 8 lanes per (token, K or V, kv head): one 16-byte load, the
//         group's amax by an xor butterfly, one 8-byte store.  Bound: HBM, 2 D
//         bytes in and D + 4 out a row.
//  load   8 values a thread of the same rows back as bf16(code * s), through
//         the block tables.  Bound: HBM, D + 4 bytes in and 2 D out a row.
#include "common.h"

namespace lfs {
namespace {

template <int D, bool VEC>
__global__ __launch_bounds__(256) void store_kvcache_fp8_kernel(
    const uint16_t* __restrict__ key, int64_t ks, const uint16_t* __restrict__ value, int64_t vs,
    uint8_t* __restrict__ kc, uint8_t* __restrict__ vc, float* __restrict__ ksc, float* __restrict__ vsc,
    const int64_t* __restrict__ slots, int64_t rows, int Hkv, int BS, int64_t num_slots) {
  constexpr int LPR = D / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / LPR;  // (token, K or V, kv head)
  const int c = (int)(i % LPR);
  if (row >= rows) return;  // a row's lanes all in or all out
  const int64_t t = row / (2 * Hkv);
  const int r = (int)(row - t * 2 * Hkv), h = r < Hkv ? r : r - Hkv;
  const int64_t slot = slots[t];
  if (slot < 0 || slot >= num_slots) return;
  const uint16_t* src = (r < Hkv ? key + t * ks : value + t * vs) + h * D + c * 8;
  uint4 w;
  if constexpr (VEC) {
    w = *reinterpret_cast<const uint4*>(src);
  } else {
    uint32_t p[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] = (uint32_t)src[2 * e] | (uint32_t)src[2 * e + 1] << 16;
    w = make_uint4(p[0], p[1], p[2], p[3]);
  }
  float f[8], amax = 0.f;
  unpack8(w, f);
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(f[e]));
  amax = group_max<LPR>(amax);
  const float s = scale_from_amax(amax, false);
  *reinterpret_cast<uint2*>((r < Hkv ? kc : vc) + (slot * Hkv + h) * D + c * 8) = quant8(f, s);
  if (c == 0) {
    const int64_t blk = slot / BS;
    (r < Hkv ? ksc : vsc)[(blk * Hkv + h) * BS + (slot - blk * BS)] = s;
  }
}

template <int D>
__global__ __launch_bounds__(256) void load_kvcache_fp8_kernel(
    const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc, const float* __restrict__ ksc,
    const float* __restrict__ vsc, const int32_t* __restrict__ bt, int64_t bt_stride, int max_blocks,
    const int32_t* __restrict__ cu, int B, int64_t total, uint16_t* __restrict__ k, uint16_t* __restrict__ v, int Hkv,
    int BS, int64_t NB) {
  constexpr int LPR = D / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = i / (LPR * Hkv);
  const int c = (int)(i - t * LPR * Hkv), h = c / LPR;
  if (t >= total) return;
  int lo = 0, hi = B;  // the last sequence that begins at or before row t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  int64_t blk = -1;
  int off = 0;
  if (B > 0 && t >= cu[lo] && t < cu[lo + 1]) {
    const int64_t pos = t - cu[lo], col = pos / BS;
    off = (int)(pos - col * BS);
    if (col < max_blocks) blk = bt[lo * bt_stride + col];
  }
  uint4 ko = make_uint4(0, 0, 0, 0), vo = ko;
  if (blk >= 0 && blk < NB) {
    const int64_t at = (blk * BS + off) * Hkv * D + c * 8, sat = (blk * Hkv + h) * BS + off;
    const uint2 kw = *reinterpret_cast<const uint2*>(kc + at), vw = *reinterpret_cast<const uint2*>(vc + at);
    const float a = ksc[sat], b = vsc[sat];
    float f[8];
    e4m3x4_to_f32(kw.x, f), e4m3x4_to_f32(kw.y, f + 4);
    ko = make_uint4(pack_bf16x2(f[0] * a, f[1] * a), pack_bf16x2(f[2] * a, f[3] * a),
                    pack_bf16x2(f[4] * a, f[5] * a), pack_bf16x2(f[6] * a, f[7] * a));
    e4m3x4_to_f32(vw.x, f), e4m3x4_to_f32(vw.y, f + 4);
    vo = make_uint4(pack_bf16x2(f[0] * b, f[1] * b), pack_bf16x2(f[2] * b, f[3] * b),
                    pack_bf16x2(f[4] * b, f[5] * b), pack_bf16x2(f[6] * b, f[7] * b));
  }
  *reinterpret_cast<uint4*>(k + (t * Hkv * LPR + c) * 8) = ko;
  *reinterpret_cast<uint4*>(v + (t * Hkv * LPR + c) * 8) = vo;
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
  const int64_t rows = T * 2 * Hkv, wgs = (rows * (D / 8) + 255) / 256;
#define LFS_STORE(DD, VEC)                                                                                            \
  hipLaunchKernelGGL((store_kvcache_fp8_kernel<DD, VEC>), dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream,     \
                     (const uint16_t*)key, k_stride_t, (const uint16_t*)value, v_stride_t, (uint8_t*)k_cache,         \
                     (uint8_t*)v_cache, k_scale, v_scale, slot_mapping, rows, Hkv, BS, num_blocks * BS)
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
  const int64_t wgs = (total * Hkv * (D / 8) + 255) / 256;
#define LFS_LOAD(DD)                                                                                                  \
  hipLaunchKernelGGL((load_kvcache_fp8_kernel<DD>), dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream,           \
                     (const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, block_tables, bt_stride,     \
                     max_blocks, cu_seqlens, (int)B, total, (uint16_t*)k, (uint16_t*)v, Hkv, BS, num_blocks)
  if (D == 64) LFS_LOAD(64);
  else LFS_LOAD(128);
#undef LFS_LOAD
  return check_launch("load_kvcache_fp8");
}
