// RMSNorm of every query and key head by itself, the rotation by position and
// the KV slot write, one launch.  For head x of D values of a token at
// position p, with weight w [D]:
//   y = w * x * rsqrt(mean(x^2) + eps)
//   for d < R / 2:  z[d]         = y[d] cos[p][d] - y[d + R/2] sin[p][d]
//                   z[d + R / 2] = y[d + R/2] cos[p][d] + y[d] sin[p][d]
//   z[d] = y[d] for d >= R,
// all in fp32 and rounded to bf16 once.  Values are copied.
//
// A lane owns one 16-byte chunk of a head, D / 8 neighbouring lanes a head:
// the sum of squares and the rotation's other half are exchanges within them,
// so no LDS and no barrier.  Bound: HBM, each byte read and written once.
#include "common.h"

#include <algorithm>

namespace lfs {
namespace {

template <int D>
__global__ __launch_bounds__(256) void qk_head_norm_rope_store_kernel(
    const uint16_t* __restrict__ qkv, int64_t ld, const float* __restrict__ qw, const float* __restrict__ kw,
    const float* __restrict__ cos_sin, int R, const int64_t* __restrict__ pos, const int64_t* __restrict__ slots,
    uint16_t* __restrict__ q_out, uint16_t* __restrict__ kc, uint16_t* __restrict__ vc, uint16_t* __restrict__ k_out,
    uint16_t* __restrict__ v_out, int64_t T, int Hq, int Hkv, int64_t num_slots, int64_t max_pos, float eps) {
  constexpr int C = D / 8;  // lanes of a head
  const int heads = Hq + 2 * Hkv, c = threadIdx.x % C, r2 = R / 16;  // r2: chunks of half the rotated dims
  const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / C;
  if (unit >= T * heads) return;  // whole heads: the exchanges below stay among live lanes
  const int64_t t = unit / heads;
  const int h = (int)(unit - t * heads);
  const uint4 x = *reinterpret_cast<const uint4*>(qkv + t * ld + h * D + 8 * c);
  const int64_t slot = h >= Hq && slots != nullptr ? slots[t] : -1;
  const bool store = slot >= 0 && slot < num_slots;
  if (h >= Hq + Hkv) {
    const int64_t e = (int64_t)(h - Hq - Hkv) * D + 8 * c;
    if (store) *reinterpret_cast<uint4*>(vc + slot * Hkv * D + e) = x;
    if (v_out != nullptr) *reinterpret_cast<uint4*>(v_out + t * Hkv * D + e) = x;
    return;
  }
  float f[8], y[8], other[8];
  unpack8(x, f);
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
  const float inv = rsqrtf(group_sum<C>(ss) * (1.0f / D) + eps);
  const float* w = (h < Hq ? qw : kw) + 8 * c;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = f[e] * inv * w[e];
  const bool low = c < r2, turned = c < 2 * r2;
  const int src = (threadIdx.x & 63) + (low ? r2 : turned ? -r2 : 0);
#pragma unroll
  for (int e = 0; e < 8; ++e) other[e] = __shfl(y[e], src, 64);
  if (turned) {
    int64_t p = pos[t];
    p = p < 0 ? 0 : (p >= max_pos ? max_pos - 1 : p);
    const float* cs = cos_sin + p * R + 8 * (low ? c : c - r2);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float s = cs[R / 2 + e];
      y[e] = fmaf(y[e], cs[e], low ? -other[e] * s : other[e] * s);
    }
  }
  const uint4 z = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                             pack_bf16x2(y[6], y[7]));
  if (h < Hq) {
    *reinterpret_cast<uint4*>(q_out + (t * Hq + h) * D + 8 * c) = z;
  } else {
    const int64_t e = (int64_t)(h - Hq) * D + 8 * c;
    if (store) *reinterpret_cast<uint4*>(kc + slot * Hkv * D + e) = z;
    if (k_out != nullptr) *reinterpret_cast<uint4*>(k_out + t * Hkv * D + e) = z;
  }
}

}  // namespace
}  // namespace lfs

using namespace lfs;

extern "C" int lfs_qk_head_norm_rope_store(const void* qkv, int64_t ld, const float* q_weight, const float* k_weight,
                                           const float* cos_sin, int32_t rotary_dim, const int64_t* positions,
                                           const int64_t* slot_mapping, void* q_out, void* k_cache, void* v_cache,
                                           void* k_out, void* v_out, int64_t T, int32_t num_q_heads,
                                           int32_t num_kv_heads, int32_t head_dim, int64_t num_slots,
                                           int64_t max_positions, float eps, void* stream) {
  const int Hq = num_q_heads, Hkv = num_kv_heads, D = head_dim, R = rotary_dim;
  LFS_REQUIRE(T >= 0 && Hq > 0 && Hkv > 0 && num_slots >= 0, "qk_head_norm_rope_store: bad shape");
  LFS_REQUIRE(D == 64 || D == 128, "qk_head_norm_rope_store: head_dim must be 64 or 128 (got %d)", D);
  LFS_REQUIRE(R > 0 && R <= D && R % 16 == 0,
              "qk_head_norm_rope_store: rotary_dim must be a multiple of 16, at most head_dim (got %d)", R);
  LFS_REQUIRE(ld >= (int64_t)(Hq + 2 * (int64_t)Hkv) * D && ld % 8 == 0, "qk_head_norm_rope_store: bad row stride");
  LFS_REQUIRE(max_positions > 0, "qk_head_norm_rope_store: empty rotation table");
  if (T == 0) return 0;
  LFS_REQUIRE(qkv && q_weight && k_weight && cos_sin && positions && q_out, "qk_head_norm_rope_store: null pointer");
  LFS_REQUIRE(slot_mapping == nullptr || (k_cache && v_cache), "qk_head_norm_rope_store: null cache");
  LFS_REQUIRE((k_out == nullptr) == (v_out == nullptr), "qk_head_norm_rope_store: k_out and v_out go together");
  LFS_REQUIRE(((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)k_out |
               (uintptr_t)v_out) % 16 == 0,
              "qk_head_norm_rope_store: buffers must be 16-byte aligned");
  const int64_t heads = Hq + 2 * (int64_t)Hkv;
  LFS_REQUIRE(T < ((1ll << 32) - 256) / (D / 8) / heads, "qk_head_norm_rope_store: too many tokens");
  const int64_t wgs = (T * heads * (D / 8) + 255) / 256;
#define LFS_HN(DD)                                                                                                   \
  hipLaunchKernelGGL(qk_head_norm_rope_store_kernel<DD>, dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream,      \
                     (const uint16_t*)qkv, ld, q_weight, k_weight, cos_sin, R, positions, slot_mapping,              \
                     (uint16_t*)q_out, (uint16_t*)k_cache, (uint16_t*)v_cache, (uint16_t*)k_out, (uint16_t*)v_out, T, \
                     Hq, Hkv, num_slots, max_positions, eps)
  if (D == 64) LFS_HN(64);
  else LFS_HN(128);
#undef LFS_HN
  return check_launch("qk_head_norm_rope_store");
}
