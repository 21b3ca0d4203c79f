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
// so no LDS and no barrier.  Few tokens have a thread per chunk, many a wave
// per token (kHeadRowsT).  Bound: HBM, each byte read and written once: 16383
// tokens of 32 / 8 heads of 128 take 73 us, 5.5 TB/s; 128 tokens 3 us, the
// launch and three dependent loads.
#include "common.h"

#include <algorithm>

namespace lfs {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The call's pointers and sizes.
struct HeadNorm {
  const uint16_t* qkv;
  int64_t ld;
  const float *qw, *kw, *cos_sin;
  const int64_t *pos, *slots;
  uint16_t *q_out, *kc, *vc, *k_out, *v_out;
  int64_t num_slots, max_pos;
  float eps;
  int R, Hq, Hkv;
  unsigned T;
};

// What a lane's chunk c of any head of a token needs besides the chunk.
template <int D>
struct Turn {
  static constexpr int C = D / 8;  // lanes of a head
  float w[2][8], cs[8], sn[8];     // of q and k; sn has the sign of its product
  int src;                         // the lane with the other half's chunk
  bool turned;

  __device__ __forceinline__ static void load8(const float* p, float* f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = p[e];
  }
  __device__ __forceinline__ void load_weights(const HeadNorm& a, int c) {
    load8(a.qw + 8 * c, w[0]);
    load8(a.kw + 8 * c, w[1]);
  }
  __device__ __forceinline__ void load_row(const HeadNorm& a, int c, int64_t t) {
    const int r2 = a.R / 16;  // chunks of half the rotated dims
    const bool low = c < r2;
    turned = c < 2 * r2;
    src = (int)(threadIdx.x & 63) + (low ? r2 : turned ? -r2 : 0);
    if (!turned) return;
    int64_t p = a.pos[t];
    p = p < 0 ? 0 : (p >= a.max_pos ? a.max_pos - 1 : p);
    const float* row = a.cos_sin + p * a.R + 8 * (low ? c : c - r2);
    load8(row, cs);
    load8(row + a.R / 2, sn);
#pragma unroll
    for (int e = 0; e < 8; ++e) sn[e] = low ? -sn[e] : sn[e];
  }
  // the chunk of a head of q (k: isk): every lane of the head calls it
  __device__ __forceinline__ u32x4 head(const u32x4& x, bool isk, float eps) const {
    float f[8], y[8], other[8], ss = 0.f;
    unpack8(make_uint4(x[0], x[1], x[2], x[3]), f);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
    const float inv = rsqrtf(group_sum<C>(ss) * (1.0f / D) + eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = f[e] * inv * (isk ? w[1][e] : w[0][e]);
#pragma unroll
    for (int e = 0; e < 8; ++e) other[e] = __shfl(y[e], src, 64);
    if (turned) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = fmaf(y[e], cs[e], other[e] * sn[e]);
    }
    return u32x4{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7])};
  }
};

template <bool NT>
__device__ __forceinline__ void put(uint16_t* p, const u32x4& x) {
  if constexpr (NT) __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(p));
  else *reinterpret_cast<u32x4*>(p) = x;
}
// chunk c of head h (q, k, v heads in turn) of token t, as it leaves
template <int D, bool NT>
__device__ __forceinline__ void store_head(const HeadNorm& a, int64_t t, int h, int c, int64_t slot, const u32x4& x) {
  if (h < a.Hq) {
    put<NT>(a.q_out + (t * a.Hq + h) * D + 8 * c, x);
    return;
  }
  const bool isv = h >= a.Hq + a.Hkv;
  const int64_t e = (int64_t)(h - a.Hq - (isv ? a.Hkv : 0)) * D + 8 * c;
  if (slot >= 0 && slot < a.num_slots) put<NT>((isv ? a.vc : a.kc) + slot * a.Hkv * D + e, x);
  if (a.k_out != nullptr) put<NT>((isv ? a.v_out : a.k_out) + t * a.Hkv * D + e, x);
}

// Few tokens: D / 8 lanes per (token, head).
template <int D>
__global__ __launch_bounds__(256) void qk_head_norm_rope_store_kernel(HeadNorm a) {
  constexpr int C = D / 8;
  const unsigned heads = a.Hq + 2 * a.Hkv, unit = blockIdx.x * (256 / C) + threadIdx.x / C, t = unit / heads;
  const int c = threadIdx.x % C, h = (int)(unit - t * heads);
  if (t >= a.T) return;  // whole heads: the exchanges stay among live lanes
  u32x4 x = *reinterpret_cast<const u32x4*>(a.qkv + t * a.ld + h * D + 8 * c);
  const int64_t slot = h >= a.Hq && a.slots != nullptr ? a.slots[t] : -1;
  if (h < a.Hq + a.Hkv) {
    Turn<D> turn;
    turn.load_weights(a, c);
    turn.load_row(a, c, t);
    x = turn.head(x, h >= a.Hq, a.eps);
  }
  store_head<D, false>(a, t, h, c, slot, x);
}

// Many tokens: a wave per token, 512 / D heads at a time, so that the weights
// and the token's row of the table are read once for all of its heads.
constexpr int HU = 4;  // heads of a lane whose loads are in flight together
template <int D>
__global__ __launch_bounds__(256) void qk_head_norm_rope_store_rows(HeadNorm a) {
  constexpr int C = D / 8, HW = 64 / C;
  const int lane = threadIdx.x & 63, c = lane % C, heads = a.Hq + 2 * a.Hkv;
  Turn<D> turn;
  turn.load_weights(a, c);
  for (unsigned t = blockIdx.x * 4 + (threadIdx.x >> 6); t < a.T; t += gridDim.x * 4) {
    const uint16_t* row = a.qkv + t * a.ld + 8 * c;
    turn.load_row(a, c, t);
    const int64_t slot = a.slots != nullptr ? a.slots[t] : -1;
    for (int h0 = lane / C; h0 < heads; h0 += HU * HW) {
      u32x4 x[HU];
#pragma unroll
      for (int i = 0; i < HU; ++i)
        x[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(row + min(h0 + i * HW, heads - 1) * D));
#pragma unroll
      for (int i = 0; i < HU; ++i) {
        const int h = h0 + i * HW;
        if (h < a.Hq + a.Hkv) x[i] = turn.head(x[i], h >= a.Hq, a.eps);
        if (h < heads) store_head<D, true>(a, t, h, c, slot, x[i]);
      }
    }
  }
}
// Tokens from which a wave takes a whole token.  A thread per chunk / a wave per
// token, us: 32 / 8 heads of 128, 128 tokens 2.9 / 6.3, 1024 8.3 / 9.2, 2048
// 12.2 / 12.2, 4096 20.2 / 19.8, 16383 97 / 73.6; 12 / 4 of 64, 128 tokens
// 2.6 / 3.1, 2048 4.5 / 4.3, 4096 7.9 / 7.2, 16383 19.4 / 20.5 (one number for
// all shapes: the wrong side costs 6 % there).
constexpr int64_t kHeadRowsT = 2048;

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
  const HeadNorm a{(const uint16_t*)qkv, ld, q_weight, k_weight, cos_sin, positions, slot_mapping, (uint16_t*)q_out,
                   (uint16_t*)k_cache, (uint16_t*)v_cache, (uint16_t*)k_out, (uint16_t*)v_out, num_slots, max_positions,
                   eps, R, Hq, Hkv, (unsigned)T};
  hipStream_t st = (hipStream_t)stream;
  if (T >= kHeadRowsT) {
    const dim3 grid((unsigned)std::min<int64_t>((T + 3) / 4, 4096));
    if (D == 64) hipLaunchKernelGGL(qk_head_norm_rope_store_rows<64>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(qk_head_norm_rope_store_rows<128>, grid, dim3(256), 0, st, a);
  } else {
    const dim3 grid((unsigned)((T * heads * (D / 8) + 255) / 256));
    if (D == 64) hipLaunchKernelGGL(qk_head_norm_rope_store_kernel<64>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(qk_head_norm_rope_store_kernel<128>, grid, dim3(256), 0, st, a);
  }
  return check_launch("qk_head_norm_rope_store");
}
