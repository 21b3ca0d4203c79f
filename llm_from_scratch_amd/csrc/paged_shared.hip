// GQA decode over a bf16 pool for groups of sequences that share their first
// blocks.
//
// A wave per (sequence, query head) walks the context a token at a time, D / 64
// values a lane, with the running maximum and sum of the softmax in fp32.
#include "decode_wave.h"

namespace lfs {
namespace {

template <int D, bool FP8>
__global__ __launch_bounds__(64) void paged_decode_tokens(
    const uint16_t* __restrict__ q, const void* __restrict__ kc, const void* __restrict__ vc,
    const float* __restrict__ ksc, const float* __restrict__ vsc, const int64_t* __restrict__ ctx_lens,
    const int32_t* __restrict__ bt, int64_t bt_stride, uint16_t* __restrict__ out, int Hq, int Hkv, int BS, int64_t NB,
    int max_blocks, float scale_log2) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x, h = blockIdx.x, b = blockIdx.y, kh = h / (Hq / Hkv);
  const int64_t L = min(ctx_lens[b], (int64_t)max_blocks * BS);
  float qf[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qf[e] = bf16_to_f32(q[((int64_t)b * Hq + h) * D + lane * E + e]) * scale_log2;
    acc[e] = 0.f;
  }
  auto value = [&](const void* c, int64_t at) {
    if constexpr (FP8) return __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t*)c)[at], 0);
    else return bf16_to_f32(((const uint16_t*)c)[at]);
  };
  for (int64_t t = 0; t < L; ++t) {
    const int64_t col = t / BS;
    const int off = (int)(t - col * BS);
    const int64_t blk = bt[(int64_t)b * bt_stride + col];
    if (blk < 0 || blk >= NB) continue;  // an invalid block contributes nothing
    const int64_t at = ((blk * BS + off) * Hkv + kh) * D + lane * E, sat = (blk * Hkv + kh) * BS + off;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(qf[e], value(kc, at + e), s);
    s = group_sum<64>(s);
    if constexpr (FP8) s *= ksc[sat];
    const float mn = fmaxf(m, s), a = exp2f(m - mn), p = exp2f(s - mn);
    l = l * a + p;
    const float w = FP8 ? p * vsc[sat] : p;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(w, value(vc, at + e), acc[e] * a);
    m = mn;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    out[((int64_t)b * Hq + h) * D + lane * E + e] = (uint16_t)f32_to_bf16(l > 0.f ? acc[e] / l : 0.f);
}

template <bool FP8>
int launch_tokens(const char* what, const void* q, const void* kc, const void* vc, const float* ks, const float* vs,
                  const int64_t* cl, const int32_t* bt, int64_t bts, void* out, int64_t B, int Hq, int Hkv, int D, int BS,
                  int64_t NB, int max_blocks, float scale, void* q_out, float* q_scale, void* stream) {
  const float sl2 = scale * 1.4426950408889634f;
  if (D == 64)
    hipLaunchKernelGGL((paged_decode_tokens<64, FP8>), dim3((unsigned)Hq, (unsigned)B), dim3(64), 0, (hipStream_t)stream,
                       (const uint16_t*)q, kc, vc, ks, vs, cl, bt, bts, (uint16_t*)out, Hq, Hkv, BS, NB, max_blocks, sl2);
  else
    hipLaunchKernelGGL((paged_decode_tokens<128, FP8>), dim3((unsigned)Hq, (unsigned)B), dim3(64), 0,
                       (hipStream_t)stream, (const uint16_t*)q, kc, vc, ks, vs, cl, bt, bts, (uint16_t*)out, Hq, Hkv, BS,
                       NB, max_blocks, sl2);
  const int rc = check_launch(what);
  if (rc || q_out == nullptr) return rc;
  return lfs_act_quant(out, Hq * D, q_out, q_scale, B, Hq * D, 128, 0, stream);
}

}  // namespace
}  // namespace lfs

using namespace lfs;

extern "C" int64_t lfs_paged_decode_shared_workspace_bytes(int64_t B, int64_t num_groups, int32_t num_q_heads,
                                                           int32_t num_kv_heads, int32_t head_dim) {
  if (B < 0 || num_groups < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return -1;
  return 1024;
}

extern "C" int lfs_paged_decode_shared(const void* q, const void* k_cache, const void* v_cache,
                                       const int64_t* context_lens, const int32_t* block_tables, int64_t bt_stride,
                                       const int32_t* cu_groups, const int32_t* shared_blocks, int64_t num_groups,
                                       void* out, void* workspace, int64_t workspace_bytes, int64_t B,
                                       int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                       int64_t num_blocks, int32_t max_blocks, float scale, void* q_out, float* q_scale,
                                       void* stream) {
  LFS_REQUIRE(num_groups >= 0, "paged_decode_shared: bad shape");
  const int rc = check_decode("paged_decode_shared", q, k_cache, v_cache, context_lens, block_tables, bt_stride, out,
                              workspace, workspace_bytes,
                              lfs_paged_decode_shared_workspace_bytes(B, num_groups, num_q_heads, num_kv_heads, head_dim),
                              B, num_q_heads, num_kv_heads, head_dim, block_size, num_blocks, max_blocks, q_out, q_scale);
  if (rc || B == 0) return rc;
  LFS_REQUIRE(num_groups == 0 || (cu_groups && shared_blocks), "paged_decode_shared: null pointer");
  LFS_REQUIRE(B <= 8192 && num_groups <= 8192, "paged_decode_shared: at most 8192 sequences and groups");
  return launch_tokens<false>("paged_decode_shared", q, k_cache, v_cache, nullptr, nullptr, context_lens, block_tables,
                              bt_stride, out, B, num_q_heads, num_kv_heads, head_dim, block_size, num_blocks, max_blocks,
                              scale, q_out, q_scale, stream);
}
