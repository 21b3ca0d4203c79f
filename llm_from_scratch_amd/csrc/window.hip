// Causal attention over a sliding window with sinks: the query at position p
// of its sequence sees key j where j <= p and (j > p - window or j < sinks),
//   o = sum_j softmax_j(scale * q . k_j) v_j  over the visible j,
// and 0 where it sees none.  Hidden keys are never read, so their blocks may
// be freed.
//
// One wave per (query token, query head): lane l takes the score of the l-th
// key of a chunk of 64, then dims l (and l + 64) of the chunk's P V, with the
// running maximum and sum of an online softmax in fp32.
#include "common.h"

namespace lfs {
namespace {

template <int D>
__global__ __launch_bounds__(64) void window_attention_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
    const int32_t* __restrict__ cu_q, const int32_t* __restrict__ cu_k, const int64_t* __restrict__ ctx_lens,
    const int32_t* __restrict__ bt, int64_t bt_stride, int64_t max_blocks, int BS, int64_t num_slots,
    uint16_t* __restrict__ out, int Hkv, int64_t window, int64_t sinks, float scale_log2) {
  __shared__ float qs[D];
  const int lane = threadIdx.x, h = blockIdx.y, Hq = gridDim.y, kh = h / (Hq / Hkv);
  const int64_t b = blockIdx.z, t = blockIdx.x;
  int64_t row, p, n, k0 = 0;  // query row, its position, keys of the context, row of key 0
  if (ctx_lens != nullptr) {
    row = b;
    p = ctx_lens[b] - 1;
    n = min(p + 1, max_blocks * BS);
  } else {
    const int64_t lq = cu_q[b + 1] - cu_q[b], lk = cu_k[b + 1] - cu_k[b];
    if (t >= lq) return;
    row = cu_q[b] + t;
    p = lk - lq + t;
    n = lk;
    k0 = cu_k[b];
  }
  const int64_t hi = min(p + 1, n), first = max((int64_t)0, p + 1 - window);
  const int64_t s = max((int64_t)0, min(min(sinks, first), hi));  // visible keys before the window
  const int64_t count = s + max((int64_t)0, hi - first);
  const uint16_t* qr = q + (row * Hq + h) * D;
  for (int d = lane; d < D; d += 64) qs[d] = bf16_to_f32(qr[d]);
  __syncthreads();
  auto key_row = [&](int64_t j) -> int64_t {  // -1: its block is not in the pool
    if (bt == nullptr) return k0 + j;
    const int64_t blk = bt[b * bt_stride + min(j / BS, bt_stride - 1)];
    if (blk < 0 || blk * BS >= num_slots) return -1;
    return blk * BS + j % BS;
  };
  float m = -INFINITY, l = 0.f, o[D / 64] = {};
  for (int64_t c = 0; c < count; c += 64) {
    const int64_t i = c + lane;
    int64_t kr = -1;
    if (i < count) kr = key_row(i < s ? i : first + i - s);
    if (i < count && kr < 0 && ctx_lens == nullptr) kr = 0;
    float x = -INFINITY;
    if (kr >= 0) {
      const uint16_t* kp = k + (kr * Hkv + kh) * D;
      float a = 0.f;
      for (int d = 0; d < D; d += 8) {
        float f[8];
        unpack8(*reinterpret_cast<const uint4*>(kp + d), f);
#pragma unroll
        for (int e = 0; e < 8; ++e) a = fmaf(f[e], qs[d + e], a);
      }
      x = a * scale_log2;
    }
    const float m_new = fmaxf(m, group_max<64>(x));
    const float alpha = m_new == m ? 1.f : exp2f(m - m_new);
    const float w = kr >= 0 ? exp2f(x - m_new) : 0.f;
    l = l * alpha + group_sum<64>(w);
    m = m_new;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] *= alpha;
    const int rows = (int)min((int64_t)64, count - c);
    for (int r = 0; r < rows; ++r) {
      const int64_t vr = __shfl(kr, r, 64);
      if (vr < 0) continue;
      const float wr = __shfl(w, r, 64);
#pragma unroll
      for (int e = 0; e < D / 64; ++e) o[e] = fmaf(wr, bf16_to_f32(v[(vr * Hkv + kh) * D + lane + 64 * e]), o[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < D / 64; ++e)
    out[(row * Hq + h) * D + lane + 64 * e] = (uint16_t)f32_to_bf16(count > 0 ? (l != 0.f ? o[e] / l : 0.f) : 0.f);
}

int window_launch(const char* what, const void* q, const void* k, const void* v, const int32_t* cu_q,
                  const int32_t* cu_k, const int64_t* ctx_lens, const int32_t* bt, int64_t bt_stride,
                  int64_t max_blocks, int BS, int64_t num_slots, void* out, int64_t B, int Hq, int Hkv, int D,
                  int64_t max_q, int64_t window, int64_t sinks, float scale, hipStream_t st) {
  const dim3 grid((unsigned)max_q, (unsigned)Hq, (unsigned)B);
  const float sl2 = scale * 1.4426950408889634f;
#define LFS_W(DD)                                                                                                     \
  hipLaunchKernelGGL(window_attention_kernel<DD>, grid, dim3(64), 0, st, (const uint16_t*)q, (const uint16_t*)k,      \
                     (const uint16_t*)v, cu_q, cu_k, ctx_lens, bt, bt_stride, max_blocks, BS, num_slots,              \
                     (uint16_t*)out, Hkv, window, sinks, sl2)
  if (D == 64) LFS_W(64);
  else LFS_W(128);
#undef LFS_W
  return check_launch(what);
}

}  // namespace
}  // namespace lfs

using namespace lfs;

extern "C" int lfs_prefill_attention_window(const void* q, const void* k, const void* v, const int32_t* cu_seqlens_q,
                                            const int32_t* cu_seqlens_k, const int32_t* block_tables,
                                            int64_t bt_stride, int32_t block_size, int64_t num_slots, void* out,
                                            int64_t B, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                            int32_t max_seqlen_q, int32_t window, int32_t sinks, float scale,
                                            void* stream) {
  const int Hq = num_q_heads, Hkv = num_kv_heads, D = head_dim;
  LFS_REQUIRE(B >= 0 && Hq > 0 && Hkv > 0 && max_seqlen_q >= 0, "prefill_attention_window: bad shape");
  LFS_REQUIRE(D == 64 || D == 128, "prefill_attention_window: head_dim must be 64 or 128 (got %d)", D);
  LFS_REQUIRE(Hq % Hkv == 0 && Hq / Hkv <= 8,
              "prefill_attention_window: num_q_heads (%d) must be a multiple of num_kv_heads (%d), ratio <= 8", Hq, Hkv);
  LFS_REQUIRE(window >= 1 && sinks >= 0, "prefill_attention_window: window must be >= 1 and sinks >= 0 (got %d, %d)",
              window, sinks);
  if (B == 0 || max_seqlen_q == 0) return 0;
  LFS_REQUIRE(q && k && v && cu_seqlens_q && cu_seqlens_k && out, "prefill_attention_window: null pointer");
  LFS_REQUIRE(((((uintptr_t)q) | ((uintptr_t)k) | ((uintptr_t)v) | ((uintptr_t)out)) & 15u) == 0,
              "prefill_attention_window: q, k, v and out must be 16-byte aligned");
  if (block_tables != nullptr)
    LFS_REQUIRE(block_size > 0 && block_size % 16 == 0 && num_slots >= block_size && bt_stride > 0,
                "prefill_attention_window: bad paged KV geometry (block_size must be a multiple of 16)");
  LFS_REQUIRE(B < 65536 && Hq < 65536, "prefill_attention_window: grid too large");
  return window_launch("prefill_attention_window", q, k, v, cu_seqlens_q, cu_seqlens_k, nullptr, block_tables,
                       bt_stride, 0, block_tables != nullptr ? block_size : 1, num_slots, out, B, Hq, Hkv, D,
                       max_seqlen_q, window, sinks, scale, (hipStream_t)stream);
}

extern "C" int64_t lfs_paged_decode_window_workspace_bytes(int64_t B, int32_t num_q_heads, int32_t head_dim) {
  return B < 0 || num_q_heads <= 0 || head_dim <= 0 ? -1 : 0;
}

extern "C" int lfs_paged_decode_window(const void* q, const void* k_cache, const void* v_cache,
                                       const int64_t* context_lens, const int32_t* block_tables, int64_t bt_stride,
                                       void* out, void* workspace, int64_t workspace_bytes, int64_t B,
                                       int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                       int32_t block_size, int64_t num_blocks, int32_t max_blocks, int32_t window,
                                       int32_t sinks, float scale, void* q_out, float* q_scale, void* stream) {
  const int Hq = num_q_heads, Hkv = num_kv_heads, D = head_dim, BS = block_size;
  LFS_REQUIRE(B >= 0 && Hq > 0 && Hkv > 0 && BS > 0 && num_blocks >= 0 && max_blocks >= 0,
              "paged_decode_window: bad shape");
  LFS_REQUIRE(D == 64 || D == 128, "paged_decode_window: head_dim must be 64 or 128 (got %d)", D);
  LFS_REQUIRE(Hq % Hkv == 0 && Hq / Hkv <= 8,
              "paged_decode_window: num_q_heads (%d) must be a multiple of num_kv_heads (%d), ratio <= 8", Hq, Hkv);
  LFS_REQUIRE(BS % 16 == 0, "paged_decode_window: block_size must be a multiple of 16 (got %d)", BS);
  LFS_REQUIRE(window >= 1 && sinks >= 0, "paged_decode_window: window must be >= 1 and sinks >= 0 (got %d, %d)", window,
              sinks);
  LFS_REQUIRE(bt_stride >= max_blocks, "paged_decode_window: block table stride < max_blocks");
  LFS_REQUIRE(num_blocks >= 1 || max_blocks == 0, "paged_decode_window: empty KV pool");
  if (B == 0) return 0;
  LFS_REQUIRE(q && k_cache && v_cache && context_lens && out, "paged_decode_window: null pointer");
  LFS_REQUIRE(max_blocks == 0 || block_tables, "paged_decode_window: null block table");
  LFS_REQUIRE(((((uintptr_t)q) | ((uintptr_t)k_cache) | ((uintptr_t)v_cache) | ((uintptr_t)out)) & 15u) == 0,
              "paged_decode_window: q, caches and out must be 16-byte aligned");
  LFS_REQUIRE(B < 65536 && Hq < 65536, "paged_decode_window: batch too large");
  LFS_REQUIRE((q_out == nullptr) == (q_scale == nullptr), "paged_decode_window: q_out and q_scale go together");
  LFS_REQUIRE(q_out == nullptr || Hq * D % 128 == 0, "paged_decode_window: the quantised output needs Hq*D %% 128 == 0");
  const int64_t need = lfs_paged_decode_window_workspace_bytes(B, Hq, D);
  LFS_REQUIRE(workspace_bytes >= need && (need == 0 || workspace),
              "paged_decode_window: workspace of %lld bytes < required %lld", (long long)workspace_bytes, (long long)need);
  const int rc = window_launch("paged_decode_window", q, k_cache, v_cache, nullptr, nullptr, context_lens, block_tables,
                               bt_stride, max_blocks, BS, num_blocks * BS, out, B, Hq, Hkv, D, 1, window, sinks, scale,
                               (hipStream_t)stream);
  if (rc != 0 || q_out == nullptr) return rc;
  return lfs_act_quant(out, Hq * D, q_out, q_scale, B, Hq * D, 128, 0, stream);
}
