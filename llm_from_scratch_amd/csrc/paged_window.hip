// Paged decode over a sliding window with sinks: with L tokens in a
// sequence's context, the newest at L - 1,
//   o = sum_t softmax_t(scale * q . k_t) v_t  over t < L with t >= L - window
//       or t < sinks,
// and 0 for a sequence without context.  Hidden tokens are never read, so
// their blocks may be freed (table entry -1).
//
// A sequence's visible tokens are tiles (decode_wave.h) of two ranges: the
// window, whose first tile may begin with hidden rows, and the sinks before
// it, whose last may end with them.  One 4-wave workgroup takes a split of
// both for one (sequence, kv head), its waves every fourth tile of the split;
// the waves' partials (o, m, l) meet in LDS.  With one split that is the
// output, in one launch; else the splits' partials go to the workspace and a
// second launch merges them.  Unlike contexts, windows are of one length, so
// equal splits balance: as many as give every CU a workgroup.
// Bound: HBM, the visible keys and values read once.
#include "common.h"
#include "decode_wave.h"

#include <algorithm>

namespace lfs {
namespace {

constexpr int WNW = 4;  // waves per workgroup

template <int D, int G>
__global__ __launch_bounds__(64 * WNW, 2) void paged_window_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ kc, const uint16_t* __restrict__ vc,
    const int64_t* __restrict__ ctx_lens, const int32_t* __restrict__ bt, int64_t bt_stride, float* __restrict__ ws_o,
    float* __restrict__ ws_ml, uint16_t* __restrict__ out, int Hkv, int BS, int64_t NB, int max_blocks, int tile,
    int window, int sinks, float scale_log2, int splits, int per) {
  using W = DecodeWave<D, G>;
  __shared__ __attribute__((aligned(16))) float p_lds[WNW][DecodeGeom<D>::T * W::GP];
  __shared__ __attribute__((aligned(16))) float part_o[WNW][G * D];
  __shared__ float part_m[WNW][G], part_l[WNW][G];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  // kv heads fastest: workgroups that start together read neighbouring pieces of the same token rows
  const int kh = blockIdx.x % Hkv, split = blockIdx.x / Hkv % splits;
  const int64_t b = blockIdx.x / Hkv / splits;
  const int Hq = Hkv * G;
  const int64_t L = max(ctx_lens[b], (int64_t)0), end = min(L, (int64_t)max_blocks * BS);
  // hidden: tokens sk .. first - 1
  const int64_t first = max((int64_t)0, L - window), sk = min(min((int64_t)sinks, first), end);

  W w(lane, Hkv);
  typename W::QBuf qa;
  w.load_q(qa, q, b, kh, Hq);
  const int32_t* btrow = bt + b * bt_stride;
  if (sk > 0) {  // the sinks' tiles, from the last split and wave on, which have the fewest of the window's
    const unsigned n = ((unsigned)sk + tile - 1) >> __builtin_ctz(tile);  // tiles: sk <= sinks < 2^31
    const int64_t each = splits == 1 ? n : (n + splits - 1) / (unsigned)splits;
    const int64_t t0 = (splits - 1 - split) * each * tile, t1 = min(sk, t0 + each * tile);
    const int64_t t = t0 + (WNW - 1 - wave) * tile;
    if (t < t1)
      decode_walk<D, G>(w, qa, kc, vc, btrow, BS, NB, tile, scale_log2, kh, t, t1, WNW, max_blocks, p_lds[wave]);
  }
  const int64_t w0 = first & -(int64_t)tile;  // 16, 32 or 64
  const int64_t t0 = w0 + (int64_t)split * per * tile, t1 = min(end, t0 + (int64_t)per * tile);
  const int64_t t = t0 + wave * tile;
  if (t < t1)
    decode_walk<D, G, true>(w, qa, kc, vc, btrow, BS, NB, tile, scale_log2, kh, t, t1, WNW, max_blocks, p_lds[wave],
                            NoPrologue(), first);
  w.reduce_lanes();
  if (w.ts == 0) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float* dst = &part_o[wave][g * D + w.dc * 8];
      *reinterpret_cast<float4*>(dst) = make_float4(w.acc[g][0], w.acc[g][1], w.acc[g][2], w.acc[g][3]);
      *reinterpret_cast<float4*>(dst + 4) = make_float4(w.acc[g][4], w.acc[g][5], w.acc[g][6], w.acc[g][7]);
    }
  }
  if (lane < G) part_m[wave][lane] = w.m_run, part_l[wave][lane] = w.l_run;
  __syncthreads();
  for (int e = threadIdx.x; e < G * D; e += 64 * WNW) {
    const int g = e / D;
    float M = -INFINITY, num = 0.f, den = 0.f;
#pragma unroll
    for (int i = 0; i < WNW; ++i) M = fmaxf(M, part_m[i][g]);
    if (M != -INFINITY) {
#pragma unroll
      for (int i = 0; i < WNW; ++i) {
        const float x = exp2f(part_m[i][g] - M);
        den = fmaf(x, part_l[i][g], den);
        num = fmaf(x, part_o[i][e], num);
      }
    }
    const int64_t row = b * Hq + kh * G;  // first query row
    if (splits == 1) {
      out[row * D + e] = (uint16_t)f32_to_bf16(den > 0.f ? num / den : 0.f);
    } else {
      const int64_t prow = (row + g) * splits + split;
      ws_o[prow * D + (e - g * D)] = num;
      if (e == g * D) ws_ml[prow * 2] = M, ws_ml[prow * 2 + 1] = den;
    }
  }
}

// One thread per output element; with qo also the act_quant of the 128-value
// group that its 128 neighbours hold.
__global__ __launch_bounds__(128) void paged_window_merge(const float* __restrict__ ws_o,
                                                          const float* __restrict__ ws_ml, uint16_t* __restrict__ out,
                                                          uint8_t* __restrict__ qo, float* __restrict__ qs, int64_t E,
                                                          int D, int splits) {
  __shared__ __attribute__((aligned(16))) uint16_t vals[128];
  const int64_t e = (int64_t)blockIdx.x * 128 + threadIdx.x;  // D is 64 or 128: a wave's elements are one row's
  uint16_t v = 0;
  if (e < E) {
    const int64_t row = e / D;
    v = (uint16_t)f32_to_bf16(merge_element(ws_o, ws_ml, row * splits, 1, splits, D, (int)(e - row * D)));
    out[e] = v;
  }
  if (qo == nullptr) return;
  vals[threadIdx.x] = v;
  __syncthreads();
  const int t = threadIdx.x;
  if (t >= 16) return;
  float f[8], amax = 0.f;
  unpack8(*reinterpret_cast<const uint4*>(&vals[t * 8]), f);
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(f[i]));
  amax = group_max<16>(amax);
  const float sc = scale_from_amax(amax, false);
  *reinterpret_cast<uint2*>(qo + (int64_t)blockIdx.x * 128 + t * 8) = quant8(f, sc);
  if (t == 0) qs[blockIdx.x] = sc;
}

int window_cu_count() {
  static int cached[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (cached[dev] == 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cached[dev] = n;
  }
  return cached[dev];
}

}  // namespace
}  // namespace lfs

using namespace lfs;

extern "C" int64_t lfs_paged_decode_window_workspace_bytes(int64_t B, int32_t num_q_heads, int32_t head_dim) {
  if (B < 0 || num_q_heads <= 0 || head_dim <= 0) return -1;
  // units * splits <= CUs workgroups of at most 8 query rows, D + 2 floats a row
  const int64_t cus = window_cu_count();
  return B > cus ? 0 : 4 * cus * std::min(8, num_q_heads) * ((int64_t)head_dim + 2);
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
  LFS_REQUIRE((q_out == nullptr) == (q_scale == nullptr), "paged_decode_window: q_out and q_scale go together");
  LFS_REQUIRE(q_out == nullptr || Hq * D % 128 == 0, "paged_decode_window: the quantised output needs Hq*D %% 128 == 0");
  const int64_t units = B * Hkv, cus = window_cu_count();
  LFS_REQUIRE(B < (1ll << 24) / Hkv, "paged_decode_window: too many (sequence, kv head) workgroups");
  const int64_t need = lfs_paged_decode_window_workspace_bytes(B, Hq, D);
  LFS_REQUIRE(workspace_bytes >= need && (need == 0 || workspace),
              "paged_decode_window: workspace of %lld bytes < required %lld", (long long)workspace_bytes, (long long)need);
  int tile = 16;
  for (int t = D == 64 ? 64 : 32; t >= 16; t >>= 1)
    if (BS % t == 0) { tile = t; break; }
  // a window's tiles, whatever its place in them
  const int64_t seen = std::min<int64_t>(window, (int64_t)max_blocks * BS), tiles = (seen + tile - 1) / tile + 1;
  const int splits = (int)std::max<int64_t>(1, std::min(cus / units, (tiles + WNW - 1) / WNW));
  const int per = (int)((tiles + splits - 1) / splits);
  const int G = Hq / Hkv;
  float* ws_o = (float*)workspace;
  float* ws_ml = ws_o + (int64_t)B * Hq * splits * D;
  const float sl2 = scale * 1.4426950408889634f;
  hipStream_t st = (hipStream_t)stream;
#define LFS_G(DD, GG)                                                                                                 \
  case GG:                                                                                                            \
    hipLaunchKernelGGL((paged_window_kernel<DD, GG>), dim3((unsigned)(units * splits)), dim3(64 * WNW), 0, st,        \
                       (const uint16_t*)q, (const uint16_t*)k_cache, (const uint16_t*)v_cache, context_lens,          \
                       block_tables, bt_stride, ws_o, ws_ml, (uint16_t*)out, Hkv, BS, num_blocks, max_blocks, tile,   \
                       window, sinks, sl2, splits, per);                                                              \
    break;
  if (D == 64) {
    switch (G) {
      LFS_G(64, 1) LFS_G(64, 2) LFS_G(64, 3) LFS_G(64, 4) LFS_G(64, 5) LFS_G(64, 6) LFS_G(64, 7) LFS_G(64, 8)
    }
  } else {
    switch (G) {
      LFS_G(128, 1) LFS_G(128, 2) LFS_G(128, 3) LFS_G(128, 4) LFS_G(128, 5) LFS_G(128, 6) LFS_G(128, 7) LFS_G(128, 8)
    }
  }
#undef LFS_G
  int rc = check_launch("paged_decode_window");
  if (rc != 0) return rc;
  if (splits > 1) {
    const int64_t E = B * Hq * D;
    hipLaunchKernelGGL(paged_window_merge, dim3((unsigned)((E + 127) / 128)), dim3(128), 0, st, ws_o, ws_ml,
                       (uint16_t*)out, (uint8_t*)q_out, q_scale, E, D, splits);
    return check_launch("paged_decode_window(merge)");
  }
  if (q_out == nullptr) return 0;
  return lfs_act_quant(out, Hq * D, q_out, q_scale, B, Hq * D, 128, 0, stream);
}
