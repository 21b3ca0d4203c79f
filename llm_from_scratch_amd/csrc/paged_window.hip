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
// second launch merges them.  Windows are of one length, so equal splits
// balance, unless they are long: then contexts inside the window and a last
// round of workgroups cost more than the paged decode's balanced split does
// (decode_wave.h, the same walk with one wave per kv head, an equal share of
// all visible tiles per workgroup).
// Bound: HBM, the visible keys and values read once.  256 sequences past a
// window of 4096 (32 / 8 heads of 128, 4.1 GB) take 630 us, 6.5 TB/s; 64 past one
// of 1024 (16 / 4 of 64, 67 MB) 20 us: 6 us for the launch, the table, the
// first tile and the merge in LDS, then 4.8 TB/s.
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
    Window win, float scale_log2, int splits, int per) {
  using W = DecodeWave<D, G>;
  __shared__ __attribute__((aligned(16))) float p_lds[WNW][DecodeGeom<D>::T * W::GP];
  __shared__ __attribute__((aligned(16))) float part_o[WNW][G * D];
  __shared__ float part_m[WNW][G], part_l[WNW][G];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  // kv heads fastest: workgroups that start together read neighbouring pieces of the same token rows
  const int kh = blockIdx.x % Hkv, split = blockIdx.x / Hkv % splits;
  const int64_t b = blockIdx.x / Hkv / splits;
  const int Hq = Hkv * G;
  const WindowTiles wt(ctx_lens[b], (int64_t)max_blocks * BS, tile, win);

  W w(lane, Hkv);
  typename W::QBuf qa;
  w.load_q(qa, q, b, kh, Hq);
  const int32_t* btrow = bt + b * bt_stride;
  if (wt.ns > 0) {  // the sinks' tiles, from the last split and wave on, which have the fewest of the window's
    const int each = splits == 1 ? wt.ns : (wt.ns + splits - 1) / splits;
    const int64_t t0 = (int64_t)(splits - 1 - split) * each * tile, t1 = min(wt.sk, t0 + (int64_t)each * tile);
    const int64_t t = t0 + (WNW - 1 - wave) * tile;
    if (t < t1)
      decode_walk<D, G>(w, qa, kc, vc, btrow, BS, NB, tile, scale_log2, kh, t, t1, WNW, max_blocks, p_lds[wave]);
  }
  const int64_t t0 = wt.w0 + (int64_t)split * per * tile, t1 = min(wt.end, t0 + (int64_t)per * tile);
  const int64_t t = t0 + wave * tile;
  if (t < t1)
    decode_walk<D, G, true>(w, qa, kc, vc, btrow, BS, NB, tile, scale_log2, kh, t, t1, WNW, max_blocks, p_lds[wave],
                            NoPrologue(), wt.first);
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

// Whether a call takes the balanced split: long windows (from 48 tiles, with one
// query head per kv head from 32) and at least 32 tiles of work per CU.  us,
// equal splits / balanced, contexts past the window (evenly spaced from 10
// tokens to past it): 12 / 4 heads of 64, window 4096, 32 sequences 35.2 / 35.3
// (32.4 / 28.5), 64 55 / 57 (51 / 43), 80 96 / 67 (62 / 53), 256 203 / 180; 32 / 8
// of 128, 4096, 4 22 / 27, 16 58 / 56 (54 / 41), 256 740 / 680; window 1024 (33
// tiles), 64 55 / 58 (52 / 57), 256 196 / 192 (173 / 197); 8 / 8 of 64, window
// 2048 (33 tiles), 64 61 / 55 (56 / 47), 128 120 / 98.
bool window_balanced(int64_t B, int64_t units, int64_t cus, int64_t tiles, int G) {
  return B <= BAL_MAXB && tiles >= (G == 1 ? 32 : 48) && units * tiles >= 32 * cus;
}
// Equal splits of a window otherwise: one while a wave then has at most two
// tiles (the merge costs what they do: 5 tiles 8.5 us in two splits, 8.2 in
// one), else as many as CUs allow.  us, one split / those: one sequence, 12 / 4
// heads of 64, window 512 10.0 / 8.6, 1024 13.5 / 9.2; 16 sequences 17.3 / 12.1.
int window_splits(int64_t units, int64_t cus, int64_t tiles) {
  if (tiles <= 2 * WNW) return 1;
  return (int)std::max<int64_t>(1, std::min(cus / units, (tiles + WNW - 1) / WNW));
}

}  // namespace
}  // namespace lfs

using namespace lfs;

extern "C" int64_t lfs_paged_decode_window_workspace_bytes(int64_t B, int32_t num_q_heads, int32_t head_dim) {
  if (B < 0 || num_q_heads <= 0 || head_dim <= 0) return -1;
  const int64_t cus = decode_cu_count();
  // equal splits: at most a workgroup per CU, of at most 8 query rows; the
  // balanced split: as lfs_paged_decode; D + 2 floats a row
  int64_t need = B > cus ? 0 : 4 * cus * std::min(8, num_q_heads) * ((int64_t)head_dim + 2);
  if (B <= BAL_MAXB) need = std::max(need, 4 * (8 * cus + 2 * B) * num_q_heads * ((int64_t)head_dim + 2) + 4 * (B + 1));
  return need;
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
  LFS_REQUIRE(((uintptr_t)workspace & 15u) == 0, "paged_decode_window: the workspace must be 16-byte aligned");
  LFS_REQUIRE((q_out == nullptr) == (q_scale == nullptr), "paged_decode_window: q_out and q_scale go together");
  LFS_REQUIRE(q_out == nullptr || Hq * D % 128 == 0, "paged_decode_window: the quantised output needs Hq*D %% 128 == 0");
  const int64_t units = B * Hkv, cus = decode_cu_count();
  LFS_REQUIRE(B < (1ll << 24) / Hkv, "paged_decode_window: too many (sequence, kv head) workgroups");
  const int64_t need = lfs_paged_decode_window_workspace_bytes(B, Hq, D);
  LFS_REQUIRE(workspace_bytes >= need && (need == 0 || workspace),
              "paged_decode_window: workspace of %lld bytes < required %lld", (long long)workspace_bytes, (long long)need);
  int tile = 16;
  for (int t = D == 64 ? 64 : 32; t >= 16; t >>= 1)
    if (BS % t == 0) { tile = t; break; }
  const int G = Hq / Hkv;
  const float sl2 = scale * 1.4426950408889634f;
  const Window win{window, sinks};
  hipStream_t st = (hipStream_t)stream;
  // a window's tiles, whatever its place in them
  const int64_t seen = std::min<int64_t>(window, (int64_t)max_blocks * BS), tiles = (seen + tile - 1) / tile + 1;
  if (window_balanced(B, units, cus, tiles, G)) {
    const BalancedGeom bg = balanced_geom(Hkv);
    const int64_t rows = ((int64_t)bg.nwg + B * bg.ngroups) * bg.wpg * G;
    const int64_t first = std::min<int64_t>(sinks, (int64_t)max_blocks * BS);  // of a sequence: the sinks' tiles, the window's
    LFS_REQUIRE((int64_t)bg.ngroups * B * ((first + tile - 1) / tile + tiles) < (1ll << 31),
                "paged_decode_window: too many visible tiles for the balanced split");
    float* ws_o = (float*)workspace;
    float* ws_ml = ws_o + rows * D;
    int* tp = (int*)(ws_ml + rows * 2);
    const PartMap pm{0, 0, tp, tile, bg.ngroups, bg.wpg, G, bg.nwg, (int)B};
    const bool ok = D == 64
        ? dispatch_balanced<64, true>(G, (unsigned)bg.nwg, dim3(64 * bg.wpg), st, (const uint16_t*)q,
                                      (const uint16_t*)k_cache, (const uint16_t*)v_cache, context_lens, block_tables,
                                      bt_stride, ws_o, ws_ml, tp, (uint16_t*)out, Hkv, BS, num_blocks, max_blocks,
                                      (int)B, tile, sl2, bg.ngroups, win)
        : dispatch_balanced<128, true>(G, (unsigned)bg.nwg, dim3(64 * bg.wpg), st, (const uint16_t*)q,
                                       (const uint16_t*)k_cache, (const uint16_t*)v_cache, context_lens, block_tables,
                                       bt_stride, ws_o, ws_ml, tp, (uint16_t*)out, Hkv, BS, num_blocks, max_blocks,
                                       (int)B, tile, sl2, bg.ngroups, win);
    LFS_REQUIRE(ok, "paged_decode_window: unsupported group size %d", G);
    const int rc = check_launch("paged_decode_window(balanced split)");
    if (rc) return rc;
    return paged_decode_merge_launch(ws_o, ws_ml, context_lens, out, q_out, q_scale, B, Hq, D, BS, max_blocks, pm, st);
  }
  const int splits = window_splits(units, cus, tiles);
  const int per = (int)((tiles + splits - 1) / splits);
  float* ws_o = (float*)workspace;
  float* ws_ml = ws_o + (int64_t)B * Hq * splits * D;
#define LFS_G(DD, GG)                                                                                                 \
  case GG:                                                                                                            \
    hipLaunchKernelGGL((paged_window_kernel<DD, GG>), dim3((unsigned)(units * splits)), dim3(64 * WNW), 0, st,        \
                       (const uint16_t*)q, (const uint16_t*)k_cache, (const uint16_t*)v_cache, context_lens,          \
                       block_tables, bt_stride, ws_o, ws_ml, (uint16_t*)out, Hkv, BS, num_blocks, max_blocks, tile,   \
                       win, sl2, splits, per);                                                                        \
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
