// GQA decode over a KV pool in 8 bits: codes e4m3fn [NB, BS, Hkv, D], scales
// fp32 [NB, Hkv, BS] per token and kv head.  With K = s_k k and V = s_v v,
//   o = sum_t w_t s_v,t v_t / sum_t w_t,   w_t = exp(scale s_k,t (q . k_t) - m).
//
// The walk of a wave over its tiles is pool_wave.h's.  Work is shared by the
// balanced split of decode_wave.h: one 4-wave workgroup a CU, its waves on
// adjacent heads of the same rows, so that both halves of a 128-byte line (two
// heads of 64 codes) are asked for together.
//
// What it takes (us, with the merge's launch; the same contexts in bf16): 64
// sequences of 512 to 32768 tokens, 32 / 8 heads of 128: 352 (651), 6.4 TB/s; 64 of
// 128 to 4096, 16 / 4 of 64: 23 (38); one of 3001, 12 / 4 of 64: 15 (16).  Bound:
// HBM at the first; at the second 5 us of launch, scan and first tile and 4 of the
// merge beside some 13 of reads; the last is these fixed parts alone.  A copy of the
// kernel that only loads its tiles takes as long, so the arithmetic is hidden.
#include "pool_wave.h"

namespace lfs {
namespace {

// A workgroup's four waves are 4 / hg shares of hg adjacent kv heads each.
// SCAN: a fixed grid's shares split the tiles of the batch evenly
// (paged_decode_balanced's split); else a share per (sequence, group of kv heads)
// walks the whole context.  (With a workgroup a share, whose LDS lets two onto a CU,
// one kv head took 33 us where it takes 27: 64 sequences of 128 to 8192 tokens, 8 /
// 1 heads of 128.)
template <int D, bool ONE, bool SCAN>
__global__ __launch_bounds__(256) void paged_fp8_kernel(
    const uint16_t* __restrict__ q, const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
    const float* __restrict__ ksc, const float* __restrict__ vsc, const int64_t* __restrict__ ctx_lens,
    const int32_t* __restrict__ bt, int64_t bt_stride, float* __restrict__ ws_o, float* __restrict__ ws_ml,
    int* __restrict__ tp_out, uint16_t* __restrict__ out, int Hkv, int G, int BS, int64_t NB, int max_blocks, int B,
    float scale_log2, int ngroups, int hg) {
  constexpr int T = PoolGeom<D, true>::T;
  __shared__ __attribute__((aligned(16))) float scales[4][2 * T];
  __shared__ int tp[SCAN ? BAL_MAXB + 1 : 1], lens[SCAN ? BAL_MAXB : 1];
  __shared__ int wsum[4], found[4];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int per = 4 / hg, sub = wave / hg, head = wave - sub * hg;
  const unsigned v = blockIdx.x * per + sub;  // the share (sub == per: none, of 3 heads' fourth wave)
  const int cap = max_blocks * BS;
  PoolWave<D, true, ONE> w;
  w.init(lane, kc, vc, ksc, vsc, Hkv, G, BS, NB, scale_log2);
  // a range of tiles of (sequence, group of kv heads), for the wave's head
  auto range = [&](PoolRange& r, int b, int kh, int L, int i0, int i1, int64_t slot) {
    const int64_t h = (int64_t)b * Hkv + kh;
    r.btrow = bt + (int64_t)b * bt_stride;
    r.q = q + h * G * D;
    r.t0 = i0 * T, r.t1 = min(L, i1 * T), r.kh = kh;
    r.out = r.t0 == 0 && r.t1 >= L ? out + h * G * D : nullptr;
    r.prow = (slot * hg + head) * G;
  };
  if constexpr (!SCAN) {
    const int b = (int)(v / (unsigned)ngroups), grp = (int)(v - (unsigned)b * ngroups), kh = grp * hg + head;
    if (sub >= per || b >= B || kh >= Hkv) return;
    const int L = (int)max((int64_t)0, min(ctx_lens[b], (int64_t)cap));
    if (L <= 0) {
      uint16_t* o = out + ((int64_t)b * Hkv + kh) * G * D;
      for (int i = lane; i < G * D / 2; i += 64) reinterpret_cast<uint32_t*>(o)[i] = 0;
      return;
    }
    bool left = true;
    w.run(
        [&](PoolRange& r) {
          if (!left) return false;
          left = false;
          range(r, b, kh, L, 0, (L + T - 1) / T, 0);
          return true;
        },
        scales[wave], ws_o, ws_ml);
  } else {
    const TileScan scan = scan_tiles(tp, wsum, B, [&](int b) {
      const int L = (int)max((int64_t)0, min(ctx_lens[b], (int64_t)cap));
      lens[b] = L;
      return (L + T - 1) / T;
    });
    const unsigned total = (unsigned)ngroups * (unsigned)scan.total, shares = gridDim.x * per;
    const unsigned Ct = max(1u, (total + shares - 1) / shares);
    place_tiles(tp, scan, [&](int i, int before, int after) {
      for (int k = 0; k < per; ++k) {
        const unsigned at = (blockIdx.x * per + k) * Ct;
        if ((unsigned)ngroups * (unsigned)before <= at && at < (unsigned)ngroups * (unsigned)after) found[k] = i;
      }
    });
    if (blockIdx.x == 0)
      for (int i = tid; i <= B; i += blockDim.x) tp_out[i] = tp[i];
    unsigned u = v * Ct;
    const unsigned u_end = min(total, u + Ct);
    if (sub >= per || u >= u_end) return;
    int b = __builtin_amdgcn_readfirstlane(found[sub]);
    w.run(
        [&](PoolRange& r) {
          while (u < u_end) {
            const unsigned t0 = __builtin_amdgcn_readfirstlane(tp[b]), t1 = __builtin_amdgcn_readfirstlane(tp[b + 1]);
            const unsigned nb = t1 - t0, base = (unsigned)ngroups * t0;
            if (u >= base + (unsigned)ngroups * nb) {  // past the sequence, or none of it
              ++b;
              continue;
            }
            const unsigned grp = (u - base) / nb, i0 = (u - base) - grp * nb;
            const unsigned stop = min(u_end, base + (grp + 1) * nb);
            const int kh = grp * hg + head;
            const int i1 = (int)(i0 + (stop - u));
            u = stop;
            if (kh >= Hkv) continue;
            range(r, b, kh, __builtin_amdgcn_readfirstlane(lens[b]), (int)i0, i1,
                  (int64_t)v + (int64_t)b * ngroups + grp);
            return true;
          }
          return false;
        },
        scales[wave], ws_o, ws_ml);
  }
}

}  // namespace
}  // namespace lfs

using namespace lfs;

extern "C" int64_t lfs_paged_decode_fp8_workspace_bytes(int64_t B, int32_t num_q_heads, int32_t head_dim) {
  if (B < 0 || num_q_heads <= 0 || head_dim <= 0) return -1;
  if (B > BAL_MAXB) return 0;
  // partial rows of D + 2 floats, as lfs_paged_decode's balanced split, and the scan
  return 4 * (8 * (int64_t)decode_cu_count() + 2 * B) * num_q_heads * ((int64_t)head_dim + 2) + 4 * (B + 1);
}

extern "C" int lfs_paged_decode_fp8(const void* q, const void* k_cache, const void* v_cache, const float* k_scale,
                                    const float* v_scale, const int64_t* context_lens, const int32_t* block_tables,
                                    int64_t bt_stride, void* out, void* workspace, int64_t workspace_bytes, int64_t B,
                                    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                    int64_t num_blocks, int32_t max_blocks, float scale, void* q_out, float* q_scale,
                                    void* stream) {
  const int Hq = num_q_heads, Hkv = num_kv_heads, D = head_dim, BS = block_size;
  int rc = check_decode("paged_decode_fp8", q, k_cache, v_cache, context_lens, block_tables, bt_stride, out, workspace,
                        workspace_bytes, lfs_paged_decode_fp8_workspace_bytes(B, Hq, D), B, Hq, Hkv, D, BS, num_blocks,
                        max_blocks, q_out, q_scale);
  if (rc || B == 0) return rc;
  LFS_REQUIRE(k_scale && v_scale, "paged_decode_fp8: null pointer");
  LFS_REQUIRE(((((uintptr_t)k_scale) | ((uintptr_t)v_scale)) & 15u) == 0,
              "paged_decode_fp8: the scales must be 16-byte aligned");
  LFS_REQUIRE((int64_t)Hkv * D * 128 < (1ll << 31), "paged_decode_fp8: too many kv heads (%d)", Hkv);
  const int T = 64, G = Hq / Hkv;
  const BalancedGeom bg = balanced_geom(Hkv);
  const bool scan = B <= BAL_MAXB, one = BS % T == 0;
  LFS_REQUIRE((int64_t)bg.ngroups * B * (((int64_t)max_blocks * BS + T - 1) / T) < (1ll << 31),
              "paged_decode_fp8: too many context tiles");
  LFS_REQUIRE((int64_t)max_blocks * BS < (1ll << 31) - 256, "paged_decode_fp8: block tables of 2^31 tokens");
  const int64_t rows = ((int64_t)bg.nwg + B * bg.ngroups) * bg.wpg * G;
  float* ws_o = (float*)workspace;
  float* ws_ml = ws_o + rows * D;
  int* tp = (int*)(ws_ml + rows * 2);
  const int64_t per = 4 / bg.wpg;  // shares a workgroup
  const dim3 grid((unsigned)(scan ? bg.nwg / per : (B * bg.ngroups + per - 1) / per)), block(256);
  hipStream_t st = (hipStream_t)stream;
#define LFS_FP8(DD, ONE, SCAN)                                                                                        \
  hipLaunchKernelGGL((paged_fp8_kernel<DD, ONE, SCAN>), grid, block, 0, st, (const uint16_t*)q, (const uint8_t*)k_cache, \
                     (const uint8_t*)v_cache, k_scale, v_scale, context_lens, block_tables, bt_stride, ws_o, ws_ml, tp, \
                     (uint16_t*)out, Hkv, G, BS, num_blocks, max_blocks, (int)B, scale * 1.4426950408889634f, bg.ngroups, bg.wpg)
  if (D == 64) {
    if (!scan) LFS_FP8(64, false, false);
    else if (one) LFS_FP8(64, true, true);
    else LFS_FP8(64, false, true);
  } else {
    if (!scan) LFS_FP8(128, false, false);
    else if (one) LFS_FP8(128, true, true);
    else LFS_FP8(128, false, true);
  }
#undef LFS_FP8
  rc = check_launch("paged_decode_fp8");
  if (rc) return rc;
  if (scan)
    return paged_decode_merge_launch(ws_o, ws_ml, context_lens, out, q_out, q_scale, B, Hq, D, BS, max_blocks,
                                     PartMap{0, 0, tp, T, bg.ngroups, bg.wpg, G, bg.nwg, (int)B}, st);
  if (q_out == nullptr) return 0;
  return lfs_act_quant(out, Hq * D, q_out, q_scale, B, Hq * D, 128, 0, stream);
}
