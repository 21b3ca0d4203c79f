// GQA decode over a KV pool in 8 bits: codes e4m3fn [NB, BS, Hkv, D], scales
// fp32 [NB, Hkv, BS] per token and kv head.  With K = s_k k and V = s_v v,
//   o = sum_t w_t s_v,t v_t / sum_t w_t,   w_t = exp(scale s_k,t (q . k_t) - m).
//
// One wave per (sequence, kv head, range of tiles of T tokens).  Per tile:
//   S = k q^T  v_mfma_f32_16x16x32_bf16, the codes converted (exactly) two at a
//              time.  Not the FP8 MFMAs: on gfx950 their sums are off by up to
//              2^-12 of the largest product (measured on sums of 32 to 128 random
//              products), which a weight would show.  Columns j and j + 8 of q^T
//              are the same head;
//   softmax    online, log2 domain; lane l holds the scores of head l % 8 for
//              tokens 4 (l / 16) .. +3 of every 16-token group;
//   O^T += v^T P^T  v_mfma_f32_16x16x32_bf16 (codes are exact in bf16): P^T is the
//              B operand straight from the softmax registers, k-index 8 kq + i
//              standing for token 4 kq + i of the pair's first 16-token group (i <
//              4) or 4 kq + i - 4 of its second.  Lane (m, kq) loads D / 16 codes of
//              those eight tokens, at dims m D / 16 on: pairs of tokens are put
//              beside each other by byte permutes and converted, so V is transposed
//              in registers.  Columns j and j + 8 are the weight s_v w rounded to
//              bf16 and what that left: 16 bits of it;
//   loads      a tile ahead, in two sets of registers, through buffer descriptors
//              that end behind the last visible row: rows past the context and of
//              blocks outside the pool read as zeros, whatever they hold.
// Work per CU is that of the balanced split of decode_wave.h: one 4-wave workgroup
// a CU, its waves on adjacent heads of the same rows.
#include "decode_wave.h"

namespace lfs {
namespace {


template <int D>
struct Fp8Geom {
  static constexpr int T = D == 64 ? 128 : 64;  // tokens per tile: 16 KiB of codes
  static constexpr int NG = T / 16;             // 16-token groups
  static constexpr int TU = T / 64;             // scales per lane
  static constexpr int KL = D / 64;             // 16-byte K loads per lane and group
  static constexpr int DB = D / 16;             // V codes per lane and token
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t pool_rows(const uint8_t* base, int64_t off, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base) + off, 0, bytes, 0x00020000);
}
// eight codes -> bf16 (exact)
__device__ __forceinline__ uint32_t bf16_lo(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
}
__device__ __forceinline__ uint32_t bf16_hi(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true));
}
__device__ __forceinline__ v8bf codes_bf16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(v8bf, make_uint4(bf16_lo(a), bf16_hi(a), bf16_lo(b), bf16_hi(b)));
}
constexpr int kNt = 2;  // nontemporal: every row is read once

template <int D, bool ONE>
struct Fp8Wave {
  using Geo = Fp8Geom<D>;
  static constexpr int NG = Geo::NG, TU = Geo::TU, KL = Geo::KL, DB = Geo::DB, T = Geo::T;
  struct Tile {
    u32x4 k[NG][KL];
    uint32_t v[NG][4][DB / 4];
    float ks[TU], vs[TU];
    int n;         // tokens up to the context's end (at most T)
    uint32_t bad;  // bit g: group g lies in no block of the pool
  };

  int lane, j, kq, kh, Hkv, BS, row;
  int64_t NB;
  const uint8_t *kc, *vc;
  const float *ksc, *vsc;
  v8bf q[D / 32];
  float scale_log2, acc[DB][4], m_run, l_run;
  // the walk: columns and offsets of the next tile whose ids are asked for
  const int32_t* btrow;
  int64_t id_end, left;
  int col[TU], off[TU], ids[TU], idoff[TU], sq, sr;

  // Lane (j, kq) holds dims 64 x + 16 kq .. +15 of head j % 8.
  __device__ __forceinline__ void load_q(const uint16_t* qp, int G) {
    const int h = j & 7;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (h < G) w = *reinterpret_cast<const uint4*>(qp + h * D + (c >> 1) * 64 + kq * 16 + (c & 1) * 8);
      q[c] = __builtin_bit_cast(v8bf, w);
    }
  }

  __device__ __forceinline__ void start(const int32_t* bt_row, int64_t t_begin, int64_t t_end) {
    btrow = bt_row;
    id_end = block_of(t_end - 1, BS) + 1;
    left = t_end - t_begin;
#pragma unroll
    for (int u = 0; u < TU; ++u) {
      const int64_t t = t_begin + u * 64 + (lane >> 4) * 16, c = block_of(t, BS);
      col[u] = (int)c;
      off[u] = (int)(t - c * BS);
    }
    sq = T / BS;
    sr = T - sq * BS;
#pragma unroll
    for (int e = 0; e < DB; ++e)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[e][r] = 0.f;
    m_run = -INFINITY;
    l_run = 0.f;
  }
  // Ask for the next tile's block ids; columns past the context's are not read.
  __device__ __forceinline__ void ask() {
#pragma unroll
    for (int u = 0; u < TU; ++u) {
      ids[u] = -1;
      if (col[u] < id_end) ids[u] = btrow[col[u]];
      idoff[u] = off[u];
      col[u] += sq;
      off[u] += sr;
      if (off[u] >= BS) off[u] -= BS, ++col[u];
    }
  }
  // Load the tile whose ids were asked for.
  __device__ __forceinline__ void load(Tile& t) {
    const int n = (int)max((int64_t)0, min((int64_t)T, left));
    left -= T;
    t.n = n;
    uint32_t bad = 0;
    int64_t at[TU];
#pragma unroll
    for (int u = 0; u < TU; ++u) {
      const bool ok = ids[u] >= 0 && (int64_t)ids[u] < NB;
      const int64_t slot = (int64_t)(ok ? ids[u] : 0) * BS + idoff[u];
      at[u] = slot * row + (int64_t)kh * D;
      const int tok = u * 64 + lane;
      const int64_t sat = ((int64_t)(ok ? ids[u] : 0) * Hkv + kh) * BS + idoff[u] + (lane & 15);
      const bool use = ok && tok < n;
      const float a = ksc[sat], b = vsc[sat];
      t.ks[u] = use ? a : 0.f;
      t.vs[u] = use ? b : 0.f;
      const uint64_t m = __ballot(!ok);
#pragma unroll
      for (int k = 0; k < 4; ++k) bad |= (uint32_t)(m >> (16 * k) & 1) << (u * 4 + k);
    }
    t.bad = bad;
    auto base_of = [&](int g) {
      const int u = g >> 2, l = (g & 3) * 16;
      const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)at[u], l);
      const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)at[u] >> 32), l);
      return (int64_t)((uint64_t)hi << 32 | lo);
    };
    const int kat = j * row + kq * 16, vat = kq * 4 * row + j * DB;
    const int64_t b0 = base_of(0);
    const int all = ONE && n > 0 && !(bad & 1) ? (n - 1) * row + D : 0;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      int64_t b = b0;
      int bytes = all, soff = g * 16 * row;
      if constexpr (!ONE) {
        b = base_of(g);
        const int rows = min(16, n - g * 16);
        bytes = rows > 0 && !(bad >> g & 1) ? (rows - 1) * row + D : 0;
        soff = 0;
      }
      const auto kr = pool_rows(kc, b, bytes);
#pragma unroll
      for (int x = 0; x < KL; ++x)
        t.k[g][x] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(kr, kat + x * 64, soff, kNt));
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      int64_t b = b0;
      int bytes = all, soff = g * 16 * row;
      if constexpr (!ONE) {
        b = base_of(g);
        const int rows = min(16, n - g * 16);
        bytes = rows > 0 && !(bad >> g & 1) ? (rows - 1) * row + D : 0;
        soff = 0;
      }
      const auto vr = pool_rows(vc, b, bytes);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (DB == 4) {
          t.v[g][r][0] = __builtin_amdgcn_raw_buffer_load_b32(vr, vat + r * row, soff, kNt);
        } else {
          const auto w = __builtin_amdgcn_raw_buffer_load_b64(vr, vat + r * row, soff, kNt);
          t.v[g][r][0] = w[0];
          t.v[g][r][1] = w[1];
        }
      }
    }
  }

  // pw: the wave's LDS slice, 2 T floats.
  __device__ __forceinline__ void compute(const Tile& t, float* __restrict__ pw) {
#pragma unroll
    for (int u = 0; u < TU; ++u) {
      pw[u * 64 + lane] = t.ks[u];
      pw[T + u * 64 + lane] = t.vs[u];
    }
    wave_lds_sync();
    float s[NG][4];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      v4f sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < KL; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const v8bf a = codes_bf16(t.k[g][x][2 * c], t.k[g][x][2 * c + 1]);
          sc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[2 * x + c], sc, 0, 0, 0);
        }
      const float4 ks = *reinterpret_cast<const float4*>(pw + g * 16 + kq * 4);
      const float kf[4] = {ks.x, ks.y, ks.z, ks.w};
#pragma unroll
      for (int r = 0; r < 4; ++r) s[g][r] = sc[r] * (scale_log2 * kf[r]);
    }
    if (t.n < T || t.bad) {
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if ((t.bad >> g & 1) || g * 16 + kq * 4 + r >= t.n) s[g][r] = -INFINITY;
    }
    float tmax = -INFINITY;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) tmax = fmaxf(tmax, s[g][r]);
    tmax = max_xor32(max_xor16(tmax));
    const float m_new = fmaxf(m_run, tmax);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    if (__any(m_new != m_run)) {
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
      l_run *= alpha;
#pragma unroll
      for (int e = 0; e < DB; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[e][r] *= alpha;
      m_run = m_new;
    }
    const uint32_t low = j < 8 ? 0u : 0xFFFF0000u;  // columns 8 .. 15 take what the rounding left
#pragma unroll
    for (int p = 0; p < NG / 2; ++p) {
      uint32_t w[4];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int g = 2 * p + y;
        const float4 vs = *reinterpret_cast<const float4*>(pw + T + g * 16 + kq * 4);
        const float vf[4] = {vs.x, vs.y, vs.z, vs.w};
        float x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[r] = __builtin_amdgcn_exp2f(s[g][r] - m_use);
          l_run += x[r];
          x[r] *= vf[r];
        }
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          const uint32_t hi = pack_bf16x2(x[r], x[r + 1]);
          w[y * 2 + r / 2] = pack_bf16x2(x[r] - __uint_as_float(hi << 16 & low), x[r + 1] - __uint_as_float(hi & low));
        }
      }
      const v8bf pb = __builtin_bit_cast(v8bf, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
      for (int d = 0; d < DB / 4; ++d) {
        uint32_t a[4][4];  // [code of the dword][pair of tokens]
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t t0 = t.v[2 * p + i / 2][(i & 1) * 2][d], t1 = t.v[2 * p + i / 2][(i & 1) * 2 + 1][d];
          const uint32_t x01 = __builtin_amdgcn_perm(t1, t0, 0x05010400u), x23 = __builtin_amdgcn_perm(t1, t0, 0x07030602u);
          a[0][i] = bf16_lo(x01), a[1][i] = bf16_hi(x01), a[2][i] = bf16_lo(x23), a[3][i] = bf16_hi(x23);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v4f c = {acc[4 * d + e][0], acc[4 * d + e][1], acc[4 * d + e][2], acc[4 * d + e][3]};
          c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(v8bf, make_uint4(a[e][0], a[e][1], a[e][2], a[e][3])), pb, c, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[4 * d + e][r] = c[r];
        }
      }
    }
    wave_lds_sync();
  }

  __device__ __forceinline__ void walk(const int32_t* bt_row, int64_t t_begin, int64_t t_end, float* __restrict__ pw) {
    start(bt_row, t_begin, t_end);
    const int nt = (int)((t_end - t_begin + T - 1) / T);
    Tile a, b;
    ask();
    load(a);
    ask();
    for (int i = 0; i < nt; i += 2) {
      __builtin_amdgcn_sched_barrier(0);
      load(b);
      ask();
      __builtin_amdgcn_sched_barrier(0);
      compute(a, pw);
      if (i + 1 >= nt) break;
      __builtin_amdgcn_sched_barrier(0);
      load(a);
      ask();
      __builtin_amdgcn_sched_barrier(0);
      compute(b, pw);
    }
  }

  // The normalised output of the whole context, or the partial (o, m, l) of
  // query head kh G + j to row prow + j of the workspace.
  __device__ __forceinline__ void finish(bool whole, uint16_t* __restrict__ out, float* __restrict__ ws_o,
                                         float* __restrict__ ws_ml, int64_t prow, int G) {
    const float l = sum_xor32(sum_xor16(l_run));
    const float inv = l > 0.f ? 1.f / l : 0.f;
    float o[4][DB];
#pragma unroll
    for (int e = 0; e < DB; ++e)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r][e] = xor_sum<8>(acc[e][r]) * (whole ? inv : 1.f);
    if (j >= G) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = (kq * 4 + r) * DB;
      if (whole) {
#pragma unroll
        for (int e = 0; e < DB; e += 4)
          *reinterpret_cast<uint2*>(out + (int64_t)j * D + d + e) =
              make_uint2(pack_bf16x2(o[r][e], o[r][e + 1]), pack_bf16x2(o[r][e + 2], o[r][e + 3]));
      } else {
#pragma unroll
        for (int e = 0; e < DB; e += 4)
          *reinterpret_cast<float4*>(ws_o + (prow + j) * D + d + e) =
              make_float4(o[r][e], o[r][e + 1], o[r][e + 2], o[r][e + 3]);
      }
    }
    if (!whole && kq == 0) {
      ws_ml[(prow + j) * 2 + 0] = m_run;
      ws_ml[(prow + j) * 2 + 1] = l;
    }
  }
};

// SCAN: a fixed grid shares the tiles of the batch (paged_decode_balanced's
// split); else a workgroup per (sequence, group of kv heads) walks the whole
// context.
template <int D, bool ONE, bool SCAN>
__global__ __launch_bounds__(256) void paged_fp8_kernel(
    const uint16_t* __restrict__ q, const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
    const float* __restrict__ ksc, const float* __restrict__ vsc, const int64_t* __restrict__ ctx_lens,
    const int32_t* __restrict__ bt, int64_t bt_stride, float* __restrict__ ws_o, float* __restrict__ ws_ml,
    int* __restrict__ tp_out, uint16_t* __restrict__ out, int Hkv, int G, int BS, int64_t NB, int max_blocks, int B,
    float scale_log2, int ngroups) {
  constexpr int T = Fp8Geom<D>::T;
  __shared__ __attribute__((aligned(16))) float scales[4][2 * T];
  __shared__ int tp[SCAN ? BAL_MAXB + 1 : 1];
  __shared__ int wsum[4];
  const int tid = threadIdx.x, wpg = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int64_t cap = (int64_t)max_blocks * BS;
  Fp8Wave<D, ONE> w;
  w.lane = lane, w.j = lane & 15, w.kq = lane >> 4;
  w.Hkv = Hkv, w.BS = BS, w.row = Hkv * D, w.NB = NB;
  w.scale_log2 = scale_log2;
  w.kc = kc, w.vc = vc, w.ksc = ksc, w.vsc = vsc;
  auto range = [&](int b, int grp, int64_t i0, int64_t i1, int64_t slot) {
    const int kh = grp * wpg + wave;
    if (kh >= Hkv) return;
    const int64_t Lc = min(ctx_lens[b], cap), t0 = i0 * T, t1 = min(Lc, i1 * T);
    uint16_t* o = out + ((int64_t)b * Hkv + kh) * G * D;
    if (t0 >= t1) {  // no context (SCAN: never)
      for (int i = lane; i < G * D / 2; i += 64) reinterpret_cast<uint32_t*>(o)[i] = 0;
      return;
    }
    w.kh = kh;
    w.load_q(q + ((int64_t)b * Hkv + kh) * G * D, G);
    w.walk(bt + (int64_t)b * bt_stride, t0, t1, scales[wave]);
    w.finish(t0 == 0 && t1 >= Lc, o, ws_o, ws_ml, (slot * wpg + wave) * G, G);
  };
  if constexpr (!SCAN) {
    const int b = (int)(blockIdx.x / (unsigned)ngroups), grp = (int)(blockIdx.x - (unsigned)b * ngroups);
    range(b, grp, 0, 1ll << 40, 0);
  } else {
    scan_tiles(tp, wsum, B, [&](int b) { return decode_tiles(ctx_lens, b, cap, T); });
    if (blockIdx.x == 0)
      for (int i = tid; i <= B; i += blockDim.x) tp_out[i] = tp[i];
    const unsigned total = (unsigned)ngroups * (unsigned)tp[B], nwg = gridDim.x;
    const unsigned Ct = max(1u, (total + nwg - 1) / nwg);
    unsigned u = blockIdx.x * Ct;
    const unsigned u_end = min(total, u + Ct);
    if (u >= u_end) return;
    int b = 0, b_hi = B - 1;  // the largest b with ngroups * tp[b] <= u
    while (b < b_hi) {
      const int mid = (b + b_hi + 1) >> 1;
      if ((unsigned)ngroups * (unsigned)tp[mid] <= u) b = mid;
      else b_hi = mid - 1;
    }
    while (u < u_end) {
      const unsigned nb = tp[b + 1] - tp[b], base = (unsigned)ngroups * (unsigned)tp[b];
      const unsigned grp = (u - base) / nb, i0 = (u - base) - grp * nb;
      const unsigned seg_end = min(u_end, base + (grp + 1) * nb);
      range(b, (int)grp, i0, i0 + (seg_end - u), (int64_t)blockIdx.x + (int64_t)b * ngroups + grp);
      u = seg_end;
      if (u >= base + ngroups * nb) {
        ++b;
        while (b < B && tp[b + 1] == tp[b]) ++b;
      }
    }
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
  const int T = D == 64 ? 128 : 64, G = Hq / Hkv;
  const BalancedGeom bg = balanced_geom(Hkv);
  const bool scan = B <= BAL_MAXB, one = BS % T == 0;
  LFS_REQUIRE((int64_t)bg.ngroups * B * (((int64_t)max_blocks * BS + T - 1) / T) < (1ll << 31),
              "paged_decode_fp8: too many context tiles");
  const int64_t rows = ((int64_t)bg.nwg + B * bg.ngroups) * bg.wpg * G;
  float* ws_o = (float*)workspace;
  float* ws_ml = ws_o + rows * D;
  int* tp = (int*)(ws_ml + rows * 2);
  const dim3 grid((unsigned)(scan ? bg.nwg : B * bg.ngroups)), block((unsigned)(64 * bg.wpg));
  hipStream_t st = (hipStream_t)stream;
#define LFS_FP8(DD, ONE, SCAN)                                                                                        \
  hipLaunchKernelGGL((paged_fp8_kernel<DD, ONE, SCAN>), grid, block, 0, st, (const uint16_t*)q, (const uint8_t*)k_cache, \
                     (const uint8_t*)v_cache, k_scale, v_scale, context_lens, block_tables, bt_stride, ws_o, ws_ml, tp, \
                     (uint16_t*)out, Hkv, G, BS, num_blocks, max_blocks, (int)B, scale * 1.4426950408889634f, bg.ngroups)
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
