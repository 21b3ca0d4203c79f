// One wave's walk over the tiles of one (sequence, kv head) of a paged KV pool,
// the balanced split of a batch into such walks, and their log-sum-exp merge:
// shared by the paged decode (paged_kv.hip) and the decode over a sliding
// window (paged_window.hip).
#pragma once

#include "common.h"

namespace lfs {
namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// One wave per (sequence, kv head, range of the context).  Per tile of T
// tokens (one KV block never straddled):
//   K  : MFMA A operand straight from HBM -- lane l loads token (l % 16) of a
//        16-token group, dims c*32 + (l / 16)*8 .. +7 (16 B);
//   q^T: MFMA B operand, column j = l % 16 is query head kh*G + j (zero for
//        j >= G);
//   S  = K q^T with v_mfma_f32_16x16x32_bf16: lane l ends with the scores of
//        head (l % 16) for tokens 4*(l / 16) .. +3 of each group, so the
//        online-softmax max/sum per head is a 2-step xor over lanes 16, 32;
//   P  goes through a wave-private LDS slice [T][G] to the P.V mapping;
//   V  : lane l owns token (l / (D/8)) + (64/(D/8))*i and dims
//        (l % (D/8))*8 .. +7 (coalesced 16-byte loads), fp32 FMAs into
//        acc[G][8], rescaled by exp2(m_old - m_new) read from lane g.
// Loads are software-pipelined one tile ahead (two K and two V buffers: a
// step issues the next tile's loads, then computes on the tile loaded by
// the step before) with nontemporal 16-byte loads, since every KV row is
// read exactly once.  One tile in flight per wave is 16 KiB, 16 MiB over
// the chip: enough to keep HBM busy, and a new request does not queue
// behind twice that (two tiles ahead measured 4 % slower on every decode
// shape).  There is no workgroup barrier: waves exit independently.  A
// range that covers the whole context writes the normalised bf16 output
// directly; otherwise the unnormalised partial (o, m, l) goes to the
// workspace for the merge.
template <int D>
struct DecodeGeom {
  static constexpr int LPR = D / 8;               // lanes per token row in the P.V mapping
  static constexpr int TPI = 64 / LPR;            // tokens per V load instruction
  static constexpr int T = (D == 64) ? 64 : 32;   // tokens per tile
  static constexpr int NG = T / 16;               // 16-token MFMA groups per tile
  static constexpr int NDC = D / 32;              // 32-wide head-dim chunks
  static constexpr int UV = T / TPI;              // V loads per lane per tile
};

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
// 16-byte streaming load (nontemporal: the KV rows are read exactly once)
__device__ __forceinline__ uint4 nt_load16(const uint16_t* p) {
  const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// Reductions over lanes l, l^16 (and l^32) without LDS: v_permlane16_swap
// (v_permlane32_swap) of a value with itself leaves the value of lane l in
// one result and that of lane l^16 (l^32) in the other, in both lanes of the
// pair.  Same operands in the same order as x op __shfl_xor(x, 16 / 32), so
// the results are bit-identical (IEEE add and max are commutative).
__device__ __forceinline__ float max_xor16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_xor16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float sum_xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The per-wave pieces of a decode range.  A tile is (n, off): n valid rows
// (0 for a skipped block or a look-ahead filler) starting at element offset
// off of the cache.
template <int D, int G>
struct DecodeWave {
  using Geo = DecodeGeom<D>;
  static constexpr int GP = G <= 4 ? 4 : 8;  // padded heads per token in the P slice
  typedef uint4 KBuf[Geo::NG][Geo::NDC];
  typedef uint4 VBuf[Geo::UV];
  typedef uint4 QBuf[Geo::NDC];

  int lane, j, kq, ts, dc;
  int64_t row;  // elements per token row of the cache (Hkv * D)
  float acc[G][8];
  float m_run, l_run;

  __device__ __forceinline__ DecodeWave(int lane_, int Hkv) : lane(lane_) {
    j = lane & 15;
    kq = lane >> 4;
    ts = lane / Geo::LPR;
    dc = lane % Geo::LPR;
    row = (int64_t)Hkv * D;
    reset();
  }
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[g][e] = 0.f;
    m_run = -INFINITY;
    l_run = 0.f;
  }
  // q^T columns of kv head kh of sequence b (lanes j >= G load nothing)
  __device__ __forceinline__ void load_q(QBuf& qa, const uint16_t* __restrict__ q, int64_t b, int kh, int Hq) const {
#pragma unroll
    for (int c = 0; c < Geo::NDC; ++c) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (j < G) w = *reinterpret_cast<const uint4*>(q + ((int64_t)b * Hq + kh * G + j) * D + c * 32 + kq * 8);
      qa[c] = w;
    }
  }
  // the same from a [G][D] bf16 block in LDS (this kv head's query rows)
  __device__ __forceinline__ void load_q_lds(QBuf& qa, const uint16_t* ql) const {
#pragma unroll
    for (int c = 0; c < Geo::NDC; ++c) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (j < G) w = *reinterpret_cast<const uint4*>(ql + j * D + c * 32 + kq * 8);
      qa[c] = w;
    }
  }
  // a tile whose rows are all the one token row k / v (bf16 [D] each, in
  // LDS): with n = 1 in tile() it adds that single token
  __device__ __forceinline__ void row_tile(KBuf& ka, VBuf& va, const uint16_t* kl, const uint16_t* vl) const {
#pragma unroll
    for (int g16 = 0; g16 < Geo::NG; ++g16)
#pragma unroll
      for (int c = 0; c < Geo::NDC; ++c) ka[g16][c] = *reinterpret_cast<const uint4*>(kl + c * 32 + kq * 8);
#pragma unroll
    for (int i = 0; i < Geo::UV; ++i) va[i] = *reinterpret_cast<const uint4*>(vl + dc * 8);
  }
  // Every load is issued unconditionally: rows past the valid count n read
  // row n-1 (row 0 of block 0 for a skipped block), whose scores are masked
  // and whose P is 0 (a skipped block's P.V is not run).  Offsets inside a
  // tile are 32-bit from a wave-uniform base.  LO: rows below lo (< n) are
  // hidden, read row lo and get the same treatment.
  template <bool LO = false>
  __device__ __forceinline__ void load_k(KBuf& ka, const uint16_t* __restrict__ kc, int n, int64_t off,
                                         int lo = 0) const {
    const uint16_t* kb = kc + off;
    const int nn = max(n, 1);
#pragma unroll
    for (int g16 = 0; g16 < Geo::NG; ++g16) {
      int tr = min(g16 * 16 + j, nn - 1);
      if constexpr (LO) tr = max(tr, lo);
#pragma unroll
      for (int c = 0; c < Geo::NDC; ++c)
        ka[g16][c] = nt_load16(kb + (uint32_t)(tr * (int)row + c * 32 + kq * 8));
    }
  }
  template <bool LO = false>
  __device__ __forceinline__ void load_v(VBuf& va, const uint16_t* __restrict__ vc, int n, int64_t off,
                                         int lo = 0) const {
    const uint16_t* vb = vc + off;
    const int nn = max(n, 1);
#pragma unroll
    for (int i = 0; i < Geo::UV; ++i) {
      int tr = min(ts + Geo::TPI * i, nn - 1);
      if constexpr (LO) tr = max(tr, lo);
      va[i] = nt_load16(vb + (uint32_t)(tr * (int)row + dc * 8));
    }
  }

  // One tile of n valid rows (LO: rows lo .. n - 1): scores (log2 domain),
  // online-softmax update for head j, P through the LDS slice pw, P.V into
  // acc.
  template <bool LO = false>
  __device__ __forceinline__ void tile(const KBuf& ka, const VBuf& va, const QBuf& qa, int n, float scale_log2,
                                       float* __restrict__ pw, int lo = 0) {
    float s[Geo::NG][4];
    float tmax = -INFINITY;
#pragma unroll
    for (int g16 = 0; g16 < Geo::NG; ++g16) {
      v4f sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < Geo::NDC; ++c)
        sc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, ka[g16][c]),
                                                     __builtin_bit_cast(v8bf, qa[c]), sc, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int tok = g16 * 16 + kq * 4 + r;
        s[g16][r] = tok < n && (!LO || tok >= lo) ? sc[r] * scale_log2 : -INFINITY;
        tmax = fmaxf(tmax, s[g16][r]);
      }
    }
    tmax = max_xor16(tmax);
    tmax = max_xor32(tmax);
    const float m_new = fmaxf(m_run, tmax);
    const bool live = m_new != -INFINITY;
    const float alpha = live ? exp2f(m_run - m_new) : 1.f;
    float psum = 0.f;
#pragma unroll
    for (int g16 = 0; g16 < Geo::NG; ++g16)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = live ? exp2f(s[g16][r] - m_new) : 0.f;
        psum += p;
        if (j < G) pw[(g16 * 16 + kq * 4 + r) * GP + j] = p;
      }
    psum = sum_xor16(psum);
    psum = sum_xor32(psum);
    l_run = l_run * alpha + psum;
    m_run = m_new;
    wave_lds_sync();

    // P.V (rows past n have P = 0; a skipped block adds nothing)
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float a = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(alpha), g));
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[g][e] *= a;
    }
    if (n > 0) {
#pragma unroll
      for (int iv = 0; iv < Geo::UV; ++iv) {
        const int tok = ts + Geo::TPI * iv;
        float pg[GP];
#pragma unroll
        for (int g4 = 0; g4 < GP; g4 += 4) {
          const float4 p4 = *reinterpret_cast<const float4*>(&pw[tok * GP + g4]);
          pg[g4] = p4.x; pg[g4 + 1] = p4.y; pg[g4 + 2] = p4.z; pg[g4 + 3] = p4.w;
        }
        float vf[8];
        unpack8(va[iv], vf);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[g][e] = fmaf(pg[g], vf[e], acc[g][e]);
      }
    }
    wave_lds_sync();
  }

  // End of a range: sum the token subgroups (lanes with the same dc), then
  // the normalised bf16 output of query heads kh*G + g (whole context) or
  // the unnormalised partial to workspace rows prow + g.
  // Sum acc over the token subgroups: afterwards lanes with ts == 0 hold the
  // wave's totals for dims dc*8 .. +7 of every head.
  // (distances LPR, 2 LPR, ..., 32: the same sums as acc += __shfl_xor(acc, o))
  template <int O = Geo::LPR>
  __device__ __forceinline__ void reduce_lanes() {
    if constexpr (O < 64) {
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[g][e] = xor_sum<O>(acc[g][e]);
      reduce_lanes<2 * O>();
    }
  }
  __device__ __forceinline__ void finish(bool whole, uint16_t* __restrict__ out, float* __restrict__ ws_o,
                                         float* __restrict__ ws_ml, int64_t b, int kh, int Hq, int64_t prow) {
    reduce_lanes();
    if (whole) {
      if (ts == 0) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float lg = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(l_run), g));
          const float inv = lg > 0.f ? 1.f / lg : 0.f;
          uint4 o;
          o.x = pack_bf16x2(acc[g][0] * inv, acc[g][1] * inv);
          o.y = pack_bf16x2(acc[g][2] * inv, acc[g][3] * inv);
          o.z = pack_bf16x2(acc[g][4] * inv, acc[g][5] * inv);
          o.w = pack_bf16x2(acc[g][6] * inv, acc[g][7] * inv);
          *reinterpret_cast<uint4*>(out + (b * Hq + kh * G + g) * D + dc * 8) = o;
        }
      }
    } else {
      if (ts == 0) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float* dst = ws_o + (prow + g) * D + dc * 8;
          *reinterpret_cast<float4*>(dst) = make_float4(acc[g][0], acc[g][1], acc[g][2], acc[g][3]);
          *reinterpret_cast<float4*>(dst + 4) = make_float4(acc[g][4], acc[g][5], acc[g][6], acc[g][7]);
        }
      }
      if (lane < G) {
        ws_ml[(prow + lane) * 2 + 0] = m_run;
        ws_ml[(prow + lane) * 2 + 1] = l_run;
      }
    }
  }
};

// One wave streams tiles of kv head kh of one sequence into w: tile i of the
// walk covers context rows [t_begin + i*tstride*tile, +tile) clipped to
// t_end (t_begin a multiple of `tile`, t_end <= the context length), so a
// range of consecutive tiles is tstride 1 and every S-th tile from s*tile
// is t_begin = s*tile, tstride S.  btrow: the sequence's block-table row;
// block ids at or past id_end are never loaded.  pw: the wave's private
// LDS slice (T * GP floats).  LO: rows below `first`, which lies in the first
// tile or before it, are hidden.  pro() runs once, after the first tile's loads
// are issued and before anything reads qa (a caller may fill qa there); an
// empty walk does not run it.
struct NoPrologue {
  __device__ __forceinline__ void operator()() const {}
};
// t / BS for t >= 0, by a 32-bit divide where t < 2^31 (every real pool)
__device__ __forceinline__ int64_t block_of(int64_t t, int BS) {
  return t >> 31 ? t / BS : (int64_t)((unsigned)t / (unsigned)BS);
}

template <int D, int G, bool LO = false, class Pro = NoPrologue>
__device__ __forceinline__ void decode_walk(
    DecodeWave<D, G>& w, const typename DecodeWave<D, G>::QBuf& qa, const uint16_t* __restrict__ kc,
    const uint16_t* __restrict__ vc, const int32_t* __restrict__ btrow, int BS, int64_t NB, int tile,
    float scale_log2, int kh, int64_t t_begin, int64_t t_end, int tstride, int64_t id_end,
    float* __restrict__ pw, Pro&& pro = Pro(), int64_t first = 0) {
  using W = DecodeWave<D, G>;
  const int lane = w.lane;
  const int64_t step_rows = (int64_t)tile * tstride;
  const int ntiles = (int)block_of(t_end - t_begin + step_rows - 1, (int)step_rows);
  // The walk's block ids, 256 at a time (window w0 .. w0 + 255 of the table
  // row): lane l holds ids 4l .. 4l+3 of the window, read back with
  // readlane, so no tile waits on a scalar load of its block id.  Ids at or
  // past id_end are never read (loaded as 0 to stay in bounds).  The window
  // is (re)loaded only where a group of MAXT tiles starts, and waited for
  // there: the group's tiles then read ids with no load pending on them, so
  // the compiler puts no vmcnt(0) between a tile's loads and the next
  // tile's (which would drain the tile in flight).  A group spans
  // (MAXT-1)*(tstride*tile/BS + 1) + 1 <= 256 blocks for tstride <= 35.
  int64_t w0 = -1;
  uint4 ids = make_uint4(0, 0, 0, 0);
  auto load_window = [&](int64_t wb) {
    w0 = wb;
    const int64_t e = wb + 4 * lane;
    uint32_t v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = e + c < id_end ? (uint32_t)btrow[e + c] : 0u;
    ids = make_uint4(v[0], v[1], v[2], v[3]);
    __builtin_amdgcn_s_waitcnt(0x0F70);
  };
  auto block_id = [&](int64_t bi) -> int32_t {
    const int e = __builtin_amdgcn_readfirstlane((int)(bi - w0));
    const int src = e >> 2, c = e & 3;
    const uint32_t x = c == 0 ? ids.x : c == 1 ? ids.y : c == 2 ? ids.z : ids.w;
    return (int32_t)__builtin_amdgcn_readlane((int)x, src);
  };
  // tile i of the walk: valid row count (0 for a skipped block) and the
  // element offset of its first row.  Tiles at or past `last` are
  // look-ahead fillers: n = 0 and row 0 of block 0, so their loads all hit
  // one line (they only keep the per-step load count constant).
  // The tiles are asked for in order, so the block column and the row within
  // the block of the next one are carried along: a divide per tile (64-bit,
  // some 100 instructions) would sit between a tile's arithmetic and the next
  // tile's loads.
  int last = 0;
  const int sq = (int)step_rows / BS, sr = (int)step_rows - sq * BS;
  int64_t left = t_end - t_begin, bi = block_of(t_begin, BS);
  int bo = (int)(t_begin - bi * BS);
  auto tile_at = [&](int i, int& n, int64_t& off) {
    if (i >= last) {
      n = 0;
      off = (int64_t)kh * D;
      return;
    }
    n = (int)min((int64_t)tile, left);
    const int32_t blk = block_id(bi);
    const bool ok = blk >= 0 && (int64_t)blk < NB;
    if (!ok) n = 0;  // invalid block: contributes nothing
    off = ((int64_t)(ok ? blk : 0) * BS + bo) * w.row + (int64_t)kh * D;
    left -= step_rows;
    bi += sq;
    bo += sr;
    if (bo >= BS) bo -= BS, ++bi;
  };

  // Pipeline one tile deep over two K and two V buffers: step i issues the
  // loads of tile i+1 into the other buffers, then computes tile i.  The
  // tiles of a walk are processed in straight-line code (MAXT steps
  // unrolled, with early exits), every step issuing the same loads, so the
  // compiler's in-order wait counts are exact: tile i waits only for its own
  // loads.  Walks longer than MAXT tiles go MAXT tiles at a time.
  constexpr int MAXT = 8;
  typename W::KBuf ka0, ka1;
  typename W::VBuf va0, va1;
  int nb0 = 0, nb1 = 0;
  int lo = LO ? (int)max((int64_t)0, first - t_begin) : 0;  // of the tile about to be computed: 0 past the first
  auto step = [&](int i, typename W::KBuf& ka, typename W::VBuf& va, int nb, typename W::KBuf& kx,
                  typename W::VBuf& vx, int& nbx) {
    int n1;
    int64_t o1;
    tile_at(i + 1, n1, o1);
    __builtin_amdgcn_sched_barrier(0);  // keep the issue order the wait counts assume
    w.load_k(kx, kc, n1, o1);
    w.load_v(vx, vc, n1, o1);
    __builtin_amdgcn_sched_barrier(0);
    nbx = n1;
    w.template tile<LO>(ka, va, qa, nb, scale_log2, pw, lo);
    lo = 0;
  };
  for (int base = 0; base < ntiles; base += MAXT) {
    last = min(ntiles, base + MAXT);
    {
      const int64_t bl = bi + (last - 1 - base) * (sq + 1);  // no tile of the group lies past it
      if (base == 0 || __builtin_amdgcn_readfirstlane((int)(bl >= w0 + 256))) load_window(bi);
    }
    {
      int64_t o0;
      tile_at(base, nb0, o0);
      w.template load_k<LO>(ka0, kc, nb0, o0, lo);
      w.template load_v<LO>(va0, vc, nb0, o0, lo);
    }
    if (base == 0) pro();
#pragma unroll
    for (int u = 0; u < MAXT; u += 2) {
      if (base + u >= last) break;
      step(base + u, ka0, va0, nb0, ka1, va1, nb1);
      if (base + u + 1 >= last) break;
      step(base + u + 1, ka1, va1, nb1, ka0, va0, nb0);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // drain the look-ahead loads
  }
  (void)lane;
}

// One wave: kv head kh of sequence b over context rows [t_begin, t_end)
// (t_begin a multiple of `tile`, t_end <= Lc).  A range that is the whole
// context (t_begin == 0, t_end >= Lc) writes the normalised bf16 output;
// otherwise the unnormalised partial of query head kh*G + g goes to row
// prow + g of the workspace (o: ws_o[row*D ..], (m, l): ws_ml[row*2 ..]).
// pw: the wave's private LDS slice (T * GP floats).
template <int D, int G>
__device__ __forceinline__ void decode_chunk(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ kc,
    const uint16_t* __restrict__ vc, const int32_t* __restrict__ btrow, float* __restrict__ ws_o,
    float* __restrict__ ws_ml, uint16_t* __restrict__ out, int Hkv, int BS, int64_t NB, int tile,
    float scale_log2, int b, int kh, int64_t t_begin, int64_t t_end, int64_t Lc, int64_t prow,
    float* __restrict__ pw, int lane) {
  using W = DecodeWave<D, G>;
  W w(lane, Hkv);
  const int Hq = Hkv * G;
  typename W::QBuf qa;
  w.load_q(qa, q, b, kh, Hq);
  decode_walk<D, G>(w, qa, kc, vc, btrow, BS, NB, tile, scale_log2, kh, t_begin, t_end, 1,
                    block_of(t_end - 1, BS) + 1, pw);
  w.finish(t_begin == 0 && t_end >= Lc, out, ws_o, ws_ml, b, kh, Hq, prow);
}

// Balanced split: a fixed grid of nwg workgroups (wpg waves each, one kv
// head per wave; one workgroup per CU) shares the work evenly, whatever the
// context lengths.
// Work units are (sequence b, kv-head group, tile) triples in that order,
// n_b = ceil(L_b / tile) tiles per (sequence, group), where L_b is the
// clamped context length; workgroup w takes the units [w*Ct, (w+1)*Ct),
// Ct = ceil(total / nwg), and its waves walk the same tiles for the heads of
// the group (so a workgroup reads wpg adjacent head slices of each row
// together).  A (sequence, group) range that one workgroup covers entirely
// is written out directly; otherwise workgroup w's partial of pair group
// pg = b*ngroups + group is slot (w + pg)*wpg + wave -- unique, since along
// the units both w and pg are non-decreasing and one of them grows at every
// step from one (pg, w) overlap to the next.  Every workgroup scans the
// per-sequence tile counts into LDS (B <= BAL_MAXB); workgroup 0 also
// writes the scan (B+1 ints) to tp_out for the merge.
constexpr int BAL_MAXB = 8192;

__device__ __forceinline__ int decode_tiles(const int64_t* ctx_lens, int b, int64_t cap, int tile) {
  const int64_t L = min(ctx_lens[b], cap);
  return L > 0 ? (int)((L + tile - 1) >> __builtin_ctz(tile)) : 0;  // tile is 16, 32 or 64
}

// A window over the contexts: of L tokens the last `size` are visible and the
// first `sinks`.  A sequence's visible rows are two ranges of tiles: of the
// sinks before the window, [0, sinks) clipped, and of the window, whose first
// tile may begin with hidden rows.
struct Window {
  int size, sinks;
};
struct WindowTiles {
  int64_t first, end, sk;  // the window's rows first .. end - 1, the sinks' 0 .. sk - 1
  int64_t w0;              // first row of the window's first tile
  int ns, nw;              // tiles of the sinks and of the window
  __device__ __forceinline__ WindowTiles(int64_t L, int64_t cap, int tile, const Window& w) {
    const int sh = __builtin_ctz(tile);
    L = max(L, (int64_t)0);
    first = max((int64_t)0, L - w.size);
    end = min(L, cap);
    sk = min(min((int64_t)w.sinks, first), end);
    w0 = first & -(int64_t)tile;
    ns = (int)((sk + tile - 1) >> sh);
    nw = end > first ? (int)((end - w0 + tile - 1) >> sh) : 0;
  }
};

// One wave: kv head kh of sequence b over the visible tiles i0 .. i1 - 1 (the
// sinks', then the window's), as decode_chunk.
template <int D, int G>
__device__ __forceinline__ void window_chunk(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ kc, const uint16_t* __restrict__ vc,
    const int32_t* __restrict__ btrow, float* __restrict__ ws_o, float* __restrict__ ws_ml, uint16_t* __restrict__ out,
    int Hkv, int BS, int64_t NB, int max_blocks, int tile, float scale_log2, int b, int kh, int i0, int i1,
    const WindowTiles& wt, int64_t prow, float* __restrict__ pw, int lane) {
  using W = DecodeWave<D, G>;
  W w(lane, Hkv);
  const int Hq = Hkv * G;
  typename W::QBuf qa;
  w.load_q(qa, q, b, kh, Hq);
  if (i0 < wt.ns)
    decode_walk<D, G>(w, qa, kc, vc, btrow, BS, NB, tile, scale_log2, kh, (int64_t)i0 * tile,
                      min(wt.sk, (int64_t)i1 * tile), 1, max_blocks, pw);
  const int64_t t0 = wt.w0 + (int64_t)max(0, i0 - wt.ns) * tile;
  const int64_t t1 = min(wt.end, wt.w0 + (int64_t)(i1 - wt.ns) * tile);
  if (t0 < t1)
    decode_walk<D, G, true>(w, qa, kc, vc, btrow, BS, NB, tile, scale_log2, kh, t0, t1, 1, max_blocks, pw,
                            NoPrologue(), wt.first);
  w.finish(i0 == 0 && i1 == wt.ns + wt.nw, out, ws_o, ws_ml, b, kh, Hq, prow);
}

// WIN: over a window.
template <int D, int G, bool WIN>
__global__ __launch_bounds__(256) void paged_decode_balanced(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ kc,
    const uint16_t* __restrict__ vc, const int64_t* __restrict__ ctx_lens,
    const int32_t* __restrict__ bt, int64_t bt_stride, float* __restrict__ ws_o,
    float* __restrict__ ws_ml, int* __restrict__ tp_out, uint16_t* __restrict__ out, int Hkv, int BS,
    int64_t NB, int max_blocks, int B, int tile, float scale_log2, int ngroups, Window win) {
  using Geo = DecodeGeom<D>;
  constexpr int GP = G <= 4 ? 4 : 8;
  __shared__ __attribute__((aligned(16))) float p_lds[4][Geo::T * GP];
  __shared__ int tp[BAL_MAXB + 1];
  __shared__ int wsum[4];
  const int tid = threadIdx.x, nthr = blockDim.x;
  const int wave = tid >> 6, lane = tid & 63, wpg = nthr >> 6;
  const int64_t cap = (int64_t)max_blocks * BS;

  // ---- tp[b] = sum of n_b' for b' < b (each thread a run of sequences)
  const int per = (B + nthr - 1) / nthr;
  const int lo = min(B, tid * per), hi = min(B, lo + per);
  int run = 0;
  for (int i = lo; i < hi; ++i) {
    if constexpr (WIN) {
      const WindowTiles wt(ctx_lens[i], cap, tile, win);
      run += wt.ns + wt.nw;
    } else {
      run += decode_tiles(ctx_lens, i, cap, tile);
    }
    tp[i + 1] = run;
  }
  int incl = run;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(incl, o, 64);
    if (lane >= o) incl += v;
  }
  if (lane == 63) wsum[wave] = incl;
  __syncthreads();
  int excl = incl - run;
  for (int w = 0; w < wave; ++w) excl += wsum[w];
  for (int i = lo; i < hi; ++i) tp[i + 1] += excl;
  if (tid == 0) tp[0] = 0;
  __syncthreads();
  if (blockIdx.x == 0)
    for (int i = tid; i <= B; i += nthr) tp_out[i] = tp[i];

  // 32-bit throughout: the host refuses 2^31 work units, and a 64-bit divide
  // is some 0.3 us of a chain that no other work hides
  const unsigned total = (unsigned)ngroups * (unsigned)tp[B];
  const unsigned nwg = gridDim.x;
  const unsigned Ct = max(1u, (total + nwg - 1) / nwg);
  unsigned u = blockIdx.x * Ct;
  const unsigned u_end = min(total, u + Ct);
  if (u >= u_end) return;
  // first sequence: the largest b with ngroups * tp[b] <= u (it has n_b > 0)
  int b_lo = 0, b_hi = B - 1;
  while (b_lo < b_hi) {
    const int mid = (b_lo + b_hi + 1) >> 1;
    if ((unsigned)ngroups * (unsigned)tp[mid] <= u) b_lo = mid;
    else b_hi = mid - 1;
  }
  int b = b_lo;
  float* pw = p_lds[wave];
  while (u < u_end) {
    const unsigned nb = tp[b + 1] - tp[b];
    const unsigned base = (unsigned)ngroups * (unsigned)tp[b];
    const int grp = (int)((u - base) / nb);
    const unsigned i0 = (u - base) - grp * nb;
    const unsigned seg_end = min(u_end, base + (grp + 1) * nb);
    const int kh = grp * wpg + wave;
    if (kh < Hkv) {
      const int64_t slot = ((int64_t)blockIdx.x + (int64_t)b * ngroups + grp) * wpg + wave;
      if constexpr (WIN) {
        const WindowTiles wt(ctx_lens[b], cap, tile, win);
        const int i1 = (int)(i0 + (seg_end - u));
        window_chunk<D, G>(q, kc, vc, bt + (int64_t)b * bt_stride, ws_o, ws_ml, out, Hkv, BS, NB, max_blocks, tile,
                           scale_log2, b, kh, (int)i0, i1, wt, slot * G, pw, lane);
      } else {
        const int64_t Lc = min(ctx_lens[b], cap);
        const int64_t t_begin = (int64_t)i0 * tile;
        const int64_t t_end = min(Lc, (int64_t)(i0 + (seg_end - u)) * tile);
        decode_chunk<D, G>(q, kc, vc, bt + (int64_t)b * bt_stride, ws_o, ws_ml, out, Hkv, BS, NB, tile,
                           scale_log2, b, kh, t_begin, t_end, Lc, slot * G, pw, lane);
      }
    }
    u = seg_end;
    if (u >= base + ngroups * nb) {
      ++b;
      while (b < B && tp[b + 1] == tp[b]) ++b;  // sequences with no context
    }
  }
}

// ------------------------------------------------------------ decode merge --
// Where the partials of (sequence b, query head h) live: ns of them, the
// s-th at workspace row r0 + s * rstep (o at ws_o[row * D], (m, l) at
// ws_ml[row * 2]).  ns == 1: the split kernel wrote the output itself;
// ns == 0: no context.
struct PartMap {
  int bps, max_splits;  // fixed chunks of bps blocks (bps > 0)
  const int* tp;        // balanced split (bps == 0): tile-count scan, B + 1 ints
  int tile, ngroups, wpg, G, nwg, B;
};

__device__ __forceinline__ int part_span(const PartMap& pm, int b, int h, int Hq, int64_t Lc, int BS,
                                         int64_t& r0, int64_t& rstep) {
  if (pm.bps > 0) {
    const int64_t chunk = (int64_t)pm.bps * BS;
    r0 = (int64_t)b * pm.max_splits * Hq + h;
    rstep = Hq;
    return Lc > 0 ? (int)((Lc + chunk - 1) / chunk) : 0;
  }
  r0 = 0;
  rstep = (int64_t)pm.wpg * pm.G;
  const int nb = pm.tp[b + 1] - pm.tp[b];
  if (nb == 0) return 0;
  const int kh = h / pm.G, g = h - kh * pm.G;
  const int grp = kh / pm.wpg, wv = kh - grp * pm.wpg;
  const unsigned total = (unsigned)pm.ngroups * (unsigned)pm.tp[pm.B];  // < 2^31, as in the split
  const unsigned Ct = max(1u, (total + pm.nwg - 1) / (unsigned)pm.nwg);
  const unsigned start = (unsigned)pm.ngroups * (unsigned)pm.tp[b] + (unsigned)grp * (unsigned)nb;
  const unsigned wf = start / Ct, wl = (start + nb - 1) / Ct;
  r0 = (((int64_t)wf + (int64_t)b * pm.ngroups + grp) * pm.wpg + wv) * pm.G + g;
  return (int)(wl - wf + 1);
}

// Log-sum-exp merge of one output element: partials s = 0 .. ns-1 of a
// (sequence, head) at workspace rows r0 + s*rs, element d.  All lanes of a
// wave share the (sequence, head) (D is a multiple of 64).  Up to MERGE_NS
// partials are loaded together (one memory round trip).  More (a few long
// contexts spread over the whole chip) go 64 at a time: lane s loads the
// (m, l) and computes the weight of partial s, while every lane's 64 values
// are already in flight; the sums take the weights by readlane in the same
// order as before, so the same bits.  Measured at three sequences of 583-2517
// tokens (40-69 partials a row): 28.1 -> 6.9 us against a loop of one partial
// at a time, which waits a round trip for each.  ns == 0 (no context) gives 0.
constexpr int MERGE_NS = 16;
__device__ __forceinline__ float merge_element(const float* __restrict__ ws_o, const float* __restrict__ ws_ml,
                                               int64_t r0, int64_t rs, int ns, int D, int d) {
  float res = 0.f;
  if (ns > 1 && ns <= MERGE_NS) {
    float mv[MERGE_NS], lv[MERGE_NS], ov[MERGE_NS];
#pragma unroll
    for (int s = 0; s < MERGE_NS; ++s) {
      const int64_t r = r0 + (s < ns ? s : 0) * rs;
      mv[s] = ws_ml[r * 2];
      lv[s] = ws_ml[r * 2 + 1];
      ov[s] = ws_o[r * D + d];
    }
    float M = -INFINITY;
#pragma unroll
    for (int s = 0; s < MERGE_NS; ++s)
      if (s < ns) M = fmaxf(M, mv[s]);
    float num = 0.f, den = 0.f;
    if (M != -INFINITY) {
#pragma unroll
      for (int s = 0; s < MERGE_NS; ++s)
        if (s < ns) {
          const float w = exp2f(mv[s] - M);
          den = fmaf(w, lv[s], den);
          num = fmaf(w, ov[s], num);
        }
    }
    res = den > 0.f ? num / den : 0.f;
  } else if (ns > 1) {
    const int lane = threadIdx.x & 63;
    float M = -INFINITY, num = 0.f, den = 0.f;
    for (int c = 64; c < ns; c += 64)  // the chunks past the first, whose maximum comes with its values
      M = fmaxf(M, ws_ml[(r0 + min(c + lane, ns - 1) * rs) * 2]);
    for (int c = 0; c < ns; c += 64) {
      const int n = min(64, ns - c);
      const int64_t r = r0 + c * rs;
      const float m = ws_ml[(r + min(lane, n - 1) * rs) * 2], l = ws_ml[(r + min(lane, n - 1) * rs) * 2 + 1];
      float ov[64];
#pragma unroll
      for (int s = 0; s < 64; ++s) ov[s] = ws_o[(r + min(s, n - 1) * rs) * D + d];
      if (c == 0) M = group_max<64>(fmaxf(M, m));
      if (M == -INFINITY) break;
      const float w = exp2f(m - M);
#pragma unroll
      for (int s = 0; s < 64; ++s)
        if (s < n) {
          const float ws = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), s));
          den = fmaf(ws, __int_as_float(__builtin_amdgcn_readlane(__float_as_int(l), s)), den);
          num = fmaf(ws, ov[s], num);
        }
    }
    res = den > 0.f ? num / den : 0.f;
  }
  return res;
}

// One thread per output element: workgroup (x, b) merges elements
// x*256 .. x*256+255 of sequence b's Hq*D outputs (whole heads for D = 64 /
// 128).  256-thread workgroups, one per CU at the cfg3 shapes: the same
// arithmetic as one 64 / 128-thread workgroup per (head, sequence), bit for
// bit, and 0.1-0.2 us (cfg3) to 2 us (cfg4) less kernel time -- fewer
// workgroups to dispatch; the two dependent round trips (lengths and scan,
// then the partials) remain.
constexpr int MERGE_THREADS = 256;
__global__ __launch_bounds__(MERGE_THREADS) void paged_decode_merge(
    const float* __restrict__ ws_o, const float* __restrict__ ws_ml,
    const int64_t* __restrict__ ctx_lens, uint16_t* __restrict__ out, int Hq, int D, int BS,
    int max_blocks, PartMap pm) {
  const int b = blockIdx.y;
  const int e = blockIdx.x * MERGE_THREADS + threadIdx.x;
  if (e >= Hq * D) return;
  const int h = e / D, d = e - h * D;
  const int64_t Lc = min(ctx_lens[b], (int64_t)max_blocks * BS);
  int64_t r0, rs;
  const int ns = part_span(pm, b, h, Hq, Lc, BS, r0, rs);
  if (ns == 1) return;
  out[(int64_t)b * Hq * D + e] = (uint16_t)f32_to_bf16(merge_element(ws_o, ws_ml, r0, rs, ns, D, d));
}

// The merge fused with the act_quant of its output row (the output
// projection's FP8 input): one 128-thread workgroup per (128-value act_quant
// group, sequence), every group independent.  Each thread merges one element
// of the group (the arithmetic of paged_decode_merge; ns == 1: the split
// kernel wrote the value), then 16 lanes quantise the group's 128 bf16
// values 8 each, as act_quant does: codes and scale bit-identical to
// act_quant(out row, 128).  Needs Hq * D % 128 == 0.
__global__ __launch_bounds__(128) void paged_decode_merge_quant_group(
    const float* __restrict__ ws_o, const float* __restrict__ ws_ml, const int64_t* __restrict__ ctx_lens,
    uint16_t* __restrict__ out, uint8_t* __restrict__ qo, float* __restrict__ qs, int Hq, int D, int BS,
    int max_blocks, PartMap pm) {
  __shared__ __attribute__((aligned(16))) uint16_t vals[128];
  const int g = blockIdx.x, b = blockIdx.y, t = threadIdx.x;
  const int E = Hq * D;
  const int e = g * 128 + t;
  const int h = e / D, d = e - h * D;
  const int64_t Lc = min(ctx_lens[b], (int64_t)max_blocks * BS);
  int64_t r0, rs;
  const int ns = part_span(pm, b, h, Hq, Lc, BS, r0, rs);
  uint16_t* orow = out + (int64_t)b * E;
  uint16_t v;
  if (ns == 1) {
    v = orow[e];  // written by the split kernel
  } else {
    v = (uint16_t)f32_to_bf16(merge_element(ws_o, ws_ml, r0, rs, ns, D, d));
    orow[e] = v;
  }
  vals[t] = v;
  __syncthreads();
  if (t < 16) {
    float f[8];
    unpack8(*reinterpret_cast<const uint4*>(&vals[t * 8]), f);
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(f[i]));
    amax = group_max<16>(amax);
    const float sc = scale_from_amax(amax, false);
    *reinterpret_cast<uint2*>(qo + (int64_t)b * E + g * 128 + t * 8) = quant8(f, sc);
    if (t == 0) qs[(int64_t)b * (E / 128) + g] = sc;
  }
}

template <int D, int G, bool WIN>
void launch_balanced(unsigned nwg, dim3 block, hipStream_t st, const uint16_t* q, const uint16_t* kc,
                     const uint16_t* vc, const int64_t* cl, const int32_t* bt, int64_t bts, float* wo,
                     float* wml, int* tp, uint16_t* out, int Hkv, int BS, int64_t NB, int max_blocks, int B,
                     int tile, float sl2, int ngroups, Window win) {
  hipLaunchKernelGGL((paged_decode_balanced<D, G, WIN>), dim3(nwg), block, 0, st, q, kc, vc, cl, bt, bts, wo, wml,
                     tp, out, Hkv, BS, NB, max_blocks, B, tile, sl2, ngroups, win);
}

template <int D, bool WIN = false>
bool dispatch_balanced(int G, unsigned nwg, dim3 block, hipStream_t st, const uint16_t* q,
                       const uint16_t* kc, const uint16_t* vc, const int64_t* cl, const int32_t* bt,
                       int64_t bts, float* wo, float* wml, int* tp, uint16_t* out, int Hkv, int BS,
                       int64_t NB, int max_blocks, int B, int tile, float sl2, int ngroups, Window win = Window{}) {
#define LFS_G(GG) \
  case GG: launch_balanced<D, GG, WIN>(nwg, block, st, q, kc, vc, cl, bt, bts, wo, wml, tp, out, Hkv, BS, NB, max_blocks, B, tile, sl2, ngroups, win); return true;
  switch (G) {
    LFS_G(1) LFS_G(2) LFS_G(3) LFS_G(4) LFS_G(5) LFS_G(6) LFS_G(7) LFS_G(8)
    default: return false;
  }
#undef LFS_G
}

// compute units of the current device (the balanced split's grid)
int decode_cu_count() {
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

// balanced split geometry: wpg waves (kv heads) per workgroup, ngroups
// groups, nwg workgroups -- one 4-wave workgroup per CU, one round.  Fewer,
// longer streams beat filling the kernel's occupancy (two waves per SIMD):
// measured at 1 / 2 / 3 / 4 / 8 workgroups per CU, cfg3 44.3 / 49.4 / 56.6 /
// 56.0 / 66.2 us, cfg4 1169 / 1190 / 1202 / 1212 / 1257 us (fewer tile
// pipelines to ramp up, fewer partials, fewer concurrent DRAM streams).
struct BalancedGeom {
  int wpg, ngroups, nwg;
};
BalancedGeom balanced_geom(int Hkv) {
  BalancedGeom g;
  g.wpg = Hkv < 4 ? Hkv : 4;
  g.ngroups = (Hkv + g.wpg - 1) / g.wpg;
  g.nwg = decode_cu_count() * (4 / g.wpg);
  return g;
}

int paged_decode_merge_launch(float* ws_o, float* ws_ml, const int64_t* context_lens, void* out, void* q_out,
                              float* q_scale, int64_t B, int Hq, int D, int BS, int max_blocks, const PartMap& pm,
                              hipStream_t st) {
  if (q_out != nullptr) {
    hipLaunchKernelGGL(paged_decode_merge_quant_group, dim3((unsigned)(Hq * D / 128), (unsigned)B), dim3(128), 0, st,
                       ws_o, ws_ml, context_lens, (uint16_t*)out, (uint8_t*)q_out, q_scale, Hq, D, BS, max_blocks, pm);
    return check_launch("paged_decode(merge + quant)");
  }
  hipLaunchKernelGGL(paged_decode_merge, dim3((unsigned)((Hq * D + MERGE_THREADS - 1) / MERGE_THREADS), (unsigned)B),
                     dim3(MERGE_THREADS), 0, st, ws_o, ws_ml, context_lens, (uint16_t*)out, Hq, D, BS, max_blocks, pm);
  return check_launch("paged_decode(merge)");
}

}  // namespace
}  // namespace lfs
