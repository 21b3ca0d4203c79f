// One wave's walk over a range of tiles of one (sequence, kv head) of a paged KV
// pool in 8 bits (codes and scales) or in bf16, both products on the matrix
// cores, V transposed in registers: for the decode over a pool in 8 bits
// (paged_fp8.hip) and of what sequences do not share (paged_shared.hip).
//
// Per tile of T tokens (in 8 bits K = s_k k and V = s_v v):
//   S = k q^T  v_mfma_f32_16x16x32_bf16: lane (j, kq) supplies 16 bytes of token j
//              of a 16-token group.  Codes are converted (exactly) two at a time.
//              Not the FP8 MFMAs: on gfx950 their sums are off by up to 2^-12 of
//              the largest product (measured on sums of 32 to 128 random
//              products), which a weight would show.  Columns j and j + 8 of q^T
//              are the same head;
//   softmax    online, log2 domain; lane (j, kq) holds the scores of head j % 8 for
//              tokens 4 kq .. +3 of every group;
//   O^T += v^T P^T  P^T is the B operand straight from the softmax registers,
//              k-index 8 kq + i standing for token 4 kq + i of a pair's first
//              16-token group (i < 4) or 4 kq + i - 4 of its second.  Lane (m, kq)
//              loads D / 16 values of those eight tokens, at dims m D / 16 on:
//              byte permutes put pairs of tokens beside each other, which
//              transposes V without LDS.  Columns j and j + 8 are the weight (times
//              s_v) rounded to bf16 and what that left: 16 bits of it, at no cost;
//   loads      a tile ahead, in two sets of registers, through buffer descriptors
//              that end behind the last visible row: rows past the context and of
//              blocks outside the pool read as zeros, whatever they hold.
// The cost per tile does not depend on the number of query heads (at most 8).
#pragma once

#include "decode_wave.h"

namespace lfs {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int D, bool FP8>
struct PoolGeom {
  static constexpr int ES = FP8 ? 1 : 2;             // bytes of a value
  // Tokens per tile (8 or 16 KiB).  Codes in heads of 64: 64 sequences of 128 to 4096
  // tokens 22.7 us, in tiles of 128 26.5 (fewer, longer steps at a range's ends).
  static constexpr int T = FP8 || D == 64 ? 64 : 32;
  static constexpr int NG = T / 16;                  // 16-token groups
  static constexpr int KL = D * ES / 64;             // 16-byte K loads per lane and group
  static constexpr int DB = D / 16;                  // V values per lane and token
  static constexpr int VD = DB * ES / 4;             // and their dwords
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

// Tokens t0 .. t1 - 1 of a context (t0 a multiple of 16; where ONE a tile from t0 on
// lies in one block), for kv head kh: G query heads at q, the partial to rows prow ..
// or, where out is given, the normalised output there.
struct PoolRange {
  const int32_t* btrow;
  const uint16_t* q;
  uint16_t* out;
  int64_t prow;
  int t0, t1, kh;
};

template <int D, bool FP8, bool ONE>
struct PoolWave {
  using Geo = PoolGeom<D, FP8>;
  static constexpr int NG = Geo::NG, KL = Geo::KL, DB = Geo::DB, T = Geo::T, ES = Geo::ES, VD = Geo::VD;
  // Every row is read once: nontemporal, but where a head's codes are half a line,
  // whose other half another wave asks for (64 sequences of 8192 tokens, 16 / 4
  // heads of 64: 65.4 us nontemporal, 61.1 not; of 128 92 and 102).
  static constexpr int kNt = D * ES >= 128 ? 2 : 0;
  struct Tile {
    u32x4 k[NG][KL];
    uint32_t v[NG][4][VD];
    float ks, vs;  // of token `lane`
    int n;         // tokens up to the range's end (at most T)
    uint32_t bad;  // bit g: group g lies in no block of the pool
    bool first, last;  // of its range
    PoolRange at;
  };

  int lane, j, kq, Hkv, G, BS, row;  // row: bytes of a token
  int64_t NB;
  const uint8_t *kc, *vc;
  const float *ksc, *vsc;
  v8bf q[D / 32], qnext[D / 32];
  float scale_log2, acc[DB][4], m_run, l_run;
  // the tile asked for: its range and place; lanes 16 g .. 16 g + 15 hold the block id
  // of its 16-token group g and the offset there, and the column of the next's
  PoolRange ask_at;
  int pos, ask_n, col, off, id, idoff, sq, sr;
  bool ask_first, ask_last, more;

  __device__ __forceinline__ void init(int lane_, const void* kc_, const void* vc_, const float* ksc_, const float* vsc_,
                                       int Hkv_, int G_, int BS_, int64_t NB_, float scale_log2_) {
    lane = lane_, j = lane & 15, kq = lane >> 4;
    kc = (const uint8_t*)kc_, vc = (const uint8_t*)vc_, ksc = ksc_, vsc = vsc_;
    Hkv = Hkv_, G = G_, BS = BS_, row = Hkv * D * ES, NB = NB_;
    scale_log2 = scale_log2_;
    sq = T / BS;
    sr = T - sq * BS;
  }

  // Begin the range in ask_at: its first tile's place and column.
  __device__ __forceinline__ void begin() {
    pos = ask_at.t0;
    const unsigned t = pos + (lane >> 4) * 16;
    col = (int)(t / (unsigned)BS);
    off = (int)t - col * BS;
  }
  // Of the next tile (of the range under way, else of the one that next() fills
  // in) ask for the block ids; columns past the range's are not read.
  template <class Next>
  __device__ __forceinline__ void ask(Next&& next) {
    ask_first = pos >= ask_at.t1;
    if (ask_first) {
      more = next(ask_at);
      begin();  // without another range the last one again, of which nothing is then used
    }
    ask_tile();
  }
  __device__ __forceinline__ void ask_tile() {
    ask_n = more ? min(T, ask_at.t1 - pos) : 0;
    pos += T;
    ask_last = pos >= ask_at.t1;
    const int end = (int)((unsigned)(ask_at.t1 - 1) / (unsigned)BS);
    const int at = ask_at.btrow[min(col, end)];
    id = col <= end ? at : -1;
    idoff = off;
    col += sq;
    off += sr;
    if (off >= BS) off -= BS, ++col;
  }
  // Load the tile whose ids were asked for.
  __device__ __forceinline__ void load(Tile& t) {
    const int n = ask_n, kh = ask_at.kh;
    t.n = n;
    t.first = ask_first, t.last = ask_last;
    t.at = ask_at;
    // the range's query, with its first tile: lane (j, kq) holds of head j % 8 the
    // dims of its K loads
    {
      const auto qr = pool_rows(reinterpret_cast<const uint8_t*>(ask_at.q), 0, ask_first ? G * D * 2 : 0);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const int d = FP8 ? (c >> 1) * 64 + kq * 16 + (c & 1) * 8 : c * 32 + kq * 8;
        qnext[c] = __builtin_bit_cast(v8bf, __builtin_amdgcn_raw_buffer_load_b128(qr, ((j & 7) * D + d) * 2, 0, 0));
      }
    }
    const bool ok = id >= 0 && (int64_t)id < NB;
    const int64_t blk = ok ? id : 0, at = (blk * BS + idoff) * row + (int64_t)kh * (D * ES);
    if constexpr (FP8) {
      const int64_t sat = (blk * Hkv + kh) * BS + idoff + (lane & 15);
      const bool use = ok && lane < n;
      const float a = ksc[sat], b = vsc[sat];
      t.ks = use ? a : 0.f;
      t.vs = use ? b : 0.f;
    }
    const uint64_t m = __ballot(!ok);
    uint32_t bad = 0;
#pragma unroll
    for (int g = 0; g < NG; ++g) bad |= (uint32_t)(m >> (16 * g) & 1) << g;
    t.bad = bad;
    auto base_of = [&](int g) {
      const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)at, 16 * g);
      const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)at >> 32), 16 * g);
      return (int64_t)((uint64_t)hi << 32 | lo);
    };
    const int kat = j * row + kq * 16, vat = kq * 4 * row + j * (DB * ES);
    const int64_t b0 = base_of(0);
    const int all = ONE && n > 0 && !(bad & 1) ? (n - 1) * row + D * ES : 0;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      int64_t b = b0;
      int bytes = all, soff = g * 16 * row;
      if constexpr (!ONE) {
        b = base_of(g);
        const int rows = min(16, n - g * 16);
        bytes = rows > 0 && !(bad >> g & 1) ? (rows - 1) * row + D * ES : 0;
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
        bytes = rows > 0 && !(bad >> g & 1) ? (rows - 1) * row + D * ES : 0;
        soff = 0;
      }
      const auto vr = pool_rows(vc, b, bytes);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (VD == 1) {
          t.v[g][r][0] = __builtin_amdgcn_raw_buffer_load_b32(vr, vat + r * row, soff, kNt);
        } else if constexpr (VD == 2) {
          const auto w = __builtin_amdgcn_raw_buffer_load_b64(vr, vat + r * row, soff, kNt);
          t.v[g][r][0] = w[0];
          t.v[g][r][1] = w[1];
        } else {
          const auto w = __builtin_amdgcn_raw_buffer_load_b128(vr, vat + r * row, soff, kNt);
#pragma unroll
          for (int d = 0; d < 4; ++d) t.v[g][r][d] = w[d];
        }
      }
    }
  }

  // pw: the wave's LDS slice, 2 T floats (FP8).
  __device__ __forceinline__ void compute(const Tile& t, float* __restrict__ pw) {
    if constexpr (FP8) {
      pw[lane] = t.ks;
      pw[T + lane] = t.vs;
      wave_lds_sync();
    }
    float s[NG][4];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      v4f sc = {0.f, 0.f, 0.f, 0.f};
      if constexpr (FP8) {
#pragma unroll
        for (int c = 0; c < 2 * KL; ++c)
          sc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_bf16(t.k[g][c / 2][c % 2 * 2], t.k[g][c / 2][c % 2 * 2 + 1]),
                                                       q[c], sc, 0, 0, 0);
        const float4 ks = *reinterpret_cast<const float4*>(pw + g * 16 + kq * 4);
        const float kf[4] = {ks.x, ks.y, ks.z, ks.w};
#pragma unroll
        for (int r = 0; r < 4; ++r) s[g][r] = sc[r] * (scale_log2 * kf[r]);
      } else {
#pragma unroll
        for (int c = 0; c < KL; ++c)
          sc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, t.k[g][c]), q[c], sc, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[g][r] = sc[r] * scale_log2;
      }
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
        float vf[4] = {1.f, 1.f, 1.f, 1.f};
        if constexpr (FP8) {
          const float4 vs = *reinterpret_cast<const float4*>(pw + T + g * 16 + kq * 4);
          vf[0] = vs.x, vf[1] = vs.y, vf[2] = vs.z, vf[3] = vs.w;
        }
        float x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[r] = __builtin_amdgcn_exp2f(s[g][r] - m_use);
          l_run += x[r];
          if constexpr (FP8) x[r] *= vf[r];
        }
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          const uint32_t hi = pack_bf16x2(x[r], x[r + 1]);
          w[y * 2 + r / 2] = pack_bf16x2(x[r] - __uint_as_float(hi << 16 & low), x[r + 1] - __uint_as_float(hi & low));
        }
      }
      const v8bf pb = __builtin_bit_cast(v8bf, make_uint4(w[0], w[1], w[2], w[3]));
      constexpr int VN = FP8 ? 4 : 2;  // values of a dword
#pragma unroll
      for (int d = 0; d < VD; ++d) {
        uint32_t a[VN][4];  // [value of the dword][pair of tokens]
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t t0 = t.v[2 * p + i / 2][(i & 1) * 2][d], t1 = t.v[2 * p + i / 2][(i & 1) * 2 + 1][d];
          if constexpr (FP8) {
            const uint32_t x01 = __builtin_amdgcn_perm(t1, t0, 0x05010400u);
            const uint32_t x23 = __builtin_amdgcn_perm(t1, t0, 0x07030602u);
            a[0][i] = bf16_lo(x01), a[1][i] = bf16_hi(x01), a[2][i] = bf16_lo(x23), a[3][i] = bf16_hi(x23);
          } else {
            a[0][i] = __builtin_amdgcn_perm(t1, t0, 0x05040100u), a[1][i] = __builtin_amdgcn_perm(t1, t0, 0x07060302u);
          }
        }
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          v4f c = {acc[VN * d + e][0], acc[VN * d + e][1], acc[VN * d + e][2], acc[VN * d + e][3]};
          c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(v8bf, make_uint4(a[e][0], a[e][1], a[e][2], a[e][3])), pb, c, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[VN * d + e][r] = c[r];
        }
      }
    }
    if constexpr (FP8) wave_lds_sync();
  }

  // Work through the ranges that next(range) fills in until it says false, as one
  // stream of tiles: the first tile and the query of a range are in flight while
  // the last of the one before is computed.  pw: LDS for compute().
  template <class Next>
  __device__ __forceinline__ void run(Next&& next, float* __restrict__ pw, float* __restrict__ ws_o,
                                      float* __restrict__ ws_ml) {
    // A wave may have no range at all (its heads lie past the last): ask_at then
    // holds nothing that could be read.
    if (!next(ask_at)) return;
    more = ask_first = true;
    begin();
    ask_tile();
    Tile a, b;
    load(a);
    ask(next);
    auto step = [&](Tile& cur, Tile& nxt) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) q[c] = cur.first ? qnext[c] : q[c];
      load(nxt);
      ask(next);
      __builtin_amdgcn_sched_barrier(0);
      if (cur.first) {
        m_run = -INFINITY;
        l_run = 0.f;
#pragma unroll
        for (int e = 0; e < DB; ++e)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[e][r] = 0.f;
      }
      compute(cur, pw);
      if (cur.last) finish(cur.at, ws_o, ws_ml);
    };
    while (true) {
      step(a, b);
      if (b.n == 0) break;
      step(b, a);
      if (a.n == 0) break;
    }
  }

  __device__ __forceinline__ void finish(const PoolRange& at, float* __restrict__ ws_o, float* __restrict__ ws_ml) {
    const bool whole = at.out != nullptr;
    const int64_t prow = at.prow;
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
          *reinterpret_cast<uint2*>(at.out + (int64_t)j * D + d + e) =
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

}  // namespace
}  // namespace lfs
