// GQA decode over a bf16 pool for groups of sequences that share their first
// blocks: the shared keys and values of a group are read once for all of them.
//
// A context is its group's prefix and the rest.  Attention over either leaves a
// maximum m, a sum l and an unnormalised output o, and parts a, b, .. join as
//   m = max_i m_i,  o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.
//
// One launch does both kinds of part, a second joins them.  Its workgroups have
// two roles, of which each CU holds one workgroup each, so that the matrix cores
// work on prefixes while memory streams the rest:
//  prefix  a kv head's queries of a group are a list of n G rows (n sequences, G
//          heads).  Units are (group, kv head, 128 rows, 64-key tile), in that
//          order; a workgroup takes an equal run of them.  A wave has 32 rows, the
//          waves share 64-key K and V tiles in LDS, the next tile's copies in
//          flight: the products, swizzles and copies of prefill.hip (tile32.h),
//          without the causal mask, with the keys' range cut in runs and with
//          weights of 16 bits (outputs as exact as paged_attention_decode's).
//          Consecutive workgroups hold consecutive runs of one (kv head, 128
//          rows), so those of the next 128 rows on the same keys often run on the
//          same XCD and find them in its L2.
//  rest    the walk of pool_wave.h from the prefix's end on, shared by the
//          balanced split of decode_wave.h.  A group of one sequence has no
//          prefix here, its whole context is rest; from two on it pays, but for
//          pairs with heads of 64 (64 sequences behind 4096 tokens each pair, four,
//          eight shares: 161, 95, 54 us of 32 / 8 heads of 128, 151 to 174 by
//          themselves; of 16 / 4 of 64 69, 42, 25 and 57 to 58).
// What it takes (us, in all; alone the roles 79-84 and 57): 128 sequences of 64 to 1024
// tokens behind 16384 shared ones, 32 / 8 heads of 128: 100, of which the merge 11,
// where the decode that reads every context by itself takes 1220; 64 sequences in
// 3 groups behind 1536 to 3584 tokens, 16 / 4 of 64: 24 and 47.  Bound: at the first
// the matrix cores' work beside the reads (a CU has one workgroup of each role), at
// the second five dependent round trips (boundaries, lengths, table, rows) and the
// merge's launch.  Each workgroup taking a share of both roles, half of them in
// either order, took 116 and 32 where this took 93 and 23 (weights of 8 bits then): twice the
// parts, and twice the scans.
// Group boundaries are read on the device: a running maximum of cu_groups,
// clipped to the batch, so that any values keep every access in bounds.
#include "pool_wave.h"
#include "tile32.h"

namespace lfs {
namespace {

constexpr int SMEM = 2 * 4 * (BAL_MAXB + 8);  // scans of groups and sequences, then the tiles
constexpr int PROWS = RW * NW;                // rows of a prefix unit
constexpr int KNOWN = 512;                    // sequences whose prefix and length stay in LDS, groups whose blocks do

struct SharedArgs {
  const uint16_t *q, *kc, *vc;
  const int64_t* ctx_lens;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t *cu, *shared;
  float *po, *pml, *so, *sml;  // partials: prefix, rest
  int *starts, *punits, *stiles, *group;  // [NG + 1], [NG + 1], [B + 1], [B]: for the merge
  int Hkv, G, BS, NG, B, max_blocks, hg, ngroups, nprefix, nrest;
  int64_t NB;
  float scale_log2;
};

// What a workgroup keeps in LDS beside its scans.
struct SharedLds {
  int wsum[NW], found[NW];
  int blocks[KNOWN];       // shared by a group
  int prefix[2 * KNOWN];   // of a sequence: tokens of its group's prefix, length
};

// starts[g]: running maximum of the boundaries clipped to 0 .. B, in LDS, with the
// first groups' shared blocks.
__device__ __forceinline__ void scan_starts(const SharedArgs& a, int* starts, SharedLds& s) {
  int* wmax = s.wsum;
  for (int g = threadIdx.x; g < min(a.NG, KNOWN); g += 256) s.blocks[g] = a.shared[g];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, n = a.NG + 1;
  const int per = (n + 255) / 256, lo = min(n, tid * per), hi = min(n, lo + per);
  int run = 0;
  for (int i = lo; i < hi; ++i) starts[i] = run = max(run, min(max(a.cu[i], 0), a.B));
  int incl = run;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(incl, o, 64);
    if (lane >= o) incl = max(incl, v);
  }
  if (lane == 63) wmax[wave] = incl;
  int before = __shfl_up(incl, 1, 64);
  if (lane == 0) before = 0;
  __syncthreads();
  for (int w = 0; w < wave; ++w) before = max(before, wmax[w]);
  for (int i = lo; i < hi; ++i) starts[i] = max(starts[i], before);
  __syncthreads();
}

// Tokens of group g's prefix, of n sequences.
__device__ __forceinline__ int64_t prefix_of(const SharedArgs& a, int blocks, int n) {
  return n < 2 ? 0 : (int64_t)min(max(blocks, 0), a.max_blocks) * a.BS;
}
__device__ __forceinline__ int64_t prefix_tokens(const SharedArgs& a, int g, int n) {
  return prefix_of(a, n < 2 ? 0 : a.shared[g], n);
}
// (after scan_starts)
__device__ __forceinline__ int64_t prefix_tokens(const SharedArgs& a, const SharedLds& s, int g, int n) {
  return g < KNOWN ? prefix_of(a, s.blocks[g], n) : prefix_tokens(a, g, n);
}
// Its 128-row tiles and 64-key tiles.
__device__ __forceinline__ int row_tiles(const SharedArgs& a, int n) { return (n * a.G + PROWS - 1) / PROWS; }
__device__ __forceinline__ int key_tiles(int64_t tokens) { return (int)((tokens + KT - 1) / KT); }

// The group of sequence b (-1: none) and its prefix.
__device__ __forceinline__ int group_of(const SharedArgs& a, const SharedLds& s, const int* starts, int b, int64_t& tokens) {
  tokens = 0;
  if (a.NG == 0) return -1;
  int lo = 0, hi = a.NG;  // the last boundary at or before b
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] <= b) lo = mid;
    else hi = mid - 1;
  }
  if (lo == a.NG || starts[lo] > b) return -1;
  tokens = prefix_tokens(a, s, lo, starts[lo + 1] - starts[lo]);
  return lo;
}

// Key tiles k0 .. k1 - 1 of row tile rt of kv head kh of the group whose
// sequences are first .. first + n - 1, sharing `tokens`; prow: the first of the
// partial's rows.
template <int D>
__device__ __forceinline__ void prefix_unit(const SharedArgs& a, uint8_t* smem, int first, int n, int64_t tokens, int kh,
                                            int rt, int k0, int k1, int64_t prow) {
  constexpr int NDC = D / 16, NDB = D / 32, RB = 2 * D, TB = KT * RB, RPC = 1024 / RB, NC = TB / 1024 / NW;
  constexpr int NB = KT / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c32 = lane & 31, h = lane >> 5, hoff = 16 * wave;
  const int Hq = a.Hkv * a.G, rows = n * a.G, r0 = rt * PROWS;
  const int64_t cap = (int64_t)a.max_blocks * a.BS;
  const int64_t rowb = (int64_t)a.Hkv * RB;
  auto limit_of = [&](int r) {  // keys of the prefix that row r sees
    if (r >= rows) return 0;
    return (int)max((int64_t)0, min(min(a.ctx_lens[first + r / a.G], cap), tokens));
  };
  // lanes 16 x .. 16 x + 15 look after the tile's 16-key group x: block column
  // and offset, asked for a tile ahead, the first before the rows' lengths are known
  const int32_t* btrow = a.bt + (int64_t)first * a.bt_stride;
  const int gkey = 16 * (lane >> 4);
  int col = (unsigned)(k0 * KT + gkey) / (unsigned)a.BS;
  int off = k0 * KT + gkey - col * a.BS, entry = -1, eoff = 0;
  auto ask = [&](int t0) {
    entry = -1;
    eoff = off;
    if (t0 + gkey < tokens) entry = btrow[col];
    off += KT;
    while (off >= a.BS) off -= a.BS, ++col;
  };
  ask(k0 * KT);
  // keys that any of the workgroup's rows sees: none past them is read
  int kend = max(limit_of(r0 + lane), limit_of(r0 + 64 + lane));
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) kend = max(kend, __shfl_xor(kend, o, 64));
  kend = __builtin_amdgcn_readfirstlane(kend);
  k1 = min(k1, (kend + KT - 1) / KT);
  const int row = r0 + RW * wave + c32, lim = limit_of(row);
  int wmin = lim, wmax = lim;  // of the wave's rows
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    wmin = min(wmin, __shfl_xor(wmin, o, 64));
    wmax = max(wmax, __shfl_xor(wmax, o, 64));
  }
  wmin = __builtin_amdgcn_readfirstlane(wmin), wmax = __builtin_amdgcn_readfirstlane(wmax);

  const unsigned lbase = (unsigned)(uintptr_t)(const lds_u8*)smem;
  const int crow = hoff + lane / (D / 8);
  unsigned krow[NC], vrow[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int r = crow + RPC * c;
    krow[c] = (unsigned)(r & 15) * (unsigned)rowb + (((lane % (D / 8)) ^ kswz<D>(r)) << 4);
    vrow[c] = (unsigned)(r & 15) * (unsigned)rowb + (((lane % (D / 8)) ^ vswz<D>(r)) << 4);
  }
  const uint8_t* kb = reinterpret_cast<const uint8_t*>(a.kc) + (int64_t)kh * RB;
  const uint8_t* vb = reinterpret_cast<const uint8_t*>(a.vc) + (int64_t)kh * RB;
  // copies of the tile at key t0 to buffer buf; returns which of its groups hold
  // visible keys.  A wave copies one group's K and V; one without takes the rows
  // of one with, whose values are finite, and its scores are masked.
  auto fetch = [&](int t0, int buf) -> unsigned {
    const bool ok = entry >= 0 && (int64_t)entry < a.NB && t0 + gkey < kend;
    const uint64_t m = __ballot(ok);
    const unsigned use = (unsigned)(m & 1) | (unsigned)(m >> 16 & 1) << 1 | (unsigned)(m >> 32 & 1) << 2 |
                         (unsigned)(m >> 48 & 1) << 3;
    const int src = use == 0 ? 0 : use >> wave & 1 ? wave : __builtin_ctz(use);
    const int64_t slot = ok ? (int64_t)entry * a.BS + eoff : 0;
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)slot, 16 * src);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)slot >> 32), 16 * src);
    const int64_t at = (int64_t)((uint64_t)hi << 32 | lo) * rowb;
    const int valid = use == 0 ? 0 : min(15, kend - 1 - (t0 + 16 * src));
    unsigned ko[NC], vo[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {  // rows past the last visible one read it
      const unsigned back = (unsigned)max(0, (crow & 15) + RPC * c - valid) * (unsigned)rowb;
      ko[c] = krow[c] - back;
      vo[c] = vrow[c] - back;
    }
    copy_rows<NC>(kb + at, ko, lbase + buf * TB + hoff * RB);
    copy_rows<NC>(vb + at, vo, lbase + (2 + buf) * TB + hoff * RB);
    return use;
  };

  // Q^T (B operand): lane l supplies row l % 32, dims 16c + 8h .. +7; rows past the last as the last
  v8bf qb[NDC];
  {
    const int r = min(row, rows - 1), b = first + r / a.G;
    const uint16_t* qr = a.q + ((int64_t)b * Hq + kh * a.G + r % a.G) * D + 8 * h;
#pragma unroll
    for (int c = 0; c < NDC; ++c) qb[c] = __builtin_bit_cast(v8bf, *reinterpret_cast<const uint4*>(qr + 16 * c));
  }
  v16f o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;
  const unsigned ka = lbase + c32 * RB + ((h ^ kswz<D>(c32)) << 4);
  const int il = lane & 15, gq = (lane >> 4) & 1;
  const unsigned va = lbase + 2 * TB + (4 * h + (il >> 2)) * RB +
                      (((2 * gq + ((il & 3) >> 1)) ^ vswz<D>(4 * h + (il >> 2))) << 4) + 8 * (il & 1);
  auto k_frag = [&](int i, int buf) -> u32x4 { return lds_read16((ka ^ (32 * (i / NB))) + buf * TB + i % NB * 32 * RB); };
  auto v_frag = [&](int i, int buf) -> uint4 {
    const unsigned p = (va ^ (64 * (i % NDB))) + buf * TB + (32 * (i / NDB / 2) + 8 * (i / NDB % 2)) * RB;
    const uint2 lo = lds_read_tr(p), hi = lds_read_tr(p + 16 * RB);
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  };
  constexpr int NS = NB * NDC, NP = KT / 16 * NDB, AH = 4;
  unsigned use = 0, next = 0;
  __syncthreads();  // the tiles' LDS is free
  if (k0 < k1) {
    next = fetch(k0 * KT, 0);
    ask((k0 + 1) * KT);
  }
  for (int kt = k0; kt < k1; ++kt) {
    const int t0 = kt * KT, buf = (kt - k0) & 1;
    use = next;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();  // the tile is in LDS, and every wave done with the one before
    u32x4 kf[AH];
#pragma unroll
    for (int i = 0; i < AH; ++i) kf[i] = k_frag(i, buf);
    __builtin_amdgcn_sched_barrier(0);
    if (kt + 1 < k1) {
      next = fetch(t0 + KT, buf ^ 1);
      ask(t0 + 2 * KT);
    }
    if (use == 0 || t0 >= wmax) continue;  // nothing that the wave's rows see (it still copies)
    v16f s[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      s[i % NB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, kf[i % AH]), qb[i / NB], s[i % NB], 0,
                                                          0, 0);
      if (i + AH < NS) kf[i % AH] = k_frag(i + AH, buf);
      __builtin_amdgcn_sched_barrier(0);
    }
    uint4 vf[AH];
#pragma unroll
    for (int i = 0; i < AH; ++i) vf[i] = v_frag(i, buf);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int b = 0; b < NB; ++b) s[b] *= a.scale_log2;
    if (use != 15 || t0 + KT > wmin) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!(use >> (2 * b + r / 8) & 1) || t0 + 32 * b + 8 * (r / 4) + 4 * h + r % 4 >= lim) s[b][r] = -INFINITY;
    }
    float mx = s[0][0], alpha = 1.f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
    mx = xor_max<32>(mx);
    if (__any(mx > m_run)) {
      const float m_new = fmaxf(m_run, mx);
      alpha = m_new == m_run ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
      m_run = m_new;
    }
    const float m_exp = m_run == -INFINITY ? 0.f : m_run;
    float ps = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[b][r] = __builtin_amdgcn_exp2f(s[b][r] - m_exp);
        ps += s[b][r];
      }
    l_run = fmaf(l_run, alpha, ps);  // the lane's own keys
    __builtin_amdgcn_sched_barrier(0);
    // A weight as bf16 and what that rounding left, 16 bits of it as in pool_wave.h, in
    // two products: 128 sequences behind 16384 tokens, 32 / 8 heads of 128, 104 us and
    // 0.0017 from 64 bits (the outputs' own rounding); the first product alone 97 and 0.0022.
    uint4 hi = {}, lo = {};
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if (i % NDB == 0) {
        const v16f& x = s[i / NDB / 2];
        const int at = i / NDB % 2 * 4;
        uint32_t w[4], left[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float x0 = x[at + k / 2 * 8 + k % 2 * 2], x1 = x[at + k / 2 * 8 + k % 2 * 2 + 1];
          w[k] = pack_bf16x2(x0, x1);
          left[k] = pack_bf16x2(x0 - __uint_as_float(w[k] << 16), x1 - __uint_as_float(w[k] & 0xFFFF0000u));
        }
        hi = make_uint4(w[0], w[1], w[2], w[3]), lo = make_uint4(left[0], left[1], left[2], left[3]);
      }
      const v8bf v = __builtin_bit_cast(v8bf, vf[i % AH]);
      o[i % NDB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, __builtin_bit_cast(v8bf, hi), o[i % NDB], 0, 0, 0);
      o[i % NDB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, __builtin_bit_cast(v8bf, lo), o[i % NDB], 0, 0, 0);
      if (i + AH < NP) vf[i % AH] = v_frag(i + AH, buf);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  const float l = xor_sum<32>(l_run);
  if (row >= rows) return;
  const int64_t at = prow + RW * wave + c32;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int x = 0; x < 4; ++x)
      *reinterpret_cast<float4*>(a.po + at * D + 32 * db + 8 * x + 4 * h) =
          make_float4(o[db][4 * x], o[db][4 * x + 1], o[db][4 * x + 2], o[db][4 * x + 3]);
  if (h == 0) {
    a.pml[at * 2] = m_run;
    a.pml[at * 2 + 1] = l;
  }
}

template <int D>
__device__ __forceinline__ void prefix_role(const SharedArgs& a, uint8_t* smem, SharedLds& s, int w) {
  int* starts = reinterpret_cast<int*>(smem);
  int* units = starts + BAL_MAXB + 8;
  scan_starts(a, starts, s);
  const TileScan scan = scan_tiles(units, s.wsum, a.NG, [&](int g) {
    const int n = starts[g + 1] - starts[g];
    return row_tiles(a, n) * a.Hkv * key_tiles(prefix_tokens(a, s, g, n));
  });
  const unsigned total = scan.total, Ct = max(1u, (total + a.nprefix - 1) / a.nprefix);
  unsigned u = w * Ct;
  const unsigned u_end = min(total, u + Ct);
  place_tiles(units, scan, [&](int g, int before, int after) {
    if ((unsigned)before <= u && u < (unsigned)after) s.found[0] = g;
  });
  if (w == 0)
    for (int i = threadIdx.x; i <= a.NG; i += 256) a.starts[i] = starts[i], a.punits[i] = units[i];
  if (u >= u_end) return;
  int g = s.found[0];
  unsigned base = units[g];
  int first = starts[g], end = starts[g + 1];
  while (true) {
    const int n = end - first, rts = row_tiles(a, n);
    const int64_t tokens = prefix_tokens(a, s, g, n);
    const unsigned nt = key_tiles(tokens), pairs = rts * a.Hkv;
    while (u < base + pairs * nt && u < u_end) {
      const unsigned pair = (u - base) / nt, k0 = (u - base) - pair * nt;
      const unsigned stop = min(u_end, base + (pair + 1) * nt);
      const int kh = pair / rts, rt = pair - kh * rts;
      // partial rows: 128 further for each workgroup, a pair's rows further for each pair
      const int64_t prow = (int64_t)w * PROWS + (int64_t)first * a.G * a.Hkv + (int64_t)kh * n * a.G + rt * PROWS;
      prefix_unit<D>(a, smem, first, n, tokens, kh, rt, (int)k0, (int)(k0 + (stop - u)), prow);
      u = stop;
    }
    if (u >= u_end) return;
    base += pairs * nt;  // the next group (the scans' LDS holds tiles by now)
    ++g;
    first = end;
    end = max(end, min(max(a.cu[g + 1], 0), a.B));
  }
}

// The walk works on virtual workgroups of hg waves, one per kv head of a group of
// heads: 4 / hg of them here.
template <int D, bool ONE>
__device__ __forceinline__ void rest_role(const SharedArgs& a, uint8_t* smem, SharedLds& s, int w) {
  constexpr int T = PoolGeom<D, false>::T;
  int* starts = reinterpret_cast<int*>(smem);
  int* tp = starts + BAL_MAXB + 8;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t cap = (int64_t)a.max_blocks * a.BS;
  const int b0 = scan_first(a.B);
  const int64_t len0 = b0 < a.B ? a.ctx_lens[b0] : 0;  // in flight while the boundaries are scanned
  scan_starts(a, starts, s);
  const TileScan scan = scan_tiles(tp, s.wsum, a.B, [&](int b) {
    int64_t tokens;
    const int g = group_of(a, s, starts, b, tokens);
    if (w == 0) a.group[b] = g;
    const int64_t Lc = min(b == b0 ? len0 : a.ctx_lens[b], cap), L = Lc - tokens;
    if (b < KNOWN) s.prefix[2 * b] = (int)tokens, s.prefix[2 * b + 1] = (int)max((int64_t)0, Lc);
    return L > 0 ? (int)((L + T - 1) / T) : 0;
  });
  const int sub = wave / a.hg, head = wave - sub * a.hg, per = NW / a.hg;
  const unsigned total = (unsigned)a.ngroups * (unsigned)scan.total, nwg = a.nrest * per;
  const unsigned Ct = max(1u, (total + nwg - 1) / nwg), v = w * per + sub;
  place_tiles(tp, scan, [&](int b, int before, int after) {
    for (int k = 0; k < per; ++k) {
      const unsigned at = (w * per + k) * Ct;
      if ((unsigned)a.ngroups * (unsigned)before <= at && at < (unsigned)a.ngroups * (unsigned)after) s.found[k] = b;
    }
  });
  if (w == 0)
    for (int i = threadIdx.x; i <= a.B; i += 256) a.stiles[i] = tp[i];
  if (sub >= per) return;  // hg == 3
  unsigned u = v * Ct;
  const unsigned u_end = min(total, u + Ct);
  if (u >= u_end) return;
  int b = s.found[sub];
  b = __builtin_amdgcn_readfirstlane(b);
  PoolWave<D, false, ONE> wv;
  wv.init(lane, a.kc, a.vc, nullptr, nullptr, a.Hkv, a.G, a.BS, a.NB, a.scale_log2);
  wv.run(
      [&](PoolRange& r) {
        while (u < u_end) {
          const unsigned t0 = __builtin_amdgcn_readfirstlane(tp[b]), t1 = __builtin_amdgcn_readfirstlane(tp[b + 1]);
          const unsigned nb = t1 - t0, base = (unsigned)a.ngroups * t0;
          if (u >= base + (unsigned)a.ngroups * nb) {  // past the sequence, or none of it
            ++b;
            continue;
          }
          const unsigned grp = (u - base) / nb, i0 = (u - base) - grp * nb;
          const unsigned stop = min(u_end, base + (grp + 1) * nb);
          const int kh = grp * a.hg + head, i1 = (int)(i0 + (stop - u));
          u = stop;
          if (kh >= a.Hkv) continue;
          int start, L;
          if (b < KNOWN) {
            start = __builtin_amdgcn_readfirstlane(s.prefix[2 * b]);
            L = __builtin_amdgcn_readfirstlane(s.prefix[2 * b + 1]);
          } else {
            int64_t tokens;
            group_of(a, s, starts, b, tokens);
            start = __builtin_amdgcn_readfirstlane((int)tokens);
            L = __builtin_amdgcn_readfirstlane((int)min(a.ctx_lens[b], cap));
          }
          r.btrow = a.bt + (int64_t)b * a.bt_stride;
          r.q = a.q + ((int64_t)b * a.Hkv + kh) * a.G * D;
          r.out = nullptr;
          r.prow = (((int64_t)v + (int64_t)b * a.ngroups + grp) * a.hg + head) * a.G;
          r.t0 = start + (int)i0 * T, r.t1 = min(L, start + i1 * T), r.kh = kh;
          return true;
        }
        return false;
      },
      nullptr, a.so, a.sml);
}

template <int D, bool ONE>
__global__ __launch_bounds__(256, 2) void paged_shared_kernel(SharedArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[SMEM];
  __shared__ SharedLds lds;
  static_assert(SMEM >= 4 * KT * 2 * D, "K and V tiles, two each");
  const int w = blockIdx.x;
  if (w < a.nprefix) prefix_role<D>(a, smem, lds, w);
  else rest_role<D, ONE>(a, smem, lds, w - a.nprefix);
}

// One wave per 64 elements of an output row: the weights of up to 64 parts at a
// time, one a lane, then their values in order.  With qo also the act_quant of
// the 128 values that a workgroup holds, as paged_decode_merge_quant_group.
constexpr int MU = 16;
template <int D>
__global__ __launch_bounds__(128) void paged_shared_merge(SharedArgs a, uint16_t* __restrict__ out,
                                                          uint8_t* __restrict__ qo, float* __restrict__ qs, int64_t E) {
  __shared__ __attribute__((aligned(16))) uint16_t vals[128];
  const int64_t e = (int64_t)blockIdx.x * 128 + threadIdx.x;
  const int lane = threadIdx.x & 63;
  uint16_t v = 0;
  if (e < E) {  // a wave's 64 elements are all in or all out
    const int64_t hrow = __builtin_amdgcn_readfirstlane((int)(e / D));  // (sequence, query head)
    const int d = (int)(e % D), Hq = a.Hkv * a.G;
    const int b = (int)(hrow / Hq), hq = (int)(hrow - (int64_t)b * Hq), kh = hq / a.G, gq = hq - kh * a.G;
    int np = 0, ns = 0;
    int64_t prow = 0, srow = 0;
    const int g = a.group[b];
    if (g >= 0) {
      const int first = a.starts[g], n = a.starts[g + 1] - first;
      const unsigned nt = key_tiles(prefix_tokens(a, g, n));
      if (nt > 0) {
        const unsigned total = a.punits[a.NG], Ct = max(1u, (total + a.nprefix - 1) / a.nprefix);
        const int r = (b - first) * a.G + gq, rt = r / PROWS;
        const unsigned base = a.punits[g] + (unsigned)(kh * row_tiles(a, n) + rt) * nt;
        const unsigned wf = base / Ct;
        np = (int)((base + nt - 1) / Ct - wf) + 1;
        prow = (int64_t)wf * PROWS + (int64_t)first * a.G * a.Hkv + (int64_t)kh * n * a.G + r;
      }
    }
    const unsigned nb = a.stiles[b + 1] - a.stiles[b];
    if (nb > 0) {
      const unsigned nwg = a.nrest * (NW / a.hg), total = (unsigned)a.ngroups * (unsigned)a.stiles[a.B];
      const unsigned Ct = max(1u, (total + nwg - 1) / nwg);
      const int grp = kh / a.hg;
      const unsigned base = (unsigned)a.ngroups * (unsigned)a.stiles[b] + grp * nb, wf = base / Ct;
      ns = (int)((base + nb - 1) / Ct - wf) + 1;
      srow = (((int64_t)wf + (int64_t)b * a.ngroups + grp) * a.hg + (kh - grp * a.hg)) * a.G + gq;
    }
    float M = -INFINITY, num = 0.f, den = 0.f;
    for (int c = 0; c < np + ns; c += 64) {
      const int i = c + lane;
      float m = -INFINITY, l = 0.f;
      if (i < np + ns) {
        const float* ml = i < np ? a.pml + (prow + (int64_t)i * PROWS) * 2 : a.sml + (srow + (int64_t)(i - np) * a.hg * a.G) * 2;
        m = ml[0], l = ml[1];
      }
      const float Mn = fmaxf(M, group_max<64>(m));
      if (Mn == -INFINITY) continue;
      const float old = M == -INFINITY ? 0.f : exp2f(M - Mn), w = exp2f(m - Mn);
      num *= old;
      den = fmaf(den, old, group_sum<64>(w * l));
      M = Mn;
      const int cnt = min(64, np + ns - c);
      for (int s0 = 0; s0 < cnt; s0 += MU) {  // MU values in flight
        float o[MU];
#pragma unroll
        for (int s = 0; s < MU; ++s) {
          const int k = c + min(s0 + s, cnt - 1);
          o[s] = (k < np ? a.po + (prow + (int64_t)k * PROWS) * D : a.so + (srow + (int64_t)(k - np) * a.hg * a.G) * D)[d];
        }
#pragma unroll
        for (int s = 0; s < MU; ++s)
          if (s0 + s < cnt) num = fmaf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), s0 + s)), o[s], num);
      }
    }
    v = (uint16_t)f32_to_bf16(den > 0.f ? num / den : 0.f);
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

// Partial rows of a call, at most: the prefix workgroups' and the batch's, and the
// rest's as in lfs_paged_decode's balanced split; D + 2 floats each.
int64_t prefix_rows(int64_t B, int Hq) { return (int64_t)decode_cu_count() * PROWS + B * Hq; }
int64_t rest_rows(int64_t B, int Hq) { return (8 * (int64_t)decode_cu_count() + 2 * B) * Hq; }

}  // namespace
}  // namespace lfs

using namespace lfs;

extern "C" int64_t lfs_paged_decode_shared_workspace_bytes(int64_t B, int64_t num_groups, int32_t num_q_heads,
                                                           int32_t num_kv_heads, int32_t head_dim) {
  if (B < 0 || num_groups < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return -1;
  return 4 * (prefix_rows(B, num_q_heads) + rest_rows(B, num_q_heads)) * ((int64_t)head_dim + 2) +
         4 * (2 * (num_groups + 1) + 2 * B + 1);
}

extern "C" int lfs_paged_decode_shared(const void* q, const void* k_cache, const void* v_cache,
                                       const int64_t* context_lens, const int32_t* block_tables, int64_t bt_stride,
                                       const int32_t* cu_groups, const int32_t* shared_blocks, int64_t num_groups,
                                       void* out, void* workspace, int64_t workspace_bytes, int64_t B,
                                       int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                       int64_t num_blocks, int32_t max_blocks, float scale, void* q_out, float* q_scale,
                                       void* stream) {
  const int Hq = num_q_heads, Hkv = num_kv_heads, D = head_dim, BS = block_size;
  LFS_REQUIRE(num_groups >= 0, "paged_decode_shared: bad shape");
  const int rc = check_decode("paged_decode_shared", q, k_cache, v_cache, context_lens, block_tables, bt_stride, out,
                              workspace, workspace_bytes,
                              lfs_paged_decode_shared_workspace_bytes(B, num_groups, Hq, Hkv, D), B, Hq, Hkv, D, BS,
                              num_blocks, max_blocks, q_out, q_scale);
  if (rc || B == 0) return rc;
  LFS_REQUIRE(cu_groups && (num_groups == 0 || shared_blocks), "paged_decode_shared: null pointer");
  LFS_REQUIRE(B <= BAL_MAXB && num_groups <= BAL_MAXB, "paged_decode_shared: at most %d sequences and groups (got %lld, %lld)",
              BAL_MAXB, (long long)B, (long long)num_groups);
  LFS_REQUIRE((int64_t)Hkv * D * 256 < (1ll << 31), "paged_decode_shared: too many kv heads (%d)", Hkv);
  const int T = D == 64 ? 64 : 32, G = Hq / Hkv;
  const int64_t tokens = (int64_t)max_blocks * BS;
  LFS_REQUIRE(tokens < (1ll << 31) - 4096, "paged_decode_shared: block tables of 2^31 tokens");
  SharedArgs a{};
  a.hg = Hkv < NW ? Hkv : NW;
  a.ngroups = (Hkv + a.hg - 1) / a.hg;
  LFS_REQUIRE(((B * G + PROWS - 1) / PROWS + std::min(B / 2, num_groups)) * Hkv * ((tokens + KT - 1) / KT) < (1ll << 31) &&
                  B * a.ngroups * ((tokens + T - 1) / T) < (1ll << 31),
              "paged_decode_shared: too many context tiles");
  const int64_t E = B * Hq * D;
  LFS_REQUIRE(E <= (1ll << 32) - 128, "paged_decode_shared: too many outputs");  // a thread each, less than 2^32 a launch
  const int64_t prows = prefix_rows(B, Hq), srows = rest_rows(B, Hq);
  a.q = (const uint16_t*)q, a.kc = (const uint16_t*)k_cache, a.vc = (const uint16_t*)v_cache;
  a.ctx_lens = context_lens, a.bt = block_tables, a.bt_stride = bt_stride;
  a.cu = cu_groups, a.shared = shared_blocks;
  a.po = (float*)workspace, a.so = a.po + prows * D;
  a.pml = a.so + srows * D, a.sml = a.pml + prows * 2;
  a.starts = (int*)(a.sml + srows * 2), a.punits = a.starts + num_groups + 1;
  a.stiles = a.punits + num_groups + 1, a.group = a.stiles + B + 1;
  a.Hkv = Hkv, a.G = G, a.BS = BS, a.NG = (int)num_groups, a.B = (int)B, a.max_blocks = max_blocks, a.NB = num_blocks;
  a.nprefix = a.nrest = decode_cu_count();
  a.scale_log2 = scale * 1.4426950408889634f;
  const dim3 grid((unsigned)(a.nprefix + a.nrest));
  hipStream_t st = (hipStream_t)stream;
  const bool one = BS % T == 0;
#define LFS_SHARED(DD, ONE) hipLaunchKernelGGL((paged_shared_kernel<DD, ONE>), grid, dim3(256), 0, st, a)
  if (D == 64 && one) LFS_SHARED(64, true);
  else if (D == 64) LFS_SHARED(64, false);
  else if (one) LFS_SHARED(128, true);
  else LFS_SHARED(128, false);
#undef LFS_SHARED
  const int rc2 = check_launch("paged_decode_shared");
  if (rc2) return rc2;
  if (D == 64)
    hipLaunchKernelGGL((paged_shared_merge<64>), dim3((unsigned)((E + 127) / 128)), dim3(128), 0, st, a, (uint16_t*)out,
                       (uint8_t*)q_out, q_scale, E);
  else
    hipLaunchKernelGGL((paged_shared_merge<128>), dim3((unsigned)((E + 127) / 128)), dim3(128), 0, st, a, (uint16_t*)out,
                       (uint8_t*)q_out, q_scale, E);
  return check_launch("paged_decode_shared(merge)");
}
