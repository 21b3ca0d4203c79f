// One token per row of logits by temperature, top-k, top-p and min-p, from a
// given uniform number u in [0, 1).
//
// A row's tokens are ordered by logit, largest first, equal ones by index,
// with weights w_i = exp((x_i - x_max) / T).  top-k keeps the first k of the
// order; top-p of those the shortest prefix whose weight reaches p times
// theirs; min-p the tokens with w_i >= min_p.  Each keeps a prefix of the
// order, so together they keep the shortest of the three.  The token is the
// first of the order at which the kept weight summed so far exceeds u times
// all of it.
//
// Logits are bf16, so equal logits are common and a row has at most 65280
// different ones: counts by value (bins, largest first) carry everything the
// order does.  A bin's tokens weigh the same, so a cut inside one is a
// division, and an exponential is taken per value and not per token.
// Weights and their sums are held in 64 bits: with 32 the borders of tokens
// in the tail of a wide vocabulary move by more than the tokens weigh.
//
// One workgroup per row, which it reads once, into registers (longer rows are
// read again).  Counts of all 65536 bit patterns stand in 128 KiB of LDS, two
// 16-bit ones a word, under the tokens' own bits: a token costs a few
// instructions and one LDS addition.  A count past 65535 carries or is lost,
// so that the counts no longer add up to the tokens; such a row is counted
// again in 32-bit bins, a window of them at a time.  A value that holds many
// of the row (a mask's, say) is counted by ballots and not in LDS, where its
// additions would queue up: one that 8 of 64 samples have.  One wave then
// walks the counts (512 chunks of 128 bins, a chunk an exponent and a sign)
// for the cuts, and the workgroup looks up the token among equals.
#include "common.h"

namespace lfs {
namespace {

constexpr int FNT = 1024;            // threads
constexpr int FNW = FNT / 64;
constexpr int kBins = 65536;
constexpr int kChunk = 128;          // bins of a chunk: two per lane
constexpr int kChunks = kBins / kChunk;
constexpr int CPL = kChunks / 64;    // chunks per lane
constexpr int kWindow = 32768;       // 32-bit bins counted at once
constexpr uint32_t kNever = 0xFFFFu; // a NaN, in the place of tokens past the row

// Bin of a logit, 0 the largest value; kBins for one that is never drawn
// (-infinity, NaN).  -0 and +0 are equal.
__device__ __forceinline__ int bin_of(uint32_t h) {
  if ((h & 0x7FFFu) > 0x7F80u || h == 0xFF80u) return kBins;
  if (h == 0x8000u) h = 0;
  return (h & 0x8000u) ? (int)h : 0x7FFF - (int)h;
}
__device__ __forceinline__ uint32_t bits_of(int d) { return d < 0x8000 ? 0x7FFFu - d : (uint32_t)d; }
__device__ __forceinline__ double bin_value(int d) { return (double)bf16_to_f32(bits_of(d)); }

// The weights of a row.
struct Weights {
  int top;  // the largest logit's bin
  double xmax, T;
  __device__ __forceinline__ double at(int d) const {
    if (d == top) return 1.0;
    const double w = exp((bin_value(d) - xmax) / T);
    return w == w ? w : 0.0;  // infinite logit and temperature
  }
};

// Inclusive sums over the wave's lanes.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)moved<CTRL, ROWS>((uint32_t)b) |
                                        (uint64_t)moved<CTRL, ROWS>((uint32_t)(b >> 32)) << 32);
}
template <class X>
__device__ __forceinline__ X scan_sum(X v) {
  v += moved<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  v += moved<0x142, 0xA>(v);  // row_bcast 15: rows 1 and 3
  v += moved<0x143, 0xC>(v);  // row_bcast 31: rows 2 and 3
  return v;
}
__device__ __forceinline__ double lane_d(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane);
  const uint64_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, lo | hi << 32);
}
__device__ __forceinline__ uint32_t lane_u(uint32_t v, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

// 64 * N entries of a wave in order (entry N * lane + i), each a count and a
// weight, and their sums before the lane's first.
template <int N>
struct Entries {
  uint32_t n[N], nb;
  double w[N], wb;
  __device__ __forceinline__ void scan() {
    uint32_t ns = 0;
    double ws = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) ns += n[i], ws += w[i];
    nb = scan_sum(ns) - ns;
    wb = __shfl_up(scan_sum(ws), 1, 64);
    if ((threadIdx.x & 63) == 0) wb = 0.0;
  }
  // The first entry that is not empty and at whose end pred(count, weight)
  // holds of the sums so far, which start at c and m; the last one that is not
  // empty where none does (-1: all are empty).  c and m become the sums before
  // it.
  template <class Pred>
  __device__ __forceinline__ int find(uint32_t& c, double& m, Pred&& pred) const {
    uint32_t cb = c + nb;
    double mb = m + wb;
    int hit = -1, last = -1;  // in the lane
    uint32_t hc = 0, lc = 0;
    double hm = 0.0, lm = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (n[i] != 0) {
        if (hit < 0 && pred(cb + n[i], mb + w[i])) hit = i, hc = cb, hm = mb;
        last = i, lc = cb, lm = mb;
      }
      cb += n[i], mb += w[i];
    }
    uint64_t any = __ballot(hit >= 0);
    if (any == 0) {
      any = __ballot(last >= 0);
      if (any == 0) return -1;
      any = 1ull << (63 - __builtin_clzll(any));
      hit = last, hc = lc, hm = lm;
    }
    const int src = __builtin_ctzll(any);
    c = lane_u(hc, src);
    m = lane_d(hm, src);
    return N * src + (int)lane_u((uint32_t)hit, src);
  }
};

// A place in the order: n tokens of bin d, after all of the bins before it;
// c and m: their count and weight.
struct Place {
  int d;
  uint32_t n, c;
  double m;
};

struct Filters {
  int64_t k;      // <= 0: off
  double p, m, u;
};

// The cuts and the draw, by one wave or by several alike.  hold(chunk, bins)
// fills in a chunk's two bins per lane.  d: the drawn token's bin, nth: its
// place among the bin's tokens, S: the kept weight.
template <class Hold>
__device__ __forceinline__ void draw(const Weights& wt, const Filters& f, const uint32_t* cnt, const double* mass,
                                     Hold&& hold_bins, int& d, uint32_t& nth, double& S) {
  const int lane = threadIdx.x & 63;
  Entries<CPL> ch;
#pragma unroll
  for (int i = 0; i < CPL; ++i) ch.n[i] = cnt[CPL * lane + i], ch.w[i] = ch.n[i] != 0 ? mass[CPL * lane + i] : 0.0;
  ch.scan();
  Entries<2> bn;
  int held = -1;
  auto hold = [&](int chunk) {
    if (chunk == held) return;
    held = chunk;
    hold_bins(chunk, bn.n);
#pragma unroll
    for (int i = 0; i < 2; ++i) bn.w[i] = bn.n[i] != 0 ? bn.n[i] * wt.at(chunk * kChunk + 2 * lane + i) : 0.0;
    bn.scan();
  };
  // the first bin at whose end pred holds of the count and weight so far
  auto find = [&](auto&& pred) -> Place {
    Place at{0, 0, 0, 0.0};
    const int chunk = ch.find(at.c, at.m, pred);
    hold(chunk);
    const int e = bn.find(at.c, at.m, pred);
    at.d = chunk * kChunk + e;
    at.n = lane_u((e & 1) ? bn.n[1] : bn.n[0], e >> 1);
    return at;
  };
  // top-k: the first k tokens
  Place end = find([&](uint32_t c, double) { return f.k > 0 && c >= (uint64_t)f.k; });
  if (f.k > 0 && end.c + (uint64_t)end.n > (uint64_t)f.k) end.n = (uint32_t)(f.k - end.c);
  S = end.m + end.n * wt.at(end.d);
  // top-p: the tokens before which the weight is below the target
  if (f.p < 1.0) {
    const double target = f.p * S;
    Place at = find([&](uint32_t, double m) { return m >= target; });
    const double need = ceil((target - at.m) / wt.at(at.d));
    at.n = need >= 1.0 ? (need < (double)at.n ? (uint32_t)need : at.n) : 1u;
    if (at.d < end.d || (at.d == end.d && at.n < end.n)) end = at;
  }
  // min-p: the last bin whose weight reaches it, 64 bins tried at a time
  if (f.m > 1.0) {
    end = Place{wt.top, 1, 0, 0.0};
  } else if (f.m > 0.0 && wt.at(end.d) < f.m) {
    int lo = wt.top;  // at(lo) >= m
#pragma unroll 1
    for (int step = 1024; step > 0; step >>= step == 1024 ? 6 : 4) {  // 1024, 16, 1
      const int mid = lo + step * (lane + 1);
      const uint64_t in = __ballot(mid < kBins && wt.at(min(mid, kBins - 1)) >= f.m);
      lo += step * (in == ~0ull ? 64 : __builtin_ctzll(~in));
    }
    const int chunk = lo / kChunk;
    hold(chunk);
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < CPL; ++i) n += CPL * lane + i < chunk ? ch.n[i] : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) n += chunk * kChunk + 2 * lane + i <= lo ? bn.n[i] : 0;
    n = lane_u(scan_sum(n), 63);
    end = find([&](uint32_t c, double) { return c >= n; });
  }
  S = end.m + end.n * wt.at(end.d);
  const double target = f.u * S;
  Place at = find([&](uint32_t, double m) { return m > target; });
  if (at.d > end.d) at = end;
  if (at.d == end.d) at.n = min(at.n, end.n);
  const double skip = floor((target - at.m) / wt.at(at.d));
  d = at.d;
  nth = skip > 0.0 ? (skip < (double)(at.n - 1) ? (uint32_t)skip : at.n - 1) : 0u;
}

// NR: 16-byte pieces of the row that a thread holds; 0: rows of any length.
template <int NR>
__global__ __launch_bounds__(FNT) void sample_filtered_kernel(
    const uint16_t* __restrict__ logits, int64_t ld, const float* __restrict__ temps,
    const float* __restrict__ uniforms, const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
    const float* __restrict__ min_p, int V, int64_t* __restrict__ out, float* __restrict__ logprob) {
  __shared__ __attribute__((aligned(16))) uint32_t hist[kWindow];
  __shared__ double mass[kChunks];
  __shared__ double drawn_s;
  __shared__ uint32_t cnt[kChunks];
  __shared__ uint32_t bins[kChunk];
  __shared__ uint32_t places[(NR > 0 ? NR : 1) * FNW];
  __shared__ uint32_t many_n, drawn_n;
  __shared__ int drawn_d;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t b = blockIdx.x;
  const uint16_t* row = logits + b * ld;
  // 16-byte pieces: piece i holds tokens 8i - skew .. + 7
  const int skew = (int)(((uintptr_t)row >> 1) & 7), pieces = (int)(((int64_t)V + skew + 7) / 8);
  auto piece = [&](int i) -> uint4 {
    const int64_t t = 8ll * i - skew;
    if (t >= 0 && t + 8 <= V) return *reinterpret_cast<const uint4*>(row + t);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t a = t + 2 * e;
      w[e] = (a >= 0 && a < V ? row[a] : kNever) | (a + 1 >= 0 && a + 1 < V ? row[a + 1] : kNever) << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  uint4 held[NR > 0 ? NR : 1];
  if constexpr (NR > 0) {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      held[r] = make_uint4(~0u, ~0u, ~0u, ~0u);
      if (r * FNT + tid < pieces) held[r] = piece(r * FNT + tid);
    }
  }
  // a value that many of 64 samples have (the same samples for every wave)
  const uint32_t sample = row[(int64_t)lane * V >> 6];
  const float T = temps[b];
  Filters f;
  f.k = top_k != nullptr ? top_k[b] : 0;
  if (!(T > 0.f)) f.k = 1;  // greedy
  f.p = top_p != nullptr ? (double)top_p[b] : 1.0;
  f.m = min_p != nullptr ? (double)min_p[b] : 0.0;
  f.u = fmin(fmax((double)uniforms[b], 0.0), 1.0 - 0x1p-24);  // a NaN counts as 0
  for (int i = tid; i < kWindow / 4; i += FNT) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
  if (tid == 0) many_n = 0;
  uint32_t many = ~0u;
#pragma unroll 1
  for (int e = 0; e < 64; e += 3) {  // one of its samples is met
    const uint32_t v = lane_u(sample, e);
    if (__popcll(__ballot(sample == v)) >= 8) {
      many = v;
      break;
    }
  }
  __syncthreads();

  // the counts: low half of word h & 0x7FFF for bits h < 0x8000, high half for the others
  auto add = [&](uint32_t h) { atomicAdd(&hist[h & 0x7FFFu], (h >> 15) * 0xFFFFu + 1u); };
  uint32_t many_here = 0;  // of the wave
  auto count = [&](const uint4& x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    if (many == ~0u) {
#pragma unroll
      for (int e = 0; e < 4; ++e) add(w[e] & 0xFFFFu), add(w[e] >> 16);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t h = (e & 1) ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu;
        many_here += __popcll(__ballot(h == many));
        if (h != many) add(h);
      }
    }
  };
  int waves_pieces = 0;  // of the wave
  if constexpr (NR > 0) {
#pragma unroll
    for (int r = 0; r < NR; ++r)
      if (r * FNT + wave * 64 < pieces) count(held[r]), ++waves_pieces;
  } else {
    for (int i = wave * 64; i < pieces; i += FNT) {
      uint4 x = make_uint4(~0u, ~0u, ~0u, ~0u);
      if (i + lane < pieces) x = piece(i + lane);
      count(x);
      ++waves_pieces;
    }
  }
  if (lane == 0 && many_here != 0) atomicAdd(&many_n, many_here);
  __syncthreads();
  const uint32_t many_all = many_n;
  // tokens of bin d
  auto bits_count = [&](uint32_t h) -> uint32_t {
    const uint32_t w = hist[h & 0x7FFFu];
    return ((h >> 15) ? w >> 16 : w & 0xFFFFu) + (h == many ? many_all : 0u);
  };
  auto bin_count = [&](int d) -> uint32_t {
    if (d < 0x7F || d >= 0xFF80 || d == 0x8000) return 0;  // NaN, -infinity; -0 counts as +0
    const uint32_t n = bits_count(bits_of(d));
    return d == 0x7FFF ? n + bits_count(0x8000u) : n;
  };
  uint32_t sum = 0;  // of all counts, drawable or not
  for (int i = tid; i < kWindow; i += FNT) sum += (hist[i] & 0xFFFFu) + (hist[i] >> 16);
  for (int c = wave; c < kChunks; c += FNW) {
    const uint32_t n = lane_u(scan_sum(bin_count(c * kChunk + 2 * lane) + bin_count(c * kChunk + 2 * lane + 1)), 63);
    if (lane == 0) cnt[c] = n;
  }
  sum = lane_u(scan_sum(sum), 63) + many_here - 512u * waves_pieces;
  if (tid < 128) bins[tid] = 0;
  __syncthreads();
  if (lane == 0 && sum != 0) atomicAdd(&bins[0], sum);  // modulo 2^32: 0 over the waves where nothing was lost
  __syncthreads();
  const bool counted = bins[0] == 0;

  // the largest logit
  auto first_chunk = [&]() -> int {
    int c = kChunks;
#pragma unroll
    for (int i = CPL - 1; i >= 0; --i)
      if (cnt[CPL * lane + i] != 0) c = CPL * lane + i;
    const uint64_t any = __ballot(c < kChunks);
    return any == 0 ? -1 : (int)lane_u((uint32_t)c, __builtin_ctzll(any));
  };
  auto first_bin = [&](int chunk, uint32_t n0, uint32_t n1) -> int {
    const int src = __builtin_ctzll(__ballot(n0 + n1 != 0));
    return chunk * kChunk + 2 * src + (lane_u(n0, src) != 0 ? 0 : 1);
  };
  Weights wt;
  wt.T = (double)T;
  int d = 0;
  uint32_t nth = 0;
  double S = 0.0;
  if (counted) {
    const int c0 = first_chunk();
    if (c0 < 0) {  // nothing can be drawn
      if (tid == 0) {
        out[b] = 0;
        if (logprob != nullptr) logprob[b] = -INFINITY;
      }
      return;
    }
    wt.top = first_bin(c0, bin_count(c0 * kChunk + 2 * lane), bin_count(c0 * kChunk + 2 * lane + 1));
    wt.xmax = bin_value(wt.top);
    for (int c = wave; c < kChunks; c += FNW) {
      if (cnt[c] == 0) continue;
      const int e = c * kChunk + 2 * lane;
      const uint32_t n0 = bin_count(e), n1 = bin_count(e + 1);
      const double m = (n0 != 0 ? n0 * wt.at(e) : 0.0) + (n1 != 0 ? n1 * wt.at(e + 1) : 0.0);
      const double all = lane_d(scan_sum(m), 63);
      if (lane == 0) mass[c] = all;
    }
    __syncthreads();
    if (wave == 0) {
      draw(wt, f, cnt, mass, [&](int chunk, uint32_t (&n)[2]) {
        n[0] = bin_count(chunk * kChunk + 2 * lane), n[1] = bin_count(chunk * kChunk + 2 * lane + 1);
      }, d, nth, S);
      if (lane == 0) drawn_d = d, drawn_n = nth, drawn_s = S;
    }
    __syncthreads();
    d = drawn_d, nth = drawn_n, S = drawn_s;
  } else {
    // a count did not fit: 32-bit bins, a window at a time, from the row itself
    bool found = false;
    wt.top = 0, wt.xmax = 0.0;
    auto recount = [&](int first, int n, uint32_t* to) {  // the bins first .. first + n - 1
      __syncthreads();
      for (int i = tid; i < n; i += FNT) to[i] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += FNT) {
        const int e = bin_of(row[i]) - first;
        if (e >= 0 && e < n) atomicAdd(&to[e], 1u);
      }
      __syncthreads();
    };
    for (int w0 = 0; w0 < kBins; w0 += kWindow) {
      recount(w0, kWindow, hist);
      for (int c = wave; c < kWindow / kChunk; c += FNW) {
        const uint32_t n = lane_u(scan_sum(hist[c * kChunk + 2 * lane] + hist[c * kChunk + 2 * lane + 1]), 63);
        if (lane == 0) cnt[w0 / kChunk + c] = n;
      }
      if (w0 == 0)  // not yet counted
        for (int c = kWindow / kChunk + tid; c < kChunks; c += FNT) cnt[c] = 0;
      __syncthreads();
      if (!found) {
        const int c0 = first_chunk();
        if (c0 >= 0) {
          found = true;
          const uint32_t* h = &hist[c0 * kChunk - w0];
          wt.top = first_bin(c0, h[2 * lane], h[2 * lane + 1]);
          wt.xmax = bin_value(wt.top);
        }
      }
      for (int c = wave; found && c < kWindow / kChunk; c += FNW) {
        const int e = c * kChunk + 2 * lane;
        const uint32_t n0 = hist[e], n1 = hist[e + 1];
        const double m = (n0 != 0 ? n0 * wt.at(w0 + e) : 0.0) + (n1 != 0 ? n1 * wt.at(w0 + e + 1) : 0.0);
        const double all = lane_d(scan_sum(m), 63);
        if (lane == 0) mass[w0 / kChunk + c] = all;
      }
    }
    __syncthreads();
    if (!found) {
      if (tid == 0) {
        out[b] = 0;
        if (logprob != nullptr) logprob[b] = -INFINITY;
      }
      return;
    }
    draw(wt, f, cnt, mass, [&](int chunk, uint32_t (&n)[2]) {  // the whole workgroup, the same chunk
      recount(chunk * kChunk, kChunk, bins);
      n[0] = bins[2 * lane], n[1] = bins[2 * lane + 1];
    }, d, nth, S);
  }

  // the nth of the bin's tokens by index
  auto done = [&](int64_t token) {
    out[b] = token;
    if (logprob != nullptr) logprob[b] = (float)((d == wt.top ? 0.0 : (bin_value(d) - wt.xmax) / wt.T) - log(S));
  };
  const uint32_t bits = bits_of(d), alt = bits == 0 ? 0x8000u : bits;
  auto matches = [&](const uint4& x) -> uint32_t {  // a bit for each of the eight
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t h = (e & 1) ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu;
      m |= h == bits || h == alt ? 1u << e : 0u;
    }
    return m;
  };
  // in the 64 pieces of a wave from piece i on, of which a lane's holds m: the
  // token if the nth is there, else nth less those there
  auto pick = [&](uint32_t m, int i) -> bool {
    const uint32_t mine = __popc(m), upto = scan_sum(mine), all = lane_u(upto, 63);
    if (nth >= all) {
      nth -= all;
      return false;
    }
    if (nth < upto && nth >= upto - mine) {
      for (uint32_t skip = nth - (upto - mine); skip > 0; --skip) m &= m - 1;
      done(8ll * (i + lane) - skew + __builtin_ctz(m));
    }
    return true;
  };
  if constexpr (NR > 0) {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const uint32_t n = lane_u(scan_sum((uint32_t)__popc(matches(held[r]))), 63);
      if (lane == 0) places[r * FNW + wave] = n;
    }
    __syncthreads();
    uint32_t at = 0;  // tokens of the bin before the wave's r-th pieces
    int mine = -1;
    constexpr int PPL = (NR * FNW + 63) / 64;
    uint32_t n[PPL], before = 0;
#pragma unroll
    for (int i = 0; i < PPL; ++i) {
      n[i] = PPL * lane + i < NR * FNW ? places[PPL * lane + i] : 0;
      before += n[i];
    }
    before = scan_sum(before) - before;
#pragma unroll
    for (int i = 0; i < PPL; ++i) {
      if (nth >= before && nth < before + n[i]) mine = PPL * lane + i, at = before;
      before += n[i];
    }
    const uint64_t any = __ballot(mine >= 0);
    if (any == 0) return;  // not reached: the bin holds more than nth tokens
    const int src = __builtin_ctzll(any), place = (int)lane_u((uint32_t)mine, src);
    if (place % FNW != wave) return;
    nth -= lane_u(at, src);
#pragma unroll
    for (int r = 0; r < NR; ++r)
      if (r == place / FNW) pick(matches(held[r]), r * FNT + wave * 64);
  } else {
    const int per = ((pieces + FNW - 1) / FNW + 63) & ~63;  // pieces of a wave
    const int i0 = min(pieces, wave * per), i1 = min(pieces, i0 + per);
    auto at = [&](int i) { return i + lane < i1 ? matches(piece(i + lane)) : 0u; };
    uint32_t here = 0;
    for (int i = i0; i < i1; i += 64) here += __popc(at(i));
    here = lane_u(scan_sum(here), 63);
    if (lane == 0) places[wave] = here;
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
      if (nth < places[w]) return;
      nth -= places[w];
    }
    if (nth >= here) return;
    for (int i = i0; i < i1; i += 64)
      if (pick(at(i), i)) return;
  }
}

}  // namespace
}  // namespace lfs

using namespace lfs;

extern "C" int lfs_sample_filtered(const void* logits, int64_t ld, const float* temperatures, const float* uniforms,
                                   const int32_t* top_k, const float* top_p, const float* min_p, int64_t B,
                                   int32_t vocab, int64_t* out, float* logprob, void* stream) {
  LFS_REQUIRE(B >= 0 && vocab > 0 && ld >= vocab, "sample_filtered: bad shape B=%lld V=%d ld=%lld", (long long)B, vocab,
              (long long)ld);
  if (B == 0) return 0;
  LFS_REQUIRE(logits && temperatures && uniforms && out, "sample_filtered: null pointer");
  LFS_REQUIRE(B < (1ll << 22), "sample_filtered: too many rows");
  LFS_REQUIRE(vocab <= (1 << 30), "sample_filtered: vocabulary too large");
#define LFS_SF(NR)                                                                                                  \
  hipLaunchKernelGGL(sample_filtered_kernel<NR>, dim3((unsigned)B), dim3(FNT), 0, (hipStream_t)stream,               \
                     (const uint16_t*)logits, ld, temperatures, uniforms, top_k, top_p, min_p, vocab, out, logprob)
  const int64_t pieces = ((int64_t)vocab + 7 + 7) / 8;  // at any alignment
  if (pieces <= 5 * FNT) LFS_SF(5);
  else if (pieces <= 10 * FNT) LFS_SF(10);
  else if (pieces <= 20 * FNT) LFS_SF(20);
  else LFS_SF(0);
#undef LFS_SF
  return check_launch("sample_filtered");
}
