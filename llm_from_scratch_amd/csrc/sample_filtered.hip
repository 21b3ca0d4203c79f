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
// One workgroup per row.  Counts of all 65536 bit patterns stand in 128 KiB of
// LDS, two 16-bit ones a word, under the tokens' own bits: a token costs a few
// instructions and one LDS addition.  A count past 65535 carries or is lost,
// so that the counts no longer add up to the tokens; such a row is counted
// again in 32-bit bins, a window of them at a time.  A value that holds many
// of the row (a mask's, say) is counted by ballots and not in LDS, where its
// additions would queue up: one that 8 of 64 samples have.  One wave then
// walks the counts (512 chunks of 128 bins, a chunk an exponent and a sign)
// for top-k, top-p and the draw, another for min-p's cut; meanwhile the others
// read the row again, from the caches, into registers, and find the token
// among equals there.
//
// Measured: 256 rows of 150001 with top-p and min-p 39 us, one row of 32000
// with all filters 14.5 us.  The bound is not memory (the logits of the 256 take
// 16 us), but a chain of phases: of a long row's 74000 cycles (one of 256) the
// counting takes 30000, by HBM and one LDS addition a token at nine cycles a
// wave's, the sums of counts and of weights 11000, by instructions (16 cycles
// each over the workgroup, 32 in 64 bits), the cuts 8000, by one wave's
// latencies, and the second read and its search 19000; a row of 32000 has 6200,
// 11000, 7000 and 3000 of 32000.  Loads begun while LDS is cleared and beside
// the counting took the 256 rows to 41.6 us, the cuts as a loop over one
// search one row to 16.7.
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
constexpr int FU = 8;                // 16-byte pieces of the row that a thread has in flight
constexpr int FH = 22;               // and that a thread of all waves but two holds
constexpr int FNH = FNT - 128;
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
constexpr int kList = FNT;           // equal tokens ranked as a list, one a thread

// Bin of a logit, 0 the largest value; kBins for one that is never drawn
// (-infinity, NaN).  -0 and +0 are equal.
__device__ __forceinline__ int bin_of(uint32_t h) {
  if ((h & 0x7FFFu) > 0x7F80u || h == 0xFF80u) return kBins;
  if (h == 0x8000u) h = 0;
  return (h & 0x8000u) ? (int)h : 0x7FFF - (int)h;
}
__device__ __forceinline__ uint32_t bits_of(int d) { return d < 0x8000 ? 0x7FFFu - d : (uint32_t)d; }
__device__ __forceinline__ double bin_value(int d) { return (double)bf16_to_f32(bits_of(d)); }

// The weights of a row: 2^((x - x_max) log2(e) / T), by its Taylor series at
// the exponent's nearest whole number (|f ln 2| <= 0.35: the first term left out
// is below 2^-52).  Weights below 2^-1000 count as 0.
struct Weights {
  int top;  // the largest logit's bin
  double xmax, c;
  __device__ __forceinline__ double at(int d) const { return d == top ? 1.0 : of(bin_value(d) - xmax); }
  __device__ __forceinline__ double of(double x) const {
    const double t = x * c, n = rint(t), f = (t - n) * 0.6931471805599453;
    double w = 1.0 / 479001600;
    w = fma(w, f, 1.0 / 39916800);
    w = fma(w, f, 1.0 / 3628800);
    w = fma(w, f, 1.0 / 362880);
    w = fma(w, f, 1.0 / 40320);
    w = fma(w, f, 1.0 / 5040);
    w = fma(w, f, 1.0 / 720);
    w = fma(w, f, 1.0 / 120);
    w = fma(w, f, 1.0 / 24);
    w = fma(w, f, 1.0 / 6);
    w = fma(w, f, 0.5);
    w = fma(w, f, 1.0);
    w = fma(w, f, 1.0);
    return t > -1000.0 ? ldexp(w, (int)n) : 0.0;  // NaN (an infinite logit and temperature): 0
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

// Sums over the lanes of each eight.
template <class X>
__device__ __forceinline__ X scan_sum8(X v) {
  const int at = threadIdx.x & 7;
  const X a = moved<0x111, 0xF>(v);  // row_shr: also from the eight before
  v += at >= 1 ? a : X(0);
  const X b = moved<0x112, 0xF>(v);
  v += at >= 2 ? b : X(0);
  const X c = moved<0x114, 0xF>(v);
  return v + (at >= 4 ? c : X(0));
}
template <class X>
__device__ __forceinline__ X before(X upto) {  // the lane before's; 0 in lane 0
  const X v = __shfl_up(upto, 1, 64);
  return (threadIdx.x & 63) == 0 ? X(0) : v;
}

// A place in the order: n tokens of bin d, w each, after all of the bins
// before it; c and m: their count and weight.
struct Place {
  int d;
  uint32_t n, c;
  double m, w;
};

struct Filters {
  int64_t k;      // <= 0: off
  double p, m, u;
};

// The last bin whose weight reaches m in (0, 1]: among the 64 around the one
// that the inverse formula names in 32 bits, or, where it lies outside (values
// next to 0, whose bins are narrower than that is exact), 64 bins tried at a
// time.
__device__ __forceinline__ int last_reaching(const Weights& wt, float T, double m) {
  const int lane = threadIdx.x & 63;
  const float x = (float)wt.xmax + __builtin_amdgcn_logf((float)m) * 0.6931472f * T;
  const int near = max(wt.top, min(bin_of(__float_as_uint(x) >> 16) - 32, kBins - 64));
  const uint64_t reach = __ballot(near + lane < kBins && wt.at(min(near + lane, kBins - 1)) >= m);
  if ((reach & 1) != 0 && reach != ~0ull) return near + __builtin_ctzll(~reach) - 1;
  int lo = wt.top;
#pragma unroll 1
  for (int step = 1024; step > 0; step >>= step == 1024 ? 6 : 4) {  // 1024, 16, 1
    const int mid = lo + step * (lane + 1);
    const uint64_t in = __ballot(mid < kBins && wt.at(min(mid, kBins - 1)) >= m);
    lo += step * (in == ~0ull ? 64 : __builtin_ctzll(~in));
  }
  return lo;
}

// A row's order by its counts, for the cuts and the draw: of one wave, or of several alike.  hold_bins(chunk, n)
// fills in a chunk's two bins per lane.
template <class Hold>
struct Order {
  const Weights& wt;
  const uint32_t* cnt;
  const double* mass;
  Hold hold_bins;
  int lane, held = -1;
  // sums up to the end of the lane's CPL chunks, and before them
  uint32_t lane_n = 0, lane_nb;
  double lane_w = 0.0, lane_wb;
  uint32_t n[2], upto_n = 0;  // of the chunk held: the lane's two bins, sums up to their end
  double one[2], w[2], upto_w = 0.0;  // of a token, of the bin

  __device__ __forceinline__ Order(const Weights& wt, const uint32_t* cnt, const double* mass, Hold hold_bins)
      : wt(wt), cnt(cnt), mass(mass), hold_bins(hold_bins), lane(threadIdx.x & 63) {
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      const uint32_t c = cnt[CPL * lane + i];
      lane_n += c;
      lane_w += c != 0 ? mass[CPL * lane + i] : 0.0;
    }
    lane_n = scan_sum(lane_n);
    lane_w = scan_sum(lane_w);
    lane_nb = before(lane_n);
    lane_wb = before(lane_w);
  }
  __device__ __forceinline__ void hold(int chunk) {
    if (chunk == held) return;
    held = chunk;
    hold_bins(chunk, n);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      one[i] = wt.at(chunk * kChunk + 2 * lane + i);
      w[i] = n[i] != 0 ? n[i] * one[i] : 0.0;
    }
    upto_n = scan_sum(n[0] + n[1]);
    upto_w = scan_sum(w[0] + w[1]);
  }
  // The first lane whose sums are not 0 and satisfy pred; the last that adds to
  // them where none does.
  __device__ __forceinline__ static int first_lane(bool some, bool hit) {
    const uint64_t any = __ballot(hit);
    return any != 0 ? __builtin_ctzll(any) : 63 - __builtin_clzll(__ballot(some) | 1);
  }
  // the first bin that is not empty and at whose end pred(count, weight) holds
  // of the sums so far; the last one that is not empty where none does
  template <class Pred>
  __device__ __forceinline__ Place find(Pred&& pred) {
    const bool some = lane_n != lane_nb;  // the scan's sums of a lane without tokens may differ from the one before's
    const int src = first_lane(some, some && pred(lane_n, lane_w));
    const uint32_t cb = lane_u(lane_nb, src);
    const double mb = lane_d(lane_wb, src);
    const int at8 = lane & (CPL - 1);
    const uint32_t cn = cnt[CPL * src + at8];
    const uint32_t c_upto = cb + scan_sum8(cn);
    const double m_upto = mb + scan_sum8(cn != 0 ? mass[CPL * src + at8] : 0.0);
    const int c8 = first_lane(lane < CPL && cn != 0, lane < CPL && cn != 0 && pred(c_upto, m_upto));
    Place at{0, 0, 0, 0.0, 0.0};
    at.c = c8 == 0 ? cb : lane_u(c_upto, c8 - 1);
    at.m = c8 == 0 ? mb : lane_d(m_upto, c8 - 1);
    const int chunk = CPL * src + c8;
    hold(chunk);
    // the first of the lane's bins, then the second
    const uint32_t n1 = at.c + upto_n, n0 = n1 - n[1];
    const double w1 = at.m + upto_w, w0 = at.m + (upto_w - w[1]);
    const bool hit0 = n[0] != 0 && pred(n0, w0), hit1 = n[1] != 0 && pred(n1, w1);
    const int l = first_lane((n[0] | n[1]) != 0, hit0 || hit1);
    const bool second = lane_u(hit0 || (!hit1 && n[1] == 0) ? 0 : 1, l) != 0;
    at.d = chunk * kChunk + 2 * l + second;
    at.n = lane_u(second ? n[1] : n[0], l);
    const double wb = before(upto_w);
    at.c = lane_u(second ? n0 : n0 - n[0], l);
    at.m += second ? lane_d(wb + w[0], l) : lane_d(wb, l);
    at.w = lane_d(second ? one[1] : one[0], l);
    return at;
  }
  __device__ __forceinline__ static double weight(Place at) { return at.m + at.n * at.w; }
  // the last token that top-k and top-p keep
  __device__ __forceinline__ Place first_cuts(const Filters& f) {
    const uint32_t all = lane_u(lane_n, 63);
    Place end{kBins, 0, all, lane_d(lane_w, 63), 0.0};  // all tokens
    if (f.k > 0 && f.k < (int64_t)all) {
      end = find([&](uint32_t c, double) { return c >= (uint32_t)f.k; });
      end.n = min(end.n, (uint32_t)f.k - end.c);
    }
    if (f.p < 1.0) {  // the tokens before which the weight is below the target
      const double target = f.p * weight(end);
      Place at = find([&](uint32_t, double m) { return m >= target; });
      const double need = ceil((target - at.m) / at.w);
      at.n = need >= 1.0 ? (need < (double)at.n ? (uint32_t)need : at.n) : 1u;
      end = earlier(end, at);
    }
    return end;
  }
  // that min-p keeps; lo: the last bin that reaches it, where it is in (0, 1]
  __device__ __forceinline__ Place min_cut(const Filters& f, int lo) {
    if (f.m > 1.0) return Place{wt.top, 1, 0, 0.0, 1.0};
    const int chunk = lo / kChunk;
    hold(chunk);
    uint32_t to = 0;  // tokens up to bin lo
#pragma unroll
    for (int i = 0; i < CPL; ++i) to += CPL * lane + i < chunk ? cnt[CPL * lane + i] : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) to += chunk * kChunk + 2 * lane + i <= lo ? n[i] : 0;
    to = lane_u(scan_sum(to), 63);
    return find([&](uint32_t c, double) { return c >= to; });
  }
  __device__ __forceinline__ static Place earlier(Place a, Place b) {
    const bool is_b = b.d < a.d || (b.d == a.d && b.n < a.n);
    return Place{is_b ? b.d : a.d, is_b ? b.n : a.n, is_b ? b.c : a.c, is_b ? b.m : a.m, is_b ? b.w : a.w};
  }
  // d: the drawn token's bin, nth: its place among the bin's tokens, S: the kept weight
  __device__ __forceinline__ void pick(Place end, double u, int& d, uint32_t& nth, double& S) {
    S = weight(end);
    const double target = u * S;
    Place at = find([&](uint32_t, double m) { return m > target; });
    at = Place{min(at.d, end.d), at.d >= end.d ? (at.d == end.d ? min(at.n, end.n) : end.n) : at.n, 0,
               at.d > end.d ? end.m : at.m, at.d > end.d ? end.w : at.w};
    const double skip = floor((target - at.m) / at.w);
    d = at.d;
    nth = skip > 0.0 ? (skip < (double)(at.n - 1) ? (uint32_t)skip : at.n - 1) : 0u;
  }
};

__global__ __launch_bounds__(FNT) void sample_filtered_kernel(
    const uint16_t* __restrict__ logits, int64_t ld, const float* __restrict__ temps,
    const float* __restrict__ uniforms, const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
    const float* __restrict__ min_p, int V, int64_t* __restrict__ out, float* __restrict__ logprob) {
  __shared__ __attribute__((aligned(16))) uint32_t hist[kWindow];
  __shared__ __attribute__((aligned(16))) double mass[kChunks];
  __shared__ double drawn_s;
  __shared__ __attribute__((aligned(16))) uint32_t cnt[kChunks];
  __shared__ uint32_t bins[kChunk];
  __shared__ uint32_t places[FNW + 1];
  __shared__ uint32_t many_value, many_n, lost, drawn_n, list_n, min_ready;
  __shared__ __attribute__((aligned(16))) uint32_t list[kList];
  __shared__ int drawn_d, reaching;
  __shared__ Place min_end;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t b = blockIdx.x;
  const uint16_t* row = logits + b * ld;
  // The row: `head` tokens up to a 16-byte boundary, `pieces` of 8, and the rest.
  const int head = min(V, (int)(-(uintptr_t)row >> 1 & 7)), pieces = (V - head) / 8;
  const uint4* body = reinterpret_cast<const uint4*>(row + head);
  // of the first 16 threads: a token outside the pieces, or -1
  const int edge = tid < 8 ? (tid < head ? tid : -1)
                   : tid < 16 && head + 8 * pieces + tid - 8 < V ? head + 8 * pieces + tid - 8 : -1;
  // fn(piece, its number, whether it is one) over the pieces past `from`, FU of a thread's loaded together
  auto walk = [&](int from, auto&& fn) {
    for (int first = from; first < pieces; first += FU * FNT) {
      uint4 x[FU];
#pragma unroll
      for (int u = 0; u < FU; ++u) x[u] = body[min(first + u * FNT + tid, pieces - 1)];
#pragma unroll
      for (int u = 0; u < FU; ++u)
        if (first + u * FNT + wave * 64 < pieces) fn(x[u], first + u * FNT + tid, first + u * FNT + tid < pieces);
    }
  };
  const float T = temps[b];
  Filters f;
  f.k = top_k != nullptr ? top_k[b] : 0;
  if (!(T > 0.f)) f.k = 1;  // greedy
  f.p = top_p != nullptr ? (double)top_p[b] : 1.0;
  f.m = min_p != nullptr ? (double)min_p[b] : 0.0;
  f.u = fmin(fmax((double)uniforms[b], 0.0), 1.0 - 0x1p-24);  // a NaN counts as 0
  for (int i = tid; i < kWindow / 4; i += FNT) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
  if (tid == 0) many_n = lost = list_n = min_ready = 0;
  if (wave == FNW - 1) {  // a value that 8 of 64 samples have
    const uint32_t v = row[(int64_t)lane * V >> 6];
    uint64_t alike = ~0ull;  // lanes with the same bits
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const uint64_t ones = __ballot(v >> e & 1);
      alike &= (v >> e & 1) ? ones : ~ones;
    }
    const uint64_t often = __ballot(__popcll(alike) >= 8);
    if (lane == 0) many_value = often != 0 ? 0u : ~0u;
    if (often != 0 && lane == __builtin_ctzll(often)) many_value = v;
  }
  __syncthreads();
  const uint32_t many = many_value;

  // the counts: low half of word h & 0x7FFF for bits h < 0x8000, high half for the others
  auto add = [&](uint32_t h) { atomicAdd(&hist[h & 0x7FFFu], (h >> 15) * 0xFFFFu + 1u); };
  uint32_t many_here = 0;  // of the wave
  if (many == ~0u) {
    walk(0, [&](const uint4& x, int, bool in) {
      if (!in) return;
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) add(w[e] & 0xFFFFu), add(w[e] >> 16);
    });
  } else {
    walk(0, [&](const uint4& x, int, bool in) {
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t h = (e & 1) ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu;
        many_here += __popcll(__ballot(in && h == many));
        if (in && h != many) add(h);
      }
    });
  }
  if (wave == 0) {
    const uint32_t h = edge >= 0 ? row[edge] : 0;
    many_here += __popcll(__ballot(edge >= 0 && h == many));
    if (edge >= 0 && h != many) add(h);
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
  // The chunks' counts.  Eight lanes take the 128 words of a positive and of a
  // negative chunk, a wave eight such pairs at a time; odd eights start 32 words
  // further, so that a read touches every bank once.
  uint32_t sum = 0;  // of all counts, drawable or not
  for (int g = wave * 8; g < kChunks / 2; g += FNW * 8) {
    const int pair = g + lane / 8;
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = ((i * 32 + (lane & 8) * 4) & 127) + (lane & 7) * 4;
      const uint4 x = *reinterpret_cast<const uint4*>(&hist[pair * kChunk + at]);
      lo += (x.x & 0xFFFFu) + (x.y & 0xFFFFu) + (x.z & 0xFFFFu) + (x.w & 0xFFFFu);
      hi += (x.x >> 16) + (x.y >> 16) + (x.z >> 16) + (x.w >> 16);
    }
    sum += lo + hi;
    lo = scan_sum8(lo), hi = scan_sum8(hi);
    if ((lane & 7) == 7) {
      const int above = kChunks / 2 - 1 - pair, below = kChunks / 2 + pair;  // the chunks of the two
      // what the words do not say: -0 counts as +0, NaN and -infinity not at all, the shared value is apart
      if (pair == 0) lo += hist[0] >> 16, hi -= hist[0] >> 16;
      if (above == 0) lo = hist[0x7F80] & 0xFFFFu, hi = 0;
      const int extra = many != ~0u && bin_of(many) < kBins ? bin_of(many) / kChunk : -1;
      cnt[above] = lo + (above == extra ? many_all : 0u);
      cnt[below] = hi + (below == extra ? many_all : 0u);
    }
  }
  sum = lane_u(scan_sum(sum), 63) + many_here - (wave == 0 ? (uint32_t)V : 0u);
  if (lane == 0 && sum != 0) atomicAdd(&lost, sum);  // modulo 2^32: 0 over the waves where every count fits
  __syncthreads();
  const bool counted = lost == 0;

  // the largest logit
  uint32_t have;  // a bit for each of the lane's chunks that is not empty
  auto first_chunk = [&]() -> int {
    have = 0;
#pragma unroll
    for (int i = 0; i < CPL; ++i) have |= (cnt[CPL * lane + i] != 0 ? 1u : 0u) << i;
    const uint64_t any = __ballot(have != 0);
    if (any == 0) return -1;
    const int src = __builtin_ctzll(any);
    return CPL * src + __builtin_ctz(lane_u(have, src));
  };
  auto first_bin = [&](int chunk, uint32_t n0, uint32_t n1) -> int {
    const int src = __builtin_ctzll(__ballot(n0 + n1 != 0));
    return chunk * kChunk + 2 * src + (lane_u(n0, src) != 0 ? 0 : 1);
  };
  Weights wt;
  wt.c = 1.4426950408889634 / (double)T;
  int d = 0;
  uint32_t nth = 0;
  double S = 0.0;
  uint4 held[FH];
  const int held_tid = tid - (FNT - FNH), held_wave = wave * 64 - (FNT - FNH);
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
    // The chunks that are not empty, dealt to the waves in turn; the last wave
    // looks for min-p's last bin meanwhile.
    const int waves = f.m > 0.0 ? FNW - 1 : FNW;
    static_assert(kChunks <= 64 * (FNW - 1), "a lane for each of a wave's chunks");
    const uint32_t upto = scan_sum((uint32_t)__popc(have)), chunks = lane_u(upto, 63);
    int mine = 0, num = 0;  // the wave's, one a lane
    for (uint32_t r = wave; wave < waves && r < chunks; r += waves, ++num) {
      const int src = __builtin_ctzll(__ballot(upto > r));
      uint32_t bits = lane_u(have, src);
      for (uint32_t skip = r + __builtin_popcount(bits) - lane_u(upto, src); skip > 0; --skip) bits &= bits - 1;
      mine = lane == num ? CPL * src + __builtin_ctz(bits) : mine;
    }
    // A chunk's values are evenly spaced: the weight of a bin 64 further is
    // this times its own.
    const double ratio = num > 0 ? wt.of(bin_value(mine * kChunk + 64) - bin_value(mine * kChunk)) : 0.0;
    for (int i = 0; i < num; ++i) {
      const int c = (int)lane_u((uint32_t)mine, i), e = c * kChunk + lane;
      const uint32_t n0 = bin_count(e), n1 = bin_count(e + 64);
      const double w0 = wt.at(e);
      const double w1 = c == c0 ? wt.at(e + 64) : w0 * lane_d(ratio, i);  // bins before the first: no finite weight
      const double all = lane_d(scan_sum((n0 != 0 ? n0 * w0 : 0.0) + (n1 != 0 ? n1 * w1 : 0.0)), 63);
      if (lane == 0) mass[c] = all;
    }
    if (wave >= waves) {
      const int lo = last_reaching(wt, T, f.m);
      if (lane == 0) reaching = lo;
    }
    __syncthreads();
    if (held_wave >= 0) {  // the row again, for the search after the draw
#pragma unroll
      for (int r = 0; r < FH; ++r)
        if (r * FNH + held_wave < pieces) held[r] = body[min(r * FNH + held_tid, pieces - 1)];
    } else {
      auto hold_bins = [&](int chunk, uint32_t (&n)[2]) {
        n[0] = bin_count(chunk * kChunk + 2 * lane), n[1] = bin_count(chunk * kChunk + 2 * lane + 1);
      };
      Order<decltype(hold_bins)> order(wt, cnt, mass, hold_bins);
      if (wave == 0) {
        Place end = order.first_cuts(f);
        if (f.m > 0.0) {  // wave 1's part, which waits for nothing; a barrier would also wait for the others' loads
          while (__hip_atomic_load(&min_ready, __ATOMIC_ACQUIRE, __HIP_MEMORY_SCOPE_WORKGROUP) == 0)
            __builtin_amdgcn_s_sleep(1);
          end = order.earlier(end, min_end);
        }
        order.pick(end, f.u, d, nth, S);
        if (lane == 0) drawn_d = d, drawn_n = nth, drawn_s = S;
      } else if (f.m > 0.0) {
        const Place at = order.min_cut(f, reaching);
        if (lane == 0) {
          min_end = at;
          __hip_atomic_store(&min_ready, 1u, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
      }
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
    auto hold_bins = [&](int chunk, uint32_t (&n)[2]) {  // the whole workgroup, the same chunk
      recount(chunk * kChunk, kChunk, bins);
      n[0] = bins[2 * lane], n[1] = bins[2 * lane + 1];
    };
    Order<decltype(hold_bins)> order(wt, cnt, mass, hold_bins);
    Place end = order.first_cuts(f);
    if (f.m > 0.0) end = order.earlier(end, order.min_cut(f, last_reaching(wt, T, f.m)));
    order.pick(end, f.u, d, nth, S);
  }

  // the nth of the bin's tokens by index
  auto done = [&](int64_t token) {
    out[b] = token;
    if (logprob != nullptr) logprob[b] = (float)((d == wt.top ? 0.0 : (bin_value(d) - wt.xmax) / (double)T) - log(S));
  };
  // a half of a word matches where it is 0 here; +0 also meets -0
  const uint32_t same = bits_of(d) * 0x10001u, mask = d == 0x7FFF ? 0x7FFF7FFFu : ~0u;
  auto any_match = [&](const uint4& x) {  // whether the least half is 0
    auto halves = [&](uint32_t w) { return __builtin_bit_cast(u16x2, (w ^ same) & mask); };
    const u16x2 least = __builtin_elementwise_min(__builtin_elementwise_min(halves(x.x), halves(x.y)),
                                                  __builtin_elementwise_min(halves(x.z), halves(x.w)));
    return least.x == 0 || least.y == 0;
  };
  auto matches = [&](const uint4& x) -> uint32_t {  // a bit for each of the eight
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t n = (w[e] ^ same) & mask;
      m |= ((n & 0xFFFFu) == 0 ? 1u << (2 * e) : 0u) | ((n >> 16) == 0 ? 2u << (2 * e) : 0u);
    }
    return m;
  };
  auto note = [&](uint32_t token) {
    const uint32_t at = atomicAdd(&list_n, 1u);
    if (at < kList) list[at] = token;
  };
  auto search = [&](const uint4& x, int i, bool in) {
    if (!in || !any_match(x)) return;
    for (uint32_t m = matches(x); m != 0; m &= m - 1) note(head + 8 * i + __builtin_ctz(m));
  };
  if (counted && held_wave >= 0) {
#pragma unroll
    for (int r = 0; r < FH; ++r)
      if (r * FNH + held_wave < pieces) search(held[r], r * FNH + held_tid, r * FNH + held_tid < pieces);
  }
  walk(counted ? FH * FNH : 0, search);
  auto equal_bits = [&](uint32_t h) { return ((h ^ same) & mask & 0xFFFFu) == 0; };
  if (edge >= 0 && equal_bits(row[edge])) note(edge);
  __syncthreads();
  const uint32_t equal = list_n;
  if (equal <= kList) {  // the nth smallest: a thread counts those before its own
    if (tid >= (int)equal) return;
    const uint32_t mine = list[tid];
    uint32_t less = 0, i = 0;
    for (; i + 4 <= equal; i += 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(&list[i]);
      less += (x.x < mine) + (x.y < mine) + (x.z < mine) + (x.w < mine);
    }
    for (; i < equal; ++i) less += list[i] < mine;
    if (less == nth) done(mine);
    return;
  }
  // many equals: a wave counts those of a consecutive part of the pieces, and
  // one looks through its part; the tokens before and after the pieces are in
  // the first wave
  const int per = ((pieces + FNW - 1) / FNW + 63) & ~63, i0 = min(pieces, wave * per), i1 = min(pieces, i0 + per);
  auto in_piece = [&](int i) { return i + lane < i1 ? matches(body[i + lane]) : 0u; };
  uint32_t here = 0;
  for (int i = i0; i < i1; i += 64) here += __popc(in_piece(i));
  here = lane_u(scan_sum(here), 63);
  const uint64_t edges = wave == 0 ? __ballot(edge >= 0 && equal_bits(row[max(edge, 0)])) : 0;
  if (lane == 0) places[wave] = here;
  if (tid == 0) places[FNW] = __popcll(edges & 0xFF);
  __syncthreads();
  if (nth < places[FNW]) {  // before the pieces
    if (wave == 0 && lane < 8 && (edges >> lane & 1) && __popcll(edges & ((1ull << lane) - 1)) == (int)nth) done(edge);
    return;
  }
  nth -= places[FNW];
  uint32_t sum_n = 0, before_n = 0;
  for (int w = 0; w < FNW; ++w) {
    if (w == wave) before_n = sum_n;
    sum_n += places[w];
  }
  if (nth >= sum_n) {  // after them
    nth -= sum_n;
    if (wave == 0 && lane >= 8 && (edges >> lane & 1) &&
        __popcll(edges & ((1ull << lane) - 1) & ~0xFFull) == (int)nth)
      done(edge);
    return;
  }
  if (nth < before_n || nth >= before_n + here) return;
  nth -= before_n;
  for (int i = i0; i < i1; i += 64) {
    uint32_t m = in_piece(i);
    const uint32_t mine = __popc(m), upto = scan_sum(mine), all = lane_u(upto, 63);
    if (nth < all) {
      if (nth < upto && nth >= upto - mine) {
        for (uint32_t skip = nth - (upto - mine); skip > 0; --skip) m &= m - 1;
        done(head + 8ll * (i + lane) + __builtin_ctz(m));
      }
      return;
    }
    nth -= all;
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
  hipLaunchKernelGGL(sample_filtered_kernel, dim3((unsigned)B), dim3(FNT), 0, (hipStream_t)stream,
                     (const uint16_t*)logits, ld, temperatures, uniforms, top_k, top_p, min_p, vocab, out, logprob);
  return check_launch("sample_filtered");
}
