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
// One workgroup per row.  Bins are grouped into chunks of 128; a chunk's
// count and weight stay in LDS, its bins are counted again where a cut falls.
#include "common.h"

namespace lfs {
namespace {

constexpr int FNT = 1024;            // threads
constexpr int kBins = 65536;
constexpr int kChunk = 128;          // bins of a chunk: two per lane
constexpr int kChunks = kBins / kChunk;
constexpr int kWindow = 32768;       // bins counted at once

// Bin of a logit, 0 the largest value; kBins for one that is never drawn
// (-infinity, NaN).  -0 and +0 are equal.
__device__ __forceinline__ int bin_of(uint32_t h) {
  if ((h & 0x7FFFu) > 0x7F80u || h == 0xFF80u) return kBins;
  if (h == 0x8000u) h = 0;
  return (h & 0x8000u) ? (int)h : 0x7FFF - (int)h;
}
__device__ __forceinline__ double bin_value(int d) {
  return (double)bf16_to_f32(d < 0x8000 ? 0x7FFFu - d : (uint32_t)d);
}

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

__device__ __forceinline__ double shfl_d(double v, int lane) { return __shfl(v, lane, 64); }

// The first of a wave's 64 * N entries (entry N * lane + i: a count and a
// weight) that is not empty and at whose end pred(count, weight) holds of the
// sums so far, which start at c and m; the last one that is not empty where
// none does.  c and m become the sums before it.  -1: all are empty.
template <int N, class Pred>
__device__ __forceinline__ int find_entry(const uint32_t (&n)[N], const double (&w)[N], uint32_t& c, double& m,
                                          Pred&& pred) {
  const int lane = threadIdx.x & 63;
  uint32_t cs = 0;
  double ms = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) cs += n[i], ms += w[i];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t cu = __shfl_up(cs, o, 64);
    const double mu = __shfl_up(ms, o, 64);
    if (lane >= o) cs += cu, ms += mu;
  }
  uint32_t cb = __shfl_up(cs, 1, 64);
  double mb = __shfl_up(ms, 1, 64);
  if (lane == 0) cb = 0, mb = 0.0;
  cb += c, mb += m;
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
  c = __shfl(hc, src, 64);
  m = shfl_d(hm, src);
  return N * src + __shfl(hit, src, 64);
}

// A place in the order: n tokens of bin d, after all of the bins before it;
// c and m: their count and weight.
struct Place {
  int d;
  uint32_t n, c;
  double m;
};

__global__ __launch_bounds__(FNT) void sample_filtered_kernel(
    const uint16_t* __restrict__ logits, int64_t ld, const float* __restrict__ temps,
    const float* __restrict__ uniforms, const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
    const float* __restrict__ min_p, int V, int64_t* __restrict__ out, float* __restrict__ logprob) {
  __shared__ uint32_t hist[kWindow];
  __shared__ uint32_t cnt[kChunks];
  __shared__ double mass[kChunks];
  __shared__ uint32_t bins[kChunk];
  __shared__ int red[FNT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t b = blockIdx.x;
  const uint16_t* row = logits + b * ld;

  int top = kBins;
  for (int i = tid; i < V; i += FNT) top = min(top, bin_of(row[i]));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = min(top, __shfl_xor(top, o, 64));
  if (lane == 0) red[wave] = top;
  __syncthreads();
  for (int w = 0; w < FNT / 64; ++w) top = min(top, red[w]);
  if (top == kBins) {  // nothing can be drawn
    if (tid == 0) {
      out[b] = 0;
      if (logprob != nullptr) logprob[b] = -INFINITY;
    }
    return;
  }
  const float T = temps[b];
  const Weights wt{top, bin_value(top), (double)T};
  int64_t k = top_k != nullptr ? top_k[b] : 0;
  if (!(T > 0.f)) k = 1;  // greedy
  const double p = top_p != nullptr ? (double)top_p[b] : 1.0;
  const double mp = min_p != nullptr ? (double)min_p[b] : 0.0;
  const double u = fmin(fmax((double)uniforms[b], 0.0), 1.0 - 0x1p-24);  // a NaN counts as 0

  // counts and weights of the chunks
  for (int w0 = 0; w0 < kBins; w0 += kWindow) {
    __syncthreads();
    for (int i = tid; i < kWindow; i += FNT) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < V; i += FNT) {
      const int d = bin_of(row[i]) - w0;
      if (d >= 0 && d < kWindow) atomicAdd(&hist[d], 1u);
    }
    __syncthreads();
    for (int c = wave; c < kWindow / kChunk; c += FNT / 64) {
      const uint32_t n0 = hist[c * kChunk + 2 * lane], n1 = hist[c * kChunk + 2 * lane + 1];
      const int d = w0 + c * kChunk + 2 * lane;
      double m = (n0 != 0 ? n0 * wt.at(d) : 0.0) + (n1 != 0 ? n1 * wt.at(d + 1) : 0.0);
      uint32_t n = n0 + n1;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64), m += __shfl_xor(m, o, 64);
      if (lane == 0) cnt[w0 / kChunk + c] = n, mass[w0 / kChunk + c] = m;
    }
  }
  __syncthreads();
  constexpr int CPL = kChunks / 64;
  uint32_t cn[CPL];
  double cm[CPL];
#pragma unroll
  for (int i = 0; i < CPL; ++i) cn[i] = cnt[CPL * lane + i], cm[i] = mass[CPL * lane + i];

  // the bins of a chunk: counts and weights of the lane's two
  uint32_t bn[2];
  double bm[2];
  int held = -1;
  auto hold = [&](int chunk) {  // the whole workgroup, the same chunk
    if (chunk == held) return;
    held = chunk;
    __syncthreads();
    if (tid < kChunk) bins[tid] = 0;
    __syncthreads();
    for (int i = tid; i < V; i += FNT) {
      const int d = bin_of(row[i]) - chunk * kChunk;
      if (d >= 0 && d < kChunk) atomicAdd(&bins[d], 1u);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      bn[i] = bins[2 * lane + i];
      bm[i] = bn[i] != 0 ? bn[i] * wt.at(chunk * kChunk + 2 * lane + i) : 0.0;
    }
  };
  // the first bin at whose end pred holds of the count and weight so far
  auto find = [&](auto&& pred) -> Place {
    Place at{0, 0, 0, 0.0};
    const int chunk = find_entry(cn, cm, at.c, at.m, pred);
    hold(chunk);
    const int e = find_entry(bn, bm, at.c, at.m, pred);
    at.d = chunk * kChunk + e;
    at.n = __shfl(bn[0], e >> 1, 64);
    if (e & 1) at.n = __shfl(bn[1], e >> 1, 64);
    return at;
  };
  // top-k: the weight of the first k tokens
  Place end = find([&](uint32_t c, double) { return k > 0 && c >= (uint64_t)k; });
  if (k > 0 && end.c + (uint64_t)end.n > (uint64_t)k) end.n = (uint32_t)(k - end.c);
  double S = end.m + end.n * wt.at(end.d);
  // top-p: tokens before which the weight is below the target
  if (p < 1.0) {
    const double target = p * S;
    Place at = find([&](uint32_t, double m) { return m >= target; });
    const double need = ceil((target - at.m) / wt.at(at.d));
    at.n = need >= 1.0 ? (need < (double)at.n ? (uint32_t)need : at.n) : 1u;
    if (at.d < end.d || (at.d == end.d && at.n < end.n)) end = at;
  }
  // min-p: the last bin whose weight reaches it, by bisection
  if (mp > 0.0) {
    int lo = top, hi = kBins;  // at(lo) >= mp (or the first token, always kept) > at(hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (wt.at(mid) >= mp) lo = mid;
      else hi = mid;
    }
    if (lo < end.d) {  // keep the tokens up to that bin
      const int chunk = lo / kChunk;
      hold(chunk);
      uint32_t n = 0;
#pragma unroll
      for (int i = 0; i < CPL; ++i) n += CPL * lane + i < chunk ? cn[i] : 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) n += chunk * kChunk + 2 * lane + i <= lo ? bn[i] : 0;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
      end = find([&](uint32_t c, double) { return c >= n; });
    }
    if (mp > 1.0) end = Place{top, 1, 0, 0.0};
  }
  S = end.m + end.n * wt.at(end.d);
  // the draw
  const double target = u * S;
  Place at = find([&](uint32_t, double m) { return m > target; });
  if (at.d > end.d) at = end;
  if (at.d == end.d) at.n = min(at.n, end.n);
  const double w = wt.at(at.d);
  const double skip = floor((target - at.m) / w);
  uint32_t nth = skip > 0.0 ? (skip < (double)(at.n - 1) ? (uint32_t)skip : at.n - 1) : 0u;

  // the nth token of the bin by index: a wave's consecutive slice at a time
  const int per = (V + FNT / 64 - 1) / (FNT / 64), i0 = min(V, wave * per), i1 = min(V, i0 + per);
  int mine = 0;
  for (int i = i0 + lane; i < i1; i += 64) mine += bin_of(row[i]) == at.d;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mine += __shfl_xor(mine, o, 64);
  __syncthreads();
  if (lane == 0) red[wave] = mine;
  __syncthreads();
  uint32_t before = 0;
  for (int w2 = 0; w2 < wave; ++w2) before += red[w2];
  if (nth < before || nth >= before + mine) return;
  nth -= before;
  for (int i = i0; i < i1; i += 64) {
    const uint64_t hits = __ballot(i + lane < i1 && bin_of(row[min(i + lane, V - 1)]) == at.d);
    const uint32_t n = __popcll(hits);
    if (nth < n) {
      const uint64_t below = hits & ((1ull << lane) - 1);
      if ((hits >> lane & 1) && __popcll(below) == nth) {
        out[b] = i + lane;
        if (logprob != nullptr) {
          const double x = at.d == top ? 0.0 : (bin_value(at.d) - wt.xmax) / wt.T;
          logprob[b] = (float)(x - log(S));
        }
      }
      return;
    }
    nth -= n;
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
