// Penalties, biases and a mask of allowed tokens on a batch of logits.
//
// Row b with its history tokens[b][0 .. n), n = seq_lens[b], of which the first
// prompt_lens[b] are the prompt's; c(v) counts token v among the others, seen(v)
// says whether it is in the history at all.  In fp32, in this order:
//   x = seen(v) ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - frequency c(v) - presence [c(v) > 0]
//   x = x + the biases of v, in the order of the row's list
//   x = -infinity where the row's mask has no bit for v
// and one rounding to the logits' type.
//
// A workgroup takes CHUNK tokens of the vocabulary of one row, from where the row
// of out is 16-byte aligned.  It streams the logits through the mask, eight a
// thread and step, and meanwhile counts the history's tokens among them in LDS
// (integers: any order gives the same), whose first occurrences make a list.
// After a barrier the few listed and biased tokens are read again and written as
// the formula has them.  Counting every logit's penalties in the stream instead
// took 45 us where this took 40 on that card (256 rows of 150001, histories of 50 to
// 4096, 64 biases): nearly every wave has some token with a count.  Bound: HBM, a
// read and a write of the logits; 40-44 us on several cards, 3.7-4.0 TB/s.
#include "common.h"

namespace lfs {
namespace {

constexpr int PT = 512;           // threads
constexpr int MAX_BIAS = 1024;    // a row's list of biases lies in LDS
constexpr int HIST = 4;           // of a history's tokens each thread holds this many at a time

struct PenaltyIn {
  const int32_t* tokens;
  int64_t tokens_stride;
  int width;
  const int32_t* prompt_lens;
  const int32_t* seq_lens;
  const float* repetition;
  const float* presence;
  const float* frequency;
  const int32_t* bias_ids;
  const float* bias;
  int nbias;
  const uint32_t* allowed;
  int64_t allowed_stride;
};

template <class T>
__device__ __forceinline__ float logit_in(T x) {
  if constexpr (sizeof(T) == 2) return bf16_to_f32(x);
  else return x;
}
template <class T>
__device__ __forceinline__ T logit_out(float x) {
  if constexpr (sizeof(T) == 2) return (uint16_t)f32_to_bf16(x);
  else return x;
}

// seen: in the history; n: times past the prompt
__device__ __forceinline__ float penalised(float x, bool seen, uint32_t n, float rep, float pres, float freq) {
  if (seen) x = x > 0.f ? x / rep : x * rep;
  if (n != 0) x = x - freq * (float)n - pres;
  return x;
}

// A token's count, with two marks: in the prompt, in the list of biases.  32 bits,
// or 16 where the history is shorter than 2^14, which halves the LDS: two a word
// (128 rows of 150001: 20.6 us in 32 bits, 18.9 in 16).
template <bool WIDE>
struct Counts {
  static constexpr int PER = WIDE ? 1 : 2, BITS = WIDE ? 32 : 16;
  static constexpr uint32_t SEEN = 1u << (BITS - 1), BIASED = 1u << (BITS - 2), TIMES = BIASED - 1;
  // returns the token's count before
  static __device__ __forceinline__ uint32_t add(uint32_t* c, uint32_t at, bool prompt) {
    const int sh = WIDE ? 0 : (at & 1) * 16;
    const uint32_t old = prompt ? atomicOr(&c[at / PER], SEEN << sh) : atomicAdd(&c[at / PER], 1u << sh);
    return (old >> sh) & (SEEN | TIMES);
  }
  static __device__ __forceinline__ void mark(uint32_t* c, uint32_t at) {
    atomicOr(&c[at / PER], BIASED << (WIDE ? 0 : (at & 1) * 16));
  }
  static __device__ __forceinline__ uint32_t get(const uint32_t* c, uint32_t at) {
    return WIDE ? c[at] : (c[at / 2] >> ((at & 1) * 16)) & 0xFFFFu;
  }
};

template <class T, bool WIDE, int CHUNK>
__global__ __launch_bounds__(PT) void penalties_kernel(const T* logits, int64_t ld, T* out, int64_t ldo,
                                                       int V, PenaltyIn in) {
  using C = Counts<WIDE>;
  // a chunk's tokens from index 8 on; the first chunk's few before the first aligned one from 8 - head
  __shared__ __attribute__((aligned(16))) uint32_t count[(CHUNK + 8) / C::PER];
  __shared__ uint16_t list[CHUNK + 8];  // indexes of the history's tokens, once each
  __shared__ __attribute__((aligned(16))) int32_t ids[MAX_BIAS];
  __shared__ int listed;
  const int b = blockIdx.y, tid = threadIdx.x;
  T* orow = out + (int64_t)b * ldo;
  const T* xrow = logits + (int64_t)b * ld;
  const int head = min(V, (int)(-((uintptr_t)orow / sizeof(T)) & 7));
  const int body = head + (int)blockIdx.x * CHUNK;         // the chunk's first aligned token
  const int v0 = blockIdx.x == 0 ? 0 : body;               // and its first
  const int v1 = min(V, body + CHUNK);                     // and its end
  const int zero = body - 8;                               // token of LDS index 0
  if (v0 >= v1) return;
  // the thread's logits and mask words, the first of the history (which of it
  // counts is known later) and of the list of biases
  constexpr int NQ = 8 * sizeof(T) / 16;  // 16-byte pieces of eight logits
  constexpr int ITER = CHUNK / (PT * 8);
  const uint32_t* mask = in.allowed ? in.allowed + (int64_t)b * in.allowed_stride : nullptr;
  const int nwords = (V + 31) >> 5;
  const bool counts = in.seq_lens != nullptr;
  const int32_t* row = in.tokens + (int64_t)b * in.tokens_stride;
  int32_t h[HIST];
  auto fetch = [&](int i0, int n) {
#pragma unroll
    for (int k = 0; k < HIST; ++k) {
      const int i = i0 + k * PT + tid;
      h[k] = i < n ? row[i] : -1;
    }
  };
  if (counts) fetch(0, in.width);
  constexpr int BU = MAX_BIAS / PT;
  int id[BU];
  float by[BU];
#pragma unroll
  for (int u = 0; u < BU; ++u) {
    const int i = tid + u * PT;
    id[u] = i < in.nbias ? in.bias_ids[(int64_t)b * in.nbias + i] : -1;
    by[u] = i < in.nbias ? in.bias[(int64_t)b * in.nbias + i] : 0.f;
  }
  uint4 x[ITER][NQ];
  uint32_t ok[ITER];
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const int v = body + (k * PT + tid) * 8;
    ok[k] = 0xFFu;
    if (v + 8 > v1) break;
    __builtin_memcpy(x[k], xrow + v, sizeof(x[k]));
    if (mask != nullptr) {
      const int wi = v >> 5, sh = v & 31;
      const uint32_t w0 = mask[wi], w1 = sh > 24 && wi + 1 < nwords ? mask[wi + 1] : 0u;
      ok[k] = __builtin_amdgcn_alignbit(w1, w0, sh);
    }
  }
  const float rep = in.repetition ? in.repetition[b] : 1.f;
  const float pres = in.presence ? in.presence[b] : 0.f, freq = in.frequency ? in.frequency[b] : 0.f;
  if (tid == 0) listed = 0;
  if (counts)
    for (int i = tid * 4; i < (CHUNK + 8) / C::PER; i += PT * 4) *reinterpret_cast<uint4*>(count + i) = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int u = 0; u < BU; ++u) ids[tid + u * PT] = id[u];
  __syncthreads();
  int same[BU];  // how often the token is in the list, 0 where it was earlier
#pragma unroll
  for (int u = 0; u < BU; ++u) {
    same[u] = 0;
    if (id[u] < v0 || id[u] >= v1) continue;
    if (counts) C::mark(count, id[u] - zero);
    int n = 0, before = 0;
    for (int j = 0; j < in.nbias; j += 4) {  // (past the list: -1)
      const int4 q = *reinterpret_cast<const int4*>(ids + j);
      const int i = tid + u * PT - j;
      const int m = (q.x == id[u]) | (q.y == id[u]) << 1 | (q.z == id[u]) << 2 | (q.w == id[u]) << 3;
      n += __builtin_popcount(m);
      before |= i >= 4 ? m : i > 0 ? m & ((1 << i) - 1) : 0;
    }
    same[u] = before ? 0 : n;
  }
  if (counts) {
    const int n = max(0, min(in.seq_lens[b], in.width)), np = in.prompt_lens[b];
    for (int i0 = 0; i0 < n; i0 += HIST * PT) {
      int32_t now[HIST];
#pragma unroll
      for (int k = 0; k < HIST; ++k) now[k] = i0 + k * PT + tid < n ? h[k] : -1;
      if (i0 + HIST * PT < n) fetch(i0 + HIST * PT, n);
#pragma unroll
      for (int k = 0; k < HIST; ++k)
        if (now[k] >= v0 && now[k] < v1) {
          const int at = now[k] - zero;
          if (C::add(count, at, i0 + k * PT + tid < np) == 0) list[atomicAdd(&listed, 1)] = (uint16_t)at;
        }
    }
  }
  auto allowed = [&](int v) { return mask == nullptr || (mask[v >> 5] >> (v & 31) & 1u); };
  // tokens before the first aligned one, and past the last eight
  const int tail = body + (max(0, v1 - body) & ~7);
  for (int k = tid; k < (body - v0) + (v1 - tail); k += PT) {
    const int v = k < body - v0 ? v0 + k : tail + k - (body - v0);
    if (v < v1) orow[v] = allowed(v) ? xrow[v] : logit_out<T>(-INFINITY);
  }
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const int v = body + (k * PT + tid) * 8;
    if (v + 8 > v1) break;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      uint32_t w[4] = {x[k][i].x, x[k][i].y, x[k][i].z, x[k][i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 2) {
          const uint32_t lo = (uint32_t)__builtin_amdgcn_sbfe((int)ok[k], 2 * e, 1);
          const uint32_t hi = (uint32_t)__builtin_amdgcn_sbfe((int)ok[k], 2 * e + 1, 1);
          const uint32_t m = (lo & 0xFFFFu) | (hi & 0xFFFF0000u);
          w[e] = (w[e] & m) | (0xFF80FF80u & ~m);
        } else {
          w[e] = ok[k] >> (4 * i + e) & 1u ? w[e] : 0xFF800000u;
        }
      }
      reinterpret_cast<uint4*>(orow + v)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __syncthreads();
  // the row of out now holds the chunk's logits as they came, but where masked
  auto one = [&](int v, uint32_t c) {
    return penalised(logit_in<T>(orow[v]), (c & (C::SEEN | C::TIMES)) != 0, c & C::TIMES, rep, pres, freq);
  };
  if (counts)
    for (int i = tid; i < listed; i += PT) {
      const int at = list[i], v = at + zero;
      const uint32_t c = C::get(count, at);
      if ((c & C::BIASED) == 0 && allowed(v)) orow[v] = logit_out<T>(one(v, c));
    }
#pragma unroll
  for (int u = 0; u < BU; ++u) {
    if (same[u] == 0 || !allowed(id[u])) continue;
    float y = one(id[u], counts ? C::get(count, id[u] - zero) : 0u) + by[u];
    for (int j = tid + u * PT + 1, n = same[u]; n > 1 && j < in.nbias; ++j)
      if (ids[j] == id[u]) {
        y += in.bias[(int64_t)b * in.nbias + j];
        --n;
      }
    orow[id[u]] = logit_out<T>(y);
  }
}

template <class T, bool WIDE>
void launch_penalties(const void* x, int64_t ld, void* out, int64_t ldo, int64_t B, int V, const PenaltyIn& in,
                      hipStream_t st) {
  // Small chunks where large ones would not give every CU one: small / large, us a
  // call in a graph: rows of 32000, one 4.0 / 4.4, 16 4.7 / 5.0, 64 5.7 / 5.5; of
  // 150001, 8 5.0 / 5.3, 32 8.7 / 7.8, 128 21.1 / 18.9.
  constexpr int BIG = 8192, SMALL = 4096;
  const bool big = B * ((V + BIG - 1) / BIG) >= 256;
  const dim3 grid((unsigned)(V / (big ? BIG : SMALL) + 1), (unsigned)B);
  if (big)
    hipLaunchKernelGGL((penalties_kernel<T, WIDE, BIG>), grid, dim3(PT), 0, st, (const T*)x, ld, (T*)out, ldo, V, in);
  else
    hipLaunchKernelGGL((penalties_kernel<T, WIDE, SMALL>), grid, dim3(PT), 0, st, (const T*)x, ld, (T*)out, ldo, V, in);
}

}  // namespace
}  // namespace lfs

using namespace lfs;

extern "C" int lfs_apply_penalties(const void* logits, int64_t ld, void* out, int64_t ld_out, int32_t is_f32,
                                   const int32_t* tokens, int64_t tokens_stride, int32_t width,
                                   const int32_t* prompt_lens, const int32_t* seq_lens, const float* repetition,
                                   const float* presence, const float* frequency, const int32_t* bias_ids,
                                   const float* bias, int32_t num_biases, const int32_t* allowed,
                                   int64_t allowed_stride, int64_t B, int32_t V, void* stream) {
  LFS_REQUIRE(B >= 0 && B < 65536 && V >= 0 && V < (1 << 30) && width >= 0 && width < (1 << 30),
              "apply_penalties: bad shape");
  LFS_REQUIRE(num_biases >= 0 && num_biases <= MAX_BIAS, "apply_penalties: at most %d biases a row (got %d)", MAX_BIAS,
              num_biases);
  if (B == 0 || V == 0) return 0;
  LFS_REQUIRE(logits && out, "apply_penalties: null pointer");
  LFS_REQUIRE((B == 1 || ld_out >= V), "apply_penalties: the rows of out overlap");
  LFS_REQUIRE((seq_lens == nullptr) == (prompt_lens == nullptr) && (width == 0 || seq_lens == nullptr || tokens),
              "apply_penalties: tokens, prompt_lens and seq_lens go together");
  LFS_REQUIRE(seq_lens || !(repetition || presence || frequency), "apply_penalties: penalties need the rows' tokens");
  LFS_REQUIRE(num_biases == 0 || (bias_ids && bias), "apply_penalties: bias_ids and bias go together");
  LFS_REQUIRE(!allowed || B == 1 || allowed_stride >= (V + 31) / 32, "apply_penalties: allowed has too few words a row");
  const PenaltyIn in{tokens, tokens_stride, width, prompt_lens, seq_lens, repetition, presence, frequency, bias_ids, bias,
                     num_biases, (const uint32_t*)allowed, allowed_stride};
  LFS_REQUIRE((((uintptr_t)out | (uintptr_t)logits) & (is_f32 ? 3u : 1u)) == 0, "apply_penalties: unaligned logits");
  const bool wide = width >= 1 << 14;
  hipStream_t st = (hipStream_t)stream;
  if (is_f32 && wide) launch_penalties<float, true>(logits, ld, out, ld_out, B, V, in, st);
  else if (is_f32) launch_penalties<float, false>(logits, ld, out, ld_out, B, V, in, st);
  else if (wide) launch_penalties<uint16_t, true>(logits, ld, out, ld_out, B, V, in, st);
  else launch_penalties<uint16_t, false>(logits, ld, out, ld_out, B, V, in, st);
  return check_launch("apply_penalties");
}
