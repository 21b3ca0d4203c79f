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
// A workgroup takes CHUNK tokens of the vocabulary of one row: it counts the
// history's tokens among them in LDS (integers: any order gives the same), then
// streams the logits past the counts.  The few biased tokens are written again
// at the end, after a barrier.  Bound: HBM, a read and a write of the logits.
#include "common.h"

namespace lfs {
namespace {

constexpr int PT = 256;           // threads
constexpr int MAX_BIAS = 1024;    // a row's list of biases lies in LDS
constexpr uint32_t SEEN = 1u << 31;  // in the prompt; the bits below count the other tokens

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

__device__ __forceinline__ float penalised(float x, uint32_t c, float rep, float pres, float freq) {
  if (c != 0) x = x > 0.f ? x / rep : x * rep;
  const uint32_t n = c & ~SEEN;
  if (n != 0) x = x - freq * (float)n - pres;
  return x;
}

template <class T, int CHUNK>
__global__ __launch_bounds__(PT) void penalties_kernel(const T* logits, int64_t ld, T* out, int64_t ldo,
                                                       int V, PenaltyIn in) {
  __shared__ __attribute__((aligned(16))) uint32_t count[CHUNK];
  __shared__ int32_t ids[MAX_BIAS];
  const int b = blockIdx.y, tid = threadIdx.x;
  const int v0 = blockIdx.x * CHUNK, nv = min(CHUNK, V - v0);
  const bool counts = in.seq_lens != nullptr;
  const float rep = in.repetition ? in.repetition[b] : 1.f;
  const float pres = in.presence ? in.presence[b] : 0.f, freq = in.frequency ? in.frequency[b] : 0.f;
  for (int i = tid; i < CHUNK; i += PT) count[i] = 0;
  for (int i = tid; i < in.nbias; i += PT) ids[i] = in.bias_ids[(int64_t)b * in.nbias + i];
  __syncthreads();
  if (counts) {
    const int n = max(0, min(in.seq_lens[b], in.width)), np = in.prompt_lens[b];
    const int32_t* row = in.tokens + (int64_t)b * in.tokens_stride;
    for (int i = tid; i < n; i += PT) {
      const uint32_t at = (uint32_t)row[i] - (uint32_t)v0;
      if (at < (uint32_t)nv) {
        if (i < np) atomicOr(&count[at], SEEN);
        else atomicAdd(&count[at], 1u);
      }
    }
  }
  __syncthreads();
  const T* x = logits + (int64_t)b * ld + v0;
  T* o = out + (int64_t)b * ldo + v0;
  const uint32_t* mask = in.allowed ? in.allowed + (int64_t)b * in.allowed_stride : nullptr;
  auto allowed = [&](int v) { return mask == nullptr || (mask[v >> 5] >> (v & 31) & 1u); };
  // the biased tokens' logits are read before anything is written: out may be logits
  constexpr int BU = MAX_BIAS / PT;
  float bx[BU];
#pragma unroll
  for (int u = 0; u < BU; ++u) {
    const int i = tid + u * PT;
    const uint32_t at = i < in.nbias ? (uint32_t)ids[i] - (uint32_t)v0 : ~0u;
    bx[u] = at < (uint32_t)nv ? logit_in<T>(x[at]) : 0.f;
  }
  __syncthreads();
  for (int i = tid; i < nv; i += PT) {
    const float y = penalised(logit_in<T>(x[i]), count[i], rep, pres, freq);
    o[i] = logit_out<T>(allowed(v0 + i) ? y : -INFINITY);
  }
  if (in.nbias == 0) return;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < BU; ++u) {
    const int i = tid + u * PT;
    if (i >= in.nbias) break;
    const int32_t id = ids[i];
    const uint32_t at = (uint32_t)id - (uint32_t)v0;
    if (at >= (uint32_t)nv || !allowed(id)) continue;
    bool first = true;
    float y = penalised(bx[u], count[at], rep, pres, freq);
    for (int j = 0; j < in.nbias; ++j)
      if (ids[j] == id) {
        first &= j >= i;
        y += in.bias[(int64_t)b * in.nbias + j];
      }
    if (first) o[at] = logit_out<T>(y);
  }
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
  LFS_REQUIRE(B >= 0 && B < 65536 && V >= 0 && V < (1 << 30) && width >= 0, "apply_penalties: bad shape");
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
  constexpr int CHUNK = 4096;
  const dim3 grid((unsigned)((V + CHUNK - 1) / CHUNK), (unsigned)B);
  if (is_f32)
    hipLaunchKernelGGL((penalties_kernel<float, CHUNK>), grid, dim3(PT), 0, (hipStream_t)stream, (const float*)logits, ld,
                       (float*)out, ld_out, V, in);
  else
    hipLaunchKernelGGL((penalties_kernel<uint16_t, CHUNK>), grid, dim3(PT), 0, (hipStream_t)stream,
                       (const uint16_t*)logits, ld, (uint16_t*)out, ld_out, V, in);
  return check_launch("apply_penalties");
}
