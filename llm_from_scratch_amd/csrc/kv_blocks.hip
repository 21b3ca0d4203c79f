// Whole blocks of a KV pool copied to other blocks, in every plane of the pool
// at once (the layers' K and V): what forking a sequence (its partly filled
// last block) and packing a pool towards its start need.
//
// The block pairs are host data: checked here and passed by value in the
// kernel's arguments, kPairs of them a launch, so no index array has to
// reach the GPU first or outlive the call.  Bound: HBM, each byte read and
// written once.
#include "common.h"

#include <algorithm>
#include <new>

namespace lfs {
namespace {

constexpr int kPairs = 448;  // of a launch: 3.5 of the 4 KiB a launch's arguments may take
struct Pairs {
  int32_t src[kPairs], dst[kPairs];
};
constexpr int CNT = 256;          // threads
constexpr int CPT = 4;            // 16-byte chunks per thread
constexpr int kPiece = CNT * CPT; // chunks of a workgroup

// Workgroup (x, y): piece x % pieces of pair x / pieces, in planes y, y +
// gridDim.y, ...
__global__ __launch_bounds__(CNT) void copy_kv_blocks_kernel(uint4* __restrict__ pool, int64_t planes,
                                                             int64_t plane_chunks, int64_t block_chunks, int pieces,
                                                             Pairs pairs) {
  const int pair = blockIdx.x / pieces;
  const int64_t at = (int64_t)(blockIdx.x - pair * pieces) * kPiece + threadIdx.x;
  const int64_t src = pairs.src[pair] * block_chunks, dst = pairs.dst[pair] * block_chunks;
  for (int64_t p = blockIdx.y; p < planes; p += gridDim.y) {
    uint4* plane = pool + p * plane_chunks;
    uint4 x[CPT];
#pragma unroll
    for (int c = 0; c < CPT; ++c)
      if (at + c * CNT < block_chunks) x[c] = plane[src + at + c * CNT];
#pragma unroll
    for (int c = 0; c < CPT; ++c)
      if (at + c * CNT < block_chunks) plane[dst + at + c * CNT] = x[c];
  }
}

}  // namespace
}  // namespace lfs

using namespace lfs;

extern "C" int lfs_copy_kv_blocks(void* pool, int64_t planes, int64_t num_blocks, int64_t block_bytes,
                                  const int32_t* src, const int32_t* dst, int64_t n, void* stream) {
  LFS_REQUIRE(planes >= 0 && num_blocks >= 0 && block_bytes > 0 && n >= 0, "copy_kv_blocks: bad shape");
  LFS_REQUIRE(block_bytes % 16 == 0, "copy_kv_blocks: a block must be a multiple of 16 bytes (got %lld)",
              (long long)block_bytes);
  if (n == 0) return 0;
  LFS_REQUIRE(src && dst && (pool || planes == 0), "copy_kv_blocks: null pointer");
  LFS_REQUIRE((((uintptr_t)pool) & 15u) == 0, "copy_kv_blocks: the pool must be 16-byte aligned");
  LFS_REQUIRE(n <= num_blocks, "copy_kv_blocks: %lld pairs for %lld blocks", (long long)n, (long long)num_blocks);
  for (int64_t i = 0; i < n; ++i)
    LFS_REQUIRE(src[i] >= 0 && src[i] < num_blocks && dst[i] >= 0 && dst[i] < num_blocks,
                "copy_kv_blocks: pair %lld (%d to %d) is outside the pool of %lld blocks", (long long)i, src[i], dst[i],
                (long long)num_blocks);
  // the copies run in any order: a block may be written once, and not read as well
  int32_t* to = new (std::nothrow) int32_t[n];
  LFS_REQUIRE(to != nullptr, "copy_kv_blocks: out of host memory");
  std::copy(dst, dst + n, to);
  std::sort(to, to + n);
  const int32_t* twice = std::adjacent_find(to, to + n);
  const int32_t again = twice != to + n ? *twice : -1;
  int64_t both = -1;
  for (int64_t i = 0; i < n && both < 0; ++i)
    if (std::binary_search(to, to + n, src[i])) both = src[i];
  delete[] to;
  LFS_REQUIRE(again < 0, "copy_kv_blocks: block %d is a destination twice", again);
  LFS_REQUIRE(both < 0, "copy_kv_blocks: block %lld is a source and a destination", (long long)both);
  if (planes == 0) return 0;
  const int64_t block_chunks = block_bytes / 16, pieces = (block_chunks + kPiece - 1) / kPiece;
  LFS_REQUIRE(pieces < (1ll << 31) / kPairs / CNT, "copy_kv_blocks: blocks of %lld bytes are too large",
              (long long)block_bytes);
  for (int64_t i = 0; i < n; i += kPairs) {
    const int m = (int)std::min<int64_t>(kPairs, n - i);
    Pairs pairs;
    std::copy(src + i, src + i + m, pairs.src);
    std::copy(dst + i, dst + i + m, pairs.dst);
    std::fill(pairs.src + m, pairs.src + kPairs, 0);
    std::fill(pairs.dst + m, pairs.dst + kPairs, 0);
    hipLaunchKernelGGL(copy_kv_blocks_kernel, dim3((unsigned)(m * pieces), (unsigned)std::min<int64_t>(planes, 65535)),
                       dim3(CNT), 0, (hipStream_t)stream, (uint4*)pool, planes, num_blocks * block_chunks, block_chunks,
                       (int)pieces, pairs);
    const int rc = check_launch("copy_kv_blocks");
    if (rc) return rc;
  }
  return 0;
}
