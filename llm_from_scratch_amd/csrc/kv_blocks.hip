// Whole blocks of a KV pool copied to other blocks, in every plane of the pool
// at once (the layers' K and V): what forking a sequence (its partly filled
// last block) and packing a pool towards its start need.
//
// The block pairs are host data: checked here and passed by value in the
// kernel's arguments, up to kPairs of them a launch, so no index array has to
// reach the GPU first or outlive the call.
//
// Bound: HBM, each byte read and written once.  A workgroup copies 4 KiB, one
// nontemporal 16-byte load and store a thread, pieces of a block in order,
// then pairs, then planes: 257 blocks of 128 KiB in 24 planes (1.6 GB both
// ways) take 259 us, 6.2 TB/s.  Without the nontemporal hint 275 us, and then with
// 2, 4 and 8 chunks a thread 299, 306 and 413 us.  4 blocks (25 MB): 6 us.
#include "common.h"

#include <algorithm>
#include <new>

namespace lfs {
namespace {

constexpr int kPairs = 448;  // of a launch: 3.5 of the 4 KiB a launch's arguments may take
struct Pairs {
  int32_t src[kPairs], dst[kPairs];
};
constexpr int CNT = 256;  // threads: 16-byte chunks of a workgroup
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Workgroup w: piece w % pieces of pair w / pieces % n in plane w / pieces / n.
__global__ __launch_bounds__(CNT) void copy_kv_blocks_kernel(u32x4* __restrict__ pool, int64_t plane_chunks,
                                                             int64_t block_chunks, unsigned pieces, unsigned n,
                                                             Pairs pairs) {
  const unsigned r = blockIdx.x / pieces, plane = r / n, pair = r - plane * n;
  const int64_t at = (int64_t)(blockIdx.x - r * pieces) * CNT + threadIdx.x;
  if (at >= block_chunks) return;
  u32x4* base = pool + plane * plane_chunks + at;
  const u32x4 x = __builtin_nontemporal_load(base + pairs.src[pair] * block_chunks);
  __builtin_nontemporal_store(x, base + pairs.dst[pair] * block_chunks);
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
  const int64_t block_chunks = block_bytes / 16, pieces = (block_chunks + CNT - 1) / CNT;
  // a launch takes less than 2^32 threads
  const int64_t most = planes < (1 << 24) && pieces < (1 << 24) ? std::min<int64_t>(kPairs, ((1 << 24) - 1) / (planes * pieces)) : 0;
  LFS_REQUIRE(most > 0, "copy_kv_blocks: %lld planes of blocks of %lld bytes are too large", (long long)planes,
              (long long)block_bytes);
  for (int64_t i = 0; i < n; i += most) {
    const int m = (int)std::min(most, n - i);
    Pairs pairs;
    std::copy(src + i, src + i + m, pairs.src);
    std::copy(dst + i, dst + i + m, pairs.dst);
    std::fill(pairs.src + m, pairs.src + kPairs, 0);
    std::fill(pairs.dst + m, pairs.dst + kPairs, 0);
    hipLaunchKernelGGL(copy_kv_blocks_kernel, dim3((unsigned)(m * pieces * planes)), dim3(CNT), 0, (hipStream_t)stream,
                       (u32x4*)pool, num_blocks * block_chunks, block_chunks, (unsigned)pieces, (unsigned)m, pairs);
    const int rc = check_launch("copy_kv_blocks");
    if (rc) return rc;
  }
  return 0;
}
