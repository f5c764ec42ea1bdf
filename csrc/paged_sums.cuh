// Prefix sums over rows, and the cluster that they are made in: what the kernels that move pages (csrc/paged_tables.cu, csrc/paged_share.cu)
// have in common.
#pragma once
#include "kernel_setup.h"
#include "paged_kernels.h"

#include <stdint.h>

namespace penny {
namespace paged {

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}

// Sums hold at 2^31 - 1 (of terms that do so themselves: in any order the same).
constexpr uint32_t kTop = 0x7fffffffu;
__device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) { return min(a + b, kTop); }

// Exclusive sums over the block's threads, and the whole in `total`.  The first call of a kernel needs no barrier in front.
template <int N>
__device__ __forceinline__ void block_sums(uint32_t (&v)[N], uint32_t (&total)[N], uint32_t (&part)[N][32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint32_t incl = v[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl = add(incl, u);
    }
    if (lane == 31) part[i][warp] = incl;
    const uint32_t before = __shfl_up_sync(0xffffffffu, incl, 1);
    v[i] = lane > 0 ? before : 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint32_t incl = lane < warps ? part[i][lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl = add(incl, u);
    }
    total[i] = __shfl_sync(0xffffffffu, incl, 31);
    const uint32_t before = __shfl_sync(0xffffffffu, incl, max(0, warp - 1));
    if (warp > 0) v[i] = add(v[i], before);
  }
}

// The last row r of [0, rows) with at[r] <= x (at is ascending, at[0] <= x).
__device__ __forceinline__ int row_at(const int* at, int rows, int x) {
  int lo = 0, hi = rows;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// CTAs of a cluster of 1024 threads each with up to `smem` bytes: sixteen where the device has room for one such cluster, else the eight that all have.
inline int cluster_of(const void* kernel, size_t smem) {
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, int> done;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  int& n = done[{dev, kernel}];
  if (n == 0) {
    const bool may = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
    if (!may) (void)cudaGetLastError();
    n = may && max_clusters(kernel, 16, 1024, smem) > 0 ? 16 : 8;
  }
  return n;
}

}  // namespace paged
}  // namespace penny
