// Block tables and slot maps from request lengths, on the device.
//
// Every row of a table has a length and as many pages as hold it; the other pages lie on a stack.  A call lets n[r] tokens
// come to each row (or its last -n[r] leave) and moves all that follows from it: pages from the stack to the rows and
// back, lengths, and for the tokens of all rows, one behind the other, their positions and slots.  Which page goes where is a
// matter of prefix sums over the rows, so any order of execution gives the same tables:
//   leaving tokens  the k-th released page, rows and pages ascending, of `pushed` goes to place count + pushed - 1 - k
//   coming tokens   the k-th new page comes from place count + pushed - 1 - k
// (What comes and leaves again is back in its old place.)  A row is granted its tokens if it may be that long, they end
// inside `tokens`, and the stack has pages for it and all rows before it that pass these two tests.
//
// One launch: every CTA of a cluster sums over all rows by itself (8 bytes a row, read from L2), the cluster's barrier stands
// between the last read of the lengths and their update, then the CTAs share tokens and released pages.  Latency is
// all there is to it: a few reads and prefix sums one after the other, and 12 bytes written per token.
#include "kernel_setup.h"
#include "paged_kernels.h"
#include "paged_plan.h"
#include "pdl.h"

#include <stdint.h>

namespace penny {
namespace {
using namespace paged;

constexpr int kTokensPerThread = 4;
static_assert(kPagedMaxRows <= 8 * 1024, "rows of a thread");

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

// Values of a thread's rows to shared memory.
template <int kPer>
__device__ __forceinline__ void put(int* to, int r0, int rows, const int (&v)[kPer]) {
#pragma unroll
  for (int i = 0; i < kPer; i += 4) {
    if constexpr (kPer % 4 == 0) {
      if (r0 + i < rows) *reinterpret_cast<int4*>(to + r0 + i) = make_int4(v[i], v[i + 1], v[i + 2], v[i + 3]);  // (up to three behind the last)
    } else {
      if (r0 + i < rows) to[r0 + i] = v[i];
    }
  }
}

// kPer: rows of a thread, one behind the other.
template <int kPer>
__global__ void __launch_bounds__(1024) k_page_tables(const PageTables a, const PageDiv div, int cluster) {
  extern __shared__ int smem[];
  // per row: where its tokens begin, its length (-1 - length: not granted), its first new page's number among all new
  // ones, its first released page's among all released
  const int stride = (a.rows + 3) / 4 * 4;
  int *s_off = smem, *s_old = s_off + stride, *s_new = s_old + stride, *s_gone = s_new + stride;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, rank = blockIdx.x;
  const long long most = min((long long)a.width * a.page_size, 2147483647ll), longest = min(most, (long long)a.max_len);
  const int count = max(0, min(*a.free_count, a.pages));
  const int r0 = tid * kPer;
  auto gone_of = [&](int old, int n) { return n < 0 ? pages_of(div, old) - pages_of(div, (int)max(0ll, (long long)old + n)) : 0; };
  __shared__ uint32_t s_two[2][32], s_one[1][32], s_popped;
  if (tid == 0) s_popped = 0;

  int old[kPer], n[kPer];
  uint32_t sums[2] = {0, 0}, totals[2];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const bool in = r0 + i < a.rows;
    old[i] = in ? (int)max(0ll, min((long long)a.lengths[r0 + i], most)) : 0;
    n[i] = in ? a.news[r0 + i] : 0;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    sums[0] = add(sums[0], max(0, n[i]));
    sums[1] = add(sums[1], gone_of(old[i], n[i]));
  }
  block_sums(sums, totals, s_two);
  // (more pages than the pool has: a table that holds some twice; what the stack cannot take is dropped)
  const int pushed = (int)min(totals[1], (uint32_t)(a.pages - count));
  const uint32_t pages_there = (uint32_t)(count + pushed);
  uint32_t end = sums[0], gone = sums[1], need[1] = {0}, all_need[1];
  bool granted[kPer];
  int first_token[kPer], first_gone[kPer], first_new[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    first_token[i] = (int)end;
    first_gone[i] = (int)gone;
    end = add(end, max(0, n[i]));
    gone = add(gone, gone_of(old[i], n[i]));
    granted[i] = n[i] <= 0 || (old[i] + (long long)n[i] <= longest && end <= (uint32_t)a.tokens);
    if (n[i] > 0 && granted[i]) need[0] = add(need[0], pages_of(div, old[i] + n[i]) - pages_of(div, old[i]));
  }
  block_sums(need, all_need, s_one);
  uint32_t taken = need[0], last = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    first_new[i] = (int)taken;
    if (n[i] > 0 && granted[i]) {
      const int pages = pages_of(div, old[i] + n[i]) - pages_of(div, old[i]);
      taken = add(taken, pages);
      // (once a row is refused, all behind it that need pages are: the last one that is not has the sum)
      granted[i] = pages == 0 || taken <= pages_there;
      if (granted[i] && pages > 0) last = taken;
    }
  }
  int kept[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) kept[i] = granted[i] ? old[i] : -1 - old[i];
  put<kPer>(s_off, r0, a.rows, first_token);
  put<kPer>(s_old, r0, a.rows, kept);
  put<kPer>(s_new, r0, a.rows, first_new);
  put<kPer>(s_gone, r0, a.rows, first_gone);
  last = __reduce_max_sync(0xffffffffu, last);
  if ((tid & 31) == 0 && last > 0) atomicMax(&s_popped, last);
  if (cluster > 1) cluster_barrier();
  else __syncthreads();

  // ---- the rows' own state, from here on nobody reads it ----
  if ((tid >> 5) % cluster == rank) {  // (every CTA has all rows: each writes its warps' part)
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (r0 + i >= a.rows) break;
      a.granted[r0 + i] = granted[i];
      a.offsets[r0 + i] = first_token[i];
      a.lengths[r0 + i] = granted[i] ? (int)max(0ll, (long long)old[i] + n[i]) : old[i];
    }
  }
  if (rank == 0 && tid == 0) {
    a.offsets[a.rows] = (int)totals[0];
    *a.free_count = count + pushed - (int)s_popped;
  }

  // k-th released page, rows and pages ascending
  auto released = [&](int k) {
    const int r = row_at(s_gone, a.rows, k);
    const int left = pages_of(div, (int)max(0ll, (long long)s_old[r] + a.news[r]));  // (a row that releases is granted)
    return a.table[r * a.table_stride + left + (k - s_gone[r])];
  };
  auto new_page = [&](int k) {
    const int at = count + pushed - 1 - k;
    return at < count ? a.free_pages[at] : released(k);  // pushed - 1 - (at - count) = k
  };
  const int threads = cluster * blockDim.x, me = rank * blockDim.x + tid;
  for (int k = me; k < pushed; k += threads) a.free_pages[count + pushed - 1 - k] = released(k);

  const int total = (int)min(totals[0], (uint32_t)a.tokens);
  // a token to a thread, or four where there are more than threads; their pages are read at the same time
  const int each = a.tokens <= threads ? 1 : kTokensPerThread;
  for (long long j0 = (long long)me * each; j0 < a.tokens; j0 += (long long)threads * each) {
    int row[kTokensPerThread], pos[kTokensPerThread], at[kTokensPerThread], page[kTokensPerThread];
    bool fresh[kTokensPerThread];
    int r = j0 < total ? row_at(s_off, a.rows, (int)j0) : a.rows;
#pragma unroll
    for (int i = 0; i < kTokensPerThread; ++i) {
      const int j = (int)j0 + i;
      row[i] = -1;
      pos[i] = 0;
      if (i >= each || j >= total) continue;
      while (r + 1 < a.rows && s_off[r + 1] <= j) ++r;
      const int had = s_old[r];
      if (had < 0) continue;
      row[i] = r;
      pos[i] = had + (j - s_off[r]);
      at[i] = div_page(div, pos[i]);
      page[i] = at[i] - pages_of(div, had);  // of the row's new pages; below zero: one that it had
      fresh[i] = page[i] >= 0;
    }
#pragma unroll
    for (int i = 0; i < kTokensPerThread; ++i)
      if (row[i] >= 0) page[i] = fresh[i] ? new_page(s_new[row[i]] + page[i]) : a.table[row[i] * a.table_stride + at[i]];
    long long slot[kTokensPerThread];
#pragma unroll
    for (int i = 0; i < kTokensPerThread; ++i) {
      slot[i] = -1;
      if (row[i] < 0) continue;
      const int within = pos[i] - at[i] * a.page_size;
      if (fresh[i] && within == 0) a.table[row[i] * a.table_stride + at[i]] = page[i];
      if (page[i] >= 0 && page[i] < a.pages) slot[i] = (long long)page[i] * a.page_size + within;
    }
    if (each == kTokensPerThread && j0 + kTokensPerThread <= a.tokens) {
#pragma unroll
      for (int i = 0; i < kTokensPerThread; i += 2) *reinterpret_cast<longlong2*>(a.slots + j0 + i) = make_longlong2(slot[i], slot[i + 1]);
      *reinterpret_cast<int4*>(a.positions + j0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
      for (int i = 0; i < kTokensPerThread; ++i) {
        if (i >= each || j0 + i >= a.tokens) break;
        a.slots[j0 + i] = slot[i];
        a.positions[j0 + i] = pos[i];
      }
    }
  }
}

// CTAs of a cluster for many rows or tokens: sixteen where the device has room for one such cluster, else the eight that all have.
int cluster_of(const void* kernel) {
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, int> done;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  int& n = done[{dev, kernel}];
  if (n == 0) {
    const bool may = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
    if (!may) (void)cudaGetLastError();
    n = may && max_clusters(kernel, 16, 1024, kPagedMaxRows * 4 * sizeof(int)) > 0 ? 16 : 8;
  }
  return n;
}

}  // namespace

cudaError_t launch_page_tables(const PageTables& a, cudaStream_t stream) {
  if (a.rows < 1 || a.rows > kPagedMaxRows || a.width < 1 || a.page_size < 1 || a.pages < 1 || a.tokens < 0) return cudaErrorInvalidValue;
  const size_t smem = (size_t)(a.rows + 3) / 4 * 16 * sizeof(int);
  // One CTA for a decode step; a cluster for many rows or tokens.  There and back, on the device: 64 rows of one token 5.6 us; 1000 rows
  // with 3060 tokens 9.1, in one CTA 10.2; 4000 rows with 42,209 tokens in 5342 pages 16.1, of eight CTAs instead of sixteen 3 more.
  const int threads = a.rows <= 256 && a.tokens <= 1024 ? 256 : 1024, big = a.tokens > 2048 || a.rows > 1024;
  const int per = (a.rows + threads - 1) / threads;
#define PENNY_PAGE_TABLES(N)                                                                                                          \
  do {                                                                                                                                \
    const cudaError_t rc = kernel_setup(reinterpret_cast<const void*>(k_page_tables<N>), kPagedMaxRows * 4 * (int)sizeof(int)).rc;     \
    if (rc != cudaSuccess) return rc;                                                                                                 \
    const int cluster = big ? cluster_of(reinterpret_cast<const void*>(k_page_tables<N>)) : 1;                                         \
    return launch_kernel_ex(k_page_tables<N>, dim3(cluster), dim3(threads), smem, stream, true, cluster, a, page_div(a.page_size),     \
                            cluster);                                                                                                 \
  } while (0)
  if (per == 1) PENNY_PAGE_TABLES(1);
  if (per <= 4) PENNY_PAGE_TABLES(4);
  PENNY_PAGE_TABLES(8);
#undef PENNY_PAGE_TABLES
}

}  // namespace penny
