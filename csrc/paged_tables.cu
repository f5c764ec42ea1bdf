// Block tables and slot maps from request lengths, on the device.
//
// Every row of a table has a length and as many pages as hold it; the other pages lie on a stack.  A call lets n[r] tokens
// come to each row (or its last -n[r] leave) and moves all that follows from it: pages from the stack to the rows and
// back, lengths, and for the tokens of all rows, one behind the other, their positions and slots.  Which page goes where is a
// matter of prefix sums over the rows, so any order of execution gives the same tables:
//   leaving tokens  the k-th released page, rows and pages ascending, of `pushed` goes to place count + pushed - 1 - k
//   coming tokens   the k-th new page comes from place count + pushed - 1 - k
// (What comes and leaves again is back in its old place.)  A row is granted its tokens if the table row holds them, they end
// inside `tokens`, and the stack has pages for it and all rows before it that pass these two tests.
//
// One launch: every CTA of a cluster sums over all rows by itself (8 bytes a row, read from L2), the cluster's barrier stands
// between the last read of the lengths and their update, then the CTAs share tokens and released pages.  Latency is
// all there is to it: a few reads and prefix sums one after the other, and 12 bytes written per token.
#include "kernel_setup.h"
#include "paged_kernels.h"
#include "paged_plan.h"
#include "pdl.h"

namespace penny {
namespace {
using namespace paged;

constexpr int kTokensPerThread = 4;

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Exclusive sums over the block's threads, and the whole in `total`.
template <int N>
__device__ __forceinline__ void block_sums(long long (&v)[N], long long (&total)[N]) {
  __shared__ long long part[N][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  long long own[N];
  __syncthreads();  // (part is free again)
#pragma unroll
  for (int i = 0; i < N; ++i) {
    own[i] = v[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, v[i], o);
      if (lane >= o) v[i] += u;
    }
    if (lane == 31) part[i][warp] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    long long w = lane < warps ? part[i][lane] : 0;
    const long long mine = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    total[i] = __shfl_sync(0xffffffffu, w, 31);
    v[i] += __shfl_sync(0xffffffffu, w - mine, warp) - own[i];
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

__global__ void __launch_bounds__(1024) k_page_tables(const PageTables a, const PageDiv div, int cluster) {
  extern __shared__ int smem[];
  // per row: where its tokens begin, its length (-1 - length: not granted), its first new page's number among all new
  // ones, its first released page's among all released
  int *s_off = smem, *s_old = s_off + a.rows, *s_new = s_old + a.rows, *s_gone = s_new + a.rows;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, rank = blockIdx.x;
  const long long most = min((long long)a.width * a.page_size, 2147483647ll);
  const int count = max(0, min(*a.free_count, a.pages));
  const int per = (a.rows + blockDim.x - 1) / blockDim.x, r0 = min(a.rows, tid * per), r1 = min(a.rows, r0 + per);
  auto old_of = [&](int r) { return (int)max(0ll, min((long long)a.lengths[r], most)); };
  auto gone_of = [&](int old, int n) { return n < 0 ? pages_of(div, old) - pages_of(div, (int)max(0ll, (long long)old + n)) : 0; };

  long long sums[2] = {0, 0}, totals[2];
  for (int r = r0; r < r1; ++r) {
    const int n = a.news[r], old = old_of(r);
    sums[0] += max(0, n);
    sums[1] += gone_of(old, n);
  }
  block_sums(sums, totals);
  long long end = sums[0];
  // (more pages than the pool has: a table that holds some twice; what the stack cannot take is dropped)
  const int pushed = (int)min(totals[1], (long long)(a.pages - count));
  long long gone = sums[1], need[1] = {0}, all_need[1];
  for (int r = r0; r < r1; ++r) {
    const int n = a.news[r], old = old_of(r);
    s_off[r] = (int)min(end, 2147483647ll);
    s_gone[r] = (int)min(gone, 2147483647ll);
    end += max(0, n);
    gone += gone_of(old, n);
    const bool fits = n > 0 && old + (long long)n <= most && end <= a.tokens;
    s_old[r] = fits || n <= 0 ? old : -1 - old;
    if (fits) need[0] += pages_of(div, old + n) - pages_of(div, old);
  }
  block_sums(need, all_need);
  long long taken = need[0], popped_here = 0;
  for (int r = r0; r < r1; ++r) {
    const int n = a.news[r];
    s_new[r] = (int)min(taken, 2147483647ll);
    if (n > 0 && s_old[r] >= 0) {
      const int pages = pages_of(div, s_old[r] + n) - pages_of(div, s_old[r]);
      taken += pages;
      if (pages > 0 && taken > count + pushed) s_old[r] = -1 - s_old[r];
      else popped_here += pages;
    }
  }
  long long popped[1] = {popped_here}, all_popped[1];
  block_sums(popped, all_popped);
  if (cluster > 1) cluster_barrier();
  else __syncthreads();

  // ---- the rows' own state, from here on nobody reads it ----
  if (rank == 0) {
    for (int r = r0; r < r1; ++r) {
      const int n = a.news[r], old = s_old[r] >= 0 ? s_old[r] : -1 - s_old[r];
      a.granted[r] = s_old[r] >= 0;
      a.offsets[r] = s_off[r];
      a.lengths[r] = n > 0 ? (s_old[r] >= 0 ? old + n : old) : (int)max(0ll, (long long)old + n);
    }
    if (tid == 0) {
      a.offsets[a.rows] = (int)min(totals[0], 2147483647ll);
      *a.free_count = count + pushed - (int)all_popped[0];
    }
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

  const int total = (int)min(totals[0], (long long)a.tokens);
  for (long long j0 = (long long)me * kTokensPerThread; j0 < a.tokens; j0 += (long long)threads * kTokensPerThread) {
    long long slot[kTokensPerThread];
    int pos[kTokensPerThread];
    int r = j0 < total ? row_at(s_off, a.rows, (int)j0) : a.rows, page = -1, page_at = -1;
#pragma unroll
    for (int i = 0; i < kTokensPerThread; ++i) {
      const int j = (int)j0 + i;
      slot[i] = -1;
      pos[i] = 0;
      if (j >= total) continue;
      while (r + 1 < a.rows && s_off[r + 1] <= j) {
        ++r;
        page_at = -1;
      }
      const int old = s_old[r];
      if (old < 0) continue;
      const int p = old + (j - s_off[r]), at = div_page(div, p), held = pages_of(div, old);
      if (at != page_at) {
        page_at = at;
        page = at < held ? a.table[r * a.table_stride + at] : new_page(s_new[r] + at - held);
      }
      if (at >= held && p - at * a.page_size == 0) a.table[r * a.table_stride + at] = page;
      pos[i] = p;
      if (page >= 0 && page < a.pages) slot[i] = (long long)page * a.page_size + (p - at * a.page_size);
    }
    if (j0 + kTokensPerThread <= a.tokens) {
#pragma unroll
      for (int i = 0; i < kTokensPerThread; i += 2) *reinterpret_cast<longlong2*>(a.slots + j0 + i) = make_longlong2(slot[i], slot[i + 1]);
      *reinterpret_cast<int4*>(a.positions + j0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
      for (int i = 0; i < kTokensPerThread && j0 + i < a.tokens; ++i) {
        a.slots[j0 + i] = slot[i];
        a.positions[j0 + i] = pos[i];
      }
    }
  }
}

}  // namespace

cudaError_t launch_page_tables(const PageTables& a, cudaStream_t stream) {
  if (a.rows < 1 || a.rows > kPagedMaxRows || a.width < 1 || a.page_size < 1 || a.pages < 1 || a.tokens < 0) return cudaErrorInvalidValue;
  const size_t smem = (size_t)a.rows * 4 * sizeof(int);
  const cudaError_t rc = kernel_setup(reinterpret_cast<const void*>(k_page_tables), kPagedMaxRows * 4 * (int)sizeof(int)).rc;
  if (rc != cudaSuccess) return rc;
  const int work = max(a.rows, a.tokens / kTokensPerThread);
  const int threads = work <= 256 ? 256 : 1024, cluster = a.tokens <= 4096 ? 1 : 8;
  return launch_kernel_ex(k_page_tables, dim3(cluster), dim3(threads), smem, stream, true, cluster, a, page_div(a.page_size), cluster);
}

}  // namespace penny
