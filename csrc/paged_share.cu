// Rows that have pages in common: forks of a row, the pool's pages moved together, copies of pages, and which rows share what.
//
// `refs` counts the rows of every page (zero: the page is on the stack of free ones).  As in csrc/paged_tables.cu all of it is prefix
// sums, so that any order of execution gives the same tables, and ids and lengths are looked at before they are used.
//
//   k_page_fork     an empty row becomes a copy of another: its whole pages get one row more, a page that the row ends
//                   inside is copied to one from the stack (the copies are a list for k_page_copy).  Granted in order, as long as there
//                   are pages.
//   k_page_compact  with U pages in use, the i-th page in use from U on goes to the i-th free page below U; tables and counts
//                   follow, the stack holds what is left, the lowest page on top.  Sources and targets are apart, so the copies may
//                   be made in any order.  While the tables are rewritten the count of a page that moved holds where it went (-1 - id).
//   k_page_copy     pages of all pools (k and v of all layers) in a launch: 16 bytes a thread, eight under way.  Bound by memory.
//   k_page_groups   rows with the same first page are a group (a hash table in shared memory finds the lowest row of each), what they share
//                   is the least that one of them has in common with the lowest row.  A counting sort by groups gives their
//                   rows.
//
// All but the copy are latency: a few reads one after another, prefix sums, barriers.  One CTA for a small state, a cluster of up
// to sixteen for a large one: 64 forks of 62 pages each and their leaving 17 us (fork 8 of 12 pages 5), 600 pages moved together 5.5 (and 78 for 143
// copies in 48 pools, 5.6 TB/s), groups of 64 rows 7.4, of 4000 25 (one CTA sorts, the others have returned).
// Copies of small pages are held up by the index arithmetic of their vectors: 1000 of 4 KB in 48 pools 5.2 TB/s with 63 % of the issue slots used, warps waiting
// for fixed latencies more than for loads.
#include "kernel_setup.h"
#include "paged_kernels.h"
#include "paged_plan.h"
#include "paged_sums.cuh"
#include "pdl.h"

#include <climits>
#include <stdint.h>

#include <algorithm>

namespace penny {
namespace {
using namespace paged;

constexpr int kThreads = 1024, kPerThread = kPagedMaxRows / kThreads;

__device__ __forceinline__ void barrier_of(int cluster) {
  if (cluster > 1) cluster_barrier();
  else __syncthreads();
}
__device__ __forceinline__ bool in_pool(int page, int pages) { return (unsigned)page < (unsigned)pages; }
// Threads that take a row's pages together, a power of two: as many as there are for each of `rows`, at least a warp.
__device__ __forceinline__ int threads_of_row(int rows, int threads) {
  int n = 32;
  while (n < kThreads && (long long)rows * n * 2 <= threads) n *= 2;
  return n;
}

__global__ void __launch_bounds__(kThreads) k_page_fork(const PageFork a, const PageDiv div, int cluster) {
  extern __shared__ int smem[];
  int *s_first = smem, *s_row = s_first + a.rows, *s_old = s_row + a.forks, *s_new = s_old + a.forks;  // per row, then per fork
  __shared__ uint32_t s_part[1][32], s_last;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, rank = blockIdx.x;
  const int most = (int)min((long long)a.width * a.page_size, 2147483647ll);
  const int count = max(0, min(*a.free_count, a.pages));
  const int per = (a.forks + kThreads - 1) / kThreads, f0 = tid * per;
  for (int r = tid; r < a.rows; r += kThreads) s_first[r] = INT_MAX;
  if (tid == 0) s_last = 0;
  __syncthreads();
  int dst[kPerThread], old[kPerThread];
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    dst[i] = -1, old[i] = 0;
    if (i >= per || f0 + i >= a.forks) continue;
    const int s = a.source[f0 + i], t = a.target[f0 + i];
    if ((unsigned)s >= (unsigned)a.rows || (unsigned)t >= (unsigned)a.rows || s == t || a.lengths[t] > 0) continue;
    dst[i] = t, old[i] = max(0, min(a.lengths[s], most));
    atomicMin(s_first + t, f0 + i);  // (a row that is asked for twice: the first one has it)
  }
  __syncthreads();
  uint32_t need[1] = {0}, total[1];
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    if (dst[i] >= 0 && s_first[dst[i]] != f0 + i) dst[i] = -1;
    need[0] += dst[i] >= 0 && old[i] != div_page(div, old[i]) * a.page_size;
  }
  block_sums(need, total, s_part);
  uint32_t taken = need[0], last = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    if (i >= per || f0 + i >= a.forks) break;
    const bool part = dst[i] >= 0 && old[i] != div_page(div, old[i]) * a.page_size;
    if (part && ++taken > (uint32_t)count) dst[i] = -1;
    if (part && dst[i] >= 0) last = taken;
    s_row[f0 + i] = dst[i];
    s_old[f0 + i] = old[i];
    s_new[f0 + i] = part && dst[i] >= 0 ? (int)taken - 1 : -1;  // the number of its page among those from the stack
  }
  last = __reduce_max_sync(0xffffffffu, last);
  if ((tid & 31) == 0 && last > 0) atomicMax(&s_last, last);
  barrier_of(cluster);  // (all have read the lengths)
  const int threads = cluster * kThreads, me = rank * kThreads + tid, copies = (int)s_last;
  if (me == 0) *a.free_count = count - copies;
  for (int f = me; f < a.forks; f += threads) {
    const int t = s_row[f], k = s_new[f];
    a.granted[f] = t >= 0;
    if (t >= 0) a.lengths[t] = s_old[f];
    if (f >= copies) a.copy_from[f] = a.copy_to[f] = -1;
    if (k >= 0) {
      const int full = div_page(div, s_old[f]), from = a.table[a.source[f] * a.table_stride + full], to = a.free_pages[count - 1 - k];
      a.table[t * a.table_stride + full] = to;
      if (in_pool(to, a.pages)) a.refs[to] = 1;
      a.copy_from[k] = in_pool(from, a.pages) ? from : a.pages;  // (no page: no copy)
      a.copy_to[k] = in_pool(to, a.pages) ? to : a.pages;
    }
  }
  const int group = threads_of_row(a.forks, threads);
  for (int f = me / group; f < a.forks; f += threads / group) {
    if (s_row[f] < 0) continue;
    const int full = div_page(div, s_old[f]);
    const int* const from = a.table + a.source[f] * a.table_stride;
    int* const to = a.table + s_row[f] * a.table_stride;
    for (int c = me % group; c < full; c += group) {
      const int page = from[c];
      to[c] = page;
      if (in_pool(page, a.pages)) atomicAdd(a.refs + page, 1);
    }
  }
}

__global__ void __launch_bounds__(kThreads) k_page_compact(const PageCompact a, const PageDiv div, int cluster) {
  __shared__ int s_warp[2][32], s_counts[16], s_part[2];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, rank = blockIdx.x, lane = tid & 31, warp = tid >> 5;
  const int chunk = (a.pages + cluster - 1) / cluster, p0 = min(a.pages, rank * chunk), p1 = min(a.pages, p0 + chunk);
  // The block's number of pages for which each of two tests holds; the CTAs' in front of this one, and all, through s_counts.
  auto before_and_all = [&](int mine, int& before, int& all) {  // mine: one value of the CTA, in every thread
    if (cluster > 1) {
      cluster_barrier();  // (s_counts has been read)
      if (tid < cluster) {
        uint32_t to;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"((uint32_t)__cvta_generic_to_shared(s_counts + rank)), "r"(tid));
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(mine) : "memory");
      }
      cluster_barrier();
    } else {
      __syncthreads();
      if (tid == 0) s_counts[0] = mine;
      __syncthreads();
    }
    before = all = 0;
    for (int c = 0; c < cluster; ++c) {
      before += c < rank ? s_counts[c] : 0;
      all += s_counts[c];
    }
  };
  auto block_count = [&](int mine) {
    mine = __reduce_add_sync(0xffffffffu, mine);
    __syncthreads();
    if (lane == 0) s_warp[0][warp] = mine;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, s_warp[0][lane]);
  };
  int mine = 0, before, used;
  for (int p = p0 + tid; p < p1; p += kThreads) mine += a.refs[p] > 0;
  before_and_all(block_count(mine), before, used);
  int goes = 0, room = 0, goes_before, room_before, moves, rooms;
  for (int p = p0 + tid; p < p1; p += kThreads) {
    const bool in_use = a.refs[p] > 0;
    goes += in_use && p >= used;
    room += !in_use && p < used;
  }
  goes = block_count(goes);
  room = block_count(room);
  before_and_all(goes, goes_before, moves);
  before_and_all(room, room_before, rooms);
  if (tid == 0) s_part[0] = goes_before, s_part[1] = room_before;
  for (int b = p0; b < p1; b += kThreads) {
    const int p = b + tid;
    const bool in_use = p < p1 && a.refs[p] > 0, go = in_use && p >= used, free = p < p1 && !in_use && p < used;
    const uint32_t who[2] = {__ballot_sync(0xffffffffu, go), __ballot_sync(0xffffffffu, free)};
    __syncthreads();
    if (lane < 2) s_warp[lane][warp] = __popc(who[lane]);
    __syncthreads();
    int at[2];
    for (int i = 0; i < 2; ++i) {
      at[i] = s_part[i] + __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[i][lane] : 0) + __popc(who[i] & ((1u << lane) - 1));
    }
    if (go) a.copy_from[at[0]] = p;
    if (free) a.copy_to[at[1]] = p;
    __syncthreads();
    if (tid == 0) {
      for (int i = 0; i < 2; ++i)
        for (int w = 0; w < 32; ++w) s_part[i] += s_warp[i][w];
    }
  }
  barrier_of(cluster);
  const int threads = cluster * kThreads, me = rank * kThreads + tid;
  for (int i = me; i < a.pages / 2; i += threads) {
    if (i < moves) {
      const int from = __ldcg(a.copy_from + i), to = __ldcg(a.copy_to + i);
      a.refs[to] = __ldcg(a.refs + from);
      a.refs[from] = -1 - to;
    } else {
      a.copy_from[i] = a.copy_to[i] = -1;
    }
  }
  barrier_of(cluster);
  const int most = (int)min((long long)a.width * a.page_size, 2147483647ll), group = threads_of_row(a.rows, threads);
  for (int r = me / group; r < a.rows; r += threads / group) {
    int* const row = a.table + r * a.table_stride;
    const int n = pages_of(div, max(0, min(a.lengths[r], most)));
    for (int c = me % group; c < n; c += group) {
      const int page = row[c];
      if (!in_pool(page, a.pages)) continue;
      const int to = -1 - __ldcg(a.refs + page);
      if (to >= 0 && to < used) row[c] = to;
    }
  }
  barrier_of(cluster);
  for (int i = me; i < moves; i += threads) a.refs[__ldcg(a.copy_from + i)] = 0;
  for (int i = me; i < a.pages - used; i += threads) a.free_pages[i] = a.pages - 1 - i;
  if (me == 0) *a.free_count = a.pages - used;
}

// A CTA takes pieces of a page, or the same page of `group` pools where pages are small; (copy, pools, piece) in a line, the pools of a copy one
// behind the other.  (A pool of small pages, one by one, 880 GB/s, so 4000; 48 pools 5200.)
constexpr int kCopyThreads = 256, kAhead = 8, kPiece = kCopyThreads * kAhead;  // vectors of 16 bytes
__global__ void __launch_bounds__(kCopyThreads) k_page_copy(const __grid_constant__ PageCopy a, int pieces, int group) {
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, vecs = a.run_bytes / 16, total = a.outer * a.inner * vecs;  // of a page
  const long long each = (long long)((a.pools + group - 1) / group) * pieces, units = a.copies * each;
  for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int copy = (int)(unit / each), rest = (int)(unit - copy * each);
    const int from = a.from[copy], to = a.to[copy];
    if (!in_pool(from, a.pages) || !in_pool(to, a.pages)) {  // (on to this CTA's first piece of the next pair)
      unit += (each - 1 - rest) / gridDim.x * gridDim.x;
      continue;
    }
    const int set = rest / pieces, first = (rest - set * pieces) * kPiece, pool0 = set * group;
    const int count = group > 1 ? min(group, a.pools - pool0) * total : total;  // vectors of this unit's pools
    const long long src = from * a.page_bytes, dst = to * a.page_bytes;
    uint4 v[kAhead];
    auto at = [&](int u, char*& base) {  // where a vector lies in its page, -1 behind the last
      int i = first + u * kCopyThreads + tid;
      if (i >= count) return -1ll;
      int pool = pool0;
      if (group > 1) {
        pool += i / total;
        i %= total;
      }
      base = a.pool[pool];
      if (a.outer == 1 && a.inner == 1) return (long long)i * 16;
      const int run = i / vecs, o = run / a.inner;
      return o * a.outer_bytes + (run - o * a.inner) * a.inner_bytes + (long long)(i - run * vecs) * 16;
    };
    char* base = nullptr;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const long long x = at(u, base);
      if (x >= 0) v[u] = *reinterpret_cast<const uint4*>(base + src + x);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const long long x = at(u, base);
      if (x >= 0) *reinterpret_cast<uint4*>(base + dst + x) = v[u];
    }
  }
}

constexpr int kChunks = 8;  // parts of the rows that are sorted at a time, and counters of a group
__global__ void __launch_bounds__(kThreads) k_page_groups(const PageGroups a, const PageDiv div, int slots, int cluster) {
  // a hash table of first pages: (page, lowest row); later the groups' rows in every chunk
  extern __shared__ int smem[];
  int *const s_page = smem, *const s_low = s_page + slots;
  uint16_t* const s_chunk = reinterpret_cast<uint16_t*>(smem);
  int *const s_leader = smem + max(2 * slots, kChunks * a.rows / 2), *const s_least = s_leader + a.rows;
  __shared__ uint32_t s_part[2][32];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, rank = blockIdx.x, lane = tid & 31, warp = tid >> 5;
  const int most = (int)min((long long)a.width * a.page_size, 2147483647ll);
  // pages in front of the one with the row's last position
  auto whole = [&](int r) {
    const int n = max(0, min(a.lengths[r], most));
    return n > 0 ? div_page(div, n - 1) : 0;
  };
  for (int i = tid; i < slots; i += kThreads) s_page[i] = -1, s_low[i] = INT_MAX;
  __syncthreads();
  int slot[kPerThread];
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int r = i * kThreads + tid;
    slot[i] = -1;
    if (r >= a.rows || whole(r) == 0) continue;
    const int page = a.table[r * a.table_stride];
    if (page < 0) continue;
    int s = (int)(((uint32_t)page * 2654435761u) >> 7) & (slots - 1);
    for (int tries = 0; tries < slots; ++tries, s = (s + 1) & (slots - 1)) {  // (twice as many slots as rows)
      const int was = atomicCAS(s_page + s, -1, page);
      if (was == -1 || was == page) break;
    }
    atomicMin(s_low + s, r);
    slot[i] = s;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int r = i * kThreads + tid;
    if (r < a.rows) s_leader[r] = slot[i] >= 0 ? s_low[slot[i]] : r;
  }
  __syncthreads();
  // ---- pages in common with the leader, a warp to a row ----
  const int warps = cluster * (kThreads / 32);
  for (int r = rank * (kThreads / 32) + warp; r < a.rows; r += warps) {
    const int leader = s_leader[r];
    int n = whole(r);
    if (leader != r) {
      n = min(n, whole(leader));
      const int *x = a.table + r * a.table_stride, *y = a.table + leader * a.table_stride;
      for (int c0 = 0; c0 < n; c0 += 128) {
        bool same[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int c = c0 + u * 32 + lane;
          same[u] = c >= n || (x[c] == y[c] && x[c] >= 0);
        }
        int end = INT_MAX;
#pragma unroll
        for (int u = 3; u >= 0; --u) {
          const uint32_t other = __ballot_sync(0xffffffffu, !same[u]);
          if (other != 0) end = c0 + u * 32 + __ffs(other) - 1;
        }
        if (end != INT_MAX) {
          n = end;
          break;
        }
      }
    }
    if (lane == 0) a.shared[r] = n;
  }
  barrier_of(cluster);
  if (rank != 0) return;
  // ---- the least of every group, and the groups' rows, ascending ----
  for (int r = tid; r < a.rows; r += kThreads) s_least[r] = INT_MAX;
  for (int i = tid; i < kChunks * a.rows; i += kThreads) s_chunk[i] = 0;
  __syncthreads();
  for (int r = tid; r < a.rows; r += kThreads) atomicMin(s_least + s_leader[r], __ldcg(a.shared + r));
  const int chunk = (a.rows + 32 * kChunks - 1) / (32 * kChunks) * 32;  // rows of a chunk
  // a warp takes a chunk; a row's number in its group among the chunk's is kept in order[] until the groups' places are known
  if (warp < kChunks) {
    uint16_t* const fill = s_chunk + warp * a.rows;
    for (int b = warp * chunk; b < min(a.rows, (warp + 1) * chunk); b += 32) {
      const int r = b + lane;
      const bool in = r < a.rows;
      const int leader = in ? s_leader[r] : -1;
      const uint32_t peers = __match_any_sync(0xffffffffu, leader);
      const int below = __popc(peers & ((1u << lane) - 1));
      const int base = in ? fill[leader] : 0;
      __syncwarp();
      if (in && below == 0) fill[leader] = (uint16_t)(base + __popc(peers));
      __syncwarp();
      if (in) a.order[r] = base + below;  // (this thread's own from here on)
    }
  }
  __syncthreads();
  const int per = (a.rows + kThreads - 1) / kThreads, r0 = tid * per;
  uint32_t sums[2] = {0, 0}, totals[2];  // rows of the groups of this thread's leaders, and those groups
  for (int r = r0; r < min(a.rows, r0 + per); ++r) {
    if (s_leader[r] != r) continue;
    for (int c = 0; c < kChunks; ++c) sums[0] += s_chunk[c * a.rows + r];
    ++sums[1];
  }
  block_sums(sums, totals, s_part);
  for (int r = r0; r < min(a.rows, r0 + per); ++r) {
    if (s_leader[r] != r) continue;
    a.starts[sums[1]++] = (int)sums[0];
    const uint32_t begin = sums[0];
    for (int c = 0; c < kChunks; ++c) {
      const int n = s_chunk[c * a.rows + r];
      s_chunk[c * a.rows + r] = (uint16_t)sums[0];
      sums[0] += n;
    }
    s_least[r] = sums[0] - begin > 1 ? s_least[r] : 0;
  }
  for (int g = (int)totals[1] + tid; g <= a.rows; g += kThreads) a.starts[g] = a.rows;
  __syncthreads();
  // (every row's number is read before any place is written)
  int place[kPerThread];
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int r = i * kThreads + tid;
    place[i] = r < a.rows ? __ldcg(a.order + r) + s_chunk[r / chunk * a.rows + s_leader[r]] : 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int r = i * kThreads + tid;
    if (r >= a.rows) break;
    a.order[place[i]] = r;
    a.shared[r] = s_least[s_leader[r]] * a.page_size;
  }
}

template <class Kernel, typename... Args>
cudaError_t launch_cluster(Kernel kernel, size_t smem_most, size_t smem, bool big, cudaStream_t stream, Args&&... args) {
  const void* k = reinterpret_cast<const void*>(kernel);
  const cudaError_t rc = kernel_setup(k, (int)smem_most).rc;
  if (rc != cudaSuccess) return rc;
  const int cluster = big ? cluster_of(k, smem_most) : 1;
  return launch_kernel_ex(kernel, dim3(cluster), dim3(kThreads), smem, stream, true, cluster, args..., cluster);
}

}  // namespace

cudaError_t launch_page_fork(const PageFork& a, cudaStream_t stream) {
  if (a.rows < 1 || a.rows > kPagedMaxRows || a.forks < 0 || a.forks > kPagedMaxRows || a.width < 1 || a.page_size < 1 || a.pages < 1)
    return cudaErrorInvalidValue;
  if (a.forks == 0) return cudaSuccess;
  return launch_cluster(k_page_fork, (size_t)kPagedMaxRows * 16, (size_t)(a.rows + 3 * a.forks) * 4, (long long)a.forks * a.width > 2048, stream, a,
                        page_div(a.page_size));
}

cudaError_t launch_page_compact(const PageCompact& a, cudaStream_t stream) {
  if (a.rows < 1 || a.rows > kPagedMaxRows || a.width < 1 || a.page_size < 1 || a.pages < 1) return cudaErrorInvalidValue;
  return launch_cluster(k_page_compact, 0, 0, a.pages > 8192 || (long long)a.rows * a.width > 16384, stream, a, page_div(a.page_size));
}

cudaError_t launch_page_copy(const PageCopy& a, int sms, cudaStream_t stream) {
  if (a.pools < 0 || a.pools > kPageCopyPools || a.copies < 0 || a.outer < 1 || a.inner < 1 || a.run_bytes < 16 || a.run_bytes % 16 != 0)
    return cudaErrorInvalidValue;
  if (a.pools == 0 || a.copies == 0) return cudaSuccess;
  const long long total = (long long)a.outer * a.inner * (a.run_bytes / 16);
  if (total > INT_MAX - kPiece) return cudaErrorInvalidValue;
  const int pieces = (int)((total + kPiece - 1) / kPiece);
  // (several pools only where there are CTAs for more than one round: 8 copies of 4 KB in 48 pools 2.2 us one by one, eight pools at a time 4.2)
  const long long rounds = std::max<long long>(1, (long long)a.copies * a.pools / (8 * sms));
  const int group = pieces > 1 ? 1 : (int)std::min({(long long)a.pools, kPiece / total, rounds});
  if ((long long)a.pools * pieces > INT_MAX) return cudaErrorInvalidValue;
  const long long units = (long long)a.copies * ((a.pools + group - 1) / group) * pieces;
  const int ctas = (int)std::min<long long>(units, 8ll * sms);
  return launch_kernel_ex(k_page_copy, dim3((unsigned)ctas), dim3(kCopyThreads), 0, stream, true, 1, a, pieces, group);
}

cudaError_t launch_page_groups(const PageGroups& a, cudaStream_t stream) {
  if (a.rows < 1 || a.rows > kPagedMaxRows || a.width < 1 || a.page_size < 1) return cudaErrorInvalidValue;
  int slots = 64;
  while (slots < 2 * a.rows) slots *= 2;
  auto smem = [](int rows, int n) { return (size_t)(std::max(2 * n, kChunks * rows / 2) + 2 * rows) * 4; };
  static_assert((kPagedMaxRows & (kPagedMaxRows - 1)) == 0 && kPagedMaxRows < 1 << 16, "slots, and places of 16 bits");
  return launch_cluster(k_page_groups, smem(kPagedMaxRows, 2 * kPagedMaxRows), smem(a.rows, slots), a.rows > 64 || (long long)a.rows * a.width > 16384, stream, a,
                        page_div(a.page_size), slots);
}

}  // namespace penny
