// Attention of one new token per row over a paged KV cache whose rows share pages: positions that a group of rows have in common are
// read once, as a product of all their query heads with the keys.
//
//   o[r, h] = sum_j softmax_j(scale q[r, h] . K_j) V_j = (sum_i e^(m_i - m) O_i) / (sum_i e^(m_i - m) l_i)
//
// with one part (m_i, l_i, O_i) or more from the shared positions of the row's group and one or more from its own.  (Where no
// row shares anything csrc/paged_attention.cu is the kernel to use.)
//
//   * Up to 128 (row, query head) pairs of a KV head are the M side of tcgen05 products: S = Q K^T with 128 positions on the N side, P to
//     tensor memory in S's place, O += P V with P as the operand in tensor memory.  Groups with more pairs give a CTA two such
//     tiles, which take turns: the exponentials of one run under the products of the other.  A row's own positions are products
//     whose other rows are empty; there the cache's stream is the bound, and the tiles of positions go to the two in turn.
//   * A thread has a query's row of S: no exchange between threads for maxima and sums.
//   * Keys and values are staged by TMA, boxes of 8 to 32 positions of a page; a warp zeroes what values of a tile lie behind its ends (stale
//     rows may hold NaN).  Pages of no multiple of 8 positions come by cp.async, 16 bytes at a time through a list of places, which
//     any page size and strides will do for.  e4m3 pages are converted on the way to fp16, which is exact, and bf16 queries meet them as fp16 times
//     a power of two (four conversions for a pair of values in place of one were the bound).
//   * All items (a KV head of a group, or of a row) lie in a line that is cut into equal shares, a CTA to an SM
//     (paged_shared_plan.h).  A warp walks the line and hands the pieces to the others; loads run ahead across pieces.  Pieces leave unnormalised
//     fp32 outputs in a workspace, a second kernel joins them.  No counters: a workspace holds nothing between calls.
//   * Weights count from a base that is the largest score of the first 64 positions; it follows, and the accumulators are scaled, when the
//     weights of 64 positions add up to more than 2^10 (fp16 weights, which stand 2^7 above it against what fp16 loses under 2^-14: 2^15), which is seldom.
//     Weights are rounded to their type by up to half a step of each, their sum is not; an output is then off by what the
//     roundings of many weights leave, about one of its own.
//
// Bound by chains of waits, not by a pipe: a tile of 128 positions of two times 128 queries takes 4200 clocks, 2050 of softmax and 1600 of products
// that wait for each other, in two streams; one of a row's own positions 2600, with a row's few queries of 128.  64 rows of 4000 shared and 300 own
// positions, 32 of 8 heads of 128, bf16, 56 us called one after another and 55 in a graph; 100 of 16000 and 500 104 and 97; 130 of nine prompts, e4m3,
// 93 and 89 (each row by itself 91); 64 of 2048 that share nothing 107 (each by itself 84).
//
// Every wait is bounded; one that ran out sets the error word that all tcgen05 kernels here share, and the CTA ends.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "gemm_sm100.cuh"
#include "gemm_sm100.h"
#include "kernel_setup.h"
#include "paged_kernels.h"
#include "paged_shared_plan.h"
#include "paged_sums.cuh"
#include "pdl.h"

namespace penny {
namespace {
using namespace paged;
using namespace sm100;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kRing = 8;  // pieces between the warp that walks the line and the others
constexpr uint32_t kErrWait = 0x5a;

template <int D>
struct Shape {
  static constexpr int kStreams = D <= 128 ? 2 : 1;          // tiles of 128 queries at a time
  static constexpr int kTile = tile_positions(D), kQueries = tile_queries(D);
  static_assert(kQueries == 128 * kStreams, "a tile of queries for each stream");
  static constexpr int kSlot = kTile * D * 2;                // bytes of a tile's keys, or values
  static constexpr int kSlots = D == 64 ? 8 : 4;             // keys and values in turn
  static constexpr int kQ = 128 * D * 2;
  static constexpr int kSmem = kStreams * kQ + kSlots * kSlot + 1024;
  static constexpr int kSoftmaxWarps = 4 * kStreams, kLoad = kSoftmaxWarps, kWalk = kLoad + 4, kEnds = kWalk + 1, kMma = kWalk + 3;
  // (the issuer, which polls, is not on the scheduler of each stream's first warp, which has the queries of a single row)
  static constexpr int kThreads = (kMma + 1) * 32;
  // registers: whole warpgroups; those of two streams' softmax take some from the others.  (128 for all
  // spilled, and what spills is read back through an L1 of 20 KB that all loads go through: 100 rows of 16000 + 500 positions 145 us, so 139.)
  static constexpr int kMoreRegs = kStreams == 2 ? 144 : 0, kFewerRegs = 112;
  static_assert(kThreads % 128 == 0 && (kStreams == 1 || (kThreads == 512 && kMoreRegs * 256 + kFewerRegs * 256 <= 65536)), "warpgroups");
  // tensor memory: S (and P) of each stream, then O
  static constexpr int kColsO = kStreams * kTile, kCols = kColsO + kStreams * D <= 256 ? 256 : 512;
  static_assert(kColsO + kStreams * D <= 512 && kSmem <= 200 << 10, "");
};

struct Params {
  PagedAttention a;
  PagedPool pool;
  PageDiv div;
  const int *order, *starts, *shared;
  int group, max_len, max_units, ctas;
  int box;                // positions of a TMA box, of which pages are whole multiples; 0: no TMA
  uint32_t page_step, pos_step, step_bytes;
  // workspace
  int* line;         // [2 rows + 1]: first unit of every element: groups, then rows; all units
  int2* place;       // [rows]: a row's group and its number in it
  float* out;        // [4][rows][heads][D]: first pieces: of shared positions, of own ones, two halves each
  float2* ml;        // [4][rows][heads]: base, sum of the weights
  float* more;       // [ctas][2][128][D]: pieces that do not begin an item
  float2* more_ml;
  uint32_t* error;
};

struct Element {
  int begin, end;     // positions; begin at the start of a box, what is in front of `low` is not seen
  int low;
  int queries, first; // (row, head) pairs of a KV head; the first row's place in order, or ~row
  int row;            // whose table it is
};
template <int D>
__device__ __forceinline__ Element element_of(const Params& p, int e) {
  Element x = {};
  const int rows = p.a.rows;
  if (e < rows) {
    const int s0 = min(max(p.starts[e], 0), rows), n = min(max(p.starts[e + 1], 0), rows) - s0;
    if (n < 2) return x;
    x.first = s0;
    x.row = p.order[s0];
    if ((unsigned)x.row >= (unsigned)rows) return x;
    x.queries = n * p.group;
    x.end = group_end(p.shared[x.row], p.max_len, p.a.window);
  } else {
    x.row = e - rows;
    x.first = ~x.row;
    x.queries = p.group;
    const Seen s = seen_of(p.a.lengths[x.row], p.max_len, p.a.window);
    x.end = s.end;
    x.low = takes_part(s, p.shared[x.row]) ? max(p.shared[x.row], 0) : s.first;
  }
  x.begin = p.box > 0 && x.low < x.end ? x.low & -p.box : x.low;
  return x;
}
template <int D>
__device__ __forceinline__ int items_of(const Params& p, const Element& x) {
  return p.pool.heads * query_tiles(x.queries, Shape<D>::kQueries);
}
template <int D>
__device__ __forceinline__ uint32_t units_of(const Params& p, const Element& x) {
  return (uint32_t)min((long long)items_of<D>(p, x) * item_units(tiles_of(x.end - x.begin, Shape<D>::kTile), pair_of(x.queries, Shape<D>::kQueries)), 0x7fffffffll);
}

// What a CTA has of an item, as the walking warp hands it on.
struct Piece {
  int tiles;       // 0: the end
  int begin, end;  // first position, and behind the item's last
  int low;         // as in Element
  int row;         // whose table it is
  int first;       // as in Element
  int head;        // KV head
  int query0, queries;
  int whole;       // it begins the item
  int stream;      // of its first tile, where tiles go to the streams in turn
  bool pair;       // both streams take every tile
};

__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
      "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
      "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem] B[smem], 16 of K.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void cp_async16(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float exp2_ftz(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack2(const __nv_bfloat16*, float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(const __half*, float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// two e4m3 values as fp16
__device__ __forceinline__ uint32_t widen(uint32_t x) {
  uint32_t r;
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, l;}" : "=r"(r) : "r"(x));
  return r;
}
// 16 bytes, or zeros without a look at them
__device__ __forceinline__ uint4 load_or_zero(const void* from, bool there) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(from), "r"((int)there)
      : "memory");
  return v;
}
// where 16-byte chunk c of row r lies in an operand of `rows` rows: blocks of 64 columns, 128 bytes a row, swizzled
__device__ __forceinline__ uint32_t chunk_at(int rows, int r, int c) {
  return (uint32_t)((c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}
// The values as the B operand of P V, K (positions) along the rows: blocks of 64 columns lie kTile rows apart, 8 rows 1024 bytes.
template <int kTile>
__device__ __forceinline__ uint64_t value_desc(uint32_t at) {
  uint64_t d = (uint64_t)((at & 0x3ffffu) >> 4);
  d |= (uint64_t)(kTile * 128 >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r, x = *reinterpret_cast<unsigned long long*>(&a), y = *reinterpret_cast<unsigned long long*>(&b);
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r, x = *reinterpret_cast<unsigned long long*>(&a), y = *reinterpret_cast<unsigned long long*>(&b);
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Waits for what tcgen05.ld has under way; the registers are the loads' from here on.
__device__ __forceinline__ void tmem_ld_done(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                 "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]),
                 "+r"(r[31])::"memory");
}
// The largest score of 32 positions of a thread's row of S, of those that are there.
__device__ __forceinline__ float largest(uint32_t s_cols, uint32_t mask) {
  float top = -INFINITY;
  uint32_t s[32];
  tmem_ld_32x32(s_cols, s);
  tmem_ld_done(s);
#pragma unroll
  for (int j = 0; j < 32; j += 2)
    top = max3(top, (mask >> j) & 1 ? __uint_as_float(s[j]) : -INFINITY, (mask >> (j + 1)) & 1 ? __uint_as_float(s[j + 1]) : -INFINITY);
  return top;
}
// 64 positions of a thread's row of S: weights exp2(score * factor - base), rounded to T, in pairs; returns their sum, unrounded.  kFull: all
// positions are there.  (The multiplication by itself and then the difference: a score that is the base's has weight one however large it is.)
template <typename T, bool kFull>
__device__ __forceinline__ float weights(uint32_t s_cols, uint32_t mask0, uint32_t mask1, float factor, float base, uint32_t (&packed)[32]) {
  const float2 by = make_float2(factor, factor), minus = make_float2(-base, -base);
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  uint32_t s[2][32];
  tmem_ld_32x32(s_cols, s[0]);
  tmem_ld_32x32(s_cols + 32, s[1]);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    tmem_ld_done(s[w]);
    const uint32_t mask = w == 0 ? mask0 : mask1;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float2 y = add2(mul2(make_float2(__uint_as_float(s[w][2 * j]), __uint_as_float(s[w][2 * j + 1])), by), minus);
      float2 p = make_float2(exp2_ftz(y.x), exp2_ftz(y.y));
      if (!kFull) {
        p.x = (mask >> (2 * j)) & 1 ? p.x : 0.f;
        p.y = (mask >> (2 * j + 1)) & 1 ? p.y : 0.f;
      }
      packed[w * 16 + j] = pack2((const T*)nullptr, p.x, p.y);
      sum[j & 1] = add2(sum[j & 1], p);
    }
  }
  return sum[0].x + sum[0].y + (sum[1].x + sum[1].y);
}
__device__ __forceinline__ uint32_t times(const __nv_bfloat16*, uint32_t both, float by) {
  return pack2((const __nv_bfloat16*)nullptr, __uint_as_float(both << 16) * by, __uint_as_float(both & 0xffff0000u) * by);
}
__device__ __forceinline__ uint32_t times(const __half*, uint32_t both, float by) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&both));
  return pack2((const __half*)nullptr, f.x * by, f.y * by);
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, P;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Bounded by the clock, as mbar_wait is, in less code (that of all roles has to stay in the instruction caches).
__device__ __forceinline__ bool wait_some(uint64_t* bar, uint32_t parity) {
  unsigned long long since = 0;
#pragma unroll 1
  for (uint32_t i = 1; !mbar_try_wait(bar, parity); ++i) {
    if ((i & 255u) != 0) continue;
    const unsigned long long now = gtime_ns();
    if (since == 0) since = now;
    if (now - since > kWaitNs) return false;
  }
  return true;
}
// Columns of a thread's row times `by`: fp32 values, or pairs of T.
template <typename T>
__device__ __forceinline__ void scale_columns(uint32_t cols, int n, float by, bool pairs) {
#pragma unroll 1
  for (int c = 0; c < n; c += 32) {
    uint32_t v[32];
    tmem_ld_32x32(cols + c, v);
    tmem_ld_done(v);
    if (pairs) {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = times((const T*)nullptr, v[j], by);
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * by);
    }
    tmem_st_32x32(cols + c, v);
  }
  tmem_st_wait();
}

// How keys and values come to shared memory.
enum Stage { STAGE_TMA, STAGE_COPY, STAGE_E4M3 };
template <int D, typename TQ, Stage kStage>
__global__ void __launch_bounds__(Shape<D>::kThreads, 1) k_shared_attention(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap k_map,
                                                                               const __grid_constant__ CUtensorMap v_map) {
  using L = Shape<D>;
  constexpr int kTile = L::kTile, kSlots = L::kSlots, kStreams = L::kStreams;
  using T = std::conditional_t<kStage == STAGE_E4M3, __half, TQ>;  // of the products
  constexpr bool kBf16 = __is_same(T, __nv_bfloat16), kTma = kStage == STAGE_TMA, kE4M3 = kStage == STAGE_E4M3;
  // The base is kShift under the largest score of the first 64 positions that have any, and of later ones whose weights add up to over kLimit.
  constexpr float kShift = kBf16 ? 0.f : 7.f, kLimit = kBf16 ? 0x1p10f : 0x1p15f;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t b_full[kSlots], b_free[kSlots], b_landed[kSlots], b_q[2], b_s[2], b_p[2], b_o[2], b_piece[kRing], b_taken[kRing];
  __shared__ Piece s_piece[kRing];
  __shared__ uint32_t s_tmem;
  __shared__ __align__(16) uint32_t s_there[kSlots][4];
  __shared__ uint32_t s_part[1][32];
  __shared__ int s_first[3];  // the element that the CTA's share begins in, how far behind the element's first unit, all units
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  unsigned char* const tiles = align_tiles(smem_raw);
  const uint32_t q_at = smem_u32(tiles), kv_at = q_at + kStreams * L::kQ;
  if (tid == 0) {
    for (int i = 0; i < kSlots; ++i) mbar_init(b_full + i, 128), mbar_init(b_free + i, 1), mbar_init(b_landed + i, 128);
    for (int i = 0; i < 2; ++i) mbar_init(b_q + i, 128), mbar_init(b_s + i, 1), mbar_init(b_p + i, 4), mbar_init(b_o + i, 1);
    for (int i = 0; i < kRing; ++i) mbar_init(b_piece + i, 1), mbar_init(b_taken + i, L::kSoftmaxWarps + 6);
    mbar_fence_init();
    s_first[0] = -1;
    if (kTma) tma_prefetch_desc(&k_map), tma_prefetch_desc(&v_map);
  }
  if (warp == L::kMma) tmem_alloc(&s_tmem, L::kCols);
  pdl_wait();
  // ---- the line ----
  const int elements = 2 * p.a.rows, per = (elements + L::kThreads - 1) / L::kThreads, e0 = min(elements, tid * per), e1 = min(elements, e0 + per);
  const int cta = blockIdx.x;
  {
    uint32_t sum[1] = {0}, total[1];
    for (int e = e0; e < e1; ++e) sum[0] = add(sum[0], units_of<D>(p, element_of<D>(p, e)));
    block_sums(sum, total, s_part);
    const bool sound = total[0] <= (uint32_t)p.max_units;  // (groups that overlap: nothing is done)
    const int units = sound ? (int)total[0] : 0, share = units > 0 ? unit_share(units, p.ctas) : 1;
    const long long begin = (long long)cta * share;
    long long at = sum[0];
    for (int e = e0; e < e1; ++e) {
      const uint32_t n = units_of<D>(p, element_of<D>(p, e));
      if (cta == 0) p.line[e] = sound ? (int)at : 0;
      if (begin < units && begin >= at && begin < at + n) s_first[0] = e, s_first[1] = (int)(begin - at);
      at += n;
    }
    if (tid == 0) s_first[2] = units;
    if (cta == 0 && tid == 0) p.line[elements] = units;
    for (int i = cta * L::kThreads + tid; i < p.a.rows; i += p.ctas * L::kThreads) {
      const int row = p.order[i];
      if ((unsigned)row >= (unsigned)p.a.rows) continue;
      const int g = row_at(p.starts, p.a.rows, i);
      p.place[row] = make_int2(g, i - p.starts[g]);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = s_tmem;
  const int units = s_first[2], share = units > 0 ? unit_share(units, p.ctas) : 1;
  bool ok = s_first[0] >= 0;
  // (by whole warps, which see one outcome)
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return ok = __all_sync(0xffffffffu, ok && wait_some(bar, parity));
  };
  int piece_no = 0;
  auto take = [&](Piece& x) {  // the next piece; false at the end
    if (!wait(b_piece + piece_no % kRing, (piece_no / kRing) & 1)) return false;
    x = s_piece[piece_no % kRing];
    __syncwarp();
    if (lane == 0) mbar_arrive(b_taken + piece_no % kRing);
    ++piece_no;
    return x.tiles > 0;
  };
  // tiles of a piece that a stream has, and the first of them
  auto tiles_of_stream = [&](const Piece& x, int t) { return x.pair || kStreams == 1 ? x.tiles : (x.tiles + 1 - (t ^ x.stream)) / 2; };

  if (!ok) {
    // (nothing for this CTA)
  } else if (warp < L::kSoftmaxWarps) {
    // ================= a stream's softmax: a thread has a query =================
    if constexpr (L::kMoreRegs > 0) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kMoreRegs > 0 ? L::kMoreRegs : 128));
    const int t = warp >> 2, lane_at = (warp & 3) * 32, me = lane_at + lane;
    const uint32_t s_cols = tmem + t * kTile + ((uint32_t)lane_at << 16), o_cols = tmem + L::kColsO + t * D + ((uint32_t)lane_at << 16);
    unsigned char* const q_tile = tiles + t * L::kQ;
    int tile0 = 0;
    struct Work {
      int begin, n, first_tile, tile_no;  // the piece's first position, tiles of this stream, its first one, their number among all of the CTA
      int lo, hi;                         // positions that the query sees
      long long to;                       // where its output goes
      float factor;
      bool there, idle, whole, pair;
    };
    // The next piece that this stream has tiles of: its queries to shared memory, which the products of the one before are done with.
    auto begin = [&](Work& y) {
      Piece x;
      while (take(x)) {
        y.tile_no = tile0;
        tile0 += x.tiles;
        y.n = tiles_of_stream(x, t);
        if (y.n == 0) continue;
        const int query = x.query0 + (x.pair ? t * 128 : 0) + me, member = query / p.group, head = x.head * p.group + query - member * p.group;
        y.there = query < x.query0 + x.queries && (x.pair || me < x.queries);
        int row = 0;
        if (y.there) {
          row = x.first < 0 ? ~x.first : p.order[x.first + member];
          y.there = (unsigned)row < (unsigned)p.a.rows;
        }
        y.factor = p.a.scale * kLog2e;
        if (kE4M3) y.factor *= p.pool.k_scale[x.head];
        const uint32_t flip = y.factor < 0 ? 0x80008000u : 0;  // (the maximum is that of the scores before the factor)
        y.factor = fabsf(y.factor);
        const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const TQ*>(p.a.q) + row * p.a.q_stride + head * p.a.q_head_stride);
        Seen seen = {0, 0};
        if (y.there) seen = seen_of(p.a.lengths[row], p.max_len, p.a.window);
        float up = 1.f;
        if constexpr (!__is_same(T, TQ)) {
          // bf16 queries as fp16, times the power of two that brings a row's largest value to [2^15, 2^16) (values under 2^-29 of that keep
          // 2^-40 of it); the factor takes it back
          float top = 0.f;
          if (y.there) {
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c) {
              const uint4 v = q[c];
              for (uint32_t w : {v.x, v.y, v.z, v.w}) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u))));
            }
          }
          const int e = max((__float_as_int(top) >> 23) & 255, 16);
          up = __int_as_float((269 - e) << 23);
          y.factor *= __int_as_float((e - 15) << 23);
        }
#pragma unroll 1
        for (int c0 = 0; c0 < D / 8; c0 += 8) {
          uint4 v[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) v[c] = y.there ? q[c0 + c] : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if constexpr (!__is_same(T, TQ)) w[j] = pack2((const T*)nullptr, __uint_as_float(w[j] << 16) * up, __uint_as_float(w[j] & 0xffff0000u) * up);
              w[j] ^= flip;
            }
            *reinterpret_cast<uint4*>(q_tile + chunk_at(128, me, c0 + c)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        fence_async_shared();
        mbar_arrive(b_q + t);
        y.lo = seen.first, y.hi = seen.end;
        y.begin = x.begin;
        y.first_tile = x.pair || kStreams == 1 ? 0 : t ^ x.stream;
        const int half = x.pair ? (x.whole ? 0 : t) : t ^ x.stream;
        y.to = x.whole ? (((x.first < 0 ? 2 : 0) + half) * (long long)p.a.rows + row) * p.a.heads + head : (cta * 2ll + half) * 128 + me;
        y.idle = !__any_sync(0xffffffffu, y.there);  // a warp without queries
        y.whole = x.whole;
        y.pair = x.pair;
        return true;
      }
      return false;
    };
    uint32_t s_parity = 0, o_parity = 0;
    Work x = {};
    float base = -INFINITY, sum = 0.f;  // base: minus infinity before there is a score
    bool first = true;
    while (true) {
      Work y;
      const bool more = ok && begin(y);  // (the next queries before this piece's output: their scores come meanwhile)
      if (!first) {
        if (!wait(b_o + t, o_parity)) break;
        o_parity ^= 1;
        tc_fence_after_sync();
        if (!x.idle) {
          float4* const to = reinterpret_cast<float4*>((x.whole ? p.out : p.more) + x.to * D);
          if (x.there) (x.whole ? p.ml : p.more_ml)[x.to] = make_float2(base, sum);
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32(o_cols + c, o);
            tmem_ld_done(o);
            if (x.there) {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                to[c / 4 + j] = make_float4(__uint_as_float(o[4 * j]), __uint_as_float(o[4 * j + 1]), __uint_as_float(o[4 * j + 2]), __uint_as_float(o[4 * j + 3]));
            }
          }
          tc_fence_before_sync();
        }
      }
      if (!more) break;
      x = y;
      first = false;
      base = -INFINITY, sum = 0.f;
      for (int i = 0; i < x.n; ++i) {
        const int tile = x.pair || kStreams == 1 ? i : 2 * i + x.first_tile, pos = x.begin + tile * kTile;
        const bool inside = __all_sync(0xffffffffu, !x.there || (pos >= x.lo && pos + kTile <= x.hi));  // every query sees all of the tile
        if (!wait(b_s + t, s_parity)) break;
        s_parity ^= 1;
        if (!x.idle) {
          tc_fence_after_sync();
          // positions of the tile that are there (and that this query sees)
          const uint32_t* const words = s_there[(x.tile_no + tile) % kSlots];
          uint32_t all = 0xffffffffu;
#pragma unroll
          for (int w = 0; w < kTile / 32; ++w) all &= words[w];
          const bool full = inside && all == 0xffffffffu;
          auto seen = [&](int w) {
            const int a = min(max(x.lo - pos - w * 32, 0), 32), b = min(max(x.hi - pos - w * 32, 0), 32);  // [a, b)
            return words[w] & (b >= 32 ? 0xffffffffu : (1u << b) - 1) & ~(a >= 32 ? 0xffffffffu : (1u << a) - 1);
          };
          // 64 positions at a time (straight code for more is more than the instruction caches hold): their weights against the base as it
          // is, in registers; where there is none yet, or their sum says that it lies too low, against one from their largest score.
#pragma unroll 1
          for (int h = 0; h < kTile / 64; ++h) {
            const uint32_t from_cols = s_cols + h * 64;
            const uint32_t mask0 = full ? 0xffffffffu : seen(2 * h), mask1 = full ? 0xffffffffu : seen(2 * h + 1);
            uint32_t packed[32];
            float of_half = 0.f;
            bool low = x.there && base == -INFINITY;
#pragma unroll 1
            for (int again = 0; again < 2; ++again) {
              if (__any_sync(0xffffffffu, low)) {
                float top = -INFINITY;
#pragma unroll 1
                for (int w = 0; w < 2; ++w) top = fmaxf(top, largest(from_cols + 32 * w, w == 0 ? mask0 : mask1));
                float by = 1.f;
                if (low && top > -INFINITY) {
                  const float next = __fsub_rn(__fmul_rn(top, x.factor), kShift);
                  by = exp2_ftz(base - next);
                  base = next;
                }
                sum *= by;
                if (__any_sync(0xffffffffu, by != 1.f)) {
                  if (h > 0) {  // the weights in front of these, which have to be there (a wait for loads is none for stores)
                    tmem_st_wait();
                    scale_columns<T>(s_cols, 32, by, true);
                  }
                  if (i > 0) scale_columns<T>(o_cols, D, by, false);
                }
              }
              const float from = base == -INFINITY ? 0.f : base;
              of_half = full ? weights<T, true>(from_cols, mask0, mask1, x.factor, from, packed)
                             : weights<T, false>(from_cols, mask0, mask1, x.factor, from, packed);
              low = of_half > kLimit;
              if (!__any_sync(0xffffffffu, low)) break;
            }
            sum += of_half;
            tmem_st_32x32(s_cols + h * 32, packed);
          }
          tmem_st_wait();
          tc_fence_before_sync();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(b_p + t);
      }
    }
  } else if (warp == L::kMma) {
    // ================= products, a step (a tile of positions of a stream) after another =================
    if constexpr (L::kMoreRegs > 0) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kFewerRegs));
    // The whole warp walks along and elects a lane for the instructions alone; what they take is the same in all lanes and known to
    // be (through a shuffle), else every operand of every one of them is fetched by itself (the eight of a tile took 1200 clocks, so 550).
    auto same = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    constexpr uint32_t kType = kBf16 ? (1u << 7) | (1u << 10) : 0;
    constexpr uint32_t kIdS = (1u << 4) | kType | ((uint32_t)(kTile >> 3) << 17) | (8u << 24);
    constexpr uint32_t kIdO = (1u << 4) | kType | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24);  // B: K along its rows
    const uint32_t cols = (uint32_t)same((int)tmem);
    const uint64_t q_desc = make_smem_desc((uint32_t)same((int)q_at)), k_desc = make_smem_desc((uint32_t)same((int)kv_at)),
                   v_desc = value_desc<kTile>((uint32_t)same((int)kv_at));
    const uint32_t q_hi = (uint32_t)(q_desc >> 32), q_lo = (uint32_t)q_desc, k_lo = (uint32_t)k_desc, v_hi = (uint32_t)(v_desc >> 32), v_lo = (uint32_t)v_desc;
    // What each stream has under way: a step whose scores are asked for and whose weights are not yet multiplied.  Whatever is ready goes
    // next, so that neither stream waits for the other.
    struct Step {
      int value;  // slot number of the values
      bool on, first, last, alone;
    } step[2] = {};
    int done[2] = {-1, -1};           // the values that each has last multiplied
    uint32_t q_no = 0, p_no = 0;      // a bit for each stream's parity
    auto ready = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_test(bar, parity)); };
    auto full = [&](int number) { return ready(b_full + number % kSlots, (number / kSlots) & 1); };
    int tile0 = 0, tiles_here = 0, pair = 0, stream0 = 0, i = 0, end = 0;  // the piece at work: steps done, and all of them
    bool more = true;
    uint32_t idle = 0;
    unsigned long long since = 0;
    // S = Q K^T of the next step, if its stream is free and its operands are there
    auto scores = [&]() {
      if (i >= end) return false;
      const int tile = pair ? i >> 1 : i, t = pair ? i & 1 : kStreams == 1 ? 0 : (stream0 + i) & 1;
      const int nth = pair || kStreams == 1 ? tile : i >> 1;
      const int n = pair || kStreams == 1 ? tiles_here : (tiles_here + 1 - (t ^ stream0)) / 2;
      const int number = 2 * (tile0 + tile), slot = number % kSlots;
      if ((t == 0 ? step[0].on : step[1].on) || (nth == 0 && !ready(b_q + t, (q_no >> t) & 1)) || !full(number)) return false;
      tc_fence_after_sync();
      const bool frees = !pair || t == 1;
      const uint32_t d = cols + t * kTile, q = q_lo + t * (L::kQ >> 4), k0 = k_lo + slot * (L::kSlot >> 4);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_bf16(d, make_desc(q_hi, q + ((k >> 2) * 128 * 128 + (k & 3) * 32 >> 4)), make_desc(q_hi, k0 + ((k >> 2) * kTile * 128 + (k & 3) * 32 >> 4)),
                    kIdS, k > 0);
        umma_commit(b_s + t);
        if (frees) umma_commit(b_free + slot);
      }
      __syncwarp();
      if (nth == 0) q_no ^= 1u << t;
      const Step x = {number + 1, true, nth == 0, nth + 1 == n, !pair};
      if (t == 0) step[0] = x;
      else step[1] = x;
      ++i;
      return true;
    };
    while (ok && (more || i < end || step[0].on || step[1].on)) {
      bool moved = false;
#pragma unroll 1
      for (int t = 0; t < kStreams; ++t) {  // O += P V, and the scores that most often waited for that
        const Step x = t == 0 ? step[0] : step[1];
        if (x.on && ready(b_p + t, (p_no >> t) & 1) && full(x.value)) {
          tc_fence_after_sync();
          const int slot = x.value % kSlots;
          const bool frees = x.alone || (t == 0 ? done[1] : done[0]) >= x.value;  // (the second of two)
          const uint32_t d = cols + L::kColsO + t * D, a = cols + t * kTile, v = v_lo + slot * (L::kSlot >> 4);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k) umma_ts(d, a + k * 8, make_desc(v_hi, v + (k * 16 * 128 >> 4)), kIdO, !x.first || k > 0);
            if (frees) umma_commit(b_free + slot);
            if (x.last) umma_commit(b_o + t);
          }
          __syncwarp();
          p_no ^= 1u << t;
          if (t == 0) step[0].on = false, done[0] = x.value;
          else step[1].on = false, done[1] = x.value;
          moved = true;
        }
        moved |= scores();
      }
      if (i == end && more && ready(b_piece + piece_no % kRing, (piece_no / kRing) & 1)) {
        tile0 += tiles_here;
        Piece x;
        more = take(x);
        tiles_here = same(x.tiles), pair = same(x.pair), stream0 = same(x.stream);
        i = 0;
        end = pair ? 2 * tiles_here : tiles_here;
        moved = true;
      }
      if (moved) {
        idle = 0;
        continue;
      }
      __nanosleep(20);  // (leaves the scheduler to the softmax)
      if ((++idle & 1023u) == 0) {  // (bounded, as every wait is)
        const unsigned long long now = (unsigned long long)__shfl_sync(0xffffffffu, gtime_ns(), 0);
        if (idle == 1024) since = now;
        else if (now - since > kWaitNs) ok = false;
      }
    }
  } else if (warp < L::kWalk) {
    // ================= keys and values to shared memory =================
    if constexpr (L::kMoreRegs > 0) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kFewerRegs));
    const int me = tid - L::kLoad * 32;
    // A warp has a quarter of a tile's positions, of which it finds the places by itself, a lane each; its lanes then take the chunks of 16 bytes
    // of a position one behind the other.
    constexpr int kRows = kTile / 4, kSize = kE4M3 ? 1 : 2, kChunks = D * kSize / 16, kPer = kRows * kChunks / 32, kStep = 32 / kChunks;
    static_assert(kChunks <= 32, "a position to a pass at least");
    const int row0 = (me >> 5) * kRows, c = lane % kChunks, r0 = lane / kChunks;
    int number = 0, told = 0;  // slots begun, and handed on
    auto tell = [&](int upto) {
      fence_async_shared();
      for (; told < upto; ++told) mbar_arrive(b_full + told % kSlots);
    };
    auto room = [&]() {  // for slot `number`
      if (number < kSlots) return ok;
      uint64_t* const bar = b_free + number % kSlots;
      const uint32_t parity = ((number / kSlots) & 1) ^ 1;
      if (kStage == STAGE_COPY && !mbar_try_wait(bar, parity)) {
        cp_async_wait<0>();  // (whoever frees it may be waiting for what is under way)
        tell(number);
      }
      return wait(bar, parity);
    };
    Piece x;
    x.tiles = 0;
    int tile_no = -1, tile = -1, at0 = 0, now = -1, id = -1;  // now, id: the page of this lane's position in this tile and in the next
    const char *k_src = nullptr, *v_src = nullptr;
    uint32_t place = kNoStep;
    // The next tile: where this lane's position lies, and which of the warp's are there; false at the end.
    auto advance = [&]() {
      auto page = [&](int pos) { return lane < kRows && pos < x.end ? p.a.table[x.row * p.a.table_stride + div_page(p.div, pos)] : -1; };
      if (++tile >= x.tiles) {
        if (!take(x)) return false;
        tile = 0;
        at0 = x.begin - kTile;
        id = page(x.begin + row0 + lane);
        k_src = reinterpret_cast<const char*>(p.pool.k) + x.head * p.pool.head_stride * kSize + c * 16;
        v_src = reinterpret_cast<const char*>(p.pool.v) + x.head * p.pool.head_stride * kSize + c * 16;
      }
      ++tile_no;
      at0 += kTile;
      now = id;
      const int pos = at0 + row0 + lane;
      place = lane < kRows && pos >= x.low ? step_of(now, p.pool.pages, pos, p.div, p.page_step, p.pos_step) : kNoStep;
      const uint32_t there = __ballot_sync(0xffffffffu, place != kNoStep);
      if (lane == 0) {
        if constexpr (kRows == 32) s_there[tile_no % kSlots][me >> 5] = there;
        else reinterpret_cast<uint16_t*>(s_there[tile_no % kSlots])[me >> 5] = (uint16_t)there;
      }
      if (kE4M3 && place != kNoStep) {  // (to L2: the loads, for which there are registers a tile later, come from there)
        const long long by = (long long)place * p.step_bytes + x.head * p.pool.head_stride;
#pragma unroll
        for (int i = 0; i < D; i += 128) {
          asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(p.pool.k) + by + i));
          asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(p.pool.v) + by + i));
        }
      }
      id = tile + 1 < x.tiles ? page(pos + kTile) : -1;
      return ok;
    };
    if constexpr (kTma) {
      while (advance()) {
        // boxes of positions that are seen: each warp asks for its own (a page that is none is out of the tensor, which gives zeros)
        const int from = max(x.low - at0, 0), to = min(x.end - at0, kTile);
        const int box0 = max(from - row0, 0) & -p.box, box1 = min(to - row0, kRows);
        const bool part = from > 0 || to < kTile;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!room()) continue;
          // (of a tile that is not whole the values behind its ends are zeroed by another warp, which hands it on)
          uint64_t* const bar = (part && h == 1 ? b_landed : b_full) + number % kSlots;
          unsigned char* const at = tiles + kStreams * L::kQ + (number % kSlots) * L::kSlot + row0 * 128;
          if (lane == 0 && box1 > box0) mbar_expect_tx(bar, ((box1 - box0 + p.box - 1) & -p.box) * D * 2);
          else mbar_arrive(bar);
          for (int b = box0; b < box1; b += p.box) {
            const int page = __shfl_sync(0xffffffffu, now, b), y = at0 + row0 + b, in = y - div_page(p.div, y) * p.pool.page_size;
            const int z = (unsigned)page < (unsigned)p.pool.pages ? page : p.pool.pages, head = __shfl_sync(0xffffffffu, x.head, 0);
            if (elect_one()) {
#pragma unroll
              for (int c = 0; c < D / 64; ++c) tma_load_4d(at + c * kTile * 128 + b * 128, h == 0 ? &k_map : &v_map, bar, c * 64, in, head, z);
            }
            __syncwarp();
          }
          told = ++number;
        }
      }
    } else if constexpr (kE4M3) {
      // A tile's keys and values lie in registers while they are on their way: those of the next one are asked for where this one's have
      // been converted and stored.
      uint4 v[2][kPer];
      auto load = [&](uint4 (&to)[kPer], const char* src) {
        // (all places before the first load, and no branch around a load: with either between them they went one by one, 200 clocks each)
        uint32_t at[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) at[i] = __shfl_sync(0xffffffffu, place, i * kStep + r0);
#pragma unroll
        for (int i = 0; i < kPer; ++i) to[i] = load_or_zero(src + (unsigned long long)(at[i] != kNoStep ? at[i] : 0) * p.step_bytes, at[i] != kNoStep);
      };
      auto store = [&](const uint4 (&from)[kPer]) {
        if (!room()) return;
        unsigned char* const to = tiles + kStreams * L::kQ + (number % kSlots) * L::kSlot;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const uint32_t w[4] = {from[i].x, from[i].y, from[i].z, from[i].w};
          uint32_t y[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) y[2 * j] = widen(w[j]), y[2 * j + 1] = widen(w[j] >> 16);
          const int r = row0 + i * kStep + r0;
          *reinterpret_cast<uint4*>(to + chunk_at(kTile, r, 2 * c)) = make_uint4(y[0], y[1], y[2], y[3]);
          *reinterpret_cast<uint4*>(to + chunk_at(kTile, r, 2 * c + 1)) = make_uint4(y[4], y[5], y[6], y[7]);
        }
        ++number;
        tell(number);
      };
      bool some = advance();
      if (some) load(v[0], k_src), load(v[1], v_src);
      while (some) {
        const bool more = advance();
        store(v[0]);
        if (more) load(v[0], k_src);
        store(v[1]);
        if (more) load(v[1], v_src);
        some = more;
      }
    } else {
      while (advance()) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!room()) break;
          const uint32_t to = kv_at + (number % kSlots) * L::kSlot;
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const uint32_t at = __shfl_sync(0xffffffffu, place, i * kStep + r0);
            const bool there = at != kNoStep;
            cp_async16(to + chunk_at(kTile, row0 + i * kStep + r0, c), (h == 0 ? k_src : v_src) + (there ? (unsigned long long)at * p.step_bytes : 0), there);
          }
          cp_async_commit();
          ++number;
          if (number >= kSlots - 1) {
            cp_async_wait<kSlots - 2>();
            tell(max(told, number - (kSlots - 2)));
          }
        }
      }
      cp_async_wait<0>();
      if (ok) tell(number);
    }
  } else if (warp == L::kEnds) {
    // ================= values of tiles that are not whole: zeros behind their ends =================
    if constexpr (L::kMoreRegs > 0) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kFewerRegs));
    uint32_t landed = 0;  // a bit for each slot's parity
    int tile_no = 0;
    Piece x;
    while (take(x)) {
      if constexpr (kTma) {
        for (int tile = 0; tile < x.tiles && ok; ++tile) {
          const int at0 = x.begin + tile * kTile, from = max(x.low - at0, 0), to = min(x.end - at0, kTile);
          if (from == 0 && to == kTile) continue;
          const int slot = (2 * (tile_no + tile) + 1) % kSlots;
          if (!wait(b_landed + slot, (landed >> slot) & 1)) break;
          landed ^= 1u << slot;
          unsigned char* const values = tiles + kStreams * L::kQ + slot * L::kSlot;
          for (int i = lane; i < kTile * (D / 8); i += 32) {
            const int r = i / (D / 8);
            if (r < from || r >= to) *reinterpret_cast<uint4*>(values + chunk_at(kTile, r, i % (D / 8))) = make_uint4(0, 0, 0, 0);
          }
          fence_async_shared();
          asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], 4;" ::"r"(smem_u32(b_full + slot)) : "memory");
        }
      }
      tile_no += x.tiles;
    }
  } else if (warp > L::kWalk) {
    // (completes a warpgroup)
    if constexpr (L::kMoreRegs > 0) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kFewerRegs));
  } else {
    // ================= the walk along the line =================
    if constexpr (L::kMoreRegs > 0) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kFewerRegs));
    int e = s_first[0], off = s_first[1], no = 0, parity = 0;
    long long at = (long long)cta * share;
    const long long end = min((long long)units, at + share);
    auto hand = [&](const Piece& x) {
      if (no >= kRing && !wait(b_taken + no % kRing, ((no / kRing) & 1) ^ 1)) return;
      if (lane == 0) {
        s_piece[no % kRing] = x;
        mbar_arrive(b_piece + no % kRing);
      }
      __syncwarp();
      ++no;
    };
    while (ok && at < end && e < elements) {
      // 32 elements at a time
      const Element mine = e + lane < elements ? element_of<D>(p, e + lane) : Element{};
      uint32_t some = __ballot_sync(0xffffffffu, mine.end > mine.begin);
      for (; some != 0 && at < end && ok; some &= some - 1) {
        const int l = __ffs(some) - 1;
        Element x;
        x.begin = __shfl_sync(0xffffffffu, mine.begin, l);
        x.end = __shfl_sync(0xffffffffu, mine.end, l);
        x.low = __shfl_sync(0xffffffffu, mine.low, l);
        x.queries = __shfl_sync(0xffffffffu, mine.queries, l);
        x.first = __shfl_sync(0xffffffffu, mine.first, l);
        x.row = __shfl_sync(0xffffffffu, mine.row, l);
        const bool two = pair_of(x.queries, L::kQueries);
        const int tiles = tiles_of(x.end - x.begin, kTile), each = item_units(tiles, two), cuts = query_tiles(x.queries, L::kQueries);
        const long long start = at - off;  // the element's first unit
        int item = off / each;
        off = 0;
        for (; item < p.pool.heads * cuts && start + (long long)item * each < end && ok; ++item) {
          const Tiles part = piece_of((int)(start + (long long)item * each), tiles, two, share, cta);
          if (part.to > part.from) {
            Piece y;
            y.tiles = part.to - part.from;
            y.begin = x.begin + part.from * kTile;
            y.end = x.end;
            y.low = x.low;
            y.row = x.row;
            y.first = x.first;
            y.head = item / cuts;
            y.query0 = (item - y.head * cuts) * L::kQueries;
            y.queries = min(L::kQueries, x.queries - y.query0);
            y.whole = part.from == 0;
            y.pair = y.queries > 128;
            y.stream = y.pair || kStreams == 1 ? 0 : parity;
            if (!y.pair) parity = (parity + y.tiles) & (kStreams - 1);
            else parity = 0;
            hand(y);
          }
        }
        at = start + (long long)p.pool.heads * cuts * each;
      }
      e += 32;
    }
    Piece last = {};
    hand(last);
  }
  if (!ok && s_first[0] >= 0 && lane == 0) atomicCAS(p.error, 0u, kErrWait);
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == L::kMma) tmem_dealloc(tmem, L::kCols);
}

// Joins the pieces of a row's heads: a warp takes a head at a time.
constexpr int kJoinWarps = 4;
template <int D, typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) k_shared_join(const __grid_constant__ Params p) {
  using L = Shape<D>;
  constexpr int kPer = D / 32;  // values of a lane
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x, kh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int elements = 2 * p.a.rows, units = p.line[elements], share = units > 0 ? unit_share(units, p.ctas) : 1;
  const int2 place = p.place[row];
  const Element of[2] = {element_of<D>(p, min(max(place.x, 0), p.a.rows - 1)), element_of<D>(p, p.a.rows + row)};
  const int line[2] = {p.line[min(max(place.x, 0), p.a.rows - 1)], p.line[p.a.rows + row]};
  const float v_scale = p.pool.v_scale ? p.pool.v_scale[kh] : 1.f;
  for (int g = warp; g < p.group; g += kJoinWarps) {
    const int head = kh * p.group + g;
    float top = -INFINITY, sum = 0.f, acc[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) acc[j] = 0.f;
#pragma unroll 1
    for (int kind = 0; kind < 2; ++kind) {
      const Element x = of[kind];
      if (kind == 0 && !takes_part(seen_of(p.a.lengths[row], p.max_len, p.a.window), p.shared[row])) continue;
      const int tiles = units > 0 ? tiles_of(x.end - x.begin, L::kTile) : 0;
      if (tiles == 0) continue;
      const int query = kind == 0 ? place.y * p.group + g : g;
      if ((unsigned)query >= (unsigned)x.queries) continue;
      const int cuts = query_tiles(x.queries, L::kQueries), cut = query / L::kQueries, within = query - cut * L::kQueries;
      const bool pair = min(L::kQueries, x.queries - cut * L::kQueries) > 128;
      const bool two = pair_of(x.queries, L::kQueries);
      const int begin = line[kind] + (kh * cuts + cut) * item_units(tiles, two);
      const int first = cta_of(begin, 0, two, share), pieces = cta_of(begin, tiles - 1, two, share) - first + 1;
      // parts: two halves of a piece where its tiles went to both streams
      for (int i0 = 0; i0 < 2 * pieces; i0 += 32) {
        const int i = i0 + lane, piece = i >> 1, half = i & 1;
        bool some = piece < pieces;
        long long at = 0;
        if (some) {
          const Tiles t = piece_of(begin, tiles, two, share, first + piece);
          some = half == 0 || (!pair && L::kStreams == 2 && t.to - t.from > 1);
          const int stream = pair ? within >> 7 : half, lane_of = pair ? within & 127 : within;
          at = piece == 0 ? ((2 * kind + half) * (long long)p.a.rows + row) * p.a.heads + head : ((first + piece) * 2ll + stream) * 128 + lane_of;
        }
        const float2 ml = some ? (piece == 0 ? p.ml : p.more_ml)[at] : make_float2(-INFINITY, 0.f);
        float most = ml.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float next = fmaxf(top, most), base = next == -INFINITY ? 0.f : next;
        const float old = exp2_ftz(top - base), by = exp2_ftz(ml.x - base);
        float l = by * ml.y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        sum = sum * old + l;
        top = next;
#pragma unroll
        for (int j = 0; j < kPer; ++j) acc[j] *= old;
        const float* const from = (piece == 0 ? p.out : p.more) + at * D;
        for (uint32_t who = __ballot_sync(0xffffffffu, some); who != 0; who &= who - 1) {
          const int l = __ffs(who) - 1;
          const float* const o = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(from), l)) + lane * kPer;
          const float w = __shfl_sync(0xffffffffu, by, l);
          if constexpr (kPer == 2) {
            const float2 v = *reinterpret_cast<const float2*>(o);
            acc[0] += w * v.x, acc[1] += w * v.y;
          } else {
#pragma unroll
            for (int j = 0; j < kPer; j += 4) {
              const float4 v = *reinterpret_cast<const float4*>(o + j);
              acc[j] += w * v.x, acc[j + 1] += w * v.y, acc[j + 2] += w * v.z, acc[j + 3] += w * v.w;
            }
          }
        }
      }
    }
    // (no positions: zeros, as what was added up is zero)
    const float inv = top == -INFINITY ? 0.f * sum : v_scale / sum;
    uint32_t* const out = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p.a.out) + row * p.a.out_stride + head * p.a.out_head_stride + lane * kPer);
#pragma unroll
    for (int j = 0; j < kPer; j += 2) out[j / 2] = pack2((const T*)nullptr, acc[j] * inv, acc[j + 1] * inv);
    if (p.a.lse && lane == 0) p.a.lse[(long long)row * p.a.heads + head] = (top + log2f(sum)) * kLn2;
  }
}

size_t rounded(size_t n) { return (n + 255) / 256 * 256; }
struct Workspace {
  size_t line, place, out, ml, more, more_ml, all;
  Workspace(size_t rows, size_t heads, size_t dim, size_t ctas) {
    line = 0;
    place = line + rounded((2 * rows + 1) * sizeof(int));
    out = place + rounded(rows * sizeof(int2));
    ml = out + rounded(4 * rows * heads * dim * sizeof(float));
    more = ml + rounded(4 * rows * heads * sizeof(float2));
    more_ml = more + rounded(ctas * 256 * dim * sizeof(float));
    all = more_ml + rounded(ctas * 256 * sizeof(float2));
  }
};

template <int D, typename T, bool kE4M3>
cudaError_t launch(Params p, char* workspace, int sms, cudaStream_t stream) {
  using L = Shape<D>;
  const long long most = most_units(p.a.rows, p.pool.heads, p.group, p.max_len, L::kTile, L::kQueries);
  p.max_units = (int)most;
  p.ctas = (int)std::min<long long>(sms, (most + kLeastUnits - 1) / kLeastUnits);
  const Workspace w(p.a.rows, p.a.heads, D, p.ctas);
  p.line = reinterpret_cast<int*>(workspace + w.line);
  p.place = reinterpret_cast<int2*>(workspace + w.place);
  p.out = reinterpret_cast<float*>(workspace + w.out);
  p.ml = reinterpret_cast<float2*>(workspace + w.ml);
  p.more = reinterpret_cast<float*>(workspace + w.more);
  p.more_ml = reinterpret_cast<float2*>(workspace + w.more_ml);
  // TMA boxes of whole pages or parts of one, of 8 positions up to a warp's share of a tile (so many divide a page); pools that no tensor map
  // can have, and 8-bit ones, which are converted on the way, go without
  CUtensorMap k_map = {}, v_map = {};
  p.box = L::kTile / 4;
  while (p.box > 1 && p.pool.page_size % p.box != 0) p.box /= 2;
  const PagedPool& pool = p.pool;
  const bool bf16 = __is_same(T, __nv_bfloat16);
  auto map = [&](CUtensorMap* m, const void* base) {
    return make_page_map(m, base, bf16, D, pool.page_size, pool.heads, pool.pages, pool.pos_stride * 2, pool.head_stride * 2, pool.page_stride * 2, p.box) ==
           cudaSuccess;
  };
  if (kE4M3 || p.box < 8 || !map(&k_map, pool.k) || !map(&v_map, pool.v)) p.box = 0;
  auto* kernel = k_shared_attention<D, T, kE4M3 ? STAGE_E4M3 : STAGE_COPY>;
  if constexpr (!kE4M3) kernel = p.box > 0 ? k_shared_attention<D, T, STAGE_TMA> : kernel;
  cudaError_t rc = kernel_setup(reinterpret_cast<const void*>(kernel), L::kSmem).rc;
  if (rc != cudaSuccess) return rc;
  rc = launch_kernel_ex(kernel, dim3(p.ctas), dim3(L::kThreads), (size_t)L::kSmem, stream, true, 1, p, k_map, v_map);
  if (rc != cudaSuccess) return rc;
  return launch_kernel_ex(k_shared_join<D, T>, dim3(p.a.rows, p.pool.heads), dim3(kJoinWarps * 32), 0, stream, true, 1, p);
}

}  // namespace

size_t shared_attention_workspace_bytes(int rows, int heads, int dim, int sms) { return Workspace(rows, heads, dim, sms).all; }

cudaError_t launch_shared_attention(const PagedAttention& a, PagedType type, const PagedPool& pool, PagedType cache, const SharedGroups& groups,
                                    void* workspace, int sms, uint32_t* error_word, cudaStream_t stream) {
  if (a.rows < 1 || a.rows > kPagedMaxRows || pool.heads < 1 || pool.heads > 65535 || a.heads % pool.heads != 0 || a.heads < pool.heads || type == PAGED_E4M3 ||
      (cache != PAGED_E4M3 && cache != type))
    return cudaErrorInvalidValue;
  const long long cap = (long long)a.width * pool.page_size;
  const int max_len = (int)(cap < kMaxLen ? cap : kMaxLen);
  if (!shared_fits(a.rows, pool.heads, a.heads / pool.heads, max_len, pool.dim)) return cudaErrorInvalidValue;
  Params p = {};
  p.a = a;
  p.pool = pool;
  p.div = page_div(pool.page_size);
  p.order = groups.order;
  p.starts = groups.starts;
  p.shared = groups.shared;
  p.group = a.heads / pool.heads;
  p.max_len = max_len;
  const Steps st = steps_of(pool.pages, pool.page_size, pool.page_stride, pool.pos_stride, cache == PAGED_E4M3 ? 1 : 2);
  if (st.bytes == 0) return cudaErrorInvalidValue;
  p.page_step = st.page;
  p.pos_step = st.pos;
  p.step_bytes = st.bytes;
  p.error = error_word;
  char* const w = reinterpret_cast<char*>(workspace);
#define PENNY_SHARED_TYPE(D)                                                                                                     \
  (cache == PAGED_E4M3 ? (type == PAGED_BF16 ? launch<D, __nv_bfloat16, true>(p, w, sms, stream) : launch<D, __half, true>(p, w, sms, stream)) \
                       : (type == PAGED_BF16 ? launch<D, __nv_bfloat16, false>(p, w, sms, stream) : launch<D, __half, false>(p, w, sms, stream)))
  switch (pool.dim) {
    case 64: return PENNY_SHARED_TYPE(64);
    case 128: return PENNY_SHARED_TYPE(128);
    case 256: return PENNY_SHARED_TYPE(256);
    default: return cudaErrorInvalidValue;
  }
#undef PENNY_SHARED_TYPE
}

}  // namespace penny
