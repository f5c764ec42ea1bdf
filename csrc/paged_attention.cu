// Attention of one new token per sequence over a paged KV cache.  (The attention over contiguous caches, csrc/decode_attention_fused.cu,
// rotates and appends its token itself; here csrc/paged_append.cu has done that.)
//
//   o[b, h] = sum_j softmax_j(scale * q[b, h] . K_j) V_j,  j in the last `window` of lengths[b] positions (all without one),
// position j in the pool's page table[b, j / page_size] at j % page_size.  One pass over K and V with a running maximum and sum
// (fp32); lse = the logarithm of the sum.  Rows without positions: zeros, -inf.  Positions on a page that the pool does not
// have count as not there.
//
//   * The heads of a KV head share its keys and values.  Keys and values are the M side of mma.sync (m16n8k16), the G = Hq / Hkv
//     query heads its N side: S^T = K Q^T, O^T = V^T P^T, so eight heads fill a product (sixteen take two, more go to several
//     CTAs), and P^T is S^T's accumulators, transposed in registers.  (The 128 rows of a tcgen05 tile would be empty; the bound is
//     the cache's stream.)
//   * All warps of the GPU get an equal share of the batch: for every head group the tiles (4 KB of K and 4 KB of V: 16 positions
//     of 128 bf16 values) of all rows in a line, cut every `share` tiles (paged_plan.h; every warp sums over the lengths by
//     itself).  A warp walks its part of the line with a private three-stage cp.async pipeline that does not drain between
//     rows (a CTA for each piece of a row instead took 48 us for 26 at rows of up to 1000 positions of 20 heads of 64).  64 entries
//     of the row's table stand in the lanes' registers; sixteen positions on one page take one of them, others one each, so
//     any page size and any strides will do.  What lies outside a row is filled with zeros and never read (stale rows may
//     hold anything).
//   * A row that lies in one warp's part is finished from its registers, the parts of one that spans warps of a CTA
//     meet in shared memory, those of several CTAs in a workspace, which a second kernel joins.  No counters: a workspace
//     holds nothing between calls.
//   * e4m3 caches: fp16 is exact for them, so they meet q as fp16, each row of q times the power of two that brings its largest value
//     to [2^15, 2^16) (exact for fp16 rows; of bf16 ones values under 2^-29 of the largest keep 2^-40 of it; the score's factor takes it
//     back).  A lane's four bytes of K are two adjacent pairs: the dims inside a
//     16-byte chunk are permuted on both sides of the product.  V's bytes are transposed in pairs by ldmatrix and separated
//     into even and odd dims.
//   * P is rounded to the type of the product (bf16: 2^-8 of each weight at most, averaged over the positions; the sum is of the
//     unrounded ones); q, scores, maxima and sums are not rounded.  fp16 holds nothing under 2^-25 and little under 2^-14, and a long
//     row has many such weights: the base of fp16 weights stands kShift under the maximum, so that the largest is near 2^15 and a weight
//     loses 2^-40 of the largest at most (2^-32 where the base may lag).  With a largest weight of one, 25,000 positions of a warp
//     that stood 17.4 under another one were lost whole.  Weights count from a base near the maximum so far.  Where they are
//     finer than the output (e4m3 caches with a bf16 q) it follows when it is exceeded by 2^8, which is seldom (64 rows of 4096, 28
//     of 2 heads: 34.4 us, always 38.1).  Elsewhere it follows always, so that the largest weight is one and not off: 64 rows of 2048,
//     bf16, are 0.00183 of the output's norm from 64 bits (its own rounding: 0.00166; the rest is P's), otherwise 0.0022 (and 0.5 us
//     faster).
//
// Bound by memory: 64 rows of 2048 positions, 32 of 8 heads of 128, bf16, 85 us (6.3 TB/s), 64 of 16000 598 (7.0); few or short rows by
// a chain of latencies: 6.6 us for one row of 200, 9.4 for one of 2048.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "decode_attn_common.cuh"
#include "kernel_setup.h"
#include "paged_kernels.h"
#include "paged_plan.h"
#include "pdl.h"

namespace penny {
namespace {
using namespace paged;
using attn::cp_async16;
using attn::cp_async_commit;
using attn::cp_async_wait;
using attn::ldmatrix_x4;
using attn::ldmatrix_x4_trans;
using attn::mma_bf16;

constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int D, bool kE4M3, int kBlocks>
struct Tile {
  static constexpr int kRow = kE4M3 ? D : 2 * D;               // bytes of a position
  static constexpr int kPos = kRow <= 128 ? 32 : 16;
  static constexpr int kChunks = kRow / 16;                    // 16-byte chunks of a position
  static constexpr int kPerPass = 32 / kChunks;                // positions that a warp's 32 chunks cover
  static constexpr int kStage = 2 * kPos * kRow;
  static constexpr uint32_t kAll = 0xffffffffu >> (32 - kPos);  // the mask of a full tile
  static constexpr int kFrags = kBlocks * (D / 16);            // MMA accumulators of O^T: 16 dims x 8 heads, a float4 a lane
  static constexpr int kParts = kWarps * kFrags * 512;         // room for a part of every warp
  // two CTAs to an SM where three stages (five small ones) or two of them leave room for that, else one; of 228 KB a CTA takes 1 KB
  // and its static variables, in whole KB, besides
  static constexpr int kOwn = 1024 + kBlocks * 1024, kHalf = (228 << 10) / 2 - kOwn;
  static constexpr int stages(int most, int limit) {
    int n = most;
    while (n > 2 && n * kWarps * kStage + kParts > limit) --n;
    return n;
  }
  static constexpr bool kTwo = 2 * kWarps * kStage + kParts <= kHalf;
  static constexpr int kStages = stages(kStage < 8192 ? 5 : 3, kTwo ? kHalf : (228 << 10) - kOwn);
  static constexpr int kPipes = kWarps * kStages * kStage, kSmem = kPipes + kParts;
  static_assert(kSmem <= (kTwo ? kHalf : (228 << 10) - kOwn) && kStages * kStage >= kFrags * 512, "shared memory");
  // where chunk c of position r lies: eight positions' equal chunks in eight different 16-byte banks
  static __device__ __forceinline__ uint32_t at(int r, int c) {
    if constexpr (kRow == 64) return (uint32_t)((r >> 1) * 128 + ((((r & 1) << 2) | (c ^ ((r >> 1) & 3))) << 4));
    return (uint32_t)(r * kRow + ((c ^ (r & 7)) << 4));
  }
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// two e4m3 values (the low or the high half of x) as fp16
__device__ __forceinline__ uint32_t e4m3_lo(uint32_t x) {
  uint32_t r;
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, l;}" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_hi(uint32_t x) {
  uint32_t r;
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, h;}" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float exp2_ftz(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// an 8 x 8 matrix of 16-bit values, transposed in the warp's registers
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float2 to_f32(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ float2 to_f32(__half2 v) { return __half22float2(v); }
template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return attn::pack2(lo, hi); }
};
template <>
struct Pair<__half> {
  using type = __half2;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_f16(lo, hi); }
};

struct Params {
  PagedAttention a;
  PagedPool pool;
  PageDiv div;
  int group;              // G
  int items, groups;      // (KV head, head group) pairs, head groups of a KV head
  int teams;              // CTAs of an item
  bool by_row;            // the joining kernel has a block for each row, not for each team
  int max_len;
  uint32_t page_step, pos_step, step_bytes;  // strides in units of step_bytes
  float4* parts;          // per CTA two parts: of a row that began before it, of one that ends after it
  float2* part_ml;        // their maxima (base 2) and sums
};

// The row of unit `unit` of the line and how far behind the row's first it is; `unit` of `share`, the units of a warp.  False: behind the
// line's end.  Called by whole warps, each of which sums over all rows (no barrier).
template <class UnitOf>
__device__ __forceinline__ bool locate(const Params& p, int tile, UnitOf unit, int& row, int& at, int& share, int& total) {
  const int lane = threadIdx.x & 31;
  const int per = (p.a.rows + 31) / 32, r0 = min(p.a.rows, lane * per), r1 = min(p.a.rows, r0 + per);
  auto units = [&](int r) {
    const Seen s = seen_of(p.a.lengths[r], p.max_len, p.a.window);
    return units_of(s.end - s.first, tile);
  };
  int mine = 0;
#pragma unroll 4
  for (int r = r0; r < r1; ++r) mine += units(r);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  total = __shfl_sync(0xffffffffu, incl, 31);
  share = share_of(total, p.teams * kWarps);
  const long long begin = unit(share);
  if (begin >= total) return false;
  row = r0, at = (int)begin - (incl - mine);
  const bool here = at >= 0 && at < mine;
  if (here && per > 1) {
    for (int n; at >= (n = units(row)); ++row) at -= n;
  }
  const int from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
  row = __shfl_sync(0xffffffffu, row, from);
  at = __shfl_sync(0xffffffffu, at, from);
  return true;
}

// One accumulator of O^T, rounded, to its 16 dims of up to eight heads: this thread holds dims g and g + 8
// (e4m3: 2 g and 2 g + 1) of heads 2 t and 2 t + 1.  Called by whole warps.  out: the first head's dims.
template <typename T, bool kE4M3>
__device__ __forceinline__ void store_frag(T* out, long long head_stride, int heads, int lane, const float4& o) {
  const uint32_t lo = transpose8x8(Pair<T>::pack(o.x, o.y)), hi = transpose8x8(Pair<T>::pack(o.z, o.w));
  const int g = lane >> 2, t = lane & 3;  // now head g
  if (g >= heads) return;
  T* to = out + g * head_stride;
  if constexpr (kE4M3) {
    *reinterpret_cast<uint2*>(to + 4 * t) = make_uint2(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
  } else {
    *reinterpret_cast<uint32_t*>(to + 2 * t) = lo;
    *reinterpret_cast<uint32_t*>(to + 8 + 2 * t) = hi;
  }
}
__device__ __forceinline__ float inverse(float top, float sum, float factor) { return top == -INFINITY ? 0.f * sum : factor / sum; }

// kBlocks: blocks of eight query heads of a CTA, 1 or 2.
template <int D, typename T, bool kE4M3, int kBlocks>
__global__ void __launch_bounds__(kWarps * 32) k_paged_attention(const __grid_constant__ Params p) {
  using L = Tile<D, kE4M3, kBlocks>;
  using T2 = typename Pair<T>::type;
  constexpr int kRows = 8 * kBlocks, kSteps = D / 16, kGroups = L::kPos / 16, kStages = L::kStages;
  constexpr bool kBf16 = !kE4M3 && __is_same(T, __nv_bfloat16);
  // exponents: how far the base stands under the maximum, and how far a score may be above that before it follows (fp16 weights: up to
  // 2^(kShift + kSlack) = 2^15)
  constexpr float kSlack = kE4M3 && __is_same(T, __nv_bfloat16) ? 8.f : 0.f, kShift = kBf16 ? 0.f : 15.f - kSlack;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ float2 s_ml[2][kWarps][kRows];  // of a warp's first part and of its last
  __shared__ int s_head[kWarps];             // a part of a row that began before: 0 none, 1 it ends here, 2 it does not
  __shared__ int s_tail[kWarps];             // a row that does not end here, -1: none
  // (dependents may start once all CTAs are behind the wait: the joining kernel reads the lengths before its own)
  bool waited = !p.a.early;
  auto wait = [&]() {
    pdl_wait();
    pdl_launch_dependents();
    waited = true;
  };
  if (waited) wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  auto seen = [&](int row) { return seen_of(p.a.lengths[row], p.max_len, p.a.window); };
  Walk load = {};
  {
    const int me = (int)blockIdx.y * kWarps + warp;
    int share, total;
    if (locate(p, L::kPos, [&](int each) { return (long long)me * each; }, load.row, load.at, share, total)) {
      load.left = min(share, total - me * share);
      enter_row(load, L::kPos, seen);
    }
  }
  Walk w = load;
  const int kh = kBlocks == 1 ? (int)blockIdx.x : (int)blockIdx.x / p.groups, h0 = kBlocks == 1 ? 0 : ((int)blockIdx.x - kh * p.groups) * kRows;
  const int heads = min(kRows, p.group - h0), head0 = kh * p.group + h0;  // of this CTA
  const int cta = (int)(blockIdx.y * gridDim.x + blockIdx.x);
  const uint32_t wbase = attn::smem_u32_local(smem_raw) + warp * (kStages * L::kStage);
  float4* heads_area = reinterpret_cast<float4*>(smem_raw + L::kPipes);                                  // [warps][frags][32]
  auto tail_area = [&](int i) { return reinterpret_cast<float4*>(smem_raw + i * (kStages * L::kStage)); };  // a drained pipeline's space
  constexpr int kSize = kE4M3 ? 1 : 2;
  const uint32_t pos_bytes = p.pos_step * p.step_bytes;
  const char* kbase = reinterpret_cast<const char*>(p.pool.k) + kh * p.pool.head_stride * kSize + (lane % L::kChunks) * 16;
  const char* vbase = reinterpret_cast<const char*>(p.pool.v) + kh * p.pool.head_stride * kSize + (lane % L::kChunks) * 16;

  // ---- loading: 64 entries of the row's table in the lanes' registers, the next 32 on their way ----
  int load_pos = 0, load_tiles = 0, ids_at = 0, ids[2] = {-1, -1};
  const int* table = nullptr;
  auto load_ids = [&](int at) { return at + lane < pages_of(p.div, load.end) ? table[at + lane] : -1; };
  int stage_in = 0, stage_out = 0;
  // requests the next tile; the mask of its positions that are there
  auto issue = [&]() {
    uint32_t mask = 0;
    if (load_tiles == 0) {
      while (load.left > 0 && load_tiles <= 0) {
        const WalkPart part = next_part(load, L::kPos, seen);
        load_tiles = max(0, part.to - part.from);
        load_pos = load.first + part.from * L::kPos;
      }
      if (load_tiles > 0) {
        table = p.a.table + load.row * p.a.table_stride;
        ids_at = div_page(p.div, load_pos);
        ids[0] = load_ids(ids_at);
        ids[1] = load_ids(ids_at + 32);
      }
    }
    if (load_tiles > 0) {
      if (!waited && load_pos + L::kPos >= load.end) wait();  // the tile of the row's last position
      const uint32_t sb = wbase + stage_in * L::kStage;
      const int r0 = lane / L::kChunks, c = lane % L::kChunks;
      const int page0 = div_page(p.div, load_pos) - ids_at;
      if (page0 >= 32) {  // (a tile has 32 pages at most)
        ids_at += 32;
        ids[0] = ids[1];
        ids[1] = load_ids(ids_at + 32);
      }
#pragma unroll
      for (int part = 0; part < L::kPos; part += 16) {
        const int from = load_pos + part, at0 = div_page(p.div, from) - ids_at;
        constexpr int kPasses = 16 / L::kPerPass;
        if (from + 16 <= load.end && div_page(p.div, from + 15) - ids_at == at0) {  // all of it on one page
          const int id = __shfl_sync(0xffffffffu, at0 < 32 ? ids[0] : ids[1], at0 & 31);
          const uint32_t off = step_of(id, p.pool.pages, from, p.div, p.page_step, p.pos_step);
          const bool ok = off != kNoStep;
          if (ok) mask |= 0xffffu << part;
          const unsigned long long by = ok ? (unsigned long long)off * p.step_bytes + (unsigned long long)pos_bytes * r0 : 0;
          const char *kp = kbase + by, *vp = vbase + by;
          const uint32_t pass_bytes = ok ? pos_bytes * L::kPerPass : 0;
#pragma unroll
          for (int i = 0; i < kPasses; ++i) {
            const uint32_t s = sb + L::at(part + i * L::kPerPass + r0, c);
            cp_async16(s, kp + (unsigned long long)pass_bytes * i, ok);
            cp_async16(s + L::kPos * L::kRow, vp + (unsigned long long)pass_bytes * i, ok);
          }
        } else {
          const int pos = from + lane % 16, at = div_page(p.div, pos) - ids_at;
          const int lo = __shfl_sync(0xffffffffu, ids[0], at & 31), hi = __shfl_sync(0xffffffffu, ids[1], at & 31);
          const uint32_t off = step_of(pos < load.end ? (at < 32 ? lo : hi) : -1, p.pool.pages, pos, p.div, p.page_step, p.pos_step);
          mask |= (__ballot_sync(0xffffffffu, off != kNoStep) & 0xffffu) << part;
#pragma unroll
          for (int i = 0; i < kPasses; ++i) {
            const int r = i * L::kPerPass + r0;
            const uint32_t o = __shfl_sync(0xffffffffu, off, r);
            const bool ok = o != kNoStep;
            const unsigned long long by = ok ? (unsigned long long)o * p.step_bytes : 0;
            const uint32_t s = sb + L::at(part + r, c);
            cp_async16(s, kbase + by, ok);
            cp_async16(s + L::kPos * L::kRow, vbase + by, ok);
          }
        }
      }
      load_pos += L::kPos;
      --load_tiles;
    }
    stage_in = stage_in + 1 == kStages ? 0 : stage_in + 1;
    cp_async_commit();  // always: keeps the group count in step with the tiles
    return mask;
  };
  uint32_t masks[kStages];  // of the tiles in flight
#pragma unroll
  for (int j = 0; j + 1 < kStages; ++j) masks[j] = issue();
  if (!waited) wait();
  if (lane == 0) {
    s_head[warp] = 0;
    s_tail[warp] = -1;
  }

  uint32_t qb[kBlocks][kSteps][2];
  float qs[kBlocks][2];
  // q of a row as MMA B fragments (head g of a block), and what turns the scores of heads 2 t and 2 t + 1 into exponents of two
  auto load_q = [&](int row) {
#pragma unroll
    for (int nb = 0; nb < kBlocks; ++nb) {
      const int h = min(nb * 8 + g, heads - 1);
      const T* q = reinterpret_cast<const T*>(p.a.q) + row * p.a.q_stride + (head0 + h) * p.a.q_head_stride;
      if constexpr (kE4M3) {
        float x[kSteps][4], top = 0.f;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          const uint2 raw = *reinterpret_cast<const uint2*>(q + k * 16 + 4 * t);
          const float2 lo = to_f32(*reinterpret_cast<const T2*>(&raw.x)), hi = to_f32(*reinterpret_cast<const T2*>(&raw.y));
          x[k][0] = lo.x, x[k][1] = lo.y, x[k][2] = hi.x, x[k][3] = hi.y;
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(x[k][i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // times 2^(142 - e), so that the largest is in [2^15, 2^16) (smaller where it is under 2^-111, for both powers to be fp32's)
        const int e = max((__float_as_int(top) >> 23) & 255, 16);
        const float up = __int_as_float((269 - e) << 23), factor = p.a.scale * kLog2e * p.pool.k_scale[kh] * __int_as_float((e - 15) << 23);
#pragma unroll
        for (int i = 0; i < 2; ++i) qs[nb][i] = __shfl_sync(0xffffffffu, factor, (2 * t + i) * 4);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          qb[nb][k][0] = pack_f16(x[k][0] * up, x[k][1] * up);
          qb[nb][k][1] = pack_f16(x[k][2] * up, x[k][3] * up);
        }
      } else {
        qs[nb][0] = qs[nb][1] = p.a.scale * kLog2e;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          qb[nb][k][0] = *reinterpret_cast<const uint32_t*>(q + k * 16 + 2 * t);
          qb[nb][k][1] = *reinterpret_cast<const uint32_t*>(q + k * 16 + 8 + 2 * t);
        }
      }
    }
  };
  auto mma = [&](float (&d)[4], const uint32_t (&a)[4], const uint32_t (&bb)[2]) {
    if constexpr (kBf16) mma_bf16(d, a[0], a[1], a[2], a[3], bb[0], bb[1]);
    else mma_f16(d, a[0], a[1], a[2], a[3], bb[0], bb[1]);
  };
  T* const out = reinterpret_cast<T*>(p.a.out);
  auto out_of = [&](int row, int head) { return out + row * p.a.out_stride + head * p.a.out_head_stride; };

  // ---- this warp's share, row by row ----
  while (w.left > 0) {
    const WalkPart part = next_part(w, L::kPos, seen);
    const int n = part.to - part.from;
    if (w.first == w.end) {  // an empty row
      for (int f = 0; f < L::kFrags; ++f)
        store_frag<T, kE4M3>(out_of(w.row, head0 + f / kSteps * 8) + f % kSteps * 16, p.a.out_head_stride, heads - f / kSteps * 8, lane,
                             make_float4(0.f, 0.f, 0.f, 0.f));
      if (p.a.lse && lane < heads) p.a.lse[(long long)w.row * p.a.heads + head0 + lane] = -INFINITY;
      continue;
    }
    if (n <= 0) continue;
    load_q(w.row);
    // per block of heads: the base (m: minus infinity before there is one) of heads 2 t and 2 t + 1, this thread's share of their sums, O^T
    float m[kBlocks][2], base[kBlocks][2], l[kBlocks][2], o[kBlocks][kSteps][4];
#pragma unroll
    for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
      for (int i = 0; i < 2; ++i) m[nb][i] = -INFINITY, base[nb][i] = l[nb][i] = 0.f;
#pragma unroll
      for (int k = 0; k < kSteps; ++k) o[nb][k][0] = o[nb][k][1] = o[nb][k][2] = o[nb][k][3] = 0.f;
    }
    for (int j = 0; j < n; ++j) {
      // The next tile is requested behind the scores' products, whose latency its instructions fill (64 rows of 2048 86.0 us, in front of
      // the wait for this tile 89.3; 64 of 16000, e4m3, 315 and 363); with two stages in front (16 heads of 256 61 us, behind 66).
      if constexpr (kStages == 2) {
        __syncwarp();  // everyone is done with the stage that the request overwrites
        masks[1] = issue();
        cp_async_wait<1>();
      } else {
        cp_async_wait<kStages - 2>();
      }
      __syncwarp();  // all of the tile is there (and everyone is done with the one before)
      const uint32_t sb = wbase + stage_out * L::kStage;
      stage_out = stage_out + 1 == kStages ? 0 : stage_out + 1;
      // ---- S^T = K Q^T, 16 positions at a time: this thread holds positions g and g + 8 of heads 2 t and 2 t + 1 ----
      // (even and odd steps apart: a chain of products into one accumulator is the longest wait of a tile)
      float s[kBlocks][kGroups][4];
#pragma unroll
      for (int c = 0; c < kGroups; ++c) {
        float odd[kBlocks][4];
#pragma unroll
        for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
          for (int u = 0; u < 4; ++u) s[nb][c][u] = odd[nb][u] = 0.f;
        }
        const int row = c * 16 + (lane & 15);
#pragma unroll
        for (int k2 = 0; k2 < L::kChunks / 2; ++k2) {
          uint32_t a[4];
          ldmatrix_x4(sb + L::at(row, k2 * 2 + (lane >> 4)), a);
          if constexpr (kE4M3) {  // a chunk is 16 dims
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t x[4] = {e4m3_lo(a[2 * i]), e4m3_lo(a[2 * i + 1]), e4m3_hi(a[2 * i]), e4m3_hi(a[2 * i + 1])};
#pragma unroll
              for (int nb = 0; nb < kBlocks; ++nb) mma(i ? odd[nb] : s[nb][c], x, qb[nb][k2 * 2 + i]);
            }
          } else {
#pragma unroll
            for (int nb = 0; nb < kBlocks; ++nb) mma(k2 & 1 ? odd[nb] : s[nb][c], a, qb[nb][k2]);
          }
        }
#pragma unroll
        for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
          for (int u = 0; u < 4; ++u) s[nb][c][u] += odd[nb][u];
        }
      }
      if constexpr (kStages > 2) masks[kStages - 1] = issue();
      // ---- weights exp2(score - base); the base goes up when a score of the tile is above base + kShift by more than kSlack ----
      uint32_t pb[kBlocks][kGroups][2];
#pragma unroll
      for (int nb = 0; nb < kBlocks; ++nb) {
        bool above = false;
        // exponents against the base as it is; minus infinity where nothing is
#pragma unroll
        for (int c = 0; c < kGroups; ++c) {
#pragma unroll
          for (int u = 0; u < 4; ++u) s[nb][c][u] = fmaf(s[nb][c][u], qs[nb][u & 1], -base[nb][u & 1]);
        }
        if (masks[0] != L::kAll) {
          const uint32_t mask = masks[0] >> g;
#pragma unroll
          for (int c = 0; c < kGroups; ++c) {
#pragma unroll
            for (int u = 0; u < 4; ++u) s[nb][c][u] = (mask >> (c * 16 + u / 2 * 8)) & 1 ? s[nb][c][u] : -INFINITY;
          }
        }
#pragma unroll
        for (int c = 0; c < kGroups; ++c) {
#pragma unroll
          for (int u = 0; u < 4; ++u) above = above || s[nb][c][u] > (m[nb][u & 1] == -INFINITY ? -INFINITY : kShift + kSlack);
        }
        if (__any_sync(0xffffffffu, above)) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < kGroups; ++c) top = fmaxf(top, fmaxf(s[nb][c][i], s[nb][c][2 + i]));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            if (top > (m[nb][i] == -INFINITY ? -INFINITY : kShift)) {
              // (the exponents and the base move by the same amount, rounded down: the largest one then is at most kShift and above
              // kShift - 16, however far apart the numbers of the scores' size are)
              const float by = __fsub_rd(kShift, top), corr = m[nb][i] == -INFINITY ? 0.f : exp2_ftz(by);
              m[nb][i] = base[nb][i] -= by;
              l[nb][i] *= corr;
#pragma unroll
              for (int k = 0; k < kSteps; ++k) o[nb][k][i] *= corr, o[nb][k][2 + i] *= corr;
#pragma unroll
              for (int c = 0; c < kGroups; ++c) s[nb][c][i] += by, s[nb][c][2 + i] += by;
            }
          }
        }
#pragma unroll
        for (int c = 0; c < kGroups; ++c) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float p0 = exp2_ftz(s[nb][c][2 * u]), p1 = exp2_ftz(s[nb][c][2 * u + 1]);
            l[nb][0] += p0;
            l[nb][1] += p1;
            pb[nb][c][u] = transpose8x8(kBf16 ? attn::pack2(p0, p1) : pack_f16(p0, p1));
          }
        }
      }
      // ---- O^T += V^T P^T, 16 positions at a time ----
#pragma unroll
      for (int c = 0; c < kGroups; ++c) {
#pragma unroll
        for (int d = 0; d < L::kChunks / 2; ++d) {
          uint32_t a[4];
          const uint32_t vb = sb + L::kPos * L::kRow;
          if constexpr (kE4M3) {  // two chunks of 16 dims: their even dims are rows 0 to 7, the odd ones rows 8 to 15
            ldmatrix_x4_trans(vb + L::at(c * 16 + (lane & 15), d * 2 + (lane >> 4)), a);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t lo = __byte_perm(a[2 * i], 0, 0x3120), hi = __byte_perm(a[2 * i + 1], 0, 0x3120);
              const uint32_t x[4] = {e4m3_lo(lo), e4m3_hi(lo), e4m3_lo(hi), e4m3_hi(hi)};
#pragma unroll
              for (int nb = 0; nb < kBlocks; ++nb) mma(o[nb][d * 2 + i], x, pb[nb][c]);
            }
          } else {
            ldmatrix_x4_trans(vb + L::at(c * 16 + (lane & 7) + (lane >> 4) * 8, d * 2 + ((lane >> 3) & 1)), a);
#pragma unroll
            for (int nb = 0; nb < kBlocks; ++nb) mma(o[nb][d], a, pb[nb][c]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i + 1 < kStages; ++i) masks[i] = masks[i + 1];
    }
#pragma unroll
    for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nb][i] += __shfl_xor_sync(0xffffffffu, l[nb][i], x);
      }
    }
    if (part.begins && part.ends) {
      const float v_scale = kE4M3 ? p.pool.v_scale[kh] : 1.f;
#pragma unroll
      for (int nb = 0; nb < kBlocks; ++nb) {
        const float inv[2] = {inverse(m[nb][0], l[nb][0], v_scale), inverse(m[nb][1], l[nb][1], v_scale)};
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
          store_frag<T, kE4M3>(out_of(w.row, head0 + nb * 8) + k * 16, p.a.out_head_stride, heads - nb * 8, lane,
                               make_float4(o[nb][k][0] * inv[0], o[nb][k][1] * inv[1], o[nb][k][2] * inv[0], o[nb][k][3] * inv[1]));
        if (p.a.lse && g == 0) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (nb * 8 + 2 * t + i < heads) p.a.lse[(long long)w.row * p.a.heads + head0 + nb * 8 + 2 * t + i] = (m[nb][i] + log2f(l[nb][i])) * kLn2;
        }
      }
    } else {
      __syncwarp();  // (the last tile was read by all)
      float4* area = part.begins ? tail_area(warp) : heads_area + warp * (L::kFrags * 32);
#pragma unroll
      for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
          area[(nb * kSteps + k) * 32 + lane] = make_float4(o[nb][k][0], o[nb][k][1], o[nb][k][2], o[nb][k][3]);
        if (g == 0) {
#pragma unroll
          for (int i = 0; i < 2; ++i) s_ml[part.begins][warp][nb * 8 + 2 * t + i] = make_float2(m[nb][i], l[nb][i]);
        }
      }
      if (lane == 0) {
        if (part.begins) s_tail[warp] = w.row;
        else s_head[warp] = part.ends ? 1 : 2;
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();

  // ---- parts that meet inside the CTA: a chain begins with a warp's last part, or with what the team before left ----
  static_assert(kWarps == 4, "a lane for every part and head of eight");
#pragma unroll 1
  for (int first = s_head[0] != 0 ? -1 : 0; first < kWarps; ++first) {
    const int row = first >= 0 ? s_tail[first] : 0;
    if (row < 0) continue;
    int last = first;  // the chain's last warp
    bool done = false;
    while (!done && last + 1 < kWarps && s_head[last + 1] != 0) done = s_head[++last] == 1;
    const bool whole = first >= 0 && done;
    const float v_scale = kE4M3 && whole ? p.pool.v_scale[kh] : 1.f;
    const long long slot = 2ll * cta + (first >= 0);
    // lane 8 i + h: what head h of warp i's part is multiplied by
    const int i = lane >> 3, h8 = lane & 7;
    float by[kBlocks];
#pragma unroll
    for (int nb = 0; nb < kBlocks; ++nb) {
      const int h = nb * 8 + h8;
      const float2 ml = i >= first && i <= last ? s_ml[i == first][i][h] : make_float2(-INFINITY, 0.f);
      float top = fmaxf(ml.x, __shfl_xor_sync(0xffffffffu, ml.x, 8));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
      by[nb] = exp2_ftz(ml.x - (top == -INFINITY ? 0.f : top));
      float sum = by[nb] * ml.y;
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if (whole) {
        by[nb] *= inverse(top, sum, v_scale);
        if (warp == 0 && lane < 8 && h < heads && p.a.lse) p.a.lse[(long long)row * p.a.heads + head0 + h] = (top + log2f(sum)) * kLn2;
      } else if (warp == 0 && lane < 8) {
        p.part_ml[slot * kRows + h] = make_float2(top, sum);
      }
    }
#pragma unroll
    for (int nb = 0; nb < kBlocks; ++nb) {
      float fa[kWarps], fb[kWarps];
#pragma unroll
      for (int u = 0; u < kWarps; ++u) {
        fa[u] = __shfl_sync(0xffffffffu, by[nb], u * 8 + 2 * t);
        fb[u] = __shfl_sync(0xffffffffu, by[nb], u * 8 + 2 * t + 1);
      }
#pragma unroll 1
      for (int k = warp; k < kSteps; k += kWarps) {
        const int f = nb * kSteps + k;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < kWarps; ++u) {
          if (u < first || u > last) continue;
          const float4 v = (u == first ? tail_area(u) : heads_area + u * (L::kFrags * 32))[f * 32 + lane];
          acc.x += fa[u] * v.x, acc.y += fb[u] * v.y, acc.z += fa[u] * v.z, acc.w += fb[u] * v.w;
        }
        if (whole) store_frag<T, kE4M3>(out_of(row, head0 + nb * 8) + k * 16, p.a.out_head_stride, heads - nb * 8, lane, acc);
        else p.parts[(slot * L::kFrags + f) * 32 + lane] = acc;
      }
    }
  }
}

// Joins the parts of a row that spans teams: a block has a row, or the row that begins in its team (if there is one that does not end
// there), and finds out before it waits.  A warp takes an accumulator of O^T, or, with more warps than those, every so many-th part
// of it; with gridDim.z above one a block has one accumulator.  kAhead: parts requested before the first is used.
constexpr int kJoinThreads = 512;
template <int D, typename T, bool kE4M3, int kBlocks, int kAhead>
__global__ void __launch_bounds__(kJoinThreads) k_paged_join(const __grid_constant__ Params p) {
  using L = Tile<D, kE4M3, kBlocks>;
  constexpr int kSteps = D / 16, kRows = 8 * kBlocks;
  __shared__ float4 s_acc[kJoinThreads], s_ml[kJoinThreads];
  pdl_launch_dependents();
  int row = (int)blockIdx.y, team = (int)blockIdx.y, behind = 0;  // teams behind the one that begins the row
  if (p.by_row) {
    int total = 0, before = 0;
    for (int r = threadIdx.x & 31; r < p.a.rows; r += 32) {
      const Seen s = seen_of(p.a.lengths[r], p.max_len, p.a.window);
      const int n = units_of(s.end - s.first, L::kPos);
      total += n;
      before += r < row ? n : 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      total += __shfl_xor_sync(0xffffffffu, total, o);
      before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    const int each = kWarps * share_of(total, p.teams * kWarps);
    const Seen s = seen_of(p.a.lengths[row], p.max_len, p.a.window);
    team = (before + kStart) / each;
    behind = s.end > s.first ? teams_behind(team * each, (team + 1) * each, before, units_of(s.end - s.first, L::kPos)) : 0;
  } else {
    int at, share, total;
    if (locate(p, L::kPos, [&](int each) { return ((long long)team + 1) * kWarps * each; }, row, at, share, total)) {
      const Seen s = seen_of(p.a.lengths[row], p.max_len, p.a.window);
      const int each = kWarps * share, end = (team + 1) * each;
      behind = teams_behind(end - each, end, end - at, units_of(s.end - s.first, L::kPos));
    }
  }
  pdl_wait();
  if (behind == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warps = blockDim.x / 32;
  const int kh = kBlocks == 1 ? (int)blockIdx.x : (int)blockIdx.x / p.groups, h0 = kBlocks == 1 ? 0 : ((int)blockIdx.x - kh * p.groups) * kRows;
  const int heads = min(kRows, p.group - h0), head0 = kh * p.group + h0, n = 1 + behind;
  const int frags = gridDim.z > 1 ? 1 : L::kFrags, sets = max(1, warps / frags), set = warp / frags;
  const long long cta = (long long)team * gridDim.x + blockIdx.x;
  const float v_scale = kE4M3 ? p.pool.v_scale[kh] : 1.f;
  for (int f0 = warp % frags; f0 < frags; f0 += warps) {
    const int f = f0 + (int)blockIdx.z, nb = f / kSteps, h = nb * 8 + 2 * t;
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto take = [&](const float4& ml, const float4& v) {  // maxima and sums of two heads, their values
      const float next[2] = {fmaxf(top[0], ml.x), fmaxf(top[1], ml.z)};
      const float base[2] = {next[0] == -INFINITY ? 0.f : next[0], next[1] == -INFINITY ? 0.f : next[1]};
      const float a = exp2_ftz(top[0] - base[0]), b = exp2_ftz(top[1] - base[1]), c = exp2_ftz(ml.x - base[0]), d = exp2_ftz(ml.z - base[1]);
      sum[0] = sum[0] * a + ml.y * c, sum[1] = sum[1] * b + ml.w * d;
      acc.x = acc.x * a + v.x * c, acc.y = acc.y * b + v.y * d, acc.z = acc.z * a + v.z * c, acc.w = acc.w * b + v.w * d;
      top[0] = next[0], top[1] = next[1];
    };
    for (int i0 = set; i0 < n; i0 += kAhead * sets) {
      float4 ml[kAhead], v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * sets;
        const long long slot = 2 * (cta + (long long)i * gridDim.x) + (i == 0);
        if (i < n) {
          ml[u] = *reinterpret_cast<const float4*>(p.part_ml + slot * kRows + h);
          v[u] = p.parts[(slot * L::kFrags + f) * 32 + lane];
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (i0 + u * sets < n) take(ml[u], v[u]);
    }
    if (sets > 1) {
      s_acc[threadIdx.x] = acc;
      s_ml[threadIdx.x] = make_float4(top[0], sum[0], top[1], sum[1]);
      __syncthreads();
      if (set > 0) return;
      for (int i = 1; i < sets; ++i) take(s_ml[threadIdx.x + i * frags * 32], s_acc[threadIdx.x + i * frags * 32]);
    }
    const float inv[2] = {inverse(top[0], sum[0], v_scale), inverse(top[1], sum[1], v_scale)};
    T* out = reinterpret_cast<T*>(p.a.out) + row * p.a.out_stride + (head0 + nb * 8) * p.a.out_head_stride + f % kSteps * 16;
    store_frag<T, kE4M3>(out, p.a.out_head_stride, heads - nb * 8, lane, make_float4(acc.x * inv[0], acc.y * inv[1], acc.z * inv[0], acc.w * inv[1]));
    if (p.a.lse && f % kSteps == 0 && g == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (h + e < heads) p.a.lse[(long long)row * p.a.heads + head0 + h + e] = (top[e] + log2f(sum[e])) * kLn2;
    }
  }
}

int blocks_of(int group) { return group > 8 ? 2 : 1; }
int items_of(int kv_heads, int group) { return kv_heads * ((group + 8 * blocks_of(group) - 1) / (8 * blocks_of(group))); }
// CTAs of a launch over rows that can be as long as `most`.
long long ctas_of(int rows, int items, int most, int tile, int slots) { return (long long)items * teams_of(rows, items, units_of(most, tile), kWarps, slots); }
int most_seen(int max_len, int window) { return window > 0 && window < max_len ? window : max_len; }

template <int D, typename T, bool kE4M3, int kBlocks>
cudaError_t launch(Params p, void* workspace, int sms, cudaStream_t stream) {
  using L = Tile<D, kE4M3, kBlocks>;
  auto* kernel = k_paged_attention<D, T, kE4M3, kBlocks>;
  cudaError_t rc = kernel_setup(reinterpret_cast<const void*>(kernel), L::kSmem).rc;
  if (rc != cudaSuccess) return rc;
  const long long ctas = ctas_of(p.a.rows, p.items, most_seen(p.max_len, p.a.window), L::kPos, L::kTwo ? 2 * sms : sms);
  if (ctas > 0x7fffffffll) return cudaErrorInvalidValue;
  p.parts = reinterpret_cast<float4*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.parts + ctas * 2 * L::kFrags * 32);
  p.teams = (int)(ctas / p.items);
  p.by_row = p.a.rows < p.teams;
  const dim3 grid((unsigned)p.items, (unsigned)p.teams);
  rc = launch_kernel_ex(kernel, grid, dim3(kWarps * 32), (size_t)L::kSmem, stream, true, 1, p);
  if (rc != cudaSuccess || ctas == p.items) return rc;  // (a single team finishes its rows)
  // Fewer rows than teams: a block for each row, and one for each accumulator where rows are in many parts.  A block for each team, with
  // all accumulators: 1 row of 100000 positions, 4 heads of 1, 296 parts: 37 us, so 18.7; 40 of 20000 at most: 21, so 18.5.  A block for
  // each accumulator where a row has 1 or 2 parts: 32 rows of 2048, 32 heads of 8: 55 us, so 47.5.  Eight parts under way in a warp, or
  // four with fewer registers, where so many blocks have to find room beside the attention's (8 rows of 2048 20.3 us, so 18.2).
  const bool many = p.teams > 4 * p.a.rows, long_rows = p.teams > 16 * p.a.rows;
  const int warps = long_rows ? kJoinThreads / 32 : L::kFrags < 8 && !p.by_row ? L::kFrags : 8;
  return launch_kernel_ex(many && !long_rows ? k_paged_join<D, T, kE4M3, kBlocks, 4> : k_paged_join<D, T, kE4M3, kBlocks, 8>,
                          dim3(grid.x, p.by_row ? p.a.rows : p.teams, many ? L::kFrags : 1), dim3(warps * 32), 0, stream, true, 1, p);
}

}  // namespace

size_t paged_attention_workspace_bytes(int rows, int heads, int kv_heads, int dim, int max_len, int window, int sms) {
  const int group = heads / kv_heads, blocks = blocks_of(group);
  // (of all cache types: the smallest tile, one or two CTAs an SM)
  const int items = items_of(kv_heads, group), most = most_seen(max_len, window);
  const long long one = ctas_of(rows, items, most, 16, sms), two = ctas_of(rows, items, most, 16, 2 * sms);
  const size_t ctas = (size_t)(one > two ? one : two);
  return ctas == (size_t)items ? 0 : ctas * 2 * blocks * ((size_t)(dim / 16) * 512 + 8 * sizeof(float2));
}

cudaError_t launch_paged_attention(const PagedAttention& a, PagedType type, const PagedPool& pool, PagedType cache, void* workspace, int sms,
                                   cudaStream_t stream) {
  if (a.rows < 1 || pool.heads < 1 || a.heads % pool.heads != 0 || a.heads < pool.heads || type == PAGED_E4M3 ||
      (cache != PAGED_E4M3 && cache != type))
    return cudaErrorInvalidValue;
  const long long cap = (long long)a.width * pool.page_size;
  Params p = {};
  p.a = a;
  p.pool = pool;
  p.div = page_div(pool.page_size);
  p.group = a.heads / pool.heads;
  p.max_len = (int)(cap < kMaxLen ? cap : kMaxLen);
  p.items = items_of(pool.heads, p.group);
  p.groups = p.items / pool.heads;
  if ((long long)a.rows * units_of(most_seen(p.max_len, a.window), 16) > kMaxUnits) return cudaErrorInvalidValue;
  const Steps st = steps_of(pool.pages, pool.page_size, pool.page_stride, pool.pos_stride, cache == PAGED_E4M3 ? 1 : 2);
  if (st.bytes == 0 || (unsigned long long)st.pos * st.bytes > 1u << 26) return cudaErrorInvalidValue;  // (a tile's rows are counted in 32 bits of bytes)
  p.page_step = st.page;
  p.pos_step = st.pos;
  p.step_bytes = st.bytes;
#define PENNY_PAGED_ROWS(D, T, E) (p.group <= 8 ? launch<D, T, E, 1>(p, workspace, sms, stream) : launch<D, T, E, 2>(p, workspace, sms, stream))
#define PENNY_PAGED_TYPE(D)                                                                                                   \
  (cache == PAGED_E4M3 ? (type == PAGED_BF16 ? PENNY_PAGED_ROWS(D, __nv_bfloat16, true) : PENNY_PAGED_ROWS(D, __half, true)) \
                       : (type == PAGED_BF16 ? PENNY_PAGED_ROWS(D, __nv_bfloat16, false) : PENNY_PAGED_ROWS(D, __half, false)))
  switch (pool.dim) {
    case 64: return PENNY_PAGED_TYPE(64);
    case 128: return PENNY_PAGED_TYPE(128);
    case 256: return PENNY_PAGED_TYPE(256);
    default: return cudaErrorInvalidValue;
  }
#undef PENNY_PAGED_TYPE
#undef PENNY_PAGED_ROWS
}

}  // namespace penny
