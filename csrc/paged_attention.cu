// Attention of one new token per sequence over a paged KV cache.
//
//   o[b, h] = sum_j softmax_j(scale * q[b, h] . K_j) V_j,  j in the last `window` of lengths[b] positions (all without one),
// position j in the pool's page table[b, j / page_size] at j % page_size.  One pass over K and V with a running maximum and sum
// (fp32); lse = the logarithm of the sum.  Rows without positions: zeros, -inf.  Positions on a page that the pool does not
// have count as not there.
//
//   * The heads of a KV head share its keys and values: G = Hq / Hkv query rows are the M side of mma.sync (m16n8k16), whose
//     second eight rows stay empty up to G = 8; more than 16 go to several CTAs.  (The 128 rows of a tcgen05 tile would be
//     empty; the bound is the cache's stream.)
//   * A CTA is four warps, each with a private three-stage cp.async pipeline over tiles of 4 KB of K and 4 KB of V (16
//     positions of 128 bf16 values).  A lane looks up one position's page a tile ahead, so any page size and any strides will
//     do; what lies outside the row is filled with zeros and never read (stale rows may hold anything).
//   * e4m3 caches: fp16 is exact for them, so they meet q as fp16, each row of q divided by the power of two of its
//     largest value (exact; the score's factor takes it back).  A lane's four bytes of K are two adjacent pairs: the dims inside a
//     16-byte chunk are permuted on both sides of the product.  V's bytes are transposed in pairs by ldmatrix and separated
//     into even and odd dims.
//   * P is rounded to the type of the product (bf16: 2^-8 of each weight at most, averaged over the positions; the sum is of the
//     unrounded ones); q, scores, maxima and sums are not rounded.
//   * Rows are cut into pieces of the batch's total over the CTAs that the GPU holds (paged_plan.h), found by every CTA from the
//     lengths on the device.  A second kernel joins the pieces of cut rows; no counters, so a workspace holds nothing between
//     calls.
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

constexpr int kWarps = 4, kStages = 3;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int D, bool kE4M3>
struct Tile {
  static constexpr int kRow = kE4M3 ? D : 2 * D;               // bytes of a position
  static constexpr int kPos = 4096 / kRow > 16 ? 4096 / kRow : 16;
  static constexpr int kChunks = kRow / 16;                    // 16-byte chunks of a position
  static constexpr int kPerPass = 32 / kChunks;                // positions that a warp's 32 chunks cover
  static constexpr int kStage = 2 * kPos * kRow;
  static constexpr int kSmem = kWarps * kStages * kStage;
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

struct Cut {   // where a CTA's piece comes from and goes to
  int row, item, piece, pieces;
};
// Meta of the joining kernel: the CTA of a row's first piece of item 0, and how many pieces the row has.
struct Params {
  PagedAttention a;
  PagedPool pool;
  PageDiv div;
  int group;           // G
  int items_per_row;   // (KV head, head group) pairs of a row
  int max_len, slots;  // slots 0: rows are whole
  int2* meta;
  float* part_o;   // per piece kRows rows of dim
  float2* part_ml; // maximum (base 2), sum
};

// The piece of CTA `idx`.  Called by all threads; row -1: none.
__device__ __forceinline__ Cut find_cut(const Params& p, int idx) {
  __shared__ long long s_sum[kWarps];
  __shared__ int s_cnt[kWarps];
  __shared__ Cut s_cut;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = (p.a.rows + kWarps * 32 - 1) / (kWarps * 32), r0 = min(p.a.rows, tid * per), r1 = min(p.a.rows, r0 + per);
  auto seen = [&](int r) {
    const Seen s = seen_of(p.a.lengths[r], p.max_len, p.a.window);
    return s.end - s.first;
  };
  long long sum = 0;
  for (int r = r0; r < r1; ++r) sum += seen(r);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_sum[warp] = sum;
  if (tid == 0) s_cut.row = -1;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += s_sum[w];
  const int len = piece_len(total, p.items_per_row, p.slots);
  int mine = 0;
  for (int r = r0; r < r1; ++r) mine += pieces_of(seen(r), len);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_cnt[warp] = incl;
  __syncthreads();
  int first = incl - mine;
  for (int w = 0; w < warp; ++w) first += s_cnt[w];
  long long at = idx - (long long)first * p.items_per_row;
  if (at >= 0 && at < (long long)mine * p.items_per_row) {
    for (int r = r0; r < r1; ++r) {
      const int n = pieces_of(seen(r), len);
      if (at < (long long)n * p.items_per_row) {
        const int piece = (int)at / p.items_per_row;
        s_cut = {r, (int)at - piece * p.items_per_row, piece, n};
        break;
      }
      at -= (long long)n * p.items_per_row;
    }
  }
  __syncthreads();
  return s_cut;
}

// kRows: query rows of a CTA, 8 or 16.
template <int D, typename T, bool kE4M3, int kRows>
__global__ void __launch_bounds__(kWarps * 32) k_paged_attention(const __grid_constant__ Params p) {
  using L = Tile<D, kE4M3>;
  using T2 = typename Pair<T>::type;
  constexpr int kHalves = kRows / 8, kLook = (L::kPos + 31) / 32, kSteps = D / 16, kNC = L::kPos / 8;
  constexpr bool kBf16 = !kE4M3 && sizeof(T2) == 4 && __is_same(T, __nv_bfloat16);
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  pdl_launch_dependents();
  pdl_wait();
  Cut cut;
  if (p.slots > 0) {
    cut = find_cut(p, (int)blockIdx.x);
    if (cut.row < 0) return;
  } else {
    cut.row = (int)blockIdx.x / p.items_per_row;
    cut.item = (int)blockIdx.x - cut.row * p.items_per_row;
    cut.piece = 0;
    cut.pieces = 1;
  }
  const int b = cut.row, groups = (p.group + kRows - 1) / kRows, kh = cut.item / groups, h0 = (cut.item - kh * groups) * kRows;
  const int heads = min(kRows, p.group - h0);  // valid rows of this CTA
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (p.slots > 0 && cut.piece == 0 && cut.item == 0 && threadIdx.x == 0) p.meta[b] = make_int2((int)blockIdx.x, cut.pieces);

  const Seen seen = seen_of(p.a.lengths[b], p.max_len, p.a.window);
  const int n = seen.end - seen.first;
  const int per = ((n + cut.pieces - 1) / cut.pieces + L::kPos - 1) / L::kPos * L::kPos;
  const int t0 = (int)min((long long)seen.first + (long long)cut.piece * per, (long long)seen.end), t1 = min(seen.end, t0 + min(per, n));
  const int tiles = (t1 - t0 + L::kPos - 1) / L::kPos;
  const uint32_t wbase = attn::smem_u32_local(smem_raw) + warp * (kStages * L::kStage);
  const int* table = p.a.table + (long long)b * p.a.table_stride;
  constexpr int kSize = kE4M3 ? 1 : 2;
  const char* kbase = reinterpret_cast<const char*>(p.pool.k) + kh * p.pool.head_stride * kSize + (lane % L::kChunks) * 16;
  const char* vbase = reinterpret_cast<const char*>(p.pool.v) + kh * p.pool.head_stride * kSize + (lane % L::kChunks) * 16;
  const long long page_bytes = p.pool.page_stride * kSize, pos_bytes = p.pool.pos_stride * kSize;

  // tile j of this warp: positions [t0 + (warp + 4 j) kPos, + kPos).  The page of this lane's position(s), -1: not there.
  int page[kLook];
  auto look = [&](int j) {
    const int start = t0 + (warp + kWarps * j) * L::kPos;
#pragma unroll
    for (int i = 0; i < kLook; ++i) {
      const int pos = start + i * 32 + lane;
      page[i] = i * 32 + lane < L::kPos && warp + kWarps * j < tiles && pos < t1 ? table[div_page(p.div, pos)] : -1;
    }
  };
  // requests tile j; the mask of its positions that are there
  auto issue = [&](int j) {
    unsigned long long mask = 0;
    if (warp + kWarps * j < tiles) {
      const int start = t0 + (warp + kWarps * j) * L::kPos;
      const uint32_t sb = wbase + (j % kStages) * L::kStage;
      long long off[kLook];
#pragma unroll
      for (int i = 0; i < kLook; ++i) {
        const int pos = start + i * 32 + lane;
        off[i] = place_of(page[i], p.pool.pages, pos, p.div, page_bytes, pos_bytes);
        mask |= (unsigned long long)__ballot_sync(0xffffffffu, off[i] >= 0) << (32 * i);
      }
#pragma unroll
      for (int i = 0; i < L::kPos / L::kPerPass; ++i) {
        const int r = i * L::kPerPass + lane / L::kChunks;
        const long long o = __shfl_sync(0xffffffffu, off[(i * L::kPerPass) / 32], r & 31);
        const uint32_t s = sb + L::at(r, lane % L::kChunks);
        cp_async16(s, kbase + (o < 0 ? 0 : o), o >= 0);
        cp_async16(s + L::kPos * L::kRow, vbase + (o < 0 ? 0 : o), o >= 0);
      }
    }
    cp_async_commit();  // always: keeps the group count in step with j
    return mask;
  };
  look(0);
  unsigned long long mask0 = issue(0);
  look(1);
  unsigned long long mask1 = issue(1);
  look(2);

  // ---- q as MMA A fragments, and what turns a score into the exponent of two ----
  uint32_t qa[kSteps][2 * kHalves];
  float qs[kHalves];
#pragma unroll
  for (int r = 0; r < kHalves; ++r) {
    const int h = r * 8 + g;
    const T* q = reinterpret_cast<const T*>(p.a.q) + b * p.a.q_stride + (long long)(kh * p.group + h0 + min(h, heads - 1)) * p.a.q_head_stride;
    qs[r] = p.a.scale * kLog2e;
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
      const int e = (__float_as_int(top) >> 23) & 255;
      const bool plain = e < 1 || e > 253;  // zeros, infinities
      const float down = plain ? 1.f : __int_as_float((254 - e) << 23);
      qs[r] *= p.pool.k_scale[kh] * (plain ? 1.f : __int_as_float(e << 23));
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        qa[k][r] = pack_f16(x[k][0] * down, x[k][1] * down);
        qa[k][kHalves + r] = pack_f16(x[k][2] * down, x[k][3] * down);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        qa[k][r] = *reinterpret_cast<const uint32_t*>(q + k * 16 + 2 * t);
        qa[k][kHalves + r] = *reinterpret_cast<const uint32_t*>(q + k * 16 + 8 + 2 * t);
      }
    }
  }
  auto mma = [&](float (&d)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {  // a: row g (and g + 8), k low, then k high
    const uint32_t a1 = kHalves == 2 ? a[1] : 0u, a2 = a[kHalves], a3 = kHalves == 2 ? a[3] : 0u;
    if constexpr (kBf16) mma_bf16(d, a[0], a1, a2, a3, b0, b1);
    else mma_f16(d, a[0], a1, a2, a3, b0, b1);
  };
  auto pack_p = [&](float lo, float hi) {
    if constexpr (kBf16) return attn::pack2(lo, hi);
    else return pack_f16(lo, hi);
  };

  float m[kHalves], l[kHalves], o[D / 8][4];
#pragma unroll
  for (int r = 0; r < kHalves; ++r) m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  const int my_tiles = tiles > warp ? (tiles - warp + kWarps - 1) / kWarps : 0;
  for (int j = 0; j < my_tiles; ++j) {
    __syncwarp();  // everyone is done with the stage that tile j + 2 overwrites
    const unsigned long long mask2 = issue(j + 2);
    look(j + 3);
    cp_async_wait<2>();
    __syncwarp();
    const uint32_t sb = wbase + (j % kStages) * L::kStage;
    // ---- S = Q K^T, eight positions at a time ----
    float s[kNC][4];
#pragma unroll
    for (int c = 0; c < kNC; ++c) {
      s[c][0] = s[c][1] = s[c][2] = s[c][3] = 0.f;
#pragma unroll
      for (int k4 = 0; k4 < L::kChunks / 4; ++k4) {
        uint32_t kb[4];
        ldmatrix_x4(sb + L::at(c * 8 + (lane & 7), k4 * 4 + (lane >> 3)), kb);
        if constexpr (kE4M3) {
#pragma unroll
          for (int i = 0; i < 4; ++i) mma(s[c], qa[k4 * 4 + i], e4m3_lo(kb[i]), e4m3_hi(kb[i]));
        } else {
          mma(s[c], qa[k4 * 2], kb[0], kb[1]);
          mma(s[c], qa[k4 * 2 + 1], kb[2], kb[3]);
        }
      }
    }
    // ---- running softmax; this thread holds positions c * 8 + 2 t, + 1 of rows g and g + 8 ----
    uint32_t pa[kNC / 2][2 * kHalves];
#pragma unroll
    for (int r = 0; r < kHalves; ++r) {
      float top = m[r];
#pragma unroll
      for (int c = 0; c < kNC; ++c) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = s[c][2 * r + e];
          x = (mask0 >> (c * 8 + 2 * t + e)) & 1 ? x * qs[r] : -INFINITY;
          top = fmaxf(top, x);
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float base = top == -INFINITY ? 0.f : top;  // nothing there yet: weights of zero
      const float corr = exp2f(m[r] - base);
      m[r] = top;
      l[r] *= corr;
#pragma unroll
      for (int c = 0; c < kNC; ++c) {
        const float p0 = exp2f(s[c][2 * r] - base), p1 = exp2f(s[c][2 * r + 1] - base);
        l[r] += p0 + p1;
        pa[c / 2][(c & 1) * kHalves + r] = pack_p(p0, p1);
      }
#pragma unroll
      for (int i = 0; i < D / 8; ++i) o[i][2 * r] *= corr, o[i][2 * r + 1] *= corr;
    }
    // ---- O += P V, 16 positions at a time ----
#pragma unroll
    for (int c = 0; c < kNC / 2; ++c) {
      const int row = c * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
      for (int d = 0; d < L::kChunks / 2; ++d) {
        uint32_t vb[4];
        ldmatrix_x4_trans(sb + L::kPos * L::kRow + L::at(row, d * 2 + (lane >> 4)), vb);
        if constexpr (kE4M3) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t x = __byte_perm(vb[2 * i], 0, 0x3120), y = __byte_perm(vb[2 * i + 1], 0, 0x3120);
            mma(o[(d * 2 + i) * 2], pa[c], e4m3_lo(x), e4m3_lo(y));
            mma(o[(d * 2 + i) * 2 + 1], pa[c], e4m3_hi(x), e4m3_hi(y));
          }
        } else {
          mma(o[2 * d], pa[c], vb[0], vb[1]);
          mma(o[2 * d + 1], pa[c], vb[2], vb[3]);
        }
      }
    }
    mask0 = mask1;
    mask1 = mask2;
  }
  cp_async_wait<0>();

  // ---- the four warps' sums join in shared memory (the pipelines' space) ----
  __syncthreads();
  float* sm_o = reinterpret_cast<float*>(smem_raw);             // [warps][kRows][D]
  float2* sm_ml = reinterpret_cast<float2*>(sm_o + kWarps * kRows * D);  // [warps][kRows]
#pragma unroll
  for (int r = 0; r < kHalves; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int h = warp * kRows + r * 8 + g;
    if (r * 8 + g < heads) {
      float* to = sm_o + h * D;
      if constexpr (kE4M3) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          *reinterpret_cast<float4*>(to + i * 16 + 4 * t) =
              make_float4(o[2 * i][2 * r], o[2 * i + 1][2 * r], o[2 * i][2 * r + 1], o[2 * i + 1][2 * r + 1]);
      } else {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) *reinterpret_cast<float2*>(to + i * 8 + 2 * t) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
      }
      if (t == 0) sm_ml[h] = make_float2(m[r], l[r]);
    }
  }
  __syncthreads();
  const float v_scale = kE4M3 ? p.pool.v_scale[kh] : 1.f;
  for (int i = threadIdx.x; i < heads * (D / 4); i += kWarps * 32) {
    const int h = i / (D / 4), d = (i - h * (D / 4)) * 4;
    float top = -INFINITY, sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_ml[w * kRows + h].x);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 ml = sm_ml[w * kRows + h];
      const float4 v = *reinterpret_cast<const float4*>(sm_o + (w * kRows + h) * D + d);
      const float f = exp2f(ml.x - base);
      sum += f * ml.y;
      acc[0] += f * v.x, acc[1] += f * v.y, acc[2] += f * v.z, acc[3] += f * v.w;
    }
    if (cut.pieces == 1) {
      const int head = kh * p.group + h0 + h;
      const float inv = top == -INFINITY ? 0.f : v_scale / sum;
      const uint2 raw = make_uint2(Pair<T>::pack(acc[0] * inv, acc[1] * inv), Pair<T>::pack(acc[2] * inv, acc[3] * inv));
      *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.a.out) + b * p.a.out_stride + head * p.a.out_head_stride + d) = raw;
      if (d == 0 && p.a.lse) p.a.lse[(long long)b * p.a.heads + head] = (top + log2f(sum)) * kLn2;
    } else {
      const long long slot = (long long)blockIdx.x * kRows + h;
      *reinterpret_cast<float4*>(p.part_o + slot * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (d == 0) p.part_ml[slot] = make_float2(top, sum);
    }
  }
}

// Joins the pieces of a cut row: a CTA per (row, query head), D / 4 threads per piece, 512 / D pieces at a time.
template <int D, typename T, bool kE4M3, int kRows>
__global__ void __launch_bounds__(128) k_paged_join(const __grid_constant__ Params p) {
  constexpr int kLanes = D / 4, kSets = 128 / kLanes;
  __shared__ float4 s_o[128];
  __shared__ float2 s_ml[kSets];
  pdl_launch_dependents();
  pdl_wait();
  const int b = (int)blockIdx.x / p.a.heads, head = (int)blockIdx.x - b * p.a.heads;
  const int2 meta = p.meta[b];
  if (meta.y == 1) return;
  const int groups = (p.group + kRows - 1) / kRows, kh = head / p.group, hg = (head - kh * p.group) / kRows;
  const int h = head - kh * p.group - hg * kRows;
  const int set = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  auto slot_of = [&](int i) { return ((long long)meta.x + i * p.items_per_row + kh * groups + hg) * kRows + h; };
  float top = -INFINITY, sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = set; i0 < meta.y; i0 += 4 * kSets) {
    float2 ml[4];
    float4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * kSets;
      ml[u] = i < meta.y ? p.part_ml[slot_of(i)] : make_float2(-INFINITY, 0.f);
      v[u] = i < meta.y ? *reinterpret_cast<const float4*>(p.part_o + slot_of(i) * D + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float next = top;
#pragma unroll
    for (int u = 0; u < 4; ++u) next = fmaxf(next, ml[u].x);
    const float base = next == -INFINITY ? 0.f : next, corr = exp2f(top - base);
    sum *= corr;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= corr;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float f = exp2f(ml[u].x - base);
      sum += f * ml[u].y;
      acc[0] += f * v[u].x, acc[1] += f * v[u].y, acc[2] += f * v[u].z, acc[3] += f * v[u].w;
    }
    top = next;
  }
  s_o[threadIdx.x] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  if (lane == 0) s_ml[set] = make_float2(top, sum);
  __syncthreads();
  if (set > 0) return;
  top = -INFINITY, sum = 0.f, acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
#pragma unroll
  for (int i = 0; i < kSets; ++i) top = fmaxf(top, s_ml[i].x);
  const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int i = 0; i < kSets; ++i) {
    const float f = exp2f(s_ml[i].x - base);
    const float4 v = s_o[i * kLanes + lane];
    sum += f * s_ml[i].y;
    acc[0] += f * v.x, acc[1] += f * v.y, acc[2] += f * v.z, acc[3] += f * v.w;
  }
  const float inv = top == -INFINITY ? 0.f : (kE4M3 ? p.pool.v_scale[kh] : 1.f) / sum;
  const uint2 raw = make_uint2(Pair<T>::pack(acc[0] * inv, acc[1] * inv), Pair<T>::pack(acc[2] * inv, acc[3] * inv));
  *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.a.out) + b * p.a.out_stride + head * p.a.out_head_stride + lane * 4) = raw;
  if (lane == 0 && p.a.lse) p.a.lse[(long long)b * p.a.heads + head] = (top + log2f(sum)) * kLn2;
}

struct Shape {
  int rows, items_per_row;
  long long items, extra;
};
Shape shape_of(int batch, int heads, int kv_heads, int max_len, int window, int slots) {
  Shape s;
  const int group = heads / kv_heads;
  s.rows = group > 8 ? 16 : 8;
  s.items_per_row = kv_heads * ((group + s.rows - 1) / s.rows);
  s.items = (long long)batch * s.items_per_row;
  s.extra = extra_pieces(batch, s.items_per_row, slots, window > 0 && window < max_len ? window : max_len);
  return s;
}
size_t round16(size_t n) { return (n + 15) / 16 * 16; }

template <int D, typename T, bool kE4M3, int kRows>
cudaError_t launch(Params p, const Shape& s, cudaStream_t stream) {
  auto* kernel = k_paged_attention<D, T, kE4M3, kRows>;
  constexpr int smem = Tile<D, kE4M3>::kSmem;
  static_assert(smem >= kWarps * kRows * (D * 4 + 8), "the join of the warps fits the pipelines' space");
  cudaError_t rc = kernel_setup(reinterpret_cast<const void*>(kernel), smem).rc;
  if (rc != cudaSuccess) return rc;
  rc = launch_kernel_ex(kernel, dim3((unsigned)(s.items + s.extra)), dim3(kWarps * 32), (size_t)smem, stream, true, 1, p);
  if (rc != cudaSuccess || s.extra == 0) return rc;
  return launch_kernel_ex(k_paged_join<D, T, kE4M3, kRows>, dim3((unsigned)p.a.rows * p.a.heads), dim3(128), 0, stream, true, 1, p);
}

}  // namespace

size_t paged_attention_workspace_bytes(int rows, int heads, int kv_heads, int dim, int max_len, int window, int sms) {
  const Shape s = shape_of(rows, heads, kv_heads, max_len, window, 2 * sms);
  if (s.extra == 0) return 0;
  const size_t parts = (size_t)(s.items + s.extra) * s.rows;
  return round16(rows * sizeof(int2)) + parts * (dim * sizeof(float) + sizeof(float2));
}

cudaError_t launch_paged_attention(const PagedAttention& a, PagedType type, const PagedPool& pool, PagedType cache, void* workspace, int sms,
                                   cudaStream_t stream) {
  if (a.rows < 1 || pool.heads < 1 || a.heads % pool.heads != 0 || a.heads < pool.heads || type == PAGED_E4M3 ||
      (cache != PAGED_E4M3 && cache != type))
    return cudaErrorInvalidValue;
  const long long cap = (long long)a.width * pool.page_size;
  Params p;
  p.a = a;
  p.pool = pool;
  p.div = page_div(pool.page_size);
  p.group = a.heads / pool.heads;
  p.max_len = (int)(cap < 0x7fff0000ll ? cap : 0x7fff0000ll);
  const int slots = 2 * sms;
  const Shape s = shape_of(a.rows, a.heads, pool.heads, p.max_len, a.window, slots);
  if (s.items + s.extra > 0x7fffffffll || (long long)a.rows * a.heads > 0x7fffffffll) return cudaErrorInvalidValue;
  p.items_per_row = s.items_per_row;
  p.slots = s.extra > 0 ? slots : 0;
  p.meta = reinterpret_cast<int2*>(workspace);
  p.part_o = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + round16(a.rows * sizeof(int2)));
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (size_t)(s.items + s.extra) * s.rows * pool.dim);
#define PENNY_PAGED_ROWS(D, T, E) (s.rows == 8 ? launch<D, T, E, 8>(p, s, stream) : launch<D, T, E, 16>(p, s, stream))
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
