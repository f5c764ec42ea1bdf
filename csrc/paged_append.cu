// Rotary positions of new tokens and their keys and values into the pages of a pool.
//
// A token's row of the projection is [q heads | k heads | v heads] of `dim` values.  q and k are rotated (rotate-half form:
// pair (x[d], x[d + dim / 2]) by the angle position * theta^(-2 d / dim)), in place or into `out`; the rotated k and v
// go to the token's slot.  A slot that the pool does not have (-1: padding, or a token without a page) leaves its row alone.
//
// The angle is taken in turns: position times the pair's frequency over 2 pi in fp64, of which only the fraction goes on to
// fp32 sine and cosine.  In fp32 an angle of 1e5 rad would be off by 4e-3, half of what bf16 resolves.  A token's sines and
// cosines are computed once and shared by its heads.
//
// Bound by memory: every value is read and written once.  A block has a token, a thread two pairs of 16 bytes at a time, the first
// of which are on their way while the angles are computed.  16384 tokens of 32 + 2 * 8 heads of 128 bf16 values: 72 to 74 us,
// 6 TB/s (with the loads behind the angles 88, with four tokens to a block of 448 threads 92); 64 tokens 2.9 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "paged_kernels.h"
#include "paged_plan.h"
#include "pdl.h"

namespace penny {
namespace {

constexpr int kMaxThreads = 256, kMaxHalf = 128, kItems = 2;  // kItems: of a thread at a time

struct Turns {
  double of[kMaxHalf];  // turns per position of every pair
};

__device__ __forceinline__ void unpack(const __nv_bfloat16*, const uint4& r, float (&x)[8]) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(p[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack(const __half*, const uint4& r, float (&x)[8]) {
  const __half2* p = reinterpret_cast<const __half2*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(p[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 pack(const __nv_bfloat16*, const float (&x)[8]) {
  uint4 r;
  __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
  return r;
}
__device__ __forceinline__ uint4 pack(const __half*, const float (&x)[8]) {
  uint4 r;
  __half2* p = reinterpret_cast<__half2*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
  return r;
}

// Two products, and two a b + c, of an instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r, x = *reinterpret_cast<unsigned long long*>(&a), y = *reinterpret_cast<unsigned long long*>(&b);
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r, x = *reinterpret_cast<unsigned long long*>(&a), y = *reinterpret_cast<unsigned long long*>(&b),
                        z = *reinterpret_cast<unsigned long long*>(&c);
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return *reinterpret_cast<float2*>(&r);
}

// x, or +-most where it is past that (NaN stays)
__device__ __forceinline__ float within(float x, float most) {
  float r;
  asm("min.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(most));
  return r;
}

// What values of a head are divided by.  A quotient in fp32 comes from one over the scale and the remainder that an FMA leaves exact, which
// gives the rounded one (Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, 1990) where no step
// leaves fp32's range: scales past 2^+-60 are brought nearer to one, with the values, and of quotients past e4m3's largest only
// that much is taken.  (2047 tokens of 20 heads of 64 8.6 us, with divisions 10.2, times one over the scale 8.1; but
// that puts quotients near the middle of two e4m3 values on the wrong side, and one over a scale under 2^-128 is infinite.)
struct Scale {
  float by, minus, inv;
};
__device__ __forceinline__ Scale scale_of(float scale) {
  const float by = fabsf(scale) < 0x1p-60f ? 0x1p64f : fabsf(scale) > 0x1p60f ? 0x1p-64f : 1.f;
  return {by, -(scale * by), 1.f / (scale * by)};
}

// Eight values to the pool: as they are, or e4m3 of value over scale (rounded from fp32, values past +-448 to that).
template <typename T, bool kE4M3>
__device__ __forceinline__ void store8(void* pool, long long at, const float (&x)[8], const Scale& s) {
  if constexpr (kE4M3) {
    uint2 r;
    __nv_fp8x2_storage_t* p = reinterpret_cast<__nv_fp8x2_storage_t*>(&r);
    const float2 inv = make_float2(s.inv, s.inv), minus = make_float2(s.minus, s.minus);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 v = make_float2(x[2 * i], x[2 * i + 1]);
      if (s.by != 1.f) v.x *= s.by, v.y *= s.by;
      float2 q = mul2(v, inv);
      q = make_float2(within(q.x, 512.f), within(q.y, 512.f));
      p[i] = __nv_cvt_float2_to_fp8x2(fma2(fma2(q, minus, v), inv, q), __NV_SATFINITE, __NV_E4M3);
    }
    *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(pool) + at) = r;
  } else {
    *reinterpret_cast<uint4*>(reinterpret_cast<T*>(pool) + at) = pack((const T*)nullptr, x);
  }
}

// (64 registers, so that an SM holds eight blocks of 128 threads: 2047 tokens, e4m3, 8.6 us, with 73 registers 10.4)
template <typename T, bool kE4M3>
__global__ void __launch_bounds__(kMaxThreads, 4) k_paged_append(T* qkv, long long qkv_stride, T* out, long long out_stride, const PagedPool pool,
                                                              const long long* slots, const int* positions, int heads, int items, bool early,
                                                              const paged::PageDiv by_vec, const __grid_constant__ Turns turns) {
  __shared__ float2 s_rot[kMaxHalf];  // cosine, sine: the first pairs of all vectors, the second ones, ... (no two lanes on one bank)
  pdl_launch_dependents();
  if (!early) pdl_wait();
  // work items: pairs of 8 values of the q and k heads, then pairs of 8 values of the v heads
  const int half = pool.dim / 2, vecs = half / 8, tid = threadIdx.x, threads = blockDim.x;
  T* const row = qkv + blockIdx.x * qkv_stride;
  struct Item {
    int h, d;  // head of the row, first value
    uint4 a, b;
  } it[kItems];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const int i = i0 + u * threads;
      if (i >= items) break;
      it[u].h = paged::div_page(by_vec, i);
      it[u].d = (i - it[u].h * vecs) * 8;
      const T* x = row + it[u].h * pool.dim + it[u].d;
      it[u].a = *reinterpret_cast<const uint4*>(x);
      it[u].b = *reinterpret_cast<const uint4*>(x + half);
    }
  };
  if (!early) fetch(tid);
  const long long at = paged::place_of_slot(slots[blockIdx.x], pool.pages, pool.page_size, pool.page_stride, pool.pos_stride);
  if (at >= 0) {
    for (int d = tid; d < half; d += threads) {
      const double x = (double)positions[blockIdx.x] * turns.of[d];
      float sn, cs;
      sincospif(2.0f * (float)(x - rint(x)), &sn, &cs);
      s_rot[(d & 7) * vecs + (d >> 3)] = make_float2(cs, sn);
    }
  }
  if (early) {
    pdl_wait();
    fetch(tid);
  }
  __syncthreads();
  if (at < 0) return;
  for (int i0 = tid; i0 < items; i0 += kItems * threads) {
    if (i0 != tid) fetch(i0);
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      if (i0 + u * threads >= items) break;
      const int h = it[u].h, d = it[u].d;
      const bool turned = h < heads + pool.heads;
      float a[8], b[8];
      unpack((const T*)nullptr, it[u].a, a);
      unpack((const T*)nullptr, it[u].b, b);
      if (turned) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 cs = s_rot[j * vecs + (d >> 3)];
          const float x = a[j], y = b[j];
          a[j] = x * cs.x - y * cs.y;
          b[j] = y * cs.x + x * cs.y;
        }
        T* y = out + blockIdx.x * out_stride + h * pool.dim + d;
        *reinterpret_cast<uint4*>(y) = pack((const T*)nullptr, a);
        *reinterpret_cast<uint4*>(y + half) = pack((const T*)nullptr, b);
        if (h < heads) continue;
      }
      const int kh = h - heads - (turned ? 0 : pool.heads);
      const Scale scale = kE4M3 ? scale_of((turned ? pool.k_scale : pool.v_scale)[kh]) : Scale{};
      void* const to = turned ? pool.k : pool.v;
      store8<T, kE4M3>(to, at + kh * pool.head_stride + d, a, scale);
      store8<T, kE4M3>(to, at + kh * pool.head_stride + d + half, b, scale);
    }
  }
}

template <typename T, bool kE4M3>
cudaError_t launch(void* qkv, long long qkv_stride, void* out, long long out_stride, const PagedPool& pool, const long long* slots,
                   const int* positions, int tokens, int heads, double theta, bool early, cudaStream_t stream) {
  Turns turns;
  const double step = std::pow(theta, -2.0 / pool.dim);
  double f = 0.15915494309189533577;  // 1 / (2 pi)
  for (int d = 0; d < pool.dim / 2; ++d, f *= step) turns.of[d] = f;
  const int items = (heads + 2 * pool.heads) * (pool.dim / 16);
  // few tokens: as many threads as have work (64 tokens of 448 items: 2.5 us with 224 threads, 3.0 with 128); many: small blocks, of
  // which an SM holds more (16384 tokens 3 % less time)
  const int most = tokens >= 148 * 8 ? 128 : kMaxThreads, threads = std::min(most, (items + 32 * kItems - 1) / (32 * kItems) * 32);
  return launch_kernel_ex(k_paged_append<T, kE4M3>, dim3(tokens), dim3(threads), 0, stream, true, 1, (T*)qkv, qkv_stride, (T*)(out ? out : qkv),
                          out ? out_stride : qkv_stride, pool, slots, positions, heads, items, early, paged::page_div(pool.dim / 16), turns);
}

}  // namespace

cudaError_t launch_paged_append(void* qkv, long long qkv_stride, void* out, long long out_stride, PagedType type, const PagedPool& pool,
                                PagedType cache, const long long* slots, const int* positions, int tokens, int heads, double theta,
                                bool early, cudaStream_t stream) {
  if (pool.dim < 16 || pool.dim > 2 * kMaxHalf || pool.dim % 16 != 0 || heads < 0 || pool.heads < 1 || !(theta > 0) || type == PAGED_E4M3 ||
      (cache != PAGED_E4M3 && cache != type))
    return cudaErrorInvalidValue;
  if (tokens < 1) return cudaSuccess;
#define PENNY_PAGED_APPEND(T, E) launch<T, E>(qkv, qkv_stride, out, out_stride, pool, slots, positions, tokens, heads, theta, early, stream)
  if (type == PAGED_BF16)
    return cache == PAGED_E4M3 ? PENNY_PAGED_APPEND(__nv_bfloat16, true) : PENNY_PAGED_APPEND(__nv_bfloat16, false);
  return cache == PAGED_E4M3 ? PENNY_PAGED_APPEND(__half, true) : PENNY_PAGED_APPEND(__half, false);
#undef PENNY_PAGED_APPEND
}

}  // namespace penny
