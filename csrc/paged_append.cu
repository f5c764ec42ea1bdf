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
// Bound by memory: every value is read and written once, 16 bytes a thread.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <stdint.h>

#include <cmath>

#include "paged_kernels.h"
#include "paged_plan.h"
#include "pdl.h"

namespace penny {
namespace {

constexpr int kThreads = 256, kMaxHalf = 128, kTokens = 4;

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

// Eight values to the pool: as they are, or e4m3 of value / scale (rounded once from fp32, values past +-448 to that).
template <typename T, bool kE4M3>
__device__ __forceinline__ void store8(void* pool, long long at, const float (&x)[8], float scale) {
  if constexpr (kE4M3) {
    uint2 r;
    __nv_fp8x2_storage_t* p = reinterpret_cast<__nv_fp8x2_storage_t*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      p[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i] / scale, x[2 * i + 1] / scale), __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(pool) + at) = r;
  } else {
    *reinterpret_cast<uint4*>(reinterpret_cast<T*>(pool) + at) = pack((const T*)nullptr, x);
  }
}

template <typename T, bool kE4M3>
__global__ void __launch_bounds__(kThreads) k_paged_append(T* qkv, long long qkv_stride, T* out, long long out_stride, const PagedPool pool,
                                                           const long long* slots, const int* positions, int tokens, int per, int heads,
                                                           const __grid_constant__ Turns turns) {
  __shared__ float2 s_rot[kTokens * kMaxHalf];  // cosine, sine
  __shared__ long long s_at[kTokens];           // the token's place in the pool, -1: none
  pdl_launch_dependents();
  pdl_wait();
  const int t0 = blockIdx.x * per, n = min(per, tokens - t0), half = pool.dim / 2;
  for (int i = threadIdx.x; i < n * half; i += kThreads) {
    const int t = i / half, d = i - t * half;
    const double x = (double)positions[t0 + t] * turns.of[d];
    float sn, cs;
    sincospif(2.0f * (float)(x - rint(x)), &sn, &cs);
    s_rot[t * kMaxHalf + d] = make_float2(cs, sn);
  }
  if (threadIdx.x < n) {
    s_at[threadIdx.x] = paged::place_of_slot(slots[t0 + threadIdx.x], pool.pages, pool.page_size, pool.page_stride, pool.pos_stride);
  }
  __syncthreads();
  // work items of a token: pairs of 8 values of the q and k heads, then 8 values of the v heads
  const int vecs = half / 8, turned = (heads + pool.heads) * vecs, items = turned + pool.heads * vecs * 2;
  for (int i = threadIdx.x; i < n * items; i += kThreads) {
    const int t = i / items, w = i - t * items;
    const long long at = s_at[t];
    if (at < 0) continue;
    T* row = qkv + (t0 + t) * qkv_stride;
    if (w < turned) {
      const int h = w / vecs, d = (w - h * vecs) * 8;
      const T* x = row + h * pool.dim + d;
      float a[8], b[8], ra[8], rb[8];
      unpack((const T*)nullptr, *reinterpret_cast<const uint4*>(x), a);
      unpack((const T*)nullptr, *reinterpret_cast<const uint4*>(x + half), b);
      const float2* rot = s_rot + t * kMaxHalf + d;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 cs = rot[j];
        ra[j] = a[j] * cs.x - b[j] * cs.y;
        rb[j] = b[j] * cs.x + a[j] * cs.y;
      }
      T* y = out + (t0 + t) * out_stride + h * pool.dim + d;
      *reinterpret_cast<uint4*>(y) = pack((const T*)nullptr, ra);
      *reinterpret_cast<uint4*>(y + half) = pack((const T*)nullptr, rb);
      if (h >= heads) {
        const int kh = h - heads;
        const float scale = kE4M3 ? pool.k_scale[kh] : 1.f;
        store8<T, kE4M3>(pool.k, at + kh * pool.head_stride + d, ra, scale);
        store8<T, kE4M3>(pool.k, at + kh * pool.head_stride + d + half, rb, scale);
      }
    } else {
      const int u = w - turned, kh = u / (2 * vecs), d = (u - kh * 2 * vecs) * 8;
      float x[8];
      unpack((const T*)nullptr, *reinterpret_cast<const uint4*>(row + (heads + pool.heads + kh) * pool.dim + d), x);
      store8<T, kE4M3>(pool.v, at + kh * pool.head_stride + d, x, kE4M3 ? pool.v_scale[kh] : 1.f);
    }
  }
}

template <typename T, bool kE4M3>
cudaError_t launch(void* qkv, long long qkv_stride, void* out, long long out_stride, const PagedPool& pool, const long long* slots,
                   const int* positions, int tokens, int heads, double theta, cudaStream_t stream) {
  Turns turns;
  const double step = std::pow(theta, -2.0 / pool.dim);
  double f = 0.15915494309189533577;  // 1 / (2 pi)
  for (int d = 0; d < pool.dim / 2; ++d, f *= step) turns.of[d] = f;
  const int per = tokens >= 148 * 8 * kTokens ? kTokens : 1;
  return launch_kernel_ex(k_paged_append<T, kE4M3>, dim3((tokens + per - 1) / per), dim3(kThreads), 0, stream, true, 1, (T*)qkv, qkv_stride,
                          (T*)(out ? out : qkv), out ? out_stride : qkv_stride, pool, slots, positions, tokens, per, heads, turns);
}

}  // namespace

cudaError_t launch_paged_append(void* qkv, long long qkv_stride, void* out, long long out_stride, PagedType type, const PagedPool& pool,
                                PagedType cache, const long long* slots, const int* positions, int tokens, int heads, double theta,
                                cudaStream_t stream) {
  if (pool.dim < 16 || pool.dim > 2 * kMaxHalf || pool.dim % 16 != 0 || heads < 0 || pool.heads < 1 || !(theta > 0) || type == PAGED_E4M3 ||
      (cache != PAGED_E4M3 && cache != type))
    return cudaErrorInvalidValue;
  if (tokens < 1) return cudaSuccess;
#define PENNY_PAGED_APPEND(T, E) launch<T, E>(qkv, qkv_stride, out, out_stride, pool, slots, positions, tokens, heads, theta, stream)
  if (type == PAGED_BF16)
    return cache == PAGED_E4M3 ? PENNY_PAGED_APPEND(__nv_bfloat16, true) : PENNY_PAGED_APPEND(__nv_bfloat16, false);
  return cache == PAGED_E4M3 ? PENNY_PAGED_APPEND(__half, true) : PENNY_PAGED_APPEND(__half, false);
#undef PENNY_PAGED_APPEND
}

}  // namespace penny
