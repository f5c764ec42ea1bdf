// Log probabilities of given tokens under the softmax of their logits, its entropy, and its likeliest tokens.
//
// With m a logit of the row, Z = sum exp(x - m):  log p(t) = x_t - m - log Z,  entropy = log Z - (sum exp(x - m) (x - m)) / Z.
// One pass over the logits: every thread keeps the two sums (fp32) against the largest of its first values, or one that it has met since
// and that is over e^8 times as likely, and scales them then; threads, warps and the CTAs of a row's cluster are joined against the larger of two.  So
// m is the row's largest logit or one up to 8 below it.  (No log p is above zero for that, nor an entropy below: where m is not the largest, it keeps
// every p under 1 / (1 + e^-8), far more than two roundings from one.)  The sums are taken of x - m and not of x, so that an
// fp32 logit loses nothing against a far maximum.
//
// The likeliest tokens are found in the same pass.  Of a CTA's first values the largest ones of 64 groups of lanes are ranked: at least
// `top` values of the row are as large as the top-th of those, and few others.  What is as large goes on the CTA's list, as a number that orders
// by value and then by lowest id; every number on it counts those above, which is its place, at the end and after 1, 2, 4, ... batches of the
// row, when the smallest that stays is the new bound (with the first bound kept, 370 of 128256 values came on the list at a top of 20,
// and 2047 rows took 284 us).  A row that has more than the list can hold (ascending ones, ties) is read again: every warp has a list of
// its own then, which keeps its largest `top` when it is full, and the smallest of them is the warp's new bound.
//
// Few rows: a row's cluster has up to eight CTAs, whose sums and lists meet in the first one's shared memory.
//
// Many rows: 2047 of 128256 in bf16 100 us in a graph (5.2 TB/s), 113 called one after another; with the 20 likeliest 145; 1000 in fp32 87 (5.9 TB/s).
// No pipe is at its bound (1480 rows: issue slots 71 % of active cycles, exponentials' pipe 59 %, ALU 48 %, HBM 4.8 TB/s; warps wait for fixed latencies, for
// each other and for loads in equal parts; with the likeliest tokens as much for barriers).  Few by latency: 64 rows 8.6 us, with the 20 likeliest
// 13.5; one 4.8.
// A vector with minus infinity in it goes value by value: with a tenth of the tokens left 2047 rows take 379 us, the 20 likeliest 407.  Where so few are left
// that groups of lanes have none, there is no bound, and all of the row comes on the list, which runs over: ten tokens left, 20 likeliest, 1175 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <algorithm>

#include "logprobs.h"
#include "pdl.h"

namespace penny {
namespace {

constexpr int kVecs = 4, kWarpsOfSm = 32;  // kVecs: 16 bytes of a thread at a time
constexpr int kGroups = 64, kList = 96, kMaxCluster = 8;  // of a warp's list, and of the CTA's
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kAbove = 8.f;
static_assert(kLogprobsMaxTop <= 32 && kList >= kLogprobsMaxTop + 64, "lists");

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float exp2_ftz(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t of_cta0(const void* p) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_at(p)));
  return r;
}

// `kPer` values of 16 bytes
__device__ __forceinline__ void unpack(const __nv_bfloat16*, const uint4& r, float* x) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
__device__ __forceinline__ void unpack(const __half*, const uint4& r, float* x) {
  const __half2* p = reinterpret_cast<const __half2*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(p[i]);
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack(const float*, const uint4& r, float* x) {
  x[0] = __uint_as_float(r.x), x[1] = __uint_as_float(r.y), x[2] = __uint_as_float(r.z), x[3] = __uint_as_float(r.w);
}
// The largest (NaN if there is one) and the smallest of a vector's values.
template <typename P, typename T>
__device__ __forceinline__ float2 ends_of_pairs(const uint4& r) {
  const P* p = reinterpret_cast<const P*>(&r);
  const P hi = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3])), lo = __hmin2_nan(__hmin2_nan(p[0], p[1]), __hmin2_nan(p[2], p[3]));
  return make_float2(max_nan((float)hi.x, (float)hi.y), fminf((float)lo.x, (float)lo.y));
}
__device__ __forceinline__ float2 ends(const __nv_bfloat16*, const uint4& r) { return ends_of_pairs<__nv_bfloat162, __nv_bfloat16>(r); }
__device__ __forceinline__ float2 ends(const __half*, const uint4& r) { return ends_of_pairs<__half2, __half>(r); }
__device__ __forceinline__ float2 ends(const float*, const uint4& r) {
  const float x = __uint_as_float(r.x), y = __uint_as_float(r.y), z = __uint_as_float(r.z), w = __uint_as_float(r.w);
  return make_float2(max_nan(max_nan(x, y), max_nan(z, w)), fminf(fminf(x, y), fminf(z, w)));
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
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r, x = *reinterpret_cast<unsigned long long*>(&a), y = *reinterpret_cast<unsigned long long*>(&b),
                        z = *reinterpret_cast<unsigned long long*>(&c);
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(float x) { return x; }

// Orders as the values do (NaN on top), equal ones by the lowest id.
__device__ __forceinline__ unsigned long long key_of(float x, int id) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (no negative zero)
  return ((unsigned long long)((int)b < 0 ? ~b : b | 0x80000000u) << 32) | (0xffffffffu - (uint32_t)id);
}
__device__ __forceinline__ float value_of(unsigned long long key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int id_of(unsigned long long key) { return (int)(0xffffffffu - (uint32_t)key); }

// Maximum, sum of exp2(y), sum of exp2(y) y, with y = (x - maximum) log2 e.
struct Sums {
  float m, z, e;
};
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  const float m = max_nan(a.m, b.m);
  const float ya = a.m == m ? 0.f : fmaxf((a.m - m) * kLog2e, -1e30f), yb = b.m == m ? 0.f : fmaxf((b.m - m) * kLog2e, -1e30f);
  if (m != m) return {m, m, m};
  const float ca = exp2_ftz(ya), cb = exp2_ftz(yb);
  // (a sum of nothing is zero, and so is what is multiplied by it; zero times a far maximum is not taken)
  const float ea = ca == 0.f ? 0.f : ca * fmaf(ya, a.z, a.e), eb = cb == 0.f ? 0.f : cb * fmaf(yb, b.z, b.e);
  return {m, a.z * ca + b.z * cb, ea + eb};
}

template <typename T, bool kTop, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kWarpsOfSm / kWarps) k_token_logprobs(const TokenLogprobs a, int cluster) {
  constexpr int kPer = 16 / (int)sizeof(T), kThreads = kWarps * 32, kLanes = kThreads / kGroups, kNumbers = kWarps * kList > 1024 ? kWarps * kList : 1024;
  __shared__ Sums s_sums[kWarps], s_parts[kMaxCluster];
  __shared__ unsigned long long s_list[kTop ? kNumbers : 1], s_group[kTop ? kGroups : 1], s_all[kTop ? kMaxCluster * kLogprobsMaxTop : 1];
  __shared__ float s_bound;
  __shared__ int s_count[kWarps], s_n;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = (int)(blockIdx.x / cluster), rank = (int)(blockIdx.x % cluster);
  const T* const x0 = reinterpret_cast<const T*>(a.logits) + row * a.row_stride;
  // [0, head): in front of the first 16-byte boundary, [head + kPer vecs, vocab): behind the last
  const int head = min(a.vocab, (int)((16 - ((uintptr_t)x0 & 15)) % 16 / sizeof(T))), vecs = (a.vocab - head) / kPer;
  const int per = (vecs + cluster - 1) / cluster, v0 = min(vecs, rank * per), v1 = min(vecs, v0 + per);
  const uint4* const xv = reinterpret_cast<const uint4*>(x0 + head);

  Sums s = {-INFINITY, 0.f, 0.f};  // (the maximum; the sums while they are added up: z and e)
  float bound = -INFINITY;  // values below are not among the top ones
  unsigned long long floor = 0;  // nor are keys up to this one
  int count = 0;             // on the warp's list
  unsigned long long* const list = s_list + (kTop ? warp * kList : 0);
  auto keep_top = [&]() {  // the list's largest `top`, by counting those above
    __syncwarp();
    unsigned long long mine[kList / 32];
    int place[kList / 32];
#pragma unroll
    for (int i = 0; i < kList / 32; ++i) {
      mine[i] = i * 32 + lane < count ? list[i * 32 + lane] : 0;
      place[i] = 0;
    }
    for (int j = 0; j < count; ++j) {
      const unsigned long long other = list[j];
#pragma unroll
      for (int i = 0; i < kList / 32; ++i) place[i] += other > mine[i];
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kList / 32; ++i)
      if (i * 32 + lane < count && place[i] < a.top) list[place[i]] = mine[i];
    __syncwarp();
    if (count >= a.top) {
      count = a.top;
      floor = list[a.top - 1];
      bound = value_of(floor);
    }
  };
  auto offer = [&](float x, int id, bool there) {  // (by whole warps)
    const unsigned long long key = key_of(x, id);
    const bool in = there && key > floor && !(x < bound);
    const uint32_t who = __ballot_sync(0xffffffffu, in);
    if (who == 0) return;
    if (in) list[count + __popc(who & ((1u << lane) - 1))] = key;
    count += __popc(who);
    if (count + 32 > kList) keep_top();
  };
  // the sums in pairs, of even and odd values; joined at the end
  float2 z = make_float2(0.f, 0.f), e = z;
  // The sums count from s.m, which is the largest of a thread's first values, and is raised to one that lies over kAbove above it (NaN
  // too): a warp of which one lane has a new maximum at every other vector would scale its sums all the time.
  auto raise = [&](float top) {
    if (!(top <= s.m + kAbove)) {
      const Sums x = join({s.m, z.x, e.x}, {top, 0.f, 0.f}), y = join({s.m, z.y, e.y}, {top, 0.f, 0.f});
      s.m = x.m;
      z = make_float2(x.z, y.z);
      e = make_float2(x.e, y.e);
    }
  };
  auto one_more = [&](float x) {
    raise(x);
    if (s.m == -INFINITY) return;
    // (minus infinity is exp2(-300) = 0 here, which times itself is zero)
    const float y = max_nan((x - s.m) * kLog2e, -300.f), p = exp2_ftz(y);
    z.x += p;
    e.x = fmaf(p, y, e.x);
  };
  auto add = [&](const float (&x)[kPer], const float2& of) {
    raise(of.x);
    if (s.m == -INFINITY) return;
    const float2 minus = make_float2(-s.m, -s.m), by = make_float2(kLog2e, kLog2e);
    if (of.y - s.m < -2e38f) {  // minus infinity, or what becomes that here (a mask of the type's lowest value)
#pragma unroll 1
      for (int i = 0; i < kPer; ++i) {
        float one = x[0];
#pragma unroll
        for (int j = 1; j < kPer; ++j) one = i == j ? x[j] : one;
        one_more(one);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kPer; i += 2) {
      float2 y = mul2(add2(make_float2(x[i], x[i + 1]), minus), by);
      const float2 p = make_float2(exp2_ftz(y.x), exp2_ftz(y.y));
      z = add2(z, p);
      e = fma2(p, y, e);
    }
  };

  uint4 raw[kVecs];
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int v = v0 + tid + u * kThreads;
    raw[u] = v < v1 ? xv[v] : make_uint4(0, 0, 0, 0);
  }
  float most = -INFINITY;
#pragma unroll
  for (int u = 0; u < kVecs; ++u)
    if (v0 + tid + u * kThreads < v1) most = max_nan(most, ends((const T*)nullptr, raw[u]).x);
  s.m = most;
  if constexpr (kTop) {  // the bound: the top-th of the groups' largest (minus infinity where groups have nothing)
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane % kLanes == 0) s_group[tid / kLanes] = key_of(most, tid / kLanes);
    if (tid == 0) s_n = 0;
    __syncthreads();
    if (tid < kGroups) {
      const unsigned long long mine = s_group[tid];
      int place = 0;
#pragma unroll 8
      for (int j = 0; j < kGroups; ++j) place += s_group[j] > mine;
      if (place == a.top - 1) s_bound = value_of(mine);
    }
    __syncthreads();
    bound = s_bound;
  }
  auto push = [&](float x, int id) {
    if (x < bound) return;
    const int at = atomicAdd(&s_n, 1);
    if (at < kNumbers) s_list[at] = key_of(x, id);
  };
  int batch = 0;
  for (int base = v0; base < v1; base += kThreads * kVecs) {
    if constexpr (kTop) {
      // after 1, 2, 4, ... batches: the list's largest `top`, and the smallest of them as bound
      if (batch > 0 && (batch & (batch - 1)) == 0) {
        __syncthreads();
        const int n = s_n;
        if (n > a.top && n <= kThreads) {
          const unsigned long long mine = tid < n ? s_list[tid] : 0;
          int place = 0;
          if (tid < n) {
#pragma unroll 8
            for (int j = 0; j < n; ++j) place += s_list[j] > mine;
          }
          __syncthreads();
          if (tid < n && place < a.top) s_list[place] = mine;
          if (tid < n && place == a.top - 1) s_bound = value_of(mine), s_n = a.top;
        }
        __syncthreads();
        bound = s_bound;
      }
      ++batch;
    }
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int v = base + tid + u * kThreads, next = v + kThreads * kVecs;
      if (v >= v1) continue;
      float x[kPer];
      unpack((const T*)nullptr, raw[u], x);
      const float2 of = ends((const T*)nullptr, raw[u]);
      if (next < v1) raw[u] = xv[next];
      add(x, of);
      if constexpr (kTop) {
        if (!(of.x < bound)) {
          uint32_t who = 0;
#pragma unroll
          for (int i = 0; i < kPer; ++i) who |= (x[i] < bound ? 0u : 1u) << i;
#pragma unroll 1
          for (; who != 0; who &= who - 1) {
            const int i = __ffs(who) - 1;
            float one = x[0];
#pragma unroll
            for (int j = 1; j < kPer; ++j) one = i == j ? x[j] : one;
            push(one, head + v * kPer + i);
          }
        }
      }
    }
  }
  // what is not in whole vectors: the first CTA's first warp
  if (rank == 0 && warp == 0) {
    const int tail = head + vecs * kPer, rest = head + a.vocab - tail;  // fewer than 16
    const int i = lane < head ? lane : tail + lane - head;
    const bool there = lane < rest;
    if (there) {
      const float x = to_f32(x0[i]);
      one_more(x);
      if constexpr (kTop) push(x, i);
    }
  }
  s = join({s.m, z.x, e.x}, {s.m, z.y, e.y});
  // ---- the warps' and the cluster's sums ----
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    s = join(s, {__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.z, o), __shfl_xor_sync(0xffffffffu, s.e, o)});
  if (lane == 0) s_sums[warp] = s;
  int numbers = 0;  // on the list
  if constexpr (kTop) {
    __syncthreads();
    numbers = s_n;
    if (numbers > kNumbers) {  // once more, with a list for every warp
      for (int base = v0; base < v1; base += kThreads) {
        const int v = base + tid;
        float x[kPer];
        unpack((const T*)nullptr, v < v1 ? xv[v] : make_uint4(0, 0, 0, 0), x);
#pragma unroll 1
        for (int i = 0; i < kPer; ++i) {
          float one = x[0];
#pragma unroll
          for (int j = 1; j < kPer; ++j) one = i == j ? x[j] : one;
          offer(one, head + v * kPer + i, v < v1);
        }
      }
      if (rank == 0 && warp == 0) {
        const int tail = head + vecs * kPer, i = lane < head ? lane : tail + lane - head;
        const bool there = lane < head + a.vocab - tail;
        offer(there ? to_f32(x0[i]) : 0.f, i, there);
      }
      if (count > a.top) keep_top();
      // one behind the other: the numbers first to registers, then to their places
      if (lane == 0) s_count[warp] = count;
      const unsigned long long mine = lane < count ? list[lane] : 0;  // (a.top at most)
      __syncthreads();
      int before = 0;
      numbers = 0;
      for (int w = 0; w < kWarps; ++w) {
        before += w < warp ? s_count[w] : 0;
        numbers += s_count[w];
      }
      if (lane < count) s_list[before + lane] = mine;
    }
  }
  if (cluster > 1) asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");  // (the first CTA is there)
  else __syncthreads();
  if (warp == 0) {
    s = lane < kWarps ? s_sums[lane] : Sums{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1)
      s = join(s, {__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.z, o), __shfl_xor_sync(0xffffffffu, s.e, o)});
    if (lane == 0) {
      const uint32_t to = of_cta0(&s_parts[rank]);
      asm volatile("st.shared::cluster.f32 [%0], %1;\nst.shared::cluster.f32 [%0 + 4], %2;\nst.shared::cluster.f32 [%0 + 8], %3;" ::"r"(to), "f"(s.m),
                   "f"(s.z), "f"(s.e)
                   : "memory");
    }
  }
  if constexpr (kTop) {
    // a thread has a number of the list and counts those above
    const uint32_t to = of_cta0(&s_all[rank * kLogprobsMaxTop]);
    for (int i = tid; i < numbers; i += kThreads) {
      const unsigned long long mine = s_list[i];
      int place = 0;
#pragma unroll 8
      for (int j = 0; j < numbers; ++j) place += s_list[j] > mine;
      if (place < a.top) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to + 8 * place), "l"(mine) : "memory");
    }
    if (tid >= numbers && tid < a.top) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to + 8 * tid), "l"(0ull) : "memory");  // (fewer than that)
  }
  if (cluster > 1) asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
  else __syncthreads();
  if (rank != 0) return;
  s = s_parts[0];
  for (int i = 1; i < cluster; ++i) s = join(s, s_parts[i]);
  const float log_z = s.m == -INFINITY ? 0.f : logf(s.z);
  if (tid == 0) {
    const long long token = a.tokens[row];
    const bool there = token >= 0 && token < a.vocab;
    a.logprobs[row] = !there ? __int_as_float(0x7fffffff) : s.m == -INFINITY ? -INFINITY : to_f32(x0[token]) - s.m - log_z;
    a.entropy[row] = s.m == -INFINITY ? 0.f : log_z - s.e * kLn2 / s.z;
  }
  if constexpr (kTop) {
    for (int i = tid; i < cluster * a.top; i += kThreads) {
      const unsigned long long mine = s_all[i / a.top * kLogprobsMaxTop + i % a.top];
      int place = 0;
      for (int c = 0; c < cluster; ++c) {
#pragma unroll 4
        for (int j = 0; j < a.top; ++j) place += s_all[c * kLogprobsMaxTop + j] > mine;
      }
      if (mine != 0 && place < a.top) {
        a.top_logprobs[(long long)row * a.top + place] = s.m == -INFINITY ? -INFINITY : value_of(mine) - s.m - log_z;
        a.top_ids[(long long)row * a.top + place] = id_of(mine);
      }
    }
  }
}

template <typename T, bool kTop>
cudaError_t launch(const TokenLogprobs& a, int sms, cudaStream_t stream) {
  // Many rows: a CTA of eight warps each, four to an SM, so that some read while others sort.  Few: sixteen warps and as many CTAs of a row
  // as the SMs hold, each with 4096 values at least (64 rows of 128256, top 20: 13 us, with eight warps 17).
  const bool few = a.rows <= 3 * sms;
  int cluster = 1;
  while (few && cluster < kMaxCluster && a.rows * cluster * 2 <= 2 * sms && a.vocab / (cluster * 2) >= 4096) cluster *= 2;
  return few ? launch_kernel_ex(k_token_logprobs<T, kTop, 16>, dim3((unsigned)(a.rows * cluster)), dim3(512), 0, stream, true, cluster, a, cluster)
             : launch_kernel_ex(k_token_logprobs<T, kTop, 8>, dim3((unsigned)a.rows), dim3(256), 0, stream, true, 1, a, 1);
}

}  // namespace

cudaError_t launch_token_logprobs(const TokenLogprobs& a, LogitType type, int sms, cudaStream_t stream) {
  if (a.rows < 0 || a.vocab < 1 || a.vocab > (1 << 30) || a.top < 0 || a.top > kLogprobsMaxTop || a.top > a.vocab) return cudaErrorInvalidValue;
  if (a.rows == 0) return cudaSuccess;
  switch (type) {
    case LOGITS_BF16: return a.top > 0 ? launch<__nv_bfloat16, true>(a, sms, stream) : launch<__nv_bfloat16, false>(a, sms, stream);
    case LOGITS_FP16: return a.top > 0 ? launch<__half, true>(a, sms, stream) : launch<__half, false>(a, sms, stream);
    default: return a.top > 0 ? launch<float, true>(a, sms, stream) : launch<float, false>(a, sms, stream);
  }
}

}  // namespace penny
