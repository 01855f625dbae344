// Shared pieces of the block operators (norm.cu, conv.cu, ssm.cu): activation
// types, guarded vector loads and stores, and the sum of per-block partials.
#pragma once
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <string>

#include "boa_b200.h"
#include "capi_util.h"

namespace boa {
namespace seq {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// V consecutive elements, loaded and stored as one aligned access.
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_f(const T* p, float (&out)[V]) {
  const Vec<T, V> r = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = to_f(r.v[i]);
}

template <typename T, int V>
__device__ __forceinline__ void store_f(T* p, const float (&in)[V]) {
  Vec<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = from_f<T>(in[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = r;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float sigmoid_f(float v) { return rcp(1.0f + ex2(-kLog2e * v)); }

// softplus(v) = max(v, 0) + log(1 + u), u = exp(-|v|), with
// log(1 + u) = 2 artanh(s), s = u / (2 + u) <= 1/3, and artanh(s) / s a minimax
// polynomial in s^2 (relative error 4e-9): exact to a few units in the last
// place for every v, where log2 of a rounded 1 + u would lose small u.
__device__ __forceinline__ float softplus_f(float v, float& u) {
  u = ex2(-kLog2e * fabsf(v));
  const float s = u * rcp(2.0f + u), w = s * s;
  float p = fmaf(0.14089173f, w, 0.13980299f);
  p = fmaf(p, w, 0.20012455f);
  p = fmaf(p, w, 0.33333158f);
  p = fmaf(p, w, 1.0f);
  return fmaxf(v, 0.0f) + 2.0f * s * p;
}

// Pairs of fp32 in one 64-bit register: one instruction for two operations.
struct f2 {
  unsigned long long v;
};
__device__ __forceinline__ f2 pack(float lo, float hi) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpack(f2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ f2 ex2_2(f2 a) {
  const float2 t = unpack(a);
  return pack(ex2(t.x), ex2(t.y));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum of n_parts partial rows: column c of the result is sum_p parts[p * cols + c],
// in a fixed order.  A block owns 32 columns; its 16 warps take the rows in turn
// and are joined in shared memory.  Columns [0, s1) go to o1, [s1, s2) to o2 and
// the rest to o3 (NULL: dropped), so one launch finishes up to three gradients.
static __global__ void __launch_bounds__(512) k_sum_parts(const float* __restrict__ parts, int64_t n_parts, int cols,
                                                          int s1, int s2, float* __restrict__ o1,
                                                          float* __restrict__ o2, float* __restrict__ o3) {
  __shared__ float red[16][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (c < cols)
#pragma unroll 4
    for (int64_t p = w; p < n_parts; p += 16) s += parts[p * cols + c];
  red[w][lane] = s;
  __syncthreads();
  if (w == 0 && c < cols) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += red[i][lane];
    if (c < s1) o1[c] = t;
    else if (c < s2) { if (o2) o2[c - s1] = t; }
    else if (o3) o3[c - s2] = t;
  }
}

inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

inline int n_sms(int device) {
  int n = 148;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
  return n;
}

}  // namespace seq
}  // namespace boa
