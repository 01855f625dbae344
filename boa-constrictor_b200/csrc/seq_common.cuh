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
