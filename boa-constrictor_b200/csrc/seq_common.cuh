// Shared pieces of the block operators (norm.cu, conv.cu, ssm.cu): activation
// types, guarded vector loads and stores, and the sum of per-block partials.
#pragma once
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <cstring>
#include <string>
#include <type_traits>

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

// V elements as the 32-bit words they are loaded in (an element a word for
// single-element rows), unpacked when they are used: a bf16 is the upper half
// of its fp32, two 16-bit results are rounded by one instruction.
template <typename T, int V>
struct Words {
  static constexpr int kN = V * (int)sizeof(T) >= 4 ? V * (int)sizeof(T) / 4 : 1;
  uint32_t w[kN];
  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
    const uint32_t u = w[j / 2];
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      return __uint_as_float(j & 1 ? u & 0xffff0000u : u << 16);
    } else {
      return __half2float(__ushort_as_half((unsigned short)(j & 1 ? u >> 16 : u)));
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kN; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V * sizeof(T) == 2) w[0] = *reinterpret_cast<const unsigned short*>(p);
    if constexpr (V * sizeof(T) == 4) w[0] = *reinterpret_cast<const uint32_t*>(p);
    if constexpr (V * sizeof(T) == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x;
      w[1] = v.y;
    }
    if constexpr (V * sizeof(T) == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x;
      w[1] = v.y;
      w[2] = v.z;
      w[3] = v.w;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V * sizeof(T) == 2) *reinterpret_cast<unsigned short*>(p) = (unsigned short)w[0];
    if constexpr (V * sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
    if constexpr (V * sizeof(T) == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void set(const float (&v)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(v[i]);
    } else if constexpr (V == 1) {
      const T t = from_f<T>(v[0]);
      unsigned short h;
      memcpy(&h, &t, 2);
      w[0] = h;
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        memcpy(&w[i], &t, 4);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const __half2 t = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        memcpy(&w[i], &t, 4);
      }
    }
  }
};

template <typename T, int V>
__device__ __forceinline__ void store_f(T* p, const float (&in)[V]) {
  Words<T, V> r;
  r.set(in);
  r.store(p);
}

// Rows on their way from global memory, DEPTH groups of U accesses ahead of
// their use without holding registers: every thread copies what it will itself
// read (cp.async into slots of its own), so no barrier is needed.  16-bit single
// elements, which cp.async cannot copy, are loaded when they are taken.
template <typename T, int V, int U, int DEPTH>
struct Ahead {
  static constexpr int kBytes = V * (int)sizeof(T);
  static constexpr bool kAsync = kBytes >= 4;
  // shared memory of a block of `threads`
  static constexpr size_t bytes(int threads) { return kAsync ? (size_t)DEPTH * U * threads * kBytes : 0; }
  uint32_t base, step;      // this thread's slot, bytes between its slots
  int slot = 0;
  __device__ __forceinline__ Ahead(void* smem, int thread, int threads)
      : base((uint32_t)__cvta_generic_to_shared(smem) + thread * kBytes), step(threads * kBytes) {}
  __device__ __forceinline__ void start(int s, const T* p, int64_t stride) {
    if constexpr (kAsync) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(base + (s * U + u) * step), "l"(p + u * stride),
                     "n"(kBytes) : "memory");
    }
  }
  // the end of a group of all rings of this thread; every group is ended, empty ones too
  static __device__ __forceinline__ void commit() {
    if constexpr (kAsync) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  static __device__ __forceinline__ void wait() {
    if constexpr (kAsync) asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
  }
  // the oldest group, whose rows start at p
  __device__ __forceinline__ void take(const T* p, int64_t stride, Words<T, V> (&r)[U]) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (kAsync) {
        const uint32_t at = base + (slot * U + u) * step;
        if constexpr (kBytes == 4) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r[u].w[0]) : "r"(at) : "memory");
        if constexpr (kBytes == 8)
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r[u].w[0]), "=r"(r[u].w[1]) : "r"(at) : "memory");
        if constexpr (kBytes == 16)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(r[u].w[0]), "=r"(r[u].w[1]), "=r"(r[u].w[2]), "=r"(r[u].w[3]) : "r"(at) : "memory");
      } else {
        r[u].load(p + u * stride);
      }
    }
  }
  __device__ __forceinline__ void next() { slot = slot + 1 == DEPTH ? 0 : slot + 1; }
};

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
// polynomial in s^2 (relative error 8e-9), where log2 of a rounded 1 + u would
// lose small u.  The relative error is at most (12 + 1.25 max(-v, 0)) 2^-24: a
// few roundings, and that of the exponent, which exp scales by |v|.  exp(d A)
// has the same share from its own exponent.  Below v = -87.3 u is flushed to 0.
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
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ f2 ex2_2(f2 a) {
  const float2 t = unpack(a);
  return pack(ex2(t.x), ex2(t.y));
}

// softplus_f of two values; u as there.
__device__ __forceinline__ f2 softplus2(f2 v, f2& u) {
  u = ex2_2(mul2(f2{v.v & 0x7fffffff7fffffffull}, pack(-kLog2e, -kLog2e)));
  const float2 den = unpack(add2(u, pack(2.0f, 2.0f)));
  const f2 s = mul2(u, pack(rcp(den.x), rcp(den.y))), w = mul2(s, s);
  f2 p = fma2(pack(0.14089173f, 0.14089173f), w, pack(0.13980299f, 0.13980299f));
  p = fma2(p, w, pack(0.20012455f, 0.20012455f));
  p = fma2(p, w, pack(0.33333158f, 0.33333158f));
  p = fma2(p, w, pack(1.0f, 1.0f));
  const float2 x = unpack(v);
  return fma2(add2(s, s), p, pack(fmaxf(x.x, 0.0f), fmaxf(x.y, 0.0f)));
}

// V fp32 values of neighbouring channels: pairs where V is even, one value for V = 1.
template <int V>
struct Fv {
  f2 p[V / 2];
};
template <>
struct Fv<1> {
  float p;
};
template <int V>
__device__ __forceinline__ Fv<V> splat(float x) {
  Fv<V> r;
  if constexpr (V == 1) {
    r.p = x;
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.p[i] = pack(x, x);
  }
  return r;
}
template <int V>
__device__ __forceinline__ Fv<V> from_array(const float (&x)[V]) {
  Fv<V> r;
  if constexpr (V == 1) {
    r.p = x[0];
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.p[i] = pack(x[2 * i], x[2 * i + 1]);
  }
  return r;
}
template <int V>
__device__ __forceinline__ void to_array(const Fv<V>& a, float (&x)[V]) {
  if constexpr (V == 1) {
    x[0] = a.p;
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 t = unpack(a.p[i]);
      x[2 * i] = t.x;
      x[2 * i + 1] = t.y;
    }
  }
}
template <int V>
__device__ __forceinline__ Fv<V> vfma(const Fv<V>& a, const Fv<V>& b, const Fv<V>& c) {
  Fv<V> r;
  if constexpr (V == 1) {
    r.p = fmaf(a.p, b.p, c.p);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.p[i] = fma2(a.p[i], b.p[i], c.p[i]);
  }
  return r;
}
template <int V>
__device__ __forceinline__ Fv<V> vmul(const Fv<V>& a, const Fv<V>& b) {
  Fv<V> r;
  if constexpr (V == 1) {
    r.p = a.p * b.p;
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.p[i] = mul2(a.p[i], b.p[i]);
  }
  return r;
}
template <int V>
__device__ __forceinline__ Fv<V> vadd(const Fv<V>& a, const Fv<V>& b) {
  Fv<V> r;
  if constexpr (V == 1) {
    r.p = a.p + b.p;
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.p[i] = add2(a.p[i], b.p[i]);
  }
  return r;
}
template <int V>
__device__ __forceinline__ Fv<V> vsigmoid(const Fv<V>& a) {
  Fv<V> e = vmul(a, splat<V>(-kLog2e));
  if constexpr (V == 1) {
    e.p = ex2(e.p);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) e.p[i] = ex2_2(e.p[i]);
  }
  e = vadd(e, splat<V>(1.0f));
  if constexpr (V == 1) {
    e.p = rcp(e.p);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 t = unpack(e.p[i]);
      e.p[i] = pack(rcp(t.x), rcp(t.y));
    }
  }
  return e;
}
template <typename T, int V>
__device__ __forceinline__ Fv<V> values(const Words<T, V>& w) {
  float x[V];
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = w.get(i);
  return from_array<V>(x);
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const Fv<V>& a) {
  float x[V];
  to_array<V>(a, x);
  store_f<T, V>(p, x);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum of n_parts partial rows: column c of the result is sum_p parts[p * cols + c],
// in a fixed order.  A block owns 32 columns; its 32 warps take the rows in turn
// and are joined in shared memory.  Columns [0, s1) go to o1, [s1, s2) to o2 and
// the rest to o3 (NULL: dropped), so one launch finishes up to three gradients.
static __global__ void __launch_bounds__(1024) k_sum_parts(const float* __restrict__ parts, int64_t n_parts,
                                                          int64_t cols, int64_t s1, int64_t s2,
                                                          float* __restrict__ o1, float* __restrict__ o2,
                                                          float* __restrict__ o3) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (c < cols)
#pragma unroll 8
    for (int64_t p = w; p < n_parts; p += 32) s += parts[p * cols + c];
  red[w][lane] = s;
  __syncthreads();
  if (w == 0 && c < cols) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += red[i][lane];
    if (c < s1) o1[c] = t;
    else if (c < s2) { if (o2) o2[c - s1] = t; }
    else if (o3) o3[c - s2] = t;
  }
}

// Bound on the length and the channels of a call: indexes behind the last tile,
// run or block of a row then still fit 32 bits.  Their products are 64 bits wide.
constexpr int kMaxSize = 0x7fffffff - (1 << 16);

inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

inline int n_sms(int device) {
  int n = 148;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
  return n;
}

}  // namespace seq
}  // namespace boa
