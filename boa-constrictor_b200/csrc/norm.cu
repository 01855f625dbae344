// Layer norm over the last axis, forward and backward.
//
//   y  = (x - mean) r w + b,  r = 1 / sqrt(var + eps)
//   dx = r (g - mean(g) - xh mean(g xh)),  g = dy w,  xh = (x - mean) r
//   dw = sum_rows dy xh,  db = sum_rows dy
//
// Bound by memory: the forward call reads x and writes y once, the backward
// call reads x and dy and writes dx once.  A row is held in registers (a warp
// per row up to 1024 columns, a block of 8 warps beyond), so mean and variance
// take two passes over registers and none over memory.  At 131072 x 256 bf16 on
// a B200: forward 25 us (5.4 TB/s of 6.5 measured), backward 42 us (4.8 TB/s)
// and 5 us for the sums of dw and db.
#include "seq_common.cuh"

namespace boa {
namespace seq {

constexpr int kNormWarps = 8;
constexpr int kNormMaxWidth = kNormWarps * 32 * 32;

// Sum over the LANES threads of a row; every thread gets it.
template <int ROW_WARPS>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = warp_sum(v);
  if constexpr (ROW_WARPS > 1) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < ROW_WARPS; ++i) v += red[i];
  }
  return v;
}

// VPL values of a row per thread, as VPL / V accesses of V elements, zeros
// beyond the width.
template <typename T, int V, int VPL, int ROW_WARPS>
struct NormRow {
  Words<T, V> r[VPL / V];
  __device__ __forceinline__ void load(const T* row, int width, int lane) {
#pragma unroll
    for (int c = 0; c < VPL / V; ++c) {
      const int i = (c * 32 * ROW_WARPS + lane) * V;
      r[c].clear();
      if (i < width) r[c].load(row + i);
    }
  }
  __device__ __forceinline__ void get(float (&v)[VPL]) const {
#pragma unroll
    for (int i = 0; i < VPL; ++i) v[i] = r[i / V].get(i % V);
  }
};

// Rows a warp works on together: their loads and reductions overlap.
template <int VPL, int ROW_WARPS>
constexpr int norm_rows() { return ROW_WARPS > 1 ? 1 : VPL <= 8 ? 4 : VPL <= 16 ? 2 : 1; }

// A column's parameters in registers, zeros beyond the width or without the array.
template <int V, int VPL, int ROW_WARPS>
__device__ __forceinline__ void param_load(const float* p, int width, int lane, float (&v)[VPL]) {
#pragma unroll
  for (int c = 0; c < VPL / V; ++c)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = (c * 32 * ROW_WARPS + lane) * V + j;
      v[c * V + j] = p && i < width ? p[i] : 0.0f;
    }
}

template <typename T, int V, int VPL, int ROW_WARPS>
__global__ void __launch_bounds__(kNormWarps * 32) k_norm(int64_t rows, int width, const T* __restrict__ x,
                                                          int64_t x_stride, const float* __restrict__ w,
                                                          const float* __restrict__ b, float eps, T* __restrict__ y,
                                                          float* __restrict__ stats) {
  __shared__ float red[ROW_WARPS];
  constexpr int kLanes = 32 * ROW_WARPS, R = norm_rows<VPL, ROW_WARPS>();
  constexpr int kRows = kNormWarps / ROW_WARPS * R;
  const int lane = threadIdx.x % kLanes;
  const float inv = 1.0f / (float)width;
  float wv[VPL], bv[VPL];
  param_load<V, VPL, ROW_WARPS>(w, width, lane, wv);
  param_load<V, VPL, ROW_WARPS>(b, width, lane, bv);
  NormRow<T, V, VPL, ROW_WARPS> next[R];      // the rows of the next round are in flight while these are worked on
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int k = 0; k < R; ++k) next[k].load(x + min(row + k, rows - 1) * x_stride, width, lane);
  };
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes * R;
  if (row < rows) fetch(row);
  for (; row < rows; row += (int64_t)gridDim.x * kRows) {
    float v[R][VPL], s[R], mean[R], rstd[R];
#pragma unroll
    for (int k = 0; k < R; ++k) next[k].get(v[k]);
    if (row + (int64_t)gridDim.x * kRows < rows) fetch(row + (int64_t)gridDim.x * kRows);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      s[k] = 0.0f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) s[k] += v[k][i];
    }
#pragma unroll
    for (int k = 0; k < R; ++k) mean[k] = row_sum<ROW_WARPS>(s[k], red) * inv;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      s[k] = 0.0f;
#pragma unroll
      for (int c = 0; c < VPL / V; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[k][c * V + j] -= mean[k];
          const float d = v[k][c * V + j];
          s[k] += ((c * kLanes + lane) * V < width) ? d * d : 0.0f;
        }
    }
#pragma unroll
    for (int k = 0; k < R; ++k) rstd[k] = rsqrtf(row_sum<ROW_WARPS>(s[k], red) * inv + eps);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      if (row + k >= rows) break;
      if (stats && lane == 0)
        *reinterpret_cast<float2*>(stats + 2 * (row + k)) = make_float2(mean[k], rstd[k]);
#pragma unroll
      for (int c = 0; c < VPL / V; ++c) {
        const int i = (c * kLanes + lane) * V;
        if (i < width) {
          float o[V];
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = fmaf(v[k][c * V + j] * rstd[k], wv[c * V + j], bv[c * V + j]);
          store_f<T, V>(y + (row + k) * width + i, o);
        }
      }
    }
  }
}

// dx row by row; every thread keeps the sums of its columns' dw and db over all
// rows it takes.  The block's warps are joined in shared memory, warp by warp,
// and the block's sums go to parts[block][2 * width].
template <typename T, int V, int VPL, int ROW_WARPS>
__global__ void __launch_bounds__(kNormWarps * 32)
    k_norm_backward(int64_t rows, int width, const T* __restrict__ x, int64_t x_stride, const T* __restrict__ dy,
                    int64_t dy_stride, const float* __restrict__ w, const float* __restrict__ stats,
                    T* __restrict__ dx, float* __restrict__ parts) {
  extern __shared__ float joined[];   // [2 * width]
  __shared__ float red[ROW_WARPS];
  constexpr int kLanes = 32 * ROW_WARPS, R = norm_rows<VPL, ROW_WARPS>() > 1 ? 2 : 1;
  constexpr int kSubs = kNormWarps / ROW_WARPS, kRows = kSubs * R;
  const int lane = threadIdx.x % kLanes, sub = threadIdx.x / kLanes;
  const float inv = 1.0f / (float)width;
  float wv[VPL], dw[VPL], db[VPL];
  param_load<V, VPL, ROW_WARPS>(w, width, lane, wv);
#pragma unroll
  for (int i = 0; i < VPL; ++i) dw[i] = db[i] = 0.0f;
  NormRow<T, V, VPL, ROW_WARPS> nx[R], ng[R];      // the next round's rows, in flight
  float2 nst[R];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t r = min(row + k, rows - 1);
      nx[k].load(x + r * x_stride, width, lane);
      ng[k].load(dy + r * dy_stride, row + k < rows ? width : 0, lane);   // a row past the last: dy counts as zero
      nst[k] = *reinterpret_cast<const float2*>(stats + 2 * r);
    }
  };
  int64_t row = (int64_t)blockIdx.x * kRows + sub * R;
  if (row < rows) fetch(row);
  for (; row < rows; row += (int64_t)gridDim.x * kRows) {
    float xv[R][VPL], gv[R][VPL], s[R], q[R], rstd[R];
    float2 stv[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      nx[k].get(xv[k]);
      ng[k].get(gv[k]);
      stv[k] = nst[k];
    }
    if (row + (int64_t)gridDim.x * kRows < rows) fetch(row + (int64_t)gridDim.x * kRows);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const float2 st = stv[k];
      rstd[k] = st.y;
      s[k] = q[k] = 0.0f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        xv[k][i] = (xv[k][i] - st.x) * st.y;
        dw[i] = fmaf(gv[k][i], xv[k][i], dw[i]);      // dy is 0 beyond the width
        db[i] += gv[k][i];
        gv[k][i] *= wv[i];
        s[k] += gv[k][i];
        q[k] = fmaf(gv[k][i], xv[k][i], q[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      s[k] = row_sum<ROW_WARPS>(s[k], red) * inv;
      q[k] = row_sum<ROW_WARPS>(q[k], red) * inv;
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      if (row + k >= rows) break;
#pragma unroll
      for (int c = 0; c < VPL / V; ++c) {
        const int i = (c * kLanes + lane) * V;
        if (i < width) {
          float o[V];
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = rstd[k] * (gv[k][c * V + j] - s[k] - xv[k][c * V + j] * q[k]);
          store_f<T, V>(dx + (row + k) * width + i, o);
        }
      }
    }
  }
  for (int k = 0; k < kSubs; ++k) {
    if (sub == k) {
#pragma unroll
      for (int c = 0; c < VPL / V; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int i = (c * kLanes + lane) * V + j;
          if (i < width) {
            joined[i] = (k ? joined[i] : 0.0f) + dw[c * V + j];
            joined[width + i] = (k ? joined[width + i] : 0.0f) + db[c * V + j];
          }
        }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 2 * width; i += blockDim.x) parts[(int64_t)blockIdx.x * 2 * width + i] = joined[i];
}

struct NormCall {
  int64_t rows;
  int width, dtype;
  const void* x;
  int64_t x_stride;
  const void* dy;
  int64_t dy_stride;
  const float *w, *b;
  float eps;
  void* out;
  float* stats;
  float* parts;
  int grid;
  cudaStream_t s;
};

// Blocks of the backward kernel (its workspace holds a row of sums per block):
// the 2 that each of 148 SMs holds, fewer when the rows are few.  They take row
// after row, the next rows in flight (47 us with 592 blocks, 42 us with 296, at
// 131072 x 256 bf16).
static int norm_backward_grid(int64_t rows, int width) {
  const int64_t per = width <= 512 ? 2 * kNormWarps : width <= 1024 ? kNormWarps : 1;
  const int64_t need = (rows + per - 1) / per;
  return (int)(need < 296 ? need : 296);
}

// Forward blocks an SM: about as many as it holds, so that they stay and keep the
// next rows in flight (8 against 2: 30.6 and 26.9 us at 131072 x 256 bf16, 51.4 and
// 35.2 us at 32768 x 1024); a row a block of at most 8 values a thread wants 4
// (31.1 us with 2, 24.9 us with 4, at 8192 x 2048 fp32).
static int norm_forward_blocks(int width) { return width > 1024 && width <= 2048 ? 4 : 2; }

template <typename T, int V, int VPL, int ROW_WARPS>
static void norm_launch(const NormCall& c, bool backward) {
  if (backward) {
    const size_t smem = (size_t)2 * c.width * sizeof(float);
    auto k = k_norm_backward<T, V, VPL, ROW_WARPS>;
    // the bound of all widths, not this one's size: another thread may launch between here and the launch
    if (smem > 48 * 1024)
      cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kNormMaxWidth * (int)sizeof(float));
    k<<<c.grid, kNormWarps * 32, smem, c.s>>>(c.rows, c.width, (const T*)c.x, c.x_stride, (const T*)c.dy, c.dy_stride,
                                             c.w, c.stats, (T*)c.out, c.parts);
  } else {
    k_norm<T, V, VPL, ROW_WARPS><<<c.grid, kNormWarps * 32, 0, c.s>>>(c.rows, c.width, (const T*)c.x, c.x_stride, c.w,
                                                                     c.b, c.eps, (T*)c.out, c.stats);
  }
}

template <typename T, int V>
static void norm_by_width(const NormCall& c, bool backward) {
  const int w = c.width;
  if (w <= 256) norm_launch<T, V, 8, 1>(c, backward);
  else if (w <= 512) norm_launch<T, V, 16, 1>(c, backward);
  else if (w <= 1024) norm_launch<T, V, 32, 1>(c, backward);
  else if (w <= 2048) norm_launch<T, V, 8, kNormWarps>(c, backward);
  else if (w <= 4096) norm_launch<T, V, 16, kNormWarps>(c, backward);
  else norm_launch<T, V, 32, kNormWarps>(c, backward);
}

// 16-byte accesses where every row starts on a 16-byte boundary and holds whole
// vectors, single elements otherwise.
template <typename T>
static void norm_by_vector(const NormCall& c, bool backward) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = c.width % V == 0 && c.x_stride % V == 0 && aligned(c.x, 16) && aligned(c.out, 16) &&
                   (!backward || (c.dy_stride % V == 0 && aligned(c.dy, 16)));
  if (vec) norm_by_width<T, V>(c, backward);
  else norm_by_width<T, 1>(c, backward);
}

static int norm_dispatch(const NormCall& c, bool backward) {
  if (c.dtype == BOA_DTYPE_F32) norm_by_vector<float>(c, backward);
  else if (c.dtype == BOA_DTYPE_BF16) norm_by_vector<__nv_bfloat16>(c, backward);
  else norm_by_vector<__half>(c, backward);
  BOA_CUDA(cudaGetLastError());
  return BOA_OK;
}

static int norm_check(const char* who, int64_t rows, int width, int dtype) {
  if (rows < 0 || width < 1) return boa_fail(BOA_ERR_ARG, std::string(who) + ": need rows >= 0 and width >= 1");
  if (width > kNormMaxWidth)
    return boa_fail(BOA_ERR_UNSUPPORTED, std::string(who) + ": width must be at most 8192");
  if (dtype < BOA_DTYPE_F32 || dtype > BOA_DTYPE_F16) return boa_fail(BOA_ERR_ARG, std::string(who) + ": unknown dtype");
  return BOA_OK;
}

}  // namespace seq
}  // namespace boa

using namespace boa::seq;

extern "C" {

BOA_API int boa_layer_norm(int64_t rows, int width, int dtype, const void* d_x, int64_t x_stride,
                           const float* d_weight, const float* d_bias, float eps, void* d_y, float* d_stats,
                           int device, void* stream) {
  const int rc = norm_check("boa_layer_norm", rows, width, dtype);
  if (rc) return rc;
  if (rows == 0) return BOA_OK;
  if (!d_x || !d_weight || !d_y) return boa_fail(BOA_ERR_ARG, "boa_layer_norm: null argument");
  if (!aligned(d_stats, 8)) return boa_fail(BOA_ERR_ARG, "boa_layer_norm: stats must be 8-byte aligned");
  BOA_CUDA(cudaSetDevice(device));
  NormCall c{};
  c.rows = rows; c.width = width; c.dtype = dtype; c.x = d_x; c.x_stride = x_stride;
  c.w = d_weight; c.b = d_bias; c.eps = eps; c.out = d_y; c.stats = d_stats; c.s = (cudaStream_t)stream;
  const int64_t per = width <= 256 ? 4 * kNormWarps : width <= 512 ? 2 * kNormWarps : width <= 1024 ? kNormWarps : 1;
  const int64_t need = (rows + per - 1) / per, most = (int64_t)n_sms(device) * norm_forward_blocks(width);
  c.grid = (int)(need < most ? need : most);
  return norm_dispatch(c, false);
}

BOA_API size_t boa_layer_norm_workspace_bytes(int64_t rows, int width, int dtype) {
  if (rows < 1 || width < 1 || width > kNormMaxWidth || dtype < BOA_DTYPE_F32 || dtype > BOA_DTYPE_F16) return 0;
  return (size_t)norm_backward_grid(rows, width) * 2 * width * sizeof(float);
}

BOA_API int boa_layer_norm_backward(int64_t rows, int width, int dtype, const void* d_x, int64_t x_stride,
                                    const void* d_dy, int64_t dy_stride, const float* d_weight,
                                    const float* d_stats, void* d_dx, float* d_dweight, float* d_dbias,
                                    void* d_workspace, size_t workspace_bytes, int device, void* stream) {
  const int rc = norm_check("boa_layer_norm_backward", rows, width, dtype);
  if (rc) return rc;
  if (!d_dweight) return boa_fail(BOA_ERR_ARG, "boa_layer_norm_backward: null argument");
  cudaStream_t s = (cudaStream_t)stream;
  if (rows == 0) {
    BOA_CUDA(cudaSetDevice(device));
    BOA_CUDA(cudaMemsetAsync(d_dweight, 0, (size_t)width * sizeof(float), s));
    if (d_dbias) BOA_CUDA(cudaMemsetAsync(d_dbias, 0, (size_t)width * sizeof(float), s));
    return BOA_OK;
  }
  if (!d_x || !d_dy || !d_weight || !d_stats || !d_dx)
    return boa_fail(BOA_ERR_ARG, "boa_layer_norm_backward: null argument");
  if (!aligned(d_stats, 8)) return boa_fail(BOA_ERR_ARG, "boa_layer_norm_backward: stats must be 8-byte aligned");
  if (!d_workspace || workspace_bytes < boa_layer_norm_workspace_bytes(rows, width, dtype))
    return boa_fail(BOA_ERR_ARG, "boa_layer_norm_backward: workspace too small (see boa_layer_norm_workspace_bytes)");
  BOA_CUDA(cudaSetDevice(device));
  NormCall c{};
  c.rows = rows; c.width = width; c.dtype = dtype; c.x = d_x; c.x_stride = x_stride; c.dy = d_dy;
  c.dy_stride = dy_stride; c.w = d_weight; c.out = d_dx; c.stats = const_cast<float*>(d_stats);
  c.parts = (float*)d_workspace; c.s = s;
  c.grid = norm_backward_grid(rows, width);
  const int e = norm_dispatch(c, true);
  if (e) return e;
  k_sum_parts<<<(2 * width + 31) / 32, 1024, 0, s>>>(c.parts, c.grid, 2 * width, width, 2 * width,
                                                  d_dweight, d_dbias, nullptr);
  BOA_CUDA(cudaGetLastError());
  return BOA_OK;
}

}  // extern "C"
