// Causal depthwise convolution of width K (2..4) with optional SiLU, forward,
// backward and for one token per stream.
//
//   p_t  = bias + sum_k w_k x_{t-K+1+k},  y_t = p_t sigmoid(p_t) or p_t
//   dp_t = dy_t (s + p_t s (1 - s)),  s = sigmoid(p_t)
//   dx_s = sum_k w_k dp_{s+K-1-k},  dw_k = sum_t dp_t x_{t-K+1+k},  db = sum_t dp_t
//
// Bound by memory: forward reads x and writes y, backward reads x and dy and
// writes dx.  A thread owns V channels and walks a run of tokens with the
// window in registers, so each input is read once plus a halo of K - 1 tokens
// a run (2 (K - 1) in the backward call), which mostly hits L2.
#include "seq_common.cuh"

namespace boa {
namespace seq {

constexpr int kConvThreads = 256;
constexpr int kConvUnroll = 8;

struct ConvRuns {
  int groups;        // channel vectors of a row
  int bx, by;        // threads along the channel vectors and along the runs
  int group_blocks;
  int run, n_runs;   // tokens of a run, runs of a sequence
  int64_t run_blocks;
};

// Row t of the sequence with its past: x at t >= 0, the state (or zeros) before.
template <typename T, int V, int K>
__device__ __forceinline__ void past_row(const T* x, int64_t ts, const T* state, int channels, int t, float (&v)[V]) {
  if (t >= 0) {
    load_f<T, V>(x + t * ts, v);
  } else if (state) {
    load_f<T, V>(state + (int64_t)(K - 1 + t) * channels, v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.0f;
  }
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(kConvThreads) k_conv(const boa_conv_args a, const ConvRuns r) {
  const int cg = (blockIdx.x % r.group_blocks) * r.bx + threadIdx.x % r.bx;
  const int64_t rid = (int64_t)(blockIdx.x / r.group_blocks) * r.by + threadIdx.x / r.bx;
  if (cg >= r.groups || rid >= (int64_t)a.batch * r.n_runs) return;
  const int b = (int)(rid / r.n_runs), t0 = (int)(rid % r.n_runs) * r.run, c = cg * V, E = a.channels;
  const int len = a.lens ? min(max(a.lens[b], 0), a.length) : a.length;
  const T* x = (const T*)a.x + b * a.x_bs + c;
  const T* state = a.state ? (const T*)a.state + (int64_t)b * (K - 1) * E + c : nullptr;
  T* y = (T*)a.y + (int64_t)b * a.length * E + c;
  float w[K][V], bias[V], win[K - 1][V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    bias[j] = a.bias ? a.bias[c + j] : 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][j] = a.weight[(c + j) * K + k];
  }
  const int t1 = min(t0 + r.run, a.length), end = min(t1, len);
  if (t0 < end) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) past_row<T, V, K>(x, a.x_ts, state, E, t0 - (K - 1) + k, win[k]);
  }
  for (int tb = t0; tb < end; tb += kConvUnroll) {
    Vec<T, V> raw[kConvUnroll];
#pragma unroll
    for (int u = 0; u < kConvUnroll; ++u)
      if (tb + u < end) raw[u] = *reinterpret_cast<const Vec<T, V>*>(x + (int64_t)(tb + u) * a.x_ts);
#pragma unroll
    for (int u = 0; u < kConvUnroll; ++u) {
      if (tb + u < end) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float v = to_f(raw[u].v[j]);
          float p = bias[j];
#pragma unroll
          for (int k = 0; k < K - 1; ++k) p = fmaf(w[k][j], win[k][j], p);
          p = fmaf(w[K - 1][j], v, p);
#pragma unroll
          for (int k = 0; k < K - 2; ++k) win[k][j] = win[k + 1][j];
          win[K - 2][j] = v;
          o[j] = a.silu ? p * sigmoid_f(p) : p;
        }
        store_f<T, V>(y + (int64_t)(tb + u) * E, o);
      }
    }
  }
  const float zero[V] = {};
  for (int t = max(t0, end); t < t1; ++t) store_f<T, V>(y + (int64_t)t * E, zero);
  if (t0 == 0 && a.state_out) {
    T* so = (T*)a.state_out + (int64_t)b * (K - 1) * E + c;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      float v[V];
      past_row<T, V, K>(x, a.x_ts, state, E, len - (K - 1) + k, v);
      store_f<T, V>(so + (int64_t)k * E, v);
    }
  }
}

// One thread walks tokens t of its run and K - 1 behind it: dp_t completes
// dx_{t-K+1}.  The run's own tokens add to dw and db, which the block joins
// in shared memory row by row and writes to parts[run block][(K + 1) * E].
template <typename T, int V, int K>
__global__ void __launch_bounds__(kConvThreads) k_conv_backward(const boa_conv_args a, const ConvRuns r,
                                                                float* __restrict__ parts, int64_t run_blocks) {
  extern __shared__ float joined[];   // [K + 1][V][bx]
  const int gx = threadIdx.x % r.bx, ty = threadIdx.x / r.bx;
  const int cg = (blockIdx.x % r.group_blocks) * r.bx + gx;
  const int64_t rb = blockIdx.x / r.group_blocks;
  const int c = cg * V, E = a.channels;
  const bool on = cg < r.groups;
  float w[K][V], bias[V], dw[K][V], db[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    bias[j] = on && a.bias ? a.bias[c + j] : 0.0f;
    db[j] = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      w[k][j] = on ? a.weight[(c + j) * K + k] : 0.0f;
      dw[k][j] = 0.0f;
    }
  }
  const int64_t total = (int64_t)a.batch * r.n_runs;
  for (int64_t rid = rb * r.by + ty; on && rid < total; rid += run_blocks * r.by) {
    const int b = (int)(rid / r.n_runs), t0 = (int)(rid % r.n_runs) * r.run;
    const int len = a.lens ? min(max(a.lens[b], 0), a.length) : a.length;
    const T* x = (const T*)a.x + b * a.x_bs + c;
    const T* dy = (const T*)a.dy + b * a.dy_bs + c;
    const T* state = a.state ? (const T*)a.state + (int64_t)b * (K - 1) * E + c : nullptr;
    const T* dso = a.dstate_out ? (const T*)a.dstate_out + (int64_t)b * (K - 1) * E + c : nullptr;
    T* dx = (T*)a.dx + (int64_t)b * a.length * E + c;
    T* ds = a.dstate ? (T*)a.dstate + (int64_t)b * (K - 1) * E + c : nullptr;
    const int t1 = min(t0 + r.run, a.length);
    float win[K - 1][V], dp[K][V];   // dp[k] is dp_{t-k}
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      if (t0 < len) {
        past_row<T, V, K>(x, a.x_ts, state, E, t0 - (K - 1) + k, win[k]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) win[k][j] = 0.0f;
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) dp[k][j] = 0.0f;
    const int stop = t1 + K - 1;
    for (int tb = t0; tb < stop; tb += kConvUnroll) {
      Vec<T, V> rx[kConvUnroll], rg[kConvUnroll];
#pragma unroll
      for (int u = 0; u < kConvUnroll; ++u)
        if (tb + u < min(stop, len)) {
          rx[u] = *reinterpret_cast<const Vec<T, V>*>(x + (int64_t)(tb + u) * a.x_ts);
          rg[u] = *reinterpret_cast<const Vec<T, V>*>(dy + (int64_t)(tb + u) * a.dy_ts);
        }
#pragma unroll
      for (int u = 0; u < kConvUnroll; ++u) {
        const int t = tb + u;
        if (t >= stop) break;
        const bool live = t < len, mine = t < t1;
        const int s = t - (K - 1);
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float d = 0.0f;
          if (live) {
            const float v = to_f(rx[u].v[j]), g = to_f(rg[u].v[j]);
            d = g;
            if (a.silu) {
              float p = bias[j];
#pragma unroll
              for (int k = 0; k < K - 1; ++k) p = fmaf(w[k][j], win[k][j], p);
              p = fmaf(w[K - 1][j], v, p);
              const float sg = sigmoid_f(p);
              d = g * (sg * (1.0f + p * (1.0f - sg)));
            }
            if (mine) {
              db[j] += d;
#pragma unroll
              for (int k = 0; k < K - 1; ++k) dw[k][j] = fmaf(d, win[k][j], dw[k][j]);
              dw[K - 1][j] = fmaf(d, v, dw[K - 1][j]);
            }
#pragma unroll
            for (int k = 0; k < K - 2; ++k) win[k][j] = win[k + 1][j];
            win[K - 2][j] = v;
          }
#pragma unroll
          for (int k = K - 1; k > 0; --k) dp[k][j] = dp[k - 1][j];
          dp[0][j] = d;
          o[j] = 0.0f;
#pragma unroll
          for (int k = 0; k < K; ++k) o[j] = fmaf(w[k][j], dp[k][j], o[j]);
        }
        const int tail = s - (len - (K - 1));   // row of the final window that x_s (or the state) became
        if (dso && tail >= 0 && tail < K - 1) {
          float e[V];
          load_f<T, V>(dso + (int64_t)tail * E, e);
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] += e[j];
        }
        if (s >= t0 && s >= 0) {
          if (s >= len) {
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = 0.0f;
          }
          store_f<T, V>(dx + (int64_t)s * E, o);
        } else if (s < 0 && ds) {
          store_f<T, V>(ds + (int64_t)(s + K - 1) * E, o);
        }
      }
    }
  }
  constexpr int P = (K + 1) * V;
  for (int k = 0; k < r.by; ++k) {
    if (ty == k) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int i = 0; i < K; ++i) {
          float* p = &joined[(i * V + j) * r.bx + gx];
          *p = (k ? *p : 0.0f) + dw[i][j];
        }
        float* p = &joined[(K * V + j) * r.bx + gx];
        *p = (k ? *p : 0.0f) + db[j];
      }
    }
    __syncthreads();
  }
  if (on && ty == 0) {
    float* out = parts + rb * (int64_t)(K + 1) * E;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int k = i / V, j = i % V;
      const float v = joined[i * r.bx + gx];
      if (k < K) out[(c + j) * K + k] = v;
      else out[(int64_t)K * E + c + j] = v;
    }
  }
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(kConvThreads) k_conv_step(const boa_conv_args a, int groups) {
  const int64_t i = (int64_t)blockIdx.x * kConvThreads + threadIdx.x;
  if (i >= (int64_t)a.batch * groups) return;
  const int64_t b = i / groups;
  const int c = (int)(i % groups) * V, E = a.channels;
  T* st = (T*)a.state_out + b * (K - 1) * E + c;
  Vec<T, V> win[K];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) win[k] = *reinterpret_cast<const Vec<T, V>*>(st + (int64_t)k * E);
  win[K - 1] = *reinterpret_cast<const Vec<T, V>*>((const T*)a.x + b * a.x_bs + c);
  float o[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float p = a.bias ? a.bias[c + j] : 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) p = fmaf(a.weight[(c + j) * K + k], to_f(win[k].v[j]), p);
    o[j] = a.silu ? p * sigmoid_f(p) : p;
  }
#pragma unroll
  for (int k = 0; k < K - 1; ++k) *reinterpret_cast<Vec<T, V>*>(st + (int64_t)k * E) = win[k + 1];
  store_f<T, V>((T*)a.y + b * E + c, o);
}

// Tokens a run: long runs read less halo, short ones fill the GPU when the
// sequences are few.  `halo` tokens are walked besides a run's own.
static ConvRuns conv_runs(const boa_conv_args& a, int V, int halo) {
  ConvRuns r{};
  r.groups = (a.channels + V - 1) / V;
  r.bx = 1;
  while (r.bx < r.groups && r.bx < 32) r.bx *= 2;
  r.by = kConvThreads / r.bx;
  r.group_blocks = (r.groups + r.bx - 1) / r.bx;
  const int64_t want = 148LL * 1024;   // threads
  int steps = 128;                     // walked tokens
  while (steps > 2 * kConvUnroll &&
         (int64_t)a.batch * r.groups * ((a.length + steps - halo - 1) / (steps - halo)) < want)
    steps /= 2;
  r.run = steps - halo;
  r.n_runs = a.length > 0 ? (a.length + r.run - 1) / r.run : 1;
  r.run_blocks = ((int64_t)a.batch * r.n_runs + r.by - 1) / r.by;
  return r;
}

static bool conv_vec(const boa_conv_args& a, int V, bool backward, bool step) {
  if (a.channels % V || a.x_bs % V || (!step && a.x_ts % V) || !aligned(a.x, 16)) return false;
  if (!aligned(a.state, 16) || !aligned(a.state_out, 16)) return false;
  if (!backward) return aligned(a.y, 16);
  return a.dy_bs % V == 0 && a.dy_ts % V == 0 && aligned(a.dy, 16) && aligned(a.dx, 16) && aligned(a.dstate_out, 16) &&
         aligned(a.dstate, 16);
}

// Blocks along the runs in the backward kernel, each with a row of partial
// sums in the workspace: at most about 4 blocks an SM.
static int64_t conv_backward_blocks(const ConvRuns& r) {
  const int64_t most = (592 + r.group_blocks - 1) / r.group_blocks;
  return r.run_blocks < most ? r.run_blocks : most;
}

template <typename T, int V, int K>
static int conv_launch(const boa_conv_args& a, int what, cudaStream_t s) {
  if (what == 2) {
    const int groups = (a.channels + V - 1) / V;
    const int64_t n = (int64_t)a.batch * groups;
    k_conv_step<T, V, K><<<(unsigned)((n + kConvThreads - 1) / kConvThreads), kConvThreads, 0, s>>>(a, groups);
  } else if (what == 0) {
    const ConvRuns r = conv_runs(a, V, 0);
    k_conv<T, V, K><<<(unsigned)(r.run_blocks * r.group_blocks), kConvThreads, 0, s>>>(a, r);
  } else {
    const ConvRuns r = conv_runs(a, V, K - 1);
    const int64_t blocks = conv_backward_blocks(r);
    float* parts = (float*)a.workspace;
    k_conv_backward<T, V, K><<<(unsigned)(blocks * r.group_blocks), kConvThreads,
                               (size_t)(K + 1) * V * r.bx * sizeof(float), s>>>(a, r, parts, blocks);
    const int cols = (K + 1) * a.channels;
    k_sum_parts<<<(cols + 31) / 32, 512, 0, s>>>(parts, blocks, cols, K * a.channels, cols, a.dweight, a.dbias,
                                                nullptr);
  }
  BOA_CUDA(cudaGetLastError());
  return BOA_OK;
}

template <typename T, int K>
static int conv_by_vector(const boa_conv_args& a, int what, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (conv_vec(a, V, what == 1, what == 2)) return conv_launch<T, V, K>(a, what, s);
  return conv_launch<T, 1, K>(a, what, s);
}

template <typename T>
static int conv_by_width(const boa_conv_args& a, int what, cudaStream_t s) {
  if (a.width == 2) return conv_by_vector<T, 2>(a, what, s);
  if (a.width == 3) return conv_by_vector<T, 3>(a, what, s);
  return conv_by_vector<T, 4>(a, what, s);
}

static int conv_dispatch(const boa_conv_args& a, int what, void* stream) {
  BOA_CUDA(cudaSetDevice(a.device));
  cudaStream_t s = (cudaStream_t)stream;
  if (a.dtype == BOA_DTYPE_F32) return conv_by_width<float>(a, what, s);
  if (a.dtype == BOA_DTYPE_BF16) return conv_by_width<__nv_bfloat16>(a, what, s);
  return conv_by_width<__half>(a, what, s);
}

static int conv_check(const boa_conv_args* a, const char* who) {
  if (!a) return boa_fail(BOA_ERR_ARG, std::string(who) + ": null arguments");
  if (a->batch < 0 || a->length < 0 || a->channels < 1)
    return boa_fail(BOA_ERR_ARG, std::string(who) + ": need batch >= 0, length >= 0 and channels >= 1");
  if (a->width < 2 || a->width > 4) return boa_fail(BOA_ERR_UNSUPPORTED, std::string(who) + ": width must be 2, 3 or 4");
  if (a->dtype < BOA_DTYPE_F32 || a->dtype > BOA_DTYPE_F16)
    return boa_fail(BOA_ERR_ARG, std::string(who) + ": unknown dtype");
  return BOA_OK;
}

}  // namespace seq
}  // namespace boa

using namespace boa::seq;

extern "C" {

BOA_API int boa_causal_conv(const boa_conv_args* a, void* stream) {
  const int rc = conv_check(a, "boa_causal_conv");
  if (rc) return rc;
  if (a->batch == 0 || (a->length == 0 && !a->state_out)) return BOA_OK;
  if (!a->weight || (a->length > 0 && (!a->x || !a->y)))
    return boa_fail(BOA_ERR_ARG, "boa_causal_conv: null argument");
  return conv_dispatch(*a, 0, stream);
}

BOA_API size_t boa_causal_conv_workspace_bytes(const boa_conv_args* a) {
  if (conv_check(a, "boa_causal_conv_workspace_bytes")) return 0;
  // the single-element form has the most channel vectors and blocks of rows; take the larger of the two
  const ConvRuns r1 = conv_runs(*a, 1, a->width - 1);
  const ConvRuns rv = conv_runs(*a, a->dtype == BOA_DTYPE_F32 ? 4 : 8, a->width - 1);
  const int64_t b1 = conv_backward_blocks(r1), bv = conv_backward_blocks(rv);
  return (size_t)(b1 > bv ? b1 : bv) * (a->width + 1) * a->channels * sizeof(float);
}

BOA_API int boa_causal_conv_backward(const boa_conv_args* a, void* stream) {
  const int rc = conv_check(a, "boa_causal_conv_backward");
  if (rc) return rc;
  if (!a->weight || !a->dweight) return boa_fail(BOA_ERR_ARG, "boa_causal_conv_backward: null argument");
  if (a->batch == 0) {
    BOA_CUDA(cudaSetDevice(a->device));
    BOA_CUDA(cudaMemsetAsync(a->dweight, 0, (size_t)a->channels * a->width * sizeof(float), (cudaStream_t)stream));
    if (a->dbias)
      BOA_CUDA(cudaMemsetAsync(a->dbias, 0, (size_t)a->channels * sizeof(float), (cudaStream_t)stream));
    return BOA_OK;
  }
  if (a->length > 0 && (!a->x || !a->dy || !a->dx))
    return boa_fail(BOA_ERR_ARG, "boa_causal_conv_backward: null argument");
  if (!a->workspace || a->workspace_bytes < boa_causal_conv_workspace_bytes(a))
    return boa_fail(BOA_ERR_ARG, "boa_causal_conv_backward: workspace too small (see boa_causal_conv_workspace_bytes)");
  return conv_dispatch(*a, 1, stream);
}

BOA_API int boa_causal_conv_step(const boa_conv_args* a, void* stream) {
  const int rc = conv_check(a, "boa_causal_conv_step");
  if (rc) return rc;
  if (a->batch == 0) return BOA_OK;
  if (!a->x || !a->weight || !a->state_out || !a->y) return boa_fail(BOA_ERR_ARG, "boa_causal_conv_step: null argument");
  return conv_dispatch(*a, 2, stream);
}

}  // extern "C"
