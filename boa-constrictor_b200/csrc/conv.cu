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
// a run (2 (K - 1) in the backward call), which mostly hits L2.  On a B200:
// forward of 1 x 67109 x 512 fp32 44 us (6.2 of 6.5 TB/s measured), of 16 x 4096
// x 512 bf16 35 us (3.9 TB/s), backward 65 us (3.1 TB/s, bound by instruction
// latency at 16 warps an SM), one token of 8192 x 512 bf16 12.5 us (5.4 TB/s).
#include "seq_common.cuh"

namespace boa {
namespace seq {

constexpr int kConvThreads = 256;
constexpr int kConvUnroll = 4;    // tokens worked on at once
// groups of as many in flight: 32 KB a block and tensor
template <typename T, int V>
constexpr int conv_depth() { return V * sizeof(T) > 8 ? 2 : 4; }
template <typename T, int V>
using ConvRows = Ahead<T, V, kConvUnroll, conv_depth<T, V>()>;
constexpr int kConvVec = 4;       // channels a thread

struct ConvRuns {
  int groups;        // channel vectors of a row
  int bx, by;        // threads along the channel vectors and along the runs
  int group_blocks;
  int run, n_runs;   // tokens of a run, runs of a sequence
  int64_t run_blocks;
};

// Row t of the sequence with its past: x at t >= 0, the state (or zeros) before.
template <typename T, int V, int K>
__device__ __forceinline__ Fv<V> past_row(const T* x, int64_t ts, const T* state, int channels, int t) {
  Words<T, V> r;
  r.clear();
  if (t >= 0) r.load(x + t * ts);
  else if (state) r.load(state + (int64_t)(K - 1 + t) * channels);
  return values<T, V>(r);
}

// Weights [channels][K] of V channels; rows of 4 floats as one load.
template <int V, int K>
__device__ __forceinline__ void load_weights(const boa_conv_args& a, int c, bool on, Fv<V> (&w)[K], Fv<V>& bias) {
  float b[V], v[K][V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    b[j] = on && a.bias ? a.bias[c + j] : 0.0f;
    if constexpr (K == 4) {
      const float4 r = on ? *reinterpret_cast<const float4*>(a.weight + (int64_t)(c + j) * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
      v[0][j] = r.x;
      v[1][j] = r.y;
      v[2][j] = r.z;
      v[3][j] = r.w;
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) v[k][j] = on ? a.weight[(int64_t)(c + j) * K + k] : 0.0f;
    }
  }
  bias = from_array<V>(b);
#pragma unroll
  for (int k = 0; k < K; ++k) w[k] = from_array<V>(v[k]);
}

// p_t of one channel vector: the window and the new row.
template <int V, int K>
__device__ __forceinline__ Fv<V> conv_dot(const Fv<V> (&w)[K], const Fv<V>& bias, const Fv<V> (&win)[K - 1],
                                          const Fv<V>& v) {
  Fv<V> p = bias;
#pragma unroll
  for (int k = 0; k < K - 1; ++k) p = vfma(w[k], win[k], p);
  return vfma(w[K - 1], v, p);
}
template <int V, int K>
__device__ __forceinline__ void push(Fv<V> (&win)[K - 1], const Fv<V>& v) {
#pragma unroll
  for (int k = 0; k < K - 2; ++k) win[k] = win[k + 1];
  win[K - 2] = v;
}

template <typename T, int V>
__device__ __forceinline__ Words<T, V> raw_at(const T* p) {
  Words<T, V> r;
  r.load(p);
  return r;
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(kConvThreads, 3) k_conv(const boa_conv_args a, const ConvRuns r) {
  const int cg = (blockIdx.x % r.group_blocks) * r.bx + threadIdx.x % r.bx;
  const int64_t rid = (int64_t)(blockIdx.x / r.group_blocks) * r.by + threadIdx.x / r.bx;
  if (cg >= r.groups || rid >= (int64_t)a.batch * r.n_runs) return;
  const int b = (int)(rid / r.n_runs), t0 = (int)(rid % r.n_runs) * r.run, c = cg * V, E = a.channels;
  const int len = a.lens ? min(max(a.lens[b], 0), a.length) : a.length;
  const T* x = (const T*)a.x + b * a.x_bs + c;
  const T* state = a.state ? (const T*)a.state + (int64_t)b * (K - 1) * E + c : nullptr;
  T* y = (T*)a.y + ((int64_t)b * a.length + t0) * E + c;
  const int t1 = min(t0 + r.run, a.length), end = min(t1, len);
  const T* px = x + (int64_t)t0 * a.x_ts;
  using Rows = ConvRows<T, V>;
  constexpr int kDepth = conv_depth<T, V>();
  extern __shared__ __align__(16) uint8_t smem[];
  Rows ahead(smem, threadIdx.x, kConvThreads);
  const int n = max(end - t0, 0) / kConvUnroll;      // whole groups
  const int64_t group = kConvUnroll * a.x_ts;
#pragma unroll
  for (int i = 0; i < kDepth; ++i) {
    if (i < n) ahead.start(i, px + i * group, a.x_ts);
    Rows::commit();
  }
  Fv<V> w[K], bias, win[K - 1];
  load_weights<V, K>(a, c, true, w, bias);
  if (t0 < end) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) win[k] = past_row<T, V, K>(x, a.x_ts, state, E, t0 - (K - 1) + k);
  }
  auto row = [&](const Words<T, V>& raw) {
    const Fv<V> v = values<T, V>(raw);
    Fv<V> p = conv_dot<V, K>(w, bias, win, v);
    push<V, K>(win, v);
    if (a.silu) p = vmul(p, vsigmoid<V>(p));
    store_v<T, V>(y, p);
    y += E;
  };
  for (int i = 0; i < n; ++i) {
    Words<T, V> raw[kConvUnroll];
    Rows::wait();
    ahead.take(px, a.x_ts, raw);
    if (i + kDepth < n) ahead.start(ahead.slot, px + kDepth * group, a.x_ts);
    Rows::commit();
    ahead.next();
    px += group;
#pragma unroll
    for (int u = 0; u < kConvUnroll; ++u) row(raw[u]);
  }
  int t = t0 + n * kConvUnroll;
  for (; t < end; ++t) {
    row(raw_at<T, V>(px));
    px += a.x_ts;
  }
  for (t = max(t0, end); t < t1; ++t) {
    store_v<T, V>(y, splat<V>(0.0f));
    y += E;
  }
  if (t0 == 0 && a.state_out) {
    T* so = (T*)a.state_out + (int64_t)b * (K - 1) * E + c;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      store_v<T, V>(so + (int64_t)k * E, past_row<T, V, K>(x, a.x_ts, state, E, len - (K - 1) + k));
    }
  }
}

// One thread walks tokens t of its run and K - 1 behind it: dp_t completes
// dx_{t-K+1}.  The run's own tokens add to dw and db, which the block joins
// in shared memory row by row and writes to parts[run block][(K + 1) * E].
template <typename T, int V, int K>
__global__ void __launch_bounds__(kConvThreads, 2) k_conv_backward(const boa_conv_args a, const ConvRuns r,
                                                                   float* __restrict__ parts, int64_t run_blocks) {
  using Rows = ConvRows<T, V>;
  constexpr int kDepth = conv_depth<T, V>();
  extern __shared__ __align__(16) uint8_t smem[];
  Rows ax(smem, threadIdx.x, kConvThreads), ag(smem + Rows::bytes(kConvThreads), threadIdx.x, kConvThreads);
  float* const joined = reinterpret_cast<float*>(smem);   // [K + 1][V][bx], behind the last row
  const int gx = threadIdx.x % r.bx, ty = threadIdx.x / r.bx;
  const int cg = (blockIdx.x % r.group_blocks) * r.bx + gx;
  const int64_t rb = blockIdx.x / r.group_blocks;
  const int c = cg * V, E = a.channels;
  const bool on = cg < r.groups;
  Fv<V> w[K], bias, dw[K], db = splat<V>(0.0f);
  load_weights<V, K>(a, c, on, w, bias);
#pragma unroll
  for (int k = 0; k < K; ++k) dw[k] = splat<V>(0.0f);
  const int64_t total = (int64_t)a.batch * r.n_runs;
  for (int64_t rid = rb * r.by + ty; on && rid < total; rid += run_blocks * r.by) {
    const int b = (int)(rid / r.n_runs), t0 = (int)(rid % r.n_runs) * r.run;
    const int len = a.lens ? min(max(a.lens[b], 0), a.length) : a.length;
    const int t1 = min(t0 + r.run, a.length);
    const T* x = (const T*)a.x + b * a.x_bs + c;
    const T* state = a.state ? (const T*)a.state + (int64_t)b * (K - 1) * E + c : nullptr;
    const T* dso = a.dstate_out ? (const T*)a.dstate_out + (int64_t)b * (K - 1) * E + c : nullptr;
    T* dx = (T*)a.dx + (int64_t)b * a.length * E + c;
    T* ds = a.dstate ? (T*)a.dstate + (int64_t)b * (K - 1) * E + c : nullptr;
    const int stop = t1 + K - 1;
    // tokens t0 + K - 1 .. min(stop, len) come through the rings: rows t - (K - 1) in front of the last K - 1
    const T* px = x + (int64_t)t0 * a.x_ts;
    const T* pg = (const T*)a.dy + b * a.dy_bs + (int64_t)t0 * a.dy_ts + c;
    const int n = max(min(stop, len) - (t0 + K - 1), 0) / kConvUnroll;
    const int64_t xg = kConvUnroll * a.x_ts, gg = kConvUnroll * a.dy_ts;
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      if (i < n) {
        ax.start((ax.slot + i) % kDepth, px + (K - 1) * a.x_ts + i * xg, a.x_ts);
        ag.start((ax.slot + i) % kDepth, pg + (K - 1) * a.dy_ts + i * gg, a.dy_ts);
      }
      Rows::commit();
    }
    Words<T, V> none, hx[K - 1], hg[K - 1];
    none.clear();
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      hx[k] = hg[k] = none;
      if (t0 + k < len && t0 + k < stop) {
        hx[k].load(px + k * a.x_ts);
        hg[k].load(pg + k * a.dy_ts);
      }
    }
    Fv<V> win[K - 1], dp[K - 1];   // the K - 1 rows, and dp, before the next token
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      win[k] = t0 < len ? past_row<T, V, K>(x, a.x_ts, state, E, t0 - (K - 1) + k) : splat<V>(0.0f);
      dp[k] = splat<V>(0.0f);
    }
    // token t: its dp from the row and dy, and o = sum_k w_k dp_{t-k}, the gradient of row t - (K - 1)
    auto token = [&](const Words<T, V>& rx, const Words<T, V>& rg, bool mine) {
      const Fv<V> v = values<T, V>(rx);
      Fv<V> d = values<T, V>(rg);
      if (a.silu) {
        const Fv<V> p = conv_dot<V, K>(w, bias, win, v), s = vsigmoid<V>(p);
        // silu'(p) = s (1 + p (1 - s))
        d = vmul(vmul(d, s), vfma(p, vfma(s, splat<V>(-1.0f), splat<V>(1.0f)), splat<V>(1.0f)));
      }
      if (mine) {
        db = vadd(db, d);
#pragma unroll
        for (int k = 0; k < K - 1; ++k) dw[k] = vfma(d, win[k], dw[k]);
        dw[K - 1] = vfma(d, v, dw[K - 1]);
      }
      push<V, K>(win, v);
      // w_k multiplies dp_{t-k}: dp[i] is dp_{t-(K-1)+i}
      Fv<V> o = vmul(w[0], d);
#pragma unroll
      for (int k = 1; k < K; ++k) o = vfma(w[k], dp[K - 1 - k], o);
      push<V, K>(dp, d);
      return o;
    };
    int t = t0;
    // behind the row's end dp is 0, and rows of the final window also take dstate_out
    auto edge = [&](const Words<T, V>& rx, const Words<T, V>& rg) {
      const int s = t - (K - 1), tail = t - len;
      Fv<V> o = token(rx, rg, t < t1);
      px += a.x_ts;
      pg += a.dy_ts;
      if (dso && tail >= 0 && tail < K - 1) o = vadd(o, values<T, V>(raw_at<T, V>(dso + (int64_t)tail * E)));
      if (s >= t0) store_v<T, V>(dx + (int64_t)s * E, s < len ? o : splat<V>(0.0f));
      else if (s < 0 && ds) store_v<T, V>(ds + (int64_t)(s + K - 1) * E, o);
      ++t;
    };
#pragma unroll
    for (int k = 0; k < K - 1; ++k)
      if (t < stop) edge(hx[k], hg[k]);
    T* po = dx + (int64_t)(t - (K - 1)) * E;
    for (int i = 0; i < n; ++i) {
      Words<T, V> rx[kConvUnroll], rg[kConvUnroll];
      Rows::wait();
      ax.take(px, a.x_ts, rx);
      ag.take(pg, a.dy_ts, rg);
      if (i + kDepth < n) {
        ax.start(ax.slot, px + kDepth * xg, a.x_ts);
        ag.start(ax.slot, pg + kDepth * gg, a.dy_ts);
      }
      Rows::commit();
      ax.next();
      ag.next();
      px += xg;
      pg += gg;
#pragma unroll
      for (int u = 0; u < kConvUnroll; ++u) {
        store_v<T, V>(po, token(rx[u], rg[u], t + u < t1));
        po += E;
      }
      t += kConvUnroll;
    }
    while (t < stop) edge(t < len ? raw_at<T, V>(px) : none, t < len ? raw_at<T, V>(pg) : none);
  }
  constexpr int P = (K + 1) * V;
  __syncthreads();
  for (int k = 0; k < r.by; ++k) {
    if (ty == k) {
#pragma unroll
      for (int i = 0; i <= K; ++i) {
        float v[V];
        to_array<V>(i < K ? dw[i < K ? i : 0] : db, v);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float* p = &joined[(i * V + j) * r.bx + gx];
          *p = (k ? *p : 0.0f) + v[j];
        }
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
      if (k < K) out[(int64_t)(c + j) * K + k] = v;
      else out[(int64_t)K * E + c + j] = v;
    }
  }
}

// One token of ROWS streams a thread: the weights are read once for all of
// them, and their windows are in flight together.
template <typename T, int V, int K, int ROWS>
__global__ void __launch_bounds__(kConvThreads) k_conv_step(const boa_conv_args a, int groups) {
  const int64_t i = (int64_t)blockIdx.x * kConvThreads + threadIdx.x;
  const int c = (int)(i % groups) * V, E = a.channels;
  const int64_t b0 = i / groups * ROWS;
  if (b0 >= a.batch) return;
  const int n = (int)min((int64_t)ROWS, a.batch - b0);
  T* const st = (T*)a.state_out + b0 * (K - 1) * E + c;
  Words<T, V> win[ROWS][K];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
    if (r < n) {
#pragma unroll
      for (int k = 0; k < K - 1; ++k) win[r][k].load(st + (int64_t)(r * (K - 1) + k) * E);
      win[r][K - 1].load((const T*)a.x + (b0 + r) * a.x_bs + c);
    }
  Fv<V> w[K], bias;
  load_weights<V, K>(a, c, true, w, bias);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (r >= n) break;
    Fv<V> p = bias;
#pragma unroll
    for (int k = 0; k < K; ++k) p = vfma(w[k], values<T, V>(win[r][k]), p);
    if (a.silu) p = vmul(p, vsigmoid<V>(p));
#pragma unroll
    for (int k = 0; k < K - 1; ++k) win[r][k + 1].store(st + (int64_t)(r * (K - 1) + k) * E);
    store_v<T, V>((T*)a.y + (b0 + r) * E + c, p);
  }
}

// Tokens a run: long runs read less halo, short ones give `want` threads when
// the sequences are few.
static ConvRuns conv_runs(const boa_conv_args& a, int V, int64_t want) {
  ConvRuns r{};
  r.groups = (a.channels + V - 1) / V;
  r.bx = 1;
  while (r.bx < r.groups && r.bx < 32) r.bx *= 2;
  r.by = kConvThreads / r.bx;
  r.group_blocks = (r.groups + r.bx - 1) / r.bx;
  r.run = 128;
  while (r.run > 16 && (int64_t)a.batch * r.groups * ((a.length + r.run - 1) / r.run) < want) r.run /= 2;
  r.n_runs = a.length > 0 ? (a.length + r.run - 1) / r.run : 1;
  r.run_blocks = ((int64_t)a.batch * r.n_runs + r.by - 1) / r.by;
  return r;
}
// Forward: a few waves of blocks, so that the last one is short.  Backward: about
// four rounds of the blocks that the SMs hold (512 threads each, by registers).
static ConvRuns runs_forward(const boa_conv_args& a, int V) { return conv_runs(a, V, 148LL * 2048); }
static ConvRuns runs_backward(const boa_conv_args& a, int V) { return conv_runs(a, V, 148LL * 800); }

// Whether every row of every tensor starts on a vector of kConvVec elements.
static bool conv_vec(const boa_conv_args& a, bool backward, bool step) {
  const int V = kConvVec;
  const size_t n = V * (a.dtype == BOA_DTYPE_F32 ? 4 : 2);
  if (a.channels % V || a.x_bs % V || (!step && a.x_ts % V) || !aligned(a.x, n)) return false;
  if (!aligned(a.state, n) || !aligned(a.state_out, n)) return false;
  if (!backward) return aligned(a.y, n);
  return a.dy_bs % V == 0 && a.dy_ts % V == 0 && aligned(a.dy, n) && aligned(a.dx, n) && aligned(a.dstate_out, n) &&
         aligned(a.dstate, n);
}

// Blocks along the runs in the backward kernel, each with a row of partial
// sums in the workspace: the two that an SM holds stay and take run after run.
static int64_t conv_backward_blocks(const ConvRuns& r) {
  const int64_t most = r.group_blocks < 296 ? 296 / r.group_blocks : 1;
  return r.run_blocks < most ? r.run_blocks : most;
}

template <typename T, int V, int K>
static int conv_launch(const boa_conv_args& a, int what, cudaStream_t s) {
  using Rows = ConvRows<T, V>;
  if (what == 2) {
    const int groups = (a.channels + V - 1) / V;
    // four streams a thread where that still fills the GPU, else one
    if ((int64_t)a.batch * groups >= 4 * 148LL * 512) {
      const int64_t n = (a.batch + 3LL) / 4 * groups;
      k_conv_step<T, V, K, 4><<<(unsigned)((n + kConvThreads - 1) / kConvThreads), kConvThreads, 0, s>>>(a, groups);
    } else {
      const int64_t n = (int64_t)a.batch * groups;
      k_conv_step<T, V, K, 1><<<(unsigned)((n + kConvThreads - 1) / kConvThreads), kConvThreads, 0, s>>>(a, groups);
    }
  } else if (what == 0) {
    const ConvRuns r = runs_forward(a, V);
    k_conv<T, V, K><<<(unsigned)(r.run_blocks * r.group_blocks), kConvThreads, Rows::bytes(kConvThreads), s>>>(a, r);
  } else {
    const ConvRuns r = runs_backward(a, V);
    const int64_t blocks = conv_backward_blocks(r);
    float* parts = (float*)a.workspace;
    const size_t join = (size_t)(K + 1) * V * r.bx * sizeof(float), rows = 2 * Rows::bytes(kConvThreads);
    const size_t smem = join > rows ? join : rows;
    if (smem > 48 * 1024)
      BOA_CUDA(cudaFuncSetAttribute(k_conv_backward<T, V, K>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    k_conv_backward<T, V, K><<<(unsigned)(blocks * r.group_blocks), kConvThreads, smem, s>>>(a, r, parts, blocks);
    const int64_t cols = (K + 1LL) * a.channels;
    k_sum_parts<<<(unsigned)((cols + 31) / 32), 1024, 0, s>>>(parts, blocks, cols, (int64_t)K * a.channels, cols,
                                                             a.dweight, a.dbias, nullptr);
  }
  BOA_CUDA(cudaGetLastError());
  return BOA_OK;
}

template <typename T, int K>
static int conv_by_vector(const boa_conv_args& a, int what, cudaStream_t s) {
  if (conv_vec(a, what == 1, what == 2)) return conv_launch<T, kConvVec, K>(a, what, s);
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
  if (a->length > kMaxSize || a->channels > kMaxSize)
    return boa_fail(BOA_ERR_UNSUPPORTED, std::string(who) + ": length and channels must be below 2^31 - 2^16");
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
  if (!aligned(a->weight, 16)) return boa_fail(BOA_ERR_ARG, "boa_causal_conv: weight must be 16-byte aligned");
  return conv_dispatch(*a, 0, stream);
}

BOA_API size_t boa_causal_conv_workspace_bytes(const boa_conv_args* a) {
  if (conv_check(a, "boa_causal_conv_workspace_bytes")) return 0;
  // the single-element form has the most channel vectors and blocks of rows; take the larger of the two
  const ConvRuns r1 = runs_backward(*a, 1);
  const ConvRuns rv = runs_backward(*a, kConvVec);
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
  if (!aligned(a->weight, 16))
    return boa_fail(BOA_ERR_ARG, "boa_causal_conv_backward: weight must be 16-byte aligned");
  if (!a->workspace || a->workspace_bytes < boa_causal_conv_workspace_bytes(a))
    return boa_fail(BOA_ERR_ARG, "boa_causal_conv_backward: workspace too small (see boa_causal_conv_workspace_bytes)");
  return conv_dispatch(*a, 1, stream);
}

BOA_API int boa_causal_conv_step(const boa_conv_args* a, void* stream) {
  const int rc = conv_check(a, "boa_causal_conv_step");
  if (rc) return rc;
  if (a->batch == 0) return BOA_OK;
  if (!a->x || !a->weight || !a->state_out || !a->y) return boa_fail(BOA_ERR_ARG, "boa_causal_conv_step: null argument");
  if (!aligned(a->weight, 16)) return boa_fail(BOA_ERR_ARG, "boa_causal_conv_step: weight must be 16-byte aligned");
  return conv_dispatch(*a, 2, stream);
}

}  // extern "C"
