// Selective state space scan with 16 states a channel: forward, backward and
// one token per stream.
//
//   d = softplus(dt + bias), a = exp(d A)
//   h_t = a_t h_{t-1} + d_t x_t B_t,  v_t = C_t . h_t + D x_t,  y = v silu(z)
//   g = dy silu(z),  dz = dy v silu'(z),  e_t = g_t C_t + a_{t+1} e_{t+1}
//   dC_t = sum_e g h,  dB_t = sum_e e d x,  s1 = sum_n e B,  q = e a h_{t-1}
//   dx = s1 d + D g,  ddt = (s1 x + sum_n q A) sigmoid(dt + bias),  dA = sum_t q d
//
// Four lanes share a channel, four states each; a warp covers 8 channels and a
// block 32.  Tiles of tokens are staged in shared memory as fp32 with softplus
// and the gate applied once an element.  Sequences too few to fill the GPU are
// split over their length: every part's end state is found from a zero start
// (k_ssm_ends), the parts are chained (k_ssm_join: a part's decay is
// exp(A sum d), so one number a channel carries it), and the parts then run from
// their true start states.  That doubles the exponentials, so few parts are
// taken.  The backward call does the same with the gradient of the state, in
// reverse, and restarts h from checkpoints every 8 tokens that the forward call
// leaves.
#include "seq_common.cuh"

namespace boa {
namespace seq {

constexpr int kN = 16;            // states
constexpr int kQ = 4;             // states a lane
constexpr int kCh = 32;           // channels a block pass
constexpr int kSsmThreads = 128;
constexpr int kTile = 16;         // tokens a forward tile
constexpr int kBack = 8;          // tokens a backward tile, and between checkpoints
constexpr int kPitch = 40;        // floats of a staged row: 8 mod 32, so 4 rows x 8 channels hit 32 banks
constexpr int kPasses = 8;        // channel passes of a backward block
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float softplus_of(float v) { return v > 20.0f ? v : log1pf(expf(v)); }
__device__ __forceinline__ float sigmoid_of(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

__device__ __forceinline__ int row_len(const boa_ssm_args& a, int b) {
  return a.lens ? min(max(a.lens[b], 0), a.length) : a.length;
}

// Two neighbouring channels of a token row; zeros where the token or the
// channel does not exist.  `pair`: every row starts on a pair boundary.
template <typename T>
__device__ __forceinline__ Vec<T, 2> load_pair(const T* row, int c, int E, bool live, bool pair) {
  Vec<T, 2> r;
  r.v[0] = from_f<T>(0.0f);
  r.v[1] = from_f<T>(0.0f);
  if (live) {
    if (pair) {
      if (c < E) r = *reinterpret_cast<const Vec<T, 2>*>(row + c);
    } else {
      if (c < E) r.v[0] = row[c];
      if (c + 1 < E) r.v[1] = row[c + 1];
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store_pair(T* row, int c, int E, float v0, float v1, bool pair) {
  if (pair) {
    if (c < E) {
      const float v[2] = {v0, v1};
      store_f<T, 2>(row + c, v);
    }
  } else {
    if (c < E) row[c] = from_f<T>(v0);
    if (c + 1 < E) row[c + 1] = from_f<T>(v1);
  }
}

// Sums of four values over the four lanes of a channel: lane q gets that of v[q].
__device__ __forceinline__ float quad_sum(const float (&v)[4], int q) {
  const bool hi = q & 2, odd = q & 1;
  float k0 = hi ? v[2] : v[0], k1 = hi ? v[3] : v[1];
  k0 += __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[2], 2);
  k1 += __shfl_xor_sync(0xffffffffu, hi ? v[1] : v[3], 2);
  return (odd ? k1 : k0) + __shfl_xor_sync(0xffffffffu, odd ? k0 : k1, 1);
}

struct SsmPlan {
  int cblocks;      // blocks (of 32 channels) of a row
  int parts, part;  // parts of a sequence, tokens of a part
  bool pair;        // two-element accesses
};

template <typename T>
struct RawTile {
  Vec<T, 2> x[2], dt[2], z[2];
  float bc[4];
};

// ------------------------------------------------------------------ forward
// ENDS: only the part's end state (from zero) and sum of d, into ends / dsum.
template <typename T, bool ENDS>
__global__ void __launch_bounds__(kSsmThreads) k_ssm(const boa_ssm_args a, const SsmPlan p, float* __restrict__ ends,
                                                     float* __restrict__ dsum) {
  __shared__ __align__(16) float sd[kTile][kPitch], su[kTile][kPitch], sy[kTile][kPitch];
  __shared__ __align__(16) float sbc[kTile][2 * kN];
  const int tid = threadIdx.x, lane = tid & 31, q = lane & 3, ch = (tid >> 5) * 8 + (lane >> 2);
  const int nparts = ENDS ? p.parts - 1 : p.parts;
  const int e0 = (blockIdx.x % p.cblocks) * kCh, E = a.channels;
  const int part = (blockIdx.x / p.cblocks) % nparts, b = blockIdx.x / p.cblocks / nparts;
  const int e = e0 + ch;
  const bool on = e < E;
  const int len = row_len(a, b);
  const int begin = part * p.part, stop = min(begin + p.part, a.length), end = min(stop, len);
  const int64_t slot = ((int64_t)b * p.parts + part) * E + e;
  // staging: a thread moves two channels of tokens row and row + 8, and four values of B or C
  const int row = tid >> 4, c = e0 + 2 * (tid & 15), cl = 2 * (tid & 15);
  const int brow = tid >> 3, bsub = tid & 7;
  const T* px = (const T*)a.x + b * a.x_bs;
  const T* pd = (const T*)a.dt + b * a.dt_bs;
  const T* pz = a.z ? (const T*)a.z + b * a.z_bs : nullptr;
  const T* pbc = bsub < 4 ? (const T*)a.B + b * a.B_bs + 4 * bsub : (const T*)a.C + b * a.C_bs + 4 * (bsub - 4);
  const int64_t bcts = bsub < 4 ? a.B_ts : a.C_ts;
  const bool want_bc = !ENDS || bsub < 4;
  float bias[2], Dv[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    bias[j] = a.dt_bias && c + j < E ? a.dt_bias[c + j] : 0.0f;
    Dv[j] = a.D && c + j < E ? a.D[c + j] : 0.0f;
  }
  float A2[kQ], h[kQ];
#pragma unroll
  for (int j = 0; j < kQ; ++j) {
    A2[j] = on ? a.A[(int64_t)e * kN + kQ * q + j] * kLog2e : 0.0f;
    h[j] = 0.0f;
    if (!ENDS && on) {
      if (p.parts > 1) h[j] = ends[slot * kN + kQ * q + j];
      else if (a.state) h[j] = a.state[((int64_t)b * E + e) * kN + kQ * q + j];
    }
  }
  float total = 0.0f;
  RawTile<T> r;
  auto fetch = [&](int t0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = t0 + row + 8 * i;
      const bool live = t < end;
      r.x[i] = load_pair<T>(px + (int64_t)t * a.x_ts, c, E, live, p.pair);
      r.dt[i] = load_pair<T>(pd + (int64_t)t * a.dt_ts, c, E, live, p.pair);
      if (!ENDS && pz) r.z[i] = load_pair<T>(pz + (int64_t)t * a.z_ts, c, E, live, p.pair);
    }
    const int t = t0 + brow;
#pragma unroll
    for (int j = 0; j < 4; ++j) r.bc[j] = want_bc && t < end ? to_f(pbc[(int64_t)t * bcts + j]) : 0.0f;
  };
  if (begin < end) fetch(begin);
  for (int t0 = begin; t0 < end; t0 += kTile) {
    float xs[2][2], zs[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bool live = t0 + row + 8 * i < end && c + j < E;
        const float raw = to_f(r.dt[i].v[j]) + bias[j];
        const float d = live ? (a.softplus ? softplus_of(raw) : raw) : 0.0f;
        xs[i][j] = to_f(r.x[i].v[j]);
        zs[i][j] = !ENDS && pz ? to_f(r.z[i].v[j]) : 0.0f;
        sd[row + 8 * i][cl + j] = d;
        su[row + 8 * i][cl + j] = d * xs[i][j];
      }
    *reinterpret_cast<float4*>(&sbc[brow][4 * bsub]) = make_float4(r.bc[0], r.bc[1], r.bc[2], r.bc[3]);
    __syncthreads();
    if (t0 + kTile < end) fetch(t0 + kTile);
#pragma unroll
    for (int u = 0; u < kTile; u += 4) {
      float yp[4];
      if (!ENDS && a.checkpoints && u % kBack == 0 && on && t0 + u < end) {
        const int64_t nck = (a.length + kBack - 1) / kBack;
        *reinterpret_cast<float4*>(a.checkpoints + (((int64_t)b * nck + (t0 + u) / kBack) * E + e) * kN + kQ * q) =
            make_float4(h[0], h[1], h[2], h[3]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float d = sd[u + k][ch], du = su[u + k][ch];
        const float4 B4 = *reinterpret_cast<const float4*>(&sbc[u + k][kQ * q]);
        const float Bv[4] = {B4.x, B4.y, B4.z, B4.w};
#pragma unroll
        for (int j = 0; j < kQ; ++j) h[j] = fmaf(ex2(d * A2[j]), h[j], du * Bv[j]);
        if constexpr (ENDS) {
          total += d;
        } else {
          const float4 C4 = *reinterpret_cast<const float4*>(&sbc[u + k][kN + kQ * q]);
          yp[k] = fmaf(C4.x, h[0], fmaf(C4.y, h[1], fmaf(C4.z, h[2], C4.w * h[3])));
        }
      }
      if constexpr (!ENDS) sy[u + q][ch] = quad_sum(yp, q);
    }
    __syncthreads();
    if constexpr (!ENDS) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = t0 + row + 8 * i;
        if (t < stop) {
          float o[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            o[j] = fmaf(Dv[j], xs[i][j], sy[row + 8 * i][cl + j]);
            if (pz) o[j] *= zs[i][j] * sigmoid_of(zs[i][j]);
            if (t >= end) o[j] = 0.0f;
          }
          store_pair<T>((T*)a.y + ((int64_t)b * a.length + t) * E, c, E, o[0], o[1], p.pair);
        }
      }
    }
  }
  if constexpr (ENDS) {
    if (on) {
      *reinterpret_cast<float4*>(ends + slot * kN + kQ * q) = make_float4(h[0], h[1], h[2], h[3]);
      if (q == 0) dsum[slot] = total;
    }
  } else {
    // tiles wholly behind the row's end
    const int done = begin + (max(end - begin, 0) + kTile - 1) / kTile * kTile;
    for (int t = done + row; t < stop; t += 8)
      store_pair<T>((T*)a.y + ((int64_t)b * a.length + t) * E, c, E, 0.0f, 0.0f, p.pair);
    if (a.state_out && part == p.parts - 1 && on) {
      float* so = a.state_out + ((int64_t)b * E + e) * kN + kQ * q;
#pragma unroll
      for (int j = 0; j < kQ; ++j) so[j] = h[j];
    }
  }
}

// Chains the parts of every (row, channel, state): ends[] becomes the value
// each part starts from.  Forward: from the first part with h; backward
// (`reverse`): from the last part with the gradient of the state.
static __global__ void __launch_bounds__(256) k_ssm_join(int64_t n, int E, int parts, const float* __restrict__ A,
                                                         const float* __restrict__ first, float* __restrict__ ends,
                                                         const float* __restrict__ dsum, bool reverse) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t en = (int64_t)E * kN;
  const int64_t b = i / en, r = i % en;
  const float A2 = A[r] * kLog2e;
  float carry = first ? first[i] : 0.0f;
  for (int k = 0; k < parts; ++k) {
    const int s = reverse ? parts - 1 - k : k;
    const int64_t at = (b * parts + s) * en + r;
    float own = 0.0f, decay = 0.0f;
    if (k < parts - 1) {
      own = ends[at];
      decay = ex2(A2 * dsum[(b * parts + s) * E + r / kN]);
    }
    ends[at] = carry;
    carry = fmaf(decay, carry, own);
  }
}

// ----------------------------------------------------------------- backward
// The gradient of the state that a part passes on to the part before it, from
// a zero start at its end, and the part's sum of d.
template <typename T>
__global__ void __launch_bounds__(kSsmThreads) k_ssm_back_ends(const boa_ssm_args a, const SsmPlan p,
                                                               float* __restrict__ ends, float* __restrict__ dsum) {
  __shared__ __align__(16) float sd[kTile][kPitch], sg[kTile][kPitch];
  __shared__ __align__(16) float sc[kTile][kN];
  const int tid = threadIdx.x, lane = tid & 31, q = lane & 3, ch = (tid >> 5) * 8 + (lane >> 2);
  const int e0 = (blockIdx.x % p.cblocks) * kCh, E = a.channels;
  const int part = 1 + (blockIdx.x / p.cblocks) % (p.parts - 1), b = blockIdx.x / p.cblocks / (p.parts - 1);
  const int e = e0 + ch;
  const bool on = e < E;
  const int begin = part * p.part, end = min(min(begin + p.part, a.length), row_len(a, b));
  const int64_t slot = ((int64_t)b * p.parts + part) * E + e;
  const int row = tid >> 4, c = e0 + 2 * (tid & 15), cl = 2 * (tid & 15);
  const int brow = tid >> 3, bsub = tid & 7;
  const T* pg = (const T*)a.dy + b * a.dy_bs;
  const T* pd = (const T*)a.dt + b * a.dt_bs;
  const T* pz = a.z ? (const T*)a.z + b * a.z_bs : nullptr;
  const T* pc = (const T*)a.C + b * a.C_bs + 4 * (bsub & 3);
  float bias[2], A2[kQ], g4[kQ] = {};
#pragma unroll
  for (int j = 0; j < 2; ++j) bias[j] = a.dt_bias && c + j < E ? a.dt_bias[c + j] : 0.0f;
#pragma unroll
  for (int j = 0; j < kQ; ++j) A2[j] = on ? a.A[(int64_t)e * kN + kQ * q + j] * kLog2e : 0.0f;
  float total = 0.0f;
  RawTile<T> r;   // x holds dy
  auto fetch = [&](int t0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = t0 + row + 8 * i;
      const bool live = t < end;
      r.x[i] = load_pair<T>(pg + (int64_t)t * a.dy_ts, c, E, live, p.pair);
      r.dt[i] = load_pair<T>(pd + (int64_t)t * a.dt_ts, c, E, live, p.pair);
      if (pz) r.z[i] = load_pair<T>(pz + (int64_t)t * a.z_ts, c, E, live, p.pair);
    }
    const int t = t0 + brow;
#pragma unroll
    for (int j = 0; j < 4; ++j) r.bc[j] = bsub < 4 && t < end ? to_f(pc[(int64_t)t * a.C_ts + j]) : 0.0f;
  };
  const int tiles = (max(end - begin, 0) + kTile - 1) / kTile;
  if (tiles) fetch(begin + (tiles - 1) * kTile);
  for (int k = tiles - 1; k >= 0; --k) {
    const int t0 = begin + k * kTile;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bool live = t0 + row + 8 * i < end && c + j < E;
        const float raw = to_f(r.dt[i].v[j]) + bias[j];
        float g = to_f(r.x[i].v[j]);
        if (pz) {
          const float z = to_f(r.z[i].v[j]);
          g *= z * sigmoid_of(z);
        }
        sd[row + 8 * i][cl + j] = live ? (a.softplus ? softplus_of(raw) : raw) : 0.0f;
        sg[row + 8 * i][cl + j] = live ? g : 0.0f;
      }
    if (bsub < 4)
      *reinterpret_cast<float4*>(&sc[brow][4 * bsub]) = make_float4(r.bc[0], r.bc[1], r.bc[2], r.bc[3]);
    __syncthreads();
    if (k > 0) fetch(t0 - kTile);
#pragma unroll
    for (int t = kTile - 1; t >= 0; --t) {
      const float d = sd[t][ch], g = sg[t][ch];
      const float4 C4 = *reinterpret_cast<const float4*>(&sc[t][kQ * q]);
      const float Cv[4] = {C4.x, C4.y, C4.z, C4.w};
#pragma unroll
      for (int j = 0; j < kQ; ++j) g4[j] = ex2(d * A2[j]) * fmaf(Cv[j], g, g4[j]);
      total += d;
    }
    __syncthreads();
  }
  if (on) {
    *reinterpret_cast<float4*>(ends + slot * kN + kQ * q) = make_float4(g4[0], g4[1], g4[2], g4[3]);
    if (q == 0) dsum[slot] = total;
  }
}

// Shared memory of the backward kernel, in floats.
struct BackSmem {
  static constexpr int tile = kBack * kPitch;
  static constexpr int sd = 0, su = sd + tile, sg = su + tile, s1 = sg + tile, s2 = s1 + tile, sv = s2 + tile,
                       sbc = sv + tile, red = sbc + kBack * 2 * kN, carry = red + 4 * kBack * 2 * kN;
  // per channel of the block: dh[16], dA[16], and dD, dbias by staging row
  static constexpr int per_channel = 2 * kN + 2 * kBack;
  __host__ __device__ static constexpr int floats(int passes) { return carry + passes * kCh * per_channel; }
};

template <typename T>
struct RawBack {
  Vec<T, 2> x, dt, z, g;
  float4 h;
};

// A block takes one part of a row and up to 256 channels, tile by tile from
// the end, 32 channels a pass.  A pass recomputes h over the tile from its
// checkpoint (a and h stay in registers), then runs the gradient backwards.
// dB and dC of the tile gather over the passes in registers and are summed
// over the block's lanes and warps once a tile.
template <typename T>
__global__ void __launch_bounds__(kSsmThreads, 3)
    k_ssm_backward(const boa_ssm_args a, const SsmPlan p, int passes, int groups, const float* __restrict__ starts,
                   float* __restrict__ bc_parts, float* __restrict__ param_parts) {
  extern __shared__ __align__(16) float sm[];
  using S = BackSmem;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, q = lane & 3, ch = warp * 8 + (lane >> 2);
  const int E = a.channels, group = blockIdx.x % groups;
  const int part = (blockIdx.x / groups) % p.parts, b = blockIdx.x / groups / p.parts;
  const int e0 = group * passes * kCh;
  const int np = min(passes, (E - e0 + kCh - 1) / kCh);
  const int len = row_len(a, b);
  const int begin = part * p.part, stop = min(begin + p.part, a.length), end = min(stop, len);
  const int nck = (a.length + kBack - 1) / kBack;
  const int row = tid >> 4, cl = 2 * (tid & 15);
  const int brow = tid >> 4, bsub = tid & 15;    // two values of B or C
  const T* px = (const T*)a.x + b * a.x_bs;
  const T* pd = (const T*)a.dt + b * a.dt_bs;
  const T* pz = a.z ? (const T*)a.z + b * a.z_bs : nullptr;
  const T* pg = (const T*)a.dy + b * a.dy_bs;
  const T* pbc = bsub < 8 ? (const T*)a.B + b * a.B_bs + 2 * bsub : (const T*)a.C + b * a.C_bs + 2 * (bsub - 8);
  const int64_t bcts = bsub < 8 ? a.B_ts : a.C_ts;
  const int64_t orow = (int64_t)b * a.length;
  float* dh_s = sm + S::carry;
  float* dA_s = dh_s + passes * kCh * kN;
  float* dD_s = dA_s + passes * kCh * kN;           // [row][channel]
  float* db_s = dD_s + passes * kCh * kBack;
  for (int g = 0; g < np; ++g) {
    const int e = e0 + g * kCh + ch;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (e < E) {
      if (p.parts > 1) {
        v = *reinterpret_cast<const float4*>(starts + (((int64_t)b * p.parts + part) * E + e) * kN + kQ * q);
      } else if (a.dstate_out) {
        const float* s = a.dstate_out + ((int64_t)b * E + e) * kN + kQ * q;
        v = make_float4(s[0], s[1], s[2], s[3]);
      }
    }
    *reinterpret_cast<float4*>(dh_s + (g * kCh + ch) * kN + kQ * q) = v;
    *reinterpret_cast<float4*>(dA_s + (g * kCh + ch) * kN + kQ * q) = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      dD_s[row * passes * kCh + g * kCh + cl + j] = 0.0f;
      db_s[row * passes * kCh + g * kCh + cl + j] = 0.0f;
    }
  }
  const int tiles = (max(end - begin, 0) + kBack - 1) / kBack;
  RawBack<T> r;
  auto fetch = [&](int t0, int g) {
    const int t = t0 + row, c = e0 + g * kCh + cl;
    const bool live = t < end;
    r.x = load_pair<T>(px + (int64_t)t * a.x_ts, c, E, live, p.pair);
    r.dt = load_pair<T>(pd + (int64_t)t * a.dt_ts, c, E, live, p.pair);
    r.g = load_pair<T>(pg + (int64_t)t * a.dy_ts, c, E, live, p.pair);
    if (pz) r.z = load_pair<T>(pz + (int64_t)t * a.z_ts, c, E, live, p.pair);
    const int e = e0 + g * kCh + ch;
    r.h = make_float4(0.f, 0.f, 0.f, 0.f);
    if (e < E)
      r.h = *reinterpret_cast<const float4*>(a.checkpoints + (((int64_t)b * nck + t0 / kBack) * E + e) * kN + kQ * q);
  };
  if (tiles) fetch(begin + (tiles - 1) * kBack, 0);
  for (int k = tiles - 1; k >= 0; --k) {
    const int t0 = begin + k * kBack;
    float vB[kBack][kQ], vC[kBack][kQ];
#pragma unroll
    for (int t = 0; t < kBack; ++t)
#pragma unroll
      for (int j = 0; j < kQ; ++j) vB[t][j] = vC[t][j] = 0.0f;
    {
      const int t = t0 + brow;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        sm[S::sbc + brow * 2 * kN + 2 * bsub + j] = t < end ? to_f(pbc[(int64_t)t * bcts + j]) : 0.0f;
    }
    for (int g = 0; g < np; ++g) {
      const int c = e0 + g * kCh + cl, e = e0 + g * kCh + ch;
      const bool in_row = t0 + row < end;
      float xv[2], dv[2], gv[2], sig[2], dzf[2], Dv[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bool live = in_row && c + j < E;
        const float raw = to_f(r.dt.v[j]) + (a.dt_bias && c + j < E ? a.dt_bias[c + j] : 0.0f);
        Dv[j] = a.D && c + j < E ? a.D[c + j] : 0.0f;
        dv[j] = live ? (a.softplus ? softplus_of(raw) : raw) : 0.0f;
        sig[j] = a.softplus ? sigmoid_of(raw) : 1.0f;
        xv[j] = to_f(r.x.v[j]);
        gv[j] = to_f(r.g.v[j]);
        dzf[j] = 0.0f;
        if (pz) {
          const float z = to_f(r.z.v[j]), s = sigmoid_of(z);
          dzf[j] = gv[j] * (s * (1.0f + z * (1.0f - s)));
          gv[j] *= z * s;
        }
        sm[S::sd + row * kPitch + cl + j] = dv[j];
        sm[S::su + row * kPitch + cl + j] = dv[j] * xv[j];
        sm[S::sg + row * kPitch + cl + j] = gv[j];
      }
      const float4 h4 = r.h;
      __syncthreads();
      if (g + 1 < np) fetch(t0, g + 1);
      else if (k > 0) fetch(t0 - kBack, 0);
      float Av[kQ], A2[kQ], h0[kQ] = {h4.x, h4.y, h4.z, h4.w}, h[kBack][kQ], dec[kBack][kQ];
#pragma unroll
      for (int j = 0; j < kQ; ++j) {
        Av[j] = e < E ? a.A[(int64_t)e * kN + kQ * q + j] : 0.0f;
        A2[j] = Av[j] * kLog2e;
      }
      float yp[kBack];
#pragma unroll
      for (int t = 0; t < kBack; ++t) {
        const float d = sm[S::sd + t * kPitch + ch], du = sm[S::su + t * kPitch + ch];
        const float4 B4 = *reinterpret_cast<const float4*>(&sm[S::sbc + t * 2 * kN + kQ * q]);
        const float4 C4 = *reinterpret_cast<const float4*>(&sm[S::sbc + t * 2 * kN + kN + kQ * q]);
        const float Bv[4] = {B4.x, B4.y, B4.z, B4.w}, Cv[4] = {C4.x, C4.y, C4.z, C4.w};
        yp[t] = 0.0f;
#pragma unroll
        for (int j = 0; j < kQ; ++j) {
          dec[t][j] = ex2(d * A2[j]);
          h[t][j] = fmaf(dec[t][j], t ? h[t - 1][j] : h0[j], du * Bv[j]);
          yp[t] = fmaf(Cv[j], h[t][j], yp[t]);
        }
      }
      if (pz) {
        const float lo[4] = {yp[0], yp[1], yp[2], yp[3]}, hi[4] = {yp[4], yp[5], yp[6], yp[7]};
        sm[S::sv + q * kPitch + ch] = quad_sum(lo, q);
        sm[S::sv + (4 + q) * kPitch + ch] = quad_sum(hi, q);
      }
      float4 dh4 = *reinterpret_cast<const float4*>(dh_s + (g * kCh + ch) * kN + kQ * q);
      float4 dA4 = *reinterpret_cast<const float4*>(dA_s + (g * kCh + ch) * kN + kQ * q);
      float dh[4] = {dh4.x, dh4.y, dh4.z, dh4.w}, dA[4] = {dA4.x, dA4.y, dA4.z, dA4.w};
      float p1[4], p2[4];
#pragma unroll
      for (int t = kBack - 1; t >= 0; --t) {
        const float d = sm[S::sd + t * kPitch + ch], du = sm[S::su + t * kPitch + ch];
        const float gg = sm[S::sg + t * kPitch + ch];
        const float4 B4 = *reinterpret_cast<const float4*>(&sm[S::sbc + t * 2 * kN + kQ * q]);
        const float4 C4 = *reinterpret_cast<const float4*>(&sm[S::sbc + t * 2 * kN + kN + kQ * q]);
        const float Bv[4] = {B4.x, B4.y, B4.z, B4.w}, Cv[4] = {C4.x, C4.y, C4.z, C4.w};
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int j = 0; j < kQ; ++j) {
          dh[j] = fmaf(Cv[j], gg, dh[j]);
          vB[t][j] = fmaf(dh[j], du, vB[t][j]);
          vC[t][j] = fmaf(gg, h[t][j], vC[t][j]);
          s1 = fmaf(dh[j], Bv[j], s1);
          dh[j] *= dec[t][j];
          const float w = dh[j] * (t ? h[t - 1][j] : h0[j]);
          s2 = fmaf(w, Av[j], s2);
          dA[j] = fmaf(w, d, dA[j]);
        }
        p1[t & 3] = s1;
        p2[t & 3] = s2;
        if ((t & 3) == 0) {
          sm[S::s1 + (t + q) * kPitch + ch] = quad_sum(p1, q);
          sm[S::s2 + (t + q) * kPitch + ch] = quad_sum(p2, q);
        }
      }
      *reinterpret_cast<float4*>(dh_s + (g * kCh + ch) * kN + kQ * q) = make_float4(dh[0], dh[1], dh[2], dh[3]);
      *reinterpret_cast<float4*>(dA_s + (g * kCh + ch) * kN + kQ * q) = make_float4(dA[0], dA[1], dA[2], dA[3]);
      __syncthreads();
      if (t0 + row < stop) {
        float ox[2], od[2], oz[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int at = row * kPitch + cl + j;
          const float s1 = sm[S::s1 + at];
          ox[j] = fmaf(s1, dv[j], Dv[j] * gv[j]);
          od[j] = in_row ? fmaf(s1, xv[j], sm[S::s2 + at]) * sig[j] : 0.0f;
          oz[j] = pz ? dzf[j] * fmaf(Dv[j], xv[j], sm[S::sv + at]) : 0.0f;
          float* accD = &dD_s[row * passes * kCh + g * kCh + cl + j];
          float* accb = &db_s[row * passes * kCh + g * kCh + cl + j];
          *accD = fmaf(gv[j], xv[j], *accD);
          *accb += od[j];
        }
        const int64_t o = (orow + t0 + row) * E;
        store_pair<T>((T*)a.dx + o, c, E, ox[0], ox[1], p.pair);
        store_pair<T>((T*)a.ddt + o, c, E, od[0], od[1], p.pair);
        if (pz) store_pair<T>((T*)a.dz + o, c, E, oz[0], oz[1], p.pair);
      }
    }
    // the tile's dB and dC over the warp's 8 channels: lane bits 4, 3, 2 pick C, and the state within the lane's four
    const bool up = lane & 16, hi = lane & 8, odd = lane & 4;
#pragma unroll
    for (int t = 0; t < kBack; ++t) {
      float k4[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        k4[j] = (up ? vC[t][j] : vB[t][j]) + __shfl_xor_sync(0xffffffffu, up ? vB[t][j] : vC[t][j], 16);
      const float k0 = (hi ? k4[2] : k4[0]) + __shfl_xor_sync(0xffffffffu, hi ? k4[0] : k4[2], 8);
      const float k1 = (hi ? k4[3] : k4[1]) + __shfl_xor_sync(0xffffffffu, hi ? k4[1] : k4[3], 8);
      const float s = (odd ? k1 : k0) + __shfl_xor_sync(0xffffffffu, odd ? k0 : k1, 4);
      sm[S::red + (warp * kBack + t) * 2 * kN + (up ? kN : 0) + kQ * q + (hi ? 2 : 0) + (odd ? 1 : 0)] = s;
    }
    __syncthreads();
    for (int i = tid; i < kBack * 2 * kN; i += kSsmThreads) {
      const int t = t0 + i / (2 * kN);
      if (t < stop) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) s += sm[S::red + w * kBack * 2 * kN + i];
        bc_parts[(((int64_t)group * a.batch + b) * a.length + t) * 2 * kN + i % (2 * kN)] = s;
      }
    }
  }
  // tiles wholly behind the row's end
  for (int t = begin + tiles * kBack + row; t < stop; t += kBack) {
    const int64_t o = (orow + t) * E;
    for (int g = 0; g < np; ++g) {
      const int c = e0 + g * kCh + cl;
      store_pair<T>((T*)a.dx + o, c, E, 0.0f, 0.0f, p.pair);
      store_pair<T>((T*)a.ddt + o, c, E, 0.0f, 0.0f, p.pair);
      if (pz) store_pair<T>((T*)a.dz + o, c, E, 0.0f, 0.0f, p.pair);
    }
    float* bc = bc_parts + (((int64_t)group * a.batch + b) * a.length + t) * 2 * kN + 2 * (tid & 15);
    bc[0] = 0.0f;
    bc[1] = 0.0f;
  }
  __syncthreads();
  float* pp = param_parts + ((int64_t)b * p.parts + part) * E * (kN + 2);
  for (int g = 0; g < np; ++g) {
    const int e = e0 + g * kCh + ch;
    if (e < E) {
      const float* s = dA_s + (g * kCh + ch) * kN + kQ * q;
      const float* d = dh_s + (g * kCh + ch) * kN + kQ * q;
#pragma unroll
      for (int j = 0; j < kQ; ++j) {
        pp[(int64_t)e * kN + kQ * q + j] = s[j];
        if (part == 0 && a.dstate) a.dstate[((int64_t)b * E + e) * kN + kQ * q + j] = d[j];
      }
    }
  }
  for (int i = tid; i < np * kCh; i += kSsmThreads) {
    if (e0 + i < E) {
      float sD = 0.0f, sb = 0.0f;
#pragma unroll
      for (int k = 0; k < kBack; ++k) {
        sD += dD_s[k * passes * kCh + i];
        sb += db_s[k * passes * kCh + i];
      }
      pp[(int64_t)E * kN + e0 + i] = sD;
      pp[(int64_t)E * (kN + 1) + e0 + i] = sb;
    }
  }
}

// dB and dC from the channel groups' sums.
template <typename T>
__global__ void __launch_bounds__(256) k_ssm_bc(int64_t rows, int groups, const float* __restrict__ parts,
                                                T* __restrict__ dB, T* __restrict__ dC) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t n = rows * 2 * kN;
  if (i >= n) return;
  float s = 0.0f;
  for (int g = 0; g < groups; ++g) s += parts[g * n + i];
  const int64_t r = i / (2 * kN);
  const int k = (int)(i % (2 * kN));
  if (k < kN) dB[r * kN + k] = from_f<T>(s);
  else dC[r * kN + k - kN] = from_f<T>(s);
}

// --------------------------------------------------------------- one token
template <typename T>
__global__ void __launch_bounds__(256) k_ssm_step(const boa_ssm_args a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t n = (int64_t)a.batch * a.channels * 4;
  const bool on = i < n;
  const int64_t be = (on ? i : n - 1) >> 2;
  const int q = (int)(i & 3), E = a.channels;
  const int64_t b = be / E;
  const int e = (int)(be % E);
  float4* st = reinterpret_cast<float4*>(a.state_out + be * kN + kQ * q);
  const float4 h4 = *st;
  const float4 A4 = *reinterpret_cast<const float4*>(a.A + (int64_t)e * kN + kQ * q);
  const T* B = (const T*)a.B + b * a.B_bs + kQ * q;
  const T* C = (const T*)a.C + b * a.C_bs + kQ * q;
  const float x = to_f(((const T*)a.x)[b * a.x_bs + e]);
  const float raw = to_f(((const T*)a.dt)[b * a.dt_bs + e]) + (a.dt_bias ? a.dt_bias[e] : 0.0f);
  const float d = a.softplus ? softplus_of(raw) : raw, du = d * x;
  float h[4] = {h4.x, h4.y, h4.z, h4.w};
  const float Av[4] = {A4.x, A4.y, A4.z, A4.w};
  float v = 0.0f;
#pragma unroll
  for (int j = 0; j < kQ; ++j) {
    h[j] = fmaf(ex2(d * (Av[j] * kLog2e)), h[j], du * to_f(B[j]));
    v = fmaf(to_f(C[j]), h[j], v);
  }
  if (on) *st = make_float4(h[0], h[1], h[2], h[3]);
  v += __shfl_xor_sync(0xffffffffu, v, 2);
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  if (on && q == 0) {
    if (a.D) v = fmaf(a.D[e], x, v);
    if (a.z) {
      const float z = to_f(((const T*)a.z)[b * a.z_bs + e]);
      v *= z * sigmoid_of(z);
    }
    ((T*)a.y)[be] = from_f<T>(v);
  }
}

// --------------------------------------------------------------------- host
static int round_up(int v, int m) { return (v + m - 1) / m * m; }

// Parts of the length: one where the rows alone give enough blocks, else enough
// for `want` blocks, no part shorter than 64 tokens.
static SsmPlan ssm_plan(const boa_ssm_args& a, int64_t row_blocks, int64_t enough, int64_t want) {
  SsmPlan p{};
  p.cblocks = (a.channels + kCh - 1) / kCh;
  int parts = 1;
  const int64_t blocks = (int64_t)a.batch * row_blocks;
  if (blocks < enough) {
    const int64_t most = (a.length + 63) / 64;
    const int64_t need = (want + blocks - 1) / blocks;
    parts = (int)(need < most ? need : most);
    if (parts < 1) parts = 1;
  }
  p.part = round_up((a.length + parts - 1) / parts, kTile);
  if (p.part < kTile) p.part = kTile;
  p.parts = a.length > 0 ? (a.length + p.part - 1) / p.part : 1;
  return p;
}

static int back_passes(const boa_ssm_args& a) {
  const int n = (a.channels + kCh - 1) / kCh;
  return n < kPasses ? n : kPasses;
}
static int back_groups(const boa_ssm_args& a) {
  const int per = back_passes(a) * kCh;
  return (a.channels + per - 1) / per;
}
static SsmPlan plan_forward(const boa_ssm_args& a) { return ssm_plan(a, (a.channels + kCh - 1) / kCh, 888, 1776); }
static SsmPlan plan_backward(const boa_ssm_args& a) { return ssm_plan(a, back_groups(a), 444, 1776); }

static bool even(int64_t v) { return v % 2 == 0; }

static bool ssm_pair(const boa_ssm_args& a, bool backward) {
  const size_t s = a.dtype == BOA_DTYPE_F32 ? 8 : 4;
  bool ok = even(a.channels) && even(a.x_bs) && even(a.x_ts) && even(a.dt_bs) && even(a.dt_ts) && aligned(a.x, s) &&
            aligned(a.dt, s);
  if (a.z) ok = ok && even(a.z_bs) && even(a.z_ts) && aligned(a.z, s);
  if (!backward) return ok && aligned(a.y, s);
  return ok && even(a.dy_bs) && even(a.dy_ts) && aligned(a.dy, s) && aligned(a.dx, s) && aligned(a.ddt, s) &&
         aligned(a.dz, s);
}

static size_t ends_floats(const boa_ssm_args& a, const SsmPlan& p) {
  return p.parts > 1 ? (size_t)a.batch * p.parts * a.channels * (kN + 1) : 0;
}

template <typename T>
static int ssm_forward(const boa_ssm_args& a, cudaStream_t s) {
  SsmPlan p = plan_forward(a);
  p.pair = ssm_pair(a, false);
  float* ends = (float*)a.workspace;
  float* dsum = ends + (size_t)a.batch * p.parts * a.channels * kN;
  if (p.parts > 1) {
    k_ssm<T, true><<<(unsigned)((int64_t)p.cblocks * (p.parts - 1) * a.batch), kSsmThreads, 0, s>>>(a, p, ends, dsum);
    const int64_t n = (int64_t)a.batch * a.channels * kN;
    k_ssm_join<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(n, a.channels, p.parts, a.A, a.state, ends, dsum, false);
  }
  k_ssm<T, false><<<(unsigned)((int64_t)p.cblocks * p.parts * a.batch), kSsmThreads, 0, s>>>(a, p, ends, dsum);
  BOA_CUDA(cudaGetLastError());
  return BOA_OK;
}

template <typename T>
static int ssm_backward(const boa_ssm_args& a, cudaStream_t s) {
  SsmPlan p = plan_backward(a);
  p.pair = ssm_pair(a, true);
  const int passes = back_passes(a), groups = back_groups(a);
  float* bc = (float*)a.workspace;
  float* params = bc + (size_t)groups * a.batch * a.length * 2 * kN;
  float* ends = params + (size_t)a.batch * p.parts * a.channels * (kN + 2);
  // the three sections keep 16-byte alignment: ends holds float4
  ends = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(ends) + 15) & ~uintptr_t(15));
  float* dsum = ends + (size_t)a.batch * p.parts * a.channels * kN;
  if (p.parts > 1) {
    k_ssm_back_ends<T>
        <<<(unsigned)((int64_t)p.cblocks * (p.parts - 1) * a.batch), kSsmThreads, 0, s>>>(a, p, ends, dsum);
    const int64_t n = (int64_t)a.batch * a.channels * kN;
    k_ssm_join<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(n, a.channels, p.parts, a.A, a.dstate_out, ends, dsum, true);
  }
  const int smem = BackSmem::floats(passes) * (int)sizeof(float);
  BOA_CUDA(cudaFuncSetAttribute(k_ssm_backward<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  k_ssm_backward<T><<<(unsigned)((int64_t)groups * p.parts * a.batch), kSsmThreads, smem, s>>>(a, p, passes, groups,
                                                                                             ends, bc, params);
  const int64_t rows = (int64_t)a.batch * a.length, n = rows * 2 * kN;
  if (n > 0)
    k_ssm_bc<T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(rows, groups, bc, (T*)a.dB, (T*)a.dC);
  const int cols = a.channels * (kN + 2);
  k_sum_parts<<<(cols + 31) / 32, 512, 0, s>>>(params, (int64_t)a.batch * p.parts, cols, a.channels * kN,
                                              a.channels * (kN + 1), a.dA, a.dD, a.ddt_bias);
  BOA_CUDA(cudaGetLastError());
  return BOA_OK;
}

static int ssm_check(const boa_ssm_args* a, const char* who) {
  if (!a) return boa_fail(BOA_ERR_ARG, std::string(who) + ": null arguments");
  if (a->batch < 0 || a->length < 0 || a->channels < 1)
    return boa_fail(BOA_ERR_ARG, std::string(who) + ": need batch >= 0, length >= 0 and channels >= 1");
  if (a->states != kN) return boa_fail(BOA_ERR_UNSUPPORTED, std::string(who) + ": states must be 16");
  if (a->dtype < BOA_DTYPE_F32 || a->dtype > BOA_DTYPE_F16)
    return boa_fail(BOA_ERR_ARG, std::string(who) + ": unknown dtype");
  return BOA_OK;
}

}  // namespace seq
}  // namespace boa

using namespace boa::seq;

extern "C" {

BOA_API size_t boa_ssm_checkpoint_bytes(const boa_ssm_args* a) {
  if (ssm_check(a, "boa_ssm_checkpoint_bytes")) return 0;
  return (size_t)a->batch * ((a->length + kBack - 1) / kBack) * a->channels * kN * sizeof(float);
}

BOA_API size_t boa_ssm_workspace_bytes(const boa_ssm_args* a, int backward) {
  if (ssm_check(a, "boa_ssm_workspace_bytes") || a->batch == 0) return 0;
  if (!backward) return ends_floats(*a, plan_forward(*a)) * sizeof(float);
  const SsmPlan p = plan_backward(*a);
  return (ends_floats(*a, p) + (size_t)back_groups(*a) * a->batch * a->length * 2 * kN +
          (size_t)a->batch * p.parts * a->channels * (kN + 2)) * sizeof(float) + 16;
}

BOA_API int boa_ssm_scan(const boa_ssm_args* a, void* stream) {
  const int rc = ssm_check(a, "boa_ssm_scan");
  if (rc) return rc;
  if (a->batch == 0 || (a->length == 0 && !a->state_out)) return BOA_OK;
  if (!a->A || (a->length > 0 && (!a->x || !a->dt || !a->B || !a->C || !a->y)))
    return boa_fail(BOA_ERR_ARG, "boa_ssm_scan: null argument");
  const size_t need = boa_ssm_workspace_bytes(a, 0);
  if (need && (!a->workspace || a->workspace_bytes < need))
    return boa_fail(BOA_ERR_ARG, "boa_ssm_scan: workspace too small (see boa_ssm_workspace_bytes)");
  if (!aligned(a->workspace, 16) || !aligned(a->checkpoints, 16))
    return boa_fail(BOA_ERR_ARG, "boa_ssm_scan: workspace and checkpoints must be 16-byte aligned");
  BOA_CUDA(cudaSetDevice(a->device));
  cudaStream_t s = (cudaStream_t)stream;
  if (a->dtype == BOA_DTYPE_F32) return ssm_forward<float>(*a, s);
  if (a->dtype == BOA_DTYPE_BF16) return ssm_forward<__nv_bfloat16>(*a, s);
  return ssm_forward<__half>(*a, s);
}

BOA_API int boa_ssm_scan_backward(const boa_ssm_args* a, void* stream) {
  const int rc = ssm_check(a, "boa_ssm_scan_backward");
  if (rc) return rc;
  if (!a->A || !a->dA) return boa_fail(BOA_ERR_ARG, "boa_ssm_scan_backward: null argument");
  cudaStream_t s = (cudaStream_t)stream;
  if (a->batch == 0) {
    BOA_CUDA(cudaSetDevice(a->device));
    BOA_CUDA(cudaMemsetAsync(a->dA, 0, (size_t)a->channels * kN * sizeof(float), s));
    if (a->dD) BOA_CUDA(cudaMemsetAsync(a->dD, 0, (size_t)a->channels * sizeof(float), s));
    if (a->ddt_bias) BOA_CUDA(cudaMemsetAsync(a->ddt_bias, 0, (size_t)a->channels * sizeof(float), s));
    return BOA_OK;
  }
  if (a->length > 0 && (!a->x || !a->dt || !a->B || !a->C || !a->dy || !a->dx || !a->ddt || !a->dB || !a->dC ||
                        !a->checkpoints || (a->z && !a->dz)))
    return boa_fail(BOA_ERR_ARG, "boa_ssm_scan_backward: null argument");
  if (!a->workspace || a->workspace_bytes < boa_ssm_workspace_bytes(a, 1))
    return boa_fail(BOA_ERR_ARG, "boa_ssm_scan_backward: workspace too small (see boa_ssm_workspace_bytes)");
  if (!aligned(a->workspace, 16) || !aligned(a->checkpoints, 16))
    return boa_fail(BOA_ERR_ARG, "boa_ssm_scan_backward: workspace and checkpoints must be 16-byte aligned");
  BOA_CUDA(cudaSetDevice(a->device));
  if (a->dtype == BOA_DTYPE_F32) return ssm_backward<float>(*a, s);
  if (a->dtype == BOA_DTYPE_BF16) return ssm_backward<__nv_bfloat16>(*a, s);
  return ssm_backward<__half>(*a, s);
}

BOA_API int boa_ssm_step(const boa_ssm_args* a, void* stream) {
  const int rc = ssm_check(a, "boa_ssm_step");
  if (rc) return rc;
  if (a->batch == 0) return BOA_OK;
  if (!a->A || !a->x || !a->dt || !a->B || !a->C || !a->y || !a->state_out)
    return boa_fail(BOA_ERR_ARG, "boa_ssm_step: null argument");
  if (!aligned(a->state_out, 16) || !aligned(a->A, 16))
    return boa_fail(BOA_ERR_ARG, "boa_ssm_step: state and A must be 16-byte aligned");
  BOA_CUDA(cudaSetDevice(a->device));
  cudaStream_t s = (cudaStream_t)stream;
  const unsigned grid = (unsigned)(((int64_t)a->batch * a->channels * 4 + 255) / 256);
  if (a->dtype == BOA_DTYPE_F32) k_ssm_step<float><<<grid, 256, 0, s>>>(*a);
  else if (a->dtype == BOA_DTYPE_BF16) k_ssm_step<__nv_bfloat16><<<grid, 256, 0, s>>>(*a);
  else k_ssm_step<__half><<<grid, 256, 0, s>>>(*a);
  BOA_CUDA(cudaGetLastError());
  return BOA_OK;
}

}  // extern "C"
