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
#include <cstring>

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

__device__ __forceinline__ int row_len(const boa_ssm_args& a, int b) {
  return a.lens ? min(max(a.lens[b], 0), a.length) : a.length;
}

// V neighbouring elements of a token row as loaded, zeros where the token or the
// channel does not exist.  VEC (every row starts on whole vectors): one access,
// kept as the words it arrives in, so that nothing waits for a load before the
// values are used a tile later.
template <typename T, int V, bool VEC>
struct Row {
  static constexpr int kWords = VEC ? V * (int)sizeof(T) / 4 : V;
  uint32_t w[kWords];
  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[j]);
    } else {
      const unsigned short h = VEC ? (unsigned short)(w[j / 2] >> (16 * (j & 1))) : (unsigned short)w[j];
      T t;
      memcpy(&t, &h, 2);
      return to_f(t);
    }
  }
  __device__ __forceinline__ void load(const T* p, int c, int E, bool live) {
#pragma unroll
    for (int j = 0; j < kWords; ++j) w[j] = 0;
    if constexpr (VEC) {
      if (live && c < E) {
        if constexpr (kWords == 1) w[0] = *reinterpret_cast<const uint32_t*>(p);
        if constexpr (kWords == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(p);
          w[0] = v.x;
          w[1] = v.y;
        }
        if constexpr (kWords == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(p);
          w[0] = v.x;
          w[1] = v.y;
          w[2] = v.z;
          w[3] = v.w;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (live && c + j < E) {
          if constexpr (sizeof(T) == 4) w[j] = reinterpret_cast<const uint32_t*>(p)[j];
          else w[j] = reinterpret_cast<const unsigned short*>(p)[j];
        }
    }
  }
};
template <typename T, int V, bool VEC>
__device__ __forceinline__ void store_row(T* p, int c, int E, const float (&v)[V]) {
  if constexpr (VEC) {
    if (c < E) store_f<T, V>(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (c + j < E) p[j] = from_f<T>(v[j]);
  }
}
// Parameters of V channels, zeros beyond the last or without the array.
template <int V>
__device__ __forceinline__ void load_params(const float* p, int c, int E, float (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = p && c + j < E ? p[c + j] : 0.0f;
}
__device__ __forceinline__ float step_of(float raw, bool softplus) {
  float u;
  return softplus ? softplus_f(raw, u) : raw;
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
};

// ------------------------------------------------------------------ forward
// ENDS: only the part's end state (from zero) and sum of d, into ends / dsum.
template <typename T, bool ENDS, bool VEC>
__global__ void __launch_bounds__(kSsmThreads) k_ssm(const boa_ssm_args a, const SsmPlan p, float* __restrict__ ends,
                                                     float* __restrict__ dsum) {
  __shared__ __align__(16) float sd[kTile][kPitch], su[kTile][kPitch], sy[kTile][kPitch];
  __shared__ __align__(16) float sbc[kTile][2 * kN];
  const int tid = threadIdx.x, lane = tid & 31, q = lane & 3, ch = (tid >> 5) * 8 + (lane >> 2);
  const int nparts = ENDS ? p.parts - 1 : p.parts;
  const int e0 = (blockIdx.x % p.cblocks) * kCh, E = a.channels;
  const int part = (blockIdx.x / p.cblocks) % nparts, b = blockIdx.x / p.cblocks / nparts;
  const int e = e0 + ch;
  const bool on = e < E, gated = !ENDS && a.z;
  const int len = row_len(a, b);
  const int begin = part * p.part, stop = min(begin + p.part, a.length), end = min(stop, len);
  const int64_t slot = ((int64_t)b * p.parts + part) * E + e;
  // staging: a thread moves four channels of token `row`, and four values of its B or C
  const int row = tid >> 3, sub = tid & 7, c = e0 + 4 * sub;
  const bool is_c = sub >= 4;
  int t = begin + row;
  const T* px = (const T*)a.x + b * a.x_bs + t * a.x_ts + c;
  const T* pd = (const T*)a.dt + b * a.dt_bs + t * a.dt_ts + c;
  const T* pz = (const T*)a.z + b * a.z_bs + t * a.z_ts + c;
  const T* pbc = is_c ? (const T*)a.C + b * a.C_bs + t * a.C_ts + 4 * (sub - 4)
                      : (const T*)a.B + b * a.B_bs + t * a.B_ts + 4 * sub;
  const int64_t bcts = is_c ? a.C_ts : a.B_ts;
  T* py = (T*)a.y + ((int64_t)b * a.length + t) * E + c;
  float bias[4], Dv[4];
  load_params<4>(a.dt_bias, c, E, bias);
  load_params<4>(a.D, c, E, Dv);
  f2 A2[2], h[2];
  {
    float v[kQ], s[kQ];
    const float* s0 = ENDS ? nullptr : p.parts > 1 ? ends + slot * kN : a.state ? a.state + ((int64_t)b * E + e) * kN : nullptr;
#pragma unroll
    for (int j = 0; j < kQ; ++j) {
      v[j] = on ? a.A[(int64_t)e * kN + kQ * q + j] * kLog2e : 0.0f;
      s[j] = on && s0 ? s0[kQ * q + j] : 0.0f;
    }
    A2[0] = pack(v[0], v[1]);
    A2[1] = pack(v[2], v[3]);
    h[0] = pack(s[0], s[1]);
    h[1] = pack(s[2], s[3]);
  }
  const int nck = (a.length + kBack - 1) / kBack;
  float* ck = !ENDS && a.checkpoints && on
                  ? a.checkpoints + (((int64_t)b * nck + begin / kBack) * E + e) * kN + kQ * q : nullptr;
  float total = 0.0f;
  Row<T, 4, VEC> rx, rd, rz, rb;
  auto fetch = [&]() {
    const bool live = t < end;
    rx.load(px, c, E, live);
    rd.load(pd, c, E, live);
    if (gated) rz.load(pz, c, E, live);
    rb.load(pbc, 0, 4, live && !(ENDS && is_c));
    px += kTile * a.x_ts;
    pd += kTile * a.dt_ts;
    pz += kTile * a.z_ts;
    pbc += kTile * bcts;
  };
  if (begin < end) fetch();
  for (int t0 = begin; t0 < end; t0 += kTile) {
    float xs[4], zs[4], d[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      xs[j] = rx.get(j);
      zs[j] = gated ? rz.get(j) : 0.0f;
      d[j] = t < end ? step_of(rd.get(j) + bias[j], a.softplus) : 0.0f;
    }
    *reinterpret_cast<float4*>(&sd[row][4 * sub]) = make_float4(d[0], d[1], d[2], d[3]);
    *reinterpret_cast<float4*>(&su[row][4 * sub]) = make_float4(d[0] * xs[0], d[1] * xs[1], d[2] * xs[2], d[3] * xs[3]);
    *reinterpret_cast<float4*>(&sbc[row][4 * sub]) = make_float4(rb.get(0), rb.get(1), rb.get(2), rb.get(3));
    const bool mine = t < stop, live = t < end;
    t += kTile;
    __syncthreads();
    if (t0 + kTile < end) fetch();
#pragma unroll
    for (int u = 0; u < kTile; u += 4) {
      float yp[4];
      if (!ENDS && u % kBack == 0 && ck && t0 + u < end) {
        *reinterpret_cast<ulonglong2*>(ck) = make_ulonglong2(h[0].v, h[1].v);
        ck += (int64_t)E * kN;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float dk = sd[u + k][ch], uk = su[u + k][ch];
        const f2 dd = pack(dk, dk), uu = pack(uk, uk);
        const ulonglong2 B = *reinterpret_cast<const ulonglong2*>(&sbc[u + k][kQ * q]);
        h[0] = fma2(ex2_2(mul2(dd, A2[0])), h[0], mul2(uu, f2{B.x}));
        h[1] = fma2(ex2_2(mul2(dd, A2[1])), h[1], mul2(uu, f2{B.y}));
        if constexpr (ENDS) {
          total += dk;
        } else {
          const ulonglong2 C = *reinterpret_cast<const ulonglong2*>(&sbc[u + k][kN + kQ * q]);
          const float2 y = unpack(fma2(f2{C.x}, h[0], mul2(f2{C.y}, h[1])));
          yp[k] = y.x + y.y;
        }
      }
      if constexpr (!ENDS) sy[u + q][ch] = quad_sum(yp, q);
    }
    __syncthreads();
    if constexpr (!ENDS) {
      if (mine) {
        float o[4];
        const float4 v = *reinterpret_cast<const float4*>(&sy[row][4 * sub]);
        const float vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o[j] = fmaf(Dv[j], xs[j], vv[j]);
          if (gated) o[j] *= zs[j] * sigmoid_f(zs[j]);
          if (!live) o[j] = 0.0f;
        }
        store_row<T, 4, VEC>(py, c, E, o);
      }
      py += (int64_t)kTile * E;
    }
  }
  if constexpr (ENDS) {
    if (on) {
      *reinterpret_cast<ulonglong2*>(ends + slot * kN + kQ * q) = make_ulonglong2(h[0].v, h[1].v);
      if (q == 0) dsum[slot] = total;
    }
  } else {
    const float zero[4] = {};
    for (; t < stop; t += kTile) {   // tiles wholly behind the row's end
      store_row<T, 4, VEC>(py, c, E, zero);
      py += (int64_t)kTile * E;
    }
    if (a.state_out && part == p.parts - 1 && on) {
      float* so = a.state_out + ((int64_t)b * E + e) * kN + kQ * q;
      const float2 lo = unpack(h[0]), hi = unpack(h[1]);
      so[0] = lo.x;
      so[1] = lo.y;
      so[2] = hi.x;
      so[3] = hi.y;
    }
  }
}

// Chains the parts of every (row, channel, state): ends[] becomes the value
// each part starts from.  Forward: from the first part with h; backward
// (`reverse`): from the last part with the gradient of the state.
static __global__ void __launch_bounds__(128) k_ssm_join(int64_t n, int E, int parts, const float* __restrict__ A,
                                                         const float* __restrict__ first, float* ends,
                                                         const float* __restrict__ dsum, bool reverse) {
  const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
  if (i >= n) return;
  const int64_t en = (int64_t)E * kN;
  const int64_t b = i / en, r = i % en;
  const float A2 = A[r] * kLog2e;
  float carry = first ? first[i] : 0.0f;
  const int64_t step = reverse ? -1 : 1;
  int64_t s = b * parts + (reverse ? parts - 1 : 0);
  constexpr int kAhead = 16;   // parts whose loads are in flight together
  for (int k0 = 0; k0 < parts; k0 += kAhead) {
    float own[kAhead], sum[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const bool have = k0 + j < parts - 1;
      own[j] = have ? ends[(s + j * step) * en + r] : 0.0f;
      sum[j] = have ? dsum[(s + j * step) * E + r / kN] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (k0 + j < parts) {
        ends[(s + j * step) * en + r] = carry;
        carry = fmaf(ex2(A2 * sum[j]), carry, own[j]);
      }
    s += kAhead * step;
  }
}

// ----------------------------------------------------------------- backward
// The gradient of the state that a part passes on to the part before it, from
// a zero start at its end, and the part's sum of d.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kSsmThreads) k_ssm_back_ends(const boa_ssm_args a, const SsmPlan p,
                                                               float* __restrict__ ends, float* __restrict__ dsum) {
  __shared__ __align__(16) float sd[kTile][kPitch], sg[kTile][kPitch];
  __shared__ __align__(16) float sc[kTile][kN];
  const int tid = threadIdx.x, lane = tid & 31, q = lane & 3, ch = (tid >> 5) * 8 + (lane >> 2);
  const int e0 = (blockIdx.x % p.cblocks) * kCh, E = a.channels;
  const int part = 1 + (blockIdx.x / p.cblocks) % (p.parts - 1), b = blockIdx.x / p.cblocks / (p.parts - 1);
  const int e = e0 + ch;
  const bool on = e < E, gated = a.z;
  const int begin = part * p.part, end = min(min(begin + p.part, a.length), row_len(a, b));
  const int64_t slot = ((int64_t)b * p.parts + part) * E + e;
  const int row = tid >> 3, sub = tid & 7, c = e0 + 4 * sub;
  const int tiles = (max(end - begin, 0) + kTile - 1) / kTile;
  int t = begin + (tiles - 1) * kTile + row;
  const T* pg = (const T*)a.dy + b * a.dy_bs + t * a.dy_ts + c;
  const T* pd = (const T*)a.dt + b * a.dt_bs + t * a.dt_ts + c;
  const T* pz = (const T*)a.z + b * a.z_bs + t * a.z_ts + c;
  const T* pc = (const T*)a.C + b * a.C_bs + t * a.C_ts + 4 * sub;   // lanes with sub < 4
  float bias[4];
  load_params<4>(a.dt_bias, c, E, bias);
  f2 A2[2], g2[2] = {pack(0.f, 0.f), pack(0.f, 0.f)};
  {
    float v[kQ];
#pragma unroll
    for (int j = 0; j < kQ; ++j) v[j] = on ? a.A[(int64_t)e * kN + kQ * q + j] * kLog2e : 0.0f;
    A2[0] = pack(v[0], v[1]);
    A2[1] = pack(v[2], v[3]);
  }
  float total = 0.0f;
  Row<T, 4, VEC> rg, rd, rz, rc;
  auto fetch = [&]() {
    const bool live = t < end;
    rg.load(pg, c, E, live);
    rd.load(pd, c, E, live);
    if (gated) rz.load(pz, c, E, live);
    rc.load(pc, 0, 4, live && sub < 4);
    pg -= kTile * a.dy_ts;
    pd -= kTile * a.dt_ts;
    pz -= kTile * a.z_ts;
    pc -= kTile * a.C_ts;
  };
  if (tiles) fetch();
  for (int k = tiles - 1; k >= 0; --k) {
    float d[4], g[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      g[j] = rg.get(j);
      if (gated) {
        const float z = rz.get(j);
        g[j] *= z * sigmoid_f(z);
      }
      d[j] = t < end ? step_of(rd.get(j) + bias[j], a.softplus) : 0.0f;
    }
    *reinterpret_cast<float4*>(&sd[row][4 * sub]) = make_float4(d[0], d[1], d[2], d[3]);
    *reinterpret_cast<float4*>(&sg[row][4 * sub]) = make_float4(g[0], g[1], g[2], g[3]);
    if (sub < 4)
      *reinterpret_cast<float4*>(&sc[row][4 * sub]) = make_float4(rc.get(0), rc.get(1), rc.get(2), rc.get(3));
    t -= kTile;
    __syncthreads();
    if (k > 0) fetch();
#pragma unroll
    for (int i = kTile - 1; i >= 0; --i) {
      const float dk = sd[i][ch], gk = sg[i][ch];
      const f2 dd = pack(dk, dk), gg = pack(gk, gk);
      const ulonglong2 C = *reinterpret_cast<const ulonglong2*>(&sc[i][kQ * q]);
      g2[0] = mul2(ex2_2(mul2(dd, A2[0])), fma2(f2{C.x}, gg, g2[0]));
      g2[1] = mul2(ex2_2(mul2(dd, A2[1])), fma2(f2{C.y}, gg, g2[1]));
      total += dk;
    }
    __syncthreads();
  }
  if (on) {
    *reinterpret_cast<ulonglong2*>(ends + slot * kN + kQ * q) = make_ulonglong2(g2[0].v, g2[1].v);
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

template <typename T, bool VEC>
struct RawBack {
  Row<T, 2, VEC> x, dt, z, g;
  float4 h;
};

// A block takes one part of a row and up to 256 channels, tile by tile from
// the end, 32 channels a pass.  A pass recomputes h over the tile from its
// checkpoint (a and h stay in registers), then runs the gradient backwards.
// dB and dC of the tile gather over the passes in registers and are summed
// over the block's lanes and warps once a tile.
template <typename T, bool VEC>
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
  RawBack<T, VEC> r;
  auto fetch = [&](int t0, int g) {
    const int t = t0 + row, c = e0 + g * kCh + cl;
    const bool live = t < end;
    r.x.load(px + (int64_t)t * a.x_ts + c, c, E, live);
    r.dt.load(pd + (int64_t)t * a.dt_ts + c, c, E, live);
    r.g.load(pg + (int64_t)t * a.dy_ts + c, c, E, live);
    if (pz) r.z.load(pz + (int64_t)t * a.z_ts + c, c, E, live);
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
        float u = 0.0f;
        const float raw = r.dt.get(j) + (a.dt_bias && c + j < E ? a.dt_bias[c + j] : 0.0f);
        Dv[j] = a.D && c + j < E ? a.D[c + j] : 0.0f;
        dv[j] = live ? (a.softplus ? softplus_f(raw, u) : raw) : 0.0f;
        sig[j] = a.softplus ? (raw >= 0.0f ? 1.0f : u) * rcp(1.0f + u) : 1.0f;
        xv[j] = r.x.get(j);
        gv[j] = r.g.get(j);
        dzf[j] = 0.0f;
        if (pz) {
          const float z = r.z.get(j), s = sigmoid_f(z);
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
        store_row<T, 2, VEC>((T*)a.dx + o + c, c, E, ox);
        store_row<T, 2, VEC>((T*)a.ddt + o + c, c, E, od);
        if (pz) store_row<T, 2, VEC>((T*)a.dz + o + c, c, E, oz);
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
  const float zero2[2] = {};
  for (int t = begin + tiles * kBack + row; t < stop; t += kBack) {
    const int64_t o = (orow + t) * E;
    for (int g = 0; g < np; ++g) {
      const int c = e0 + g * kCh + cl;
      store_row<T, 2, VEC>((T*)a.dx + o + c, c, E, zero2);
      store_row<T, 2, VEC>((T*)a.ddt + o + c, c, E, zero2);
      if (pz) store_row<T, 2, VEC>((T*)a.dz + o + c, c, E, zero2);
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
  const float d = step_of(raw, a.softplus), du = d * x;
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
      v *= z * sigmoid_f(z);
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

// Vector accesses where every row of every tensor starts on four elements.
static bool row_vec(const void* p, int64_t bs, int64_t ts, size_t size) {
  return bs % 4 == 0 && ts % 4 == 0 && aligned(p, 4 * size);
}
static bool ssm_vec(const boa_ssm_args& a, bool backward) {
  const size_t s = a.dtype == BOA_DTYPE_F32 ? 4 : 2;
  const bool ok = a.channels % 4 == 0 && row_vec(a.x, a.x_bs, a.x_ts, s) && row_vec(a.dt, a.dt_bs, a.dt_ts, s) &&
                  row_vec(a.B, a.B_bs, a.B_ts, s) && row_vec(a.C, a.C_bs, a.C_ts, s) &&
                  (!a.z || row_vec(a.z, a.z_bs, a.z_ts, s));
  if (!backward) return ok && aligned(a.y, 4 * s);
  return ok && row_vec(a.dy, a.dy_bs, a.dy_ts, s) && aligned(a.dx, 4 * s) && aligned(a.ddt, 4 * s) &&
         aligned(a.dz, 4 * s);
}

static size_t ends_floats(const boa_ssm_args& a, const SsmPlan& p) {
  return p.parts > 1 ? (size_t)a.batch * p.parts * a.channels * (kN + 1) : 0;
}

template <typename T, bool VEC>
static int ssm_forward_t(const boa_ssm_args& a, cudaStream_t s) {
  const SsmPlan p = plan_forward(a);
  float* ends = (float*)a.workspace;
  float* dsum = ends + (size_t)a.batch * p.parts * a.channels * kN;
  if (p.parts > 1) {
    k_ssm<T, true, VEC><<<(unsigned)((int64_t)p.cblocks * (p.parts - 1) * a.batch), kSsmThreads, 0, s>>>(a, p, ends, dsum);
    const int64_t n = (int64_t)a.batch * a.channels * kN;
    k_ssm_join<<<(unsigned)((n + 127) / 128), 128, 0, s>>>(n, a.channels, p.parts, a.A, a.state, ends, dsum, false);
  }
  k_ssm<T, false, VEC><<<(unsigned)((int64_t)p.cblocks * p.parts * a.batch), kSsmThreads, 0, s>>>(a, p, ends, dsum);
  BOA_CUDA(cudaGetLastError());
  return BOA_OK;
}

template <typename T>
static int ssm_forward(const boa_ssm_args& a, cudaStream_t s) {
  return ssm_vec(a, false) ? ssm_forward_t<T, true>(a, s) : ssm_forward_t<T, false>(a, s);
}

template <typename T, bool VEC>
static int ssm_backward_t(const boa_ssm_args& a, cudaStream_t s) {
  const SsmPlan p = plan_backward(a);
  const int passes = back_passes(a), groups = back_groups(a);
  float* bc = (float*)a.workspace;
  float* params = bc + (size_t)groups * a.batch * a.length * 2 * kN;
  float* ends = params + (size_t)a.batch * p.parts * a.channels * (kN + 2);
  // the three sections keep 16-byte alignment: ends holds float4
  ends = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(ends) + 15) & ~uintptr_t(15));
  float* dsum = ends + (size_t)a.batch * p.parts * a.channels * kN;
  if (p.parts > 1) {
    k_ssm_back_ends<T, VEC>
        <<<(unsigned)((int64_t)p.cblocks * (p.parts - 1) * a.batch), kSsmThreads, 0, s>>>(a, p, ends, dsum);
    const int64_t n = (int64_t)a.batch * a.channels * kN;
    k_ssm_join<<<(unsigned)((n + 127) / 128), 128, 0, s>>>(n, a.channels, p.parts, a.A, a.dstate_out, ends, dsum, true);
  }
  const int smem = BackSmem::floats(passes) * (int)sizeof(float);
  BOA_CUDA(cudaFuncSetAttribute(k_ssm_backward<T, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  k_ssm_backward<T, VEC><<<(unsigned)((int64_t)groups * p.parts * a.batch), kSsmThreads, smem, s>>>(a, p, passes, groups,
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

template <typename T>
static int ssm_backward(const boa_ssm_args& a, cudaStream_t s) {
  return ssm_vec(a, true) ? ssm_backward_t<T, true>(a, s) : ssm_backward_t<T, false>(a, s);
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
