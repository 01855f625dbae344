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
//
// Bound by the exponentials (16 a channel and token; 16 a clock and SM, 4.65 T/s)
// and by issue, not by memory (8 bytes in bf16 take a third of the
// exponentials' time).  At 16 x 2048 x 512 bf16 on a B200, where they take 58 us:
// forward in one part 155 us, the end pass of the backward call 87 us, the
// backward kernel 397 us.
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
constexpr int kPasses = 8;        // channel passes of a backward block (of 64 channels)

__device__ __forceinline__ int row_len(const boa_ssm_args& a, int b) {
  return a.lens ? min(max(a.lens[b], 0), a.length) : a.length;
}

// V neighbouring elements of a token row as loaded, zeros where the token or the
// channel does not exist.  VEC (every row starts on whole vectors): one access,
// kept as the words it arrives in, so that nothing waits for a load before the
// values are used a tile later.
template <typename T, int V, bool VEC>
struct Row {
  static constexpr int kVecs = VEC ? 1 : V;
  Words<T, VEC ? V : 1> v[kVecs];
  __device__ __forceinline__ float get(int j) const { return VEC ? v[0].get(j) : v[VEC ? 0 : j].get(0); }
  __device__ __forceinline__ void load(const T* p, int c, int E, bool live) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      v[j].clear();
      if (live && c + j < E) v[j].load(p + j);
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
template <typename T, bool VEC>
__device__ __forceinline__ void store_row2(T* p, int c, int E, const f2 (&v)[2]) {
  const float2 a = unpack(v[0]), b = unpack(v[1]);
  const float x[4] = {a.x, a.y, b.x, b.y};
  store_row<T, 4, VEC>(p, c, E, x);
}
__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ void st4(void* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
// Four values of shared memory as two pairs.
__device__ __forceinline__ void ld2(const float* p, f2 (&v)[2]) {
  const ulonglong2 r = *reinterpret_cast<const ulonglong2*>(p);
  v[0] = f2{r.x};
  v[1] = f2{r.y};
}
__device__ __forceinline__ void st2(float* p, const f2 (&v)[2]) {
  *reinterpret_cast<ulonglong2*>(p) = make_ulonglong2(v[0].v, v[1].v);
}
// Parameters of V channels, zeros beyond the last or without the array.
template <int V>
__device__ __forceinline__ void load_params(const float* p, int c, int E, float (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = p && c + j < E ? p[c + j] : 0.0f;
}
__device__ __forceinline__ void load_pairs(const float* p, int c, int E, f2 (&v)[2]) {
  float t[4];
  load_params<4>(p, c, E, t);
  v[0] = pack(t[0], t[1]);
  v[1] = pack(t[2], t[3]);
}
// A in units of log2, for a decay ex2(d rate).  -inf (a channel that forgets at
// once) is held at the lowest number: d is 0 behind a row's end, where the decay
// is 1 and 0 times -inf would not be.
__device__ __forceinline__ float rate_of(float A) {
  const float r = A * kLog2e;
  return r < -3.402823466e38f ? -3.402823466e38f : r;
}
__device__ __forceinline__ float step_of(float raw, bool softplus) {
  float u;
  return softplus ? softplus_f(raw, u) : raw;
}

// A warp's 8 channels x 4 state groups: the state group is in lane bits 1 and 2,
// the channel in bits 0, 3 and 4.  A 16-byte shared load takes 2 wavefronts
// instead of 4 where lanes that differ in bit 0 alone, or in bit 1 alone, share
// an address (measured); so both the loads by state (B, C) and those by channel do.
__device__ __forceinline__ int lane_q(int lane) { return (lane >> 1) & 3; }
__device__ __forceinline__ int lane_ch(int lane) { return (lane & 1) | ((lane >> 3) << 1); }

// Sums of four values over the four lanes of a channel: lane q gets that of v[q].
__device__ __forceinline__ float quad_sum(const float (&v)[4], int q) {
  const bool hi = q & 2, odd = q & 1;
  float k0 = hi ? v[2] : v[0], k1 = hi ? v[3] : v[1];
  k0 += __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[2], 4);
  k1 += __shfl_xor_sync(0xffffffffu, hi ? v[1] : v[3], 4);
  return (odd ? k1 : k0) + __shfl_xor_sync(0xffffffffu, odd ? k0 : k1, 2);
}

struct SsmPlan {
  int cblocks;      // blocks (of 32 channels) of a row
  int parts, part;  // parts of a sequence, tokens of a part
};

// ------------------------------------------------------------------ forward
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void bar_arrive(int id, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
enum { kFull = 1, kDone = 3, kScanOnly = 5 };          // barrier ids; kFull and kDone one per slot

constexpr int kScanThreads = 2 * kSsmThreads;

// One pass over a part: warps 4-7 stage a tile (softplus once an element) and
// finish it (D x and the gate), warps 0-3 carry h through it.  The two work on
// neighbouring tiles, two slots of shared memory apart.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kScanThreads, 4) k_ssm(const boa_ssm_args a, const SsmPlan p,
                                                         const float* __restrict__ starts) {
  // d and d x of every token and channel, twice each, as the paired operations take them
  __shared__ __align__(16) f2 sd[2][kTile][kCh], su[2][kTile][kCh];
  __shared__ __align__(16) float sy[2][kTile][kPitch], sbc[2][kTile][2 * kN];
  const int tid = threadIdx.x & (kSsmThreads - 1);
  const int e0 = (blockIdx.x % p.cblocks) * kCh, E = a.channels;
  const int part = (blockIdx.x / p.cblocks) % p.parts, b = blockIdx.x / p.cblocks / p.parts;
  const int len = row_len(a, b);
  const int begin = part * p.part, stop = min(begin + p.part, a.length), end = min(stop, len);
  int slot = 0;
  if (threadIdx.x < kSsmThreads) {
    const int lane = tid & 31, q = lane_q(lane), ch = (tid >> 5) * 8 + lane_ch(lane), e = e0 + ch;
    const bool on = e < E;
    f2 A2[2], h[2];
    {
      float v[kQ], s[kQ];
      const float* s0 = p.parts > 1 ? starts + (((int64_t)b * p.parts + part) * E + e) * kN
                        : a.state   ? a.state + ((int64_t)b * E + e) * kN : nullptr;
#pragma unroll
      for (int j = 0; j < kQ; ++j) {
        v[j] = on ? rate_of(a.A[(int64_t)e * kN + kQ * q + j]) : 0.0f;
        s[j] = on && s0 ? s0[kQ * q + j] : 0.0f;
      }
      A2[0] = pack(v[0], v[1]);
      A2[1] = pack(v[2], v[3]);
      h[0] = pack(s[0], s[1]);
      h[1] = pack(s[2], s[3]);
    }
    const int nck = (a.length + kBack - 1) / kBack;
    float* ck = a.checkpoints && on
                    ? a.checkpoints + (((int64_t)b * nck + begin / kBack) * E + e) * kN + kQ * q : nullptr;
    for (int t0 = begin; t0 < end; t0 += kTile) {
      bar_sync(kFull + slot, kScanThreads);
#pragma unroll
      for (int u = 0; u < kTile; u += 4) {
        float yp[4];
        if (u % kBack == 0 && ck && t0 + u < end) {
          *reinterpret_cast<ulonglong2*>(ck) = make_ulonglong2(h[0].v, h[1].v);
          ck += (int64_t)E * kN;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const f2 dd = sd[slot][u + k][ch], uu = su[slot][u + k][ch];
          const ulonglong2 B = *reinterpret_cast<const ulonglong2*>(&sbc[slot][u + k][kQ * q]);
          const ulonglong2 C = *reinterpret_cast<const ulonglong2*>(&sbc[slot][u + k][kN + kQ * q]);
          h[0] = fma2(ex2_2(mul2(dd, A2[0])), h[0], mul2(uu, f2{B.x}));
          h[1] = fma2(ex2_2(mul2(dd, A2[1])), h[1], mul2(uu, f2{B.y}));
          const float2 y = unpack(fma2(f2{C.x}, h[0], mul2(f2{C.y}, h[1])));
          yp[k] = y.x + y.y;
        }
        sy[slot][u + q][ch] = quad_sum(yp, q);
      }
      bar_arrive(kDone + slot, kScanThreads);
      slot ^= 1;
    }
    if (a.state_out && part == p.parts - 1 && on) {
      float* so = a.state_out + ((int64_t)b * E + e) * kN + kQ * q;
      const float2 lo = unpack(h[0]), hi = unpack(h[1]);
      so[0] = lo.x;
      so[1] = lo.y;
      so[2] = hi.x;
      so[3] = hi.y;
    }
  } else {
    // a thread moves four channels of token `row` of a tile, and four values of its B or C
    const bool gated = a.z;
    const int row = tid >> 3, sub = tid & 7, c = e0 + 4 * sub;
    const bool is_c = sub >= 4;
    int t = begin + row;                       // of the tile to be loaded next
    const T* px = (const T*)a.x + b * a.x_bs + t * a.x_ts + c;
    const T* pd = (const T*)a.dt + b * a.dt_bs + t * a.dt_ts + c;
    const T* pz = (const T*)a.z + b * a.z_bs + t * a.z_ts + c;
    const T* pbc = is_c ? (const T*)a.C + b * a.C_bs + t * a.C_ts + 4 * (sub - 4)
                        : (const T*)a.B + b * a.B_bs + t * a.B_ts + 4 * sub;
    const int64_t bcts = is_c ? a.C_ts : a.B_ts;
    T* py = (T*)a.y + ((int64_t)b * a.length + t) * E + c;
    f2 bias[2], Dv[2], px2[2], pz2[2];         // x and z of the tile staged before
    load_pairs(a.dt_bias, c, E, bias);
    load_pairs(a.D, c, E, Dv);
    Row<T, 4, VEC> rx, rd, rz, rb;
    auto fetch = [&]() {
      const bool live = t < end;
      rx.load(px, c, E, live);
      rd.load(pd, c, E, live);
      if (gated) rz.load(pz, c, E, live);
      rb.load(pbc, 0, 4, live);
      px += kTile * a.x_ts;
      pd += kTile * a.dt_ts;
      pz += kTile * a.z_ts;
      pbc += kTile * bcts;
      t += kTile;
    };
    auto finish = [&](int slot, int t) {       // t: this thread's token of that tile
      bar_sync(kDone + slot, kScanThreads);
      if (t < stop) {
        float o[4];
        f2 v[2];
        ld2(&sy[slot][row][4 * sub], v);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          f2 y = fma2(Dv[j], px2[j], v[j]);
          if (gated) y = mul2(y, mul2(pz2[j], vsigmoid<2>(Fv<2>{{pz2[j]}}).p[0]));
          const float2 r = unpack(y);
          o[2 * j] = t < end ? r.x : 0.0f;
          o[2 * j + 1] = t < end ? r.y : 0.0f;
        }
        store_row<T, 4, VEC>(py, c, E, o);
      }
      py += (int64_t)kTile * E;
    };
    if (begin < end) fetch();
    int at = begin + row;                      // token of the tile being staged
    for (int t0 = begin; t0 < end; t0 += kTile) {
      f2 xs[2], zs[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        xs[j] = pack(rx.get(2 * j), rx.get(2 * j + 1));
        zs[j] = gated ? pack(rz.get(2 * j), rz.get(2 * j + 1)) : f2{0ull};
        f2 d = add2(pack(rd.get(2 * j), rd.get(2 * j + 1)), bias[j]), u;
        if (a.softplus) d = softplus2(d, u);
        if (at >= end) d = f2{0ull};
        const float2 dv = unpack(d), uv = unpack(mul2(d, xs[j]));
        st4(&sd[slot][row][4 * sub + 2 * j], make_float4(dv.x, dv.x, dv.y, dv.y));
        st4(&su[slot][row][4 * sub + 2 * j], make_float4(uv.x, uv.x, uv.y, uv.y));
      }
      st4(&sbc[slot][row][4 * sub], make_float4(rb.get(0), rb.get(1), rb.get(2), rb.get(3)));
      bar_arrive(kFull + slot, kScanThreads);
      if (t0 + kTile < end) fetch();
      if (t0 > begin) finish(slot ^ 1, at - kTile);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        px2[j] = xs[j];
        pz2[j] = zs[j];
      }
      at += kTile;
      slot ^= 1;
    }
    if (begin < end) finish(slot ^ 1, at - kTile);
    const float zero[4] = {};
    for (; at < stop; at += kTile) {           // tiles wholly behind the row's end
      store_row<T, 4, VEC>(py, c, E, zero);
      py += (int64_t)kTile * E;
    }
  }
}

// Only a part's end state (from zero) and sum of d.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kSsmThreads) k_ssm_ends(const boa_ssm_args a, const SsmPlan p,
                                                          float* __restrict__ ends, float* __restrict__ dsum) {
  __shared__ __align__(16) float sd[kTile][kPitch], su[kTile][kPitch], sb[kTile][kN];
  const int tid = threadIdx.x, lane = tid & 31, q = lane_q(lane), ch = (tid >> 5) * 8 + lane_ch(lane);
  const int e0 = (blockIdx.x % p.cblocks) * kCh, E = a.channels, nparts = p.parts - 1;
  const int part = (blockIdx.x / p.cblocks) % nparts, b = blockIdx.x / p.cblocks / nparts;
  const int e = e0 + ch;
  const bool on = e < E;
  const int begin = part * p.part, end = min(min(begin + p.part, a.length), row_len(a, b));
  const int64_t slot = ((int64_t)b * p.parts + part) * E + e;
  const int row = tid >> 3, sub = tid & 7, c = e0 + 4 * sub;
  int t = begin + row;
  const T* px = (const T*)a.x + b * a.x_bs + t * a.x_ts + c;
  const T* pd = (const T*)a.dt + b * a.dt_bs + t * a.dt_ts + c;
  const T* pb = (const T*)a.B + b * a.B_bs + t * a.B_ts + 4 * sub;   // threads with sub < 4
  f2 bias[2], A2[2], h[2] = {f2{0ull}, f2{0ull}};
  load_pairs(a.dt_bias, c, E, bias);
  {
    float v[kQ];
#pragma unroll
    for (int j = 0; j < kQ; ++j) v[j] = on ? rate_of(a.A[(int64_t)e * kN + kQ * q + j]) : 0.0f;
    A2[0] = pack(v[0], v[1]);
    A2[1] = pack(v[2], v[3]);
  }
  float total = 0.0f;
  Row<T, 4, VEC> rx, rd, rb;
  auto fetch = [&]() {
    const bool live = t < end;
    rx.load(px, c, E, live);
    rd.load(pd, c, E, live);
    rb.load(pb, 0, 4, live && sub < 4);
    px += kTile * a.x_ts;
    pd += kTile * a.dt_ts;
    pb += kTile * a.B_ts;
  };
  if (begin < end) fetch();
  for (int t0 = begin; t0 < end; t0 += kTile) {
    f2 d[2], u[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      d[j] = add2(pack(rd.get(2 * j), rd.get(2 * j + 1)), bias[j]);
      if (a.softplus) d[j] = softplus2(d[j], u[j]);
      if (t >= end) d[j] = f2{0ull};
      u[j] = mul2(d[j], pack(rx.get(2 * j), rx.get(2 * j + 1)));
    }
    st2(&sd[row][4 * sub], d);
    st2(&su[row][4 * sub], u);
    if (sub < 4) st4(&sb[row][4 * sub], make_float4(rb.get(0), rb.get(1), rb.get(2), rb.get(3)));
    t += kTile;
    __syncthreads();
    if (t0 + kTile < end) fetch();
    float tile = 0.0f;
#pragma unroll
    for (int i = 0; i < kTile; ++i) {
      const float dk = sd[i][ch], uk = su[i][ch];
      const f2 dd = pack(dk, dk), uu = pack(uk, uk);
      const ulonglong2 B = *reinterpret_cast<const ulonglong2*>(&sb[i][kQ * q]);
      h[0] = fma2(ex2_2(mul2(dd, A2[0])), h[0], mul2(uu, f2{B.x}));
      h[1] = fma2(ex2_2(mul2(dd, A2[1])), h[1], mul2(uu, f2{B.y}));
      tile += dk;
    }
    total += tile;   // by tiles: a part's sum then passes tens of roundings, not one a token
    __syncthreads();
  }
  if (on) {
    *reinterpret_cast<ulonglong2*>(ends + slot * kN + kQ * q) = make_ulonglong2(h[0].v, h[1].v);
    if (q == 0) dsum[slot] = total;
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
  const float A2 = rate_of(A[r]);
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
        // nothing comes in: nothing is passed on, also where a decay above 1 has overflowed over the part
        carry = carry == 0.0f ? own[j] : fmaf(ex2(A2 * sum[j]), carry, own[j]);
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
  const int tid = threadIdx.x, lane = tid & 31, q = lane_q(lane), ch = (tid >> 5) * 8 + lane_ch(lane);
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
  f2 bias[2];
  load_pairs(a.dt_bias, c, E, bias);
  f2 A2[2], g2[2] = {pack(0.f, 0.f), pack(0.f, 0.f)};
  {
    float v[kQ];
#pragma unroll
    for (int j = 0; j < kQ; ++j) v[j] = on ? rate_of(a.A[(int64_t)e * kN + kQ * q + j]) : 0.0f;
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
    f2 d[2], g[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f2 u;
      d[j] = add2(pack(rd.get(2 * j), rd.get(2 * j + 1)), bias[j]);
      g[j] = pack(rg.get(2 * j), rg.get(2 * j + 1));
      if (a.softplus) d[j] = softplus2(d[j], u);
      if (t >= end) d[j] = f2{0ull};
      if (gated) {
        const f2 z = pack(rz.get(2 * j), rz.get(2 * j + 1));
        g[j] = mul2(g[j], mul2(z, vsigmoid<2>(Fv<2>{{z}}).p[0]));
      }
    }
    st2(&sd[row][4 * sub], d);
    st2(&sg[row][4 * sub], g);
    if (sub < 4)
      *reinterpret_cast<float4*>(&sc[row][4 * sub]) = make_float4(rc.get(0), rc.get(1), rc.get(2), rc.get(3));
    t -= kTile;
    __syncthreads();
    if (k > 0) fetch();
    float tile = 0.0f;
#pragma unroll
    for (int i = kTile - 1; i >= 0; --i) {
      const float dk = sd[i][ch], gk = sg[i][ch];
      const f2 dd = pack(dk, dk), gg = pack(gk, gk);
      const ulonglong2 C = *reinterpret_cast<const ulonglong2*>(&sc[i][kQ * q]);
      g2[0] = mul2(ex2_2(mul2(dd, A2[0])), fma2(f2{C.x}, gg, g2[0]));
      g2[1] = mul2(ex2_2(mul2(dd, A2[1])), fma2(f2{C.y}, gg, g2[1]));
      tile += dk;
    }
    total += tile;   // by tiles: a part's sum then passes tens of roundings, not one a token
    __syncthreads();
  }
  if (on) {
    *reinterpret_cast<ulonglong2*>(ends + slot * kN + kQ * q) = make_ulonglong2(g2[0].v, g2[1].v);
    if (q == 0) dsum[slot] = total;
  }
}

constexpr int kBackCh = 64;                           // channels a backward pass
constexpr int kBackPitch = 72;                        // 8 mod 32, as kPitch
constexpr int kBackScan = 256, kBackThreads = kBackScan + 128;
constexpr int kBackRegs = 168;                        // at launch
// 256 * 200 + 128 * 104 = 384 * 168.  Of 184 to 216 for the scan warps, 200 is the
// fastest (backward call at 16 x 2048 x 512 bf16: 192 512 us, 200 482, 208 517).
constexpr int kScanRegs = 200, kElementRegs = 104;
static_assert(kBackScan * kScanRegs + 128 * kElementRegs == kBackThreads * kBackRegs,
              "the warpgroups share what the block was launched with");

// Shared memory of the backward kernel, in floats.  A slot holds one pass: the
// staged {d, d, d x, d x} and {g, g} of every token and channel (twice, as the
// paired operations take them), the channels' states at the tile's start, and
// the sums the scan warps return.
struct BackSmem {
  static constexpr int kSums = kBack * kBackPitch;
  static constexpr int gg = kBack * kBackCh * 4, h0 = gg + kBack * kBackCh * 2, sums = h0 + kBackCh * kN;
  static constexpr int kSlot = sums + 3 * kSums;
  static constexpr int kBc = kBack * 2 * kN;
  static constexpr int bc = 2 * kSlot, red = bc + 2 * kBc, carry = red + kBackScan / 32 * kBc;
  // per channel of the block: dh[16], dA[16], A[16] in units of log2, D, dt_bias, and dD, ddt_bias by staging row
  static constexpr int per_channel = 3 * kN + 2 + 2 * kBack;
  __host__ __device__ static constexpr int floats(int passes) { return carry + passes * kBackCh * per_channel; }
};
static_assert(BackSmem::floats(kPasses) * 4 <= 227 * 1024, "shared memory of a block");

// A block takes one part of a row and up to 512 channels, tile by tile (8
// tokens) from the end, 64 channels a pass.  The last four warps stage a pass
// (softplus and the gate, once an element) and finish its gradients; the first
// eight recompute h over the tile from its checkpoint with a and h in registers
// and then run the gradient of the state backwards.  The two work on
// neighbouring passes, two slots of shared memory apart.  dB and dC of a tile
// gather over its passes in the scan warps' registers (hence setmaxnreg) and
// are summed over lanes and warps once a tile; with one channel group they are
// final, else the groups' sums go to bc_parts.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kBackThreads, 1)
    k_ssm_backward(const boa_ssm_args a, const SsmPlan p, int passes, int groups, const float* __restrict__ starts,
                   float* __restrict__ bc_parts, float* __restrict__ param_parts) {
  extern __shared__ __align__(16) float sm[];
  using S = BackSmem;
  const int E = a.channels, group = blockIdx.x % groups;
  const int part = (blockIdx.x / groups) % p.parts, b = blockIdx.x / groups / p.parts;
  const int width = passes * kBackCh, e0 = group * width;
  const int np = min(passes, (E - e0 + kBackCh - 1) / kBackCh);
  const int begin = part * p.part, stop = min(begin + p.part, a.length), end = min(stop, row_len(a, b));
  const int tiles = (max(end - begin, 0) + kBack - 1) / kBack;
  float* const dh_s = sm + S::carry;
  float* const dA_s = dh_s + width * kN;
  float* const A_s = dA_s + width * kN;
  float* const D_s = A_s + width * kN;
  float* const bias_s = D_s + width;
  float* const dD_s = bias_s + width;                   // [row][channel]
  float* const db_s = dD_s + width * kBack;
  const bool gated = a.z;
  if (threadIdx.x < kBackScan) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kScanRegs));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, q = lane_q(lane), ch = warp * 8 + lane_ch(lane);
    for (int g = 0; g < np; ++g) {
      const int e = e0 + g * kBackCh + ch, at = (g * kBackCh + ch) * kN + kQ * q;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f), A = v;
      if (e < E) {
        if (p.parts > 1) {
          v = ld4(starts + (((int64_t)b * p.parts + part) * E + e) * kN + kQ * q);
        } else if (a.dstate_out) {
          const float* s = a.dstate_out + ((int64_t)b * E + e) * kN + kQ * q;
          v = make_float4(s[0], s[1], s[2], s[3]);
        }
        const float* s = a.A + (int64_t)e * kN + kQ * q;
        A = make_float4(rate_of(s[0]), rate_of(s[1]), rate_of(s[2]), rate_of(s[3]));
      }
      st4(dh_s + at, v);
      st4(dA_s + at, make_float4(0.f, 0.f, 0.f, 0.f));
      st4(A_s + at, A);
    }
    int slot = 0;
    for (int k = tiles - 1; k >= 0; --k) {
      const float* const bc = sm + S::bc + (k & 1) * S::kBc + kQ * q;
      f2 vB[kBack][2], vC[kBack][2];
#pragma unroll
      for (int t = 0; t < kBack; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) vB[t][j] = vC[t][j] = f2{0ull};
      for (int g = 0; g < np; ++g) {
        float* const sl = sm + slot * S::kSlot;
        const ulonglong2* const in = reinterpret_cast<const ulonglong2*>(sl) + ch;
        const unsigned long long* const gin = reinterpret_cast<const unsigned long long*>(sl + S::gg) + ch;
        float* const s1_s = sl + S::sums + q * kBackPitch + ch;
        float* const s2_s = s1_s + S::kSums;
        float* const sv_s = s2_s + S::kSums;
        const int at = (g * kBackCh + ch) * kN + kQ * q;
        ulonglong2 r = *reinterpret_cast<const ulonglong2*>(A_s + at);
        const f2 A2[2] = {f2{r.x}, f2{r.y}};
        f2 h[kBack][2], dec[kBack][2];
        bar_sync(kFull + slot, kBackThreads);
        r = *reinterpret_cast<const ulonglong2*>(sl + S::h0 + ch * kN + kQ * q);
        const f2 h0[2] = {f2{r.x}, f2{r.y}};
        float yp[4];
#pragma unroll
        for (int t = 0; t < kBack; ++t) {
          r = in[t * kBackCh];
          const f2 dd{r.x}, uu{r.y};
          const ulonglong2 B = *reinterpret_cast<const ulonglong2*>(bc + t * 2 * kN);
          dec[t][0] = ex2_2(mul2(dd, A2[0]));
          dec[t][1] = ex2_2(mul2(dd, A2[1]));
          h[t][0] = fma2(dec[t][0], t ? h[t - 1][0] : h0[0], mul2(uu, f2{B.x}));
          h[t][1] = fma2(dec[t][1], t ? h[t - 1][1] : h0[1], mul2(uu, f2{B.y}));
          if (gated) {
            const ulonglong2 C = *reinterpret_cast<const ulonglong2*>(bc + t * 2 * kN + kN);
            const float2 y = unpack(fma2(f2{C.x}, h[t][0], mul2(f2{C.y}, h[t][1])));
            yp[t & 3] = y.x + y.y;
            if ((t & 3) == 3) sv_s[(t - 3) * kBackPitch] = quad_sum(yp, q);
          }
        }
        r = *reinterpret_cast<const ulonglong2*>(dh_s + at);
        f2 dh[2] = {f2{r.x}, f2{r.y}};
        r = *reinterpret_cast<const ulonglong2*>(dA_s + at);
        f2 dA[2] = {f2{r.x}, f2{r.y}};
        float p1[4], p2[4];
#pragma unroll
        for (int t = kBack - 1; t >= 0; --t) {
          r = in[t * kBackCh];
          const f2 dd{r.x}, uu{r.y}, gg{gin[t * kBackCh]};
          const ulonglong2 B = *reinterpret_cast<const ulonglong2*>(bc + t * 2 * kN);
          const ulonglong2 C = *reinterpret_cast<const ulonglong2*>(bc + t * 2 * kN + kN);
          const f2 Bv[2] = {f2{B.x}, f2{B.y}}, Cv[2] = {f2{C.x}, f2{C.y}};
          f2 w[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) dh[j] = fma2(Cv[j], gg, dh[j]);
          const float2 s1 = unpack(fma2(dh[0], Bv[0], mul2(dh[1], Bv[1])));
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            vB[t][j] = fma2(dh[j], uu, vB[t][j]);
            vC[t][j] = fma2(gg, h[t][j], vC[t][j]);
            dh[j] = mul2(dh[j], dec[t][j]);
            w[j] = mul2(dh[j], t ? h[t - 1][j] : h0[j]);
            dA[j] = fma2(w[j], dd, dA[j]);
          }
          const float2 s2 = unpack(fma2(w[0], A2[0], mul2(w[1], A2[1])));
          p1[t & 3] = s1.x + s1.y;
          p2[t & 3] = s2.x + s2.y;
          if ((t & 3) == 0) {
            s1_s[t * kBackPitch] = quad_sum(p1, q);
            s2_s[t * kBackPitch] = quad_sum(p2, q);
          }
        }
        *reinterpret_cast<ulonglong2*>(dh_s + at) = make_ulonglong2(dh[0].v, dh[1].v);
        *reinterpret_cast<ulonglong2*>(dA_s + at) = make_ulonglong2(dA[0].v, dA[1].v);
        bar_arrive(kDone + slot, kBackThreads);
        slot ^= 1;
      }
      // the tile's dB and dC over the warp's 8 channels: lane bits 4, 3, 0 pick C, and the state within the lane's four
      const bool up = lane & 16, hi = lane & 8, odd = lane & 1;
      const int t0 = begin + k * kBack;
#pragma unroll
      for (int t = 0; t < kBack; ++t) {
        const float2 b0 = unpack(vB[t][0]), b1 = unpack(vB[t][1]), c0 = unpack(vC[t][0]), c1 = unpack(vC[t][1]);
        const float bb[4] = {b0.x, b0.y, b1.x, b1.y}, cc[4] = {c0.x, c0.y, c1.x, c1.y};
        float k4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          k4[j] = (up ? cc[j] : bb[j]) + __shfl_xor_sync(0xffffffffu, up ? bb[j] : cc[j], 16);
        const float k0 = (hi ? k4[2] : k4[0]) + __shfl_xor_sync(0xffffffffu, hi ? k4[0] : k4[2], 8);
        const float k1 = (hi ? k4[3] : k4[1]) + __shfl_xor_sync(0xffffffffu, hi ? k4[1] : k4[3], 8);
        const float s = (odd ? k1 : k0) + __shfl_xor_sync(0xffffffffu, odd ? k0 : k1, 1);
        sm[S::red + (warp * kBack + t) * 2 * kN + (up ? kN : 0) + kQ * q + (hi ? 2 : 0) + (odd ? 1 : 0)] = s;
      }
      bar_sync(kScanOnly, kBackScan);
      static_assert(S::kBc == kBackScan, "a thread a sum");
      {
        const int t = t0 + tid / (2 * kN), n = tid % (2 * kN);
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kBackScan / 32; ++w) s += sm[S::red + w * S::kBc + tid];
        if (t >= end) s = 0.0f;
        const int64_t rowi = (int64_t)b * a.length + t;
        if (t < stop) {
          if (groups > 1) bc_parts[((int64_t)group * a.batch * a.length + rowi) * 2 * kN + n] = s;
          else if (n < kN) ((T*)a.dB)[rowi * kN + n] = from_f<T>(s);
          else ((T*)a.dC)[rowi * kN + n - kN] = from_f<T>(s);
        }
      }
      bar_sync(kScanOnly, kBackScan);
    }
    __syncthreads();
    float* const pp = param_parts + ((int64_t)b * p.parts + part) * E * (kN + 2);
    const int channels = min(np * kBackCh, E - e0);
    for (int i = tid; i < channels * kN; i += kBackScan) {
      pp[(int64_t)e0 * kN + i] = dA_s[i];
      if (part == 0 && a.dstate) a.dstate[((int64_t)b * E + e0) * kN + i] = dh_s[i];
    }
    for (int i = tid; i < channels; i += kBackScan) {
      float sD = 0.0f, sb = 0.0f;
#pragma unroll
      for (int k = 0; k < kBack; ++k) {
        sD += dD_s[k * width + i];
        sb += db_s[k * width + i];
      }
      pp[(int64_t)E * kN + e0 + i] = sD;
      pp[(int64_t)E * (kN + 1) + e0 + i] = sb;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kElementRegs));
    const int tid = threadIdx.x - kBackScan;
    const int row = tid >> 4, sub = tid & 15, cl = 4 * sub;    // four channels of token `row`; two values of its B or C
    for (int g = 0; g < np; ++g) {
      const int at = row * width + g * kBackCh + cl;
      st4(dD_s + at, make_float4(0.f, 0.f, 0.f, 0.f));
      st4(db_s + at, make_float4(0.f, 0.f, 0.f, 0.f));
    }
    for (int i = tid; i < np * kBackCh; i += 128) {
      D_s[i] = a.D && e0 + i < E ? a.D[e0 + i] : 0.0f;
      bias_s[i] = a.dt_bias && e0 + i < E ? a.dt_bias[e0 + i] : 0.0f;
    }
    bar_sync(kScanOnly + 1, 128);
    const bool is_c = sub >= 8;
    int t = begin + (tiles - 1) * kBack + row;      // of the pass to be loaded next
    int c = e0 + cl;
    int64_t out = ((int64_t)b * a.length + t) * E + c;   // of the pass to be finished next
    const T* px = (const T*)a.x + b * a.x_bs + t * a.x_ts + c;
    const T* pd = (const T*)a.dt + b * a.dt_bs + t * a.dt_ts + c;
    const T* pz = (const T*)a.z + b * a.z_bs + t * a.z_ts + c;
    const T* pg = (const T*)a.dy + b * a.dy_bs + t * a.dy_ts + c;
    const T* pbc = is_c ? (const T*)a.C + b * a.C_bs + t * a.C_ts + 2 * (sub - 8)
                        : (const T*)a.B + b * a.B_bs + t * a.B_ts + 2 * sub;
    // states 4 (tid & 3) .. of channels tid / 4 and tid / 4 + 32 at the tile's start
    const int nck = (a.length + kBack - 1) / kBack;
    const float* pck = a.checkpoints + (((int64_t)b * nck + begin / kBack + tiles - 1) * E + e0) * kN + 4 * tid;
    float4 rh[2];
    Row<T, 4, VEC> rx, rd, rz, rg;
    Row<T, 2, VEC> rb;
    int g_next = 0;
    auto fetch = [&]() {
      const bool live = t < end;
      rx.load(px, c, E, live);
      rd.load(pd, c, E, live);
      rg.load(pg, c, E, live);
      if (gated) rz.load(pz, c, E, live);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        rh[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c - cl + (tid >> 2) + 32 * j < E) rh[j] = ld4(pck + 32 * kN * j);
      }
      if (g_next == 0) {
        rb.load(pbc, 0, 2, live);
        pbc -= kBack * (is_c ? a.C_ts : a.B_ts);
      }
      px += kBackCh;
      pd += kBackCh;
      pz += kBackCh;
      pg += kBackCh;
      pck += kBackCh * kN;
      c += kBackCh;
      if (++g_next == np) {
        const int back = np * kBackCh;
        g_next = 0;
        t -= kBack;
        c -= back;
        px -= kBack * a.x_ts + back;
        pd -= kBack * a.dt_ts + back;
        pz -= kBack * a.z_ts + back;
        pg -= kBack * a.dy_ts + back;
        pck -= ((int64_t)E + back) * kN;
      }
    };
    f2 ps[2], pz2[2], px2[2], pd2[2], pg2[2];   // of the pass staged before: sigmoid, dy silu'(z), x, d, g
    const f2 one = pack(1.0f, 1.0f), minus = pack(-1.0f, -1.0f), ln2 = pack(kLn2, kLn2);
    auto finish = [&](int slot, int g, bool store, bool in_row) {
      bar_sync(kDone + slot, kBackThreads);
      const float* const sums = sm + slot * S::kSlot + S::sums + row * kBackPitch + cl;
      float* const dD = dD_s + row * width + g * kBackCh + cl;
      float* const db = db_s + row * width + g * kBackCh + cl;
      f2 s1[2], s2[2], sv[2], Dv[2], aD[2], ab[2], ox[2], od[2], oz[2];
      ld2(sums, s1);
      ld2(sums + S::kSums, s2);
      ld2(sums + 2 * S::kSums, sv);
      ld2(D_s + g * kBackCh + cl, Dv);
      ld2(dD, aD);
      ld2(db, ab);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // behind the row's end every gradient is 0, whatever D or the gradient of the state hold
        ox[j] = in_row ? fma2(s1[j], pd2[j], mul2(Dv[j], pg2[j])) : f2{0ull};
        od[j] = in_row ? mul2(fma2(s1[j], px2[j], mul2(ln2, s2[j])), ps[j]) : f2{0ull};   // s2 is in units of log2
        oz[j] = gated && in_row ? mul2(pz2[j], fma2(Dv[j], px2[j], sv[j])) : f2{0ull};
        aD[j] = fma2(pg2[j], px2[j], aD[j]);
        ab[j] = add2(ab[j], od[j]);
      }
      st2(dD, aD);
      st2(db, ab);
      if (store) {
        const int oc = e0 + g * kBackCh + cl;
        store_row2<T, VEC>((T*)a.dx + out, oc, E, ox);
        store_row2<T, VEC>((T*)a.ddt + out, oc, E, od);
        if (gated) store_row2<T, VEC>((T*)a.dz + out, oc, E, oz);
      }
      out += kBackCh;
      if (g == np - 1) out -= (int64_t)kBack * E + np * kBackCh;
    };
    if (tiles) fetch();
    int slot = 0;
    bool have = false;
    for (int k = tiles - 1; k >= 0; --k) {
      const int ts = begin + k * kBack + row;
      const bool in_row = ts < end;
      for (int g = 0; g < np; ++g) {
        f2 bias[2], sg[2], dz[2], xs[2], ds[2], gs[2];
        ld2(bias_s + g * kBackCh + cl, bias);
        float* const sl = sm + slot * S::kSlot;
        float* const in = sl + 4 * (row * kBackCh + cl);
        float* const gg = sl + S::gg + 2 * (row * kBackCh + cl);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const f2 raw = add2(pack(rd.get(2 * j), rd.get(2 * j + 1)), bias[j]);
          xs[j] = pack(rx.get(2 * j), rx.get(2 * j + 1));
          gs[j] = pack(rg.get(2 * j), rg.get(2 * j + 1));
          f2 d = raw;
          sg[j] = one;
          dz[j] = f2{0ull};
          if (a.softplus) {
            f2 u;
            d = softplus2(raw, u);
            // sigmoid(raw) = (raw >= 0 ? 1 : u) / (1 + u), u = exp(-|raw|)
            const float2 r = unpack(raw), uv = unpack(u), q = unpack(add2(u, one));
            sg[j] = pack((r.x >= 0.0f ? 1.0f : uv.x) * rcp(q.x), (r.y >= 0.0f ? 1.0f : uv.y) * rcp(q.y));
          }
          if (!in_row) d = f2{0ull};
          if (gated) {
            const f2 z = pack(rz.get(2 * j), rz.get(2 * j + 1)), s = vsigmoid<2>(Fv<2>{{z}}).p[0], zs = mul2(z, s);
            // silu'(z) = s + z s (1 - s)
            dz[j] = mul2(gs[j], fma2(zs, fma2(s, minus, one), s));
            gs[j] = mul2(gs[j], zs);
          }
          const float2 dv = unpack(d), uv = unpack(mul2(d, xs[j])), gv = unpack(gs[j]);
          st4(in + 8 * j, make_float4(dv.x, dv.x, uv.x, uv.x));
          st4(in + 8 * j + 4, make_float4(dv.y, dv.y, uv.y, uv.y));
          st4(gg + 4 * j, make_float4(gv.x, gv.x, gv.y, gv.y));
          ds[j] = d;
        }
        st4(sl + S::h0 + 4 * tid, rh[0]);
        st4(sl + S::h0 + 32 * kN + 4 * tid, rh[1]);
        if (g == 0)
          *reinterpret_cast<float2*>(sm + S::bc + (k & 1) * S::kBc + row * 2 * kN + 2 * sub) =
              make_float2(rb.get(0), rb.get(1));
        bar_arrive(kFull + slot, kBackThreads);
        if (g + 1 < np || k > 0) fetch();
        if (have) {
          // the pass before: of this tile, or the last of the tile behind
          const int tp = g ? ts : ts + kBack;
          finish(slot ^ 1, g ? g - 1 : np - 1, tp < stop, tp < end);
        }
        have = true;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          ps[j] = sg[j];
          pz2[j] = dz[j];
          px2[j] = xs[j];
          pd2[j] = ds[j];
          pg2[j] = gs[j];
        }
        slot ^= 1;
      }
    }
    if (have) finish(slot ^ 1, np - 1, begin + row < stop, begin + row < end);
    // tiles wholly behind the row's end
    const float zero[4] = {};
    for (int tz = begin + tiles * kBack + row; tz < stop; tz += kBack) {
      const int64_t rowi = (int64_t)b * a.length + tz;
      for (int g = 0; g < np; ++g) {
        const int oc = e0 + g * kBackCh + cl;
        const int64_t o = rowi * E + oc;
        store_row<T, 4, VEC>((T*)a.dx + o, oc, E, zero);
        store_row<T, 4, VEC>((T*)a.ddt + o, oc, E, zero);
        if (gated) store_row<T, 4, VEC>((T*)a.dz + o, oc, E, zero);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = 2 * sub + j;
        if (groups > 1) bc_parts[((int64_t)group * a.batch * a.length + rowi) * 2 * kN + n] = 0.0f;
        else if (n < kN) ((T*)a.dB)[rowi * kN + n] = from_f<T>(0.0f);
        else ((T*)a.dC)[rowi * kN + n - kN] = from_f<T>(0.0f);
      }
    }
    __syncthreads();
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
// Four states of a channel a thread, for ROWS streams: A is read once for all of
// them, and their states are in flight together.  VEC: B and C rows start on
// four elements.
template <typename T, int ROWS, bool VEC>
__global__ void __launch_bounds__(256) k_ssm_step(const boa_ssm_args a) {
  const int E = a.channels;
  const int64_t per = E * 4LL;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t b0 = i / per * ROWS, r = i % per;
  const int e = (int)(r >> 2), q = (int)(r & 3);
  // the four lanes of a channel take the same streams: per and the block are multiples of four
  if (b0 >= a.batch) return;
  const unsigned mask = 0xfu << (threadIdx.x & 28);
  const int n = (int)min((int64_t)ROWS, a.batch - b0);
  float4* const st = reinterpret_cast<float4*>(a.state_out + (b0 * E + e) * kN + kQ * q);
  float4 h4[ROWS];
  Row<T, 4, VEC> B[ROWS], C[ROWS];
  T x[ROWS], dt[ROWS], z[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k)
    if (k < n) {
      const int64_t b = b0 + k;
      h4[k] = st[(int64_t)k * E * kQ];
      B[k].load((const T*)a.B + b * a.B_bs + kQ * q, 0, 4, true);
      C[k].load((const T*)a.C + b * a.C_bs + kQ * q, 0, 4, true);
      x[k] = ((const T*)a.x)[b * a.x_bs + e];
      dt[k] = ((const T*)a.dt)[b * a.dt_bs + e];
      if (a.z) z[k] = ((const T*)a.z)[b * a.z_bs + e];
    }
  const float4 A4 = *reinterpret_cast<const float4*>(a.A + (int64_t)e * kN + kQ * q);
  const f2 A2[2] = {pack(rate_of(A4.x), rate_of(A4.y)), pack(rate_of(A4.z), rate_of(A4.w))};
  const float bias = a.dt_bias ? a.dt_bias[e] : 0.0f, D = a.D ? a.D[e] : 0.0f;
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    if (k >= n) break;
    const float xk = to_f(x[k]), d = step_of(to_f(dt[k]) + bias, a.softplus), du = d * xk;
    const f2 dd = pack(d, d), uu = pack(du, du);
    const f2 lo = fma2(ex2_2(mul2(dd, A2[0])), pack(h4[k].x, h4[k].y), mul2(uu, pack(B[k].get(0), B[k].get(1))));
    const f2 hi = fma2(ex2_2(mul2(dd, A2[1])), pack(h4[k].z, h4[k].w), mul2(uu, pack(B[k].get(2), B[k].get(3))));
    const float2 l = unpack(lo), g = unpack(hi);
    st[(int64_t)k * E * kQ] = make_float4(l.x, l.y, g.x, g.y);
    const float2 yy = unpack(fma2(pack(C[k].get(0), C[k].get(1)), lo, mul2(pack(C[k].get(2), C[k].get(3)), hi)));
    float v = yy.x + yy.y;
    v += __shfl_xor_sync(mask, v, 2);
    v += __shfl_xor_sync(mask, v, 1);
    if (q == 0) {
      v = fmaf(D, xk, v);
      if (a.z) {
        const float zk = to_f(z[k]);
        v *= zk * sigmoid_f(zk);
      }
      ((T*)a.y)[(b0 + k) * E + e] = from_f<T>(v);
    }
  }
}

// --------------------------------------------------------------------- host
static int round_up(int v, int m) { return (v + m - 1) / m * m; }

// Parts of the length for the forward call.  One where the rows alone give 256
// blocks; one part against many (1776 blocks), bf16: at 256 blocks 159 and 206 us
// (16 x 2048 x 512), 45 and 71 us (64 x 512 x 128), at 512 blocks 538 and 698 us
// (32 x 4096 x 512); at 192 blocks 307 and 292 us (12 x 4096 x 512), at 128 blocks
// 265 and 212 us (8 x 4096 x 512), at 64 blocks 262 and 116 us (4 x 4096 x 512).
// Else enough parts for three rounds of the four blocks that an SM holds (two
// rounds and one and a half: 410 and 441 against 404 us at 1 x 67109 x 512, 208
// and 222 against 212 us at 8 x 4096 x 512), no part shorter than 64 tokens.
static SsmPlan plan_forward(const boa_ssm_args& a) {
  SsmPlan p{};
  p.cblocks = (a.channels + kCh - 1) / kCh;
  const int64_t blocks = (int64_t)a.batch * p.cblocks;
  int64_t parts = 1;
  if (blocks < 256) {
    const int64_t most = (a.length + 63) / 64, need = (1776 + blocks - 1) / blocks;
    parts = need < most ? need : most;
    if (parts < 1) parts = 1;
  }
  p.part = round_up((int)((a.length + parts - 1) / parts), kTile);
  if (p.part < kTile) p.part = kTile;
  p.parts = a.length > 0 ? (a.length - 1) / p.part + 1 : 1;
  return p;
}

static int back_passes(const boa_ssm_args& a) {
  const int n = (a.channels + kBackCh - 1) / kBackCh;
  return n < kPasses ? n : kPasses;
}
static int back_groups(const boa_ssm_args& a) {
  const int per = back_passes(a) * kBackCh;
  return (a.channels + per - 1) / per;
}
// Parts for the backward call, whose blocks have an SM each: of 1 to 8 rounds of
// 148 blocks, the one with the least tokens to walk one after the other (about
// 6 tokens' time a block for its start and end), more rounds where they cost
// at most 3 % more, since rows of different lengths then even out.  The pass for
// the parts' end gradients is not in this cost, and neither are the rows' lengths,
// which the host does not know.  One part against the parts taken, at 512 channels
// bf16: rows of half to full length gain (148 x 4096: 6603 and 6485 us; 128 x 4096:
// 6499 and 5436 us), full rows enough to fill the SMs lose (128 x 4096: 6629 and
// 7082 us; 148 x 4096: 6684 and 8037 us; 296 x 2048: 6631 and 7847 us), fewer gain
// (64 x 4096: 6590 and 3566 us; 32 x 4096: 6537 and 1882 us).
static SsmPlan plan_backward(const boa_ssm_args& a) {
  SsmPlan p{};
  p.cblocks = (a.channels + kCh - 1) / kCh;
  const int64_t blocks = (int64_t)a.batch * back_groups(a), most = (a.length + 31) / 32;
  int64_t best = -1;
  for (int rounds = 1; rounds <= 8; ++rounds) {
    int64_t parts = 148LL * rounds / blocks;
    parts = parts < 1 ? 1 : parts < most ? parts : most < 1 ? 1 : most;
    const int part = round_up((int)((a.length + parts - 1) / parts), kBack);
    const int n = part > 0 ? (a.length - 1) / part + 1 : 1;
    const int64_t cost = (blocks * n + 147) / 148 * (part + 6);
    if (best < 0 || cost * 100 <= best * 103) {
      p.part = part > kBack ? part : kBack;
      p.parts = n > 1 ? n : 1;
      best = best < 0 || cost < best ? cost : best;
    }
  }
  return p;
}

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
    k_ssm_ends<T, VEC><<<(unsigned)((int64_t)p.cblocks * (p.parts - 1) * a.batch), kSsmThreads, 0, s>>>(a, p, ends, dsum);
    const int64_t n = (int64_t)a.batch * a.channels * kN;
    k_ssm_join<<<(unsigned)((n + 127) / 128), 128, 0, s>>>(n, a.channels, p.parts, a.A, a.state, ends, dsum, false);
  }
  k_ssm<T, VEC><<<(unsigned)((int64_t)p.cblocks * p.parts * a.batch), kScanThreads, 0, s>>>(a, p, ends);
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
  float* params = bc + (groups > 1 ? (size_t)groups * a.batch * a.length * 2 * kN : 0);
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
  // setmaxnreg moves registers between the two warpgroups: the launch has to hold exactly their sum
  cudaFuncAttributes fa{};
  BOA_CUDA(cudaFuncGetAttributes(&fa, k_ssm_backward<T, VEC>));
  if (fa.numRegs != kBackRegs)
    return boa_fail(BOA_ERR_UNSUPPORTED, "boa_ssm_scan_backward: built with another register count than its split");
  // the bound of all calls, not this one's size: another thread may launch between here and the launch
  BOA_CUDA(cudaFuncSetAttribute(k_ssm_backward<T, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                BackSmem::floats(kPasses) * (int)sizeof(float)));
  k_ssm_backward<T, VEC><<<(unsigned)((int64_t)groups * p.parts * a.batch), kBackThreads, smem, s>>>(a, p, passes, groups,
                                                                                             ends, bc, params);
  const int64_t rows = (int64_t)a.batch * a.length, n = rows * 2 * kN;
  if (n > 0 && groups > 1)
    k_ssm_bc<T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(rows, groups, bc, (T*)a.dB, (T*)a.dC);
  const int64_t E = a.channels, cols = E * (kN + 2);
  k_sum_parts<<<(unsigned)((cols + 31) / 32), 1024, 0, s>>>(params, (int64_t)a.batch * p.parts, cols, E * kN,
                                                           E * (kN + 1), a.dA, a.dD, a.ddt_bias);
  BOA_CUDA(cudaGetLastError());
  return BOA_OK;
}

template <typename T>
static int ssm_backward(const boa_ssm_args& a, cudaStream_t s) {
  return ssm_vec(a, true) ? ssm_backward_t<T, true>(a, s) : ssm_backward_t<T, false>(a, s);
}

template <typename T, int ROWS>
static void ssm_step_rows(const boa_ssm_args& a, cudaStream_t s) {
  const int64_t n = (a.batch + (ROWS - 1LL)) / ROWS * a.channels * 4;
  const unsigned grid = (unsigned)((n + 255) / 256);
  if (row_vec(a.B, a.B_bs, 0, sizeof(T)) && row_vec(a.C, a.C_bs, 0, sizeof(T)))
    k_ssm_step<T, ROWS, true><<<grid, 256, 0, s>>>(a);
  else
    k_ssm_step<T, ROWS, false><<<grid, 256, 0, s>>>(a);
}

// Two streams a thread where that still fills the GPU, else one: at 8192 x 512
// bf16 one takes 165 us, two 112, four 120 (fewer warps an SM), of 87 us that the
// bytes take.
template <typename T>
static void ssm_step_launch(const boa_ssm_args& a, cudaStream_t s) {
  if ((int64_t)a.batch * a.channels * 4 >= 2 * 148LL * 2048) ssm_step_rows<T, 2>(a, s);
  else ssm_step_rows<T, 1>(a, s);
}

static int ssm_check(const boa_ssm_args* a, const char* who) {
  if (!a) return boa_fail(BOA_ERR_ARG, std::string(who) + ": null arguments");
  if (a->batch < 0 || a->length < 0 || a->channels < 1)
    return boa_fail(BOA_ERR_ARG, std::string(who) + ": need batch >= 0, length >= 0 and channels >= 1");
  if (a->length > kMaxSize || a->channels > kMaxSize)
    return boa_fail(BOA_ERR_UNSUPPORTED, std::string(who) + ": length and channels must be below 2^31 - 2^16");
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
  const size_t groups = back_groups(*a);
  return (ends_floats(*a, p) + (groups > 1 ? groups * a->batch * a->length * 2 * kN : 0) +
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
  if (a->dtype == BOA_DTYPE_F32) ssm_step_launch<float>(*a, s);
  else if (a->dtype == BOA_DTYPE_BF16) ssm_step_launch<__nv_bfloat16>(*a, s);
  else ssm_step_launch<__half>(*a, s);
  BOA_CUDA(cudaGetLastError());
  return BOA_OK;
}

}  // extern "C"
