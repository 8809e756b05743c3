// The selective scan as an operator of its own, with its gradient: per lane l,
// channel c and state n, over the lane's positions t,
//
//   delta = softplus(x + bias[c]),  a[n] = e^(delta A[c][n])
//   h[n]  = a[n] h[n] + delta B[t][n] u
//   y     = sum_n C[t][n] h[n] + D[c] u,   out = y z sigmoid(z)
//
// and backwards, with dy = dout z sigmoid(z) and g the gradient of the state
// that t + 1 received:
//
//   dh[n] = g[n] + C[t][n] dy,   g[n] = a[n] dh[n]
//   m[n]  = g[n] h[t - 1][n],    I = sum_n dh[n] B[t][n]
//   du = D dy + delta I,  dx = (sum_n m[n] A[n] + u I) sigmoid(x + bias)
//   dz = dout y sigmoid(z) (1 + z (1 - sigmoid(z)))
//   dB[t][n] = sum_c dh delta u,  dC[t][n] = sum_c h dy
//   dA = sum m delta,  dD = sum dy u,  dbias = sum dx
//
// Four states of a channel belong to a thread, so 4 (or 8, with 32 states)
// neighbouring lanes hold a channel and a wave 16 (8) of them: sums over n
// are two or three DPP adds and sums over the wave's channels fold eight
// values with lane swaps.  A block takes 64 channels of one lane and walks
// tiles of SCAN_TILE positions; the values that are the same for all states
// of a (position, channel) -- softplus, the gate, the products with u -- are
// computed once per tile by the thread that owns them and pass through LDS.
// The backward pass recomputes a tile's states from the one that the forward
// pass saved at the tile's start and keeps them and the decays in registers.
//
// Bound by VALU issue: four states of a position take 23 instructions in the
// segments' passes, 33 forward and 99 backward, four of them exponentials that
// take as long as three or four others and, backward, seven lane swaps as long
// as those.  32 lanes x 1024 positions x 512 channels of 16 states, bf16,
// in 8 segments: 43 us and 72 forward (VALU busy 100 and 99 %), 46 and 217
// backward (100 and 90 %), 13 for the blocks' sums; the rows alone would take 72
// at the rate of a copy.
#include <algorithm>

#include "scan_lanes.h"
#include "train_kernels.h"

namespace boa {

namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.693147180559945309417f;
constexpr int CH = 64;  // channels of a block
constexpr float NEVER = -__builtin_huge_valf();  // the x whose delta is 0
// Positions whose staged values are read from LDS ahead of their use: left to
// itself the compiler reads them right before, and waits.
constexpr int AHEAD = 2;

// log(1 + e^x) = max(x, 0) + log(1 + e), e = e^-|x| in (0, 1]: the logarithm of
// y = 1 + e rounded, whose hardware form is good to an ulp down to y = 1, plus
// what the rounding lost (over y, which is 1 where that counts).  Without
// branches; x = -inf gives 0.
__device__ __forceinline__ float softplus_full(float x) {
  const float e = __builtin_amdgcn_exp2f(-__builtin_fabsf(x) * LOG2E);
  const float y = 1.0f + e, lost = e - (y - 1.0f);
  // max(NaN, 0) is 0, but e is a NaN then
  return __builtin_fmaxf(x, 0.0f) + __builtin_fmaf(__builtin_amdgcn_logf(y), LN2, lost);
}
__device__ __forceinline__ float sigmoid_hw(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-x * LOG2E));
}

// A in powers of two, kept finite: where delta is 0 (past a lane's end), 0 times
// an infinity would not leave the state as it is
__device__ __forceinline__ float rate2(float A) {
  constexpr float MOST = 3.402823466e38f;
  const float r = A * LOG2E;
  return r < -MOST ? -MOST : r > MOST ? MOST : r;  // a NaN stays one
}

// The elements of a row tensor that a thread owns: in each tile of lane l the
// same ones, off elements from the tile's first row.  The tile's address is
// uniform (scalar registers), a thread keeps 32 bits of its own.
template <typename P>
struct Tensor {
  P* lane;
  int64_t row;
  uint32_t off;
  template <typename R>
  __device__ __forceinline__ Tensor(const R& r, int l, int t, int i)
      : lane((P*)r.d + l * r.lane), row(r.row), off((uint32_t)t * (uint32_t)r.row + i) {}
  __device__ __forceinline__ P* at(int tile) const {
    uint32_t o = off;
    // not known to be the same in every tile: lane + off would take two
    // registers for each tensor throughout
    asm volatile("" : "+v"(o));
    return lane + (int64_t)tile * SCAN_TILE * row + o;
  }
};

// EV neighbouring elements of a row, as 32-bit words: EV fp32, or EV / 2 pairs of bf16
template <typename TE, int EV>
struct Raw {
  uint32_t w[EV * sizeof(TE) / 4];
};
template <typename TE, int EV, bool VEC>
__device__ __forceinline__ Raw<TE, EV> ld_raw(const Tensor<const TE>& x, int tile, int c, int C,
                                              bool ok) {
  Raw<TE, EV> r;
  constexpr int W = EV * sizeof(TE) / 4;
#pragma unroll
  for (int i = 0; i < W; ++i) r.w[i] = 0;
  const TE* p = x.at(tile);
  if constexpr (VEC) {
    if (ok && c < C) {
      if constexpr (W == 4) {
        const uint4 t = *reinterpret_cast<const uint4*>(p);
        r.w[0] = t.x; r.w[1] = t.y; r.w[2] = t.z; r.w[3] = t.w;
      } else if constexpr (W == 2) {
        const uint2 t = *reinterpret_cast<const uint2*>(p);
        r.w[0] = t.x; r.w[1] = t.y;
      } else {
        r.w[0] = *reinterpret_cast<const uint32_t*>(p);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < EV; ++i)
      if (ok && c + i < C) {
        if constexpr (sizeof(TE) == 4) r.w[i] = f2u(p[i]);
        else r.w[i / 2] |= (uint32_t)p[i] << (16 * (i % 2));
      }
  }
  return r;
}
template <typename TE, int EV>
__device__ __forceinline__ float raw_at(const Raw<TE, EV>& r, int i) {
  if constexpr (sizeof(TE) == 4) return u2f(r.w[i]);
  else return u2f(i % 2 ? r.w[i / 2] & 0xFFFF0000u : r.w[i / 2] << 16);
}
// EV neighbouring floats of a staged row
template <int EV>
__device__ __forceinline__ void st_lds(float* p, const float (&v)[EV]) {
  if constexpr (EV == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
}
template <int EV>
__device__ __forceinline__ void ld_lds(const float* p, float (&v)[EV]) {
  if constexpr (EV == 4) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  } else {
    const float2 t = *reinterpret_cast<const float2*>(p);
    v[0] = t.x; v[1] = t.y;
  }
}
template <typename TE, int EV, bool VEC>
__device__ __forceinline__ void st_row(const Tensor<TE>& x, int tile, int c, int C, bool ok,
                                       const float (&v)[EV]) {
  TE* p = x.at(tile);
  if constexpr (VEC) {
    if (ok && c < C) {
      constexpr int W = EV * sizeof(TE) / 4;
      uint32_t w[W];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if constexpr (sizeof(TE) == 4) w[i] = f2u(v[i]);
        else w[i] = bf16_pair(v[2 * i], v[2 * i + 1]);
      }
      if constexpr (W == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
      else if constexpr (W == 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(p) = w[0];
    }
  } else {
#pragma unroll
    for (int i = 0; i < EV; ++i)
      if (ok && c + i < C) stv(p + i, v[i]);
  }
}

// N states of a channel on TPC lanes
template <int N>
struct Shape {
  static constexpr int TPC = N / 4, BT = CH * TPC;  // lanes a channel, threads a block
  static constexpr int EV = SCAN_TILE * CH / BT;    // row elements a thread owns in a tile
  static constexpr int WAVES = BT / 64;
};

// a thread's four states, at any float's address; zero where there are none
__device__ __forceinline__ void ld_states(const float* p, bool ok, float (&v)[4]) {
  f4_any t = {0.0f, 0.0f, 0.0f, 0.0f};
  if (p && ok) t = *reinterpret_cast<const f4_any*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = t[i];
}

// sum over the TPC lanes of a channel, in all of them
template <int TPC>
__device__ __forceinline__ float sum_states(float x) {
  x = dpp_add<DPP_XOR1>(x);
  x = dpp_add<DPP_XOR2>(x);
  if constexpr (TPC == 8) x = dpp_add<DPP_HALF_MIRROR>(x);
  return x;
}

// the lane operations of scan_lanes.h
struct Lanes {
  int i;
  struct Pair {
    float a, b;
  };
  __device__ __forceinline__ float xor1(float x) const { return dpp_move<DPP_XOR1>(x); }
  __device__ __forceinline__ float xor2(float x) const { return dpp_move<DPP_XOR2>(x); }
  __device__ __forceinline__ float half_mirror(float x) const { return dpp_move<DPP_HALF_MIRROR>(x); }
  __device__ __forceinline__ float ror8(float x) const { return dpp_move<DPP_ROR8>(x); }
  __device__ __forceinline__ float fold16(float x, float y) const { return boa::fold16(x, y); }
  __device__ __forceinline__ Pair swap32(float x, float y) const {
    const auto s = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(y), false, false);
    return Pair{u2f(s[0]), u2f(s[1])};
  }
  __device__ __forceinline__ float pick(int bit, float x, float y) const { return i & bit ? x : y; }
  __device__ __forceinline__ float fma(float x, float y, float z) const { return __builtin_fmaf(x, y, z); }
};

// How the blocks divide the work: lane, segment of the tiles, channel block.
// Few lanes are cut into segments, so that there are blocks for every CU: a
// pass over a segment from a zero state gives the state that it adds, the
// segments' states are chained (their decay is e^(A sum of delta)), and the
// main pass starts every segment from its own.  That pass costs about half of
// the main one, so lanes that give every SIMD two waves by themselves stay whole
// (512 positions x 512 channels bf16, forward and gradient: 64 lanes whole 315
// us, in two 363; 32 lanes whole 224, in 8 215).  Up to eight waves a SIMD even
// out lanes of different lengths (16 x up to 1041 fp32: 239, 229 and 196 us with
// two, four and eight); lanes of one length would take four (32 x 512 and 32 x
// 1024 bf16: 204 and 385 us, with eight 215 and 391).  More segments than 256
// cost more to chain than they save (1 x 16,001 x 128, forward: 37, 33 and 36 us
// with 128, 256 and 512).
struct Plan {
  int tiles, cblocks, segs, seg_tiles;
};
constexpr int WHOLE_WAVES = 2048, SEG_WAVES = 8192, MAX_SEGS = 256;
Plan scan_plan(int lanes, int T, int C, int ds) {
  Plan p;
  p.tiles = (T + SCAN_TILE - 1) / SCAN_TILE;
  p.cblocks = (C + CH - 1) / CH;
  const int64_t waves =
      (int64_t)lanes * p.cblocks * (ds == 16 ? Shape<16>::WAVES : Shape<32>::WAVES);
  int64_t segs = waves >= WHOLE_WAVES ? 1 : SEG_WAVES / waves;
  segs = std::min<int64_t>(std::max<int64_t>(segs, 1), std::min(p.tiles, MAX_SEGS));
  p.seg_tiles = (int)((p.tiles + segs - 1) / segs);
  p.segs = (p.tiles + p.seg_tiles - 1) / p.seg_tiles;
  return p;
}
// a block's part of it
struct Part {
  int l, seg, cb;
};
__device__ __forceinline__ Part block_part(const Plan& p, int segs) {
  const int cb = blockIdx.x % p.cblocks, r = blockIdx.x / p.cblocks;
  return Part{r / segs, r % segs, cb};
}
// The segments' states [lane][seg][C][N] and sums of delta [lane][seg][C].  Up
// to CHAIN_SEGS segments every block of the main pass chains those before its
// own itself; more would read too much, and a kernel between the passes puts
// what enters each segment in their place (`entered`).  (4 lanes x 257, 17
// segments, forward and gradient: 43 us with that kernel, 38 without; 4 x 2000
// and 1 x 16,001 x 128, forward: 25 and 33 us with it, 50 and 61 without.)  So does
// a call whose state is updated in place: a lane's last segment stores it, and
// blocks of its other segments may not have begun by then.
constexpr int CHAIN_SEGS = 32;
struct Carry {
  float *state, *sum;
  bool entered;
};

// A state after a segment whose decay is 2^x and that adds s to it.  The decay
// is r^2, r = 2^(x / 2): it may leave fp32's range where the state that goes
// through it does not.  r stays finite, since infinity times a state of zero
// would be NaN; any other state overflows with the largest r as well.
__device__ __forceinline__ float half_decay(float x) {
  return __builtin_fminf(__builtin_amdgcn_exp2f(0.5f * x), 3.402823466e38f);
}
__device__ __forceinline__ float pass_segment(float r, float h, float s) {
  return __builtin_fmaf(r, r * h, s);
}

// What enters segment `seg` of lane l for a thread's four states of channel c:
// the chain from `first` (null: zero) over the segments before it (REV: after
// it, from the last).
template <int N, bool REV>
__device__ __forceinline__ void enter_segment(const Carry& cy, const float* first, int segs, int l,
                                              int seg, int c, int C, int q, const float (&A2)[4],
                                              float (&h)[4]) {
  const bool on = c < C;
  if (cy.entered) {
    ld_states(cy.state + (((size_t)l * segs + seg) * C + c) * N + 4 * q, on, h);
    return;
  }
  ld_states(first ? first + ((size_t)l * C + c) * N + 4 * q : nullptr, on, h);
  if (!on) return;
  const int n = REV ? segs - 1 - seg : seg;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const size_t at = ((size_t)l * segs + (REV ? segs - 1 - i : i)) * C + c;
    float s[4];
    ld_states(cy.state + at * N + 4 * q, true, s);
    const float d = cy.sum[at];
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = pass_segment(half_decay(A2[j] * d), h[j], s[j]);
  }
}

// What a segment does to the state that enters it.  Forward: the state that
// it leaves when it starts from zero.  Backward (REV): the gradient of the
// state that enters it, when that of the state it leaves is zero.  And the
// sum of its deltas.
template <typename TE, int N, bool VEC, bool REV>
__global__ __launch_bounds__((Shape<N>::BT)) void scan_local_kernel(const ScanGradArgs g, Plan pl,
                                                                    Carry cy) {
  using S = Shape<N>;
  constexpr int TPC = S::TPC, BT = S::BT, EV = S::EV;
  __shared__ __align__(16) float s_delta[SCAN_TILE][CH], s_x[SCAN_TILE][CH];
  __shared__ __align__(16) float s_v[SCAN_TILE][N];
  const ScanArgs& a = g.f;
  const Part pt = block_part(pl, pl.segs - 1);  // the last (REV: the first) is not asked for
  const int tid = threadIdx.x, cb = pt.cb, l = pt.l, seg = pt.seg + (REV ? 1 : 0);
  const int len = seq_len(a.q, l), q = tid % TPC, ch = tid / TPC, c = cb * CH + ch;
  const int ot = tid / (CH / EV), oc = (tid % (CH / EV)) * EV, gc = cb * CH + oc;
  float h[4] = {0.0f, 0.0f, 0.0f, 0.0f}, A2[4], sum = 0.0f;
  ld_states(a.A + (size_t)c * N + 4 * q, c < a.C, A2);
#pragma unroll
  for (int i = 0; i < 4; ++i) A2[i] = rate2(A2[i]);
  float bias[EV];
#pragma unroll
  for (int j = 0; j < EV; ++j) bias[j] = gc + j < a.C ? a.bias[gc + j] : 0.0f;
  constexpr int NBC = SCAN_TILE * N / BT;
  Raw<TE, EV> ru, rx, ro;
  TE rv[NBC];  // as they are: to convert them here would wait for every load before
  const RowsIn &ri = REV ? a.z : a.u, &rows_v = REV ? a.c : a.b;
  using In = Tensor<const TE>;
  const In xu(ri, l, ot, gc), xx(a.delta, l, ot, gc), xo(REV ? g.dout : ri, l, ot, gc);
  auto fetch = [&](int tile) {
    const int t = tile * SCAN_TILE + ot;
    const bool ok = t < len;
    rx = ld_raw<TE, EV, VEC>(xx, tile, gc, a.C, ok);
    ru = ld_raw<TE, EV, VEC>(xu, tile, gc, a.C, ok);
    if constexpr (REV) ro = ld_raw<TE, EV, VEC>(xo, tile, gc, a.C, ok);
#pragma unroll
    for (int i = 0; i < NBC; ++i) {
      const int e = tid + i * BT;
      rv[i] = tile * SCAN_TILE + e / N < len ? *In(rows_v, l, e / N, e % N).at(tile) : TE(0);
    }
  };
  const int all = (len + SCAN_TILE - 1) / SCAN_TILE;
  const int lo = seg * pl.seg_tiles, n = min(all, lo + pl.seg_tiles) - lo;
  if (n > 0) fetch(REV ? lo + n - 1 : lo);
  for (int i = 0; i < n; ++i) {
    const int tile = REV ? lo + n - 1 - i : lo + i;
    const bool ok = tile * SCAN_TILE + ot < len;
    __syncthreads();
    float o_d[EV], o_x[EV];
#pragma unroll
    for (int j = 0; j < EV; ++j) {
      const float in = raw_at(rx, j) + bias[j], x = raw_at(ru, j);
      o_d[j] = softplus_full(ok ? in : NEVER);
      if constexpr (REV) o_x[j] = raw_at(ro, j) * (x * sigmoid_hw(x));
      else o_x[j] = o_d[j] * x;
    }
    st_lds(&s_delta[ot][oc], o_d);
    st_lds(&s_x[ot][oc], o_x);
#pragma unroll
    for (int j = 0; j < NBC; ++j) (&s_v[0][0])[tid + j * BT] = ldv(&rv[j]);
    __syncthreads();
    if (i + 1 < n) fetch(REV ? tile - 1 : tile + 1);
    float d[2][AHEAD], x[2][AHEAD];
    float4 V[2][AHEAD];
    auto read = [&](int p) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int k = REV ? SCAN_TILE - 1 - (p * AHEAD + j) : p * AHEAD + j;
        d[p & 1][j] = s_delta[k][ch];
        x[p & 1][j] = s_x[k][ch];
        V[p & 1][j] = *reinterpret_cast<const float4*>(&s_v[k][4 * q]);
      }
    };
    read(0);
#pragma unroll
    for (int p = 0; p < SCAN_TILE / AHEAD; ++p) {
      if (p + 1 < SCAN_TILE / AHEAD) read(p + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const float delta = d[p & 1][j], xk = x[p & 1][j];
        const float4 V4 = V[p & 1][j];
        const float v[4] = {V4.x, V4.y, V4.z, V4.w};
        sum += delta;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const float e = __builtin_amdgcn_exp2f(delta * A2[m]);
          h[m] = REV ? e * __builtin_fmaf(v[m], xk, h[m]) : __builtin_fmaf(e, h[m], xk * v[m]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (c < a.C) {
    const size_t at = ((size_t)l * pl.segs + seg) * a.C + c;
    *reinterpret_cast<float4*>(cy.state + at * N + 4 * q) = make_float4(h[0], h[1], h[2], h[3]);
    if (q == 0) cy.sum[at] = sum;
  }
}

// The state (REV: the gradient) that enters each segment, over what the
// segments added: chains of segs steps, cut among up to 16 groups of 64 (channel,
// state) pairs, each of which first finds what its own segments do.  Bound by
// latency, so a thread's whole part is under way at once and stays in registers
// (251 segments: 7 us; four loads at a time, and again for the second walk: 10).
constexpr int CARRY_GROUPS = 16, CARRY_PER = MAX_SEGS / CARRY_GROUPS;  // at most
template <bool REV>
__global__ __launch_bounds__(64 * CARRY_GROUPS) void scan_carry_kernel(
    const float* __restrict__ A, const float* __restrict__ first, int C, int N, int segs,
    Carry cy) {
  __shared__ float s_h[CARRY_GROUPS][64], s_sum[CARRY_GROUPS][64];
  const int width = C * N, cols = (width + 63) / 64, l = blockIdx.x / cols;
  const int ln = threadIdx.x & 63, g = threadIdx.x >> 6, i = (blockIdx.x % cols) * 64 + ln;
  const bool on = i < width;
  const int at = on ? i : 0, c = at / N;
  const float A2 = rate2(A[at]);
  const int groups = blockDim.x >> 6, per = (segs + groups - 1) / groups;
  const int k0 = min(segs, g * per), k1 = min(segs, k0 + per);
  // k-th segment of the chain; the last one's effect is not known and not needed
  auto seg_at = [&](int k) { return (size_t)l * segs + (REV ? segs - 1 - k : k); };
  float e[CARRY_PER], s[CARRY_PER], h = 0.0f, sum = 0.0f;
#pragma unroll
  for (int j = 0; j < CARRY_PER; ++j) {  // without branches: what is not there is read as segment 0
    const int k = k0 + j < min(k1, segs - 1) ? k0 + j : 0;
    e[j] = cy.sum[seg_at(k) * C + c];
    s[j] = cy.state[seg_at(k) * width + at];
  }
#pragma unroll
  for (int j = 0; j < CARRY_PER; ++j) {
    const bool in = k0 + j < min(k1, segs - 1);
    sum += in ? e[j] : 0.0f;
    e[j] = half_decay(A2 * (in ? e[j] : 0.0f));
    s[j] = in ? s[j] : 0.0f;
    h = pass_segment(e[j], h, s[j]);
  }
  s_h[g][ln] = h;
  s_sum[g][ln] = sum;
  __syncthreads();
  if (!on) return;
  h = first ? first[(size_t)l * width + i] : 0.0f;
#pragma unroll 4
  for (int k = 0; k < g; ++k)
    h = pass_segment(half_decay(A2 * s_sum[k][ln]), h, s_h[k][ln]);
#pragma unroll
  for (int j = 0; j < CARRY_PER; ++j) {
    if (k0 + j < k1) cy.state[seg_at(k0 + j) * width + i] = h;
    h = pass_segment(e[j], h, s[j]);
  }
}

// ---------------------------------------------------------------- forward
template <typename TE, int N, bool VEC>
__global__ __launch_bounds__((Shape<N>::BT)) void scan_kernel(const ScanArgs a, Plan pl,
                                                              Carry cy) {
  using S = Shape<N>;
  constexpr int TPC = S::TPC, BT = S::BT, EV = S::EV, YS = CH + 16;
  __shared__ __align__(16) float s_delta[SCAN_TILE][CH], s_du[SCAN_TILE][CH];
  __shared__ __align__(16) float s_b[SCAN_TILE][N], s_c[SCAN_TILE][N];
  __shared__ __align__(16) float s_y[SCAN_TILE][YS];  // stride: the lanes of a channel on other banks
  const Part pt = block_part(pl, pl.segs);
  const int tid = threadIdx.x, cb = pt.cb, l = pt.l;
  const int len = seq_len(a.q, l), q = tid % TPC, ch = tid / TPC, c = cb * CH + ch;
  const int all = (len + SCAN_TILE - 1) / SCAN_TILE, first = pt.seg * pl.seg_tiles;
  if (pt.seg > 0 && first >= all) return;  // past the lane's end
  const int tiles = min(all, first + pl.seg_tiles);
  // the row elements that this thread owns: position ot of the tile, channels oc ..
  const int ot = tid / (CH / EV), oc = (tid % (CH / EV)) * EV, gc = cb * CH + oc;
  float h[4], A2[4];
  ld_states(a.A + (size_t)c * N + 4 * q, c < a.C, A2);
#pragma unroll
  for (int i = 0; i < 4; ++i) A2[i] = rate2(A2[i]);
  enter_segment<N, false>(cy, a.state_in, pl.segs, l, pt.seg, c, a.C, q, A2, h);
  float bias[EV], D[EV];
#pragma unroll
  for (int j = 0; j < EV; ++j) {
    bias[j] = gc + j < a.C ? a.bias[gc + j] : 0.0f;
    D[j] = gc + j < a.C ? a.D[gc + j] : 0.0f;
  }
  constexpr int NBC = SCAN_TILE * N / BT;  // elements of B (and of C) a thread stages
  Raw<TE, EV> ru, rx, rz;
  TE rb[NBC], rc[NBC];  // as they are: to convert them here would wait for every load before
  using In = Tensor<const TE>;
  const In xu(a.u, l, ot, gc), xx(a.delta, l, ot, gc), xz(a.z, l, ot, gc);
  const Tensor<TE> xout(a.out, l, ot, gc);
  auto fetch = [&](int tile) {
    const int t = tile * SCAN_TILE + ot;
    const bool ok = t < len;
    ru = ld_raw<TE, EV, VEC>(xu, tile, gc, a.C, ok);
    rx = ld_raw<TE, EV, VEC>(xx, tile, gc, a.C, ok);
    rz = ld_raw<TE, EV, VEC>(xz, tile, gc, a.C, ok);
#pragma unroll
    for (int i = 0; i < NBC; ++i) {
      const int e = tid + i * BT;
      const bool in = tile * SCAN_TILE + e / N < len;
      rb[i] = in ? *In(a.b, l, e / N, e % N).at(tile) : TE(0);
      rc[i] = in ? *In(a.c, l, e / N, e % N).at(tile) : TE(0);
    }
  };
  if (first < tiles) fetch(first);
  for (int tile = first; tile < tiles; ++tile) {
    const int t = tile * SCAN_TILE + ot;
    const bool ok = t < len;
    float u[EV], gate[EV], o_d[EV], o_x[EV];
#pragma unroll
    for (int j = 0; j < EV; ++j) {
      u[j] = raw_at(ru, j);
      const float z = raw_at(rz, j);
      gate[j] = z * sigmoid_hw(z);
      // past the lane's end delta = 0: the state passes unchanged
      const float in = raw_at(rx, j) + bias[j];
      o_d[j] = softplus_full(ok ? in : NEVER);
      o_x[j] = o_d[j] * u[j];
    }
    st_lds(&s_delta[ot][oc], o_d);
    st_lds(&s_du[ot][oc], o_x);
#pragma unroll
    for (int i = 0; i < NBC; ++i) {
      const int e = tid + i * BT;
      (&s_b[0][0])[e] = ldv(&rb[i]);
      (&s_c[0][0])[e] = ldv(&rc[i]);
    }
    __syncthreads();
    if (tile + 1 < tiles) fetch(tile + 1);
    if (a.saved && c < a.C) {
      float* p = a.saved + (((size_t)l * pl.tiles + tile) * a.C + c) * N + 4 * q;
      *reinterpret_cast<float4*>(p) = make_float4(h[0], h[1], h[2], h[3]);
    }
    float y[SCAN_TILE / TPC];
    float d[2][AHEAD], x[2][AHEAD];
    float4 B[2][AHEAD], C[2][AHEAD];
    auto read = [&](int p) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int k = p * AHEAD + j;
        d[p & 1][j] = s_delta[k][ch];
        x[p & 1][j] = s_du[k][ch];
        B[p & 1][j] = *reinterpret_cast<const float4*>(&s_b[k][4 * q]);
        C[p & 1][j] = *reinterpret_cast<const float4*>(&s_c[k][4 * q]);
      }
    };
    read(0);
#pragma unroll
    for (int p = 0; p < SCAN_TILE / AHEAD; ++p) {
      if (p + 1 < SCAN_TILE / AHEAD) read(p + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int k = p * AHEAD + j;
        const float delta = d[p & 1][j], du = x[p & 1][j];
        const float4 B4 = B[p & 1][j], C4 = C[p & 1][j];
        const float bv[4] = {B4.x, B4.y, B4.z, B4.w}, cv[4] = {C4.x, C4.y, C4.z, C4.w};
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(delta * A2[i]);
          h[i] = __builtin_fmaf(e, h[i], du * bv[i]);
          s = __builtin_fmaf(cv[i], h[i], s);
        }
        s = sum_states<TPC>(s);
        // lane q of the channel keeps the positions q, q + TPC, ...
        y[k / TPC] = k % TPC == 0 || q == k % TPC ? s : y[k / TPC];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int k = 0; k < SCAN_TILE / TPC; ++k) s_y[k * TPC + q][ch] = y[k];
    __syncthreads();
    float o[EV];
    ld_lds(&s_y[ot][oc], o);
#pragma unroll
    for (int j = 0; j < EV; ++j) o[j] = __builtin_fmaf(D[j], u[j], o[j]) * gate[j];
    st_row<TE, EV, VEC>(xout, tile, gc, a.C, ok, o);
  }
  if (a.state_out && tiles == all && c < a.C)
    *reinterpret_cast<float4*>(a.state_out + ((size_t)l * a.C + c) * N + 4 * q) =
        make_float4(h[0], h[1], h[2], h[3]);
}

// One position a lane: the decode step, bound by the states' bytes.  Without
// tiles a thread computes its channel's delta and gate itself (the lanes of a
// channel the same ones), every load is under way at once, and a CU holds
// twice the blocks of the tiled kernel (1000 lanes x 512 channels of 16 states,
// fp32, states in and out: 14.6 us or 5 TB/s; the tiled kernel 40).
template <typename TE, int N>
__global__ __launch_bounds__((Shape<N>::BT)) void scan_step_kernel(const ScanArgs a, Plan pl) {
  constexpr int TPC = Shape<N>::TPC;
  const Part pt = block_part(pl, 1);
  const int l = pt.l, q = threadIdx.x % TPC, c = pt.cb * CH + threadIdx.x / TPC;
  if (c >= a.C) return;
  using In = Tensor<const TE>;
  const size_t at = ((size_t)l * a.C + c) * N + 4 * q;
  const bool on = seq_len(a.q, l) > 0;
  float h[4], A2[4];
  ld_states(a.state_in ? a.state_in + at : nullptr, true, h);
  if (a.saved) *reinterpret_cast<float4*>(a.saved + at) = make_float4(h[0], h[1], h[2], h[3]);
  if (on) {
    ld_states(a.A + (size_t)c * N + 4 * q, true, A2);
    const float u = ldv(In(a.u, l, 0, c).at(0)), z = ldv(In(a.z, l, 0, c).at(0));
    const float x = ldv(In(a.delta, l, 0, c).at(0)) + a.bias[c], D = a.D[c];
    const TE *pb = In(a.b, l, 0, 4 * q).at(0), *pc = In(a.c, l, 0, 4 * q).at(0);
    float b[4], cv[4], y = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = ldv(pb + i), cv[i] = ldv(pc + i);
    const float delta = softplus_full(x), du = delta * u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e = __builtin_amdgcn_exp2f(delta * rate2(A2[i]));
      h[i] = __builtin_fmaf(e, h[i], du * b[i]);
      y = __builtin_fmaf(cv[i], h[i], y);
    }
    y = __builtin_fmaf(D, u, sum_states<TPC>(y)) * (z * sigmoid_hw(z));
    if (q == 0) stv(Tensor<TE>(a.out, l, 0, c).at(0), y);
  }
  if (a.state_out) *reinterpret_cast<float4*>(a.state_out + at) = make_float4(h[0], h[1], h[2], h[3]);
}

// --------------------------------------------------------------- backward
// Partial sums of a block: dA [lane][seg][C][N], dD and dbias [lane][seg][C],
// and with more than one channel block dB | dC [cblock][row][2 N]
struct GradWork {
  float *bc, *da, *dd, *dbias;
};

template <typename TE, int N, bool VEC>
__global__ __launch_bounds__((Shape<N>::BT)) __attribute__((amdgpu_waves_per_eu(2, 2))) void scan_grad_kernel(const ScanGradArgs g, Plan pl,
                                                                   GradWork wk, Carry cy) {
  using S = Shape<N>;
  constexpr int TPC = S::TPC, BT = S::BT, EV = S::EV, SUMS = SCAN_TILE * CH + 16;
  __shared__ __align__(16) float s_delta[SCAN_TILE][CH], s_u[SCAN_TILE][CH], s_dy[SCAN_TILE][CH];
  __shared__ __align__(16) float s_b[SCAN_TILE][N], s_c[SCAN_TILE][N];
  // y, I and sum m A log2(e) of every (position, channel); the three on different banks
  __shared__ __align__(16) float s_sums[3 * SUMS];
  __shared__ __align__(16) float s_bc[S::WAVES][SCAN_TILE][2 * N];
  __shared__ __align__(16) float s_dd[SCAN_TILE][CH], s_dbias[SCAN_TILE][CH], s_bias[CH], s_dcoef[CH];
  const ScanArgs& a = g.f;
  const Part pt = block_part(pl, pl.segs);
  const int tid = threadIdx.x, cb = pt.cb, l = pt.l;
  const Lanes lanes{tid & 63};
  const int len = seq_len(a.q, l), q = lane_states<TPC>(tid), ch = tid / TPC, c = cb * CH + ch;
  const int ot = tid / (CH / EV), oc = (tid % (CH / EV)) * EV, gc = cb * CH + oc;
  const int w = tid >> 6;
  const int first = pt.seg * pl.seg_tiles, last = min(pl.tiles, first + pl.seg_tiles);
  float* sums = s_sums + min(tid & 3, 2) * SUMS + ch;
  float A2[4], G[4], dA[4];
  ld_states(a.A + (size_t)c * N + 4 * q, c < a.C, A2);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    A2[i] = rate2(A2[i]);
    dA[i] = 0.0f;
  }
  enter_segment<N, true>(cy, g.dstate_out, pl.segs, l, pt.seg, c, a.C, q, A2, G);
  // the owners' parameters and sums live in LDS, to leave the registers to the states
#pragma unroll
  for (int j = 0; j < EV; ++j) s_dd[ot][oc + j] = s_dbias[ot][oc + j] = 0.0f;
  if (tid < CH) {
    s_bias[tid] = cb * CH + tid < a.C ? a.bias[cb * CH + tid] : 0.0f;
    s_dcoef[tid] = cb * CH + tid < a.C ? a.D[cb * CH + tid] : 0.0f;
  }
  __syncthreads();
  constexpr int NBC = SCAN_TILE * N / BT;
  Raw<TE, EV> ru, rx, rz, ro;
  TE rb[NBC], rc[NBC];  // as they are: to convert them here would wait for every load before
  float4 rh;
  using In = Tensor<const TE>;
  const In xu(a.u, l, ot, gc), xx(a.delta, l, ot, gc), xz(a.z, l, ot, gc);
  using Out = Tensor<TE>;
  const In xo(g.dout, l, ot, gc);
  const Out odu(g.du, l, ot, gc), odx(g.ddelta, l, ot, gc), odz(g.dz, l, ot, gc);
  auto fetch = [&](int tile) {
    const int t = tile * SCAN_TILE + ot;
    const bool ok = t < len;
    ru = ld_raw<TE, EV, VEC>(xu, tile, gc, a.C, ok);
    rx = ld_raw<TE, EV, VEC>(xx, tile, gc, a.C, ok);
    rz = ld_raw<TE, EV, VEC>(xz, tile, gc, a.C, ok);
    ro = ld_raw<TE, EV, VEC>(xo, tile, gc, a.C, ok);
#pragma unroll
    for (int i = 0; i < NBC; ++i) {
      const int e = tid + i * BT;
      const bool in = tile * SCAN_TILE + e / N < len;
      rb[i] = in ? *In(a.b, l, e / N, e % N).at(tile) : TE(0);
      rc[i] = in ? *In(a.c, l, e / N, e % N).at(tile) : TE(0);
    }
    rh = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (c < a.C)
      rh = *reinterpret_cast<const float4*>(
          a.saved + (((size_t)l * pl.tiles + tile) * a.C + c) * N + 4 * q);
  };
  // dB and dC of a tile: one value of one position a thread
  auto store_bc = [&](int tile, bool zero) {
#pragma unroll
    for (int j = 0; j < SCAN_TILE * 2 * N / BT; ++j) {
      const int e = tid + j * BT, k = e / (2 * N), n = e % (2 * N), t = tile * SCAN_TILE + k;
      if (t >= a.q.T) continue;
      float v = 0.0f;
      if (!zero)
#pragma unroll
        for (int i = 0; i < S::WAVES; ++i) v += s_bc[i][k][n];
      v = t < len ? v : 0.0f;
      if (pl.cblocks > 1)
        wk.bc[(((size_t)cb * a.q.lanes + l) * a.q.T + t) * (2 * N) + n] = v;
      else if (n < N)
        stv(Out(g.db, l, k, n).at(tile), v);
      else
        stv(Out(g.dc, l, k, n - N).at(tile), v);
    }
  };
  const int tiles = max(first, min(last, (len + SCAN_TILE - 1) / SCAN_TILE));
  // positions past the lane's end take no part: their gradients are zero
  for (int tile = last - 1; tile >= tiles; --tile) {
    const int t = tile * SCAN_TILE + ot;
    const float zero[EV] = {};
    const bool ok = t < a.q.T;
    st_row<TE, EV, VEC>(odu, tile, gc, a.C, ok, zero);
    st_row<TE, EV, VEC>(odx, tile, gc, a.C, ok, zero);
    st_row<TE, EV, VEC>(odz, tile, gc, a.C, ok, zero);
    store_bc(tile, true);
  }
  if (tiles > first) fetch(tiles - 1);
  for (int tile = tiles - 1; tile >= first; --tile) {
    const int t = tile * SCAN_TILE + ot;
    const bool ok = t < len;
    float dzy[EV], xsig[EV];  // dz / y, d delta / dx; the rest is read back from LDS
    float bias[EV], o_d[EV], o_x[EV], o_y[EV];
    ld_lds(&s_bias[oc], bias);
#pragma unroll
    for (int j = 0; j < EV; ++j) {
      const float z = raw_at(rz, j), sig = sigmoid_hw(z), dout = raw_at(ro, j);
      const float in = raw_at(rx, j) + bias[j], x = ok ? in : NEVER;
      dzy[j] = dout * (sig * __builtin_fmaf(z, 1.0f - sig, 1.0f));
      xsig[j] = sigmoid_hw(x);
      o_d[j] = softplus_full(x);
      o_x[j] = raw_at(ru, j);
      o_y[j] = dout * (z * sig);
      // now, and not where they are used: that would keep what they are made of
      asm volatile("" : "+v"(dzy[j]), "+v"(xsig[j]));
    }
    st_lds(&s_delta[ot][oc], o_d);
    st_lds(&s_u[ot][oc], o_x);
    st_lds(&s_dy[ot][oc], o_y);
#pragma unroll
    for (int i = 0; i < NBC; ++i) {
      const int e = tid + i * BT;
      (&s_b[0][0])[e] = ldv(&rb[i]);
      (&s_c[0][0])[e] = ldv(&rc[i]);
    }
    const float h0[4] = {rh.x, rh.y, rh.z, rh.w};
    const int rem = len - tile * SCAN_TILE;  // positions of the tile within the lane
    __syncthreads();
    // the tile's states and decays again; two positions are read ahead
    float hs[SCAN_TILE][4], es[SCAN_TILE][4];
    {
      float d[4], x[4];
      float4 B[4];
      auto read = [&](int k) {
        d[k & 3] = s_delta[k][ch];
        x[k & 3] = s_u[k][ch];
        B[k & 3] = *reinterpret_cast<const float4*>(&s_b[k][4 * q]);
      };
      read(0), read(1);
#pragma unroll
      for (int k = 0; k < SCAN_TILE; ++k) {
        if (k % 2 == 0) {
          if (k + 2 < SCAN_TILE) read(k + 2), read(k + 3);
          __builtin_amdgcn_sched_barrier(0);
        }
        const float dl = d[k & 3], du = dl * x[k & 3];
        const float bv[4] = {B[k & 3].x, B[k & 3].y, B[k & 3].z, B[k & 3].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          es[k][i] = __builtin_amdgcn_exp2f(dl * A2[i]);
          hs[k][i] = __builtin_fmaf(es[k][i], k ? hs[k > 0 ? k - 1 : 0][i] : h0[i], du * bv[i]);
        }
      }
    }
    // and backwards, one position read ahead.  The staged values are read again,
    // at indices that the compiler does not know to be the same: kept from
    // above they would take 96 registers
    int rch = ch, rq = q;
    asm volatile("" : "+v"(rch), "+v"(rq) : "v"(hs[SCAN_TILE - 1][0]));
    float d[2], x[2], dys[2];
    float4 Bs[2], Cs[2];
    auto read = [&](int k) {
      d[k & 1] = s_delta[k][rch];
      x[k & 1] = s_u[k][rch];
      dys[k & 1] = s_dy[k][rch];
      Bs[k & 1] = *reinterpret_cast<const float4*>(&s_b[k][4 * rq]);
      Cs[k & 1] = *reinterpret_cast<const float4*>(&s_c[k][4 * rq]);
    };
    read(SCAN_TILE - 1);
#pragma unroll
    for (int k = SCAN_TILE - 1; k >= 0; --k) {
      if (k > 0) read(k - 1);
      // the next tile's rows, once half of the states' registers are free
      if (k == SCAN_TILE / 2 - 1 && tile > first) fetch(tile - 1);
      __builtin_amdgcn_sched_barrier(0);
      // Positions past the lane's end are left out: dA's terms there would be
      // zeros, but NaN beside a state or a gradient that is not finite.  (A branch
      // a position: 1.5 % of a pass of 32 x 1024 x 512 bf16; one that only clears
      // dA at the lane's last position 2.8 %, a second form for such tiles spills.)
      if (k >= rem) continue;
      const float dl = d[k & 1], du = dl * x[k & 1], dyk = dys[k & 1];
      const float4 B = Bs[k & 1], C = Cs[k & 1];
      const float bv[4] = {B.x, B.y, B.z, B.w}, cv[4] = {C.x, C.y, C.z, C.w};
      float y = 0.0f, I = 0.0f, M = 0.0f, v[4];
      const Lanes::Pair cf = lanes.swap32(du, dyk);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float dh = __builtin_fmaf(cv[i], dyk, G[i]);
        y = __builtin_fmaf(cv[i], hs[k][i], y);
        I = __builtin_fmaf(dh, bv[i], I);
        G[i] = es[k][i] * dh;
        const float m = G[i] * (k ? hs[k > 0 ? k - 1 : 0][i] : h0[i]);
        M = __builtin_fmaf(m, A2[i], M);
        dA[i] = __builtin_fmaf(m, dl, dA[i]);
        // here: put off to the end of the tile these sums would keep 64 m
        asm volatile("" : "+v"(dA[i]));
        v[i] = bc_term(lanes, dh, hs[k][i], cf);
      }
      sums[k * CH] = channel_sums<TPC>(lanes, y, I, M);
      s_bc[w][k][bc_slot<TPC>(lanes.i)] = bc_sums<TPC>(lanes, v);
    }
    __syncthreads();
    float o_u[EV], o_z[EV], I[EV], y[EV], M[EV], D[EV], u[EV], dy[EV], dl[EV], sd[EV], sb[EV];
    const int at = ot * CH + oc;
    ld_lds(&s_sums[at], y), ld_lds(&s_sums[SUMS + at], I), ld_lds(&s_sums[2 * SUMS + at], M);
    ld_lds(&s_dcoef[oc], D), ld_lds(&s_u[ot][oc], u), ld_lds(&s_dy[ot][oc], dy);
    ld_lds(&s_delta[ot][oc], dl), ld_lds(&s_dd[ot][oc], sd), ld_lds(&s_dbias[ot][oc], sb);
#pragma unroll
    for (int j = 0; j < EV; ++j) {
      o_u[j] = __builtin_fmaf(D[j], dy[j], dl[j] * I[j]);
      o_x[j] = __builtin_fmaf(u[j], I[j], M[j] * LN2) * xsig[j];
      o_z[j] = dzy[j] * __builtin_fmaf(D[j], u[j], y[j]);
      // past the lane's end the sums are whatever LDS held
      o_u[j] = ok ? o_u[j] : 0.0f;
      o_x[j] = ok ? o_x[j] : 0.0f;
      o_z[j] = ok ? o_z[j] : 0.0f;
      sd[j] = __builtin_fmaf(dy[j], u[j], sd[j]);
      sb[j] += o_x[j];
    }
    st_lds(&s_dd[ot][oc], sd);
    st_lds(&s_dbias[ot][oc], sb);
    const bool in = t < a.q.T;
    st_row<TE, EV, VEC>(odu, tile, gc, a.C, in, o_u);
    st_row<TE, EV, VEC>(odx, tile, gc, a.C, in, o_x);
    st_row<TE, EV, VEC>(odz, tile, gc, a.C, in, o_z);
    store_bc(tile, false);
    __syncthreads();
  }
  const size_t part = (size_t)l * pl.segs + pt.seg;
  if (c < a.C) {
    *reinterpret_cast<float4*>(wk.da + (part * a.C + c) * N + 4 * q) =
        make_float4(dA[0], dA[1], dA[2], dA[3]);
    if (g.dstate_in && pt.seg == 0)
      *reinterpret_cast<float4*>(g.dstate_in + ((size_t)l * a.C + c) * N + 4 * q) =
          make_float4(G[0], G[1], G[2], G[3]);
  }
  // the owners' sums over the tile's positions
  __syncthreads();
  if (tid < 2 * CH) {
    const int cc = tid % CH;
    float s = 0.0f;
    for (int k = 0; k < SCAN_TILE; ++k) s += tid < CH ? s_dd[k][cc] : s_dbias[k][cc];
    if (cb * CH + cc < a.C)
      (tid < CH ? wk.dd : wk.dbias)[part * a.C + cb * CH + cc] = s;
  }
}

// The blocks' sums of the gradient.  The first bc_blocks blocks sum dB and dC
// over the channel blocks, a value a thread; the others the parameters'
// gradients over n partials -- dA's `width` values, then dD's and dbias's C --,
// 16 columns a block, 16 groups of partials, the groups added in order.
template <typename TE>
__global__ __launch_bounds__(256) void scan_sums_kernel(GradWork wk, uint32_t bc_blocks,
                                                        int cblocks, uint32_t rows, int T, int N,
                                                        RowsOut db, RowsOut dc, int n, int width,
                                                        int C, float* __restrict__ dA,
                                                        float* __restrict__ dD,
                                                        float* __restrict__ dbias) {
  __shared__ float sm[16][16];
  if (blockIdx.x < bc_blocks) {
    const uint64_t all = (uint64_t)rows * 2 * N, step = (uint64_t)bc_blocks * 256;
    for (uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x; e < all; e += step) {
      float s = 0.0f;
#pragma unroll 4
      for (int k = 0; k < cblocks; ++k) s += wk.bc[k * all + e];
      const uint32_t r = (uint32_t)(e / (2 * N)), i = (uint32_t)(e - (uint64_t)r * 2 * N);
      const uint32_t l = r / (uint32_t)T, t = r - l * T;
      if (i < (uint32_t)N) stv((TE*)db.d + l * db.lane + t * db.row + i, s);
      else stv((TE*)dc.d + l * dc.lane + t * dc.row + i - N, s);
    }
    return;
  }
  const int ba = (width + 15) / 16, bc = (C + 15) / 16, b = blockIdx.x - bc_blocks;
  const int which = b < ba ? 0 : b < ba + bc ? 1 : 2;
  const float* part = which == 0 ? wk.da : which == 1 ? wk.dd : wk.dbias;
  float* out = which == 0 ? dA : which == 1 ? dD : dbias;
  if (which) width = C;
  const int i = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int col = (b - (which == 0 ? 0 : which == 1 ? ba : ba + bc)) * 16 + i;
  float s = 0.0f;
  if (col < width)
#pragma unroll 8
    for (int k = g; k < n; k += 16) s += part[(size_t)k * width + col];
  sm[g][i] = s;
  __syncthreads();
  if (g == 0 && col < width) {
    for (int k = 1; k < 16; ++k) s += sm[k][i];
    out[col] = s;
  }
}

// whether a thread's elements of a row can be moved at once (32 x 1024 x 512 bf16,
// forward and gradient: 391 us; element by element 527)
bool rows_vec(const void* d, int64_t lane, int64_t row, int ev, int size) {
  return ((uintptr_t)d % (ev * size)) == 0 && lane % ev == 0 && row % ev == 0;
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

int64_t scan_saved_floats(int lanes, int T, int C, int ds) {
  return (int64_t)lanes * ((T + SCAN_TILE - 1) / SCAN_TILE) * C * ds;
}

namespace {

// the workspace in 256-byte aligned parts; at null, only their sizes are counted
struct Take {
  char* at;
  size_t used = 0;
  float* operator()(size_t floats) {
    float* p = at ? (float*)(at + used) : nullptr;
    used += round256(floats * 4);
    return p;
  }
};
Carry take_carry(Take& take, const Plan& p, size_t lanes, size_t C, size_t ds, bool in_place) {
  if (p.segs == 1) return Carry{nullptr, nullptr, false};
  return Carry{take(lanes * p.segs * C * ds), take(lanes * p.segs * C),
               in_place || p.segs > CHAIN_SEGS};
}
GradWork take_grad(Take& take, const Plan& p, size_t lanes, size_t T, size_t C, size_t ds) {
  GradWork w{};
  w.da = take(lanes * p.segs * C * ds);
  w.dd = take(lanes * p.segs * C);
  w.dbias = take(lanes * p.segs * C);
  if (p.cblocks > 1) w.bc = take(p.cblocks * lanes * T * 2 * ds);
  return w;
}

template <bool REV>
void launch_carry(const ScanArgs& a, const Plan& pl, const float* first, const Carry& cy,
                  hipStream_t s) {
  const int groups = std::min(CARRY_GROUPS, (pl.segs + 3) / 4);
  BOA_LAUNCH(scan_carry_kernel<REV>, dim3((uint32_t)a.q.lanes * ((a.C * a.ds + 63) / 64)),
             dim3(64 * groups), 0, s, a.A, first, a.C, a.ds, pl.segs, cy);
}

}  // namespace

size_t scan_work(int lanes, int T, int C, int ds, bool grad) {
  const Plan p = scan_plan(lanes, T, C, ds);
  Take take{nullptr};
  take_carry(take, p, lanes, C, ds, false);
  if (grad) take_grad(take, p, lanes, T, C, ds);
  return take.used;
}

#define BOA_SCAN_N(TE, V)              \
  if (a.ds == 16) BOA_SCAN(TE, 16, V); \
  else BOA_SCAN(TE, 32, V)
#define BOA_SCAN_ALL                          \
  if (a.bf16) {                               \
    if (vec) { BOA_SCAN_N(uint16_t, true); }  \
    else { BOA_SCAN_N(uint16_t, false); }     \
  } else {                                    \
    if (vec) { BOA_SCAN_N(float, true); }     \
    else { BOA_SCAN_N(float, false); }        \
  }

hipError_t launch_scan(const ScanArgs& a, hipStream_t s) {
  const Plan pl = scan_plan(a.q.lanes, a.q.T, a.C, a.ds);
  const int ev = a.ds == 16 ? Shape<16>::EV : Shape<32>::EV, size = a.bf16 ? 2 : 4;
  auto ok = [&](const auto& r) { return rows_vec(r.d, r.lane, r.row, ev, size); };
  const bool vec = a.C % ev == 0 && ok(a.u) && ok(a.delta) && ok(a.z) && ok(a.out);
  if (a.q.T == 1) {
    const dim3 grid((uint32_t)a.q.lanes * pl.cblocks);
#define BOA_STEP(TE, N) \
  BOA_LAUNCH((scan_step_kernel<TE, N>), grid, dim3(Shape<N>::BT), 0, s, a, pl)
    if (a.bf16) {
      if (a.ds == 16) BOA_STEP(uint16_t, 16);
      else BOA_STEP(uint16_t, 32);
    } else {
      if (a.ds == 16) BOA_STEP(float, 16);
      else BOA_STEP(float, 32);
    }
#undef BOA_STEP
    return hipGetLastError();
  }
  Take take{(char*)a.work};
  const Carry cy = take_carry(take, pl, a.q.lanes, a.C, a.ds,
                              a.state_in && a.state_out == a.state_in);
  if (pl.segs > 1) {
    const dim3 grid((uint32_t)a.q.lanes * (pl.segs - 1) * pl.cblocks);
    ScanGradArgs g{};
    g.f = a;
#define BOA_SCAN(TE, N, V) \
  BOA_LAUNCH((scan_local_kernel<TE, N, V, false>), grid, dim3(Shape<N>::BT), 0, s, g, pl, cy)
    BOA_SCAN_ALL
#undef BOA_SCAN
    if (cy.entered) launch_carry<false>(a, pl, a.state_in, cy, s);
  }
  const dim3 grid((uint32_t)a.q.lanes * pl.segs * pl.cblocks);
#define BOA_SCAN(TE, N, V) \
  BOA_LAUNCH((scan_kernel<TE, N, V>), grid, dim3(Shape<N>::BT), 0, s, a, pl, cy)
  BOA_SCAN_ALL
#undef BOA_SCAN
  return hipGetLastError();
}

hipError_t launch_scan_grad(const ScanGradArgs& g, hipStream_t s) {
  const ScanArgs& a = g.f;
  const Plan pl = scan_plan(a.q.lanes, a.q.T, a.C, a.ds);
  const int ev = a.ds == 16 ? Shape<16>::EV : Shape<32>::EV, size = a.bf16 ? 2 : 4;
  auto ok = [&](const auto& r) { return rows_vec(r.d, r.lane, r.row, ev, size); };
  const bool vec = a.C % ev == 0 && ok(a.u) && ok(a.delta) && ok(a.z) && ok(g.dout) && ok(g.du) &&
                   ok(g.ddelta) && ok(g.dz);
  const size_t rows = (size_t)a.q.lanes * a.q.T;
  Take take{(char*)a.work};
  const Carry cy = take_carry(take, pl, a.q.lanes, a.C, a.ds,
                              g.dstate_out && g.dstate_in == g.dstate_out);
  const GradWork wk = take_grad(take, pl, a.q.lanes, a.q.T, a.C, a.ds);
  if (pl.segs > 1) {
    const dim3 grid((uint32_t)a.q.lanes * (pl.segs - 1) * pl.cblocks);
#define BOA_SCAN(TE, N, V) \
  BOA_LAUNCH((scan_local_kernel<TE, N, V, true>), grid, dim3(Shape<N>::BT), 0, s, g, pl, cy)
    BOA_SCAN_ALL
#undef BOA_SCAN
    if (cy.entered) launch_carry<true>(a, pl, g.dstate_out, cy, s);
  }
  const dim3 grid((uint32_t)a.q.lanes * pl.segs * pl.cblocks);
#define BOA_SCAN(TE, N, V) \
  BOA_LAUNCH((scan_grad_kernel<TE, N, V>), grid, dim3(Shape<N>::BT), 0, s, g, pl, wk, cy)
  BOA_SCAN_ALL
#undef BOA_SCAN
#undef BOA_SCAN_ALL
#undef BOA_SCAN_N
  const int width = a.C * a.ds;
  const uint32_t gb = pl.cblocks == 1 ? 0
                      : (uint32_t)std::min<size_t>(MAX_BLOCKS, (rows * 2 * a.ds + 255) / 256);
  const dim3 gs(gb + (width + 15) / 16 + 2 * ((a.C + 15) / 16));
#define BOA_SUMS(TE)                                                                            \
  BOA_LAUNCH(scan_sums_kernel<TE>, gs, dim3(256), 0, s, wk, gb, pl.cblocks, (uint32_t)rows,     \
             a.q.T, a.ds, g.db, g.dc, a.q.lanes * pl.segs, width, a.C, g.dA, g.dD, g.dbias)
  if (a.bf16) BOA_SUMS(uint16_t);
  else BOA_SUMS(float);
#undef BOA_SUMS
  return hipGetLastError();
}

}  // namespace boa
