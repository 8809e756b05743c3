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
#include <algorithm>

#include "train_kernels.h"

namespace boa {

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int CH = 64;  // channels of a block

// log(1 + e^x): e = e^-|x| in (0, 1], log(1 + e) = 2 atanh(s), s = e / (2 + e)
// <= 1/3, by its odd series to s^15 (the next term is under 2^-27 of the sum)
__device__ __forceinline__ float softplus_full(float x) {
  const float e = __builtin_amdgcn_exp2f(-__builtin_fabsf(x) * LOG2E);
  const float s = e * __builtin_amdgcn_rcpf(2.0f + e), s2 = s * s;
  float p = 0.0666666666666666667f;
  p = __builtin_fmaf(p, s2, 0.0769230769230769231f);
  p = __builtin_fmaf(p, s2, 0.0909090909090909091f);
  p = __builtin_fmaf(p, s2, 0.111111111111111111f);
  p = __builtin_fmaf(p, s2, 0.142857142857142857f);
  p = __builtin_fmaf(p, s2, 0.2f);
  p = __builtin_fmaf(p, s2, 0.333333333333333333f);
  p = __builtin_fmaf(p * s2, s, s);
  return __builtin_fmaxf(x, 0.0f) + 2.0f * p;  // a NaN stays one in p
}
__device__ __forceinline__ float sigmoid_hw(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-x * LOG2E));
}

// EV neighbouring elements of a row, as 32-bit words: EV fp32, or EV / 2 pairs of bf16
template <typename TE, int EV>
struct Raw {
  uint32_t w[EV * sizeof(TE) / 4];
};
template <typename TE, int EV, bool VEC>
__device__ __forceinline__ Raw<TE, EV> ld_raw(const void* base, int64_t off, int c, int C, bool ok) {
  Raw<TE, EV> r;
  constexpr int W = EV * sizeof(TE) / 4;
#pragma unroll
  for (int i = 0; i < W; ++i) r.w[i] = 0;
  const TE* p = (const TE*)base + off + c;
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
template <typename TE, int EV, bool VEC>
__device__ __forceinline__ void st_row(void* base, int64_t off, int c, int C, bool ok,
                                       const float (&v)[EV]) {
  TE* p = (TE*)base + off + c;
  if constexpr (VEC) {
    if (ok && c < C) {
      constexpr int W = EV * sizeof(TE) / 4;
      uint32_t w[W];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if constexpr (sizeof(TE) == 4) w[i] = f2u(v[i]);
        else w[i] = (uint32_t)f32_to_bf16(v[2 * i]) | ((uint32_t)f32_to_bf16(v[2 * i + 1]) << 16);
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

// sum over the TPC lanes of a channel, in all of them
template <int TPC>
__device__ __forceinline__ float sum_states(float x) {
  x = dpp_add<DPP_XOR1>(x);
  x = dpp_add<DPP_XOR2>(x);
  if constexpr (TPC == 8) x = dpp_add<DPP_HALF_MIRROR>(x);
  return x;
}

// How the blocks divide the work: lane, channel block (and later segment)
struct Plan {
  int tiles, cblocks;
};
Plan scan_plan(int T, int C) {
  return Plan{(T + SCAN_TILE - 1) / SCAN_TILE, (C + CH - 1) / CH};
}

// ---------------------------------------------------------------- forward
template <typename TE, int N, bool VEC>
__global__ __launch_bounds__((Shape<N>::BT)) void scan_kernel(const ScanArgs a, Plan pl) {
  using S = Shape<N>;
  constexpr int TPC = S::TPC, BT = S::BT, EV = S::EV, YS = CH + 16;
  __shared__ __align__(16) float s_delta[SCAN_TILE][CH], s_du[SCAN_TILE][CH];
  __shared__ __align__(16) float s_b[SCAN_TILE][N], s_c[SCAN_TILE][N];
  __shared__ __align__(16) float s_y[SCAN_TILE][YS];  // stride: the lanes of a channel on other banks
  const int tid = threadIdx.x, cb = blockIdx.x % pl.cblocks, l = blockIdx.x / pl.cblocks;
  const int len = seq_len(a.q, l), q = tid % TPC, ch = tid / TPC, c = cb * CH + ch;
  // the row elements that this thread owns: position ot of the tile, channels oc ..
  const int ot = tid / (CH / EV), oc = (tid % (CH / EV)) * EV, gc = cb * CH + oc;
  float h[4], A2[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    A2[i] = c < a.C ? a.A[(size_t)c * N + 4 * q + i] * LOG2E : 0.0f;
    h[i] = c < a.C && a.state_in ? a.state_in[((size_t)l * a.C + c) * N + 4 * q + i] : 0.0f;
  }
  float bias[EV], D[EV];
#pragma unroll
  for (int j = 0; j < EV; ++j) {
    bias[j] = gc + j < a.C ? a.bias[gc + j] : 0.0f;
    D[j] = gc + j < a.C ? a.D[gc + j] : 0.0f;
  }
  constexpr int NBC = SCAN_TILE * N / BT;  // elements of B (and of C) a thread stages
  Raw<TE, EV> ru, rx, rz;
  float rb[NBC], rc[NBC];
  auto fetch = [&](int tile) {
    const int t = tile * SCAN_TILE + ot;
    const bool ok = t < len;
    ru = ld_raw<TE, EV, VEC>(a.u.d, l * a.u.lane + t * a.u.row, gc, a.C, ok);
    rx = ld_raw<TE, EV, VEC>(a.delta.d, l * a.delta.lane + t * a.delta.row, gc, a.C, ok);
    rz = ld_raw<TE, EV, VEC>(a.z.d, l * a.z.lane + t * a.z.row, gc, a.C, ok);
#pragma unroll
    for (int i = 0; i < NBC; ++i) {
      const int e = tid + i * BT, bt = tile * SCAN_TILE + e / N, n = e % N;
      rb[i] = bt < len ? ldv((const TE*)a.b.d + l * a.b.lane + bt * a.b.row + n) : 0.0f;
      rc[i] = bt < len ? ldv((const TE*)a.c.d + l * a.c.lane + bt * a.c.row + n) : 0.0f;
    }
  };
  const int tiles = (len + SCAN_TILE - 1) / SCAN_TILE;
  if (tiles > 0) fetch(0);
  for (int tile = 0; tile < tiles; ++tile) {
    const int t = tile * SCAN_TILE + ot;
    const bool ok = t < len;
    float u[EV], gate[EV];
#pragma unroll
    for (int j = 0; j < EV; ++j) {
      u[j] = raw_at(ru, j);
      const float z = raw_at(rz, j);
      gate[j] = z * sigmoid_hw(z);
      // past the lane's end delta = 0: the state passes unchanged
      const float delta = ok ? softplus_full(raw_at(rx, j) + bias[j]) : 0.0f;
      s_delta[ot][oc + j] = delta;
      s_du[ot][oc + j] = delta * u[j];
    }
#pragma unroll
    for (int i = 0; i < NBC; ++i) {
      const int e = tid + i * BT;
      (&s_b[0][0])[e] = rb[i];
      (&s_c[0][0])[e] = rc[i];
    }
    __syncthreads();
    if (tile + 1 < tiles) fetch(tile + 1);
    if (a.saved && c < a.C) {
      float* p = a.saved + (((size_t)l * pl.tiles + tile) * a.C + c) * N + 4 * q;
      *reinterpret_cast<float4*>(p) = make_float4(h[0], h[1], h[2], h[3]);
    }
    float y[SCAN_TILE / TPC];
#pragma unroll
    for (int k = 0; k < SCAN_TILE; ++k) {
      const float delta = s_delta[k][ch], du = s_du[k][ch];
      const float4 B = *reinterpret_cast<const float4*>(&s_b[k][4 * q]);
      const float4 C = *reinterpret_cast<const float4*>(&s_c[k][4 * q]);
      const float bv[4] = {B.x, B.y, B.z, B.w}, cv[4] = {C.x, C.y, C.z, C.w};
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
#pragma unroll
    for (int k = 0; k < SCAN_TILE / TPC; ++k) s_y[k * TPC + q][ch] = y[k];
    __syncthreads();
    float o[EV];
#pragma unroll
    for (int j = 0; j < EV; ++j) o[j] = __builtin_fmaf(D[j], u[j], s_y[ot][oc + j]) * gate[j];
    st_row<TE, EV, VEC>(a.out.d, l * a.out.lane + t * a.out.row, gc, a.C, ok, o);
  }
  if (a.state_out && c < a.C)
    *reinterpret_cast<float4*>(a.state_out + ((size_t)l * a.C + c) * N + 4 * q) =
        make_float4(h[0], h[1], h[2], h[3]);
}

// --------------------------------------------------------------- backward
// Partial sums of a block: dA [lane][C][N], dD and dbias [lane][C], and with
// more than one channel block dB | dC [cblock][row][2 N]
struct GradWork {
  float *bc, *da, *dd, *dbias;
};

template <typename TE, int N, bool VEC>
__global__ __launch_bounds__((Shape<N>::BT)) void scan_grad_kernel(const ScanGradArgs g, Plan pl,
                                                                   GradWork wk) {
  using S = Shape<N>;
  constexpr int TPC = S::TPC, BT = S::BT, EV = S::EV, YS = CH + 16;
  __shared__ __align__(16) float s_delta[SCAN_TILE][CH], s_u[SCAN_TILE][CH], s_dy[SCAN_TILE][CH];
  __shared__ __align__(16) float s_b[SCAN_TILE][N], s_c[SCAN_TILE][N];
  __shared__ __align__(16) float s_y[SCAN_TILE][YS], s_i[SCAN_TILE][YS], s_m[SCAN_TILE][YS];
  __shared__ __align__(16) float s_bc[S::WAVES][SCAN_TILE][2 * N];
  const ScanArgs& a = g.f;
  const int tid = threadIdx.x, cb = blockIdx.x % pl.cblocks, l = blockIdx.x / pl.cblocks;
  const int len = seq_len(a.q, l), q = tid % TPC, ch = tid / TPC, c = cb * CH + ch;
  const int ot = tid / (CH / EV), oc = (tid % (CH / EV)) * EV, gc = cb * CH + oc;
  const int w = tid >> 6, ln = tid & 63;
  float A[4], G[4], dA[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    A[i] = c < a.C ? a.A[(size_t)c * N + 4 * q + i] : 0.0f;
    G[i] = c < a.C && g.dstate_out ? g.dstate_out[((size_t)l * a.C + c) * N + 4 * q + i] : 0.0f;
    dA[i] = 0.0f;
  }
  float bias[EV], D[EV], dD[EV], dbias[EV];
#pragma unroll
  for (int j = 0; j < EV; ++j) {
    bias[j] = gc + j < a.C ? a.bias[gc + j] : 0.0f;
    D[j] = gc + j < a.C ? a.D[gc + j] : 0.0f;
    dD[j] = dbias[j] = 0.0f;
  }
  constexpr int NBC = SCAN_TILE * N / BT;
  Raw<TE, EV> ru, rx, rz, ro;
  float rb[NBC], rc[NBC];
  float4 rh;
  auto fetch = [&](int tile) {
    const int t = tile * SCAN_TILE + ot;
    const bool ok = t < len;
    ru = ld_raw<TE, EV, VEC>(a.u.d, l * a.u.lane + t * a.u.row, gc, a.C, ok);
    rx = ld_raw<TE, EV, VEC>(a.delta.d, l * a.delta.lane + t * a.delta.row, gc, a.C, ok);
    rz = ld_raw<TE, EV, VEC>(a.z.d, l * a.z.lane + t * a.z.row, gc, a.C, ok);
    ro = ld_raw<TE, EV, VEC>(g.dout.d, l * g.dout.lane + t * g.dout.row, gc, a.C, ok);
#pragma unroll
    for (int i = 0; i < NBC; ++i) {
      const int e = tid + i * BT, bt = tile * SCAN_TILE + e / N, n = e % N;
      rb[i] = bt < len ? ldv((const TE*)a.b.d + l * a.b.lane + bt * a.b.row + n) : 0.0f;
      rc[i] = bt < len ? ldv((const TE*)a.c.d + l * a.c.lane + bt * a.c.row + n) : 0.0f;
    }
    rh = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (c < a.C)
      rh = *reinterpret_cast<const float4*>(
          a.saved + (((size_t)l * pl.tiles + tile) * a.C + c) * N + 4 * q);
  };
  // dB and dC of a tile: one value of one position a thread
  auto store_bc = [&](int tile, bool zero) {
    for (int e = tid; e < SCAN_TILE * 2 * N; e += BT) {
      const int k = e / (2 * N), n = e % (2 * N), t = tile * SCAN_TILE + k;
      if (t >= a.q.T) continue;
      float v = 0.0f;
      if (!zero)
#pragma unroll
        for (int i = 0; i < S::WAVES; ++i) v += s_bc[i][k][n];
      if (pl.cblocks > 1)
        wk.bc[(((size_t)cb * a.q.lanes + l) * a.q.T + t) * (2 * N) + n] = v;
      else if (n < N)
        stv((TE*)g.db.d + l * g.db.lane + t * g.db.row + n, v);
      else
        stv((TE*)g.dc.d + l * g.dc.lane + t * g.dc.row + n - N, v);
    }
  };
  const int tiles = (len + SCAN_TILE - 1) / SCAN_TILE;
  // positions past the lane's end take no part: their gradients are zero
  for (int tile = pl.tiles - 1; tile >= tiles; --tile) {
    const int t = tile * SCAN_TILE + ot;
    const float zero[EV] = {};
    const bool ok = t < a.q.T;
    st_row<TE, EV, VEC>(g.du.d, l * g.du.lane + t * g.du.row, gc, a.C, ok, zero);
    st_row<TE, EV, VEC>(g.ddelta.d, l * g.ddelta.lane + t * g.ddelta.row, gc, a.C, ok, zero);
    st_row<TE, EV, VEC>(g.dz.d, l * g.dz.lane + t * g.dz.row, gc, a.C, ok, zero);
    store_bc(tile, true);
  }
  if (tiles > 0) fetch(tiles - 1);
  for (int tile = tiles - 1; tile >= 0; --tile) {
    const int t = tile * SCAN_TILE + ot;
    const bool ok = t < len;
    float u[EV], z[EV], sig[EV], dout[EV], dy[EV], delta[EV], xsig[EV];
#pragma unroll
    for (int j = 0; j < EV; ++j) {
      u[j] = raw_at(ru, j);
      z[j] = raw_at(rz, j);
      dout[j] = raw_at(ro, j);
      sig[j] = sigmoid_hw(z[j]);
      dy[j] = dout[j] * (z[j] * sig[j]);
      const float x = raw_at(rx, j) + bias[j];
      delta[j] = ok ? softplus_full(x) : 0.0f;
      xsig[j] = ok ? sigmoid_hw(x) : 0.0f;
      s_delta[ot][oc + j] = delta[j];
      s_u[ot][oc + j] = u[j];
      s_dy[ot][oc + j] = dy[j];
    }
#pragma unroll
    for (int i = 0; i < NBC; ++i) {
      const int e = tid + i * BT;
      (&s_b[0][0])[e] = rb[i];
      (&s_c[0][0])[e] = rc[i];
    }
    const float h0[4] = {rh.x, rh.y, rh.z, rh.w};
    __syncthreads();
    if (tile > 0) fetch(tile - 1);
    // the tile's states and decays again
    float hs[SCAN_TILE][4], es[SCAN_TILE][4];
#pragma unroll
    for (int k = 0; k < SCAN_TILE; ++k) {
      const float dl = s_delta[k][ch], du = dl * s_u[k][ch];
      const float4 B = *reinterpret_cast<const float4*>(&s_b[k][4 * q]);
      const float bv[4] = {B.x, B.y, B.z, B.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        es[k][i] = __builtin_amdgcn_exp2f(dl * (A[i] * LOG2E));
        hs[k][i] = __builtin_fmaf(es[k][i], k ? hs[k > 0 ? k - 1 : 0][i] : h0[i], du * bv[i]);
      }
    }
    float ys[SCAN_TILE / TPC], is[SCAN_TILE / TPC], ms[SCAN_TILE / TPC];
#pragma unroll
    for (int k = SCAN_TILE - 1; k >= 0; --k) {
      const float dl = s_delta[k][ch], du = dl * s_u[k][ch], dyk = s_dy[k][ch];
      const float4 B = *reinterpret_cast<const float4*>(&s_b[k][4 * q]);
      const float4 C = *reinterpret_cast<const float4*>(&s_c[k][4 * q]);
      const float bv[4] = {B.x, B.y, B.z, B.w}, cv[4] = {C.x, C.y, C.z, C.w};
      float y = 0.0f, I = 0.0f, M = 0.0f, db[4], dc[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float dh = __builtin_fmaf(cv[i], dyk, G[i]);
        y = __builtin_fmaf(cv[i], hs[k][i], y);
        I = __builtin_fmaf(dh, bv[i], I);
        dc[i] = hs[k][i] * dyk;
        db[i] = dh * du;
        G[i] = es[k][i] * dh;
        const float m = G[i] * (k ? hs[k > 0 ? k - 1 : 0][i] : h0[i]);
        M = __builtin_fmaf(m, A[i], M);
        dA[i] = __builtin_fmaf(m, dl, dA[i]);
      }
      y = sum_states<TPC>(y);
      I = sum_states<TPC>(I);
      M = sum_states<TPC>(M);
      const bool keep = k % TPC == TPC - 1 || q == k % TPC;
      ys[k / TPC] = keep ? y : ys[k / TPC];
      is[k / TPC] = keep ? I : is[k / TPC];
      ms[k / TPC] = keep ? M : ms[k / TPC];
      // dB, dC over the wave's channels: the halves of the wave take dB and dC,
      // the odd rows of 16 lanes states 2 and 3, lanes with bit 3 set 1 and 3
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = fold32(db[i], dc[i]);
      const float x0 = fold16(v[0], v[2]), x1 = fold16(v[1], v[3]);
      const bool odd = ln & 8;
      float r = (odd ? x1 : x0) + dpp_move<DPP_ROR8>(odd ? x0 : x1);
      if constexpr (TPC == 4) r = dpp_add<DPP_ROR4>(r);
      s_bc[w][k][(ln >> 5) * N + 4 * q + ((ln >> 4) & 1) * 2 + ((ln >> 3) & 1)] = r;
    }
#pragma unroll
    for (int k = 0; k < SCAN_TILE / TPC; ++k) {
      s_y[k * TPC + q][ch] = ys[k];
      s_i[k * TPC + q][ch] = is[k];
      s_m[k * TPC + q][ch] = ms[k];
    }
    __syncthreads();
    float o_u[EV], o_x[EV], o_z[EV];
#pragma unroll
    for (int j = 0; j < EV; ++j) {
      const float I = s_i[ot][oc + j], y = __builtin_fmaf(D[j], u[j], s_y[ot][oc + j]);
      o_u[j] = __builtin_fmaf(D[j], dy[j], delta[j] * I);
      o_x[j] = __builtin_fmaf(u[j], I, s_m[ot][oc + j]) * xsig[j];
      o_z[j] = dout[j] * y * (sig[j] * __builtin_fmaf(z[j], 1.0f - sig[j], 1.0f));
      dD[j] = __builtin_fmaf(dy[j], u[j], dD[j]);
      dbias[j] += o_x[j];
    }
    const bool in = t < a.q.T;
    st_row<TE, EV, VEC>(g.du.d, l * g.du.lane + t * g.du.row, gc, a.C, in, o_u);
    st_row<TE, EV, VEC>(g.ddelta.d, l * g.ddelta.lane + t * g.ddelta.row, gc, a.C, in, o_x);
    st_row<TE, EV, VEC>(g.dz.d, l * g.dz.lane + t * g.dz.row, gc, a.C, in, o_z);
    store_bc(tile, false);
  }
  if (c < a.C) {
    const size_t at = ((size_t)l * a.C + c) * N + 4 * q;
    *reinterpret_cast<float4*>(wk.da + at) = make_float4(dA[0], dA[1], dA[2], dA[3]);
    if (g.dstate_in)
      *reinterpret_cast<float4*>(g.dstate_in + at) = make_float4(G[0], G[1], G[2], G[3]);
  }
  // the owners' sums over the tile's positions
#pragma unroll
  for (int j = 0; j < EV; ++j) {
    s_u[ot][oc + j] = dD[j];
    s_dy[ot][oc + j] = dbias[j];
  }
  __syncthreads();
  if (tid < 2 * CH) {
    const int cc = tid % CH;
    float s = 0.0f;
    for (int k = 0; k < SCAN_TILE; ++k) s += tid < CH ? s_u[k][cc] : s_dy[k][cc];
    if (cb * CH + cc < a.C)
      (tid < CH ? wk.dd : wk.dbias)[(size_t)l * a.C + cb * CH + cc] = s;
  }
}

// dB and dC over the channel blocks
template <typename TE>
__global__ __launch_bounds__(256) void scan_bc_sum_kernel(const float* __restrict__ part,
                                                          int cblocks, uint32_t rows, int T, int N,
                                                          RowsOut db, RowsOut dc) {
  const uint64_t n = (uint64_t)rows * 2 * N, step = (uint64_t)gridDim.x * 256;
  for (uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += step) {
    float s = 0.0f;
#pragma unroll 4
    for (int k = 0; k < cblocks; ++k) s += part[k * n + e];
    const uint32_t r = (uint32_t)(e / (2 * N)), i = (uint32_t)(e - (uint64_t)r * 2 * N);
    const uint32_t l = r / (uint32_t)T, t = r - l * T;
    if (i < (uint32_t)N) stv((TE*)db.d + l * db.lane + t * db.row + i, s);
    else stv((TE*)dc.d + l * dc.lane + t * dc.row + i - N, s);
  }
}

// sums over n partials of `width` values: 64 columns a block, 16 groups of
// rows, the groups added in order
__global__ __launch_bounds__(1024) void scan_part_sum_kernel(const float* __restrict__ part, int n,
                                                             int width, float* __restrict__ out) {
  __shared__ float sm[16][64];
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), g = threadIdx.x >> 6;
  float s = 0.0f;
  if (col < width)
#pragma unroll 8
    for (int k = g; k < n; k += 16) s += part[(size_t)k * width + col];
  sm[g][threadIdx.x & 63] = s;
  __syncthreads();
  if (g == 0 && col < width) {
    for (int k = 1; k < 16; ++k) s += sm[k][threadIdx.x];
    out[col] = s;
  }
}

bool rows_vec(const void* d, int64_t lane, int64_t row, int ev, int size) {
  return ((uintptr_t)d % (ev * size)) == 0 && lane % ev == 0 && row % ev == 0;
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

int64_t scan_saved_floats(int lanes, int T, int C, int ds) {
  return (int64_t)lanes * ((T + SCAN_TILE - 1) / SCAN_TILE) * C * ds;
}

size_t scan_work(int lanes, int T, int C, int ds, bool grad) {
  if (!grad) return 0;
  const Plan p = scan_plan(T, C);
  const size_t L = lanes;
  size_t n = round256(L * C * ds * 4) + 2 * round256(L * C * 4);
  if (p.cblocks > 1) n += round256((size_t)p.cblocks * L * T * 2 * ds * 4);
  return n;
}

hipError_t launch_scan(const ScanArgs& a, hipStream_t s) {
  const Plan pl = scan_plan(a.q.T, a.C);
  const int ev = a.ds == 16 ? Shape<16>::EV : Shape<32>::EV, size = a.bf16 ? 2 : 4;
  auto ok = [&](const auto& r) { return rows_vec(r.d, r.lane, r.row, ev, size); };
  const bool vec = a.C % ev == 0 && ok(a.u) && ok(a.delta) && ok(a.z) && ok(a.out);
  const dim3 grid((uint32_t)a.q.lanes * pl.cblocks);
#define BOA_SCAN(TE, N, V) \
  BOA_LAUNCH((scan_kernel<TE, N, V>), grid, dim3(Shape<N>::BT), 0, s, a, pl)
#define BOA_SCAN_N(TE, V)             \
  if (a.ds == 16) BOA_SCAN(TE, 16, V); \
  else BOA_SCAN(TE, 32, V)
  if (a.bf16) {
    if (vec) { BOA_SCAN_N(uint16_t, true); }
    else { BOA_SCAN_N(uint16_t, false); }
  } else {
    if (vec) { BOA_SCAN_N(float, true); }
    else { BOA_SCAN_N(float, false); }
  }
#undef BOA_SCAN
  return hipGetLastError();
}

hipError_t launch_scan_grad(const ScanGradArgs& g, hipStream_t s) {
  const ScanArgs& a = g.f;
  const Plan pl = scan_plan(a.q.T, a.C);
  const int ev = a.ds == 16 ? Shape<16>::EV : Shape<32>::EV, size = a.bf16 ? 2 : 4;
  auto ok = [&](const auto& r) { return rows_vec(r.d, r.lane, r.row, ev, size); };
  const bool vec = a.C % ev == 0 && ok(a.u) && ok(a.delta) && ok(a.z) && ok(g.dout) && ok(g.du) &&
                   ok(g.ddelta) && ok(g.dz);
  const size_t L = a.q.lanes, rows = L * a.q.T;
  char* at = (char*)a.work;
  auto take = [&](size_t floats) {
    float* p = (float*)at;
    at += round256(floats * 4);
    return p;
  };
  GradWork wk{};
  wk.da = take(L * a.C * a.ds);
  wk.dd = take(L * a.C);
  wk.dbias = take(L * a.C);
  if (pl.cblocks > 1) wk.bc = take((size_t)pl.cblocks * rows * 2 * a.ds);
  const dim3 grid((uint32_t)a.q.lanes * pl.cblocks);
#define BOA_SCAN(TE, N, V) \
  BOA_LAUNCH((scan_grad_kernel<TE, N, V>), grid, dim3(Shape<N>::BT), 0, s, g, pl, wk)
  if (a.bf16) {
    if (vec) { BOA_SCAN_N(uint16_t, true); }
    else { BOA_SCAN_N(uint16_t, false); }
  } else {
    if (vec) { BOA_SCAN_N(float, true); }
    else { BOA_SCAN_N(float, false); }
  }
#undef BOA_SCAN
#undef BOA_SCAN_N
  if (pl.cblocks > 1) {
    const dim3 gb((uint32_t)std::min<size_t>(MAX_BLOCKS, (rows * 2 * a.ds + 255) / 256));
    if (a.bf16)
      BOA_LAUNCH(scan_bc_sum_kernel<uint16_t>, gb, dim3(256), 0, s, wk.bc, pl.cblocks,
                 (uint32_t)rows, a.q.T, a.ds, g.db, g.dc);
    else
      BOA_LAUNCH(scan_bc_sum_kernel<float>, gb, dim3(256), 0, s, wk.bc, pl.cblocks, (uint32_t)rows,
                 a.q.T, a.ds, g.db, g.dc);
  }
  auto sum = [&](const float* p, int width, float* out) {
    BOA_LAUNCH(scan_part_sum_kernel, dim3((width + 63) / 64), dim3(1024), 0, s, p, (int)L, width,
               out);
  };
  sum(wk.da, a.C * a.ds, g.dA);
  sum(wk.dd, a.C, g.dD);
  sum(wk.dbias, a.C, g.dbias);
  return hipGetLastError();
}

}  // namespace boa
