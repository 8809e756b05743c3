// The gated delta rule and its gradient.  For every lane and value head, with
// unit (or raw) rows q, k and a state S [d_k][d_v]:
//   S~ = e^g S        e = v - S~^T k        S = S~ + beta k e^T        o = scale S^T q
//
// Few positions are taken one after the other, the state in registers
// (delta_step_kernel).  Many are taken in chunks of 64: with sums G of the log
// decays within the chunk, D_ij = e^(G_i - G_j) and the chunk's first state S,
//   A_ij = beta_i D_ij k_i.k_j (j < i)       T = (1 + A)^-1
//   W = T diag(beta e^G) K      U = T diag(beta) V      N = U - W S      (the e, times beta)
//   P_ij = scale D_ij q_i.k_j (j <= i)       O = scale diag(e^G) Q S + P N
//   S' = e^G_64 S + sum_j e^(G_64 - G_j) k_j N_j^T
// W, U and T belong to the chunk alone (prep kernel, all chunks at once); the
// states follow one from the other, two products a chunk (chain kernel, the
// columns of S shared out); then O, all chunks at once (out kernel).
// The gradient, with dO and the gradient dS of the chunk's last state:
//   dN = P^T dO + diag(e^(G_64 - G)) K dS                   dR = T^T dN
//   dS_before = e^G_64 dS + scale (diag(e^G) Q)^T dO - W^T dN
//   dV = diag(beta) dR      dA = -dR N^T (j < i)      dP = dO N^T (j <= i)
// and dQ, dK, dbeta, dG from these, the products dO S^T, dR S^T, N dS^T and
// the elementwise rules.  Again what belongs to one chunk alone runs for all
// chunks at once, around a chain for dS.
//
// T comes from substitution within blocks of 16 and products between them, so
// keys that are equal or nearly so (the same byte again and again) do not
// spoil it.  Sums of log decays and their differences are held in 64 bits: a
// decay of -1e4 forgets all that is before it and leaves what is after it
// exact.  All else is fp32: products on the fp32 MFMA.
#include <algorithm>

#include "predictor_ops.h"

namespace boa {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
constexpr int C = 64;          // positions of a chunk
constexpr int CP = C + 4;      // pitch of a [64][64] tile in LDS
constexpr float EPS = 1e-6f;   // under the root of a row's length

// e^x for x in 64 bits, to an fp32's precision whatever its size
__device__ __forceinline__ float exp_of(double x) {
  const double y = x * 1.4426950408889634074;
  const double n = __builtin_rint(y);
  const float m = n > 1000.0 ? 1000.0f : (n < -1000.0 ? -1000.0f : (float)n);
  const float e = __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f((float)(y - n)), (int)m);
  return x != x ? (float)x : e;
}

// the log decay as it is summed: below -1e4 nothing is left of a state
__device__ __forceinline__ double log_decay(float g) {
  return g < -1e4f ? -1e4 : (double)g;
}

template <typename T>
__device__ __forceinline__ float ld1(const T* p) {
  if constexpr (sizeof(T) == 4) return *p;
  else return bf16_to_f32(*p);
}
template <typename T>
__device__ __forceinline__ void st1(T* p, float x) {
  if constexpr (sizeof(T) == 4) *p = x;
  else *p = f32_to_bf16(x);
}
// four elements from column c on of a row of d, zero past d; wide: in one piece
template <typename T>
__device__ __forceinline__ f4 ld4(const T* row, int c, int d, bool wide) {
  f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (wide) {
    if (c < d) {
      if constexpr (sizeof(T) == 4) {
        v = *reinterpret_cast<const f4*>(row + c);
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(row + c);
        v = f4{u2f(w.x << 16), u2f(w.x & 0xFFFF0000u), u2f(w.y << 16), u2f(w.y & 0xFFFF0000u)};
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < d) v[i] = ld1(row + c + i);
  }
  return v;
}

// sum over the 16 lanes of a row of lanes, in each of them
__device__ __forceinline__ float sum16(float x) {
  x = dpp_add<DPP_XOR1>(x);
  x = dpp_add<DPP_XOR2>(x);
  x = dpp_add<DPP_HALF_MIRROR>(x);
  return dpp_add<DPP_MIRROR>(x);
}

// ---- products of tiles on v_mfma_f32_16x16x4f32 ----------------------------
// Lane (i = lane % 16, g = lane / 16) holds of A row i, of B column i and of
// the result rows 4 g + r of column i.  Of every 16 of k the MFMA's step j
// takes k = 4 g + j, so an operand with k along its rows is read four at once.
// a(kk) and b(kk, n) give those four of the kk-th 16.
template <int NT, int K, typename A, typename B>
__device__ __forceinline__ void mma(f4 (&acc)[NT], A a, B b) {
#pragma unroll
  for (int kk = 0; kk < K / 16; ++kk) {
    const f4 x = a(kk);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const f4 y = b(kk, n);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], acc[n], 0, 0, 0);
    }
  }
}
// of a tile with k along its rows: rows i0 + i, k from 16 kk + 4 g
__device__ __forceinline__ f4 along(const float* t, int pitch, int i0, int kk, int lane) {
  return *reinterpret_cast<const f4*>(t + (i0 + lane % 16) * pitch + kk * 16 + lane / 16 * 4);
}
// of a tile with k across its rows: column i0 + i of rows 16 kk + 4 g ..
__device__ __forceinline__ f4 across(const float* t, int pitch, int i0, int kk, int lane) {
  const float* p = t + (kk * 16 + lane / 16 * 4) * pitch + i0 + lane % 16;
  return f4{p[0], p[pitch], p[2 * pitch], p[3 * pitch]};
}

// ---- what belongs to a (lane, value head, chunk) ---------------------------
// Everything that passes between the kernels lies in one record per chunk,
// chunks of a (lane, value head) one after the other: S [DK][DV], N [64][DV]
// (U at first), W [64][DK], T [64][64].
template <int DK, int DV>
struct Record {
  static constexpr int S = 0, N = DK * DV, W = N + C * DV, T = W + C * DK, SIZE = T + C * C;
};
// and of the gradient: dS [DK][DV], dN [64][DV]
template <int DK, int DV>
struct GradRecord {
  static constexpr int S = 0, N = DK * DV, SIZE = N + C * DV;
};

struct Place {
  int l, h, c;     // lane, value head, chunk
  int n;           // positions of the chunk within the lane's length
};
__device__ __forceinline__ Place place_of(const DeltaArgs& a, uint64_t b, int heads, int chunks) {
  Place p;
  p.c = (int)(b % chunks);
  const uint64_t lh = b / chunks;
  p.h = (int)(lh % heads);
  p.l = (int)(lh / heads);
  const int left = seq_len(a.q, p.l) - p.c * C;
  p.n = left < 0 ? 0 : (left < C ? left : C);
  return p;
}

// a tile of the chunk's rows, heads d wide at head h, into LDS; zero elsewhere
template <typename T, int D>
__device__ __forceinline__ void bring(float* t, const RowsIn& r, const Place& p, int h, int d,
                                      bool wide) {
  constexpr int PITCH = D + 4;
  for (int i = threadIdx.x; i < C * D / 4; i += blockDim.x) {
    const int row = i / (D / 4), col = i % (D / 4) * 4;
    f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (row < p.n)
      v = ld4((const T*)r.d + p.l * r.lane + (int64_t)(p.c * C + row) * r.row + (int64_t)h * d,
              col, d, wide);
    *reinterpret_cast<f4*>(t + row * PITCH + col) = v;
  }
}
// ... of floats [64][D] that lie one after the other
template <int D>
__device__ __forceinline__ void bring_dense(float* t, const float* from) {
  constexpr int PITCH = D + 4;
  for (int i = threadIdx.x; i < C * D / 4; i += blockDim.x)
    *reinterpret_cast<f4*>(t + i / (D / 4) * PITCH + i % (D / 4) * 4) =
        *reinterpret_cast<const f4*>(from + i * 4);
}

// the chunk's coefficients, by the block's first wave
struct Coef {
  double sum[C];   // G
  float beta[C];
  float since[C];  // e^G
  float left[C];   // e^(G_64 - G)
  float rk[C];     // 1 / length of k (1 where rows are taken raw)
  float rq[C];     // scale / length of q
};
__device__ __forceinline__ void decays_of(Coef& s, const DeltaArgs& a, const Place& p) {
  const int i = threadIdx.x;
  if (i >= C) return;
  double g = 0.0;
  float beta = 0.0f;
  if (i < p.n) {
    const int64_t t = p.c * C + i;
    g = log_decay(*((const float*)a.g.d + p.l * a.g.lane + t * a.g.row + p.h));
    beta = *((const float*)a.beta.d + p.l * a.beta.lane + t * a.beta.row + p.h);
  }
#pragma unroll
  for (int m = 1; m < C; m *= 2) {
    const double y = __shfl_up(g, m);
    if (i >= m) g += y;
  }
  const double all = __shfl(g, C - 1);
  s.sum[i] = g;
  s.beta[i] = beta;
  s.since[i] = exp_of(g);
  s.left[i] = exp_of(all - g);
}
// 1 / length of the tile's 64 rows, four threads a row; needs 256 threads
template <int D>
__device__ __forceinline__ void lengths_of(float* r, const float* t, bool unit, float scale) {
  constexpr int PITCH = D + 4;
  const int row = threadIdx.x / 4, part = threadIdx.x % 4;
  float s = 0.0f;
  if (unit) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const f4 v = *reinterpret_cast<const f4*>(t + row * PITCH + (i * 4 + part) * 4);
      s += v[0] * v[0] + v[1] * v[1] + v[2] * v[2] + v[3] * v[3];
    }
    s = dpp_add<DPP_XOR1>(s);
    s = dpp_add<DPP_XOR2>(s);
    s = scale / __builtin_sqrtf(s + EPS);
  } else {
    s = scale;
  }
  if (part == 0) r[row] = s;
}
__device__ __forceinline__ float between(const Coef& s, int i, int j) {
  return exp_of(s.sum[i] - s.sum[j]);
}

// ---- prep: W, U and T of every chunk ---------------------------------------
template <typename T, int DK, int DV>
__global__ __launch_bounds__(256) void delta_prep_kernel(const DeltaArgs a, float* rec, int chunks,
                                                         uint64_t blocks, bool wide) {
  using R = Record<DK, DV>;
  constexpr int D = DK > DV ? DK : DV;
  __shared__ __align__(16) float x[C * (D + 4)];
  __shared__ __align__(16) float am[C * CP], tm[C * CP];
  __shared__ Coef s;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane % 16, g4 = lane / 16 * 4;
  for (uint64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const Place p = place_of(a, b, a.HV, chunks);
    if (!p.n) continue;
    __syncthreads();
    bring<T, DK>(x, a.k, p, p.h / (a.HV / a.H), a.dk, wide);
    decays_of(s, a, p);
    __syncthreads();
    lengths_of<DK>(s.rk, x, a.unit, 1.0f);
    for (int i = threadIdx.x; i < C * C; i += 256) tm[i / C * CP + i % C] = 0.0f;
    __syncthreads();
    {
      f4 acc[4] = {};
      mma<4, DK>(acc, [&](int kk) { return along(x, DK + 4, wave * 16, kk, lane); },
                 [&](int kk, int n) { return along(x, DK + 4, n * 16, kk, lane); });
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = wave * 16 + g4 + r, j = n * 16 + i16;
          am[i * CP + j] =
              j < i ? acc[n][r] * (s.beta[i] * s.rk[i] * s.rk[j] * between(s, i, j)) : 0.0f;
        }
    }
    __syncthreads();
    // the diagonal blocks of T by substitution, a column in each of 16 lanes
    if (lane < 16) {
      float t[16];
      const float* ab = am + wave * 16 * CP + wave * 16;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float v = i == lane ? 1.0f : 0.0f;
#pragma unroll
        for (int m = 0; m < i; ++m) v -= ab[i * CP + m] * t[m];
        t[i] = v;
        tm[(wave * 16 + i) * CP + wave * 16 + lane] = v;
      }
    }
    __syncthreads();
    // blocks below the diagonal: T_21 = -T_22 (A_21 T_11), of 16, then of 32; a
    // product's result lies as the next one's right operand
    if (wave < 2) {
      const int o = wave * 32;
      f4 at[1] = {}, t21[1] = {};
      mma<1, 16>(at, [&](int kk) { return along(am + o, CP, o + 16, kk, lane); },
                 [&](int kk, int) { return across(tm + o * CP + o, CP, 0, kk, lane); });
      mma<1, 16>(t21, [&](int kk) { return along(tm + o + 16, CP, o + 16, kk, lane); },
                 [&](int, int) { return at[0]; });
#pragma unroll
      for (int r = 0; r < 4; ++r) tm[(o + 16 + g4 + r) * CP + o + i16] = -t21[0][r];
    }
    __syncthreads();
    {
      const int ri = 32 + wave / 2 * 16, cj = wave % 2 * 16;
      f4 at[2][1] = {}, t21[1] = {};
#pragma unroll
      for (int m = 0; m < 2; ++m)
        mma<1, 32>(at[m], [&](int kk) { return along(am, CP, 32 + m * 16, kk, lane); },
                   [&](int kk, int) { return across(tm, CP, cj, kk, lane); });
      mma<1, 32>(t21, [&](int kk) { return along(tm + 32, CP, ri, kk, lane); },
                 [&](int kk, int) { return at[kk][0]; });
#pragma unroll
      for (int r = 0; r < 4; ++r) tm[(ri + g4 + r) * CP + cj + i16] = -t21[0][r];
    }
    __syncthreads();
    float* out = rec + b * R::SIZE;
    if (a.saved)
      for (int i = threadIdx.x; i < C * C / 4; i += 256)
        *reinterpret_cast<f4*>(out + R::T + i * 4) =
            *reinterpret_cast<const f4*>(tm + i / (C / 4) * CP + i % (C / 4) * 4);
    {
      f4 acc[DK / 16] = {};
      mma<DK / 16, C>(
          acc,
          [&](int kk) {
            f4 v = along(tm, CP, wave * 16, kk, lane);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int m = kk * 16 + g4 + j;
              v[j] *= s.beta[m] * s.since[m] * s.rk[m];
            }
            return v;
          },
          [&](int kk, int n) { return across(x, DK + 4, n * 16, kk, lane); });
#pragma unroll
      for (int n = 0; n < DK / 16; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          out[R::W + (wave * 16 + g4 + r) * DK + n * 16 + i16] = acc[n][r];
    }
    __syncthreads();
    bring<T, DV>(x, a.v, p, p.h, a.dv, wide);
    __syncthreads();
    {
      f4 acc[DV / 16] = {};
      mma<DV / 16, C>(
          acc,
          [&](int kk) {
            f4 v = along(tm, CP, wave * 16, kk, lane);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] *= s.beta[kk * 16 + g4 + j];
            return v;
          },
          [&](int kk, int n) { return across(x, DV + 4, n * 16, kk, lane); });
#pragma unroll
      for (int n = 0; n < DV / 16; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          out[R::N + (wave * 16 + g4 + r) * DV + n * 16 + i16] = acc[n][r];
    }
  }
}

// ---- chain: the states of a (lane, value head), BV columns a block ---------
constexpr int BV = 32;
template <typename T, int DK, int DV>
__global__ __launch_bounds__(256) void delta_chain_kernel(const DeltaArgs a, float* rec, int chunks,
                                                          uint64_t blocks, bool wide) {
  using R = Record<DK, DV>;
  constexpr int SP = BV + 4, ST = DK / 64;  // row tiles of S a wave
  __shared__ __align__(16) float kt[C * (DK + 4)], sm[DK * SP], nm[C * SP];
  __shared__ Coef s;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane % 16, g4 = lane / 16 * 4;
  for (uint64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int v0 = (int)(b % (DV / BV)) * BV;
    const uint64_t lh = b / (DV / BV);
    Place p;
    p.h = (int)(lh % a.HV);
    p.l = (int)(lh / a.HV);
    const int len = seq_len(a.q, p.l);
    f4 st[ST][2];
    const int64_t state = (int64_t)lh * a.dk * a.dv;
#pragma unroll
    for (int m = 0; m < ST; ++m)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = wave * (DK / 4) + m * 16 + g4 + r, j = v0 + n * 16 + i16;
          st[m][n][r] = a.state_in && i < a.dk && j < a.dv
                            ? a.state_in[state + (int64_t)i * a.dv + j] : 0.0f;
        }
    for (p.c = 0; p.c * C < len; ++p.c) {
      p.n = min(C, len - p.c * C);
      float* at = rec + (lh * chunks + p.c) * R::SIZE;
      __syncthreads();
      bring<T, DK>(kt, a.k, p, p.h / (a.HV / a.H), a.dk, wide);
      decays_of(s, a, p);
#pragma unroll
      for (int m = 0; m < ST; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = wave * (DK / 4) + m * 16 + g4 + r, j = n * 16 + i16;
            sm[i * SP + j] = st[m][n][r];
            at[R::S + i * DV + v0 + j] = st[m][n][r];
          }
      __syncthreads();
      lengths_of<DK>(s.rk, kt, a.unit, 1.0f);
      f4 acc[2];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[n][r] = -at[R::N + (wave * 16 + g4 + r) * DV + v0 + n * 16 + i16];
      mma<2, DK>(acc,
                 [&](int kk) {
                   return *reinterpret_cast<const f4*>(at + R::W + (wave * 16 + i16) * DK +
                                                       kk * 16 + g4);
                 },
                 [&](int kk, int n) { return across(sm, SP, n * 16, kk, lane); });
      __syncthreads();
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = wave * 16 + g4 + r, j = n * 16 + i16;
          at[R::N + i * DV + v0 + j] = -acc[n][r];
          nm[i * SP + j] = -acc[n][r] * (s.left[i] * s.rk[i]);
        }
      __syncthreads();
      const float all = s.since[C - 1];
#pragma unroll
      for (int m = 0; m < ST; ++m) {
#pragma unroll
        for (int n = 0; n < 2; ++n) st[m][n] *= all;
        mma<2, C>(st[m],
                  [&](int kk) {
                    return across(kt, DK + 4, wave * (DK / 4) + m * 16, kk, lane);
                  },
                  [&](int kk, int n) { return across(nm, SP, n * 16, kk, lane); });
      }
    }
    if (a.state_out) {
#pragma unroll
      for (int m = 0; m < ST; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = wave * (DK / 4) + m * 16 + g4 + r, j = v0 + n * 16 + i16;
            if (i < a.dk && j < a.dv) a.state_out[state + (int64_t)i * a.dv + j] = st[m][n][r];
          }
    }
  }
}

// P [64][64] into pm from the tiles of q and k
template <int DK>
__device__ __forceinline__ void scores(float* pm, const float* qt, const float* kt, const Coef& s,
                                       int wave, int lane) {
  f4 acc[4] = {};
  mma<4, DK>(acc, [&](int kk) { return along(qt, DK + 4, wave * 16, kk, lane); },
             [&](int kk, int n) { return along(kt, DK + 4, n * 16, kk, lane); });
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = wave * 16 + lane / 16 * 4 + r, j = n * 16 + lane % 16;
      pm[i * CP + j] = j <= i ? acc[n][r] * (s.rq[i] * s.rk[j] * between(s, i, j)) : 0.0f;
    }
}

// ---- out: O of every chunk ---------------------------------------------------
template <typename T, int DK, int DV>
__global__ __launch_bounds__(256) void delta_out_kernel(const DeltaArgs a, const float* rec,
                                                        int chunks, uint64_t blocks, bool wide) {
  using R = Record<DK, DV>;
  constexpr int D = DK > DV ? DK : DV;
  extern __shared__ __align__(16) float lds[];
  float* qt = lds;                    // [64][DK + 4]
  float* x = qt + C * (DK + 4);       // [64][D + 4]: k, then N, then 64 rows of S at a time
  float* pm = x + C * (D + 4);        // [64][CP]
  Coef& s = *reinterpret_cast<Coef*>(pm + C * CP);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane % 16, g4 = lane / 16 * 4;
  for (uint64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const Place p = place_of(a, b, a.HV, chunks);
    if (!p.n) continue;
    const float* at = rec + b * R::SIZE;
    const int kh = p.h / (a.HV / a.H);
    __syncthreads();
    bring<T, DK>(qt, a.qr, p, kh, a.dk, wide);
    bring<T, DK>(x, a.k, p, kh, a.dk, wide);
    decays_of(s, a, p);
    __syncthreads();
    lengths_of<DK>(s.rk, x, a.unit, 1.0f);
    lengths_of<DK>(s.rq, qt, a.unit, a.scale);
    __syncthreads();
    scores<DK>(pm, qt, x, s, wave, lane);
    __syncthreads();
    f4 acc[DV / 16] = {};
#pragma unroll
    for (int part = 0; part < DK / 64; ++part) {
      bring_dense<DV>(x, at + R::S + part * 64 * DV);
      __syncthreads();
      mma<DV / 16, 64>(acc,
                       [&](int kk) { return along(qt + part * 64, DK + 4, wave * 16, kk, lane); },
                       [&](int kk, int n) { return across(x, DV + 4, n * 16, kk, lane); });
      __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < DV / 16; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = wave * 16 + g4 + r;
        acc[n][r] *= s.rq[i] * s.since[i];
      }
    bring_dense<DV>(x, at + R::N);
    __syncthreads();
    mma<DV / 16, C>(acc, [&](int kk) { return along(pm, CP, wave * 16, kk, lane); },
                    [&](int kk, int n) { return across(x, DV + 4, n * 16, kk, lane); });
#pragma unroll
    for (int n = 0; n < DV / 16; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = wave * 16 + g4 + r, j = n * 16 + i16;
        if (i < p.n && j < a.dv)
          st1((T*)a.out.d + p.l * a.out.lane + (int64_t)(p.c * C + i) * a.out.row +
                  (int64_t)p.h * a.dv + j, acc[n][r]);
      }
  }
}

// ---- the gradient's first part: P^T dO of every chunk ----------------------
template <typename T, int DK, int DV>
__global__ __launch_bounds__(256) void delta_grad_first_kernel(const DeltaGradArgs ga, float* grec,
                                                               int chunks, uint64_t blocks,
                                                               bool wide) {
  using GR = GradRecord<DK, DV>;
  constexpr int D = DK > DV ? DK : DV;
  extern __shared__ __align__(16) float lds[];
  const DeltaArgs& a = ga.f;
  float* qt = lds;
  float* x = qt + C * (DK + 4);
  float* pm = x + C * (D + 4);
  Coef& s = *reinterpret_cast<Coef*>(pm + C * CP);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane % 16, g4 = lane / 16 * 4;
  for (uint64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const Place p = place_of(a, b, a.HV, chunks);
    if (!p.n) continue;
    float* at = grec + b * GR::SIZE;
    const int kh = p.h / (a.HV / a.H);
    __syncthreads();
    bring<T, DK>(qt, a.qr, p, kh, a.dk, wide);
    bring<T, DK>(x, a.k, p, kh, a.dk, wide);
    decays_of(s, a, p);
    __syncthreads();
    lengths_of<DK>(s.rk, x, a.unit, 1.0f);
    lengths_of<DK>(s.rq, qt, a.unit, a.scale);
    __syncthreads();
    scores<DK>(pm, qt, x, s, wave, lane);
    __syncthreads();
    bring<T, DV>(x, ga.dout, p, p.h, a.dv, wide);
    __syncthreads();
    f4 acc[DV / 16] = {};
    mma<DV / 16, C>(acc, [&](int kk) { return across(pm, CP, wave * 16, kk, lane); },
                    [&](int kk, int n) { return across(x, DV + 4, n * 16, kk, lane); });
#pragma unroll
    for (int n = 0; n < DV / 16; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        at[GR::N + (wave * 16 + g4 + r) * DV + n * 16 + i16] = acc[n][r];
  }
}

// ---- the gradient's chain: dS from the last chunk to the first -------------
template <typename T, int DK, int DV>
__global__ __launch_bounds__(256) void delta_grad_chain_kernel(const DeltaGradArgs ga,
                                                               const float* rec, float* grec,
                                                               int chunks, uint64_t blocks,
                                                               bool wide) {
  using R = Record<DK, DV>;
  using GR = GradRecord<DK, DV>;
  constexpr int SP = BV + 4, ST = DK / 64;
  extern __shared__ __align__(16) float lds[];
  const DeltaArgs& a = ga.f;
  float* kt = lds;                    // [64][DK + 4]: k, then W
  float* qt = kt + C * (DK + 4);      // [64][DK + 4]
  float* sm = qt + C * (DK + 4);      // [DK][SP]: dS
  float* om = sm + DK * SP;           // [64][SP]: dO
  float* nm = om + C * SP;            // [64][SP]: dN
  Coef& s = *reinterpret_cast<Coef*>(nm + C * SP);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane % 16, g4 = lane / 16 * 4;
  for (uint64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int v0 = (int)(b % (DV / BV)) * BV;
    const uint64_t lh = b / (DV / BV);
    Place p;
    p.h = (int)(lh % a.HV);
    p.l = (int)(lh / a.HV);
    const int kh = p.h / (a.HV / a.H);
    const int len = seq_len(a.q, p.l);
    f4 st[ST][2];
    const int64_t state = (int64_t)lh * a.dk * a.dv;
#pragma unroll
    for (int m = 0; m < ST; ++m)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = wave * (DK / 4) + m * 16 + g4 + r, j = v0 + n * 16 + i16;
          st[m][n][r] = ga.dstate_out && i < a.dk && j < a.dv
                            ? ga.dstate_out[state + (int64_t)i * a.dv + j] : 0.0f;
        }
    for (p.c = (len + C - 1) / C - 1; p.c >= 0; --p.c) {
      p.n = min(C, len - p.c * C);
      const float* at = rec + (lh * chunks + p.c) * R::SIZE;
      float* gat = grec + (lh * chunks + p.c) * GR::SIZE;
      __syncthreads();
      bring<T, DK>(kt, a.k, p, kh, a.dk, wide);
      bring<T, DK>(qt, a.qr, p, kh, a.dk, wide);
      decays_of(s, a, p);
#pragma unroll
      for (int m = 0; m < ST; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = wave * (DK / 4) + m * 16 + g4 + r, j = n * 16 + i16;
            sm[i * SP + j] = st[m][n][r];
            gat[GR::S + i * DV + v0 + j] = st[m][n][r];
          }
      __syncthreads();
      lengths_of<DK>(s.rk, kt, a.unit, 1.0f);
      lengths_of<DK>(s.rq, qt, a.unit, a.scale);
      __syncthreads();
      for (int i = threadIdx.x; i < C * BV; i += 256) {
        const int row = i / BV, col = v0 + i % BV;
        float v = 0.0f;
        if (row < p.n && col < a.dv)
          v = ld1((const T*)ga.dout.d + p.l * ga.dout.lane +
                  (int64_t)(p.c * C + row) * ga.dout.row + (int64_t)p.h * a.dv + col);
        om[row * SP + i % BV] = v * (s.rq[row] * s.since[row]);
      }
      f4 acc[2] = {};
      mma<2, DK>(acc, [&](int kk) { return along(kt, DK + 4, wave * 16, kk, lane); },
                 [&](int kk, int n) { return across(sm, SP, n * 16, kk, lane); });
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = wave * 16 + g4 + r, j = n * 16 + i16;
          float* d = gat + GR::N + i * DV + v0 + j;
          const float v = *d + acc[n][r] * (s.left[i] * s.rk[i]);
          *d = v;
          nm[i * SP + j] = -v;
        }
      __syncthreads();
      bring_dense<DK>(kt, at + R::W);
      __syncthreads();
      const float all = s.since[C - 1];
#pragma unroll
      for (int m = 0; m < ST; ++m) {
        const int i0 = wave * (DK / 4) + m * 16;
#pragma unroll
        for (int n = 0; n < 2; ++n) st[m][n] *= all;
        mma<2, C>(st[m], [&](int kk) { return across(qt, DK + 4, i0, kk, lane); },
                  [&](int kk, int n) { return across(om, SP, n * 16, kk, lane); });
        mma<2, C>(st[m], [&](int kk) { return across(kt, DK + 4, i0, kk, lane); },
                  [&](int kk, int n) { return across(nm, SP, n * 16, kk, lane); });
      }
    }
    if (ga.dstate_in) {
#pragma unroll
      for (int m = 0; m < ST; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = wave * (DK / 4) + m * 16 + g4 + r, j = v0 + n * 16 + i16;
            if (i < a.dk && j < a.dv) ga.dstate_in[state + (int64_t)i * a.dv + j] = st[m][n][r];
          }
    }
  }
}

// ---- the gradient's last part: the rows' gradients of every chunk ----------
// A block takes a chunk of a head of k and all value heads that share it, so
// that their gradients of q and k are summed in registers, in one order.
template <typename T, int DK, int DV>
__global__ __launch_bounds__(256) void delta_grad_last_kernel(const DeltaGradArgs ga,
                                                              const float* rec, const float* grec,
                                                              int chunks, uint64_t blocks,
                                                              bool wide) {
  using R = Record<DK, DV>;
  using GR = GradRecord<DK, DV>;
  constexpr int NK = DK / 16, NV = DV / 16;
  extern __shared__ __align__(16) float lds[];
  const DeltaArgs& a = ga.f;
  float* kt = lds;                    // [64][DK + 4]
  float* qt = kt + C * (DK + 4);      // [64][DK + 4]
  float* dr = qt + C * (DK + 4);      // [64][DV + 4]
  float* e1 = dr + C * (DV + 4);      // [64][CP]: dP scale D
  float* e2 = e1 + C * CP;            // [64][CP]: dA beta D
  float* col = e2 + C * CP;           // [4][64]: a wave's column sums
  float* dsum = col + 4 * C;          // [64]: gradient of G
  float* tail = dsum + C;             // [4]: a wave's part of <dS, S>
  Coef& s = *reinterpret_cast<Coef*>(tail + 4);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane % 16, g4 = lane / 16 * 4;
  const int group = a.HV / a.H, r0 = wave * 16 + g4;  // this lane's rows of results: r0 ..
  for (uint64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    Place p = place_of(a, b, a.H, chunks);
    const int kh = p.h, rows = min(C, a.q.T - p.c * C);
    f4 dq[NK] = {}, dk[NK] = {};
    __syncthreads();
    if (p.n) {
      bring<T, DK>(kt, a.k, p, kh, a.dk, wide);
      bring<T, DK>(qt, a.qr, p, kh, a.dk, wide);
      __syncthreads();
      lengths_of<DK>(s.rk, kt, a.unit, 1.0f);
      lengths_of<DK>(s.rq, qt, a.unit, a.scale);
    }
    for (int vh = kh * group; vh < (kh + 1) * group; ++vh) {
      p.h = vh;
      if (!p.n) {  // rows past the length: zero
        for (int i = threadIdx.x; i < rows; i += 256) {
          const int64_t t = p.c * C + i;
          ((float*)ga.dg.d)[p.l * ga.dg.lane + t * ga.dg.row + vh] = 0.0f;
          ((float*)ga.dbeta.d)[p.l * ga.dbeta.lane + t * ga.dbeta.row + vh] = 0.0f;
        }
        for (int i = threadIdx.x; i < rows * a.dv; i += 256)
          st1((T*)ga.dv.d + p.l * ga.dv.lane + (int64_t)(p.c * C + i / a.dv) * ga.dv.row +
                  (int64_t)vh * a.dv + i % a.dv, 0.0f);
        continue;
      }
      const uint64_t at = ((uint64_t)p.l * a.HV + vh) * chunks + p.c;
      const float *S = rec + at * R::SIZE + R::S, *N = rec + at * R::SIZE + R::N,
                  *tm = rec + at * R::SIZE + R::T, *dS = grec + at * GR::SIZE + GR::S,
                  *dN = grec + at * GR::SIZE + GR::N;
      __syncthreads();
      decays_of(s, a, p);
      __syncthreads();
      float dbeta[4] = {}, dg[4] = {};
      {
        // dR = T^T dN; dV; dR . v into dbeta
        f4 acc[NV] = {};
        mma<NV, C>(acc, [&](int kk) { return across(tm, C, wave * 16, kk, lane); },
                   [&](int kk, int n) { return across(dN, DV, n * 16, kk, lane); });
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = r0 + r;
          const int64_t t = p.c * C + i;
          const T* v = (const T*)a.v.d + p.l * a.v.lane + t * a.v.row + (int64_t)vh * a.dv;
          T* o = (T*)ga.dv.d + p.l * ga.dv.lane + t * ga.dv.row + (int64_t)vh * a.dv;
          float dot = 0.0f;
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            const int j = n * 16 + i16;
            dr[i * (DV + 4) + j] = acc[n][r];
            if (j < a.dv && i < rows) {
              if (i < p.n) dot += acc[n][r] * ld1(v + j);
              st1(o + j, i < p.n ? acc[n][r] * s.beta[i] : 0.0f);
            }
          }
          dbeta[r] += sum16(dot);
        }
      }
      __syncthreads();
      // this lane's row of dO as an operand: k along the row
      const int oi = wave * 16 + i16;
      const T* drow = (const T*)ga.dout.d + p.l * ga.dout.lane +
                      (int64_t)(p.c * C + oi) * ga.dout.row + (int64_t)vh * a.dv;
      auto dout = [&](int kk) {
        return oi < p.n ? ld4(drow, kk * 16 + g4, a.dv, wide) : f4{0.0f, 0.0f, 0.0f, 0.0f};
      };
      auto drop = [&](int kk) { return along(dr, DV + 4, wave * 16, kk, lane); };
      auto dense = [&](const float* m, int pitch, int n, int kk) {
        return *reinterpret_cast<const f4*>(m + (n * 16 + i16) * pitch + kk * 16 + g4);
      };
      {
        f4 da[4] = {}, dp[4] = {}, kk_[4] = {}, qk[4] = {};
        mma<4, DV>(da, drop, [&](int kk, int n) { return dense(N, DV, n, kk); });
        mma<4, DV>(dp, dout, [&](int kk, int n) { return dense(N, DV, n, kk); });
        mma<4, DK>(kk_, [&](int kk) { return along(kt, DK + 4, wave * 16, kk, lane); },
                   [&](int kk, int n) { return along(kt, DK + 4, n * 16, kk, lane); });
        mma<4, DK>(qk, [&](int kk) { return along(qt, DK + 4, wave * 16, kk, lane); },
                   [&](int kk, int n) { return along(kt, DK + 4, n * 16, kk, lane); });
        float down[4] = {};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = r0 + r;
          float across_row = 0.0f, with_beta = 0.0f;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int j = n * 16 + i16;
            const float d = j <= i ? between(s, i, j) : 0.0f;
            const float dA = j < i ? -da[n][r] * d : 0.0f, dP = dp[n][r] * d;
            const float unit_kk = kk_[n][r] * (s.rk[i] * s.rk[j]);
            const float m = dA * s.beta[i] * unit_kk + dP * (qk[n][r] * (s.rq[i] * s.rk[j]));
            across_row += m;
            down[n] += m;
            with_beta += dA * unit_kk;
            e1[i * CP + j] = dP;
            e2[i * CP + j] = dA * s.beta[i];
          }
          dg[r] += sum16(across_row);
          dbeta[r] += sum16(with_beta);
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          float x = down[n];
          x += __shfl_xor(x, 16);
          x += __shfl_xor(x, 32);
          if (lane < 16) col[wave * C + n * 16 + i16] = x;
        }
      }
      float last[4];
      {
        f4 os[NK] = {}, rs[NK] = {}, ns[NK] = {};
        mma<NK, DV>(os, dout, [&](int kk, int n) { return dense(S, DV, n, kk); });
        mma<NK, DV>(rs, drop, [&](int kk, int n) { return dense(S, DV, n, kk); });
        mma<NK, DV>(ns, [&](int kk) { return dense(N, DV, wave, kk); },
                    [&](int kk, int n) { return dense(dS, DV, n, kk); });
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = r0 + r;
          float o = 0.0f, d = 0.0f, e = 0.0f;
#pragma unroll
          for (int n = 0; n < NK; ++n) {
            const float kv = kt[i * (DK + 4) + n * 16 + i16], qv = qt[i * (DK + 4) + n * 16 + i16];
            o += os[n][r] * qv;
            d += rs[n][r] * kv;
            e += ns[n][r] * kv;
          }
          o = sum16(o) * (s.rq[i] * s.since[i]);
          d = sum16(d) * (s.rk[i] * s.since[i]);
          last[r] = sum16(e) * (s.rk[i] * s.left[i]);
          dbeta[r] -= d;
          dg[r] += o - d * s.beta[i] - last[r];
#pragma unroll
          for (int n = 0; n < NK; ++n) {
            dq[n][r] += os[n][r] * (s.since[i] * a.scale);
            dk[n][r] += ns[n][r] * s.left[i] - rs[n][r] * (s.since[i] * s.beta[i]);
          }
        }
      }
      {
        // <dS, S>, a quarter in each wave
        float x = 0.0f;
        for (int i = threadIdx.x; i < DK * DV / 4; i += 256) {
          const f4 u = *reinterpret_cast<const f4*>(S + i * 4);
          const f4 v = *reinterpret_cast<const f4*>(dS + i * 4);
          x += u[0] * v[0] + u[1] * v[1] + u[2] * v[2] + u[3] * v[3];
        }
        x *= s.since[C - 1];
        if (i16 == 0) x += last[0] + last[1] + last[2] + last[3];
#pragma unroll
        for (int m = 1; m < 64; m *= 2) x += __shfl_xor(x, m);
        if (lane == 0) tail[wave] = x;
        if (i16 == 0)
#pragma unroll
          for (int r = 0; r < 4; ++r) dsum[r0 + r] = dg[r];
      }
      __syncthreads();
      mma<NK, C>(dq,
                 [&](int kk) {
                   f4 v = along(e1, CP, wave * 16, kk, lane);
#pragma unroll
                   for (int j = 0; j < 4; ++j) v[j] *= s.rk[kk * 16 + g4 + j] * a.scale;
                   return v;
                 },
                 [&](int kk, int n) { return across(kt, DK + 4, n * 16, kk, lane); });
      mma<NK, C>(dk,
                 [&](int kk) {
                   f4 v = across(e1, CP, wave * 16, kk, lane);
#pragma unroll
                   for (int j = 0; j < 4; ++j) v[j] *= s.rq[kk * 16 + g4 + j];
                   return v;
                 },
                 [&](int kk, int n) { return across(qt, DK + 4, n * 16, kk, lane); });
      mma<NK, C>(dk,
                 [&](int kk) {
                   f4 v = along(e2, CP, wave * 16, kk, lane) + across(e2, CP, wave * 16, kk, lane);
#pragma unroll
                   for (int j = 0; j < 4; ++j) v[j] *= s.rk[kk * 16 + g4 + j];
                   return v;
                 },
                 [&](int kk, int n) { return across(kt, DK + 4, n * 16, kk, lane); });
      if (i16 == 0)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (r0 + r < rows)
            ((float*)ga.dbeta.d)[p.l * ga.dbeta.lane + (int64_t)(p.c * C + r0 + r) * ga.dbeta.row +
                                 vh] = r0 + r < p.n ? dbeta[r] : 0.0f;
      if (wave == 0) {
        // dg: the sums of dG from each position to the chunk's last
        double x = (double)dsum[lane] - (double)col[lane] - (double)col[C + lane] -
                   (double)col[2 * C + lane] - (double)col[3 * C + lane];
        if (lane == C - 1) x += (double)tail[0] + tail[1] + tail[2] + tail[3];
#pragma unroll
        for (int m = 1; m < C; m *= 2) {
          const double y = __shfl_down(x, m);
          if (lane + m < C) x += y;
        }
        if (lane < rows)
          ((float*)ga.dg.d)[p.l * ga.dg.lane + (int64_t)(p.c * C + lane) * ga.dg.row + vh] =
              lane < p.n ? (float)x : 0.0f;
      }
    }
    // through the rows' lengths: d = r (d^ - u (u . d^)), u the unit row
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = r0 + r;
      if (i >= rows) continue;
      const int64_t t = p.c * C + i;
      T* oq = (T*)ga.dq.d + p.l * ga.dq.lane + t * ga.dq.row + (int64_t)kh * a.dk;
      T* ok = (T*)ga.dk.d + p.l * ga.dk.lane + t * ga.dk.row + (int64_t)kh * a.dk;
      float fq = 0.0f, fk = 0.0f, rq = 1.0f, rk = 1.0f;
      const bool live = i < p.n;
      if (live && a.unit) {
#pragma unroll
        for (int n = 0; n < NK; ++n) {
          fq += dq[n][r] * qt[i * (DK + 4) + n * 16 + i16];
          fk += dk[n][r] * kt[i * (DK + 4) + n * 16 + i16];
        }
        rk = s.rk[i];
        // the scale is in s.rq too
        float ss = 0.0f;
#pragma unroll
        for (int n = 0; n < NK; ++n) {
          const float x = qt[i * (DK + 4) + n * 16 + i16];
          ss += x * x;
        }
        rq = 1.0f / __builtin_sqrtf(sum16(ss) + EPS);
        fq = sum16(fq) * rq * rq;
        fk = sum16(fk) * rk * rk;
      }
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        const int j = n * 16 + i16;
        if (j >= a.dk) continue;
        float x = 0.0f, y = 0.0f;
        if (live) {
          x = rq * (dq[n][r] - qt[i * (DK + 4) + j] * fq);
          y = rk * (dk[n][r] - kt[i * (DK + 4) + j] * fk);
        }
        st1(oq + j, x);
        st1(ok + j, y);
      }
    }
  }
}

// ---- few positions, one after the other ------------------------------------
// A block per (lane, value head): 256 threads hold the state, thread (x, y)
// columns 4 x .. 4 x + 3 of rows y + RG i.  With S^T k and S^T q of the state
// before, o = scale (e^g S^T q + beta (k . q) e): one sum over the rows, and
// one barrier, a position.
template <typename T, int DK, int CX>
__global__ __launch_bounds__(256) void delta_step_kernel(const DeltaArgs a, uint64_t blocks,
                                                         bool wide, bool wide_state) {
  constexpr int RG = 256 / CX, RPT = DK / RG;
  __shared__ __align__(16) float kq[2][2][DK];
  __shared__ __align__(16) f4 part[2][4][2][CX];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, x = tid % CX, y = tid / CX;
  for (uint64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int h = (int)(b % a.HV), l = (int)(b / a.HV), kh = h / (a.HV / a.H);
    const int len = seq_len(a.q, l);
    __syncthreads();
    f4 st[RPT];
    const int64_t state = (int64_t)b * a.dk * a.dv;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int row = y + RG * i;
      st[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
      if (a.state_in && row < a.dk)
        st[i] = ld4(a.state_in + state + (int64_t)row * a.dv, 4 * x, a.dv, wide_state);
    }
    for (int t = 0; t < len; ++t) {
      const int buf = t & 1;
      // k and q: every wave sums their lengths, the first two share them out
      float kv[2] = {}, qv[2] = {};
      const T* kr = (const T*)a.k.d + l * a.k.lane + t * a.k.row + (int64_t)kh * a.dk;
      const T* qr = (const T*)a.qr.d + l * a.qr.lane + t * a.qr.row + (int64_t)kh * a.dk;
#pragma unroll
      for (int i = 0; i < DK / 64; ++i)
        if (lane + 64 * i < a.dk) {
          kv[i] = ld1(kr + lane + 64 * i);
          qv[i] = ld1(qr + lane + 64 * i);
        }
      const f4 v = ld4((const T*)a.v.d + l * a.v.lane + t * a.v.row + (int64_t)h * a.dv, 4 * x,
                       a.dv, wide);
      const float g = *((const float*)a.g.d + l * a.g.lane + t * a.g.row + h);
      const float beta = *((const float*)a.beta.d + l * a.beta.lane + t * a.beta.row + h);
      const float decay = exp_of(log_decay(g));
      float kk = kv[0] * kv[0] + kv[1] * kv[1], qq = qv[0] * qv[0] + qv[1] * qv[1],
            qk = qv[0] * kv[0] + qv[1] * kv[1];
#pragma unroll
      for (int m = 1; m < 64; m *= 2) {
        kk += __shfl_xor(kk, m);
        qq += __shfl_xor(qq, m);
        qk += __shfl_xor(qk, m);
      }
      const float rk = a.unit ? 1.0f / __builtin_sqrtf(kk + EPS) : 1.0f;
      const float rq = a.unit ? a.scale / __builtin_sqrtf(qq + EPS) : a.scale;
      if (wave < 2) {
#pragma unroll
        for (int i = 0; i < DK / 64; ++i)
          kq[buf][wave][lane + 64 * i] = wave ? qv[i] * rq : kv[i] * rk;
      }
      __syncthreads();
      f4 sk = {0.0f, 0.0f, 0.0f, 0.0f}, sq = sk;
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        sk += st[i] * kq[buf][0][y + RG * i];
        sq += st[i] * kq[buf][1][y + RG * i];
      }
#pragma unroll
      for (int m = CX; m < 64; m *= 2)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sk[j] += __shfl_xor(sk[j], m);
          sq[j] += __shfl_xor(sq[j], m);
        }
      if (lane < CX) part[buf][wave][0][x] = sk, part[buf][wave][1][x] = sq;
      __syncthreads();
      sk = (part[buf][0][0][x] + part[buf][1][0][x]) + (part[buf][2][0][x] + part[buf][3][0][x]);
      const f4 e = (v - sk * decay) * beta;
#pragma unroll
      for (int i = 0; i < RPT; ++i) st[i] = st[i] * decay + e * kq[buf][0][y + RG * i];
      if (tid < CX) {
        sq = (part[buf][0][1][x] + part[buf][1][1][x]) + (part[buf][2][1][x] + part[buf][3][1][x]);
        const f4 o = sq * decay + e * (qk * rk * rq);
        T* out = (T*)a.out.d + l * a.out.lane + t * a.out.row + (int64_t)h * a.dv + 4 * x;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (4 * x + j < a.dv) st1(out + j, o[j]);
      }
    }
    if (a.state_out) {
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const int row = y + RG * i;
        if (row >= a.dk) continue;
        float* o = a.state_out + state + (int64_t)row * a.dv + 4 * x;
        if (wide_state) {
          if (4 * x < a.dv) *reinterpret_cast<f4*>(o) = st[i];
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (4 * x + j < a.dv) o[j] = st[i][j];
        }
      }
    }
  }
}

// widths that the kernels are built for
int built(int d) { return d <= 64 ? 64 : 128; }
int chunks_of(int T) { return (T + C - 1) / C; }
int64_t record_floats(int dk, int dv) {
  const int k = built(dk), v = built(dv);
  return (int64_t)k * v + C * v + C * k + C * C;
}
int64_t grad_record_floats(int dk, int dv) {
  return (int64_t)built(dk) * built(dv) + C * built(dv);
}

// Positions taken one after the other rather than in chunks.
bool by_steps(int T) { return T <= 4; }

template <typename F>
hipError_t for_widths(int dk, int dv, F&& f) {
  using std::integral_constant;
  if (built(dk) == 64)
    return built(dv) == 64 ? f(integral_constant<int, 64>(), integral_constant<int, 64>())
                           : f(integral_constant<int, 64>(), integral_constant<int, 128>());
  return built(dv) == 64 ? f(integral_constant<int, 128>(), integral_constant<int, 64>())
                         : f(integral_constant<int, 128>(), integral_constant<int, 128>());
}

template <typename K>
hipError_t room(K kernel, size_t bytes) {
  if (bytes <= 65536) return hipSuccess;
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}
uint32_t grid(uint64_t blocks) { return (uint32_t)std::min<uint64_t>(blocks, MAX_BLOCKS); }

bool wide_rows(const RowsIn& r, int d, int size) {
  return rows_by_16(r.d, r.lane, r.row, d, size);
}

template <typename T>
hipError_t delta_of(const DeltaArgs& a, hipStream_t s) {
  const int size = sizeof(T);
  const bool wide = wide_rows(a.qr, a.dk, size) && wide_rows(a.k, a.dk, size) &&
                    wide_rows(a.v, a.dv, size);
  const uint64_t heads = (uint64_t)a.q.lanes * a.HV;
  if (by_steps(a.q.T) && !a.saved) {
    const bool wide_state = a.dv % 4 == 0 && (uintptr_t)a.state_in % 16 == 0;
    auto go = [&](auto kernel) {
      BOA_LAUNCH(kernel, grid(heads), 256, 0, s, a, heads, wide, wide_state);
      return hipGetLastError();
    };
    if (built(a.dk) == 64)
      return a.dv <= 64 ? go(delta_step_kernel<T, 64, 16>) : go(delta_step_kernel<T, 64, 32>);
    return a.dv <= 64 ? go(delta_step_kernel<T, 128, 16>) : go(delta_step_kernel<T, 128, 32>);
  }
  return for_widths(a.dk, a.dv, [&](auto dk, auto dv) {
    constexpr int DK = dk, DV = dv, D = DK > DV ? DK : DV;
    const int chunks = chunks_of(a.q.T);
    float* rec = a.saved ? a.saved : (float*)a.work;
    const uint64_t all = heads * chunks;
    BOA_LAUNCH((delta_prep_kernel<T, DK, DV>), grid(all), 256, 0, s, a, rec, chunks, all, wide);
    hipError_t e = hipGetLastError();
    if (e) return e;
    const uint64_t tiles = heads * (DV / BV);
    BOA_LAUNCH((delta_chain_kernel<T, DK, DV>), grid(tiles), 256, 0, s, a, rec, chunks, tiles,
               wide);
    if ((e = hipGetLastError())) return e;
    const size_t lds = 4 * (C * (DK + 4) + C * (D + 4) + C * CP) + sizeof(Coef);
    if ((e = room(delta_out_kernel<T, DK, DV>, lds))) return e;
    BOA_LAUNCH((delta_out_kernel<T, DK, DV>), grid(all), 256, lds, s, a, (const float*)rec, chunks,
               all, wide);
    return hipGetLastError();
  });
}

template <typename T>
hipError_t delta_grad_of(const DeltaGradArgs& ga, hipStream_t s) {
  const DeltaArgs& a = ga.f;
  const int size = sizeof(T);
  const bool wide = wide_rows(a.qr, a.dk, size) && wide_rows(a.k, a.dk, size) &&
                    wide_rows(a.v, a.dv, size) && wide_rows(ga.dout, a.dv, size);
  const uint64_t heads = (uint64_t)a.q.lanes * a.HV;
  return for_widths(a.dk, a.dv, [&](auto dk, auto dv) {
    constexpr int DK = dk, DV = dv, D = DK > DV ? DK : DV;
    const int chunks = chunks_of(a.q.T);
    const float* rec = a.saved;
    float* grec = (float*)a.work;
    const uint64_t all = heads * chunks;
    size_t lds = 4 * (C * (DK + 4) + C * (D + 4) + C * CP) + sizeof(Coef);
    hipError_t e = room(delta_grad_first_kernel<T, DK, DV>, lds);
    if (e) return e;
    BOA_LAUNCH((delta_grad_first_kernel<T, DK, DV>), grid(all), 256, lds, s, ga, grec, chunks, all,
               wide);
    if ((e = hipGetLastError())) return e;
    const uint64_t tiles = heads * (DV / BV);
    lds = 4 * (2 * C * (DK + 4) + DK * (BV + 4) + 2 * C * (BV + 4)) + sizeof(Coef);
    if ((e = room(delta_grad_chain_kernel<T, DK, DV>, lds))) return e;
    BOA_LAUNCH((delta_grad_chain_kernel<T, DK, DV>), grid(tiles), 256, lds, s, ga, rec, grec,
               chunks, tiles, wide);
    if ((e = hipGetLastError())) return e;
    lds = 4 * (2 * C * (DK + 4) + C * (DV + 4) + 2 * C * CP + 5 * C + 4) + sizeof(Coef);
    if ((e = room(delta_grad_last_kernel<T, DK, DV>, lds))) return e;
    const uint64_t last = (uint64_t)a.q.lanes * a.H * chunks;
    BOA_LAUNCH((delta_grad_last_kernel<T, DK, DV>), grid(last), 256, lds, s, ga, rec,
               (const float*)grec, chunks, last, wide);
    return hipGetLastError();
  });
}

}  // namespace

int64_t delta_saved_floats(int lanes, int T, int, int HV, int dk, int dv) {
  return (int64_t)lanes * HV * chunks_of(T) * record_floats(dk, dv);
}

int64_t delta_work_bytes(int lanes, int T, int, int HV, int dk, int dv, bool grad) {
  const int64_t n = (int64_t)lanes * HV * chunks_of(T);
  // a forward call without `saved` keeps its chunks' records here
  const int64_t forward = by_steps(T) ? 0 : n * record_floats(dk, dv);
  return 4 * (grad ? std::max(forward, n * grad_record_floats(dk, dv)) : forward);
}

hipError_t launch_delta(const DeltaArgs& a, hipStream_t s) {
  return a.bf16 ? delta_of<uint16_t>(a, s) : delta_of<float>(a, s);
}

hipError_t launch_delta_grad(const DeltaGradArgs& a, hipStream_t s) {
  return a.f.bf16 ? delta_grad_of<uint16_t>(a, s) : delta_grad_of<float>(a, s);
}

}  // namespace boa
