// The gated delta rule and its gradient.  For every lane and value head, with
// unit (or raw) rows q, k and a state S [d_k][d_v]:
//   S~ = e^g S        e = v - S~^T k        S = S~ + beta k e^T        o = scale S^T q
//
// Few positions are taken one after the other, the state in registers
// (delta_step_kernel).  Many are taken in chunks of 64: with sums G of the log
// decays within the chunk, D_ij = e^(G_i - G_j) and the chunk's first state S,
//   A_ij = beta_i D_ij k_i.k_j (j < i)       T = (1 + A)^-1
//   P_ij = scale D_ij q_i.k_j (j <= i)
//   R = diag(beta) (V - diag(e^G) K S)       N = T R      (the e, times beta)
//   O = scale diag(e^G) Q S + P N            S' = e^G_64 S + sum_j e^(G_64 - G_j) k_j N_j^T
// T and P belong to the chunk alone (prep kernel, all chunks at once).  The rest
// follows the states from chunk to chunk (chain kernel), but no column of S, N
// and O needs another: a wave takes 16 columns and keeps them in registers from
// product to product.
// The gradient, with dO and the gradient dS of the chunk's last state:
//   dN = P^T dO + diag(e^(G_64 - G)) K dS                   dR = T^T dN
//   dS_before = e^G_64 dS + scale Q^T diag(e^G) dO - K^T diag(beta e^G) dR
// is a chain of the same kind, backwards, and
//   dV = diag(beta) dR      dA = -dR N^T (j < i)      dP = dO N^T (j <= i)
// and dQ, dK, dbeta, dG, from these, the products dO S^T, dR S^T, N dS^T and the
// elementwise rules, again belong to one chunk (last kernel).
//
// T comes from substitution within blocks of 16 and products between them, so
// keys that are equal or nearly so (the same byte again and again) do not
// spoil it.  Sums of log decays and their differences are held in 64 bits: a
// decay of -1e4 forgets all that is before it and leaves what is after it
// exact.  All else has fp32's precision.  For fp32 rows the products are on the
// fp32 MFMA; for bf16 rows on the bf16 MFMA, sixteen times as fast, where an
// fp32 operand is the sum of three bf16 ones (24 bits) and products of parts
// below 2^-24 are left out: three products against rows, which are exact, six
// between fp32 operands.
#include <algorithm>

#include "predictor_ops.h"

namespace boa {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
constexpr int C = 64;          // positions of a chunk
constexpr int CP = C + 4;      // pitch of a [64][64] tile of floats in LDS
constexpr float EPS = 1e-6f;   // under the root of a row's length
constexpr f4 ZERO = {0.0f, 0.0f, 0.0f, 0.0f};

// A sum of log decays in 64 bits as a power of two, a whole one and a fraction:
// e^(a - b) then has an fp32's precision however large a and b are.
struct Power {
  int whole;
  float part;
};
__device__ __forceinline__ Power power_of(double x) {
  const double y = x * 1.4426950408889634074;
  const double n = __builtin_fmin(__builtin_fmax(__builtin_rint(y), -1e9), 1e9);
  return Power{(int)n, (float)(y - n)};
}
__device__ __forceinline__ float raised(int whole, float part) {
  return __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(part), min(max(whole, -1000), 1000));
}
__device__ __forceinline__ float exp_of(double x) {
  const Power p = power_of(x);
  return raised(p.whole, p.part);
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
// Four elements of a row as they lie in memory, from column c on of d; W: in one
// piece (d and the addresses are multiples of 16 bytes).  No branch and no use of
// what is loaded (either would wait for it): what lies past d is the row's first
// or last elements, until `cut` clears it.
template <typename T>
struct Raw {
  using V = std::conditional_t<sizeof(T) == 4, f4, u2>;
  V v;
  // from the element `row` on of what `from` gives by element
  template <bool W, typename F>
  __device__ __forceinline__ void load(const F& from, uint32_t row, int c, int d) {
    if constexpr (W) {
      v = *reinterpret_cast<const V*>(from.at(row + (c < d ? c : 0)));
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *from.at(row + min(c + i, d - 1));
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        v[i] = *from.at(row + min(c + 2 * i, d - 1)) |
               (uint32_t)*from.at(row + min(c + 2 * i + 1, d - 1)) << 16;
    }
  }
  // zero from element n on
  template <bool W>
  __device__ __forceinline__ void cut(int n) {
    if constexpr (W || sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < (int)(sizeof(V) / 4); ++i)
        if (W ? n <= 0 : i >= n) v[i] = 0;
    } else {
      v[0] = n <= 0 ? 0 : (n == 1 ? v[0] & 0xFFFFu : v[0]);
      v[1] = n <= 2 ? 0 : (n == 3 ? v[1] & 0xFFFFu : v[1]);
    }
  }
  // as the first `left` elements (of four) from `element` on
  template <bool W, typename F>
  __device__ __forceinline__ void store(const F& to, uint32_t element, int left) const {
    if constexpr (W) {
      if (left > 0) *reinterpret_cast<V*>(to.at(element)) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < left) {
          if constexpr (sizeof(T) == 4) *to.at(element + i) = v[i];
          else *to.at(element + i) = (uint16_t)(v[i / 2] >> (16 * (i % 2)));
        }
    }
  }
  __device__ __forceinline__ f4 value() const {
    if constexpr (sizeof(T) == 4) return v;
    else return f4{u2f(v[0] << 16), u2f(v[0] & 0xFFFF0000u), u2f(v[1] << 16), u2f(v[1] & 0xFFFF0000u)};
  }
};
template <typename T>
struct Plain {
  const T* p;
  __device__ __forceinline__ const T* at(uint32_t element) const { return p + element; }
};
template <typename T, bool W>
__device__ __forceinline__ f4 ld4(const T* row, int c, int d) {
  Raw<T> r;
  r.template load<W>(Plain<T>{row}, 0, c, d);
  r.template cut<W>(d - c);
  return r.value();
}
template <typename T, bool W>
__device__ __forceinline__ void st4(T* row, int c, int d, f4 v) {
  if constexpr (W) {
    if (c >= d) return;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<f4*>(row + c) = v;
    else *reinterpret_cast<u2*>(row + c) = u2{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < d) st1(row + c + i, v[i]);
  }
}

// ---- products --------------------------------------------------------------
// Lane (i = lane % 16, g = lane / 16) holds of a left operand row i, of a right
// one column i, of a 16 x 16 result rows 4 g .. 4 g + 3 of column i.  Of every 32
// of k it holds eight, 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3: then two
// results, one under the other, are the right operand of the next product as
// they lie.  (Which k a slot stands for matters to neither MFMA, as long as both
// operands agree.)
//
// An operand's eight values are P pieces of 16 bytes.  bf16 rows: one piece,
// exact; fp32 values beside them: three, x = hi + mid + lo in bf16.  fp32 rows
// and values beside them: two pieces of four floats.
template <int P>
struct Frag {
  u4 p[P];
};
template <typename T>
struct Mode;
template <>
struct Mode<uint16_t> {
  static constexpr int ROWS = 1, FULL = 3;
};
template <>
struct Mode<float> {
  static constexpr int ROWS = 2, FULL = 2;
};

// one of three parts of a pair of floats; x and y keep the rest
__device__ __forceinline__ uint32_t part_of(float& x, float& y) {
  const uint32_t h = bf16_pair(x, y);
  x -= u2f(h << 16);
  y -= u2f(h & 0xFFFF0000u);
  return h;
}
template <typename T>
__device__ __forceinline__ Frag<Mode<T>::FULL> full(f4 a, f4 b) {
  Frag<Mode<T>::FULL> r;
  if constexpr (sizeof(T) == 4) {
    r.p[0] = __builtin_bit_cast(u4, a);
    r.p[1] = __builtin_bit_cast(u4, b);
  } else {
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      float x0 = a[0], x1 = a[1], x2 = a[2], x3 = a[3], y0 = b[0], y1 = b[1], y2 = b[2], y3 = b[3];
      r.p[p] = u4{part_of(x0, x1), part_of(x2, x3), part_of(y0, y1), part_of(y2, y3)};
      a = f4{x0, x1, x2, x3};
      b = f4{y0, y1, y2, y3};
    }
  }
  return r;
}
// of values that rows hold exactly
template <typename T>
__device__ __forceinline__ Frag<Mode<T>::ROWS> rows_of(f4 a, f4 b) {
  Frag<Mode<T>::ROWS> r;
  if constexpr (sizeof(T) == 4) {
    r.p[0] = __builtin_bit_cast(u4, a);
    r.p[1] = __builtin_bit_cast(u4, b);
  } else {
    r.p[0] = u4{bf16_pair(a[0], a[1]), bf16_pair(a[2], a[3]), bf16_pair(b[0], b[1]),
                bf16_pair(b[2], b[3])};
  }
  return r;
}
template <typename T, int PA, int PB>
__device__ __forceinline__ void mma(f4& acc, const Frag<PA>& a, const Frag<PB>& b) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f4 x = __builtin_bit_cast(f4, a.p[h]), y = __builtin_bit_cast(f4, b.p[h]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], acc, 0, 0, 0);
    }
  } else {
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    // the small parts first
#pragma unroll
    for (int s = 2; s >= 0; --s)
#pragma unroll
      for (int i = 0; i < PA; ++i)
        if (s - i >= 0 && s - i < PB)
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a.p[i]),
                                                        __builtin_bit_cast(b8, b.p[s - i]), acc, 0,
                                                        0, 0);
  }
}

// the same right operand under N left ones: products that do not wait for each
// other, part by part
template <typename T, int N, int PA, int PB>
__device__ __forceinline__ void mma(f4 (&acc)[N], const Frag<PA> (&a)[N], const Frag<PB>& b) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f4 y = __builtin_bit_cast(f4, b.p[h]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int n = 0; n < N; ++n)
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f4, a[n].p[h])[e], y[e],
                                                        acc[n], 0, 0, 0);
    }
  } else {
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
#pragma unroll
    for (int s = 2; s >= 0; --s)
#pragma unroll
      for (int i = 0; i < PA; ++i)
        if (s - i >= 0 && s - i < PB)
#pragma unroll
          for (int n = 0; n < N; ++n)
            acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a[n].p[i]),
                                                             __builtin_bit_cast(b8, b.p[s - i]),
                                                             acc[n], 0, 0, 0);
  }
}

// ---- operands in LDS -------------------------------------------------------
// A block is 16 rows x 32 of k as the lanes hold it, piece by piece, 16 bytes a
// lane; a tile of U blocks across.  The rows of each g, and of each block, are in
// another order, so that what is written at once (rows of several blocks, or
// groups of k) falls into different banks.
__device__ __forceinline__ int slot_of(int i, int g) { return (i ^ g) + 16 * g; }
__device__ __forceinline__ int slot_in(int block, int slot) { return slot ^ (block & 3); }
template <int P>
__device__ __forceinline__ Frag<P> get(const u4* tile, int block, int slot) {
  Frag<P> r;
#pragma unroll
  for (int p = 0; p < P; ++p) r.p[p] = tile[(block * P + p) * 64 + slot_in(block, slot)];
  return r;
}
// blocks b0, b0 + step, ..
template <int P, int N>
__device__ __forceinline__ void get(Frag<P> (&r)[N], const u4* tile, int b0, int step, int slot) {
#pragma unroll
  for (int n = 0; n < N; ++n) r[n] = get<P>(tile, b0 + n * step, slot);
}
// four values of one row, k .. k + 3 (k a multiple of 4)
template <typename T, int P>
__device__ __forceinline__ void put(u4* tile, int U, int row, int k, f4 v) {
  const int block = row / 16 * U + k / 32, h = k / 16 % 2;
  const int slot = slot_in(block, slot_of(row % 16, k / 4 % 4));
  if constexpr (sizeof(T) == 4) {
    tile[(block * 2 + h) * 64 + slot] = __builtin_bit_cast(u4, v);
  } else {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float a = v[0], b = v[1], c = v[2], d = v[3];
      const u2 w = {part_of(a, b), part_of(c, d)};
      reinterpret_cast<u2*>(tile + (block * P + p) * 64 + slot)[h] = w;
      v = f4{a, b, c, d};
    }
  }
}

// Four rows x four columns of floats at a time, a thread
struct Four {
  f4 v[4];
};
__device__ __forceinline__ Four turned(const Four& x) {
  Four t;
#pragma unroll
  for (int c = 0; c < 4; ++c) t.v[c] = f4{x.v[0][c], x.v[1][c], x.v[2][c], x.v[3][c]};
  return t;
}
template <typename T>
__device__ __forceinline__ void put_full(u4* tile, int U, int row, int k, const Four& x) {
#pragma unroll
  for (int e = 0; e < 4; ++e) put<T, Mode<T>::FULL>(tile, U, row + e, k, x.v[e]);
}

// a value that is the same in all lanes, kept in scalar registers
__device__ __forceinline__ int same(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t same(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)same((int)(x >> 32)) << 32 | (uint32_t)same((int)x));
}
// p[i] of elements of T, i of 32 bits beside a scalar address
template <typename T, typename P>
__device__ __forceinline__ T* at32(P* p, uint32_t i) {
  return reinterpret_cast<T*>((char*)p + (uint64_t)(i * (uint32_t)sizeof(T)));
}

struct Place {
  int l, h, c;     // lane, head, chunk
  int n;           // positions of the chunk within the lane's length
};
__device__ __forceinline__ int within(int len, int c) {
  const int left = len - c * C;
  return left < 0 ? 0 : (left < C ? left : C);
}
// The rows of a chunk, one head of d columns: where the first begins and how far
// apart they are.  All of it is the same in the whole block, so an element's
// address is a scalar one plus 32 bits (64 rows with strides up to 2^23 elements).
template <typename T>
struct Chunk {
  T* p;
  uint32_t row;  // elements
  template <typename R>
  __device__ __forceinline__ Chunk(const R& r, const Place& at, int h, int d)
      : p((T*)r.d + same(at.l * r.lane + (int64_t)at.c * C * r.row + (int64_t)h * d)),
        row((uint32_t)r.row) {}
  __device__ __forceinline__ T* at(uint32_t element) const { return at32<T>(p, element); }
};

// Rows pos .. pos + 3, columns col .. col + 3 of a chunk's rows, a thread: loaded,
// later put as rows (k along them) or across (k over the positions), with zeros
// past the chunk's positions and past d
template <typename T>
struct Rows4 {
  Raw<T> r[4];
  // n: the chunk's positions, one at least
  template <bool W>
  __device__ __forceinline__ void load(const Chunk<const T>& from, int n, int d, int pos, int col) {
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e].template load<W>(from, min(pos + e, n - 1) * from.row, col, d);
  }
  // rows from n on and columns from d on
  template <bool W>
  __device__ __forceinline__ void cut(int n, int d) {
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e].template cut<W>(e < n ? d : 0);
  }
  __device__ __forceinline__ Rows4 turned() const {
    Rows4 t;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int c = 0; c < 4; ++c) t.r[c].v = f4{r[0].v[c], r[1].v[c], r[2].v[c], r[3].v[c]};
    } else {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t a = r[0].v[c], b = r[1].v[c], x = r[2].v[c], y = r[3].v[c];
        t.r[2 * c].v = u2{__builtin_amdgcn_perm(b, a, 0x05040100), __builtin_amdgcn_perm(y, x, 0x05040100)};
        t.r[2 * c + 1].v = u2{__builtin_amdgcn_perm(b, a, 0x07060302), __builtin_amdgcn_perm(y, x, 0x07060302)};
      }
    }
    return t;
  }
  // as the rows `row` .. row + 3 of a tile, k .. k + 3
  __device__ __forceinline__ void put(u4* tile, int U, int row, int k) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int block = (row + e) / 16 * U + k / 32;
      const int slot = slot_in(block, slot_of((row + e) % 16, k / 4 % 4));
      if constexpr (sizeof(T) == 4)
        tile[(block * 2 + k / 16 % 2) * 64 + slot] = __builtin_bit_cast(u4, r[e].v);
      else reinterpret_cast<u2*>(tile + block * 64 + slot)[k / 16 % 2] = r[e].v;
    }
  }
};
// the rows that a lane holds of a 16 x 16 result: two of them, one under the other,
// from an operand across their rows
template <typename T>
__device__ __forceinline__ void results_of(f4& a, f4& b, const Frag<Mode<T>::ROWS>& f) {
  if constexpr (sizeof(T) == 4) {
    a = __builtin_bit_cast(f4, f.p[0]);
    b = __builtin_bit_cast(f4, f.p[1]);
  } else {
    a = Raw<T>{u2{f.p[0][0], f.p[0][1]}}.value();
    b = Raw<T>{u2{f.p[0][2], f.p[0][3]}}.value();
  }
}

// ---- what passes between the kernels, of a (lane, value head, chunk) -------
// T and P, lower triangles of 64 x 64, as operands: six blocks each (row tile t,
// 32 of k u: t = 0, 1: u = 0; t = 2, 3: u = 0, 1), transposed for the gradient
// (t = 0, 1: u = 0, 1; t = 2, 3: u = 1).
constexpr int TRI = 6;
template <bool TRANS>
__device__ __forceinline__ constexpr int tri_block(int t, int u) {
  return TRANS ? (t < 2 ? 2 * t + u : t + 2) : (t < 2 ? t : 2 * t - 2 + u);
}
// acc += triangle x b
template <typename T, bool TRANS, int PB>
__device__ __forceinline__ void triangle(f4 (&acc)[4], const u4* tri, const Frag<PB> (&b)[2],
                                         int slot) {
  constexpr int FULL = Mode<T>::FULL, U = TRANS ? 1 : 0;  // the 32 of k that all tiles have
  Frag<FULL> x[4], y[2];
#pragma unroll
  for (int t = 0; t < 4; ++t) x[t] = get<FULL>(tri, tri_block<TRANS>(t, U), slot);
#pragma unroll
  for (int t = 0; t < 2; ++t) y[t] = get<FULL>(tri, tri_block<TRANS>(TRANS ? t : 2 + t, 1 - U), slot);
  mma<T>(acc, x, b[U]);
  f4 two[2] = {acc[TRANS ? 0 : 2], acc[TRANS ? 1 : 3]};
  mma<T>(two, y, b[1 - U]);
  acc[TRANS ? 0 : 2] = two[0];
  acc[TRANS ? 1 : 3] = two[1];
}
// Coefficients of the rows, floats: beta; beta e^G / |k|; e^(G_64 - G) / |k|;
// scale e^G / |q|; then e^G_64; for the rows' gradients G as a power of two, e^G,
// e^(G_64 - G), 1 / |k| and 1 / |q| as well.
constexpr int CHAIN_COEF = 4 * C + 4, COEF = CHAIN_COEF + 6 * C;
template <typename T>
constexpr int IMAGE = 2 * TRI * Mode<T>::FULL * 64;  // 16-byte pieces of T and P
// the larger of the types': bf16's, 39 KB; fp32 rows leave a third of it unused
constexpr int64_t PREP_BYTES = 2 * TRI * 3 * 1024 + COEF * 4;

// the block's sums of log decays and betas, by its first wave
struct Decays {
  int whole[C];    // G, as a power of two
  float part[C];
  float beta[C];
  float since[C];  // e^G
  float left[C];   // e^(G_64 - G)
};
__device__ __forceinline__ void decays_of(Decays& s, const DeltaArgs& a, const Place& p) {
  const int i = threadIdx.x;
  if (i >= C) return;
  const int64_t t = p.c * C + min(i, p.n - 1);
  double g = log_decay(*((const float*)a.g.d + p.l * a.g.lane + t * a.g.row + p.h));
  float beta = *((const float*)a.beta.d + p.l * a.beta.lane + t * a.beta.row + p.h);
  if (i >= p.n) g = 0.0, beta = 0.0f;
#pragma unroll
  for (int m = 1; m < C; m *= 2) {
    const double y = __shfl_up(g, m);
    if (i >= m) g += y;
  }
  const double all = __shfl(g, C - 1);
  const Power at = power_of(g);
  s.whole[i] = at.whole;
  s.part[i] = at.part;
  s.beta[i] = beta;
  s.since[i] = exp_of(g);
  s.left[i] = exp_of(all - g);
}

// ---- prep ------------------------------------------------------------------
// products of [64][64] tiles of floats on the fp32 MFMA, for T alone: rows i0 +
// i, k from 16 kk + 4 g along the rows or across them
__device__ __forceinline__ f4 along(const float* t, int i0, int kk, int lane) {
  return *reinterpret_cast<const f4*>(t + (i0 + lane % 16) * CP + kk * 16 + lane / 16 * 4);
}
__device__ __forceinline__ f4 across(const float* t, int i0, int kk, int lane) {
  const float* p = t + (kk * 16 + lane / 16 * 4) * CP + i0 + lane % 16;
  return f4{p[0], p[CP], p[2 * CP], p[3 * CP]};
}
__device__ __forceinline__ void mma16(f4& acc, f4 x, f4 y) {
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], acc, 0, 0, 0);
}

// A block per (lane, value head, chunk): T and P as the chain reads them, and
// the coefficients.  Bound by a block's chain of steps (the substitution of 16
// columns, then the products between blocks) and by the 39 KB that it writes: 2048
// chunks of 64 columns of k 46 us, 1.8 TB/s.  All chunks are at hand at once, so as
// many blocks as registers and LDS allow share a CU: four for bf16 rows and d_k up to
// 64, three at 128 (two: 74 and not 59 us for the prompts of 64 x 521, 8 heads); two
// or three for fp32 rows, one at 128, whose K and Q take 64 KB.
template <typename T, int DK, bool TRANS, bool W>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? (DK == 64 ? 4 : 3) : DK == 64 ? 2 : 1)
void delta_prep_kernel(const DeltaArgs a, unsigned char* prep, int chunks, uint32_t* order,
                       uint64_t blocks) {
  using M = Mode<T>;
  constexpr int U = DK / 32, P = M::ROWS;
  constexpr int TILE = 4 * U * P * 64;
  __shared__ union {
    u4 kq[2 * TILE];  // K and Q, until their products are there
    float t[C * CP];
  } lds;
  u4 *ka = lds.kq, *qa = lds.kq + TILE;
  float* tm = lds.t;
  __shared__ __align__(16) float am[C * CP];
  __shared__ float ssk[C], ssq[C], rk[C], rq[C];
  __shared__ Decays s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane % 16, g = lane / 16, g4 = 4 * g, sl = slot_of(i16, g);
  // the lanes' order, the longest first, for the chain
  for (int l = blockIdx.x; order && l < a.q.lanes; l += gridDim.x) {
    const int own = seq_len(a.q, l);
    int rank = 0;
    for (int j0 = 0; j0 < a.q.lanes; j0 += 256) {
      const int j = j0 + tid, other = seq_len(a.q, min(j, a.q.lanes - 1));
      rank += __syncthreads_count(j < a.q.lanes && (other > own || (other == own && j < l)));
    }
    if (tid == 0) order[rank] = l;
  }
  for (uint64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    Place p;
    p.c = same((int)(b % chunks));
    p.h = same((int)(b / chunks % a.HV));
    p.l = same((int)(b / chunks / a.HV));
    p.n = same(within(seq_len(a.q, p.l), p.c));
    if (!p.n) continue;
    const int kh = same(p.h / (a.HV / a.H));
    const int pos = tid / 16 * 4, col = tid % 16 * 4;
    Rows4<T> k[DK / 64], q[DK / 64];
#pragma unroll
    for (int i = 0; i < DK / 64; ++i) {
      k[i].template load<W>(Chunk<const T>(a.k, p, kh, a.dk), p.n, a.dk, pos, i * 64 + col);
      q[i].template load<W>(Chunk<const T>(a.qr, p, kh, a.dk), p.n, a.dk, pos, i * 64 + col);
    }
    __syncthreads();
    decays_of(s, a, p);
#pragma unroll
    for (int i = 0; i < DK / 64; ++i) {
      k[i].template cut<W>(p.n - pos, a.dk - i * 64 - col);
      q[i].template cut<W>(p.n - pos, a.dk - i * 64 - col);
      k[i].put(ka, U, pos, i * 64 + col);
      q[i].put(qa, U, pos, i * 64 + col);
    }
    __syncthreads();
    // this wave's 16 rows of K K^T and Q K^T up to the diagonal; Q Q^T for the
    // lengths, as K K^T's diagonal has those of k
    f4 kk[4] = {}, qk[4] = {}, qq = ZERO;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Frag<P> x = get<P>(ka, wave * U + u, sl), y = get<P>(qa, wave * U + u, sl);
      mma<T>(qq, y, y);
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (n <= wave) {
          const Frag<P> z = get<P>(ka, n * U + u, sl);
          mma<T>(kk[n], x, z);
          mma<T>(qk[n], y, z);
        }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n == wave && g4 + r == i16) ssk[wave * 16 + i16] = kk[n][r], ssq[wave * 16 + i16] = qq[r];
    __syncthreads();
    if (tid < C) {
      rk[tid] = a.unit ? 1.0f / __builtin_sqrtf(ssk[tid] + EPS) : 1.0f;
      rq[tid] = a.unit ? a.scale / __builtin_sqrtf(ssq[tid] + EPS) : a.scale;
    }
    for (int i = tid; i < C * CP / 4; i += 256) reinterpret_cast<f4*>(tm)[i] = ZERO;
    __syncthreads();
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = wave * 16 + g4 + r, j = n * 16 + i16;
        float d = 0.0f;
        if (n <= wave && j <= i) d = raised(s.whole[i] - s.whole[j], s.part[i] - s.part[j]);
        am[i * CP + j] = n <= wave && j < i ? kk[n][r] * (s.beta[i] * rk[i] * rk[j] * d) : 0.0f;
        qk[n][r] = n <= wave && j <= i ? qk[n][r] * (rq[i] * rk[j] * d) : 0.0f;
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
      f4 at = ZERO, t21 = ZERO;
      mma16(at, along(am + o, o + 16, 0, lane), across(tm + o * CP + o, 0, 0, lane));
      mma16(t21, along(tm + o + 16, o + 16, 0, lane), at);
#pragma unroll
      for (int r = 0; r < 4; ++r) tm[(o + 16 + g4 + r) * CP + o + i16] = -t21[r];
    }
    __syncthreads();
    {
      const int ri = 32 + wave / 2 * 16, cj = wave % 2 * 16;
      f4 t21 = ZERO;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        f4 at = ZERO;
#pragma unroll
        for (int kk2 = 0; kk2 < 2; ++kk2)
          mma16(at, along(am, 32 + m * 16, kk2, lane), across(tm, cj, kk2, lane));
        mma16(t21, along(tm + 32, ri, m, lane), at);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) tm[(ri + g4 + r) * CP + cj + i16] = -t21[r];
    }
    __syncthreads();  // am has been read: P takes its place
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) am[(wave * 16 + g4 + r) * CP + n * 16 + i16] = qk[n][r];
    __syncthreads();
    unsigned char* at = prep + b * PREP_BYTES;
    u4* image = reinterpret_cast<u4*>(at);
#pragma unroll
    for (int it = 0; it < 3; ++it) {
      const int job = it * 4 + wave;  // of T's and P's six blocks
      const int block = job % TRI;
      const float* m = job < TRI ? tm : am;
      int t, u;
      if (TRANS) t = block < 4 ? block / 2 : block - 2, u = block < 4 ? block % 2 : 1;
      else t = block < 2 ? block : block / 2 + 1, u = block < 2 ? 0 : block % 2;
      f4 lo, hi;
      if (TRANS) {
        lo = across(m, t * 16, 2 * u, lane);
        hi = across(m, t * 16, 2 * u + 1, lane);
      } else {
        lo = along(m, t * 16, 2 * u, lane);
        hi = along(m, t * 16, 2 * u + 1, lane);
      }
      const Frag<M::FULL> f = full<T>(lo, hi);
#pragma unroll
      for (int i = 0; i < M::FULL; ++i) image[(job * M::FULL + i) * 64 + slot_in(block, sl)] = f.p[i];
    }
    float* coef = reinterpret_cast<float*>(at + PREP_BYTES - COEF * 4);
    if (tid < C) {
      coef[tid] = s.beta[tid];
      coef[C + tid] = s.beta[tid] * s.since[tid] * rk[tid];
      coef[2 * C + tid] = s.left[tid] * rk[tid];
      coef[3 * C + tid] = rq[tid] * s.since[tid];
      if (tid == C - 1) coef[4 * C] = s.since[tid];
      if (TRANS) {
        float* more = coef + CHAIN_COEF + tid;
        more[0] = s.part[tid];
        reinterpret_cast<int*>(more)[C] = s.whole[tid];
        more[2 * C] = s.since[tid];
        more[3 * C] = s.left[tid];
        more[4 * C] = rk[tid];
        more[5 * C] = a.unit ? 1.0f / __builtin_sqrtf(ssq[tid] + EPS) : 1.0f;
      }
    }
  }
}

// ---- chain -----------------------------------------------------------------
// A block per (lane, value head, 64 columns), a wave 16 of them.  Of a chunk the
// block's LDS holds K as rows and across, Q as rows (the gradient's chain: across),
// T and P (there: transposed), v across and the coefficients; the next chunk's are
// under way in registers.  The state, 16 columns of it, stays in the wave's registers.
template <typename T, int DK, bool TRANS>
struct ChainLds {
  u4 ka[4 * (DK / 32) * Mode<T>::ROWS * 64], kt[DK / 16 * 2 * Mode<T>::ROWS * 64];
  u4 q[4 * (DK / 32) * Mode<T>::ROWS * 64];  // rows, or across: as many blocks
  u4 v[4 * 2 * Mode<T>::ROWS * 64];  // v (dO), across: 16 columns a wave; then its results
  u4 tri[IMAGE<T>];
  float coef[CHAIN_COEF];
};
template <typename T, int DK>
struct ChainNext {
  static constexpr int IMG = (IMAGE<T> + 255) / 256;
  Rows4<T> k[DK / 64], q[DK / 64], v;
  u4 img[IMG];
  float coef[2];
  template <bool W>
  __device__ __forceinline__ void load(const DeltaArgs& a, const unsigned char* prep, const Place& p,
                                       int kh, const RowsIn& rows, int v0) {
    const int tid = threadIdx.x, pos = tid / 16 * 4, col = tid % 16 * 4;
#pragma unroll
    for (int i = 0; i < IMG; ++i)
      img[i] = *at32<const u4>(prep, min(tid + 256 * i, IMAGE<T> - 1));
    const unsigned char* c = prep + PREP_BYTES - COEF * 4;
    coef[0] = *at32<const float>(c, tid);
    coef[1] = *at32<const float>(c, 4 * C);
#pragma unroll
    for (int i = 0; i < DK / 64; ++i) {
      k[i].template load<W>(Chunk<const T>(a.k, p, kh, a.dk), p.n, a.dk, pos, i * 64 + col);
      q[i].template load<W>(Chunk<const T>(a.qr, p, kh, a.dk), p.n, a.dk, pos, i * 64 + col);
    }
    v.template load<W>(Chunk<const T>(rows, p, p.h, a.dv), p.n, a.dv, pos, v0 + col);
  }
  // n: the chunk's positions
  template <bool W, bool TRANS>
  __device__ __forceinline__ void store(ChainLds<T, DK, TRANS>& s, int n, int dk, int dv) {
    const int tid = threadIdx.x, pos = tid / 16 * 4, c4 = tid % 16 * 4;
    // dv: columns of v left from the block's first one on
    if (n < C || dv < 64) v.template cut<W>(n - pos, dv - c4);
    v.turned().put(s.v, 2, c4, pos);
    if (n < C || dk < DK) {
#pragma unroll
      for (int i = 0; i < DK / 64; ++i) {
        k[i].template cut<W>(n - pos, dk - i * 64 - c4);
        q[i].template cut<W>(n - pos, dk - i * 64 - c4);
      }
    }
#pragma unroll
    for (int i = 0; i < DK / 64; ++i) {
      const int col = i * 64 + c4;
      k[i].put(s.ka, DK / 32, pos, col);
      k[i].turned().put(s.kt, 2, col, pos);
      if (TRANS) q[i].turned().put(s.q, 2, col, pos);
      else q[i].put(s.q, DK / 32, pos, col);
    }
#pragma unroll
    for (int i = 0; i < IMG; ++i)
      if (tid + 256 * i < IMAGE<T>) s.tri[tid + 256 * i] = img[i];
    s.coef[tid] = coef[0];
    if (tid == 0) s.coef[4 * C] = coef[1];
  }
};

// The compiler moves nothing across: left alone it brings all of a loop's operands
// in first, for which the registers do not suffice.
__device__ __forceinline__ void apart() { __builtin_amdgcn_sched_barrier(0); }

// rows 4 g .. of tile t of a [64] array
__device__ __forceinline__ f4 four_rows(const float* c, int t, int g) {
  return *reinterpret_cast<const f4*>(c + t * 16 + 4 * g);
}

// A wave's 64 x 16 results as rows from column v0 on: each lane puts its column
// into its slots of the wave's two blocks and takes four rows of four columns.
template <typename T, bool W>
__device__ __forceinline__ void put_result(u4* tile, const f4 (&o)[4], int wave, int lane, int slot,
                                           const Chunk<T>& out, int n, int v0, int dv) {
  constexpr int P = Mode<T>::ROWS;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const Frag<P> f = rows_of<T>(o[2 * u], o[2 * u + 1]);
#pragma unroll
    for (int p = 0; p < P; ++p)
      tile[((wave * 2 + u) * P + p) * 64 + slot_in(wave * 2 + u, slot)] = f.p[p];
  }
  // the wave's own LDS accesses are in order; the compiler's have to be
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const int pg = lane / 4, cg = lane % 4, block = wave * 2 + pg / 8, h = pg / 4 % 2;
  Rows4<T> x;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int s = slot_in(block, slot_of(cg * 4 + c, pg % 4));
    if constexpr (sizeof(T) == 4) x.r[c].v = __builtin_bit_cast(f4, tile[(block * 2 + h) * 64 + s]);
    else x.r[c].v = reinterpret_cast<const u2*>(tile + block * 64 + s)[h];
  }
  x = x.turned();
  const int col = v0 + cg * 4;
  const uint32_t first = 4 * pg * out.row + col;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (4 * pg + e < n) x.r[e].template store<W>(out, first + e * out.row, dv - col);
}

// Few sequences of many chunks are cut into segments.  A first pass takes each
// from a zero state, and beside it (LOCAL's tiles past those of d_v) from the
// columns of the identity without v: its last state is then what the segment adds
// and what it makes of the state before it.  The combine kernel chains those, and
// the main pass takes every segment from its own first state.
struct Segments {
  int n, chunks;  // segments of a sequence, chunks of a segment
  float* local;   // [lane][v head][segment][64 tiles + 2 d_k][d_k]: a row for each column;
                  // the identity's as rows, too
  float* first;   // [lane][v head][segment][64 tiles columns][d_k]: the states it is taken from
};

// The states from chunk to chunk and O.  A block's four waves, 16 columns of S, N
// and O each, share K, Q, T, P and v in LDS (69 KB for bf16 rows and d_k up to 64, so
// that two blocks share a CU: forward of 64 x 512, 4 heads of 64 and 128 columns, 105
// us and not 123; 93 KB at 128 and 91 KB for fp32 rows, one block: there a bound of two
// saves registers only, which aligned rows do not lack and for which others spill, 227
// and not 209 us for 64 x 512 fp32 rows in odd places).  S stays in registers as the next
// product's right operand, so a wave has no exchange with others but the barriers
// around a chunk's loads, which are a chunk ahead.  6 us a chunk; the matrix
// instructions take 0.15 (d_k up to 64, with S and N kept) to 0.18 of the SIMDs' time.
// Where S and N are kept for the gradient, their bytes bound it: 98 us for 32 x 1024
// bf16 rows, 4 heads of 64 and 128 columns, 150 KB a chunk, 80 of them written, 3.1
// TB/s.  Else the latency of a chunk's dependent products (S -> R -> N -> S), with one
// wave a SIMD.  O by a second wave beside the one that carries S: 102 us there, and a
// prefill of 64 x 521, 8 heads of 128 x 128, 255 us in all and not 240.
template <typename T, int DK, bool W, bool LOCAL>
__global__ __launch_bounds__(256, DK == 64 && (sizeof(T) == 2 || W) ? 2 : 1)
void delta_chain_kernel(
    const DeltaArgs a, const unsigned char* prep, float* rec, int chunks, int tiles,
    const Segments seg, const uint32_t* order, uint32_t blocks) {
  using M = Mode<T>;
  constexpr int U = DK / 32, MT = DK / 16, FULL = M::FULL, P = M::ROWS;
  extern __shared__ __align__(16) unsigned char lds[];
  ChainLds<T, DK, false>& s = *reinterpret_cast<ChainLds<T, DK, false>*>(lds);
  const int per = LOCAL ? tiles + DK / 64 : tiles;
  for (uint32_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    // (computed here, not kept from before the loop, for which registers lack)
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, wave = same(tid >> 6);
    const int i16 = lane % 16, g = lane / 16, sl = slot_of(i16, g);
    const uint32_t ls = same((int)(b / per)), nth = same((int)(ls / seg.n));
    const int sg = ls - nth * seg.n;
    Place p;
    p.l = same((int)(nth / a.HV));
    p.h = nth - p.l * a.HV;
    if (order) p.l = same((int)order[p.l]);
    const uint32_t lh = (uint32_t)p.l * a.HV + p.h;
    const int kh = same(p.h / (a.HV / a.H)), len = same(seq_len(a.q, p.l)), all = (len + C - 1) / C;
    const int from = sg * seg.chunks, last = min(all, from + seg.chunks);
    const int vb = same((int)(b - ls * per) * 64), v0 = vb + wave * 16, col = v0 + i16;
    const bool mine = col < a.dv;
    const int left = LOCAL && vb >= tiles * 64 ? 0 : a.dv - vb;  // columns of v from vb on
    const int64_t state = (int64_t)lh * a.dk * a.dv;
    f4 st[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      st[m] = ZERO;
      if constexpr (LOCAL) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (m * 16 + 4 * g + r == col - tiles * 64) st[m][r] = 1.0f;
      } else if (seg.n > 1) {
        st[m] = *at32<const f4>(seg.first + same((int64_t)ls * tiles * 64 * DK),
                                col * (DK / 4) + m * 4 + g);
      } else if (a.state_in && mine) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (m * 16 + 4 * g + r < a.dk)
            st[m][r] = a.state_in[state + (int64_t)(m * 16 + 4 * g + r) * a.dv + col];
      }
    }
    ChainNext<T, DK> next;
    auto bring = [&](int c) {
      p.c = c;
      p.n = within(len, c);
      next.template load<W>(a, prep + same(((int64_t)lh * chunks + c) * PREP_BYTES), p, kh, a.v, vb);
    };
    if (last > from) bring(from);
    for (int c = from; c < last; ++c) {
      __syncthreads();
      next.template store<W>(s, p.n, a.dk, left);
      const int n = p.n;
      __syncthreads();
      if (c + 1 < last) bring(c + 1);
      if (!LOCAL && v0 >= a.dv) continue;
      float* at = rec + same(((int64_t)lh * chunks + c) * (a.dv * (DK + C)));
      if (!LOCAL && rec && mine) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
          *at32<f4>(at, col * (DK / 4) + m * 4 + g) = st[m];
      }
      f4 o[4], x[4];
      {
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = o[t] = ZERO;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const Frag<FULL> sf = full<T>(st[2 * u], st[2 * u + 1]);
          Frag<P> k[4], q[4];
          get<P>(k, s.ka, u, U, sl);
          mma<T>(x, k, sf);
          if constexpr (!LOCAL) {
            get<P>(q, s.q, u, U, sl);
            mma<T>(o, q, sf);
          }
          if constexpr (DK == 64) apart();
        }
      }
      f4 nn[4];
      {
        f4 vc[4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
          results_of<T>(vc[2 * u], vc[2 * u + 1], get<P>(s.v, wave * 2 + u, sl));
#pragma unroll
        for (int t = 0; t < 4; ++t)
          x[t] = four_rows(s.coef, t, g) * vc[t] - four_rows(s.coef + C, t, g) * x[t];
        Frag<FULL> rf[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) rf[u] = full<T>(x[2 * u], x[2 * u + 1]);
#pragma unroll
        for (int t = 0; t < 4; ++t) nn[t] = ZERO;
        triangle<T, false>(nn, s.tri, rf, sl);
      }
      if constexpr (!LOCAL) {
        Frag<FULL> nf[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) nf[u] = full<T>(nn[2 * u], nn[2 * u + 1]);
#pragma unroll
        for (int t = 0; t < 4; ++t) o[t] *= four_rows(s.coef + 3 * C, t, g);
        triangle<T, false>(o, s.tri + TRI * FULL * 64, nf, sl);
      }
      {
        Frag<FULL> nf[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
          nf[u] = full<T>(nn[2 * u] * four_rows(s.coef + 2 * C, 2 * u, g),
                          nn[2 * u + 1] * four_rows(s.coef + 2 * C, 2 * u + 1, g));
        const float all = s.coef[4 * C];
#pragma unroll
        for (int m = 0; m < MT; ++m) st[m] *= all;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          Frag<P> k[MT];
          get<P>(k, s.kt, u, 2, sl);
          mma<T>(st, k, nf[u]);
          if constexpr (DK == 64) apart();
        }
      }
      if constexpr (LOCAL) continue;
      if (rec && mine) {
#pragma unroll
        for (int t = 0; t < 4; ++t) *at32<f4>(at + a.dv * DK, col * (C / 4) + t * 4 + g) = nn[t];
      }
      // O, from a column to a row in each lane: through the wave's own part of v
      Place here = p;
      here.c = c;
      put_result<T, W>(s.v, o, wave, lane, sl, Chunk<T>(a.out, here, p.h, a.dv), n, v0, a.dv);
    }
    if constexpr (LOCAL) {
      float* to = seg.local + same((int64_t)ls * (tiles * 64 + 2 * DK) * DK);
#pragma unroll
      for (int m = 0; m < MT; ++m) *at32<f4>(to, col * (DK / 4) + m * 4 + g) = st[m];
      if (vb >= tiles * 64)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            to[(tiles * 64 + DK + m * 16 + 4 * g + r) * DK + col - tiles * 64] = st[m][r];
    } else if (a.state_out && mine && sg == max(0, (all - 1) / seg.chunks)) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (m * 16 + 4 * g + r < a.dk)
            a.state_out[state + (int64_t)(m * 16 + 4 * g + r) * a.dv + col] = st[m][r];
    }
    __syncthreads();
  }
}

// The gradient's chain, from the last chunk to the first: dS and dR of every
// chunk, both with a column of d_v after the other, as S and N are kept.  Bound as
// the forward chain: 90 us for 32 x 1024, 4 heads of 64 and 128 columns, 3.0 TB/s.
template <typename T, int DK, bool W, bool LOCAL>
__global__ __launch_bounds__(256, 1) void delta_grad_chain_kernel(
    const DeltaGradArgs ga, const unsigned char* prep, float* grec, int chunks, int tiles,
    const Segments seg, const uint32_t* order, uint32_t blocks) {
  using M = Mode<T>;
  constexpr int U = DK / 32, MT = DK / 16, FULL = M::FULL, P = M::ROWS;
  extern __shared__ __align__(16) unsigned char lds[];
  const DeltaArgs& a = ga.f;
  ChainLds<T, DK, true>& s = *reinterpret_cast<ChainLds<T, DK, true>*>(lds);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane % 16, g = lane / 16, sl = slot_of(i16, g);
  for (uint32_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const uint32_t ls = same((int)(b / tiles)), nth = same((int)(ls / seg.n));
    const int sg = ls - nth * seg.n;
    Place p;
    p.l = same((int)(nth / a.HV));
    p.h = nth - p.l * a.HV;
    if (order) p.l = same((int)order[p.l]);
    const uint32_t lh = (uint32_t)p.l * a.HV + p.h;
    const int kh = same(p.h / (a.HV / a.H)), len = same(seq_len(a.q, p.l)), all = (len + C - 1) / C;
    const int from = sg * seg.chunks, last = min(all, from + seg.chunks);
    const int vb = same((int)(b - ls * tiles) * 64), v0 = vb + wave * 16, col = v0 + i16;
    const bool mine = col < a.dv;
    const int64_t state = (int64_t)lh * a.dk * a.dv;
    f4 st[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      st[m] = ZERO;
      if constexpr (LOCAL) {
      } else if (seg.n > 1) {
        st[m] = *at32<const f4>(seg.first + same((int64_t)ls * tiles * 64 * DK),
                                col * (DK / 4) + m * 4 + g);
      } else if (ga.dstate_out && mine) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (m * 16 + 4 * g + r < a.dk)
            st[m][r] = ga.dstate_out[state + (int64_t)(m * 16 + 4 * g + r) * a.dv + col];
      }
    }
    ChainNext<T, DK> next;
    auto bring = [&](int c) {
      p.c = c;
      p.n = within(len, c);
      next.template load<W>(a, prep + same(((int64_t)lh * chunks + c) * PREP_BYTES), p, kh, ga.dout, vb);
    };
    if (last > from) bring(last - 1);
    for (int c = last - 1; c >= from; --c) {
      __syncthreads();
      next.template store<W>(s, p.n, a.dk, a.dv - vb);
      __syncthreads();
      if (c > from) bring(c - 1);
      if (v0 >= a.dv) continue;
      float* at = grec + same(((int64_t)lh * chunks + c) * (a.dv * (DK + C)));
      if (!LOCAL && mine) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
          *at32<f4>(at, col * (DK / 4) + m * 4 + g) = st[m];
      }
      f4 dn[4], dout[4];
      {
        Frag<FULL> sf[U];
#pragma unroll
        for (int u = 0; u < U; ++u) sf[u] = full<T>(st[2 * u], st[2 * u + 1]);
        Frag<P> of[2];
        get<P>(of, s.v, wave * 2, 1, sl);
#pragma unroll
        for (int u = 0; u < 2; ++u) results_of<T>(dout[2 * u], dout[2 * u + 1], of[u]);
#pragma unroll
        for (int t = 0; t < 4; ++t) dn[t] = ZERO;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          Frag<P> k[4];
          get<P>(k, s.ka, u, U, sl);
          mma<T>(dn, k, sf[u]);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) dn[t] *= four_rows(s.coef + 2 * C, t, g);
        triangle<T, true>(dn, s.tri + TRI * FULL * 64, of, sl);
      }
      f4 dr[4];
      {
        Frag<FULL> nf[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) nf[u] = full<T>(dn[2 * u], dn[2 * u + 1]);
#pragma unroll
        for (int t = 0; t < 4; ++t) dr[t] = ZERO;
        triangle<T, true>(dr, s.tri, nf, sl);
      }
      if (!LOCAL && mine) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
          *at32<f4>(at + a.dv * DK, col * (C / 4) + t * 4 + g) = dr[t];
      }
      {
        Frag<FULL> of[2], rf[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          of[u] = full<T>(dout[2 * u] * four_rows(s.coef + 3 * C, 2 * u, g),
                          dout[2 * u + 1] * four_rows(s.coef + 3 * C, 2 * u + 1, g));
          rf[u] = full<T>(dr[2 * u] * -four_rows(s.coef + C, 2 * u, g),
                          dr[2 * u + 1] * -four_rows(s.coef + C, 2 * u + 1, g));
        }
        const float all = s.coef[4 * C];
#pragma unroll
        for (int m = 0; m < MT; ++m) st[m] *= all;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          Frag<P> k[MT], q[MT];
          get<P>(q, s.q, u, 2, sl);
          get<P>(k, s.kt, u, 2, sl);
          mma<T>(st, q, of[u]);
          mma<T>(st, k, rf[u]);
        }
      }
    }
    if constexpr (LOCAL) {
      float* to = seg.local + same((int64_t)ls * tiles * 64 * DK);
#pragma unroll
      for (int m = 0; m < MT; ++m) *at32<f4>(to, col * (DK / 4) + m * 4 + g) = st[m];
    } else if (ga.dstate_in && mine && sg == 0) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (m * 16 + 4 * g + r < a.dk)
            ga.dstate_in[state + (int64_t)(m * 16 + 4 * g + r) * a.dv + col] = st[m][r];
    }
    __syncthreads();
  }
}

// The segments' first states, one from the other: S = M S + what the segment adds,
// M its last states from the identity; or backwards, dS = M^T dS + what it adds.
// A block per 16 columns of a (lane, value head), a quarter of the rows a wave; the
// next segment's M is under way while the states pass through LDS.  Bound by the
// latency of one step: 63 segments of 64 columns 48 us (with one wave a block, which
// reads M's columns as they lie, 245).
template <int DK, bool BACK>
__global__ __launch_bounds__(256) void delta_combine_kernel(const DeltaArgs a, const float* first,
                                                            const float* moves, const float* adds,
                                                            int adds_columns, float* states,
                                                            int tiles, int segments, uint32_t blocks) {
  constexpr int MT = DK / 16, MW = MT / 4;
  __shared__ f4 now[2][MT][64];
  const int tid = threadIdx.x, lane = tid & 63, w = same(tid >> 6), i16 = lane % 16, g = lane / 16;
  for (uint32_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    const uint32_t lh = b / (4 * tiles);
    const int col = (int)(b - lh * 4 * tiles) * 16 + i16;
    f4 st[MW], add[MW], move[MW][MT];
    auto bring = [&](int i) {
      const int64_t at = (int64_t)lh * segments + (BACK ? segments - 1 - i : i);
      const float* m_ = moves + (at * (tiles * 64 + 2 * DK) + tiles * 64 + (BACK ? 0 : DK)) * DK;
#pragma unroll
      for (int m = 0; m < MW; ++m) {
        const int row = (w * MW + m) * 16;
        add[m] = *reinterpret_cast<const f4*>(adds + (at * adds_columns + col) * DK + row + 4 * g);
#pragma unroll
        for (int n = 0; n < MT; ++n)
          move[m][n] = *reinterpret_cast<const f4*>(m_ + (row + i16) * DK + n * 16 + 4 * g);
      }
    };
#pragma unroll
    for (int m = 0; m < MW; ++m) {
      st[m] = ZERO;
      const int row = (w * MW + m) * 16 + 4 * g;
      if (first && col < a.dv)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (row + r < a.dk) st[m][r] = first[((int64_t)lh * a.dk + row + r) * a.dv + col];
    }
    bring(0);
    for (int i = 0; i < segments; ++i) {
      const int64_t at = (int64_t)lh * segments + (BACK ? segments - 1 - i : i);
#pragma unroll
      for (int m = 0; m < MW; ++m) {
        now[i % 2][w * MW + m][lane] = st[m];
        *reinterpret_cast<f4*>(states + (at * tiles * 64 + col) * DK + (w * MW + m) * 16 + 4 * g) =
            st[m];
        st[m] = add[m];
      }
      if (i + 1 == segments) break;
      __syncthreads();
#pragma unroll
      for (int n = 0; n < MT; ++n) {
        const f4 y = now[i % 2][n][lane];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int m = 0; m < MW; ++m)
            st[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(move[m][n][j], y[j], st[m], 0, 0, 0);
      }
      bring(min(i + 1, segments - 2));  // (none after the last)
    }
    __syncthreads();
  }
}

// ---- the rows' gradients of a chunk ----------------------------------------
// A block of eight waves per (lane, head of k, chunk) takes all value heads that
// share the head.  Wave w of the first four and wave w of the other four have 16
// of the positions, "own".  Products over d_v come 32 columns at a time, N, dR,
// dO, S and dS as left operands in LDS and the own rows of them (the same pieces)
// as right ones.  The first four waves take dP and dA,
//   m < w:  dP^T, dA^T (rows j of tile m, column i own)      m > w:  dP, dA (rows i of tile m, column j own)
// and both for the own tile w, so that sums over rows and over columns of dP P
// and dA A stay within the wave, and what K and Q are multiplied with lies as the
// right operand; then those products.  The other four take what comes from the
// states, dO S^T, dR S^T and N dS^T.  (By the same wave the two do not fit its
// registers: forward and gradient of 4 x 777 rows, 4 heads of 128 and 8 of 128
// columns, 341 us and not 319.)  Bound by the two roles' waits for each other and by
// the LDS between products: 194 us for 32 x 1024 rows, 4 heads of 64 and 128 columns,
// 2.2 TB/s; the matrix instructions take 0.14.  K and Q kept in LDS rather than
// in registers: 234; the products' operands brought one tile ahead in the first four
// waves: 218.  At 128 columns of k the second role's seven arrays (dq, dk, qo, ko, os,
// rs, ns) are 224 registers: 218 to 272 are spilled, 600 to 700 bytes a lane, and with
// 208 blocks of two value heads each a ragged 4 x 777 rows take 93 us.  At 64 columns
// 31 (bf16, aligned) to 77 (fp32, not) are spilled.
// dQ^T and dK^T [d_k][own] leave as four neighbouring columns a lane.
template <typename T, int DK>
struct LastLds {
  static constexpr int P = Mode<T>::ROWS, FULL = Mode<T>::FULL;
  union {
    struct {
      u4 a[4 * (DK / 32) * P * 64], b[4 * (DK / 32) * P * 64];  // K, Q: rows; then across
      f4 states[2 * DK / 16][4][64];  // what the first waves have of dQ and dK
    } k;
    struct {
      u4 n[4 * FULL * 64], r[4 * FULL * 64], o[4 * P * 64];
      u4 s[DK / 16 * FULL * 64], d[DK / 16 * FULL * 64];
    } v;
  };
  float dot[8][C];  // dR . v, by groups of four columns
  float dsum[C], from[C], dots[C], tail[8];
  struct {
    float beta[C], unused[3 * C], all[4], part[C];
    int whole[C];
    float since[C], left[C], rk[C], uq[C];
  } coef;
};
static_assert(sizeof(LastLds<float, 64>::coef) == COEF * 4, "as prep leaves them");

template <int P>
__device__ __forceinline__ Frag<P> either(bool first, const Frag<P>& a, const Frag<P>& b) {
  Frag<P> r;
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int i = 0; i < 4; ++i) r.p[p][i] = first ? a.p[p][i] : b.p[p][i];
  return r;
}
__device__ __forceinline__ f4 either(bool first, f4 a, f4 b) {
  return f4{first ? a[0] : b[0], first ? a[1] : b[1], first ? a[2] : b[2], first ? a[3] : b[3]};
}
__device__ __forceinline__ f4 one_of(const f4 (&x)[4], int w) {
  return either(w < 2, either(w == 0, x[0], x[1]), either(w == 2, x[2], x[3]));
}

// What a thread brings of 32 columns of d_v: of the first 256, four columns of
// four positions of N and dO, or of dR and v; of the others, four columns of two
// rows (of 64) of S and dS.
template <typename T>
struct LastRows {
  Four x;
  Rows4<T> rows;
  template <bool W>
  __device__ __forceinline__ void load(const float* x_, const Chunk<const T>& from, int n, int dv,
                                       int v4, int pg) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x.v[i] = *at32<const f4>(x_, min(v4 + i, dv - 1) * (C / 4) + pg);
    rows.template load<W>(from, n, dv, pg * 4, v4);
  }
};
typedef float f2 __attribute__((ext_vector_type(2)));
typedef int i4 __attribute__((ext_vector_type(4)));
template <int DK>
struct LastStates {
  f2 s[DK / 64][4], d[DK / 64][4];
  __device__ __forceinline__ void load(const float* S, const float* dS, int dv, int v4, int d2) {
#pragma unroll
    for (int i = 0; i < DK / 64; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t at = min(v4 + j, dv - 1) * (DK / 2) + i * 32 + d2;
        s[i][j] = *at32<const f2>(S, at);
        d[i][j] = *at32<const f2>(dS, at);
      }
  }
};

template <typename T, int DK, bool W>
__global__ __launch_bounds__(512, 2) void delta_grad_last_kernel(
    const DeltaGradArgs ga, const unsigned char* prep, const float* rec, const float* grec,
    int chunks, uint64_t blocks) {
  constexpr int U = DK / 32, MT = DK / 16, FULL = Mode<T>::FULL, P = Mode<T>::ROWS;
  extern __shared__ __align__(16) unsigned char lds[];
  const DeltaArgs& a = ga.f;
  LastLds<T, DK>& s = *reinterpret_cast<LastLds<T, DK>*>(lds);
  const int group = a.HV / a.H;
  for (uint64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    // what follows from the thread's number is computed here, not kept from
    // before the loop: there are no registers to keep it in
    int all = threadIdx.x;
    asm volatile("" : "+v"(all));
    const bool states = same(all >> 8) != 0;
    const int tid = all & 255, lane = tid & 63, w = same(tid >> 6);
    const int i16 = lane % 16, g = lane / 16, g4 = 4 * g, sl = slot_of(i16, g), own = w * 16 + i16;
    // the wave again, but as a vector: what it decides by selects is no branch
    const int wv = tid >> 6;
    Place p;
    p.c = same((int)(b % chunks));
    const int kh = same((int)(b / chunks % a.H));
    p.l = same((int)(b / chunks / a.H));
    p.n = same(within(seq_len(a.q, p.l), p.c));
    const int rows = min(C, a.q.T - p.c * C);
    if (!p.n) {  // past the lane's length: zero
      for (int i = all; i < rows * group; i += 512) {
        const int64_t t = p.c * C + i / group, h = kh * group + i % group;
        ((float*)ga.dg.d)[p.l * ga.dg.lane + t * ga.dg.row + h] = 0.0f;
        ((float*)ga.dbeta.d)[p.l * ga.dbeta.lane + t * ga.dbeta.row + h] = 0.0f;
      }
      const int wide = group * a.dv;
      for (int i = all; i < rows * wide; i += 512)
        st1(Chunk<T>(ga.dv, p, kh, wide).at(i / wide * (uint32_t)ga.dv.row + i % wide), 0.0f);
      for (int i = all; i < rows * a.dk; i += 512) {
        st1(Chunk<T>(ga.dq, p, kh, a.dk).at(i / a.dk * (uint32_t)ga.dq.row + i % a.dk), 0.0f);
        st1(Chunk<T>(ga.dk, p, kh, a.dk).at(i / a.dk * (uint32_t)ga.dk.row + i % a.dk), 0.0f);
      }
      continue;
    }
    auto across_g = [&](float x) {
      x = fold16(x, x);
      return fold32(x, x);
    };
    // Each four waves have a loop of their own, with as many barriers, so that
    // neither keeps registers for the other.
    if (!states) {
      // K and Q, put twice: as rows, for their products, and across
      Rows4<T> k[DK / 64], q[DK / 64];
      const int kpos = tid / 16 * 4, kcol = tid % 16 * 4;
#pragma unroll
      for (int i = 0; i < DK / 64; ++i) {
        k[i].template load<W>(Chunk<const T>(a.k, p, kh, a.dk), p.n, a.dk, kpos, i * 64 + kcol);
        q[i].template load<W>(Chunk<const T>(a.qr, p, kh, a.dk), p.n, a.dk, kpos, i * 64 + kcol);
      }
      for (int vh = kh * group; vh < (kh + 1) * group; ++vh) {
        p.h = vh;
        const int64_t record = same(((int64_t)p.l * a.HV + vh) * chunks + p.c);
        const float *S = rec + record * (a.dv * (DK + C)), *N = S + a.dv * DK;
        const float *dS = grec + record * (a.dv * (DK + C)), *dR = dS + a.dv * DK;
        const unsigned char* coef = prep + ((record + 1) * PREP_BYTES - COEF * 4);
        const float co0 = *at32<const float>(coef, min(all, COEF - 1));
        const float co1 = *at32<const float>(coef, min(all + 512, COEF - 1));
        __syncthreads();
        reinterpret_cast<float*>(&s.coef)[min(all, COEF - 1)] = co0;
        if (all + 512 < COEF) reinterpret_cast<float*>(&s.coef)[all + 512] = co1;
        // the first two waves take N and dO, the others dR and v
        const int half = w / 2, pg = tid % 16, vg = tid / 16 % 8;
        const float* x_ = half ? dR : N;
        const Chunk<const T> from(half ? a.v : ga.dout, p, vh, a.dv);
        const Chunk<T> out(ga.dv, p, vh, a.dv);
        LastRows<T> next;
        next.template load<W>(x_, from, p.n, a.dv, vg * 4, pg);
        f4 pp[4] = {}, aa[4] = {}, mid_p = ZERO, mid_a = ZERO;
        f4 dots = ZERO;
        for (int v0 = 0; v0 < a.dv; v0 += 32) {
          const int v4 = v0 + vg * 4;
          __syncthreads();
#pragma unroll
          for (int i = 0; i < 4; ++i) next.x.v[i] = either(v4 + i < a.dv, next.x.v[i], ZERO);
          const Four xt = turned(next.x);  // rows: positions
          next.rows.template cut<W>(p.n - pg * 4, a.dv - v4);
          put_full<T>(half ? s.v.r : s.v.n, 1, pg * 4, vg * 4, xt);
          if (half) {
            // dV, and dR . v
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const f4 d = xt.v[i] * next.rows.r[i].value();
              dots[i] += d[0] + d[1] + d[2] + d[3];
              const int pos = pg * 4 + i;
              if (pos < rows)
                st4<T, W>(out.at(pos * out.row), v4, a.dv,
                          pos < p.n ? xt.v[i] * s.coef.beta[pos] : ZERO);
            }
          } else {
            next.rows.put(s.v.o, 1, pg * 4, vg * 4);
          }
          __syncthreads();
          apart();
          if (v0 + 32 < a.dv) next.template load<W>(x_, from, p.n, a.dv, v4 + 32, pg);
          const Frag<FULL> no = get<FULL>(s.v.n, w, sl), ro = get<FULL>(s.v.r, w, sl);
          const Frag<P> oo = get<P>(s.v.o, w, sl);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            // N of tile m with dO and dR of own, or dO and dR of tile m with N of own
            mma<T>(aa[m], get<FULL>(m <= w ? s.v.n : s.v.r, m, sl), either(m <= wv, ro, no));
            if constexpr (P == FULL) {
              mma<T>(pp[m], get<P>(m <= w ? s.v.n : s.v.o, m, sl), either(m <= wv, oo, no));
            } else {
              // one part of dO, three of N, whichever is on the left: the small first
#pragma unroll
              for (int i = FULL - 1; i >= 0; --i) {
                Frag<1> x, y;
                x.p[0] = *((m <= w ? s.v.n + (m * FULL + i) * 64 : s.v.o + m * 64) + slot_in(m, sl));
#pragma unroll
                for (int j = 0; j < 4; ++j) y.p[0][j] = m <= wv ? oo.p[0][j] : no.p[i][j];
                mma<T>(pp[m], x, y);
              }
            }
            apart();
          }
          mma<T>(mid_p, oo, no);
          mma<T>(mid_a, ro, no);
        }
        if (half) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s.dot[vg][pg * 4 + i] = dots[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < DK / 64; ++i) {
          if (vh == kh * group) {
            k[i].template cut<W>(p.n - kpos, a.dk - i * 64 - kcol);
            q[i].template cut<W>(p.n - kpos, a.dk - i * 64 - kcol);
          }
          k[i].put(s.k.a, U, kpos, i * 64 + kcol);
          q[i].put(s.k.b, U, kpos, i * 64 + kcol);
        }
        __syncthreads();
        // kk: rows of tile m, column own; qk: m <= w: q of own, k of tile m; m > w: q
        // of tile m, k of own; the wave's own tile has both (mid: the second).  Which
        // it is decides addresses and selects, not branches.
        f4 kk[4] = {}, qk[4] = {}, mid_qk = ZERO;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const Frag<P> kw = get<P>(s.k.a, w * U + u, sl), qw = get<P>(s.k.b, w * U + u, sl);
          mma<T>(mid_qk, qw, kw);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            mma<T>(kk[m], get<P>(s.k.a, m * U + u, sl), kw);
            mma<T>(qk[m], get<P>(m <= w ? s.k.a : s.k.b, m * U + u, sl), either(m <= wv, qw, kw));
          }
          apart();
        }
        // what K and Q are multiplied with; sums over a row of dP P and dA A, over a
        // column, and of dA k.k D
        f4 e[4] = {}, mid_e = ZERO, f[4] = {}, mid_f = ZERO;
        const int whole = s.coef.whole[own];
        const float part = s.coef.part[own], beta = s.coef.beta[own], rk = s.coef.rk[own];
        const float uq = s.coef.uq[own];
        float over = 0.0f, down = 0.0f, with_beta = 0.0f;
        // of the four o = at .. at + 3; row: own is the row and o the column, else the
        // other way.  Of a tile that is not the wave's own all elements count.
        auto elements = [&](int at, bool row, bool whole_tile, f4 p4, f4 a4, f4 q4, f4 k4, f4& eo,
                            f4& fo) {
          const i4 whole4 = *reinterpret_cast<const i4*>(s.coef.whole + at);
          const f4 part4 = *reinterpret_cast<const f4*>(s.coef.part + at);
          const f4 rk4 = *reinterpret_cast<const f4*>(s.coef.rk + at);
          const f4 rq4 = *reinterpret_cast<const f4*>(s.coef.uq + at);
          const f4 b4 = *reinterpret_cast<const f4*>(s.coef.beta + at);
          const f4 of_k = either(row, rk4, rq4) * a.scale, of_b = either(row, f4{beta, beta, beta, beta}, b4);
          // what lies below the diagonal by how much
          const int flip = row ? -1 : 0;
          const float signf = row ? -1.0f : 1.0f;
          const int by = whole_tile ? C : ((at - own) ^ flip) - flip;
          float with_q = 0.0f, with_k = 0.0f, kb = 0.0f;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float d = raised(((whole4[r] - whole) ^ flip) - flip, (part4[r] - part) * signf);
            const int below = by + (r ^ flip) - flip;
            const float dP = below >= 0 ? p4[r] * d : 0.0f;
            const float dA = below > 0 ? -a4[r] * d : 0.0f;
            const float e = dP * of_k[r], f = dA * rk4[r], fk = f * k4[r];
            eo[r] += e;
            fo[r] += f * of_b[r];
            with_q += e * q4[r];
            with_k += fk;
            kb += fk * of_b[r];
          }
          const float both = with_q * (row ? uq : rk) + kb * rk;
          over += row ? both : 0.0f;
          down += row ? 0.0f : both;
          with_beta += row ? with_k * rk : 0.0f;
        };
        const f4 mid_k = one_of(kk, wv);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          elements(m * 16 + g4, m <= wv, m != wv, pp[m], aa[m], qk[m], kk[m], e[m], f[m]);
          apart();
        }
        elements(w * 16 + g4, false, false, mid_p, mid_a, mid_qk, mid_k, mid_e, mid_f);
        over = across_g(over);
        down = across_g(down);
        with_beta = across_g(with_beta);
        if (g == 0) s.dsum[own] = over - down, s.dots[own] = with_beta;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < DK / 64; ++i) {
          k[i].turned().put(s.k.a, 2, i * 64 + kcol, kpos);
          q[i].turned().put(s.k.b, 2, i * 64 + kcol, kpos);
        }
        // e: q's part below (rows j), k's above (rows i); the own tile has both
        f4 ek[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          ek[m] = either(m == wv, mid_e, either(m > wv, e[m], ZERO));
          e[m] = either(m <= wv, e[m], ZERO);
          f[m] += either(m == wv, mid_f, ZERO);
        }
        Frag<FULL> ef[2], kf[2], ff[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          ef[u] = full<T>(e[2 * u], e[2 * u + 1]);
          kf[u] = full<T>(ek[2 * u], ek[2 * u + 1]);
          ff[u] = full<T>(f[2 * u], f[2 * u + 1]);
        }
        __syncthreads();  // K and Q are there, across
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          f4 q0 = ZERO, k0 = ZERO;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const Frag<P> kt = get<P>(s.k.a, m * 2 + u, sl);
            mma<T>(q0, kt, ef[u]);
            mma<T>(k0, kt, ff[u]);
            mma<T>(k0, get<P>(s.k.b, m * 2 + u, sl), kf[u]);
          }
          s.k.states[m][w][lane] = q0;
          s.k.states[MT + m][w][lane] = k0;
          apart();
        }
        __syncthreads();
      }
    } else {
      f4 dq[MT] = {}, dk[MT] = {}, qo[MT], ko[MT];  // the other waves'; qo, ko: own rows of q and k
      for (int vh = kh * group; vh < (kh + 1) * group; ++vh) {
        p.h = vh;
        const int64_t record = same(((int64_t)p.l * a.HV + vh) * chunks + p.c);
        const float *S = rec + record * (a.dv * (DK + C));
        const float* dS = grec + record * (a.dv * (DK + C));
        const unsigned char* coef = prep + ((record + 1) * PREP_BYTES - COEF * 4);
        const float co0 = *at32<const float>(coef, min(all, COEF - 1));
        const float co1 = *at32<const float>(coef, min(all + 512, COEF - 1));
        __syncthreads();
        reinterpret_cast<float*>(&s.coef)[min(all, COEF - 1)] = co0;
        if (all + 512 < COEF) reinterpret_cast<float*>(&s.coef)[all + 512] = co1;
        const int d2 = tid % 32, vg = tid / 32;
        LastStates<DK> next;
        next.load(S, dS, a.dv, vg * 4, d2);
        f4 os[MT] = {}, rs[MT] = {}, ns[MT] = {};
        float tail = 0.0f;
        for (int v0 = 0; v0 < a.dv; v0 += 32) {
          const int v4 = v0 + vg * 4;
          __syncthreads();
          // rows of d_k, columns of d_v along them; and <dS, S>
#pragma unroll
          for (int i = 0; i < DK / 64; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              f4 sv, dv;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                sv[j] = v4 + j < a.dv ? next.s[i][j][r] : 0.0f;
                dv[j] = v4 + j < a.dv ? next.d[i][j][r] : 0.0f;
              }
              const f4 both = sv * dv;
              tail += both[0] + both[1] + both[2] + both[3];
              put<T, FULL>(s.v.s, 1, i * 64 + d2 * 2 + r, vg * 4, sv);
              put<T, FULL>(s.v.d, 1, i * 64 + d2 * 2 + r, vg * 4, dv);
            }
          __syncthreads();
          apart();
          if (v0 + 32 < a.dv) next.load(S, dS, a.dv, v4 + 32, d2);
          const Frag<FULL> no = get<FULL>(s.v.n, w, sl), ro = get<FULL>(s.v.r, w, sl);
          const Frag<P> oo = get<P>(s.v.o, w, sl);
          Frag<FULL> sm = get<FULL>(s.v.s, 0, sl), dm = get<FULL>(s.v.d, 0, sl);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            // the next ones are under way
            Frag<FULL> s1, d1;
            if (m + 1 < MT) s1 = get<FULL>(s.v.s, m + 1, sl), d1 = get<FULL>(s.v.d, m + 1, sl);
            mma<T>(os[m], sm, oo);
            mma<T>(rs[m], sm, ro);
            mma<T>(ns[m], dm, no);
            sm = s1;
            dm = d1;
            apart();
          }
        }
        tail = over64(tail, Sum());
        __syncthreads();
        __syncthreads();  // K and Q are there
#pragma unroll
        for (int u = 0; u < U; ++u) {
          results_of<T>(ko[2 * u], ko[2 * u + 1], get<P>(s.k.a, w * U + u, sl));
          results_of<T>(qo[2 * u], qo[2 * u + 1], get<P>(s.k.b, w * U + u, sl));
        }
        const float beta = s.coef.beta[own], since = s.coef.since[own], left = s.coef.left[own];
        const float rk = s.coef.rk[own], rq = s.coef.uq[own] * a.scale;
        float oq = 0.0f, rsk = 0.0f, nsk = 0.0f;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            oq += os[m][r] * qo[m][r];
            rsk += rs[m][r] * ko[m][r];
            nsk += ns[m][r] * ko[m][r];
          }
          dq[m] += os[m] * (since * a.scale);
          dk[m] += ns[m] * left - rs[m] * (since * beta);
        }
        oq = across_g(oq) * (rq * since);
        rsk = across_g(rsk) * (rk * since);
        nsk = across_g(nsk) * (rk * left);
        if (g == 0) s.from[own] = oq - nsk - rsk * beta;
        const float lasts = over16(nsk, Sum());
        if (lane == 0) s.tail[w] = lasts, s.tail[4 + w] = tail * s.coef.since[C - 1];
        __syncthreads();
        if (g == 0 && own < rows) {
          float x = s.dots[own] - rsk;
#pragma unroll
          for (int i = 0; i < 8; ++i) x += s.dot[i][own];
          ((float*)ga.dbeta.d)[p.l * ga.dbeta.lane + (int64_t)(p.c * C + own) * ga.dbeta.row + vh] =
              own < p.n ? x : 0.0f;
        }
        __syncthreads();
        if (w == 0) {
          // dg: the sums of dG from each position to the chunk's last
          double x = (double)s.dsum[lane] + (double)s.from[lane];
          if (lane == C - 1)
            for (int i = 0; i < 8; ++i) x += (double)s.tail[i];
#pragma unroll
          for (int m = 1; m < C; m *= 2) {
            const double y = __shfl_down(x, m);
            if (lane + m < C) x += y;
          }
          if (lane < rows)
            ((float*)ga.dg.d)[p.l * ga.dg.lane + (int64_t)(p.c * C + lane) * ga.dg.row + vh] =
                lane < p.n ? (float)x : 0.0f;
        }
        __syncthreads();
        // the two parts meet
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          dq[m] += s.k.states[m][w][lane];
          dk[m] += s.k.states[MT + m][w][lane];
        }
      }
      // through the rows' lengths: d = r (d^ - u (u . d^)), u the unit row
      float fq = 0.0f, fk = 0.0f;
      const float rk = s.coef.rk[own], by = s.coef.uq[own];
      if (a.unit) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            fq += dq[m][r] * qo[m][r];
            fk += dk[m][r] * ko[m][r];
          }
        fq = across_g(fq) * by * by;
        fk = across_g(fk) * rk * rk;
      }
      if (own < rows) {
        const bool live = own < p.n;
        const Chunk<T> oq_(ga.dq, p, kh, a.dk), ok_(ga.dk, p, kh, a.dk);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          st4<T, W>(oq_.at(own * oq_.row), m * 16 + g4, a.dk,
                    live ? (dq[m] - qo[m] * fq) * by : ZERO);
          st4<T, W>(ok_.at(own * ok_.row), m * 16 + g4, a.dk,
                    live ? (dk[m] - ko[m] * fk) * rk : ZERO);
        }
      }
    }
    __syncthreads();
  }
}

// ---- few positions, one after the other ------------------------------------
// A block per (lane, value head): 256 threads hold the state, thread (x, y)
// columns 4 x .. 4 x + 3 of rows y + RG i.  With S^T k and S^T q of the state
// before, o = scale (e^g S^T q + beta (k . q) e): one sum over the rows and
// two barriers a position.  Bound by the states, read and written once: 1000 lanes
// of 4 of 64 x 128, one position, 58 us, 4.6 TB/s (a copy: 5.1); 50 where the caches
// hold a part of the states.
template <typename T, int DK, int CX, bool W>
__global__ __launch_bounds__(256) void delta_step_kernel(const DeltaArgs a, uint64_t blocks) {
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
      st[i] = ZERO;
      if (a.state_in && row < a.dk)
        st[i] = ld4<float, W>(a.state_in + state + (int64_t)row * a.dv, 4 * x, a.dv);
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
      const f4 v = ld4<T, W>((const T*)a.v.d + l * a.v.lane + t * a.v.row + (int64_t)h * a.dv, 4 * x,
                             a.dv);
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
      f4 sk = ZERO, sq = ZERO;
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
        st4<float, W>(a.state_out + state + (int64_t)row * a.dv, 4 * x, a.dv, st[i]);
      }
    }
  }
}

// widths that the kernels are built for
int built(int d) { return d <= 64 ? 64 : 128; }
int chunks_of(int T) { return (T + C - 1) / C; }
// S and N of a chunk, dS and dR of it
int64_t record_floats(int dk, int dv) { return (int64_t)dv * (built(dk) + C); }

// Segments of a sequence: as many as keep the two passes (about 5 and 6.5 us a
// chunk) and the chain of the segments (0.75 us each) together shortest, where there
// are CUs for them and they come to three at least.  With and without, us:
//   positions:                      384           512          1024          4096
//   2 of 64 x 64, fp32           37 and 54     38 and 66    44 and 115    69 and 411
//   8 of 128 x 128, bf16         53 and 49     59 and 59    69 and 99    127 and 336
//   32 of 64 x 64, bf16          45 and 42     48 and 51    65 and 86    160 and 280
// so from 8 chunks on, where none is slower.
struct Cut {
  int n, chunks;
};
Cut segments_of(int64_t heads, int chunks, int dk, int dv) {
  const int tiles = (dv + 63) / 64 + built(dk) / 64;
  int64_t n = 1;
  while ((n + 1) * (n + 1) <= 16 * (int64_t)chunks) ++n;
  n = std::min<int64_t>(n, 256 / (heads * tiles));
  if (chunks < 8 || n < 3) return {1, chunks};
  const int each = (int)((chunks + n - 1) / n);
  return {(chunks + each - 1) / each, each};
}
// floats of Segments::local (of the gradient: without the identity's columns) and first
int64_t local_floats(int64_t heads, const Cut& c, int dk, int dv, bool moves) {
  if (c.n == 1) return 0;
  return heads * c.n * ((dv + 63) / 64 * 64 + (moves ? 2 * built(dk) : 0)) * built(dk);
}

// Lanes of different lengths: the chains take the longest first where there are more
// blocks than CUs, so that none starts late (64 x 521, 8 heads of 128 x 128, lengths
// up to that: 145 and 168 us).  `at`: where the order is kept, of lanes' size.
// Each lane is ranked among all of them, which takes what it brings from about 4000
// lanes on and far more beyond.  With and without the order, whole calls of lanes up to
// T long, one head of 64 x 64, bf16, us:
//   lanes:       1000          2000          4000            16,000        65,535
//   T = 100   69 and  69   125 and 120   271 and  249   1,388 and   938   11,763 and 3,779
//   T = 520  184 and 207   355 and 380   721 and  717   3,117 and 2,702
constexpr int ORDER_LANES = 2048;
uint32_t* order_of(const DeltaArgs& a, uint64_t blocks, int chunks, const Cut& cut, void* at) {
  return a.q.lens && cut.n == 1 && chunks > 1 && blocks > 256 && a.q.lanes <= ORDER_LANES
             ? (uint32_t*)at : nullptr;
}

// Positions taken one after the other rather than in chunks: what a position takes
// (1.4 us where few states wait for their rows, 2.5 at 64 lanes of 8 states of 128 x
// 128) against a chunk's three kernels.  Measured, us:
//   positions:                           4             8            16
//   1 lane, 2 of 64 x 64, fp32      10 and 22     14 and 22     25 and 22
//   the same, bf16                  10 and 19     15 and 19     27 and 20
//   64 lanes, 8 of 128 x 128, bf16  22 and 72     32 and 72     52 and 72
//   1000 lanes, 4 of 64 x 128       78 and 455   115 and 457   191 and 459
// T alone decides: what a call needs and whether its bits are those of single steps
// must not depend on the batch, which a server fills as it can.  12 is where few lanes
// break even; many lanes would up to about 40 positions, and pay up to 2.4 times in
// between.
bool by_steps(int T) { return T <= 12; }

template <typename F>
hipError_t for_width(int dk, F&& f) {
  if (built(dk) == 64) return f(std::integral_constant<int, 64>());
  return f(std::integral_constant<int, 128>());
}

template <typename K>
hipError_t room(K kernel, size_t bytes) {
  if (bytes <= 65536) return hipSuccess;
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}
uint32_t grid(uint64_t blocks) { return (uint32_t)std::min<uint64_t>(blocks, MAX_BLOCKS); }

template <typename R>
bool wide_rows(const R& r, int d, int size) {
  return rows_by_16(r.d, r.lane, r.row, d, size);
}

template <typename T, bool W>
hipError_t delta_steps_of(const DeltaArgs& a, hipStream_t s) {
  const uint64_t heads = (uint64_t)a.q.lanes * a.HV;
  auto go = [&](auto kernel) {
    BOA_LAUNCH(kernel, grid(heads), 256, 0, s, a, heads);
    return hipGetLastError();
  };
  if (built(a.dk) == 64)
    return a.dv <= 64 ? go(delta_step_kernel<T, 64, 16, W>) : go(delta_step_kernel<T, 64, 32, W>);
  return a.dv <= 64 ? go(delta_step_kernel<T, 128, 16, W>) : go(delta_step_kernel<T, 128, 32, W>);
}

template <typename T, bool W>
hipError_t delta_of(const DeltaArgs& a, hipStream_t s) {
  const uint64_t heads = (uint64_t)a.q.lanes * a.HV;
  return for_width(a.dk, [&](auto dk) {
    constexpr int DK = dk;
    const int chunks = chunks_of(a.q.T), tiles = (a.dv + 63) / 64;
    unsigned char* prep = (unsigned char*)a.work;
    const uint64_t all = heads * chunks;
    const Cut cut = segments_of(heads, chunks, a.dk, a.dv);
    uint32_t* order = order_of(a, heads * tiles, chunks, cut, prep + all * PREP_BYTES);
    BOA_LAUNCH((delta_prep_kernel<T, DK, false, W>), grid(all), 256, 0, s, a, prep, chunks, order,
               all);
    hipError_t e = hipGetLastError();
    if (e) return e;
    const size_t lds = sizeof(ChainLds<T, DK, false>);
    Segments seg{cut.n, cut.chunks, nullptr, nullptr};
    if (cut.n > 1) {
      seg.first = (float*)(prep + all * PREP_BYTES);
      // where the gradient follows, it needs what the segments make of a state
      seg.local = a.saved ? a.saved + all * record_floats(a.dk, a.dv)
                          : seg.first + local_floats(heads, cut, a.dk, a.dv, false);
      const uint32_t blocks = (uint32_t)(heads * cut.n * (tiles + DK / 64));
      if ((e = room(delta_chain_kernel<T, DK, W, true>, lds))) return e;
      BOA_LAUNCH((delta_chain_kernel<T, DK, W, true>), blocks, 256, lds, s, a,
                 (const unsigned char*)prep, (float*)nullptr, chunks, tiles, seg,
                 (const uint32_t*)nullptr, blocks);
      if ((e = hipGetLastError())) return e;
      const uint32_t columns = (uint32_t)(heads * tiles * 4);
      BOA_LAUNCH((delta_combine_kernel<DK, false>), columns, 256, 0, s, a, a.state_in,
                 (const float*)seg.local, (const float*)seg.local, tiles * 64 + 2 * DK, seg.first,
                 tiles, cut.n, columns);
      if ((e = hipGetLastError())) return e;
    }
    if ((e = room(delta_chain_kernel<T, DK, W, false>, lds))) return e;
    const uint64_t blocks = heads * cut.n * tiles;
    BOA_LAUNCH((delta_chain_kernel<T, DK, W, false>), grid(blocks), 256, lds, s, a,
               (const unsigned char*)prep, a.saved, chunks, tiles, seg,
               (const uint32_t*)order, (uint32_t)blocks);
    return hipGetLastError();
  });
}

template <typename T, bool W>
hipError_t delta_grad_of(const DeltaGradArgs& ga, hipStream_t s) {
  const DeltaArgs& a = ga.f;
  const uint64_t heads = (uint64_t)a.q.lanes * a.HV;
  return for_width(a.dk, [&](auto dk) {
    constexpr int DK = dk;
    const int chunks = chunks_of(a.q.T), tiles = (a.dv + 63) / 64;
    const uint64_t all = heads * chunks;
    unsigned char* prep = (unsigned char*)a.work;
    float* grec = (float*)(prep + all * PREP_BYTES);
    const Cut cut = segments_of(heads, chunks, a.dk, a.dv);
    uint32_t* order =
        order_of(a, heads * tiles, chunks, cut, grec + all * record_floats(a.dk, a.dv));
    BOA_LAUNCH((delta_prep_kernel<T, DK, true, W>), grid(all), 256, 0, s, a, prep, chunks, order,
               all);
    hipError_t e = hipGetLastError();
    if (e) return e;
    size_t lds = sizeof(ChainLds<T, DK, true>);
    Segments seg{cut.n, cut.chunks, nullptr, nullptr};
    if (cut.n > 1) {
      seg.first = grec + all * record_floats(a.dk, a.dv);
      seg.local = seg.first + local_floats(heads, cut, a.dk, a.dv, false);
      const uint32_t blocks = (uint32_t)(heads * cut.n * tiles);
      if ((e = room(delta_grad_chain_kernel<T, DK, W, true>, lds))) return e;
      BOA_LAUNCH((delta_grad_chain_kernel<T, DK, W, true>), blocks, 256, lds, s, ga,
                 (const unsigned char*)prep, grec, chunks, tiles, seg,
                 (const uint32_t*)nullptr, blocks);
      if ((e = hipGetLastError())) return e;
      const uint32_t columns = (uint32_t)(heads * tiles * 4);
      BOA_LAUNCH((delta_combine_kernel<DK, true>), columns, 256, 0, s, a, ga.dstate_out,
                 (const float*)(a.saved + all * record_floats(a.dk, a.dv)), (const float*)seg.local,
                 tiles * 64, seg.first, tiles, cut.n, columns);
      if ((e = hipGetLastError())) return e;
    }
    if ((e = room(delta_grad_chain_kernel<T, DK, W, false>, lds))) return e;
    const uint64_t blocks = heads * cut.n * tiles;
    BOA_LAUNCH((delta_grad_chain_kernel<T, DK, W, false>), grid(blocks), 256, lds, s, ga,
               (const unsigned char*)prep, grec, chunks, tiles, seg,
               (const uint32_t*)order, (uint32_t)blocks);
    if ((e = hipGetLastError())) return e;
    lds = sizeof(LastLds<T, DK>);
    if ((e = room(delta_grad_last_kernel<T, DK, W>, lds))) return e;
    const uint64_t last = (uint64_t)a.q.lanes * a.H * chunks;
    BOA_LAUNCH((delta_grad_last_kernel<T, DK, W>), grid(last), 512, lds, s, ga,
               (const unsigned char*)prep, (const float*)a.saved, (const float*)grec, chunks, last);
    return hipGetLastError();
  });
}

// f(row type, whether all rows can be moved 16 bytes at a time)
template <typename F>
hipError_t for_rows(bool bf16, bool wide, F&& f) {
  using std::bool_constant;
  if (bf16) return wide ? f(uint16_t(), bool_constant<true>()) : f(uint16_t(), bool_constant<false>());
  return wide ? f(float(), bool_constant<true>()) : f(float(), bool_constant<false>());
}

}  // namespace

int64_t delta_saved_floats(int lanes, int T, int, int HV, int dk, int dv) {
  const int64_t heads = (int64_t)lanes * HV;
  const int chunks = chunks_of(T);
  return heads * chunks * record_floats(dk, dv) +
         local_floats(heads, segments_of(heads, chunks, dk, dv), dk, dv, true);
}

int64_t delta_work_bytes(int lanes, int T, int, int HV, int dk, int dv, bool grad) {
  if (!grad && by_steps(T)) return 0;
  const int64_t heads = (int64_t)lanes * HV;
  const int chunks = chunks_of(T);
  const Cut cut = segments_of(heads, chunks, dk, dv);
  const int64_t first = local_floats(heads, cut, dk, dv, false);
  // what a forward call needs, and a gradient's as well if it is to be one's
  int64_t floats = first + local_floats(heads, cut, dk, dv, true);
  if (grad) floats = std::max(floats, heads * chunks * record_floats(dk, dv) + 2 * first);
  if (cut.n == 1) floats += std::min((lanes + 3) / 4 * 4, ORDER_LANES);  // the lanes' order
  return heads * chunks * PREP_BYTES + 4 * floats;
}

hipError_t launch_delta(const DeltaArgs& a, hipStream_t s) {
  const int size = a.bf16 ? 2 : 4;
  if (by_steps(a.q.T) && !a.saved) {
    const bool wide = wide_rows(a.v, a.dv, size) && a.dv % 4 == 0;  // states are 16-byte aligned
    return for_rows(a.bf16, wide, [&](auto t, auto w) { return delta_steps_of<decltype(t), w>(a, s); });
  }
  const bool wide = wide_rows(a.qr, a.dk, size) && wide_rows(a.k, a.dk, size) &&
                    wide_rows(a.v, a.dv, size) && wide_rows(a.out, a.dv, size);
  return for_rows(a.bf16, wide, [&](auto t, auto w) { return delta_of<decltype(t), w>(a, s); });
}

hipError_t launch_delta_grad(const DeltaGradArgs& g, hipStream_t s) {
  const DeltaArgs& a = g.f;
  const int size = a.bf16 ? 2 : 4;
  const bool wide = wide_rows(a.qr, a.dk, size) && wide_rows(a.k, a.dk, size) &&
                    wide_rows(a.v, a.dv, size) && wide_rows(g.dout, a.dv, size) &&
                    wide_rows(g.dq, a.dk, size) && wide_rows(g.dk, a.dk, size) &&
                    wide_rows(g.dv, a.dv, size);
  return for_rows(a.bf16, wide, [&](auto t, auto w) { return delta_grad_of<decltype(t), w>(g, s); });
}

}  // namespace boa
