// Root-mean-square norm of rows with the residual's addition before it and an
// output in 8 bits after it, its gradient, and rows in 8 bits without a norm.
//
//   h = x + residual          r = 1 / sqrt(mean h^2 + eps)      y = h r w
//   in 8 bits: t = h w, top = max |t|, q = rint(127 t / top), scale = top r / 127
// so q does not depend on r.  t and q are computed in 64 bits: a value next to
// the border of two steps goes to the side that the formula puts it on.
//   dh = r (w dy - n mean(n w dy)) + dsum,  n = h r;      dw = sum of rows dy n
// Sums are in fp32; where squares of a row would leave its range, they are taken
// again from the row times a power of two.
//
// All of it is bound by the rows' bytes: a row is read once, held in registers
// by G threads of U vectors each (16 bytes a vector, or single elements where
// the rows are not aligned), and written once.
#include <algorithm>

#include "predictor_ops.h"

namespace boa {

namespace {

template <typename T> constexpr int vec_of = 16 / sizeof(T);

template <int V, typename T>
__device__ __forceinline__ void load_row(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    if constexpr (sizeof(T) == 4) v[0] = *p;
    else v[0] = bf16_to_f32(*p);
  } else if constexpr (V == 4) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  } else {
    const uint4 t = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = u2f(w[i] << 16);
      v[2 * i + 1] = u2f(w[i] & 0xFFFF0000u);
    }
  }
}
template <int V, typename T>
__device__ __forceinline__ void store_row(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    if constexpr (sizeof(T) == 4) *p = v[0];
    else *p = f32_to_bf16(v[0]);
  } else if constexpr (V == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]),
                                              bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7]));
  }
}

// where thread g's u-th vector of a row is read
template <int V, int G>
__device__ __forceinline__ int column(int u, int g, int width) {
  const int i = (u * G + g) * V;
  return i < width ? i : 0;
}

// x over the G threads of a row, in every one of them; a row of a block's 256
// threads passes through `part`
template <int G, typename F>
__device__ __forceinline__ float row_all(float x, F f, float* part) {
  x = G == 16 ? over16(x, f) : over64(x, f);
  if constexpr (G == 256) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = f(f(part[0], part[1]), f(part[2], part[3]));
  }
  return x;
}
template <int G, typename F>
__device__ __forceinline__ double row_all64(double x, F f, double* part) {
#pragma unroll
  for (int m = 1; m < (G < 64 ? G : 64); m *= 2) x = f(x, __shfl_xor(x, m));
  if constexpr (G == 256) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = f(f(part[0], part[1]), f(part[2], part[3]));
  }
  return x;
}
struct Most {  // NaN wins
  template <typename X>
  __device__ X operator()(X a, X b) const { return a != a ? a : (b > a || b != b ? b : a); }
};

// A row's r: n = h r, where h may have been multiplied by a power of two, and what
// the formula has r before is multiplied by `first` and by `second`, of which no
// product leaves fp32's range before the result does.
struct Root {
  float r, first, second;
};
// From the mean of h^2 plus eps as it is.  From LEAST on, squares below the least
// normal number are off by less than 2^-40 of it; up to MOST no sum of 8192 of them
// overflows.  Else scale(f) multiplies the row by f, and squares() sums it again (a
// NaN goes either way): what f = 2^-71 takes from small elements is under 2^-129 of n.
template <int G, typename S, typename F>
__device__ __forceinline__ Root root_of(float mean, const S& scale, const F& squares, int width,
                                        float eps, float* part) {
  constexpr float LEAST = 0x1p-110f, MOST = 0x1p100f;
  // a branch for the wave, whose other rows are multiplied by one: a divergent one
  // takes registers for h twice
  Root rn = {1.0f / __builtin_sqrtf(mean), 1.0f, 1.0f};
  const bool small = mean < LEAST, within = mean >= LEAST && mean < MOST;
  if (__any(!within)) {
    const float f = within ? 1.0f : small ? 0x1p90f : 0x1p-71f;
    scale(f);
    rn.r = 1.0f / __builtin_sqrtf(row_all<G>(squares(), Sum(), part) / (float)width + eps * f * f);
    if (!within) rn.first = small ? 0x1p45f : 0x1p-35f, rn.second = small ? 0x1p45f : 0x1p-36f;
  }
  rn.first *= rn.r;
  return rn;
}

// 127 t / top to the nearest whole number.  f is the quotient in fp32, off by
// under 5e-5 (h, t, the step and the product are rounded, 127 being the most);
// where that leaves the number open, t and the product are taken in 64 bits, and
// next to a border the quotient itself.
__device__ __forceinline__ int step_of(float f, float x, float res, float w, double top,
                                       double step) {
  const float r = __builtin_rintf(f);
  if (__builtin_fabsf(f - r) <= 0.5f - 1e-4f) return (int)r;
  const double t = ((double)x + (double)res) * (double)w;
  double q = t * step;
  if (__builtin_fabs(q - __builtin_rint(q)) > 0.5 - 1e-9) q = t * 127.0 / top;
  return (int)__builtin_rint(q);
}

// G threads a row, which stays in registers from the sums to the results, so each
// row is read once.  Bound by the bytes: 65,000 of 130,250 x 256 fp32 rows, two in
// and two out, 53 us (5.0 TB/s); 33,360 x 512 bf16 rows with a sum and 8 bits, 36 us
// (3.3 TB/s), 21 without the 8 bits: 480 vector instructions a row are issued 0.6 of
// the time.
// (The bound: 64 registers and eight waves a SIMD for two vectors of bf16; left to
// itself the compiler takes 66, and 39,000 x 256 rows 24 us and not 21.)
template <typename T, int V, int G, int U, bool OUT8>
__global__ __launch_bounds__(256, !OUT8 && V == 8 && U == 2 ? 8 : 1) void norm_kernel(
    const NormArgs a, uint32_t rows) {
  __shared__ double part[4];
  constexpr int R = 256 / G;  // rows of a block
  // over 8192 columns: rows in 8 bits and nothing else, so neither weights nor a
  // residual take registers
  constexpr bool PLAIN = G * U * V > 8192;
  const int g = threadIdx.x % G;
  const uint32_t len = a.q.T;
  float w[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = (u * G + g) * V + j;
      w[u][j] = PLAIN ? 1.0f : i < a.width ? (a.weight ? a.weight[i] : 1.0f) : 0.0f;
    }
  for (uint64_t b = (uint64_t)blockIdx.x * R; b < rows; b += (uint64_t)gridDim.x * R) {
    const uint64_t r = b + threadIdx.x / G;
    const uint32_t l = r < rows ? (uint32_t)r / len : 0, t = r < rows ? (uint32_t)r - l * len : 0;
    const bool live = r < rows && (int)t < seq_len(a.q, l);
    const T* x = (const T*)a.x.d + l * a.x.lane + t * a.x.row;
    const T* res = !PLAIN && a.res.d ? (const T*)a.res.d + l * a.res.lane + t * a.res.row : nullptr;
    float h[U][V], hr[U][V];
    // no branch between a row's loads, each of which would wait for the last:
    // threads past its end read its first elements
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) h[u][j] = hr[u][j] = 0.0f;
    if (live) {
#pragma unroll
      for (int u = 0; u < U; ++u) load_row<V>(x + column<V, G>(u, g, a.width), h[u]);
      if (res)
#pragma unroll
        for (int u = 0; u < U; ++u) load_row<V>(res + column<V, G>(u, g, a.width), hr[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if ((u * G + g) * V >= a.width) h[u][j] = hr[u][j] = 0.0f;
    // only rows in 8 bits need x and the residual for themselves
    if constexpr (!OUT8) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) h[u][j] += hr[u][j];
    }
    auto sum = [&](int u, int j) { return OUT8 ? h[u][j] + hr[u][j] : h[u][j]; };
    auto squares = [&] {
      float ss = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) ss += sum(u, j) * sum(u, j);
      return ss;
    };
    float mean = 0.0f, rn = 1.0f;
    if (!PLAIN && a.norm) mean = row_all<G>(squares(), Sum(), (float*)part) / (float)a.width + a.eps;
    if (!PLAIN && a.sum.d && live) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = (u * G + g) * V;
        float s[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = sum(u, j);
        if (i < a.width) store_row<V>((T*)a.sum.d + l * a.sum.lane + t * a.sum.row + i, s);
      }
    }
    if (!PLAIN && a.norm)
      rn = root_of<G>(mean, [&](float f) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < V; ++j) h[u][j] *= f, OUT8 ? hr[u][j] *= f : 0.0f;
      }, squares, a.width, a.eps, (float*)part).r;
    if (!PLAIN && a.out.d && live) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = (u * G + g) * V;
        if (i < a.width) {
          float y[V];
#pragma unroll
          for (int j = 0; j < V; ++j) y[j] = sum(u, j) * rn * w[u][j];
          store_row<V>((T*)a.out.d + l * a.out.lane + t * a.out.row + i, y);
        }
      }
    }
    if constexpr (OUT8) {
      float most = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j)
          most = Most()(most, __builtin_fabsf(sum(u, j) * w[u][j]));
      most = row_all<G>(most, Most(), (float*)part);
      // the greatest in 64 bits is among those next to the greatest in fp32
      // (all of them, where fp32 has few digits left or none)
      const float near = most < 1e-30f || !(most < __builtin_inff()) ? 0.0f : most * (1.0f - 0x1p-21f);
      double top = 0.0;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (!(__builtin_fabsf((h[u][j] + hr[u][j]) * w[u][j]) < near))
            top = Most()(top, __builtin_fabs(((double)h[u][j] + (double)hr[u][j]) * (double)w[u][j]));
      top = row_all64<G>(top, Most(), part);
      const double step = top > 0.0 ? 127.0 / top : 0.0;
      const float step32 = near > 0.0f ? (float)step : __builtin_nanf("");  // NaN: all in 64 bits
      if (live) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = (u * G + g) * V;
          if (i < a.width) {
            int q[V];
#pragma unroll
            for (int j = 0; j < V; ++j)
              q[j] = top > 0.0 ? step_of((h[u][j] + hr[u][j]) * w[u][j] * step32, h[u][j], hr[u][j],
                                         w[u][j], top, step)
                               : 0;
            int8_t* o = (int8_t*)a.out8.d + l * a.out8.lane + t * a.out8.row + i;
            if constexpr (V >= 4) {
              uint32_t p[V / 4] = {};
#pragma unroll
              for (int j = 0; j < V; ++j) p[j / 4] |= (uint32_t)(q[j] & 255) << (8 * (j % 4));
              if constexpr (V == 4) *reinterpret_cast<uint32_t*>(o) = p[0];
              else *reinterpret_cast<uint2*>(o) = make_uint2(p[0], p[1]);
            } else {
              o[0] = (int8_t)q[0];
            }
          }
        }
        if (g == 0) a.scale8[r] = (float)(top * (double)rn / 127.0);
      }
    }
  }
}

// As above; what a row adds to dweight stays in registers over the block's rows,
// and the blocks' sums are added in order by norm_dweight_kernel.  130,250 x 256
// fp32 rows, half of them past their lane's length, 77 us (4.3 TB/s).
template <typename T, int V, int G, int U>
__global__ __launch_bounds__(256) void norm_grad_kernel(const NormGradArgs a, uint32_t rows) {
  __shared__ float part[4];
  __shared__ float group[U * V * 256];  // partial sums of the block's row groups
  constexpr int R = 256 / G;
  const int g = threadIdx.x % G;
  const uint32_t len = a.q.T;
  float w[U][V], dw[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = (u * G + g) * V + j;
      w[u][j] = i < a.width ? (a.weight ? a.weight[i] : 1.0f) : 0.0f;
      dw[u][j] = 0.0f;
    }
  for (uint64_t b = (uint64_t)blockIdx.x * R; b < rows; b += (uint64_t)gridDim.x * R) {
    const uint64_t r = b + threadIdx.x / G;
    const bool there = r < rows;
    const uint32_t l = there ? (uint32_t)r / len : 0, t = there ? (uint32_t)r - l * len : 0;
    const bool live = there && (int)t < seq_len(a.q, l);
    float h[U][V], dy[U][V], ds[U][V];
    const T* hp = (const T*)a.h.d + l * a.h.lane + t * a.h.row;
    const T* dp = (const T*)a.dout.d + l * a.dout.lane + t * a.dout.row;
    const T* sp = a.dsum.d ? (const T*)a.dsum.d + l * a.dsum.lane + t * a.dsum.row : nullptr;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) h[u][j] = dy[u][j] = ds[u][j] = 0.0f;
    if (live) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        load_row<V>(hp + column<V, G>(u, g, a.width), h[u]);
        load_row<V>(dp + column<V, G>(u, g, a.width), dy[u]);
      }
      if (sp)
#pragma unroll
        for (int u = 0; u < U; ++u) load_row<V>(sp + column<V, G>(u, g, a.width), ds[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if ((u * G + g) * V >= a.width) h[u][j] = dy[u][j] = 0.0f;
    auto squares = [&] {
      float ss = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) ss += h[u][j] * h[u][j];
      return ss;
    };
    const float mean = row_all<G>(squares(), Sum(), part) / (float)a.width + a.eps;
    float c = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) c += h[u][j] * (w[u][j] * dy[u][j]);
    c = row_all<G>(c, Sum(), part);
    const Root rn = root_of<G>(mean, [&](float f) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) h[u][j] *= f;
    }, squares, a.width, a.eps, part);
    // the mean of n w dy: r taken out of the sum, unless its terms or their sum
    // leave fp32's range
    const float cr = c * rn.r;
    float m = cr / (float)a.width;
    const bool within = rn.second == 1.0f && __builtin_fabsf(c) >= 0x1p-100f &&
                        __builtin_fabsf(cr) >= 0x1p-110f && __builtin_fabsf(cr) < 0x1p120f;
    if (__any(live && !within)) {
      c = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) c += h[u][j] * (rn.r * w[u][j]) * dy[u][j];
      c = row_all<G>(c, Sum(), part) / (float)a.width;
      if (!within) m = c;
    }
    if (there) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = (u * G + g) * V;
        float dx[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float n = h[u][j] * rn.r;
          if (live) dw[u][j] += dy[u][j] * n;
          const float d = rn.first * (w[u][j] * dy[u][j] - n * m) * rn.second;
          dx[j] = live ? d + ds[u][j] : 0.0f;
        }
        if (i < a.width) store_row<V>((T*)a.dx.d + l * a.dx.lane + t * a.dx.row + i, dx);
      }
    }
  }
  if (!a.dweight) return;
  // the block's sums: of its R row groups, in order
  float* out = (float*)a.work + (size_t)blockIdx.x * a.width;
  constexpr int N = U * V * G;  // elements of a row, padded
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < V; ++j) group[threadIdx.x / G * N + (u * G + g) * V + j] = dw[u][j];
  __syncthreads();
  for (int i = threadIdx.x; i < a.width; i += 256) {
    float s = group[i];
    for (int k = 1; k < R; ++k) s += group[k * N + i];
    out[i] = s;
  }
}

// dweight[i] = sum of n partial rows in 64 bits, in an order that the sizes
// decide: eight columns a block, so that few blocks do not sum it all
__global__ __launch_bounds__(1024) void norm_dweight_kernel(const float* part, int n, int width,
                                                            float* dweight) {
  __shared__ double sum[128][9];
  const int c = threadIdx.x % 8, col = blockIdx.x * 8 + c, first = threadIdx.x / 8;
  double s = 0.0;
  if (col < width) {
#pragma unroll 8
    for (int k = first; k < n; k += 128) s += (double)part[(size_t)k * width + col];
  }
  sum[first][c] = s;
  __syncthreads();
#pragma unroll
  for (int m = 64; m; m /= 2) {
    if (first < m) sum[first][c] += sum[first + m][c];
    __syncthreads();
  }
  if (threadIdx.x < 8 && col < width) dweight[col] = (float)sum[0][c];
}

// Threads and vectors of a row: a row of nv vectors takes 16 threads up to 32
// of them (four rows a wave), a wave up to 256, a block beyond.
struct Shape {
  int G, U;
};
Shape shape_of(int nv) {
  if (nv <= 16) return {16, 1};
  if (nv <= 32) return {16, 2};
  if (nv <= 64) return {64, 1};
  if (nv <= 128) return {64, 2};
  if (nv <= 256) return {64, 4};
  if (nv <= 1024) return {256, 4};
  if (nv <= 2048) return {256, 8};
  return {256, 32};
}

template <typename F>
void for_shape(const Shape& s, F&& f) {
#define BOA_SHAPE(g, u) \
  if (s.G == g && s.U == u) return f(std::integral_constant<int, g>(), std::integral_constant<int, u>())
  BOA_SHAPE(16, 1);
  BOA_SHAPE(16, 2);
  BOA_SHAPE(64, 1);
  BOA_SHAPE(64, 2);
  BOA_SHAPE(64, 4);
  BOA_SHAPE(256, 4);
  BOA_SHAPE(256, 8);
#undef BOA_SHAPE
}

template <typename T, int V>
hipError_t norm_of(const NormArgs& a, hipStream_t s) {
  const uint32_t rows = (uint32_t)a.q.lanes * (uint32_t)a.q.T;
  auto go = [&](auto G, auto U) {
    // eight blocks a CU, which keep the weight in registers from row to row
    const uint32_t blocks = std::min<uint32_t>(((uint64_t)rows * G + 255) / 256, 2048);
    if constexpr (G * U * V <= 8192)
      if (!a.out8.d) {
        BOA_LAUNCH((norm_kernel<T, V, G, U, false>), blocks, 256, 0, s, a, rows);
        return;
      }
    BOA_LAUNCH((norm_kernel<T, V, G, U, true>), blocks, 256, 0, s, a, rows);
  };
  // rows in 8 bits without a norm may be as wide as the product takes them, 16384
  if (a.width > 8192) {
    go(std::integral_constant<int, 256>(), std::integral_constant<int, 64 / V>());
    return hipGetLastError();
  }
  const Shape sh = shape_of((a.width + V - 1) / V);
  if constexpr (V == 1) {
    if (sh.U == 32) {
      go(std::integral_constant<int, 256>(), std::integral_constant<int, 32>());
      return hipGetLastError();
    }
  }
  for_shape(sh, go);
  return hipGetLastError();
}

// Blocks of the gradient, each with its own partial sums: with 512, 1024, 2048 of
// them 79, 61, 57 us (130,250 x 256, fp32), 13, 15, 22 (8103 x 512, bf16) and 40,
// 39, 44 (32,768 x 1024, bf16), all without dsum and with h as dout, too: 1024 is
// never far from the best
constexpr uint32_t GRAD_BLOCKS = 1024;
uint32_t grad_blocks(int64_t rows, int G) {
  return (uint32_t)std::min<int64_t>((rows * G + 255) / 256, GRAD_BLOCKS);
}

template <typename T, int V>
hipError_t norm_grad_of(const NormGradArgs& a, hipStream_t s) {
  const uint32_t rows = (uint32_t)a.q.lanes * (uint32_t)a.q.T;
  const Shape sh = shape_of((a.width + V - 1) / V);
  const uint32_t blocks = grad_blocks(rows, sh.G);
  auto go = [&](auto G, auto U) {
    BOA_LAUNCH((norm_grad_kernel<T, V, G, U>), blocks, 256, 0, s, a, rows);
  };
  bool done = false;
  if constexpr (V == 1) {
    if (sh.U == 32) {
      go(std::integral_constant<int, 256>(), std::integral_constant<int, 32>());
      done = true;
    }
  }
  if (!done) for_shape(sh, go);
  hipError_t e = hipGetLastError();
  if (e || !a.dweight) return e;
  BOA_LAUNCH(norm_dweight_kernel, (a.width + 7) / 8, 1024, 0, s, (const float*)a.work,
             (int)blocks, a.width, a.dweight);
  return hipGetLastError();
}

bool by_16(const RowsIn& r, int width, int size) {
  return !r.d || rows_by_16(r.d, r.lane, r.row, width, size);
}
bool by_16(const RowsOut& r, int width, int size) {
  return !r.d || rows_by_16(r.d, r.lane, r.row, width, size);
}

}  // namespace

hipError_t launch_norm(const NormArgs& a, hipStream_t s) {
  const int size = a.bf16 ? 2 : 4, v = 16 / size;
  const bool wide = by_16(a.x, a.width, size) && by_16(a.res, a.width, size) &&
                    by_16(a.sum, a.width, size) && by_16(a.out, a.width, size) &&
                    (!a.out8.d || ((uintptr_t)a.out8.d % v == 0 && a.out8.lane % v == 0 &&
                                   a.out8.row % v == 0));
  if (a.bf16) return wide ? norm_of<uint16_t, 8>(a, s) : norm_of<uint16_t, 1>(a, s);
  return wide ? norm_of<float, 4>(a, s) : norm_of<float, 1>(a, s);
}

size_t norm_grad_work(int64_t rows, int width) {
  // the most partial rows of either vector width
  int64_t n = 0;
  for (int v : {1, 4, 8}) {
    const Shape sh = shape_of((width + v - 1) / v);
    n = std::max<int64_t>(n, grad_blocks(rows, sh.G));
  }
  return (size_t)n * width * 4;
}

hipError_t launch_norm_grad(const NormGradArgs& a, hipStream_t s) {
  const int size = a.bf16 ? 2 : 4;
  const bool wide = by_16(a.h, a.width, size) && by_16(a.dout, a.width, size) &&
                    by_16(a.dsum, a.width, size) && by_16(a.dx, a.width, size);
  if (a.bf16) return wide ? norm_grad_of<uint16_t, 8>(a, s) : norm_grad_of<uint16_t, 1>(a, s);
  return wide ? norm_grad_of<float, 4>(a, s) : norm_grad_of<float, 1>(a, s);
}

}  // namespace boa
