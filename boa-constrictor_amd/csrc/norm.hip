// Root-mean-square norm of rows with the residual's addition before it and an
// output in 8 bits after it, its gradient, and rows in 8 bits without a norm.
//
//   h = x + residual          r = 1 / sqrt(mean h^2 + eps)      y = h r w
//   in 8 bits: t = h w, top = max |t|, q = rint(127 t / top), scale = top r / 127
// so q does not depend on r.  t and q are computed in 64 bits: a value next to
// the border of two steps goes to the side that the formula puts it on.
//   dh = r (w dy - n mean(n w dy)) + dsum,  n = h r;      dw = sum of rows dy n
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

// sums and greatest values over the G threads of a row, in every one of them;
// rows of a block's 256 threads pass through `part`
template <int G, typename F, typename X>
__device__ __forceinline__ X row_all(X x, F f, X* part) {
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
struct Add {
  template <typename X> __device__ X operator()(X a, X b) const { return a + b; }
};
struct Most {  // NaN wins
  __device__ double operator()(double a, double b) const {
    return a != a ? a : (b > a || b != b ? b : a);
  }
};

template <typename T, int V, int G, int U, bool OUT8>
__global__ __launch_bounds__(256) void norm_kernel(const NormArgs a, uint32_t rows) {
  __shared__ double part[4];
  constexpr int R = 256 / G;  // rows of a block
  const int g = threadIdx.x % G;
  const uint32_t len = a.q.T;
  for (uint64_t b = (uint64_t)blockIdx.x * R; b < rows; b += (uint64_t)gridDim.x * R) {
    const uint64_t r = b + threadIdx.x / G;
    const uint32_t l = r < rows ? (uint32_t)r / len : 0, t = r < rows ? (uint32_t)r - l * len : 0;
    const bool live = r < rows && (int)t < seq_len(a.q, l);
    const T* x = (const T*)a.x.d + l * a.x.lane + t * a.x.row;
    const T* res = a.res.d ? (const T*)a.res.d + l * a.res.lane + t * a.res.row : nullptr;
    float h[U][V], hr[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (u * G + g) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) h[u][j] = hr[u][j] = 0.0f;
      if (live && i < a.width) {
        load_row<V>(x + i, h[u]);
        if (res) load_row<V>(res + i, hr[u]);
      }
    }
    float ss = 0.0f;
    if (a.norm) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float s = h[u][j] + hr[u][j];
          ss += s * s;
        }
      ss = row_all<G>(ss, Add(), (float*)part);
    }
    const float rn = a.norm ? 1.0f / __builtin_sqrtf(ss / (float)a.width + a.eps) : 1.0f;
    if (a.sum.d && live) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = (u * G + g) * V;
        float s[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = h[u][j] + hr[u][j];
        if (i < a.width) store_row<V>((T*)a.sum.d + l * a.sum.lane + t * a.sum.row + i, s);
      }
    }
    if (a.out.d && live) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = (u * G + g) * V;
        if (i < a.width) {
          float y[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            y[j] = (h[u][j] + hr[u][j]) * rn;
            if (a.weight) y[j] *= a.weight[i + j];
          }
          store_row<V>((T*)a.out.d + l * a.out.lane + t * a.out.row + i, y);
        }
      }
    }
    if constexpr (OUT8) {
      double top = 0.0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = (u * G + g) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          double v = (double)h[u][j] + (double)hr[u][j];
          if (a.weight && i < a.width) v *= (double)a.weight[i + j];
          top = Most()(top, __builtin_fabs(v));
        }
      }
      top = row_all<G>(top, Most(), part);
      const double step = top > 0.0 ? 127.0 / top : 0.0;
      if (live) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = (u * G + g) * V;
          if (i < a.width) {
            int8_t q[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
              double v = (double)h[u][j] + (double)hr[u][j];
              if (a.weight) v *= (double)a.weight[i + j];
              // (where the product may be on the other side of a border, the quotient)
              double f = v * step;
              if (__builtin_fabs(f - __builtin_rint(f)) > 0.5 - 1e-9) f = v * 127.0 / top;
              q[j] = (int8_t)(int)__builtin_rint(f);
            }
            int8_t* o = (int8_t*)a.out8.d + l * a.out8.lane + t * a.out8.row + i;
            if constexpr (V == 4) {
              uint32_t w = 0;
#pragma unroll
              for (int j = 0; j < 4; ++j) w |= (uint32_t)(uint8_t)q[j] << (8 * j);
              *reinterpret_cast<uint32_t*>(o) = w;
            } else if constexpr (V == 8) {
              uint32_t w[2] = {0, 0};
#pragma unroll
              for (int j = 0; j < 8; ++j) w[j / 4] |= (uint32_t)(uint8_t)q[j] << (8 * (j % 4));
              *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1]);
            } else {
              o[0] = q[0];
            }
          }
        }
        if (g == 0) a.scale8[r] = (float)(top * (double)rn / 127.0);
      }
    }
  }
}

template <typename T, int V, int G, int U>
__global__ __launch_bounds__(256) void norm_grad_kernel(const NormGradArgs a, uint32_t rows) {
  __shared__ float part[4];
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
    float ss = 0.0f, c = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (u * G + g) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) h[u][j] = dy[u][j] = ds[u][j] = 0.0f;
      if (live && i < a.width) {
        load_row<V>(hp + i, h[u]);
        load_row<V>(dp + i, dy[u]);
        if (sp) load_row<V>(sp + i, ds[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        ss += h[u][j] * h[u][j];
        c += h[u][j] * (w[u][j] * dy[u][j]);
      }
    ss = row_all<G>(ss, Add(), part);
    c = row_all<G>(c, Add(), part);
    const float rn = 1.0f / __builtin_sqrtf(ss / (float)a.width + a.eps);
    const float m = c * rn / (float)a.width;  // mean of n w dy
    if (there) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = (u * G + g) * V;
        float dx[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float n = h[u][j] * rn;
          if (live) dw[u][j] += dy[u][j] * n;
          dx[j] = live ? rn * (w[u][j] * dy[u][j] - n * m) + ds[u][j] : 0.0f;
        }
        if (i < a.width) store_row<V>((T*)a.dx.d + l * a.dx.lane + t * a.dx.row + i, dx);
      }
    }
  }
  if (!a.dweight) return;
  // the block's rows of partial sums, one for each of its R row groups
  float* out = (float*)a.work + ((size_t)blockIdx.x * R + threadIdx.x / G) * a.width;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = (u * G + g) * V + j;
      if (i < a.width) out[i] = dw[u][j];
    }
}

// dweight[i] = sum of n partial rows, in an order that the sizes decide
__global__ __launch_bounds__(1024) void norm_dweight_kernel(const float* part, int n, int width,
                                                            float* dweight) {
  __shared__ float sum[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x % 32, first = threadIdx.x / 32;
  float s = 0.0f;
  if (col < width)
    for (int k = first; k < n; k += 32) s += part[(size_t)k * width + col];
  sum[first][threadIdx.x % 32] = s;
  __syncthreads();
  if (threadIdx.x < 32 && col < width) {
    s = 0.0f;
    for (int k = 0; k < 32; ++k) s += sum[k][threadIdx.x];
    dweight[col] = s;
  }
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
    const uint32_t blocks = std::min<uint32_t>(((uint64_t)rows * G + 255) / 256, MAX_BLOCKS);
    if (a.out8.d)
      BOA_LAUNCH((norm_kernel<T, V, G, U, true>), blocks, 256, 0, s, a, rows);
    else
      BOA_LAUNCH((norm_kernel<T, V, G, U, false>), blocks, 256, 0, s, a, rows);
  };
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

// Blocks of the gradient: as many as the CUs hold at eight waves a SIMD, each
// with its own partial sums
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
  BOA_LAUNCH(norm_dweight_kernel, (a.width + 31) / 32, 1024, 0, s, (const float*)a.work,
             (int)(blocks * (256 / sh.G)), a.width, a.dweight);
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
    n = std::max<int64_t>(n, (int64_t)grad_blocks(rows, sh.G) * (256 / sh.G));
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
