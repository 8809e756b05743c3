// Product of rows in 8 bits with weights in 8 bits:
//   out[r][n] = xscale[r] wscale[n] sum_k x[r][k] w[n][k] + bias[n]
// The sums are integers in 32 bits (K at most 16384), so they do not depend on
// the order, the tile or the batch: a lane's results are the same bits however
// many lanes run beside it.  The two scales' product, its product with the sum
// and the bias's addition are rounded in fp32, then once to the row type.
#include <algorithm>

#include "predictor_ops.h"

namespace boa {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// Weights as the 32x32x32 MFMA takes them: of every 32 channels, for every 32
// of K, lane i's 16 bytes are channel i % 32, k = 16 (i / 32) ..; channels are
// padded to 128, K to 64, with zeros.
constexpr int N_PAD = 128, K_PAD = 64;
int padded(int n, int to) { return (n + to - 1) / to * to; }

__global__ __launch_bounds__(256) void int8_pack_kernel(const int8_t* w, int N, int K, int ksteps,
                                                        uint32_t pieces, uint4* packed) {
  for (uint32_t p = blockIdx.x * 256 + threadIdx.x; p < pieces; p += gridDim.x * 256) {
    const uint32_t lane = p % 64, step = p / 64 % ksteps, tile = p / 64 / ksteps;
    const int n = tile * 32 + lane % 32, k0 = step * 32 + lane / 32 * 16;
    uint32_t v[4] = {0, 0, 0, 0};
    if (n < N) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (k0 + i < K) v[i / 4] |= (uint32_t)(uint8_t)w[(size_t)n * K + k0 + i] << (8 * (i % 4));
    }
    packed[p] = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

// 16 bytes of a row from k on, zero past K; by single bytes unless `wide`
__device__ __forceinline__ uint4 row16(const int8_t* row, int k, int K, bool wide) {
  if (wide && k + 16 <= K) return *reinterpret_cast<const uint4*>(row + k);
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (k + i < K) v[i / 4] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i % 4));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// A block of four waves computes BM rows x BN channels, a wave WM x WN of them
// in tiles of 32 x 32.  Rows pass through LDS in steps of 64 of K, two steps in
// turn; the weights, laid out as the MFMA takes them, come straight from the
// caches.
template <int BM, int BN, int WM, int WN, typename T>
__global__ __launch_bounds__(256) void int8_kernel(const Int8Args a, uint32_t rows, int ksteps,
                                                   uint32_t row_tiles, uint32_t col_tiles,
                                                   bool wide) {
  constexpr int PITCH = 80;  // bytes of 64 of K in LDS: 16 rows' pieces in different banks
  constexpr int TM = WM / 32, TN = WN / 32, WCOLS = BN / WN;
  constexpr int PIECES = BM * 4 / 256;  // 16-byte pieces a thread brings of a step
  static_assert((BM / WM) * (BN / WN) == 4 && PIECES >= 1, "four waves");
  __shared__ __align__(16) uint8_t xs[2][BM * PITCH];
  __shared__ int64_t row_at[BM];
  __shared__ int64_t out_at[BM];
  __shared__ float row_scale[BM];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave / WCOLS * WM, wn = wave % WCOLS * WN;
  const uint32_t len = a.q.T;
  for (uint64_t b = blockIdx.x; b < (uint64_t)row_tiles * col_tiles; b += gridDim.x) {
    const uint32_t r0 = (uint32_t)(b / col_tiles) * BM, n0 = (uint32_t)(b % col_tiles) * BN;
    __syncthreads();
    bool any = false;
    if (tid < BM) {
      const uint64_t r = (uint64_t)r0 + tid;
      row_at[tid] = out_at[tid] = -1;
      if (r < rows) {
        const uint32_t l = (uint32_t)r / len, t = (uint32_t)r - l * len;
        if ((int)t < seq_len(a.q, l)) {
          row_at[tid] = l * a.x.lane + t * a.x.row;
          out_at[tid] = l * a.out.lane + t * a.out.row;
          row_scale[tid] = a.xscale[r];
          any = true;
        }
      }
    }
    if (!__syncthreads_or(any)) continue;
    uint4 next[PIECES];
    auto bring = [&](int k0) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int i = tid + 256 * p, row = i / 4, k = k0 + i % 4 * 16;
        const int64_t at = row_at[row];
        next[p] = at < 0 || k >= a.K ? make_uint4(0, 0, 0, 0)
                                     : row16((const int8_t*)a.x.d + at, k, a.K, wide);
      }
    };
    auto put = [&](int buf) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int i = tid + 256 * p;
        *reinterpret_cast<uint4*>(&xs[buf][i / 4 * PITCH + i % 4 * 16]) = next[p];
      }
    };
    i32x16 acc[TM][TN] = {};
    const i32x4* w = (const i32x4*)a.packed + ((size_t)(n0 + wn) / 32 * ksteps) * 64 + lane;
    bring(0);
    put(0);
    __syncthreads();
    for (int ks = 0, buf = 0; ks < ksteps; ks += 2, buf ^= 1) {
      const bool more = ks + 2 < ksteps;
      if (more) bring((ks + 2) * 32);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        i32x4 wf[TN], xf[TM];
#pragma unroll
        for (int n = 0; n < TN; ++n) wf[n] = w[((size_t)n * ksteps + ks + s) * 64];
#pragma unroll
        for (int m = 0; m < TM; ++m)
          xf[m] = *reinterpret_cast<const i32x4*>(
              &xs[buf][(wm + m * 32 + lane % 32) * PITCH + s * 32 + lane / 32 * 16]);
#pragma unroll
        for (int m = 0; m < TM; ++m)
#pragma unroll
          for (int n = 0; n < TN; ++n)
            acc[m][n] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xf[m], wf[n], acc[m][n], 0, 0, 0);
      }
      if (more) put(buf ^ 1);
      __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < TN; ++n) {
      const int col = n0 + wn + n * 32 + lane % 32;
      if (col >= a.N) continue;
      const float sw = a.wscale[col], bias = a.bias ? a.bias[col] : 0.0f;
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int row = wm + m * 32 + 8 * (i / 4) + 4 * (lane / 32) + i % 4;
          const int64_t at = out_at[row];
          if (at < 0) continue;
          const float y = (float)acc[m][n][i] * (row_scale[row] * sw) + bias;
          if constexpr (sizeof(T) == 4) ((float*)a.out.d)[at + col] = y;
          else ((uint16_t*)a.out.d)[at + col] = f32_to_bf16(y);
        }
    }
  }
}

template <typename T>
hipError_t int8_of(const Int8Args& a, hipStream_t s) {
  const uint32_t rows = (uint32_t)a.q.lanes * (uint32_t)a.q.T;
  const int ksteps = padded(a.K, K_PAD) / 32;
  const bool wide = ((uintptr_t)a.x.d & 15) == 0 && a.x.lane % 16 == 0 && a.x.row % 16 == 0;
  auto go = [&](auto kernel, int bm, int bn) {
    const uint32_t rt = (rows + bm - 1) / bm, ct = (a.N + bn - 1) / bn;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((uint64_t)rt * ct, MAX_BLOCKS);
    BOA_LAUNCH(kernel, blocks, 256, 0, s, a, rows, ksteps, rt, ct, wide);
    return hipGetLastError();
  };
  if ((uint64_t)((rows + 127) / 128) * ((a.N + 127) / 128) >= 256)
    return go(int8_kernel<128, 128, 64, 64, T>, 128, 128);
  return go(int8_kernel<64, 64, 32, 32, T>, 64, 64);
}

}  // namespace

int64_t int8_packed_bytes(int N, int K) {
  return (int64_t)padded(N, N_PAD) * padded(K, K_PAD);
}

hipError_t launch_int8_pack(const int8_t* w, int N, int K, void* packed, hipStream_t s) {
  const uint32_t pieces = (uint32_t)(int8_packed_bytes(N, K) / 16);
  const uint32_t blocks = std::min<uint32_t>((pieces + 255) / 256, MAX_BLOCKS);
  BOA_LAUNCH(int8_pack_kernel, blocks, 256, 0, s, w, N, K, padded(K, K_PAD) / 32, pieces,
             (uint4*)packed);
  return hipGetLastError();
}

hipError_t launch_int8(const Int8Args& a, hipStream_t s) {
  return a.bf16 ? int8_of<uint16_t>(a, s) : int8_of<float>(a, s);
}

}  // namespace boa
