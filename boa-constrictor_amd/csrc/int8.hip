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

// 16 bytes of a row from k on; past K whatever the row holds, for the weights
// are zero there.  WIDE: in one piece (K is a multiple of 16); else byte by byte.
// No branch lies between a step's loads, each of which would wait for the last.
template <bool WIDE>
__device__ __forceinline__ uint4 row16(const int8_t* row, int k, int K) {
  if constexpr (WIDE) return *reinterpret_cast<const uint4*>(row + min(k, K - 16));
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    v[i / 4] |= (uint32_t)(uint8_t)row[min(k + i, K - 1)] << (8 * (i % 4));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// where a tile's rows lie; out -1: past the end or a lane's length (such a row
// reads the weights instead, K bytes of them, and its results go nowhere)
template <int BM>
struct Tile {
  const int8_t* row[BM];
  int64_t out[BM];
  float scale[BM];
  // true where the tile has a row at all; a barrier for the block of 256
  __device__ __forceinline__ bool find(const Int8Args& a, uint32_t r0, uint32_t rows) {
    const int i = threadIdx.x;
    const uint32_t len = a.q.T;
    bool any = false;
    if (i < BM) {
      const uint64_t r = (uint64_t)r0 + i;
      row[i] = (const int8_t*)a.packed;
      out[i] = -1;
      scale[i] = 0.0f;
      if (r < rows) {
        const uint32_t l = (uint32_t)r / len, t = (uint32_t)r - l * len;
        if ((int)t < seq_len(a.q, l)) {
          row[i] = (const int8_t*)a.x.d + l * a.x.lane + t * a.x.row;
          out[i] = l * a.out.lane + t * a.out.row;
          scale[i] = a.xscale[r];
          any = true;
        }
      }
    }
    return __syncthreads_or(any);
  }
};

__device__ __forceinline__ float result_of(int acc, float sx, float sw, float bias) {
  return (float)acc * (sx * sw) + bias;
}

// Many rows: a block of four waves computes 128 rows x 128 channels, a wave
// 64 x 64 in tiles of 32 x 32.  256 of K at a time: rows pass through LDS, the
// weights of a wave, laid out as the MFMA takes them, come straight from the
// caches; all of a step's loads are under way together, the next rows' while
// the present are multiplied.  Two blocks a CU, so one's stores overlap the
// other's products.  Blocks that follow each other on an XCD take the columns of
// one row tile, whose rows its L2 then holds.  Results pass through LDS and
// leave as whole rows of 16-byte pieces.
template <typename T, bool WIDE>
__global__ __launch_bounds__(256, 2) void int8_kernel(const Int8Args a, uint32_t rows, int ksteps,
                                                      uint32_t row_tiles, uint32_t col_tiles,
                                                      bool wide_out) {
  constexpr int BM = 128, BN = 128, KB = 256, PITCH = KB + 16;
  constexpr int PIECES = BM * KB / 16 / 256;
  constexpr int OP = BN + 16 / sizeof(T);  // pitch of the results in LDS
  __shared__ __align__(16) uint8_t xs[BM * PITCH];
  __shared__ Tile<BM> tile;
  static_assert(64 * OP * sizeof(T) <= sizeof xs, "half of the results at a time");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave / 2 * 64, wn = wave % 2 * 64;
  const uint64_t all = (uint64_t)((row_tiles + 7) / 8) * 8 * col_tiles;
  for (uint64_t b = blockIdx.x; b < all; b += gridDim.x) {
    const uint32_t rt = (uint32_t)(b / 8 / col_tiles) * 8 + (uint32_t)(b % 8);
    if (rt >= row_tiles) continue;
    const uint32_t r0 = rt * BM, n0 = (uint32_t)(b / 8 % col_tiles) * BN;
    __syncthreads();
    if (!tile.find(a, r0, rows)) continue;
    uint4 next[PIECES];
    auto bring = [&](int k0) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int i = tid + 256 * p;
        next[p] = row16<WIDE>(tile.row[i / (KB / 16)], k0 + i % (KB / 16) * 16, a.K);
      }
    };
    i32x16 acc[2][2] = {};
    const i32x4* w = (const i32x4*)a.packed + ((size_t)(n0 + wn) / 32 * ksteps) * 64 + lane;
    bring(0);
    for (int ks = 0; ks < ksteps; ks += KB / 32) {
      if (ks) __syncthreads();
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int i = tid + 256 * p;
        *reinterpret_cast<uint4*>(&xs[i / (KB / 16) * PITCH + i % (KB / 16) * 16]) = next[p];
      }
      i32x4 wf[KB / 32][2];
#pragma unroll
      for (int s = 0; s < KB / 32; ++s)
#pragma unroll
        for (int n = 0; n < 2; ++n)
          wf[s][n] = w[((size_t)n * ksteps + min(ks + s, ksteps - 1)) * 64];
      if (ks + KB / 32 < ksteps) bring((ks + KB / 32) * 32);
      __syncthreads();
#pragma unroll
      for (int s = 0; s < KB / 32; ++s) {
        if (ks + s >= ksteps) break;
        i32x4 xf[2];
#pragma unroll
        for (int m = 0; m < 2; ++m)
          xf[m] = *reinterpret_cast<const i32x4*>(
              &xs[(wm + m * 32 + lane % 32) * PITCH + s * 32 + lane / 32 * 16]);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int n = 0; n < 2; ++n)
            acc[m][n] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xf[m], wf[s][n], acc[m][n], 0, 0, 0);
      }
    }
    float sw[2], bias[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int col = min(n0 + wn + n * 32 + lane % 32, (uint32_t)a.N - 1);
      sw[n] = a.wscale[col];
      bias[n] = a.bias ? a.bias[col] : 0.0f;
    }
    // half of the rows at a time
    T* os = reinterpret_cast<T*>(xs);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
      if (wm == half * 64) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int row = m * 32 + 8 * (i / 4) + 4 * (lane / 32) + i % 4;
              const float y = result_of(acc[m][n][i], tile.scale[wm + row], sw[n], bias[n]);
              T* o = os + row * OP + wn + n * 32 + lane % 32;
              if constexpr (sizeof(T) == 4) *o = y;
              else *o = f32_to_bf16(y);
            }
      }
      __syncthreads();
      constexpr int V = 16 / sizeof(T), PER = BN / V;
      for (int i = tid; i < 64 * PER; i += 256) {
        const int row = i / PER, c = i % PER * V, col = n0 + c;
        const int64_t at = tile.out[half * 64 + row];
        if (at < 0 || col >= a.N) continue;
        T* o = (T*)a.out.d + at + col;
        const T* from = os + row * OP + c;
        if (wide_out && col + V <= a.N) {
          typedef uint32_t u4 __attribute__((ext_vector_type(4)));
          *reinterpret_cast<u4*>(o) = *reinterpret_cast<const u4*>(from);
        } else {
          for (int j = 0; j < V && col + j < a.N; ++j) o[j] = from[j];
        }
      }
    }
  }
}

// Few rows: a block computes 32 rows x 32 channels, its four waves every fourth
// 32 of K each, straight from the caches, so that all of a short K is under way
// at once; the sums meet in LDS.
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void int8_few_kernel(const Int8Args a, uint32_t rows, int ksteps,
                                                       uint32_t row_tiles,
                                                       uint32_t col_tiles) {
  __shared__ int sums[4][32 * 33];
  __shared__ Tile<32> tile;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (uint64_t b = blockIdx.x; b < (uint64_t)row_tiles * col_tiles; b += gridDim.x) {
    const uint32_t r0 = (uint32_t)(b / col_tiles) * 32, n0 = (uint32_t)(b % col_tiles) * 32;
    __syncthreads();
    const i32x4* w = (const i32x4*)a.packed + (size_t)n0 / 32 * ksteps * 64 + lane;
    if (!tile.find(a, r0, rows)) continue;
    const int8_t* x = tile.row[lane % 32];
    i32x16 acc = {};
#pragma unroll 4
    for (int ks = wave; ks < ksteps; ks += 4) {
      const uint4 v = row16<WIDE>(x, ks * 32 + lane / 32 * 16, a.K);
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, v), w[(size_t)ks * 64],
                                                  acc, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      sums[wave][(8 * (i / 4) + 4 * (lane / 32) + i % 4) * 33 + lane % 32] = acc[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = tid / 32 + 8 * i, c = tid % 32, col = n0 + c;
      const int64_t o = tile.out[row];
      if (o < 0 || col >= a.N) continue;
      const int s = sums[0][row * 33 + c] + sums[1][row * 33 + c] + sums[2][row * 33 + c] +
                    sums[3][row * 33 + c];
      const float y = result_of(s, tile.scale[row], a.wscale[col], a.bias ? a.bias[col] : 0.0f);
      if constexpr (sizeof(T) == 4) ((float*)a.out.d)[o + col] = y;
      else ((uint16_t*)a.out.d)[o + col] = f32_to_bf16(y);
    }
  }
}

template <typename T, bool WIDE>
hipError_t int8_of(const Int8Args& a, hipStream_t s) {
  const uint32_t rows = (uint32_t)a.q.lanes * (uint32_t)a.q.T;
  const int ksteps = padded(a.K, K_PAD) / 32;
  const uint32_t rt = (rows + 127) / 128, ct = (a.N + 127) / 128;
  if ((uint64_t)rt * ct >= 256) {
    constexpr int V = 16 / sizeof(T);
    const bool wide_out = ((uintptr_t)a.out.d & 15) == 0 && a.out.lane % V == 0 && a.out.row % V == 0;
    const uint32_t blocks =
        (uint32_t)std::min<uint64_t>((uint64_t)((rt + 7) / 8) * 8 * ct, MAX_BLOCKS);
    BOA_LAUNCH((int8_kernel<T, WIDE>), blocks, 256, 0, s, a, rows, ksteps, rt, ct, wide_out);
    return hipGetLastError();
  }
  const uint32_t frt = (rows + 31) / 32, fct = (a.N + 31) / 32;
  const uint32_t blocks = (uint32_t)std::min<uint64_t>((uint64_t)frt * fct, MAX_BLOCKS);
  BOA_LAUNCH((int8_few_kernel<T, WIDE>), blocks, 256, 0, s, a, rows, ksteps, frt, fct);
  return hipGetLastError();
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
  if (rows_by_16(a.x.d, a.x.lane, a.x.row, a.K, 1))
    return a.bf16 ? int8_of<uint16_t, true>(a, s) : int8_of<float, true>(a, s);
  return a.bf16 ? int8_of<uint16_t, false>(a, s) : int8_of<float, false>(a, s);
}

}  // namespace boa
