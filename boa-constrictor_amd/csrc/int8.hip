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

// Weights as v_mfma_i32_16x16x64_i8 takes them: of every 16 channels, for every
// 64 of K, lane i's 16 bytes are channel i % 16, k = 16 (i / 16) ..; channels
// are padded to 128, K to 64 (beyond 512 to 256), with zeros.
constexpr int N_PAD = 128, K_STEP = 64;
int padded(int n, int to) { return (n + to - 1) / to * to; }
int steps_of(int K) { return K <= 512 ? padded(K, K_STEP) / K_STEP : padded(K, 256) / K_STEP; }

__global__ __launch_bounds__(256) void int8_pack_kernel(const int8_t* w, int N, int K, int ksteps,
                                                        uint32_t pieces, uint4* packed) {
  for (uint32_t p = blockIdx.x * 256 + threadIdx.x; p < pieces; p += gridDim.x * 256) {
    const uint32_t lane = p % 64, step = p / 64 % ksteps, tile = p / 64 / ksteps;
    const int n = tile * 16 + lane % 16, k0 = step * K_STEP + lane / 16 * 16;
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

// where a tile's rows lie, counted from x; out -1: past the end or a lane's
// length (such a row reads the weights instead, K bytes of them, and its results
// go nowhere)
template <int BM>
struct Tile {
  int64_t row[BM], out[BM];
  float scale[BM];
  // true where the tile has a row at all; a barrier for the block
  __device__ __forceinline__ bool find(const Int8Args& a, uint32_t r0, uint32_t rows) {
    const int i = threadIdx.x;
    const uint32_t len = a.q.T;
    bool any = false;
    if (i < BM) {
      const uint64_t r = (uint64_t)r0 + i;
      row[i] = (int64_t)((uintptr_t)a.packed - (uintptr_t)a.x.d);
      out[i] = -1;
      scale[i] = 0.0f;
      if (r < rows) {
        const uint32_t l = (uint32_t)r / len, t = (uint32_t)r - l * len;
        const float s = a.xscale[r];
        if ((int)t < seq_len(a.q, l)) {
          row[i] = l * a.x.lane + t * a.x.row;
          out[i] = l * a.out.lane + t * a.out.row;
          scale[i] = s;
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

// A wave's results, 64 rows x 64 channels from n0 on.  fp32 leaves as it lies
// (16 channels are 64 bytes); bf16 through the wave's own piece of LDS, 16
// rows at a time, as 16-byte pieces of whole rows.
constexpr int OUT_PITCH = 64 + 8;
template <typename T>
__device__ __forceinline__ void put_results(const Int8Args& a, i32x4 (&acc)[4][4], uint16_t* os,
                                            const int64_t* out, const float* scale, int n0,
                                            int lane, bool wide_out) {
  float sw[4], bias[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int col = min(n0 + n * 16 + lane % 16, a.N - 1);
    sw[n] = a.wscale[col];
    bias[n] = a.bias ? a.bias[col] : 0.0f;
  }
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = m * 16 + lane / 16 * 4 + r;
        const int64_t at = out[row];
        const float sx = scale[row];
        float* o = (float*)a.out.d + at + n0 + lane % 16;
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (at >= 0 && n0 + n * 16 + lane % 16 < a.N)
            o[n * 16] = result_of(acc[m][n][r], sx, sw[n], bias[n]);
      }
  } else {
#pragma unroll
    for (int m = 0; m < 4; ++m) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = lane / 16 * 4 + r;
        const float sx = scale[m * 16 + row];
#pragma unroll
        for (int n = 0; n < 4; ++n)
          os[row * OUT_PITCH + n * 16 + lane % 16] =
              f32_to_bf16(result_of(acc[m][n][r], sx, sw[n], bias[n]));
      }
      // the wave's own LDS accesses are in order; the compiler's have to be
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      const int c = lane % 8 * 8, col = n0 + c;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = i * 8 + lane / 8;
        const int64_t at = out[m * 16 + row];
        const uint16_t* from = os + row * OUT_PITCH + c;
        uint16_t* o = (uint16_t*)a.out.d + at + col;
        if (wide_out) {  // N is a multiple of 8
          typedef uint32_t u4 __attribute__((ext_vector_type(4)));
          const u4 v = *reinterpret_cast<const u4*>(from);
          if (at >= 0 && col < a.N) *reinterpret_cast<u4*>(o) = v;
        } else if (at >= 0) {
          for (int j = 0; j < 8; ++j)
            if (col + j < a.N) o[j] = from[j];
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// Many rows: a block of four waves takes 128 rows x `group` tiles of 128 channels, a
// wave 64 x 64 of a tile (128 x 64, for which the weights would have to come half as
// often, does not fit the registers of two waves a SIMD: 110 us and not 71 for 33,360 x
// 2064 x 512, bf16, rows in the caches).  64 KS of K at a time the rows lie in LDS (all
// of K up to 512, brought once for the block's tiles); the weights come straight from
// the caches into registers, one or two steps ahead and across tiles.  Two blocks a CU,
// so one's stores overlap the other's products.  Blocks that follow each other on an
// XCD take the groups of one row tile, whose rows its L2 then holds.  33,360 x 2064 x
// 512, bf16: 82 us, 0.86 Pop/s and 1.9 TB/s (73 with the same rows and results again,
// which the caches hold); fp32 results 122.  Bound by eight steps of products, a fifth
// of the time, and then as much work for the results, which two blocks a CU overlap
// only in part.  Rows that are not wide are put together byte by byte, for which the
// form of KS = 3 spills 112 to 118 registers and those of 5 .. 8 keep 128 bytes a lane
// in scratch.
template <typename T, int KS, bool WIDE>
__global__ __launch_bounds__(256, 2) void int8_kernel(const Int8Args a, uint32_t rows, int ksteps,
                                                      uint32_t row_tiles, uint32_t col_tiles,
                                                      uint32_t groups, uint32_t group,
                                                      bool wide_out) {
  constexpr int BM = 128, KB = KS * K_STEP, PITCH = KB + 16, PER = KB / 16;
  constexpr int PIECES = BM * PER / 256, R = KS % 2 == 0 ? 2 : 1;
  __shared__ __align__(16) uint8_t xs[BM * PITCH];
  __shared__ __align__(16) uint16_t os[sizeof(T) == 4 ? 1 : 4][sizeof(T) == 4 ? 8 : 16 * OUT_PITCH];
  __shared__ Tile<BM> tile;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave / 2 * 64, wn = wave % 2 * 64;
  const uint64_t all = (uint64_t)((row_tiles + 7) / 8) * 8 * groups;
  for (uint64_t b = blockIdx.x; b < all; b += gridDim.x) {
    const uint32_t rt = (uint32_t)(b / 8 / groups) * 8 + (uint32_t)(b % 8);
    if (rt >= row_tiles) continue;
    const uint32_t first = (uint32_t)(b / 8 % groups) * group;
    const uint32_t last = min(first + group, col_tiles);
    __syncthreads();
    if (!tile.find(a, rt * BM, rows)) continue;
    auto bring = [&](int k0) {
      uint4 v[PIECES];
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int i = tid + 256 * p;
        v[p] = row16<WIDE>((const int8_t*)a.x.d + tile.row[i / PER], k0 + i % PER * 16, a.K);
      }
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int i = tid + 256 * p;
        *reinterpret_cast<uint4*>(&xs[i / PER * PITCH + i % PER * 16]) = v[p];
      }
    };
    const i32x4* w = (const i32x4*)a.packed + ((size_t)(first * 128 + wn) / 16 * ksteps) * 64 + lane;
    i32x4 wf[R][4];
#pragma unroll
    for (int s = 0; s < R; ++s)
#pragma unroll
      for (int n = 0; n < 4; ++n) wf[s][n] = w[((size_t)n * ksteps + s) * 64];
    bring(0);
    __syncthreads();
    for (uint32_t ct = first; ct < last; ++ct) {
      i32x4 acc[4][4] = {};
      // where the weights go on after this tile (its own, behind the last one)
      const i32x4* after = ct + 1 < last ? w + (size_t)8 * ksteps * 64 : w;
      for (int k0 = 0; k0 < ksteps; k0 += KS) {
        if (k0 || (ksteps > KS && ct > first)) {
          __syncthreads();
          bring(k0 * K_STEP);
          __syncthreads();
        }
        const i32x4* next = k0 + KS < ksteps ? w + (k0 + KS) * 64 : after;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          i32x4 xf[4];
#pragma unroll
          for (int m = 0; m < 4; ++m)
            xf[m] = *reinterpret_cast<const i32x4*>(
                &xs[(wm + m * 16 + lane % 16) * PITCH + s * K_STEP + lane / 16 * 16]);
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int n = 0; n < 4; ++n)
              acc[m][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xf[m], wf[s % R][n], acc[m][n], 0,
                                                               0, 0);
          const i32x4* from = s + R < KS ? w + (k0 + s + R) * 64 : next + (s + R - KS) * 64;
#pragma unroll
          for (int n = 0; n < 4; ++n) wf[s % R][n] = from[(size_t)n * ksteps * 64];
        }
      }
      put_results<T>(a, acc, os[sizeof(T) == 4 ? 0 : wave], tile.out + wm, tile.scale + wm,
                     ct * 128 + wn, lane, wide_out);
      w = after;
    }
  }
}

// Few rows: a block computes 32 rows x 32 channels, its four waves every fourth
// 64 of K each, straight from the caches, so that all of a short K is under way
// at once; the sums meet in LDS.  Bound by the latency of one such chain: 64 x 1032 x
// 256 3.6 us.
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void int8_few_kernel(const Int8Args a, uint32_t rows, int ksteps,
                                                       uint32_t row_tiles, uint32_t col_tiles) {
  __shared__ int sums[4][32 * 33];
  __shared__ Tile<32> tile;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (uint64_t b = blockIdx.x; b < (uint64_t)row_tiles * col_tiles; b += gridDim.x) {
    const uint32_t r0 = (uint32_t)(b / col_tiles) * 32, n0 = (uint32_t)(b % col_tiles) * 32;
    __syncthreads();
    const i32x4* w = (const i32x4*)a.packed + (size_t)n0 / 16 * ksteps * 64 + lane;
    if (!tile.find(a, r0, rows)) continue;
    const int8_t* x[2] = {(const int8_t*)a.x.d + tile.row[lane % 16],
                          (const int8_t*)a.x.d + tile.row[16 + lane % 16]};
    i32x4 acc[2][2] = {};
#pragma unroll 2
    for (int ks = wave; ks < ksteps; ks += 4) {
      i32x4 wf[2], xf[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        wf[i] = w[((size_t)i * ksteps + ks) * 64];
        xf[i] = __builtin_bit_cast(i32x4, row16<WIDE>(x[i], ks * K_STEP + lane / 16 * 16, a.K));
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
          acc[m][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xf[m], wf[n], acc[m][n], 0, 0, 0);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          sums[wave][(m * 16 + lane / 16 * 4 + r) * 33 + n * 16 + lane % 16] = acc[m][n][r];
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
  const int ksteps = steps_of(a.K);
  const uint32_t rt = (rows + 127) / 128, ct = (a.N + 127) / 128;
  const bool wide_out = rows_by_16(a.out.d, a.out.lane, a.out.row, a.N, sizeof(T));
  // Tiles of 32 x 32 while those of 128 x 128 leave most CUs without work.  Small
  // and large, us: 1024 rows, N 1032, K 256 (72 large tiles) 5.3 and 6.0; 512 rows,
  // 2064, 512 (68) 6.4 and 7.6; 6000, 256, 256 (94) 6.8 and 6.1; 768, 2064, 512
  // (102) 9.0 and 7.6; 64, 2064, 512 (17) 3.9 and 7.2.
  if ((uint64_t)rt * ct < 80) {
    const uint32_t frt = (rows + 31) / 32, fct = (a.N + 31) / 32;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((uint64_t)frt * fct, MAX_BLOCKS);
    BOA_LAUNCH((int8_few_kernel<T, WIDE>), blocks, 256, 0, s, a, rows, ksteps, frt, fct);
  } else {
    // a block's tiles: four rounds of blocks at least, so that the last one's gaps
    // are short
    const uint32_t group = std::max<uint64_t>(1, std::min<uint64_t>(8, (uint64_t)rt * ct / 2048));
    const uint32_t groups = (ct + group - 1) / group;
    const uint32_t blocks =
        (uint32_t)std::min<uint64_t>((uint64_t)((rt + 7) / 8) * 8 * groups, MAX_BLOCKS);
    auto go = [&](auto kernel) {
      BOA_LAUNCH(kernel, blocks, 256, 0, s, a, rows, ksteps, rt, ct, groups, group, wide_out);
    };
    switch (ksteps <= 8 ? ksteps : 4) {
      case 1: go(int8_kernel<T, 1, WIDE>); break;
      case 2: go(int8_kernel<T, 2, WIDE>); break;
      case 3: go(int8_kernel<T, 3, WIDE>); break;
      case 4: go(int8_kernel<T, 4, WIDE>); break;
      case 5: go(int8_kernel<T, 5, WIDE>); break;
      case 6: go(int8_kernel<T, 6, WIDE>); break;
      case 7: go(int8_kernel<T, 7, WIDE>); break;
      default: go(int8_kernel<T, 8, WIDE>);
    }
  }
  return hipGetLastError();
}

}  // namespace

int64_t int8_packed_bytes(int N, int K) {
  return (int64_t)padded(N, N_PAD) * steps_of(K) * K_STEP;
}

hipError_t launch_int8_pack(const int8_t* w, int N, int K, void* packed, hipStream_t s) {
  const uint32_t pieces = (uint32_t)(int8_packed_bytes(N, K) / 16);
  const uint32_t blocks = std::min<uint32_t>((pieces + 255) / 256, MAX_BLOCKS);
  BOA_LAUNCH(int8_pack_kernel, blocks, 256, 0, s, w, N, K, steps_of(K), pieces,
             (uint4*)packed);
  return hipGetLastError();
}

hipError_t launch_int8(const Int8Args& a, hipStream_t s) {
  if (rows_by_16(a.x.d, a.x.lane, a.x.row, a.K, 1))
    return a.bf16 ? int8_of<uint16_t, true>(a, s) : int8_of<float, true>(a, s);
  return a.bf16 ? int8_of<uint16_t, false>(a, s) : int8_of<float, false>(a, s);
}

}  // namespace boa
