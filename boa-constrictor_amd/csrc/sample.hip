// The choice of a byte from its logits, with a given random number u in [0, 1):
//   x = logits + bias;  weight = exp((x - max x) / temperature)
// ranked by x, the lowest byte first among equals; kept are the first top_k,
// of those the shortest prefix that holds top_p of their weight, of those the
// bytes of weight at least min_p (the first has 1); the byte is the first one,
// in order of its value, up to which the kept weights exceed u times their sum.
// All of it in 64 bits: u may lie next to a border.
#include <algorithm>

#include "predictor_ops.h"

namespace boa {

namespace {

template <typename F>
__device__ __forceinline__ double wave_all(double x, F f) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) x = f(x, __shfl_xor(x, m));
  return x;
}
// sum over the lanes below
__device__ __forceinline__ double wave_before(double x, int lane) {
  double s = x;
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    const double y = __shfl_up(s, m);
    if (lane >= m) s += y;
  }
  s = __shfl_up(s, 1);
  return lane ? s : 0.0;
}

// A wave per row, bytes 4 i .. 4 i + 3 in lane i.
template <typename T>
__global__ __launch_bounds__(256) void sample_kernel(const SampleArgs a, uint32_t rows) {
  __shared__ double xs[4][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t len = a.q.T;
  for (uint64_t b = (uint64_t)blockIdx.x * 4; b < rows; b += (uint64_t)gridDim.x * 4) {
    __syncthreads();
    const uint64_t r = b + wave;
    const uint32_t l = r < rows ? (uint32_t)r / len : 0, t = r < rows ? (uint32_t)r - l * len : 0;
    const bool live = r < rows && (int)t < seq_len(a.q, l);
    double x[4], w[4];
    double top = -__builtin_inf();
    bool bad = false;
    const T* p = (const T*)a.logits.d + l * a.logits.lane + t * a.logits.row + 4 * lane;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = -__builtin_inf();
      if (live) {
        if constexpr (sizeof(T) == 4) x[j] = (double)p[j];
        else x[j] = (double)bf16_to_f32(p[j]);
        if (a.bias) x[j] += (double)a.bias[4 * lane + j];
      }
      bad |= !(x[j] < __builtin_inf());
      top = __builtin_fmax(top, x[j]);
    }
    top = wave_all(top, [](double u, double v) { return __builtin_fmax(u, v); });
    bad = __any(bad) || !(top > -__builtin_inf());
    const SampleHow h = a.each && live ? a.each[l] : a.how;
    const bool greedy = !(h.temperature > 0.0f);
    // how many stand before each, and the weights in order of rank
    int ahead[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = ::exp((x[j] - top) / (greedy ? 1.0 : (double)h.temperature));
      xs[wave][4 * lane + j] = x[j];
    }
    __syncthreads();
    const bool some = live && !bad;
    if (some)
      for (int i = 0; i < 256; ++i) {
        const double y = xs[wave][i];
#pragma unroll
        for (int j = 0; j < 4; ++j) ahead[j] += y > x[j] || (y == x[j] && i < 4 * lane + j);
      }
    __syncthreads();
    const bool by_k = h.top_k >= 1.0f, by_p = h.top_p < 1.0f;
    if (some)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        xs[wave][ahead[j]] = by_k && !((float)ahead[j] < h.top_k) ? 0.0 : w[j];
    __syncthreads();
    int cut = 256;  // ranks from here on are left out
    if (some) {
      double v[4], s = 0.0;
#pragma unroll
      for (int j = 0; j < 4; ++j) s += v[j] = xs[wave][4 * lane + j];
      double before = wave_before(s, lane);
      const double total = wave_all(s, [](double u, double v2) { return u + v2; });
      int first = 256;
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        double at = before;
        for (int i = 0; i < j; ++i) at += v[i];
        const int rank = 4 * lane + j;
        if (rank && ((by_p && !(at < (double)h.top_p * total)) ||
                     (by_k && !((float)rank < h.top_k)) || v[j] < (double)h.min_p || greedy))
          first = rank;
      }
#pragma unroll
      for (int m = 1; m < 64; m *= 2) first = min(first, __shfl_xor(first, m));
      cut = first;
    }
    double kept[4], sum = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += kept[j] = ahead[j] < cut ? w[j] : 0.0;
    const double before = wave_before(sum, lane);
    const double total = wave_all(sum, [](double u, double v) { return u + v; });
    // (a number outside [0, 1) is taken as the nearest inside, NaN as 0)
    const double u = live ? fmin(fmax((double)a.uniform[r], 0.0), 0x1.fffffep-1) * total : 0.0;
    // the first byte whose running sum exceeds u
    int byte = 256;
    double mine = 0.0, at = before;
    double run[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) run[j] = at += kept[j];
#pragma unroll
    for (int j = 3; j >= 0; --j)
      if (run[j] > u && kept[j] > 0.0) byte = 4 * lane + j, mine = kept[j];
    const int own = byte;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) byte = min(byte, __shfl_xor(byte, m));
    if (live && bad && lane == 0) {
      a.bytes[l * a.stride + t] = 0;
      if (a.logp) a.logp[r] = __builtin_nanf("");
    } else if (some && own == byte && own < 256) {
      a.bytes[l * a.stride + t] = (uint8_t)byte;
      if (a.logp) a.logp[r] = (float)::log(mine / total);
    }
  }
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, hipStream_t s) {
  const uint32_t rows = (uint32_t)a.q.lanes * (uint32_t)a.q.T;
  const uint32_t blocks = std::min<uint32_t>((rows + 3) / 4, MAX_BLOCKS);
  if (a.bf16) BOA_LAUNCH(sample_kernel<uint16_t>, blocks, 256, 0, s, a, rows);
  else BOA_LAUNCH(sample_kernel<float>, blocks, 256, 0, s, a, rows);
  return hipGetLastError();
}

}  // namespace boa
