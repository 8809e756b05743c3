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

// x of lane i ^ M
template <int M>
__device__ __forceinline__ uint32_t other(uint32_t x, int lane) {
  if constexpr (M == 63) {
    return other<32>(other<31>(x, lane), lane);
  } else if constexpr (M == 31) {
    return other<16>(other<15>(x, lane), lane);
  } else if constexpr (M == 32) {
    const auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return lane & 32 ? s[0] : s[1];
  } else if constexpr (M == 16) {
    const auto s = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return lane & 16 ? s[0] : s[1];
  } else if constexpr (M == 4) {
    return other<3>(other<7>(x, lane), lane);
  } else {
    constexpr int CTRL = M == 1 ? DPP_XOR1 : M == 2 ? DPP_XOR2 : M == 3 ? 0x1B
                         : M == 7 ? DPP_HALF_MIRROR : M == 8 ? DPP_ROR8 : DPP_MIRROR;
    static_assert(M == 1 || M == 2 || M == 3 || M == 7 || M == 8 || M == 15, "no such move");
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true);
  }
}
template <int M>
__device__ __forceinline__ double other(double x, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint64_t lo = other<M>((uint32_t)b, lane), hi = other<M>((uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, hi << 32 | lo);
}
template <typename X, typename F>
__device__ __forceinline__ X wave_all(X x, int lane, F f) {
  x = f(x, other<1>(x, lane));
  x = f(x, other<2>(x, lane));
  x = f(x, other<7>(x, lane));
  x = f(x, other<15>(x, lane));
  x = f(x, other<16>(x, lane));
  return f(x, other<32>(x, lane));
}
struct Add64 {
  __device__ double operator()(double a, double b) const { return a + b; }
};
struct Max64 {
  __device__ double operator()(double a, double b) const { return __builtin_fmax(a, b); }
};
struct Min32 {
  __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return a < b ? a : b; }
};
// sum over the lanes below: after step m a lane has its block of 2 m lanes'
// sum and that of the lanes before it there
template <int M>
__device__ __forceinline__ void before_step(double& sum, double& before, int lane) {
  const double o = other<M>(sum, lane);
  if (lane & M) before += o;
  sum += o;
}
__device__ __forceinline__ double wave_before(double x, int lane, double& total) {
  double before = 0.0;
  before_step<1>(x, before, lane);
  before_step<2>(x, before, lane);
  before_step<4>(x, before, lane);
  before_step<8>(x, before, lane);
  before_step<16>(x, before, lane);
  before_step<32>(x, before, lane);
  total = x;
  return before;
}

// The wave's 256 values from the greatest to the least, value 4 i + j in
// element j of lane i.  Sorted runs of n are merged in pairs: a run against the
// next one backwards (lane ^ M, element 3 - j), then halves of halves (lane ^ M,
// the same element), the greater always to the lower place, so steps within a
// lane are two instructions.
__device__ __forceinline__ void order(double& hi, double& lo) {
  const double a = __builtin_fmax(hi, lo), b = __builtin_fmin(hi, lo);
  hi = a;
  lo = b;
}
template <int M, bool BACK>
__device__ __forceinline__ void cross(double (&x)[4], int lane) {
  // lane ^ M is the lower one where the highest bit of M is set
  const bool low = !(lane & (BACK ? (M + 1) / 2 : M));
  double y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = other<M>(x[BACK ? 3 - j : j], lane);
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = (x[j] < y[j]) == low ? y[j] : x[j];
}
__device__ __forceinline__ void within(double (&x)[4]) {
  order(x[0], x[2]);
  order(x[1], x[3]);
  order(x[0], x[1]);
  order(x[2], x[3]);
}
__device__ __forceinline__ void sort_wave(double (&x)[4], int lane) {
  order(x[0], x[1]);
  order(x[2], x[3]);
  order(x[0], x[3]);
  order(x[1], x[2]);
  order(x[0], x[1]);
  order(x[2], x[3]);
  cross<1, true>(x, lane);
  within(x);
  cross<3, true>(x, lane);
  cross<1, false>(x, lane);
  within(x);
  cross<7, true>(x, lane);
  cross<2, false>(x, lane);
  cross<1, false>(x, lane);
  within(x);
  cross<15, true>(x, lane);
  cross<4, false>(x, lane);
  cross<2, false>(x, lane);
  cross<1, false>(x, lane);
  within(x);
  cross<31, true>(x, lane);
  cross<8, false>(x, lane);
  cross<4, false>(x, lane);
  cross<2, false>(x, lane);
  cross<1, false>(x, lane);
  within(x);
  cross<63, true>(x, lane);
  cross<16, false>(x, lane);
  cross<8, false>(x, lane);
  cross<4, false>(x, lane);
  cross<2, false>(x, lane);
  cross<1, false>(x, lane);
  within(x);
}

// A wave per row, bytes 4 i .. 4 i + 3 in lane i.  Bound by the vector
// instructions, which the SIMDs issue without a pause: 1500 a row, of them 600 the
// sort's where top_k or top_p ask for it, most others the exponentials' and the
// sums' in 64 bits.  32,500 rows: 87 us; 64 rows: 7 us, what a launch takes.
template <typename T>
__global__ __launch_bounds__(256) void sample_kernel(const SampleArgs a, uint32_t rows, bool wide) {
  const int lane = threadIdx.x & 63;
  const uint32_t len = a.q.T;
  float bias[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) bias[j] = a.bias ? a.bias[4 * lane + j] : 0.0f;
  const uint64_t first = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  for (uint64_t r = first; r < rows; r += (uint64_t)gridDim.x * 4) {
    const uint32_t l = (uint32_t)r / len, t = (uint32_t)r - l * len;
    if ((int)t >= seq_len(a.q, l)) continue;
    const T* p = (const T*)a.logits.d + l * a.logits.lane + t * a.logits.row + 4 * lane;
    float raw[4];
    if (wide) {
      if constexpr (sizeof(T) == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        raw[0] = v.x, raw[1] = v.y, raw[2] = v.z, raw[3] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        raw[0] = u2f(v.x << 16), raw[1] = u2f(v.x & 0xFFFF0000u);
        raw[2] = u2f(v.y << 16), raw[3] = u2f(v.y & 0xFFFF0000u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) raw[j] = p[j];
        else raw[j] = bf16_to_f32(p[j]);
      }
    }
    const SampleHow h = a.each ? a.each[l] : a.how;
    const float number = a.uniform[r];
    double x[4], top;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = (double)raw[j] + (double)bias[j];
      bad |= !(x[j] < __builtin_inf());
    }
    top = __builtin_fmax(__builtin_fmax(x[0], x[1]), __builtin_fmax(x[2], x[3]));
    top = wave_all(top, lane, Max64());
    if (__any(bad) || !(top > -__builtin_inf())) {
      if (lane == 0) {
        a.bytes[l * a.stride + t] = 0;
        if (a.logp) a.logp[r] = __builtin_nanf("");
      }
      continue;
    }
    uint32_t byte = 256;
    double share = 1.0;
    if (!(h.temperature > 0.0f) || h.min_p > 1.0f) {  // the first in rank alone
#pragma unroll
      for (int j = 3; j >= 0; --j)
        if (x[j] == top) byte = 4 * lane + j;
      byte = wave_all(byte, lane, Min32());
    } else {
      // (not 0 for an infinite temperature: a logit of -inf has to stay one)
      const double sharp = __builtin_fmax(1.0 / (double)h.temperature, 1e-300);
      double w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = ::exp((x[j] - top) * sharp);
        if (w[j] < (double)h.min_p) w[j] = 0.0;
      }
      const bool by_k = h.top_k >= 1.0f && h.top_k < 256.0f, by_p = h.top_p < 1.0f;
      if (by_k || by_p) {
        double s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = x[j];
        sort_wave(s, lane);
        uint32_t cut = 256;  // the first rank that is left out
#pragma unroll
        for (int j = 3; j >= 0; --j)
          if (by_k && !((float)(4 * lane + j) < h.top_k)) cut = 4 * lane + j;
        if (by_p) {
          double v[4], total;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            v[j] = by_k && !((float)(4 * lane + j) < h.top_k) ? 0.0 : ::exp((s[j] - top) * sharp);
          double at = wave_before(v[0] + v[1] + v[2] + v[3], lane, total);
          const double enough = (double)h.top_p * total;
          bool out[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            out[j] = !(at < enough);
            at += v[j];
          }
#pragma unroll
          for (int j = 3; j >= 0; --j)
            if (out[j] && 4 * lane + j > 0) cut = min(cut, (uint32_t)(4 * lane + j));
        }
        cut = wave_all(cut, lane, Min32());
        if (cut < 256) {
          // the last value kept and how many of its equals are: all above it
          // stay, and of its equals the lowest bytes
          const int holder = (int)(cut - 1) / 4;
          double last = s[0];
          last = (cut - 1) % 4 == 1 ? s[1] : last;
          last = (cut - 1) % 4 == 2 ? s[2] : last;
          last = (cut - 1) % 4 == 3 ? s[3] : last;
          last = __shfl(last, holder);
          uint32_t above = 0, equal = 0, before = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            above += __popcll(__ballot(x[j] > last));
            const uint64_t e = __ballot(x[j] == last);
            equal += __popcll(e);
            before += __popcll(e & (((uint64_t)1 << lane) - 1));
          }
          const uint32_t stay = cut - above;  // of the equals
          if (equal > stay) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (x[j] == last && before++ >= stay) w[j] = 0.0;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (x[j] < last) w[j] = 0.0;
        }
      }
      double total;
      double at = wave_before(w[0] + w[1] + w[2] + w[3], lane, total);
      // (a number outside [0, 1) is taken as the nearest inside, NaN as 0)
      const double u = __builtin_fmin(__builtin_fmax((double)number, 0.0), 0x1.fffffep-1) * total;
      uint32_t some = 256;
      double run[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) run[j] = at += w[j];
#pragma unroll
      for (int j = 3; j >= 0; --j)
        if (run[j] > u && w[j] > 0.0) some = 4 * lane + j;
      byte = wave_all(some, lane, Min32());
      if (byte == some) {
        double mine = w[0];
        mine = byte % 4 == 1 ? w[1] : mine;
        mine = byte % 4 == 2 ? w[2] : mine;
        mine = byte % 4 == 3 ? w[3] : mine;
        share = mine / total;
      }
    }
    if (lane == (int)(byte / 4)) {
      a.bytes[l * a.stride + t] = (uint8_t)byte;
      if (a.logp) a.logp[r] = (float)::log(share);
    }
  }
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, hipStream_t s) {
  const uint32_t rows = (uint32_t)a.q.lanes * (uint32_t)a.q.T;
  const uint32_t blocks = std::min<uint32_t>((rows + 3) / 4, MAX_BLOCKS);
  const bool wide = rows_by_16(a.logits.d, a.logits.lane, a.logits.row, 256, a.bf16 ? 2 : 4);
  if (a.bf16) BOA_LAUNCH(sample_kernel<uint16_t>, blocks, 256, 0, s, a, rows, wide);
  else BOA_LAUNCH(sample_kernel<float>, blocks, 256, 0, s, a, rows, wide);
  return hipGetLastError();
}

}  // namespace boa
