// Kernel-level interface of the operators of a gated-delta-rule predictor
// (internal to the library): the norm with its residual and its gradient, rows
// and products in 8 bits, the gated delta rule and its gradient, the choice of
// a byte.  Rows are (lane, position) pairs as in train_kernels.h.
#pragma once
#include "train_kernels.h"

namespace boa {

// whether rows of `width` elements can be moved 16 bytes at a time
inline bool rows_by_16(const void* d, int64_t lane, int64_t row, int width, int size) {
  const int v = 16 / size;
  return ((uintptr_t)d & 15) == 0 && lane % v == 0 && row % v == 0 && width % v == 0;
}

// x with f applied over the 16 lanes of a row of lanes, and over all 64
template <typename F>
__device__ __forceinline__ float over16(float x, F f) {
  x = f(x, dpp_move<DPP_XOR1>(x));
  x = f(x, dpp_move<DPP_XOR2>(x));
  x = f(x, dpp_move<DPP_HALF_MIRROR>(x));
  return f(x, dpp_move<DPP_MIRROR>(x));
}
template <typename F>
__device__ __forceinline__ float over64(float x, F f) {
  x = over16(x, f);
  const auto a = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
  x = f(u2f(a[0]), u2f(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return f(u2f(b[0]), u2f(b[1]));
}
struct Sum {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};

// ---- norm and rows in 8 bits (norm.hip) ------------------------------------
struct NormArgs {
  Seqs q;
  int width;
  float eps;
  bool norm;            // false: the rows in 8 bits as they are
  bool bf16;
  RowsIn x, res;        // res.d may be null
  const float* weight;  // [width] or null (ones)
  RowsOut sum, out;     // d may be null
  RowsOut out8;         // int8 rows; d may be null
  float* scale8;        // [lanes][T]
};
hipError_t launch_norm(const NormArgs& a, hipStream_t s);

struct NormGradArgs {
  Seqs q;
  int width;
  float eps;
  bool bf16;
  RowsIn h, dout, dsum;  // dsum.d may be null
  const float* weight;   // or null (ones)
  RowsOut dx;
  float* dweight;        // [width] or null
  void* work;
};
size_t norm_grad_work(int64_t rows, int width);
hipError_t launch_norm_grad(const NormGradArgs& a, hipStream_t s);

// ---- products in 8 bits (int8.hip) -----------------------------------------
// weights [N][K] as the product reads them, zero past N and K
int64_t int8_packed_bytes(int N, int K);
hipError_t launch_int8_pack(const int8_t* w, int N, int K, void* packed, hipStream_t s);
struct Int8Args {
  Seqs q;
  int N, K;
  RowsIn x;             // int8 rows
  const float* xscale;  // [lanes][T]
  const void* packed;
  const float* wscale;  // [N]
  const float* bias;    // [N] or null
  RowsOut out;
  bool bf16;
};
hipError_t launch_int8(const Int8Args& a, hipStream_t s);

// ---- the choice of a byte (sample.hip) -------------------------------------
struct SampleHow {
  float temperature, top_k, top_p, min_p;
};
struct SampleArgs {
  Seqs q;
  RowsIn logits;
  const float* bias;     // [256] or null
  const float* uniform;  // [lanes][T]
  SampleHow how;
  const SampleHow* each; // [lanes] on the device, or null: `how` for all
  uint8_t* bytes;        // byte (l, t) at l * stride + t
  int64_t stride;
  float* logp;           // [lanes][T] or null
  bool bf16;
};
hipError_t launch_sample(const SampleArgs& a, hipStream_t s);

// ---- the gated delta rule (delta_rule.hip) ---------------------------------
struct DeltaArgs {
  Seqs q;
  int H, HV, dk, dv;      // heads of q and k, heads of v, their widths
  float scale;
  bool unit;              // q and k through their lengths
  bool bf16;
  RowsIn qr, k, v, g, beta;
  const float* state_in;  // [lanes][HV][dk][dv] or null (zero)
  RowsOut out;
  float* state_out;       // or null
  float* saved;           // or null
  void* work;
};
struct DeltaGradArgs {
  DeltaArgs f;  // the forward's inputs and what it saved
  RowsIn dout;
  const float* dstate_out;  // or null (zero)
  RowsOut dq, dk, dv, dg, dbeta;
  float* dstate_in;         // or null
};
int64_t delta_saved_floats(int lanes, int T, int H, int HV, int dk, int dv);
int64_t delta_work_bytes(int lanes, int T, int H, int HV, int dk, int dv, bool grad);
hipError_t launch_delta(const DeltaArgs& a, hipStream_t s);
hipError_t launch_delta_grad(const DeltaGradArgs& a, hipStream_t s);

}  // namespace boa
