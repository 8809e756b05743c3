// Kernel-level interface of the training operators (internal to the library):
// embedding and its gradient, the selective scan and its gradient, the
// next-byte loss.  Rows are (lane, position) pairs of `lanes` sequences of T.
#pragma once
#include <cstddef>

#include "boa_kernels.h"

namespace boa {

// most blocks of a launch whose blocks loop over what is left: a grid's
// threads have to stay under 2^32
constexpr uint32_t MAX_BLOCKS = 1u << 22;

// rows of a tensor: element (l, t, i) at d[l * lane + t * row + i]
struct RowsIn {
  const void* d;
  int64_t lane, row;
};
struct RowsOut {
  void* d;
  int64_t lane, row;
};

// the sequences: lane l has min(max(lens[l], 0), T) positions, T where lens is null
struct Seqs {
  int lanes, T;
  const int32_t* lens;
};
__device__ __forceinline__ int seq_len(const Seqs& q, int l) {
  if (!q.lens) return q.T;
  const int n = q.lens[l];
  return n < 0 ? 0 : (n < q.T ? n : q.T);
}

// four floats at any float's address
typedef float f4_any __attribute__((ext_vector_type(4), aligned(4)));

// bfloat16 of two floats by one instruction, x in the low half
__device__ __forceinline__ uint32_t bf16_pair(float x, float y) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{x, y}, b2));
}

// x + x of the lane that CTRL names within the row of 16 lanes
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140,
              DPP_ROR8 = 0x128;
template <int CTRL>
__device__ __forceinline__ float dpp_move(float x) {
  return u2f((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f2u(x), CTRL, 0xF, 0xF, true));
}
template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) { return x + dpp_move<CTRL>(x); }
// sum of x's lower half and y's upper half partner: lanes 0 .. 31 get x[i] +
// x[i + 32], lanes 32 .. 63 get y[i - 32] + y[i]
__device__ __forceinline__ float fold32(float x, float y) {
  const auto s = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(y), false, false);
  return u2f(s[0]) + u2f(s[1]);
}
// likewise for the rows of 16 lanes: even rows get x, odd rows y
__device__ __forceinline__ float fold16(float x, float y) {
  const auto s = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(y), false, false);
  return u2f(s[0]) + u2f(s[1]);
}
// ---- embedding (train_ops.hip) -------------------------------------------
struct EmbedArgs {
  Seqs q;
  const uint8_t* tok;  // token (l, t) at tok[l * tok_lane + t]
  int64_t tok_lane;
  const void* table;   // [256][width]
  int width;
  float scale;
  RowsOut out;
  bool bf16;
};
hipError_t launch_embed(const EmbedArgs& a, hipStream_t s);

struct EmbedGradArgs {
  Seqs q;
  const uint8_t* tok;
  int64_t tok_lane;
  RowsIn dout;
  int width;
  float scale;
  float* dtable;  // [256][width]
  void* work;
  bool bf16;
};
size_t embed_grad_work(int64_t rows, int width);
hipError_t launch_embed_grad(const EmbedGradArgs& a, hipStream_t s);

// ---- next-byte loss (train_ops.hip) --------------------------------------
struct LossArgs {
  Seqs q;
  RowsIn logits;
  const uint8_t* tgt;
  int64_t tgt_lane;
  const float* bias;  // [256] or null
  float scale;
  float* loss;        // [lanes][T]
  float* total;       // [1] or null
  RowsOut dlogits;    // d may be null
  float* dbias;       // [256] or null
  void* work;
  bool bf16;
};
size_t loss_work(int64_t rows);
hipError_t launch_loss(const LossArgs& a, hipStream_t s);

// ---- selective scan (train_scan.hip) -------------------------------------
constexpr int SCAN_TILE = 16;  // positions between two saved states
struct ScanArgs {
  Seqs q;
  int C;      // channels
  int ds;     // states a channel: 16 or 32
  RowsIn u, delta, z, b, c;
  const float *A, *D, *bias;
  const float* state_in;  // [lanes][C][ds] or null (zero)
  RowsOut out;
  float* state_out;       // or null
  float* saved;           // [lanes][tiles][C][ds] or null
  void* work;
  bool bf16;
};
struct ScanGradArgs {
  ScanArgs f;  // the forward's inputs and its saved states
  RowsIn dout;
  const float* dstate_out;  // or null (zero)
  RowsOut du, ddelta, dz, db, dc;
  float *dA, *dD, *dbias;
  float* dstate_in;         // or null
};
int64_t scan_saved_floats(int lanes, int T, int C, int ds);
size_t scan_work(int lanes, int T, int C, int ds, bool grad);
hipError_t launch_scan(const ScanArgs& a, hipStream_t s);
hipError_t launch_scan_grad(const ScanGradArgs& a, hipStream_t s);

}  // namespace boa
