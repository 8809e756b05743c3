// The selective scan's sums across the lanes of a wave, over a type L of lane
// operations: the kernel's (DPP moves and lane swaps), or 64 modelled lanes on
// the CPU, where a test checks what every lane holds and that lanes that store
// to one address hold the same bits.
//
// Lanes i of a wave: TPC neighbours hold a channel, four states each; rows are
// 16 lanes.  L has, for a value x of each lane,
//   xor1(x), xor2(x)    x of lane i ^ 1, i ^ 2
//   half_mirror(x)      x of lane i ^ 7
//   ror8(x)             x of lane i ^ 8
//   fold16(x, y)        x + x of lane i ^ 16 in even rows, the same of y in odd ones
//   swap32(x, y)        x of lanes i and i + 32 in the lower half of the wave,
//                       y of lanes i - 32 and i in the upper one
//   pick(bit, x, y)     x where i has the bit, else y
//   fma(x, y, z)        x y + z, rounded once
#pragma once
#include <hip/hip_runtime.h>

namespace boa {

#define BOA_LANES __host__ __device__ __forceinline__

// Which four states of its channel a lane holds.  With four lanes a channel
// every other channel has them in reverse, so that half_mirror leads to the
// same states of the channel beside it (a rotation by four would cross into
// lanes that hold other states' sums by then).
template <int TPC>
BOA_LANES int lane_states(int lane) {
  return TPC == 4 && (lane & 4) ? 3 - lane % 4 : lane % TPC;
}

// The sums of y, I and M over a channel's lanes, in its lanes 0, 1 and from 2
// on (the same again in lanes 4 to 7)
template <int TPC, class L, class F>
BOA_LANES F channel_sums(const L& l, F y, F I, F M) {
  if constexpr (TPC == 8) {
    y = y + l.half_mirror(y);
    I = I + l.half_mirror(I);
    M = M + l.half_mirror(M);
  }
  const F yi = l.pick(1, I, y) + l.xor1(l.pick(1, y, I));
  M = M + l.xor1(M);
  return l.pick(2, M, yi) + l.xor2(l.pick(2, yi, M));
}

// A state's terms of dB and dC: dh du of lanes i and i + 32 in the lower half
// of the wave, h dy of lanes i - 32 and i in the upper one.  `c` is
// swap32(du, dy).
template <class L, class F, class P>
BOA_LANES F bc_term(const L& l, F dh, F h, const P& c) {
  const auto x = l.swap32(dh, h);
  return l.fma(x.b, c.b, x.a * c.a);
}

// dB and dC over the wave's channels from those terms: one state's sum a lane,
// at bc_slot of the 2 N sums.  With four lanes a channel two lanes have each.
template <int TPC, class L, class F>
BOA_LANES F bc_sums(const L& l, const F (&v)[4]) {
  const F x0 = l.fold16(v[0], v[2]), x1 = l.fold16(v[1], v[3]);
  F r = l.pick(8, x1, x0) + l.ror8(l.pick(8, x0, x1));
  if constexpr (TPC == 4) r = r + l.half_mirror(r);
  return r;
}
template <int TPC>
BOA_LANES int bc_slot(int lane) {
  return (lane >> 5) * 4 * TPC + 4 * lane_states<TPC>(lane) + ((lane >> 4) & 1) * 2 +
         ((lane >> 3) & 1);
}

}  // namespace boa
