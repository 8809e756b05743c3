// The steps of scan_lanes.h on 64 modelled lanes, on the CPU (host code only).
#include <cmath>
#include <utility>

#include "../boa-constrictor_amd/csrc/scan_lanes.h"

namespace {

struct Wave {
  float v[64];
};
Wave operator+(const Wave& x, const Wave& y) {
  Wave r;
  for (int i = 0; i < 64; ++i) r.v[i] = x.v[i] + y.v[i];
  return r;
}
Wave operator*(const Wave& x, const Wave& y) {
  Wave r;
  for (int i = 0; i < 64; ++i) r.v[i] = x.v[i] * y.v[i];
  return r;
}

// the instructions that the kernel uses, by their definitions
struct Model {
  struct Pair {
    Wave a, b;
  };
  template <class F>
  static Wave each(F f) {
    Wave r;
    for (int i = 0; i < 64; ++i) r.v[i] = f(i);
    return r;
  }
  Wave xor1(const Wave& x) const { return each([&](int i) { return x.v[i ^ 1]; }); }  // quad_perm 1 0 3 2
  Wave xor2(const Wave& x) const { return each([&](int i) { return x.v[i ^ 2]; }); }  // quad_perm 2 3 0 1
  Wave half_mirror(const Wave& x) const {  // lanes of 8 in reverse
    return each([&](int i) { return x.v[i / 8 * 8 + 7 - i % 8]; });
  }
  Wave ror8(const Wave& x) const {  // a row rotated by 8
    return each([&](int i) { return x.v[i / 16 * 16 + (i + 8) % 16]; });
  }
  // x's odd rows exchanged with y's even ones, and the sum of the two results
  Wave fold16(Wave x, Wave y) const {
    for (int i = 0; i < 64; ++i)
      if (i & 16) std::swap(x.v[i], y.v[i - 16]);
    return x + y;
  }
  // x's upper half exchanged with y's lower one
  Pair swap32(Wave x, Wave y) const {
    for (int i = 32; i < 64; ++i) std::swap(x.v[i], y.v[i - 32]);
    return Pair{x, y};
  }
  Wave pick(int bit, const Wave& x, const Wave& y) const {
    return each([&](int i) { return i & bit ? x.v[i] : y.v[i]; });
  }
  Wave fma(const Wave& x, const Wave& y, const Wave& z) const {
    return each([&](int i) { return std::fma(x.v[i], y.v[i], z.v[i]); });
  }
};

template <int TPC>
void run(const Wave* in, float* sums, float* bc, int* states, int* slot) {
  const Model l;
  const Wave s = boa::channel_sums<TPC>(l, in[0], in[1], in[2]);
  const Model::Pair c = l.swap32(in[3], in[4]);
  Wave v[4];
  for (int k = 0; k < 4; ++k) v[k] = boa::bc_term(l, in[5 + k], in[9 + k], c);
  const Wave r = boa::bc_sums<TPC>(l, v);
  for (int i = 0; i < 64; ++i) {
    sums[i] = s.v[i];
    bc[i] = r.v[i];
    states[i] = boa::lane_states<TPC>(i);
    slot[i] = boa::bc_slot<TPC>(i);
  }
}

}  // namespace

// in: 64 lanes each of y, I, M, du, dy, four dh and four h
extern "C" void lane_model(int tpc, const float* in, float* sums, float* bc, int* states, int* slot) {
  if (tpc == 4) run<4>((const Wave*)in, sums, bc, states, slot);
  else run<8>((const Wave*)in, sums, bc, states, slot);
}
