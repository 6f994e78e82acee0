// Heads as the kernels that rotate them hold them: slots of twice V channels, which a lane reads, normalises and rotates by
// itself.
#pragma once

#include "common.hpp"
#include "numerics.hpp"
#include "unholy/kernels/rope.hpp"

namespace unholy::kernels::turn {

using namespace uh;

// V values of bf16, as one load.
template <int V>
struct Raw;
template <>
struct Raw<8> { using type = uint4; };
template <>
struct Raw<4> { using type = uint2; };
template <>
struct Raw<2> { using type = uint32_t; };
template <>
struct Raw<1> { using type = uint16_t; };
template <int V>
using raw_t = typename Raw<V>::type;

template <int V>
__device__ __forceinline__ void unpack(const raw_t<V>& x, float* v) {
  if constexpr (V == 1) {
    v[0] = bf16_to_f32(x);
  } else {
    uint32_t w[V / 2];
    __builtin_memcpy(w, &x, sizeof(w));
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <int V>
__device__ __forceinline__ raw_t<V> pack(const float* v) {
  if constexpr (V == 1) {
    return f32_to_bf16(v[0]);
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {  // (both in one instruction)
      typedef float f32x2 __attribute__((ext_vector_type(2)));
      typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
      w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[2 * i], v[2 * i + 1]}, bf16x2));
    }
    raw_t<V> x;
    __builtin_memcpy(&x, w, sizeof(w));
    return x;
  }
}

// A head's slots: first those of the rotated part, each V pairs (pair V s + j of slot s: halves: channel j of both pieces;
// interleaved: channels 2j and 2j + 1 of the two pieces side by side), then the other channels, two pieces a slot, of which the
// last may be alone. rot % 2V, first % V and dim % V are 0.
struct Slot {
  int a, b;  // the first channels of its pieces; b < 0: none
  bool turned;
};
template <int V>
__host__ __device__ __forceinline__ int slots_of(int dim, int rot) {
  return rot / (2 * V) + (dim - rot + 2 * V - 1) / (2 * V);
}
template <int V>
__device__ __forceinline__ Slot slot_of(int s, int dim, int first, int rot, bool interleaved) {
  const int turned = rot / (2 * V);
  if (s < turned)
    return interleaved ? Slot{first + 2 * V * s, first + 2 * V * s + V, true} : Slot{first + V * s, first + rot / 2 + V * s, true};
  const int u = 2 * V * (s - turned), w = u + V;  // of the channels that are not rotated
  return Slot{u < first ? u : u + rot, w >= dim - rot ? -1 : w < first ? w : w + rot, false};
}

// The two factors of a rotation: (cos, sin) of pos * freq, times mscale, rounded once. In 64 bits, a rotation's factors serve
// many channels: the angle in quarters of a turn, of which whole ones are cut off, and at most an eighth of a turn is left,
// whose sine and cosine are their Taylor series (up to the 11th and 12th power: the next terms are below 2^-37). Far positions
// lose nothing: quarters a position are two numbers, of which the first has 21 bits and its product with a position (32 bits) is
// exact, and the second is below 2^-20 of it and holds what 2 / pi and freq's product have past 64 bits (an angle is off by
// 2^-72 of it, and by 2^-52 of what is left; one rounded product for the angle is off by 2^-52 of it: 2^-21 at position 2^31).
__device__ __forceinline__ float2 turn_of(int pos, double freq, float mscale) {
#pragma clang fp contract(off)
  constexpr double kQuarters = 0.63661977236758134308, kQuartersRest = -3.9357353350364972e-17;  // 2 / pi: 64 bits, the rest
  constexpr double kQuarter = 1.57079632679489661923;  // in radians
  const double p = double(pos);
  const double hi = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, freq * kQuarters) & 0xffffffff00000000u);
  const double lo = __builtin_fma(freq, kQuartersRest, __builtin_fma(freq, kQuarters, -hi));
  const double much = p * hi, quarters = rint(__builtin_fma(p, lo, much));
  const double a = __builtin_fma(p, lo, much - quarters) * kQuarter, z = a * a;
  double s = -1.0 / 39916800.0, c = 1.0 / 479001600.0;
  s = __builtin_fma(s, z, 1.0 / 362880.0);
  c = __builtin_fma(c, z, -1.0 / 3628800.0);
  s = __builtin_fma(s, z, -1.0 / 5040.0);
  c = __builtin_fma(c, z, 1.0 / 40320.0);
  s = __builtin_fma(s, z, 1.0 / 120.0);
  c = __builtin_fma(c, z, -1.0 / 720.0);
  s = __builtin_fma(s, z, -1.0 / 6.0);
  c = __builtin_fma(c, z, 1.0 / 24.0);
  s = __builtin_fma(s * z, a, a);
  c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  const int q = int(__builtin_bit_cast(uint64_t, quarters + 0x1.8p52)) & 3;  // (the sum's last bits are a whole number's)
  const double x = q & 1 ? -s : c, y = q & 1 ? c : s, m = q & 2 ? -double(mscale) : double(mscale);
  return make_float2(float(x * m), float(y * m));
}

// The slot's V pairs rotated; cs: (cos, sin) of each. v: the two pieces one after the other.
template <int V>
__device__ __forceinline__ void rotate(float (&v)[2 * V], const float2* cs, bool interleaved) {
#pragma clang fp contract(off)  // (each product and sum as written: every kernel that rotates rounds alike)
  const auto pair = [&](float& a, float& b, int j) {
    const float c = cs[j].x, s = cs[j].y, x = a, y = b;
    a = __builtin_fmaf(x, c, -(y * s));
    b = __builtin_fmaf(x, s, y * c);
  };
  if (interleaved) {
#pragma unroll
    for (int j = 0; j < V; ++j) pair(v[2 * j], v[2 * j + 1], j);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) pair(v[j], v[V + j], j);
  }
}

// 1 / root of the mean square of a head whose channels' squares sum to ss.
__device__ __forceinline__ float rms_scale(float ss, int dim, float eps) {
#pragma clang fp contract(off)
  return 1.0f / sqrtf(ss / float(dim) + eps);
}
template <int V>
__device__ __forceinline__ float sum_squares(const float (&v)[2 * V], float ss) {
#pragma unroll
  for (int j = 0; j < 2 * V; ++j) ss = __builtin_fmaf(v[j], v[j], ss);
  return ss;
}
// A normalised head is r w x, rotated: the products w x of two bf16 numbers are exact, and r, which all of a head's channels
// have in common, comes last, so that a channel has a rounding less.
template <int V>
__device__ __forceinline__ void weigh(float (&v)[2 * V], const float (&w)[2 * V]) {
#pragma unroll
  for (int j = 0; j < 2 * V; ++j) v[j] *= w[j];
}
template <int V>
__device__ __forceinline__ void scale(float (&v)[2 * V], float r) {
#pragma unroll
  for (int j = 0; j < 2 * V; ++j) v[j] *= r;
}

// Argument checks of every entry that rotates.
inline void check_rope(const char* who, const Rope& r, int dim) {
  const auto fail = [&](const char* what) { throw std::runtime_error(std::string(who) + ": " + what); };
  if (r.rot < 0 || r.rot % 2 || r.first < 0 || r.first > dim || r.rot > dim - r.first) fail("rot even, first + rot <= dim");
  if (!(r.mscale - r.mscale == 0.0f)) fail("mscale is not finite");
  if (r.rot && !r.freq) fail("null frequencies");
  if (reinterpret_cast<uintptr_t>(r.freq) % 8) fail("frequencies not 8-byte aligned");
}

}  // namespace unholy::kernels::turn
