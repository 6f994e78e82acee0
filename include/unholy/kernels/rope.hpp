// Rotary positions of heads, alone and behind the norms of queries and keys. No reference counterpart. (kv_append_rope of
// kv_cache.hpp is the form of a serving step, which also puts the keys and values into the paged cache.)
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace unholy::kernels {

using bf16 = uint16_t;

// How heads are rotated: channels [first, first + rot) of a head, in pairs (2i, 2i + 1) of that part (interleaved) or
// (i, i + rot / 2) (halves), pair i by the angle position * freq[i]:
//   (a, b) -> mscale (a cos - b sin, a sin + b cos).
// freq [rot / 2] (device, 8-byte aligned; null where rot is 0): radians a position. An angle's turns are cut off and its sine and
// cosine taken in 64 bits, these rounded once to 32 (with mscale), and what a far angle's product has past 64 bits counts: far
// positions are as exact as near ones (any position; |angles| below 2^40). rot even; rot 0: nothing is rotated. The other
// channels are left as they are.
struct Rope {
  const double* freq;
  int first, rot;
  bool interleaved;
  float mscale;
};

// Which frequencies of a longer context are slowed by `factor` (the context over the trained one):
//   kNone    none: base^(-2i / rot);
//   kLinear  all;
//   kTurns   in proportion between those that turn `low` times over the trained length (slowed) and `high` times (kept);
//   kPairs   between the same two, in proportion to the pair's number, ends rounded outwards to whole numbers.
enum class RopeScaling { kNone = 0, kLinear = 1, kTurns = 2, kPairs = 3 };
// h_freq [rot / 2] on the host. base > 1; factor >= 1; trained > 0 and high > low > 0 for kTurns and kPairs.
void rope_frequencies(double* h_freq, int rot, double base, RopeScaling scaling, double factor, double low, double high,
                      double trained);

// Rows x [rows, heads, dim] (row stride ldx), row r at position pos[r] (any int32; device), into y (row stride ldy). inverse:
// the transpose, which turns back (and, of a rotation with mscale 1, undoes it): the gradient of x from that of y. dim up to
// 1024, even or odd. y may be x (with ldy = ldx: then only the rotated part is read and written), otherwise they share no
// element. The operands need no alignment past their type's: the widest loads that strides and addresses allow are taken.
void rope(const bf16* x, int ldx, bf16* y, int ldy, const int32_t* pos, int rows, int heads, int dim, const Rope& r,
          bool inverse, hipStream_t st);

// Queries q [rows, Hq, dim] and keys k [rows, Hkv, dim], each head x divided by the root of (its mean square + eps) and times
// the weight of each channel, wq and wk [dim], then rotated as above, into qo and ko, in one launch. Sums and the rotation in
// fp32, one rounding to bf16 at the end (a head whose squares pass fp32, channels past 10^18, has no finite norm, and a channel
// whose product with its weight does no finite value; a head of zeros with eps 0 is 0 / 0). Row strides at least heads * dim; Hq
// or Hkv 0: no such operand. Aliasing as in rope.
void qk_norm_rope(const bf16* q, int ldq, bf16* qo, int ldqo, int Hq, const bf16* wq, const bf16* k, int ldk, bf16* ko,
                  int ldko, int Hkv, const bf16* wk, float eps, const int32_t* pos, int rows, int dim, const Rope& r,
                  hipStream_t st);

}  // namespace unholy::kernels
