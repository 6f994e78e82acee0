// Rotary positions, alone and behind the norms of queries and keys (include/unholy/kernels/rope.hpp has the contracts).
#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>

#include "common.hpp"
#include "turn.hpp"

namespace unholy::kernels {

using namespace uh;
using namespace turn;

namespace {

constexpr int RT_NT = 256;

struct Side {
  const bf16* x;
  bf16* y;
  const bf16* w;
  int ldx, ldy, heads;
};
struct Turns {
  Side side[2];
  const int32_t* pos;
  Rope r;
  int rows, dim;
  int slots;       // of a head that are read and written
  int lanes;       // of a head: a power of two
  int wg_rows, wg_heads;  // of a workgroup
  float eps;
  bool inverse;
};

// A workgroup takes the heads [wg_heads y, ..) of wg_rows rows, a head a group of lanes: the rotations of its rows are worked
// out once, a pair a thread, and kept in LDS, while the first heads are on their way; a lane reads both channels of each of
// its pairs, so that only the sum of squares crosses lanes, and a head stays in registers between its norm and its rotation.
// Bound by HBM for many rows: each value is read and written once (8191 rows of 64 + 8 heads of 128 with norms: 62 us, 4.9
// TB/s, 4099 rows of 64 heads of 192 without: 43 us, 4.7 TB/s; a large copy reaches 4.8). A few rows take what a launch takes,
// with one load, one exchange through LDS and one store behind each other: 3.0 us for 7 x 40 heads of 80, 3.6 for 32 x 40 of
// 128.
template <int V, int N, bool NORM>
__global__ __launch_bounds__(RT_NT) void turn_kernel(Turns a) {
  extern __shared__ float2 cs[];  // [row][pair]
  const int tid = threadIdx.x, lane = tid & (a.lanes - 1), group = tid / a.lanes, groups = RT_NT / a.lanes;
  const int r0 = blockIdx.x * a.wg_rows, rows = min(a.wg_rows, a.rows - r0);
  const int heads = a.side[0].heads + a.side[1].heads, h0 = blockIdx.y * a.wg_heads, hn = min(a.wg_heads, heads - h0);
  const int vectors = rows * hn, pairs = a.r.rot / 2;

  Slot at[N];
  bool mine[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = lane + i * a.lanes;
    mine[i] = s < a.slots;
    at[i] = slot_of<V>(min(s, a.slots - 1), a.dim, a.r.first, a.r.rot, a.r.interleaved);
  }
  float w[2][NORM ? N : 1][2 * V];
  if constexpr (NORM) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        raw_t<V> x{}, y{};
        if (mine[i] && a.side[k].heads) {
          x = *reinterpret_cast<const raw_t<V>*>(a.side[k].w + at[i].a);
          if (at[i].b >= 0) y = *reinterpret_cast<const raw_t<V>*>(a.side[k].w + at[i].b);
        }
        unpack<V>(x, w[k][i]);
        unpack<V>(y, w[k][i] + V);
      }
  }
  raw_t<V> next[N][2];
  int row = 0;
  bool second = false;
  const auto head_of = [&](int v, int& row, int& h, bool& second) {
    row = v / hn;
    h = h0 + v - row * hn;
    second = h >= a.side[0].heads;
    if (second) h -= a.side[0].heads;
  };
  const auto load = [&](int v) {
    int h;
    head_of(v, row, h, second);
    const Side& s = a.side[second];
    const bf16* x = s.x + size_t(r0 + row) * s.ldx + size_t(h) * a.dim;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      next[i][0] = next[i][1] = raw_t<V>{};
      if (!mine[i]) continue;
      next[i][0] = *reinterpret_cast<const raw_t<V>*>(x + at[i].a);
      if (at[i].b >= 0) next[i][1] = *reinterpret_cast<const raw_t<V>*>(x + at[i].b);
    }
  };
  if (group < vectors) load(group);
  for (int i = tid; i < rows * pairs; i += RT_NT) {
    cs[i] = turn_of(a.pos[r0 + i / pairs], a.r.freq[i % pairs], a.r.mscale);
    if (a.inverse) cs[i].y = -cs[i].y;
  }
  __syncthreads();
  for (int v = group; v < vectors; v += groups) {  // (the lanes of a head leave together)
    float x[N][2 * V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      unpack<V>(next[i][0], x[i]);
      unpack<V>(next[i][1], x[i] + V);
    }
    int h, rr;
    bool k;
    head_of(v, rr, h, k);
    if (v + groups < vectors) load(v + groups);
    float scaled = 1.0f;
    if constexpr (NORM) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) ss = sum_squares<V>(x[i], ss);
      for (int o = a.lanes / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
      scaled = rms_scale(ss, a.dim, a.eps);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float ww[2 * V];
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) ww[j] = k ? w[1][i][j] : w[0][i][j];
        weigh<V>(x[i], ww);
      }
    }
    const Side& s = a.side[k];
    bf16* y = s.y + size_t(r0 + rr) * s.ldy + size_t(h) * a.dim;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!mine[i]) continue;
      if (at[i].turned) {
        float2 c[V];
#pragma unroll
        for (int j = 0; j < V; ++j) c[j] = cs[rr * pairs + (lane + i * a.lanes) * V + j];
        rotate<V>(x[i], c, a.r.interleaved);
      }
      if constexpr (NORM) scale<V>(x[i], scaled);
      *reinterpret_cast<raw_t<V>*>(y + at[i].a) = pack<V>(x[i]);
      if (at[i].b >= 0) *reinterpret_cast<raw_t<V>*>(y + at[i].b) = pack<V>(x[i] + V);
    }
  }
}

// Whether pieces of V channels fit: slots, strides and addresses.
bool fits(const Turns& a, int V, bool norm) {
  if (a.r.rot % (2 * V) || a.r.first % V || a.dim % V) return false;
  for (const Side& s : a.side) {
    if (!s.heads) continue;
    const uintptr_t p = reinterpret_cast<uintptr_t>(s.x) | reinterpret_cast<uintptr_t>(s.y) |
                        (norm ? reinterpret_cast<uintptr_t>(s.w) : 0);
    if (p % (2 * V) || s.ldx % V || s.ldy % V) return false;
  }
  return true;
}

template <int V, bool NORM>
void launch(Turns a, bool part, hipStream_t st) {
  a.slots = part ? a.r.rot / (2 * V) : slots_of<V>(a.dim, a.r.rot);
  if (a.slots == 0) return;
  a.lanes = 1;
  while (a.lanes < 64 && a.lanes < a.slots) a.lanes *= 2;
  const int heads = a.side[0].heads + a.side[1].heads, groups = RT_NT / a.lanes;
  a.wg_rows = std::clamp(groups / heads, 1, a.rows);
  const int chunks = int(cdiv(heads, groups));
  // As many heads as are done at a time, or where the rows fill the chip all of them, whose rotations are then worked out once
  // (40 heads of 128: 32 rows 3.6 us, all heads a workgroup 4.6; 768 rows 7.9 and 8.1, 1024 10.1 and 9.2, 2048 14.5 and 13.4)
  a.wg_heads = a.rows >= 1024 ? heads : int(cdiv(heads, chunks));
  const dim3 grid(cdiv(a.rows, a.wg_rows), cdiv(heads, a.wg_heads));
  const size_t lds = size_t(a.wg_rows) * (a.r.rot / 2) * sizeof(float2);
  const auto go = [&]<int N>() {
    turn_kernel<V, N, NORM><<<grid, RT_NT, lds, st>>>(a);
    UH_CHECK_LAUNCH();
  };
  const int per = int(cdiv(a.slots, a.lanes));  // slots a lane: 1024 channels are 8 / V of them at most
  if (per == 1) return go.template operator()<1>();
  if constexpr (V <= 4)
    if (per == 2) return go.template operator()<2>();
  if constexpr (V <= 2)
    if (per <= 4) return go.template operator()<4>();
  if constexpr (V == 1) go.template operator()<8>();
}
// The widest pieces that fit (8191 rows of 72 heads of 128: 59 us with pieces of 8 channels, 74 with 4; 32 rows of 40: 3.6 and
// 3.5).
template <bool NORM>
void launch_widest(const Turns& a, bool part, hipStream_t st) {
  if (fits(a, 8, NORM)) launch<8, NORM>(a, part, st);
  else if (fits(a, 4, NORM)) launch<4, NORM>(a, part, st);
  else if (fits(a, 2, NORM)) launch<2, NORM>(a, part, st);
  else launch<1, NORM>(a, part, st);
}

void check(const char* who, const Turns& a, bool norm) {
  const auto fail = [&](const char* what) { throw std::runtime_error(std::string(who) + ": " + what); };
  if (a.rows < 0) fail("rows < 0");
  if (a.dim < 1 || a.dim > 1024) fail("dim must be in [1, 1024]");
  check_rope(who, a.r, a.dim);
  for (const Side& s : a.side) {
    if (s.heads < 0 || s.heads > 65535) fail("heads must be in [0, 65535]");
    if (!s.heads || !a.rows) continue;
    if (!s.x || !s.y || (norm && !s.w)) fail("null operand");
    if (int64_t(s.ldx) < int64_t(s.heads) * a.dim || int64_t(s.ldy) < int64_t(s.heads) * a.dim)
      fail("row strides must be at least heads * dim");
    if (s.x == s.y && s.ldx != s.ldy) fail("in place with two strides");
    if ((reinterpret_cast<uintptr_t>(s.x) | reinterpret_cast<uintptr_t>(s.y) | reinterpret_cast<uintptr_t>(s.w)) % 2)
      fail("operands not 2-byte aligned");
  }
  if (a.rows && !a.pos) fail("null positions");
  if (reinterpret_cast<uintptr_t>(a.pos) % 4) fail("positions not 4-byte aligned");
}

}  // namespace

void rope_frequencies(double* h_freq, int rot, double base, RopeScaling scaling, double factor, double low, double high,
                      double trained) {
  const auto fail = [](const char* what) { throw std::runtime_error(std::string("rope_frequencies: ") + what); };
  if (rot < 0 || rot % 2) fail("rot even and not negative");
  if (!(base > 1.0) || !std::isfinite(base)) fail("base must be greater than 1 and finite");
  const int kind = int(scaling);
  if (kind < 0 || kind > 3) fail("unknown scaling");
  const bool some = scaling == RopeScaling::kTurns || scaling == RopeScaling::kPairs;
  if (scaling != RopeScaling::kNone && (!(factor >= 1.0) || !std::isfinite(factor))) fail("factor must be at least 1 and finite");
  if (some && (!(trained > 0.0) || !std::isfinite(trained) || !(low > 0.0) || !(high > low) || !std::isfinite(high)))
    fail("trained > 0 and high > low > 0 are wanted");
  if (rot && !h_freq) fail("null operand");
  const double turn = 2.0 * M_PI, lnb = std::log(base);
  // the pair, as a real number, that turns n times over the trained length
  const auto pair_of = [&](double n) { return rot * std::log(trained / (n * turn)) / (2.0 * lnb); };
  double from = 0.0, to = 0.0;  // kPairs: pairs up to `from` are kept, those from `to` on are slowed
  if (scaling == RopeScaling::kPairs) {
    from = std::max(std::floor(pair_of(high)), 0.0);
    to = std::max(std::min(std::ceil(pair_of(low)), double(rot - 1)), from);
  }
  for (int i = 0; i < rot / 2; ++i) {
    const double f = std::exp(-lnb * (2.0 * i / rot));
    double keep = 1.0;
    if (scaling == RopeScaling::kLinear) keep = 0.0;
    else if (scaling == RopeScaling::kTurns) keep = std::clamp((f * trained / turn - low) / (high - low), 0.0, 1.0);
    else if (scaling == RopeScaling::kPairs) keep = to > from ? std::clamp((to - i) / (to - from), 0.0, 1.0) : i <= from ? 1.0 : 0.0;
    h_freq[i] = keep == 1.0 ? f : f * (keep + (1.0 - keep) / factor);
  }
}

void rope(const bf16* x, int ldx, bf16* y, int ldy, const int32_t* pos, int rows, int heads, int dim, const Rope& r,
          bool inverse, hipStream_t st) {
  Turns a{{{x, y, nullptr, ldx, ldy, heads}, {}}, pos, r, rows, dim, 0, 0, 0, 0, 0.0f, inverse};
  check("rope", a, false);
  if (rows == 0 || heads == 0) return;
  launch_widest<false>(a, x == y, st);
}

void qk_norm_rope(const bf16* q, int ldq, bf16* qo, int ldqo, int Hq, const bf16* wq, const bf16* k, int ldk, bf16* ko,
                  int ldko, int Hkv, const bf16* wk, float eps, const int32_t* pos, int rows, int dim, const Rope& r,
                  hipStream_t st) {
  Turns a{{{q, qo, wq, ldq, ldqo, Hq}, {k, ko, wk, ldk, ldko, Hkv}}, pos, r, rows, dim, 0, 0, 0, 0, eps, false};
  check("qk_norm_rope", a, true);
  if (!(eps >= 0.0f) || !std::isfinite(eps)) throw std::runtime_error("qk_norm_rope: eps must be finite and not negative");
  if (rows == 0 || Hq + Hkv == 0) return;
  launch_widest<true>(a, false, st);
}

}  // namespace unholy::kernels
