// Attention of a step's rows over the 8-bit paged key / value cache (include/unholy/kernels/kv_cache.hpp has the layout
// and the contract).
#include <algorithm>
#include <cmath>

#include "kv_internal.hpp"
#include "numerics.hpp"

namespace unholy::kernels {

using namespace uh;
using namespace kv;

namespace {

constexpr int TILE = 64;          // tokens a wave takes at a time
constexpr int AT_NT = 256;        // threads of a workgroup
constexpr int AT_WAVES = AT_NT / 64;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

// Bits of the first n of up to 16 tokens.
__device__ __forceinline__ uint32_t first_bits(int n) { return (1u << min(max(n, 0), 16)) - 1; }
// Which of the 16 tokens from t on a row at position p sees.
__device__ __forceinline__ uint32_t seen_bits(int p, int t, int window, int sinks) {
  uint32_t see = first_bits(p - t + 1);
  if (window > 0) see &= ~first_bits(int(min(int64_t(p) - window - t + 1, int64_t(16)))) | first_bits(sinks - t);
  return see;
}
// Inclusive sum over the wave's lanes (all active): DPP shifts within rows of 16, then the rows' last lanes.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  const auto step = [](uint32_t x, auto ctrl, auto rows) {
    return x + uint32_t(__builtin_amdgcn_update_dpp(0, int(x), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  v = step(v, integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});  // row_shr:1
  v = step(v, integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  v = step(v, integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  v = step(v, integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  v = step(v, integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // row_bcast:15 into rows 1 and 3
  return step(v, integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});  // row_bcast:31 into rows 2 and 3
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) { return uint32_t(__builtin_amdgcn_readlane(int(v), lane)); }

// What every workgroup knows of the call.
struct Attend {
  const bf16* q;
  bf16* out;
  float* lse;
  KvStep st;
  KvCache c;
  int ldq, ldo, group, page_shift, window, sinks;
  float scale2;  // scale * log2(e): the kernels take powers of two
  int target;    // workgroups that the chip holds at a time
  int rounds;    // of them, where segments are many
  uint32_t* counters;  // of finished pieces, [slot]; zero between launches
  float *po, *pml;     // partial sums: values [slot][ROWS][D]; maximum and weight sum [slot][ROWS][2]
};

// The 64-token tiles that some row of a sequence sees: with a window the sinks' tiles [0, sink_tiles) and those from
// `skip` on, else all; count of them, numbered in order.
struct Tiles {
  int sink_tiles, skip, count;
  __device__ __forceinline__ int at(int i) const { return i < sink_tiles ? i : i - sink_tiles + skip; }
};
__device__ __forceinline__ Tiles tiles_of(const Attend& a, const Seq& q) {
  const int64_t cap = int64_t(a.st.max_blocks) << a.page_shift;
  const int end = int((min(int64_t(q.len), cap) + TILE - 1) / TILE);
  Tiles t{0, 0, end};
  if (a.window > 0) {
    const int64_t lo = int64_t(q.first) - a.window + 1;  // the first token in the first row's window
    t.skip = min(int(max(lo, int64_t(0)) / TILE), end);
    t.sink_tiles = min(int((int64_t(a.sinks) + TILE - 1) / TILE), t.skip);
    t.count = end - t.skip + t.sink_tiles;
  }
  return t;
}
__device__ __forceinline__ int row_groups(int rows, int per) { return (rows + per - 1) / per; }

// The split of a launch's work, worked out by every workgroup from the lengths, which only the device knows: a segment is
// a (sequence, key / value head, row group) and its tiles; each is cut into pieces of at most `share` tiles, as equal as
// they can be, a workgroup each. share makes about `target` pieces, so that long and short sequences load the chip evenly.
// A segment of several pieces leaves partial sums in slots slot0 .. slot0 + pieces - 1: with u the tiles before it in the
// launch and f = u / share, slots from 2 f on, of which there are 2 (f' - f) >= 2 floor(tiles / share) >= pieces before the
// next segment's.
struct Piece {
  int b, h, rg, index, pieces, i0, i1, slot0;
};
__device__ __forceinline__ uint32_t pieces_of(uint32_t tiles, uint32_t share) {
  return max((tiles + share - 1) / share, 1u);  // (no tiles: a piece that writes zeros)
}
// Every wave for itself, a sequence a lane: no barriers, and for up to 64 sequences one pass over registers.
template <int ROWS, int LEAST>
__device__ __forceinline__ bool find_piece(const Attend& a, Piece& p, Seq& q, Tiles& t) {
  const int lane = threadIdx.x & 63;
  Tiles mt{0, 0, 0};
  uint32_t segs = 0;  // of this lane's sequence
  const auto look = [&](int b) {
    segs = 0;
    mt = Tiles{0, 0, 0};
    if (b < a.st.B) {
      q = seq_of(a.st, b);
      segs = uint32_t(row_groups((q.r1 - q.r0) * a.group, ROWS)) * a.c.heads;
      if (segs) mt = tiles_of(a, q);
    }
  };
  float tiles = 0.0f;
  uint32_t all = 0;
  for (int b0 = 0; b0 < a.st.B; b0 += 64) {
    look(b0 + lane);
    tiles += wave_sum(float(mt.count) * float(segs));
    all += lane_of(wave_scan(segs), 63);
  }
  // about `target` pieces where the segments are few, one round of the chip; else more and smaller ones than it holds, which
  // even out as they come and go
  const float want = float(all <= uint32_t(a.target) / 2 ? a.target - int(all) : a.target * a.rounds);
  // (past 2^31 tiles the prefix below would wrap: no segment is cut then)
  const uint32_t share = tiles < 2.0e9f ? max(uint32_t(ceilf(tiles * 1.0001f / want)), uint32_t(LEAST)) : 1u << 30;
  uint32_t wg0 = 0, u0 = 0;
  for (int b0 = 0; b0 < a.st.B; b0 += 64) {
    if (a.st.B > 64) look(b0 + lane);
    const uint32_t n = segs * pieces_of(uint32_t(mt.count), share), u = segs * uint32_t(mt.count);
    const uint32_t wg_end = wg0 + wave_scan(n), u_end = u0 + wave_scan(u);
    const uint64_t hit = __ballot(blockIdx.x < wg_end);
    if (hit) {
      const int l = __ffsll((unsigned long long)hit) - 1;  // (a lane of no segments ends where the one before it does)
      p.b = b0 + l;
      q = Seq{int(lane_of(q.r0, l)), int(lane_of(q.r1, l)), int(lane_of(q.len, l)), int(lane_of(q.first, l))};
      t = Tiles{int(lane_of(mt.sink_tiles, l)), int(lane_of(mt.skip, l)), int(lane_of(mt.count, l))};
      const uint32_t sg = lane_of(segs, l), first = lane_of(wg_end - n, l), ut = lane_of(u_end - u, l);
      const uint32_t rgs = sg / uint32_t(a.c.heads), pieces = pieces_of(uint32_t(t.count), share);
      const uint32_t in = blockIdx.x - first, seg = in / pieces, i = in % pieces;
      const uint32_t each = uint32_t(t.count) / pieces, more = uint32_t(t.count) % pieces;
      p.index = int(i);
      p.pieces = int(pieces);
      p.h = int(seg / rgs);
      p.rg = int(seg % rgs);
      p.i0 = int(i * each + min(i, more));
      p.i1 = p.i0 + int(each + (i < more ? 1 : 0));
      p.slot0 = int((ut + seg * uint32_t(t.count)) / share * 2);
      return true;
    }
    wg0 = lane_of(wg_end, 63);
    u0 = lane_of(u_end, 63);
  }
  return false;
}

__device__ __forceinline__ bf16x8 bf16x8_of(uint4 v) { return __builtin_bit_cast(bf16x8, v); }
__device__ __forceinline__ uint4 ld16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ uint32_t nan_bytes(uint32_t x) {  // the high bit of each byte that is a NaN code
  return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// ---- few rows a sequence: decode and verify steps ---------------------------------------------------------------------
// Bound by reading the cache once. A wave takes 16 rows ((token, query head) pairs that share a key / value head) and
// 16 J tokens at a time straight from the cache into registers, no LDS: with S^T = K Q^T the 16x16 product leaves lane
// (row c, group g) the scores of tokens 4g .. 4g + 3 of a 16-token tile, and the tiles' rows are taken in such an order of
// tokens (tile j, row r: token 4J (r / 4) + 4j + r % 4) that over the J tiles these are tokens 4J g .. 4J g + 4J - 1: the
// very tokens whose values one load of the transposed cache gives it for O^T = V^T P^T. The weights go from one product
// to the other in place, and a row's running maximum and sum are its lane's own.
// The codes become bf16 exactly (v_cvt_scalef32, the block's scale with them), the products sum in fp32; the weights are
// rounded to bf16 for the second product (2^-8 of each at most, as much as the output's own rounding), their sum is taken in
// fp32 before that.
// The four waves are RW sets of 16 rows (they read the same tokens, which L1 serves) times 4 / RW that take every
// (4 / RW)-th tile and are joined in LDS. The workgroup that finishes last of those that share rows adds their partial
// sums, in the order of the tiles whichever it is: the result does not depend on timing.
template <int D, int RW>
struct Split {
  static constexpr int J = D == 256 ? 2 : 4;  // (four tiles of 256 channels do not leave room for two waves)
  static constexpr int TOK = 16 * J;
  static constexpr int TW = AT_WAVES / RW;  // waves that share rows
  static constexpr int ROWS = 16 * RW;
  static constexpr int KL = D / 64;  // 16-byte loads of a key row's quarter
  static constexpr int DT = D / 16;  // 16-channel tiles
  struct Lds {
    float o[TW > 1 ? AT_WAVES / 2 : 1][16 * D];
    float ml[AT_WAVES][16][2];
  };
};
constexpr int kTarget = 512;  // two workgroups on each CU
constexpr int kMostSlots = 4 * kTarget;
constexpr size_t kCounterBytes = kMostSlots * sizeof(uint32_t);
constexpr int rounds_of(int rw) { return rw == 4 ? 1 : 2; }
constexpr int slots_of(int rw) { return 2 * kTarget * rounds_of(rw); }  // two a share of the tiles

// Partial sums pass between workgroups on different XCDs, whose L2 caches do not see each other's lines: stored through
// to memory and read from there (device-scope accesses), which for these few KiB is far cheaper than the fences that
// write back and invalidate a whole L2 (a layer of a single-token step over 4097 tokens, 17 pieces a
// head: 25.0 us with fences, 13.9 with these).
constexpr int SC1 = 16;  // the cache policy of a device-scope access
constexpr int JOIN = 8;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t sums_of(float* p) {
  return __builtin_amdgcn_make_buffer_rsrc(p, 0, 0x7fffffff, 0x00027000);
}
__device__ __forceinline__ void put4(__amdgpu_buffer_rsrc_t p, int at, v4f v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(__attribute__((ext_vector_type(4))) unsigned, v), p, at * 4, 0,
                                         SC1);
}
__device__ __forceinline__ void put2(__amdgpu_buffer_rsrc_t p, int at, float x, float y) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  __builtin_amdgcn_raw_buffer_store_b64(u2{__float_as_uint(x), __float_as_uint(y)}, p, at * 4, 0, SC1);
}
__device__ __forceinline__ v4f get4(__amdgpu_buffer_rsrc_t p, int at) {
  return __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(p, at * 4, 0, SC1));
}
__device__ __forceinline__ float2 get2(__amdgpu_buffer_rsrc_t p, int at) {
  const auto v = __builtin_amdgcn_raw_buffer_load_b64(p, at * 4, 0, SC1);
  return make_float2(__uint_as_float(v[0]), __uint_as_float(v[1]));
}

template <int D>
__device__ __forceinline__ void store_out(const Attend& a, int row, int hq, int d, v4f o, float l, float m, bool first) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = f32_to_bf16(l == 0.0f ? 0.0f : o[e] * inv);
  *reinterpret_cast<uint2*>(a.out + size_t(row) * a.ldo + size_t(hq) * D + d) =
      make_uint2(uint32_t(w[0]) | uint32_t(w[1]) << 16, uint32_t(w[2]) | uint32_t(w[3]) << 16);
  if (first && a.lse) a.lse[size_t(row) * (a.group * a.c.heads) + hq] = l == 0.0f ? -INFINITY : m * LN2 + logf(l);
}

template <int D, int RW>
__global__ __launch_bounds__(AT_NT, 2) void kv_split_kernel(Attend a) {
  using S = Split<D, RW>;
  constexpr int J = S::J, TOK = S::TOK, TW = S::TW;
  __shared__ __align__(16) typename S::Lds lds;
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
  Piece pc;
  Seq q;
  Tiles tiles;
  if (!find_piece<S::ROWS, TW>(a, pc, q, tiles)) return;
  const int b = pc.b, h = pc.h, nrows = (q.r1 - q.r0) * a.group, row0 = pc.rg * S::ROWS + wave / TW * 16;

  // this lane's row (the last one where there are fewer): its position
  const int ri = min(row0 + c, nrows - 1), my_row = q.r0 + ri / a.group, my_hq = h * a.group + ri % a.group;
  const int pos = q.first + ri / a.group;
  const int pos_lo = q.first + min(row0, nrows - 1) / a.group;  // of the wave's rows
  const int pos_hi = q.first + min(row0 + 15, nrows - 1) / a.group;

  v4f o[S::DT];
  float mx = -INFINITY, l = 0.0f;
#pragma unroll
  for (int d = 0; d < S::DT; ++d) o[d] = v4f{0, 0, 0, 0};

  const int mask = a.c.page - 1, sh = a.page_shift;
  const auto lookup = [&](int t0, int& pk, int& pv) {  // the pages of this lane's key rows and of its values
    pk = page_of(a.st.table, a.st.max_blocks, a.c.pages, b, (t0 + 4 * J * (c >> 2)) >> sh);
    pv = page_of(a.st.table, a.st.max_blocks, a.c.pages, b, (t0 + 4 * J * g) >> sh);
  };
  uint4 kr[J][S::KL];
  uint32_t vr[S::DT][J];
  int ksb, vsb;
  const auto load_k = [&](int t0, int pk) {
    const size_t ph = size_t(max(pk, 0)) * a.c.heads + h;
    const uint8_t* p = a.c.k + ((ph << sh) + ((t0 + 4 * J * (c >> 2) + (c & 3)) & mask)) * D + 16 * g;
    ksb = a.c.ks[ph];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int m = 0; m < S::KL; ++m) kr[j][m] = ld16(p + 4 * j * D + 64 * m);
  };
  const auto load_v = [&](int t0, int pv) {
    const size_t ph = size_t(max(pv, 0)) * a.c.heads + h;
    const uint8_t* p = a.c.v + ((ph * D + c) << sh) + ((t0 + 4 * J * g) & mask);
    vsb = a.c.vs[ph];
#pragma unroll
    for (int d = 0; d < S::DT; ++d) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(p);
      p += 16 << sh;
      if constexpr (J == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(w);
        vr[d][0] = x.x, vr[d][1] = x.y, vr[d][2] = x.z, vr[d][3] = x.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(w);
        vr[d][0] = x.x, vr[d][1] = x.y;
      }
    }
  };
  // a 64-token tile is 64 / TOK steps; steps go to the waves in turn
  constexpr int PER = TILE / TOK;
  const auto token = [&](int i) { return tiles.at(i / PER) * TILE + i % PER * TOK; };
  const int i1 = pc.i1 * PER;
  int i = pc.i0 * PER + wave % TW, pk = 0, pv = 0, pk1 = 0, pv1 = 0;
  if (row0 >= nrows) i = i1;  // no rows for this wave
  if (i < i1) lookup(token(i), pk, pv);
  bf16x8 qf[2 * S::KL];
  {
    const bf16* x = a.q + size_t(my_row) * a.ldq + size_t(my_hq) * D + 16 * g;
#pragma unroll
    for (int m = 0; m < S::KL; ++m) {
      qf[2 * m] = bf16x8_of(*reinterpret_cast<const uint4*>(x + 64 * m));
      qf[2 * m + 1] = bf16x8_of(*reinterpret_cast<const uint4*>(x + 64 * m + 8));
    }
  }
  if (i < i1) {
    load_k(token(i), pk);
    load_v(token(i), pv);
    if (i + TW < i1) lookup(token(i + TW), pk1, pv1);
  }
  for (; i < i1; i += TW) {
    const int t0 = token(i);
    const bool more = i + TW < i1;
    const int tn = token(more ? i + TW : i);
    const float ks = e8m0_to_f32(uint8_t(ksb));
    v4f s[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      s[j] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int m = 0; m < S::KL; ++m) {
        s[j] = mfma_bf16(fp8x8_to_bf16(kr[j][m].x, kr[j][m].y, ks), qf[2 * m], s[j]);
        s[j] = mfma_bf16(fp8x8_to_bf16(kr[j][m].z, kr[j][m].w, ks), qf[2 * m + 1], s[j]);
      }
    }
    const int pvt = pv;
    if (more) {
      pk = pk1, pv = pv1;
      load_k(tn, pk);
      if (i + 2 * TW < i1) lookup(token(i + 2 * TW), pk1, pv1);
    }
    // what a row does not see: only in the tiles at the ends of what the rows see
    const bool masked = t0 + TOK - 1 > pos_lo || __any(pvt < 0) ||
                        (a.window > 0 && int64_t(t0) + a.window <= pos_hi && t0 + TOK > a.sinks);
    uint32_t see = 0xffff;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < J; ++j) s[j] *= a.scale2;
    if (masked) {
      see = pvt < 0 ? 0 : seen_bits(pos, t0 + 4 * J * g, a.window, a.sinks);
#pragma unroll
      for (int k = 0; k < 4 * J; ++k) s[k / 4][k % 4] = see >> k & 1 ? s[k / 4][k % 4] : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < 4 * J; ++k) top = fmaxf(top, s[k / 4][k % 4]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float m1 = fmaxf(mx, top), ref = m1 == -INFINITY ? 0.0f : m1;
    if (__any(m1 != mx)) {
      const float al = __builtin_amdgcn_exp2f(mx - ref);
#pragma unroll
      for (int d = 0; d < S::DT; ++d) o[d] *= al;
      l *= al;
    }
    mx = m1;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[j][e] = __builtin_amdgcn_exp2f(s[j][e] - ref);
        l += s[j][e];
      }
    const float vs = e8m0_to_f32(uint8_t(vsb));
    bf16x8 p[J / 2];
#pragma unroll
    for (int hf = 0; hf < J / 2; ++hf)
#pragma unroll
      for (int e = 0; e < 8; ++e) p[hf][e] = __bf16(s[2 * hf + e / 4][e % 4]);
    uint32_t bad = 0;
    if (masked) {  // slots past the last token hold anything: zero; NaN among the values that some row sees: below
      const int n = pvt < 0 ? 0 : min(max(q.len - (t0 + 4 * J * g), 0), 4 * J);
#pragma unroll
      for (int k = 0; k < J; ++k) {
        const uint32_t keep = n >= 4 * k + 4 ? ~0u : n <= 4 * k ? 0u : (1u << (8 * (n - 4 * k))) - 1;
#pragma unroll
        for (int d = 0; d < S::DT; ++d) {
          vr[d][k] &= keep;
          bad |= nan_bytes(vr[d][k]);
        }
      }
    }
    if (__builtin_expect(!__any(bad != 0), 1)) {
#pragma unroll
      for (int d = 0; d < S::DT; ++d)
#pragma unroll
        for (int hf = 0; hf < J / 2; ++hf)
          o[d] = mfma_bf16(fp8x8_to_bf16(vr[d][2 * hf], vr[d][2 * hf + 1], vs), p[hf], o[d]);
    } else {
      // 0 x NaN is NaN: the NaN values are taken out, and a product of 0 / 1 operands counts for each row and channel the
      // NaN that it sees.
#pragma unroll
      for (int d = 0; d < S::DT; ++d) {
        v4f n{0, 0, 0, 0};
#pragma unroll
        for (int hf = 0; hf < J / 2; ++hf) {
          bf16x8 nv, sv;
          uint32_t x[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t nb = nan_bytes(vr[d][2 * hf + k]) >> 7;  // 0 / 1 in each byte
            x[k] = vr[d][2 * hf + k] & ~(nb * 0xffu);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              nv[4 * k + e] = __bf16(float(nb >> (8 * e) & 1));
              sv[4 * k + e] = __bf16(float(see >> (8 * hf + 4 * k + e) & 1));
            }
          }
          n = mfma_bf16(nv, sv, n);
          o[d] = mfma_bf16(fp8x8_to_bf16(x[0], x[1], vs), p[hf], o[d]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n[e] > 0.0f) o[d][e] = __builtin_nanf("");
      }
    }
    if (more) load_v(tn, pv);
  }

  // join the waves that share rows
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if constexpr (TW > 1) {
    if (g == 0) lds.ml[wave][c][0] = mx, lds.ml[wave][c][1] = l;
    __syncthreads();
    const int w0 = wave / TW * TW;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < TW; ++w) m = fmaxf(m, lds.ml[w0 + w][c][0]);
    const float ref = m == -INFINITY ? 0.0f : m, f = __builtin_amdgcn_exp2f(mx - ref);
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < TW; ++w) l += lds.ml[w0 + w][c][1] * __builtin_amdgcn_exp2f(lds.ml[w0 + w][c][0] - ref);
    mx = m;
#pragma unroll
    for (int d = 0; d < S::DT; ++d) o[d] *= f;
    const auto at = [&](int buf, int d) { return reinterpret_cast<v4f*>(&lds.o[buf][(d * 64 + lane) * 4]); };
#pragma unroll
    for (int half = TW / 2; half; half /= 2) {  // the upper half of the waves hands its sums to the lower
      const int k = wave % TW, buf = wave / TW * (TW / 2) + k % half;
      if (k >= half && k < 2 * half)
#pragma unroll
        for (int d = 0; d < S::DT; ++d) *at(buf, d) = o[d];
      __syncthreads();
      if (k < half)
#pragma unroll
        for (int d = 0; d < S::DT; ++d) o[d] += *at(buf, d);
      __syncthreads();
    }
  }
  const bool mine = wave % TW == 0 && row0 + c < nrows;
  if (pc.pieces == 1) {
    if (mine)
#pragma unroll
      for (int d = 0; d < S::DT; ++d) store_out<D>(a, my_row, my_hq, 16 * d + 4 * g, o[d], l, mx, d == 0 && g == 0);
    return;
  }
  if (mine) {
    const int r = (pc.slot0 + pc.index) * S::ROWS + wave / TW * 16 + c;
#pragma unroll
    for (int d = 0; d < S::DT; ++d) put4(sums_of(a.po), r * D + 4 * g + 16 * d, o[d]);
    if (g == 0) put2(sums_of(a.pml), r * 2, mx, l);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's sums have left
  __syncthreads();
  if (tid == 0)
    last = __hip_atomic_fetch_add(&a.counters[pc.slot0], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
           uint32_t(pc.pieces - 1);
  __syncthreads();
  if (!last) return;
  if (tid == 0)  // as it was found
    __hip_atomic_store(&a.counters[pc.slot0], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // a thread per row and four channels, the loads of eight pieces in flight at a time
  const int rows = min(S::ROWS, nrows - pc.rg * S::ROWS);
  const __amdgpu_buffer_rsrc_t po = sums_of(a.po + size_t(pc.slot0) * S::ROWS * D);
  const __amdgpu_buffer_rsrc_t pml = sums_of(a.pml + size_t(pc.slot0) * S::ROWS * 2);
  for (int it = tid; it < rows * (D / 4); it += AT_NT) {
    const int r = it / (D / 4), d = it % (D / 4) * 4;
    float m = -INFINITY, sum = 0.0f;
    v4f acc{0, 0, 0, 0};
    for (int k0 = 0; k0 < pc.pieces; k0 += JOIN) {
      v4f y[JOIN];
      float2 x[JOIN];
#pragma unroll
      for (int k = 0; k < JOIN; ++k) {
        const int at = min(k0 + k, pc.pieces - 1) * S::ROWS + r;
        x[k] = get2(pml, at * 2);
        y[k] = get4(po, at * D + d);
      }
      float m1 = m;
#pragma unroll
      for (int k = 0; k < JOIN; ++k) m1 = fmaxf(m1, x[k].x);
      const float ref = m1 == -INFINITY ? 0.0f : m1, al = __builtin_amdgcn_exp2f(m - ref);
      m = m1;
      acc *= al;
      sum *= al;
#pragma unroll
      for (int k = 0; k < JOIN; ++k) {
        const float f = k0 + k < pc.pieces ? __builtin_amdgcn_exp2f(x[k].x - ref) : 0.0f;
        if (k0 + k < pc.pieces) {
          sum += f * x[k].y;
          acc += f * y[k];
        }
      }
    }
    const int rr = pc.rg * S::ROWS + r;
    store_out<D>(a, q.r0 + rr / a.group, h * a.group + rr % a.group, d, acc, sum, m, d == 0);
  }
}

int most_rows(int rows, int max_new, int group) {
  return int(std::min<int64_t>(int64_t(std::min(rows, max_new)) * group, INT32_MAX));
}
int row_waves(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

}  // namespace

size_t kv_attend_workspace(int rows, int max_new, int B, int Hq, int heads, int dim) {
  if (rows < 0 || max_new < 0 || B < 0 || heads < 1 || Hq < heads || dim < 1) return 0;
  const int rw = row_waves(most_rows(rows, max_new, Hq / heads));
  return kCounterBytes + size_t(slots_of(rw)) * 16 * rw * (size_t(dim) + 2) * sizeof(float);
}

void kv_attend(const bf16* q, int ldq, const KvStep& s, const KvCache& c, int Hq, float scale, int window, int sinks,
               bf16* out, int ldo, float* lse, void* ws, size_t ws_bytes, hipStream_t st) {
  const auto fail = [](const std::string& what) { throw std::runtime_error("kv_attend: " + what); };
  check_cache("kv_attend", c);
  check_step("kv_attend", s);
  if (Hq < 1 || Hq % c.heads || Hq > 65535) fail("Hq must be a multiple of heads, up to 65535");
  if (sinks < 0) fail("sinks < 0");
  if (!std::isfinite(scale)) fail("scale is not finite");
  if (s.B == 0 || s.rows == 0 || s.max_new == 0) return;
  if (!q || !out) fail("null operand");
  const int64_t width = int64_t(Hq) * c.dim;
  if (ldq < width || ldo < width || ldq % 8 || ldo % 8) fail("ldq / ldo >= Hq * dim, % 8");
  if (!aligned16(q) || !aligned16(out)) fail("rows not 16-byte aligned");
  if (int64_t(s.rows) * Hq > INT32_MAX) fail("rows * Hq past 31 bits");
  const size_t need = kv_attend_workspace(s.rows, s.max_new, s.B, Hq, c.heads, c.dim);
  if (!ws) fail("null workspace");
  if (!aligned16(ws)) fail("workspace not 16-byte aligned");
  if (ws_bytes < need) fail("workspace of " + std::to_string(ws_bytes) + " bytes, " + std::to_string(need) + " needed");

  Attend a{q, out, lse, s, c, ldq, ldo, Hq / c.heads, 0, window, sinks, scale * LOG2E, kTarget, 1, nullptr,
           nullptr, nullptr};
  while (1 << a.page_shift < c.page) ++a.page_shift;
  const int rows = most_rows(s.rows, s.max_new, a.group), rw = row_waves(rows);
  a.counters = static_cast<uint32_t*>(ws);
  a.po = reinterpret_cast<float*>(static_cast<char*>(ws) + kCounterBytes);
  a.pml = a.po + size_t(slots_of(rw)) * 16 * rw * c.dim;
  a.rounds = rounds_of(rw);
  const int64_t segs = int64_t(s.B) * c.heads * cdiv(rows, 16 * rw);  // at most; each is a piece too many at most
  if (segs + kMostSlots > INT32_MAX) fail("too many rows");
  const unsigned grid = unsigned(segs + a.target * a.rounds);
  const auto by_rw = [&]<int D>() {
    if (rw == 1) kv_split_kernel<D, 1><<<grid, AT_NT, 0, st>>>(a);
    else if (rw == 2) kv_split_kernel<D, 2><<<grid, AT_NT, 0, st>>>(a);
    else kv_split_kernel<D, 4><<<grid, AT_NT, 0, st>>>(a);
  };
  if (c.dim == 64) by_rw.template operator()<64>();
  else if (c.dim == 128) by_rw.template operator()<128>();
  else by_rw.template operator()<256>();
  UH_CHECK_LAUNCH();
}

}  // namespace unholy::kernels
