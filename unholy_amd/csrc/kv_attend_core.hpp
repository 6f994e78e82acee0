// What the kernels of attention over the 8-bit paged cache are made of: the split of a launch's work, and the two ways of going
// through a sequence's tokens, by few rows and by many.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv_internal.hpp"
#include "numerics.hpp"
#include "pipe.hpp"

namespace unholy::kernels::kv {

using namespace uh;

constexpr int TILE = 64;          // tokens a wave takes at a time
constexpr int AT_NT = 256;        // threads of a workgroup: four waves
constexpr int AT_WAVES = AT_NT / 64;
constexpr int FEW = 16;           // rows (of a key / value head) of a sequence that the split kernel takes
constexpr int PR_ROWS = 128;      // rows of a workgroup of the tiled kernel
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

// Bits of the first n of up to 16 tokens.
__device__ __forceinline__ uint32_t first_bits(int n) { return (1u << min(max(n, 0), 16)) - 1; }
// Which of the 16 tokens from t on a row at position p sees.
__device__ __forceinline__ uint32_t seen_bits(int p, int t, int window, int sinks) {
  uint32_t see = first_bits(p - t + 1);
  if (window > 0) see &= ~first_bits(int(max(min(int64_t(p) - window - t + 1, int64_t(16)), int64_t(0)))) | first_bits(sinks - t);
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

// Rows whose sums the parts [slot, slot + step, ...) of a launch hold.
struct Block {
  int parts, step;
  int row0, rows;  // from the sequence's first (row, query head) on
  int r0, h;       // the sequence's first row, the head
  int over, pad;   // some sequence brings more than max_new rows
};

// Where partial sums begin, of how many parts.
struct Common {
  int row, parts;
};

// What every workgroup knows of the call.
struct Attend {
  const bf16* q;
  bf16* out;
  float* lse;
  KvStep st;
  KvCache c;
  int ldq, ldo, group, page_shift, window, sinks;
  float scale2;  // scale * log2(e): the kernels take powers of two
  int few;  // sequences of up to this many rows (FEW or none) are the split kernel's, the others the tiled kernel's
  uint32_t target;     // workgroups that the work is cut for
  uint32_t* counters;  // of finished parts, by the workgroup of the first; zero between launches (split kernel)
  Block* blocks;       // by the workgroup of the first part (tiled kernel; null where it is not launched)
  float *po, *pml;     // partial sums: values [slot][rows][D]; maximum and weight sum [slot][rows][2]
};
// The same of kv_attend_shared. (A struct of its own: kv_attend's kernels have less to load before their first key.)
struct AttendShared : Attend {
  Share share;
  Common *common, *own;  // by block of a group and head; by sequence, FEW of its rows and head (the first workgroup of these)
  float *so, *sml;       // the groups' partial sums: values [row][D]; maximum and weight sum [row][2]
  float *lo, *lml;       // those of a sequence's own tiles that are one part, by (row in the lists, query head), the same way
  int most_parts;        // of FEW rows, of a sequence
  int lists, sum_rows;   // rows that the lists have room for, and the groups' sums
};

__device__ __forceinline__ size_t own_at(const AttendShared& a, int b, int part, int h) {
  return (size_t(b) * a.most_parts + part) * a.c.heads + h;
}

// Where a sequence's rows begin in the groups' lists. (A plan that was made for other rows than the step has, which its caller
// should not use, gives wrong results, but no place outside of the workspace.)
__device__ __forceinline__ int list_of(const AttendShared& a, const ShareSeq& s, const Seq& q) {
  return max(min(s.row0 + s.at, a.lists - (q.r1 - q.r0)), 0);
}

// Where the sums of a sequence's r-th (row, query head) of head h are, of the sequences in groups.
__device__ __forceinline__ size_t list_row(const Attend& a, int list, int h, int r) {
  return (size_t(list) * a.group + r) * a.c.heads + h;
}

// The 64-token tiles from `from` on that some row of a sequence sees: with a window sink_tiles of the sinks' and those from
// `skip` on, else all; count of them, numbered in order.
struct Tiles {
  int sink_tiles, skip, count, from;
  __device__ __forceinline__ int at(int i) const { return i < sink_tiles ? from + i : i - sink_tiles + skip; }
};
__device__ __forceinline__ Tiles tiles_of(const Attend& a, const Seq& q, int from = 0) {
  const int64_t cap = int64_t(a.st.max_blocks) << a.page_shift;
  const int end = int((min(int64_t(q.len), cap) + TILE - 1) / TILE);
  from = from > 0 ? min(from, end) : 0;
  Tiles t{0, from, end - from, from};
  if (a.window > 0) {
    const int64_t lo = int64_t(q.first) - a.window + 1;  // the first token in the first row's window
    t.skip = max(min(int(max(lo, int64_t(0)) / TILE), end), from);
    t.sink_tiles = max(min(int((int64_t(a.sinks) + TILE - 1) / TILE), t.skip) - from, 0);
    t.count = end - t.skip + t.sink_tiles;
  }
  return t;
}
__device__ __forceinline__ int row_groups(int rows, int per) { return (rows + per - 1) / per; }

// The split of a launch's work, worked out by every workgroup from the lengths, which only the device knows. A segment is a
// (sequence, key / value head) and its tiles.
// Many segments: workgroup w takes the tiles [w share, (w + 1) share) of all segments in order, so that long and short
// sequences load the chip evenly; it may end one segment, do some whole ones and begin another, and each beginning costs it
// START tiles' time. Few segments (an eighth of the workgroups): each is cut into parts as equal as they can be, a workgroup
// each, and no workgroup has two beginnings. (256 segments of 18 tiles under a window, four layers: 67 us cut anywhere, 75 in
// two equal parts, each joined, 71 whole; 8 of 65 tiles, sixteen layers: 203 us cut anywhere, 159 in equal parts; between
// them, 32 of some 1700 tiles are 176 and 178.)
// The parts of a segment are those of consecutive workgroups; the part of workgroup w that begins a segment leaves its sums
// in slot 2 w + 1, one that goes on with it in slot 2 w.
struct Walk {
  int b, h;     // the sequence and the head
  int part;     // kv_attend_shared: which FEW of the sequence's rows
  int list;     // the same: where its rows begin in the lists of the groups
  uint32_t at;  // where the segment begins, in units (tiles, or parts of equal segments)
  Seq q;
  Tiles t;
};
struct Part {
  int i0, i1, index, parts;
};
constexpr uint32_t START = 2;  // a segment's start, in tiles: the time that its first loads and its end take
// The parts that n tiles make.
__device__ __forceinline__ uint32_t parts_of(uint32_t tiles, uint32_t share) {
  return max((tiles + share - 1) / share, 1u);  // (no tiles: a part that writes zeros)
}
// The smallest share, `least` at least, with which n things of `tiles` tiles in each lane make `target` parts or fewer: all
// is their number over the lanes (<= target), sum their tiles. ceil(sum / target) is too small or right, and
// ceil(sum / (target - all)) is large enough: each adds a part at most to its exact share.
__device__ __forceinline__ uint32_t smallest_share(uint32_t n, uint32_t tiles, uint32_t sum, uint32_t all, uint32_t target,
                                                   uint32_t least) {
  uint32_t lo = max((sum + target - 1) / target, least);
  uint32_t hi = max(all < target ? (sum + target - all - 1) / (target - all) : wave_reduce_u32<true>(tiles), least);
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    if (lane_of(wave_scan(n * parts_of(tiles, mid)), 63) <= target) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// The root of a times n items' average of `sum`.
__device__ __forceinline__ uint32_t root(float a, uint32_t sum, uint32_t n) {
  return uint32_t(__builtin_amdgcn_sqrtf(a * float(sum) * __builtin_amdgcn_rcpf(float(max(n, 1u)))));
}

struct Split {
  bool whole;            // equal parts of each segment
  uint32_t share, unit;  // tiles of a part at most; units of a workgroup
};
__device__ __forceinline__ uint32_t units_of(const Split& s, uint32_t tiles) {
  return s.whole ? parts_of(tiles, s.share) : tiles + START;
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Zeros (lse: -inf) in the rows of the sequences that bring more than max_new, which see nothing: workgroup w's of n.
__device__ __forceinline__ void clear_rows(const Attend& a, int w, int n) {
  const int heads = a.group * a.c.heads, quads = heads * a.c.dim / 8;
  for (int b = 0; b < a.st.B; ++b) {
    const Seq q = seq_of(a.st, b);
    if (!too_many(a.st, q)) continue;
    for (int i = w; i < q.r1 - q.r0; i += n) {
      uint4* out = reinterpret_cast<uint4*>(a.out + size_t(q.r0 + i) * a.ldo);
      for (int j = int(threadIdx.x); j < quads; j += AT_NT) out[j] = make_uint4(0, 0, 0, 0);
      if (a.lse)
        for (int j = int(threadIdx.x); j < heads; j += AT_NT) a.lse[size_t(q.r0 + i) * heads + j] = -INFINITY;
    }
  }
}

// A sequence's segments: its heads, times (kv_attend_shared) the parts of FEW rows that it brings.
template <class A>
__device__ __forceinline__ int segments_of(const A& a, const Seq& q) {
  return std::is_same_v<A, AttendShared> ? a.c.heads * row_groups((q.r1 - q.r0) * a.group, FEW) : a.c.heads;
}
__device__ __forceinline__ bool is_few(const Attend& a, const Seq& q) {
  return q.r1 > q.r0 && (q.r1 - q.r0) * a.group <= a.few && !too_many(a.st, q);
}
// Workgroup wg's part of the segment, from unit u on.
__device__ __forceinline__ Part part_of(const Split& s, const Walk& w, uint32_t u, uint32_t wg) {
  Part p;
  const uint32_t count = uint32_t(w.t.count), size = units_of(s, count), w0 = w.at / s.unit;
  p.index = int(wg - w0);
  p.parts = int((w.at + size - 1) / s.unit - w0 + 1);
  if (s.whole) {
    const uint32_t each = count / size, more = count % size, i = uint32_t(p.index);
    p.i0 = int(i * each + min(i, more));
    p.i1 = p.i0 + int(each + (i < more ? 1 : 0));
  } else {
    const uint32_t i0 = u - w.at, i1 = min(size, (wg + 1) * s.unit - w.at);  // the start's units hold no tile
    p.i0 = int(max(i0, START) - START);
    p.i1 = int(max(i1, START) - START);
  }
  return p;
}
// The next segment, if the units of workgroup wg reach it.
template <class A>
__device__ __forceinline__ bool next_segment(const A& a, const Split& s, Walk& w, uint32_t wg) {
  constexpr bool SH = std::is_same_v<A, AttendShared>;
  w.at += units_of(s, uint32_t(w.t.count));
  if (s.whole || w.at >= (wg + 1) * s.unit) return false;
  if (++w.h < a.c.heads) return true;
  w.h = 0;
  if (SH && ++w.part * FEW < (w.q.r1 - w.q.r0) * a.group) return true;
  w.part = 0;
  do {
    if (++w.b >= a.st.B) return false;
    const Seq q = seq_of(a.st, w.b);
    w.q = Seq{uniform(q.r0), uniform(q.r1), uniform(q.len), uniform(q.first)};
  } while (!is_few(a, w.q));
  if constexpr (SH) {
    const ShareSeq s = a.share.seqs[w.b];
    w.t = tiles_of(a, w.q, share_fits(a.share.head, a.st, a.c.page) ? uniform(s.tiles) : 0);
    w.list = uniform(list_of(a, s, w.q));
  } else {
    w.t = tiles_of(a, w.q);
  }
  return true;
}

__device__ __forceinline__ bf16x8 bf16x8_of(uint4 v) { return __builtin_bit_cast(bf16x8, v); }
__device__ __forceinline__ uint4 ld16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ uint32_t nan_bytes(uint32_t x) {  // the high bit of each byte that is a NaN code
  return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// A scale byte that is no number, as e8m0 has it (in fp32: infinity; the products' conversions make NaN of any code with
// it), and four codes that are none.
constexpr int NAN_SCALE = 0xff;
constexpr uint32_t NAN_CODES = 0x7f7f7f7fu;

// The first n bytes of four.
__device__ __forceinline__ uint32_t first_bytes(int n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1; }
// bf16 operands of 0 and 1: of the NaN among eight codes, and of eight bits; and codes with zeros for their NaN.
__device__ __forceinline__ uint32_t two_ones(uint32_t x, uint32_t y) { return (x & 1) * 0x3f80u | (y & 1) * 0x3f800000u; }
__device__ __forceinline__ bf16x8 nan_ones(uint32_t lo, uint32_t hi) {
  const uint32_t a = nan_bytes(lo) >> 7, b = nan_bytes(hi) >> 7;
  return bf16x8_of(make_uint4(two_ones(a, a >> 8), two_ones(a >> 16, a >> 24), two_ones(b, b >> 8), two_ones(b >> 16, b >> 24)));
}
__device__ __forceinline__ bf16x8 bit_ones(uint32_t z) {
  return bf16x8_of(make_uint4(two_ones(z, z >> 1), two_ones(z >> 2, z >> 3), two_ones(z >> 4, z >> 5), two_ones(z >> 6, z >> 7)));
}
__device__ __forceinline__ uint32_t no_nan(uint32_t x) { return x & ~((nan_bytes(x) >> 7) * 0xffu); }

// ---- few rows a sequence: decode and verify steps ---------------------------------------------------------------------
// Bound by reading the cache once (64 sequences of 0 to 8190 tokens, 8 heads of 128: 105 us, 5.3 TB/s; four of 90,000 to
// 131,000: 178 us, 5.4 TB/s; a sum over a large array reads 6.1 TB/s here), and where there is little of it by the chain of
// loads that depend on each other: lengths, table, keys, partial sums. A wave takes 16 rows ((token, query head) pairs that
// share a key / value head) and 64 tokens at a time straight from the cache into registers, no LDS: with S^T = K Q^T the
// 16x16 product leaves lane (row c, group g) the scores of tokens 4g .. 4g + 3 of a 16-token tile, and the tiles' rows are
// taken in such an order of tokens (tile j, row r: token 16 (r / 4) + 4j + r % 4) that over four tiles these are tokens
// 16g .. 16g + 15: the very tokens whose values one 16-byte load of the transposed cache gives it for O^T = V^T P^T. The
// weights go from one product to the other in place, and a row's running maximum and sum are its lane's own.
// The codes become bf16 exactly (v_cvt_scalef32, the block's scale with them), the products sum in fp32; the weights are
// rounded to bf16 for the second product (2^-8 of each at most, as much as the output's own rounding), their sum is taken in
// fp32 before that.
// The four waves take every fourth tile and are joined in LDS. The workgroup that finishes last of those that share rows adds
// their partial sums, in the same order whichever it is: the result does not depend on timing. (Workgroups of eight waves, one
// a CU, have half as many parts to join, but a CU then waits for twice the bytes: sixteen layers of one token over 4097 take
// 202 us for 160.)
template <int D>
struct Shape {
  static constexpr int KL = D / 64;  // 16-byte loads of a key row's quarter
  static constexpr int DT = D / 16;  // 16-channel tiles
  static constexpr int QUADS = FEW * D / 4;  // four channels of a row
  struct Lds {
    v4f o[AT_WAVES * QUADS];  // the waves' sums, later the groups' (of the join)
    float2 ml[AT_WAVES][FEW], group_ml[AT_NT];
  };
};
// Workgroups that a launch's work is cut for: two a CU, by their registers, or one (and two for 64 channels, of whose tiled
// kernel a CU holds three).
constexpr int target_of(int dim) { return dim <= 128 ? 512 : 256; }
constexpr int FLIGHT = 10;  // partial sums that a thread reads at a time
constexpr size_t kHeadBytes = 512 * (sizeof(uint32_t) + sizeof(Block));  // counters and blocks

// Partial sums pass between workgroups on different XCDs, whose L2 caches do not see each other's lines: stored through
// to memory and read from there (device-scope accesses), which for these few KiB is far cheaper than the fences that
// write back and invalidate a whole L2 (sixteen layers of one token over 4097 tokens, 17 parts a head: 375 us with fences,
// 159 with these).
constexpr int SC1 = 16;  // the cache policy of a device-scope access
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

// A tile of a wave's rows: its keys and values in registers (kr, vr, with their scales' bytes) into the rows' sums. pvt: the
// page of this lane's values; mid: what to do once the keys are used.
struct FewRow {
  int pos, pos_lo, pos_hi, len;  // this lane's row's position, all rows' lowest and highest, the sequence's length
};
template <int D, class Mid>
__device__ __forceinline__ void few_tile(const Attend& a, const uint4 (&kr)[4][Shape<D>::KL], uint32_t (&vr)[Shape<D>::DT][4],
                                         const bf16x8 (&qf)[2 * Shape<D>::KL], int ksb, int vsb, int pvt, int t0, const FewRow& row,
                                         int g, v4f (&o)[Shape<D>::DT], float& mx, float& l, Mid mid) {
  using S = Shape<D>;
  const float ks = e8m0_to_f32(uint8_t(ksb));
  v4f s[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    s[j] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int m = 0; m < S::KL; ++m) {
      s[j] = mfma_bf16(fp8x8_to_bf16(kr[j][m].x, kr[j][m].y, ks), qf[2 * m], s[j]);
      s[j] = mfma_bf16(fp8x8_to_bf16(kr[j][m].z, kr[j][m].w, ks), qf[2 * m + 1], s[j]);
    }
  }
  mid();
  // what a row does not see: only in the tiles at the ends of what the rows see
  const bool masked = t0 + TILE - 1 > row.pos_lo || __any(pvt < 0) ||
                      (a.window > 0 && int64_t(t0) + a.window <= row.pos_hi && t0 + TILE > a.sinks);
  uint32_t see = 0xffff;
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < 4; ++j) s[j] *= a.scale2;
  if (masked) {
    see = pvt < 0 ? 0 : seen_bits(row.pos, t0 + 16 * g, a.window, a.sinks);
#pragma unroll
    for (int k = 0; k < 16; ++k) s[k / 4][k % 4] = see >> k & 1 ? s[k / 4][k % 4] : -INFINITY;
  }
#pragma unroll
  for (int k = 0; k < 16; ++k) top = fmaxf(top, s[k / 4][k % 4]);
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
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[j][e] = __builtin_amdgcn_exp2f(s[j][e] - ref);
      l += s[j][e];
    }
  bf16x8 p[2];
#pragma unroll
  for (int hf = 0; hf < 2; ++hf)
#pragma unroll
    for (int e = 0; e < 8; ++e) p[hf][e] = __bf16(s[2 * hf + e / 4][e % 4]);
  if (masked) {  // slots past the last token hold anything: zero
    const int n = pvt < 0 ? 0 : min(max(row.len - (t0 + 16 * g), 0), 16);
    const uint32_t all = vsb == NAN_SCALE ? NAN_CODES : 0;  // its codes are NaN, under a scale that is a number then
    vsb = all ? 127 : vsb;
    uint32_t bad = 0;
#pragma unroll
    for (int d = 0; d < S::DT; ++d)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        vr[d][k] = (vr[d][k] | all) & first_bytes(n - 4 * k);
        bad |= nan_bytes(vr[d][k]);
      }
    if (__builtin_expect(__any(bad != 0), 0)) {
      // NaN among the values that some row sees, and 0 x NaN is NaN: they are taken out, and a product of 0 / 1 operands
      // counts for each row and channel the NaN that it sees.
#pragma unroll
      for (int d = 0; d < S::DT; ++d) {
        v4f many = mfma_bf16(nan_ones(vr[d][0], vr[d][1]), bit_ones(see), v4f{0, 0, 0, 0});
        many = mfma_bf16(nan_ones(vr[d][2], vr[d][3]), bit_ones(see >> 8), many);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          vr[d][k] = no_nan(vr[d][k]);
          if (many[k] > 0.0f) o[d][k] = __builtin_nanf("");
        }
        __builtin_amdgcn_sched_barrier(0);  // (one channel tile at a time: registers)
      }
    }
  }
  const float vs = e8m0_to_f32(uint8_t(vsb));
#pragma unroll
  for (int d = 0; d < S::DT; ++d)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
      o[d] = mfma_bf16(fp8x8_to_bf16(vr[d][2 * hf], vr[d][2 * hf + 1], vs), p[hf], o[d]);
}

// ---- many rows a sequence: prompts ------------------------------------------------------------------------------------
// Bound by the matrix rate and by the vector work next to it: 8192 rows of 32 heads of 128 take 527 to 562 us, 0.98 to 1.04
// PFLOP/s (a large bf16 product reaches 1.17 here), the matrix units busy for half of the cycles and the vector units for 72%;
// with 64 channels, where a score's exponential, scaling and sum come with half as many products, 0.56 PFLOP/s (28%, 78%). With
// 256 the registers do not suffice (14 are spilled), and in pages of 16 and 32 tokens each tile's reload waits for the direct
// loads as well: 4096 rows of 32 heads over 4 take 355 us, in pages of 16 396 (128 channels: 153 and 166).
// A workgroup takes 128 rows (4 waves of 32) of one (sequence, key / value head) and goes through the 64-token tiles that they
// see, which arrive in LDS as codes by direct loads, two tiles ahead, in a ring of three. The 32x32x16 product with the same
// order of tokens as above: S^T = K Q^T with row 8a + 4h + i of a 32-token half taken as token 16h + 4a + i, so that lane
// (row, half h) has the scores of 16 consecutive tokens and O^T = V^T P^T finds their values in one 16-byte read.
// LDS: the 16-byte pieces of a key row (D bytes) and of a channel's values (64 bytes) are permuted among themselves such
// that the sixteen lanes that a read serves at a time find theirs in different banks.
// Pages and scales are read for 16 tiles at a time: their loads are waited for with all others, direct ones among them.
// The running maximum is left alone until a row's scores pass it by more than 2^8: the weights stay small enough, and most
// tiles need no scaling of the sums. The largest weight is not 1 then, as it is above, but rounded to bf16 like the others: an
// output is off by 2.2e-3 of its norm, the split kernel's by 1.8e-3, and the output's own rounding alone is 1.65e-3.
constexpr int PR_STAGES = 3;
constexpr int PR_META = 16;  // tiles
constexpr float PR_LAG = 8.0f;

// The larger of a lane's value and its counterpart's in the wave's other half.
__device__ __forceinline__ float max_halves(float v) {
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}

// The place among a key row's pieces of piece p of row (token) t, and among a channel's pieces of piece p of channel d.
template <int D>
__device__ __forceinline__ int key_piece(int t, int p) {
  const int b1 = t >> 1 & 1, b2 = t >> 2 & 1, b4 = t >> 4 & 1;
  return p ^ (D == 64 ? b2 | b4 << 1 : D == 128 ? b1 | b2 << 1 | b4 << 2 : (t & 3) | b2 << 2 | b4 << 3);
}
__device__ __forceinline__ int value_piece(int d, int p) { return p ^ (d >> 2 & 3); }

template <int D>
struct Tiled {
  static constexpr int KV = TILE * D;                   // bytes of a tile's keys, and of its values
  static constexpr int LOADS = KV / 16 / AT_NT;         // direct loads a thread makes for each
  static constexpr int DT = D / 32;
  struct Lds {
    uint8_t k[PR_STAGES][KV], v[PR_STAGES][KV];
    int page[2][PR_META * 4];
    uint64_t missing[2];  // a bit for every 16 tokens without a page
    float ks[2][PR_META * 4], vs[2][PR_META * 4];  // of every 16 tokens
  };
};

// A workgroup's rows and tiles. The row blocks of all sequences times the heads, and where these do not fill the chip each
// block's tiles are cut into parts of at most `share`: as few as still fill it. A sequence's last blocks, which see the most,
// come first; the heads are inner, so that with 8 heads or a multiple an XCD's workgroups read the same ones' keys and
// values.
struct BlockPart {
  int b, h, row0;
  Seq q;
  Tiles t;                       // that the block's rows see
  int i0, i1;                    // the part's of them
  int index, parts;              // which part of how many
};
__device__ __forceinline__ Tiles block_tiles(const Attend& a, const Seq& q, int row0) {
  const int last = min(row0 + PR_ROWS, (q.r1 - q.r0) * a.group) - 1;
  return tiles_of(a, Seq{0, 0, max(min(q.len, q.first + last / a.group + 1), 0), q.first + row0 / a.group});
}
// Find names the call (Find::Call, what every workgroup knows) and finds this workgroup's part of a block of rows. COMMON
// (kv_attend_shared): of a group's list, whose sums are partial ones throughout, in rows from `sums` on. (Written as the kernel
// itself: the same body as a function that two kernels call is compiled to other registers, and kv_attend 1% slower.)
template <int D, class Find>
__global__ __launch_bounds__(AT_NT, D == 64 ? 3 : D == 128 ? 2 : 1) void kv_tiled_kernel(typename Find::Call a) {
  constexpr bool COMMON = std::is_same_v<typename Find::Call, AttendShared>;
  BlockPart bp;
  int sums = 0;
  if (!Find::template find<D>(a, bp, sums)) return;
  using S = Tiled<D>;
  __shared__ __align__(1024) typename S::Lds lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), c = lane & 31, h2 = lane >> 5;
  const int b = bp.b, h = bp.h, row0 = bp.row0;
  const Seq q = bp.q;
  const Tiles tiles = bp.t;
  const int nrows = (q.r1 - q.r0) * a.group, parts = bp.parts;

  // this lane's row
  const int wrow = row0 + 32 * wave, ri = min(wrow + c, nrows - 1);
  int row = q.r0 + ri / a.group, pos = q.first + ri / a.group;
  const int hq = h * a.group + ri % a.group;
  if constexpr (COMMON) {
    const int2 listed = a.share.list[row];
    row = listed.x;
    // A group's tiles lie before all of its rows: where a row is matters to a window only, and that moves on with the lengths
    // of this step, not those of the plan's.
    pos = 1 << 30;
    if (a.window > 0) {
      const Seq s = seq_of(a.st, listed.y);
      pos = s.first + row - s.r0;
    }
  }
  const int pos_lo = COMMON ? INT32_MAX : uniform(q.first + min(wrow, nrows - 1) / a.group);
  const int pos_hi = COMMON ? INT32_MAX : uniform(q.first + min(wrow + 31, nrows - 1) / a.group);
  const float sc = fmaxf(fabsf(a.scale2), 0x1p-126f);  // (not 0: hidden scores are -inf, and stay so)

  const int n = bp.i1 - bp.i0;
  const auto token = [&](int i) { return tiles.at(bp.i0 + i) * TILE; };
  // pages and scales of tiles [16 chunk, 16 chunk + 16), four groups of tokens a tile and one a lane
  static_assert(PR_META * 4 == 64);
  const auto look = [&](int chunk) {
    const int i = chunk * PR_META + lane / 4;
    return i < n ? page_of(a.st.table, a.st.max_blocks, a.c.pages, b, (token(i) + lane % 4 * 16) >> a.page_shift) : -1;
  };
  const auto meta = [&](int chunk) {
    if (wave == 0) {
      const int pg = look(chunk);
      const size_t ph = size_t(max(pg, 0)) * a.c.heads + h;
      const uint64_t none = __ballot(pg < 0);
      if (tid == 0) lds.missing[chunk & 1] = none;
      lds.page[chunk & 1][lane] = pg;
      lds.ks[chunk & 1][lane] = e8m0_to_f32(a.c.ks[ph]);
      lds.vs[chunk & 1][lane] = e8m0_to_f32(a.c.vs[ph]);
    }
  };
  const int mask = a.c.page - 1, sh = a.page_shift;
  // Tile i on its way to its stage; pg: its page, where a page holds whole tiles (then only the base differs from tile to
  // tile), else its four groups of tokens are looked up by their lanes.
  uint32_t koff[S::LOADS], voff[S::LOADS];
#pragma unroll
  for (int x = 0; x < S::LOADS; ++x) {  // the 16-byte slots that this lane fills
    const int at = (x * AT_WAVES + wave) * 64 + lane, t = at / (D / 16), d = at / 4;
    koff[x] = uint32_t(t * D + 16 * key_piece<D>(t, at % (D / 16)));
    voff[x] = uint32_t((d << sh) + 16 * value_piece(d, at % 4));
  }
  const bool whole = a.c.page >= TILE;
  const auto page_at = [&](int i) { return lds.page[i / PR_META & 1][i % PR_META * 4]; };
  const auto fetch = [&](int i, int pg) {
    const int t0 = token(i), st = i % PR_STAGES;
    const auto to = [&](uint8_t* stage, int x) { return pipe::lds_addr(stage + (x * AT_WAVES + wave) * 1024); };
    if (whole) {
      const size_t ph = size_t(uniform(max(pg, 0))) * a.c.heads + h;
      const uint8_t* kb = a.c.k + ((ph << sh) + (t0 & mask)) * D;
      const uint8_t* vb = a.c.v + ((ph * D) << sh) + (t0 & mask);
#pragma unroll
      for (int x = 0; x < S::LOADS; ++x) pipe::dma16(kb, koff[x], to(lds.k[st], x));
#pragma unroll
      for (int x = 0; x < S::LOADS; ++x) pipe::dma16(vb, voff[x], to(lds.v[st], x));
    } else {
      const int* pages = &lds.page[i / PR_META & 1][i % PR_META * 4];
#pragma unroll
      for (int x = 0; x < S::LOADS; ++x) {
        const uint32_t t = koff[x] / D;
        const size_t ph = size_t(max(pages[t / 16], 0)) * a.c.heads + h;
        pipe::dma16_at(a.c.k + ((ph << sh) + ((t0 + t) & mask)) * D + koff[x] % D, to(lds.k[st], x));
      }
#pragma unroll
      for (int x = 0; x < S::LOADS; ++x) {
        const int d = ((x * AT_WAVES + wave) * 64 + lane) / 4, p = int(voff[x] - (uint32_t(d) << sh)) / 16;
        const size_t ph = size_t(max(pages[p], 0)) * a.c.heads + h;
        pipe::dma16_at(a.c.v + ((ph * D + d) << sh) + ((t0 + 16 * p) & mask), to(lds.v[st], x));
      }
    }
  };

  pipe::v16f_t o[S::DT];
#pragma unroll
  for (int d = 0; d < S::DT; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
  float ref2 = -INFINITY, l = 0.0f;  // what the weights are relative to (a power of two's exponent); their sum
  int next = 0;  // the page of the next tile to fetch, read ahead
  uint64_t missing = 0;
  // The start, with as few loads behind each other as there can be: the pages are looked up while the rows' numbers are on
  // their way, by every wave for itself (all write the same numbers; a wave reads its own), then rows, scales and the first
  // two tiles together.
  bf16x8 qf[2 * D / 32];
  {
    const int pg = look(0);
    const size_t ph = size_t(max(pg, 0)) * a.c.heads + h;
    const bf16* x = a.q + size_t(row) * a.ldq + size_t(hq) * D + 16 * h2;
    uint4 y[2 * D / 32];
#pragma unroll
    for (int m = 0; m < 2 * D / 32; ++m) y[m] = *reinterpret_cast<const uint4*>(x + 16 * m - 8 * (m & 1));
    const uint8_t ksb = a.c.ks[ph], vsb = a.c.vs[ph];
    const uint64_t none = __ballot(pg < 0);
    lds.page[0][lane] = pg;
    if (n > 0) fetch(0, page_at(0));
    if (n > 1) fetch(1, page_at(1));
    if (n > 2) next = page_at(2);
    lds.missing[0] = none;
    lds.ks[0][lane] = e8m0_to_f32(ksb);
    lds.vs[0][lane] = e8m0_to_f32(vsb);
    const uint32_t flip = a.scale2 < 0.0f ? 0x80008000u : 0;  // scores times |scale|: their largest is the largest weight's
#pragma unroll
    for (int m = 0; m < 2 * D / 32; ++m) {
      y[m].x ^= flip, y[m].y ^= flip, y[m].z ^= flip, y[m].w ^= flip;
      qf[m] = bf16x8_of(y[m]);
    }
  }
  const int krow = 16 * (c >> 2 & 1) + 4 * (c >> 3) + (c & 3);  // the token that is this lane's row of a half
  const int kat = krow * D + 16 * key_piece<D>(krow, h2), vat = c * 64;
  for (int t = 0; t < n; ++t) {
    if (t + 1 < n) pipe::wait_vm<2 * S::LOADS>();
    else pipe::wait_vm<0>();
    pipe::lds_barrier();  // tile t is there, and every wave is done with tile t - 1
    if (t % PR_META == PR_META - 4 && t / PR_META * PR_META + PR_META < n) meta(t / PR_META + 1);
    if (t + 2 < n) fetch(t + 2, next);
    if (t + 3 < n) next = page_at(t + 3);
    const int t0 = token(t), mt = t / PR_META & 1, mi = t % PR_META * 4;
    if (t % PR_META == 0) {
      const uint64_t x = lds.missing[mt];
      missing = uint64_t(uint32_t(uniform(int(x >> 32)))) << 32 | uint32_t(uniform(int(x)));
    }
    if (wrow >= nrows || t0 > pos_hi) continue;
    const uint8_t *kt = lds.k[t % PR_STAGES], *vt = lds.v[t % PR_STAGES];
    const bool masked = t0 + TILE - 1 > pos_lo || (missing >> mi & 15) != 0 ||
                        (a.window > 0 && int64_t(t0) + a.window <= pos_hi && t0 + TILE > a.sinks);

    uint4 kx[2][D / 32];
    float ks[2], vs[2];
#pragma unroll
    for (int T = 0; T < 2; ++T) {
      ks[T] = lds.ks[mt][mi + 2 * T + (c >> 2 & 1)];
      vs[T] = lds.vs[mt][mi + 2 * T + h2];
#pragma unroll
      for (int m = 0; m < D / 32; ++m) kx[T][m] = ld16(kt + 32 * T * D + (kat ^ 32 * m));
    }
    __builtin_amdgcn_sched_barrier(0);  // every read on its way before the first product waits for one
    pipe::v16f_t s[2];  // (products that follow one another add to different sums: none waits for the one before)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[0][r] = s[1][r] = 0.0f;
#pragma unroll
    for (int m = 0; m < D / 32; ++m) {
#pragma unroll
      for (int T = 0; T < 2; ++T)
        s[T] = pipe::mfma32_bf16(fp8x8_to_bf16(kx[T][m].x, kx[T][m].y, ks[T]), qf[2 * m], s[T]);
#pragma unroll
      for (int T = 0; T < 2; ++T)
        s[T] = pipe::mfma32_bf16(fp8x8_to_bf16(kx[T][m].z, kx[T][m].w, ks[T]), qf[2 * m + 1], s[T]);
    }
    uint4 vx[2][S::DT];
#pragma unroll
    for (int T = 0; T < 2; ++T)
#pragma unroll
      for (int d = 0; d < S::DT; ++d) vx[T][d] = ld16(vt + vat + 16 * value_piece(c, 2 * T + h2) + d * 2048);
    __builtin_amdgcn_sched_barrier(0);
    uint32_t see[2] = {0xffff, 0xffff};
    int there[2] = {16, 16};  // of this lane's 16 values, those of tokens that are there
    if (masked) {
#pragma unroll
      for (int T = 0; T < 2; ++T) {
        const int tt = t0 + 32 * T + 16 * h2;
        const bool none = missing >> (mi + 2 * T + h2) & 1;
        see[T] = none ? 0 : seen_bits(pos, tt, a.window, a.sinks);
        there[T] = none ? 0 : min(max(q.len - tt, 0), 16);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[T][r] = see[T] >> r & 1 ? s[T][r] : -INFINITY;
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int T = 0; T < 2; ++T)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[T][r]);
    top = max_halves(top) * sc;
    if (__any(top > ref2 + PR_LAG)) {
      const float to = fmaxf(ref2, top), al = __builtin_amdgcn_exp2f(ref2 - (to == -INFINITY ? 0.0f : to));
#pragma unroll
      for (int d = 0; d < S::DT; ++d) o[d] *= al;
      l *= al;
      ref2 = to;
    }
    const float base = ref2 == -INFINITY ? 0.0f : ref2;
#pragma unroll
    for (int T = 0; T < 2; ++T)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[T][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[T][r], sc, -base));
        l += s[T][r];  // (before the rounding to bf16: lse is as exact as fp32 is)
      }
    bf16x8 p[2][2];
#pragma unroll
    for (int T = 0; T < 2; ++T)
#pragma unroll
      for (int e = 0; e < 16; ++e) p[T][e / 8][e % 8] = __bf16(s[T][e]);
    if (masked) {  // slots past the last token hold anything: zero
      if (__builtin_expect(__any(fmaxf(vs[0], vs[1]) == INFINITY), 0)) {  // NAN_SCALE: its codes are NaN
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int d = 0; d < S::DT; ++d)
            if (vs[T] == INFINITY) vx[T][d] = make_uint4(NAN_CODES, NAN_CODES, NAN_CODES, NAN_CODES);
      }
      uint32_t bad = 0;
#pragma unroll
      for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int d = 0; d < S::DT; ++d) {
          uint4& x = vx[T][d];
          x.x &= first_bytes(there[T]), x.y &= first_bytes(there[T] - 4), x.z &= first_bytes(there[T] - 8);
          x.w &= first_bytes(there[T] - 12);
          bad |= nan_bytes(x.x) | nan_bytes(x.y) | nan_bytes(x.z) | nan_bytes(x.w);
        }
      if (__builtin_expect(__any(bad != 0), 0)) {
        // 0 x NaN is NaN: the NaN among the values are taken out, and each is set by itself in the sums of the rows that see
        // it, from the codes in LDS (few registers; how long it takes does not matter).
#pragma unroll
        for (int d = 0; d < S::DT; ++d)
          for (int k = 0; k < 8; ++k) {
            const int T = k >> 2, j = 4 * (k & 3);  // tokens j .. j + 3 of the lane's 16
            uint32_t x = *reinterpret_cast<const uint32_t*>(vt + vat + 16 * value_piece(c, 2 * T + h2) + d * 2048 + j);
            if ((T ? vs[1] : vs[0]) == INFINITY) x = NAN_CODES;
            const uint32_t nan = nan_bytes(x & first_bytes((T ? there[1] : there[0]) - j));
            for (uint64_t left = __ballot(nan != 0); left; left &= left - 1) {
              const int from = __ffsll((unsigned long long)left) - 1;  // its channel: row 8a + 4h + i of the products
              const uint32_t bits = lane_of(nan, from);
              for (int e = 0; e < 4; ++e) {
                if (!(bits >> (8 * e + 7) & 1)) continue;
                const int tok = t0 + 32 * T + (from & 32) / 2 + j + e, to = from / 8 % 4 * 4 + from % 4;
                const bool hit = h2 == (from >> 2 & 1) && (seen_bits(pos, tok, a.window, a.sinks) & 1);
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] = hit && r == to ? __builtin_nanf("") : o[d][r];
              }
            }
          }
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int d = 0; d < S::DT; ++d) {
            uint4& x = vx[T][d];
            x = make_uint4(no_nan(x.x), no_nan(x.y), no_nan(x.z), no_nan(x.w));
          }
      }
#pragma unroll
      for (int T = 0; T < 2; ++T) vs[T] = vs[T] == INFINITY ? 1.0f : vs[T];
    }
#pragma unroll
    for (int T = 0; T < 2; ++T) {
#pragma unroll
      for (int d = 0; d < S::DT; ++d)
        o[d] = pipe::mfma32_bf16(fp8x8_to_bf16(vx[T][d].x, vx[T][d].y, vs[T]), p[T][0], o[d]);
#pragma unroll
      for (int d = 0; d < S::DT; ++d)
        o[d] = pipe::mfma32_bf16(fp8x8_to_bf16(vx[T][d].z, vx[T][d].w, vs[T]), p[T][1], o[d]);
    }
  }
  l += __shfl_xor(l, 32, 64);
  const auto four = [&](int d, int r) { return v4f{o[d][4 * r], o[d][4 * r + 1], o[d][4 * r + 2], o[d][4 * r + 3]}; };
  if constexpr (COMMON) {  // [row][D]: they are joined by sequences
    if (wrow + c >= nrows) return;
    const size_t at = size_t(sums) + 32 * wave + c;
#pragma unroll
    for (int d = 0; d < S::DT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) *reinterpret_cast<v4f*>(a.so + at * D + 32 * d + 8 * r + 4 * h2) = four(d, r);
    if (h2 == 0) *reinterpret_cast<float2*>(a.sml + at * 2) = make_float2(ref2, l);
    return;
  }
  if (parts == 1) {
    if (wrow + c >= nrows) return;
#pragma unroll
    for (int d = 0; d < S::DT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        store_out<D>(a, row, hq, 32 * d + 8 * r + 4 * h2, four(d, r), l, ref2, d == 0 && r == 0 && h2 == 0);
    return;
  }
  // Partial sums as the lanes hold them: [slot][wave][four channels of a lane][lane], whole lines.
  if (wrow >= nrows) return;
#pragma unroll
  for (int d = 0; d < S::DT; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<v4f*>(a.po + (size_t(blockIdx.x) * (PR_ROWS * D / 4) + ((wave * S::DT + d) * 4 + r) * 64 + lane) * 4) =
          four(d, r);
  if (h2 == 0) *reinterpret_cast<float2*>(a.pml + (size_t(blockIdx.x) * PR_ROWS + 32 * wave + c) * 2) = make_float2(ref2, l);
}

// ---- host -------------------------------------------------------------------------------------------------------------
// f.operator()<D>() for the cache's dim.
template <class F>
void by_dim(int dim, F&& f) {
  if (dim == 64) f.template operator()<64>();
  else if (dim == 128) f.template operator()<128>();
  else f.template operator()<256>();
  UH_CHECK_LAUNCH();
}
// Which kernels a step takes.
struct Way {
  int few;  // rows (of a key / value head) of a sequence up to which it is the split kernel's
  bool split, tiled;
};
// The operands' checks; false: there is nothing to do.
bool check_attend(const char* who, const bf16* q, int ldq, const KvStep& s, const KvCache& c, int Hq, float scale, int sinks,
                  const bf16* out, int ldo, const void* ws, size_t ws_bytes, size_t need);
Attend attend_of(const bf16* q, int ldq, const KvStep& s, const KvCache& c, int Hq, float scale, int window, int sinks, bf16* out,
                 int ldo, float* lse, const Way& way, void* ws);
// The tiled kernel and its join: blocks of rows times heads, at most so many.
void launch_tiled(const Attend& a, int64_t blocks, hipStream_t st);

}  // namespace unholy::kernels::kv
