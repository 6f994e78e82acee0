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

__device__ __forceinline__ bool visible(int p, int t, int window, int sinks) {
  return t <= p && (window <= 0 || p - t < window || t < sinks);
}

// What every workgroup knows of the call.
struct Attend {
  const bf16* q;
  bf16* out;
  float* lse;
  KvStep st;
  KvCache c;
  int ldq, ldo, group, page_shift, window, sinks;
  float scale2;  // scale * log2(e): the kernels take powers of two
  float* po;     // partial results: values [slot][16 RT][D], then maximum and sum [slot][16 RT][2]
  float* pml;
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

// Sums over the workgroup's threads before this one, and over all (wsum: AT_WAVES of LDS).
__device__ __forceinline__ int64_t scan64(int64_t v, int64_t* wsum, int64_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) wsum[w] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < AT_WAVES; ++i) {
    before += i < w ? wsum[i] : 0;
    total += wsum[i];
  }
  return before + x - v;
}

// The split of a launch's work, the same in every workgroup and in the launch that joins them. The units are the tiles of
// every (sequence, key / value head, row group), in this order; workgroup w takes units [w share, (w + 1) share), so that
// long and short sequences load the chip evenly whatever their lengths, which only the device knows.
template <int ROWS>
__device__ __forceinline__ int64_t units_of(const Attend& a, int b, int& rg) {
  const Seq q = seq_of(a.st, b);
  rg = row_groups((q.r1 - q.r0) * a.group, ROWS);
  return rg ? int64_t(tiles_of(a, q).count) * rg * a.c.heads : 0;
}
__device__ __forceinline__ int64_t share_of(int64_t units, int wgs) {
  return max((units + wgs - 1) / wgs, int64_t(AT_WAVES));  // a tile for each wave at least
}

__device__ __forceinline__ bf16x8 bf16x8_of(uint4 v) { return __builtin_bit_cast(bf16x8, v); }
__device__ __forceinline__ uint4 ld16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ uint32_t nan_bytes(uint32_t x) {  // the high bit of each byte that is a NaN code
  return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// ---- few rows a sequence: decode and verify steps ---------------------------------------------------------------------
// Bound by reading the cache once. A wave takes 16 RT rows (the (token, query head) pairs that share a key / value head) and
// 64 tokens at a time straight from the cache into registers, no LDS: with S^T = K Q^T the 16x16 product leaves lane
// (row c, group g) the scores of tokens 4g .. 4g + 3 of a 16-token tile, and the tiles' rows are taken in such an order of
// tokens (tile j, row r: token 16 (r / 4) + 4j + r % 4) that over four tiles these are tokens 16g .. 16g + 15: the
// very tokens whose values one 16-byte load of the transposed cache gives it for O^T = V^T P^T. The weights go from one
// product to the other in place, and a row's running maximum and sum are its lane's own.
// The codes become bf16 exactly (v_cvt_scalef32, the block's scale with them), the products sum in fp32; the weights are
// rounded to bf16 for the second product (2^-8 of each at most, as much as the output's own rounding), their sum is taken in
// fp32 before that.
// The waves of a workgroup take every fourth tile and are joined in LDS; workgroups that share rows leave partial sums
// and kv_join_kernel adds them, in the order of the tiles.
constexpr int wgs_per_cu(int dim, int rt) { return rt * dim <= 128 ? 2 : 1; }  // by their registers
template <int D, int RT>
struct Split {
  static constexpr int ROWS = 16 * RT;
  static constexpr int KL = D / 64;  // 16-byte loads of a key row's quarter
  static constexpr int DT = D / 16;  // 16-channel tiles
  struct Lds {
    float o[2][ROWS * D];
    float ml[AT_WAVES][ROWS][2];
  };
};

template <int D, int RT>
__global__ __launch_bounds__(AT_NT, wgs_per_cu(D, RT)) void kv_split_kernel(Attend a) {
  using S = Split<D, RT>;
  __shared__ __align__(16) char lds_raw[sizeof(typename S::Lds)];
  auto& lds = *reinterpret_cast<typename S::Lds*>(lds_raw);
  __shared__ int64_t wsum[AT_WAVES];
  __shared__ int64_t found_at;
  __shared__ int found_b;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;

  // the whole, and where this workgroup's share begins
  int64_t total = 0, sum, mine = 0, before = 0;
  int rg;
  for (int b0 = 0; b0 < a.st.B; b0 += AT_NT) {
    mine = b0 + tid < a.st.B ? units_of<S::ROWS>(a, b0 + tid, rg) : 0;
    before = total + scan64(mine, wsum, sum);
    total += sum;
  }
  const int64_t share = share_of(total, gridDim.x), u0 = share * blockIdx.x, u1 = min(u0 + share, total);
  if (u0 >= total) return;
  if (a.st.B <= AT_NT) {
    if (u0 >= before && u0 < before + mine) found_b = tid, found_at = before;
  } else {
    int64_t at = 0;
    for (int b0 = 0; b0 < a.st.B && at <= u0; b0 += AT_NT) {
      mine = b0 + tid < a.st.B ? units_of<S::ROWS>(a, b0 + tid, rg) : 0;
      before = at + scan64(mine, wsum, sum);
      if (u0 >= before && u0 < before + mine) found_b = b0 + tid, found_at = before;
      at += sum;
    }
  }
  __syncthreads();
  int b = found_b;
  int64_t base = found_at;

  for (int64_t u = u0; u < u1; ++b) {
    const int64_t in_b = units_of<S::ROWS>(a, b, rg);
    const Seq q = seq_of(a.st, b);
    const Tiles tiles = tiles_of(a, q);
    const int nrows = (q.r1 - q.r0) * a.group;
    for (; u < min(u1, base + in_b);) {
      const int seg = int((u - base) / tiles.count), h = seg / rg, row0 = seg % rg * S::ROWS;
      const int64_t seg_at = base + int64_t(seg) * tiles.count;
      const int i0 = int(u - seg_at), i1 = int(min(int64_t(tiles.count), u1 - seg_at));
      u = seg_at + i1;

      // this lane's rows: their positions and queries
      int pos[RT];
      bf16x8 qf[RT][2 * S::KL];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int ri = min(row0 + 16 * r + c, nrows - 1), tok = ri / a.group, hq = h * a.group + ri % a.group;
        pos[r] = q.first + tok;
        const bf16* x = a.q + size_t(q.r0 + tok) * a.ldq + size_t(hq) * D + 16 * g;
#pragma unroll
        for (int m = 0; m < S::KL; ++m) {
          qf[r][2 * m] = bf16x8_of(*reinterpret_cast<const uint4*>(x + 64 * m));
          qf[r][2 * m + 1] = bf16x8_of(*reinterpret_cast<const uint4*>(x + 64 * m + 8));
        }
      }
      const int pos_lo = q.first + row0 / a.group;  // of all rows here
      const int pos_hi = q.first + min(row0 + S::ROWS - 1, nrows - 1) / a.group;

      v4f o[RT][S::DT];
      float mx[RT], l[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        mx[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int d = 0; d < S::DT; ++d) o[r][d] = v4f{0, 0, 0, 0};
      }

      const int mask = a.c.page - 1, sh = a.page_shift;
      const auto lookup = [&](int t0, int& pk, int& pv) {  // the pages of this lane's key rows and of its values
        pk = page_of(a.st.table, a.st.max_blocks, a.c.pages, b, (t0 + 16 * (c >> 2)) >> sh);
        pv = page_of(a.st.table, a.st.max_blocks, a.c.pages, b, (t0 + 16 * g) >> sh);
      };
      uint4 kr[4][S::KL], vr[S::DT];
      int ksb, vsb;
      const auto load_k = [&](int t0, int pk) {
        const size_t ph = size_t(max(pk, 0)) * a.c.heads + h;
        const uint8_t* p = a.c.k + ((ph << sh) + ((t0 + 16 * (c >> 2) + (c & 3)) & mask)) * D + 16 * g;
        ksb = a.c.ks[ph];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int m = 0; m < S::KL; ++m) kr[j][m] = ld16(p + 4 * j * D + 64 * m);
      };
      const auto load_v = [&](int t0, int pv) {
        const size_t ph = size_t(max(pv, 0)) * a.c.heads + h;
        const uint8_t* p = a.c.v + ((ph * D + c) << sh) + ((t0 + 16 * g) & mask);
        vsb = a.c.vs[ph];
#pragma unroll
        for (int d = 0; d < S::DT; ++d) vr[d] = ld16(p + (size_t(16 * d) << sh));
      };

      int i = i0 + wave, pk = 0, pv = 0, pk1 = 0, pv1 = 0;
      if (i < i1) {
        lookup(tiles.at(i) * TILE, pk, pv);
        load_k(tiles.at(i) * TILE, pk);
        load_v(tiles.at(i) * TILE, pv);
        if (i + AT_WAVES < i1) lookup(tiles.at(i + AT_WAVES) * TILE, pk1, pv1);
      }
      for (; i < i1; i += AT_WAVES) {
        const int t0 = tiles.at(i) * TILE, tn = tiles.at(min(i + AT_WAVES, i1 - 1)) * TILE;
        const bool more = i + AT_WAVES < i1;
        const float ks = e8m0_to_f32(uint8_t(ksb)), vs = e8m0_to_f32(uint8_t(vsb));
        v4f s[RT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int r = 0; r < RT; ++r) s[r][j] = v4f{0, 0, 0, 0};
#pragma unroll
          for (int m = 0; m < S::KL; ++m) {
            const bf16x8 k0 = fp8x8_to_bf16(kr[j][m].x, kr[j][m].y, ks), k1 = fp8x8_to_bf16(kr[j][m].z, kr[j][m].w, ks);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              s[r][j] = mfma_bf16(k0, qf[r][2 * m], s[r][j]);
              s[r][j] = mfma_bf16(k1, qf[r][2 * m + 1], s[r][j]);
            }
          }
        }
        const int pvt = pv;
        if (more) {
          pk = pk1, pv = pv1;
          load_k(tn, pk);
          if (i + 2 * AT_WAVES < i1) lookup(tiles.at(i + 2 * AT_WAVES) * TILE, pk1, pv1);
        }
        // what a row does not see: only in the tiles at the ends of what the rows see
        const bool masked = t0 + TILE - 1 > pos_lo || (a.window > 0 && int64_t(t0) + a.window <= pos_hi && t0 + TILE > a.sinks) ||
                            __any(pvt < 0);
        uint32_t see[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          see[r] = 0xffff;
          float top = -INFINITY;
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[r][j][e] *= a.scale2;
              if (masked) {
                const int t = t0 + 16 * g + 4 * j + e;
                if (pvt < 0 || !visible(pos[r], t, a.window, a.sinks)) {
                  s[r][j][e] = -INFINITY;
                  see[r] &= ~(1u << (4 * j + e));
                }
              }
              top = fmaxf(top, s[r][j][e]);
            }
          top = fmaxf(top, __shfl_xor(top, 16, 64));
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          const float m1 = fmaxf(mx[r], top), ref = m1 == -INFINITY ? 0.0f : m1;
          const float al = __builtin_amdgcn_exp2f(mx[r] - ref);
          if (__any(m1 != mx[r])) {
#pragma unroll
            for (int d = 0; d < S::DT; ++d) o[r][d] *= al;
            l[r] *= al;
          }
          mx[r] = m1;
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[r][j][e] = __builtin_amdgcn_exp2f(s[r][j][e] - ref);
              l[r] += s[r][j][e];
            }
        }
        bool nans = false;
        if (masked) {  // slots past the last token hold anything: zero; NaN among the values that some row sees: below
          const int n = pvt < 0 ? 0 : min(max(q.len - (t0 + 16 * g), 0), 16);
          uint32_t keep[4], bad = 0;
#pragma unroll
          for (int w = 0; w < 4; ++w) keep[w] = n >= 4 * w + 4 ? ~0u : n <= 4 * w ? 0u : (1u << (8 * (n - 4 * w))) - 1;
#pragma unroll
          for (int d = 0; d < S::DT; ++d) {
            vr[d].x &= keep[0], vr[d].y &= keep[1], vr[d].z &= keep[2], vr[d].w &= keep[3];
            bad |= nan_bytes(vr[d].x) | nan_bytes(vr[d].y) | nan_bytes(vr[d].z) | nan_bytes(vr[d].w);
          }
          nans = __any(bad != 0);
        }
        bf16x8 p[RT][2];
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int e = 0; e < 8; ++e) p[r][hf][e] = __bf16(s[r][2 * hf + e / 4][e % 4]);
        if (!nans) {
#pragma unroll
          for (int d = 0; d < S::DT; ++d) {
            const bf16x8 v0 = fp8x8_to_bf16(vr[d].x, vr[d].y, vs), v1 = fp8x8_to_bf16(vr[d].z, vr[d].w, vs);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              o[r][d] = mfma_bf16(v0, p[r][0], o[r][d]);
              o[r][d] = mfma_bf16(v1, p[r][1], o[r][d]);
            }
          }
        } else {
          // 0 x NaN is NaN: the NaN values are taken out, and a product of 0 / 1 operands counts for each row and channel
          // the NaN that it sees.
#pragma unroll
          for (int d = 0; d < S::DT; ++d) {
            uint32_t x[4] = {vr[d].x, vr[d].y, vr[d].z, vr[d].w};
            bf16x8 nv[2];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t nb = nan_bytes(x[w]) >> 7;  // 0 / 1 in each byte
              x[w] &= ~(nb * 0xffu);
#pragma unroll
              for (int e = 0; e < 4; ++e) nv[w / 2][w % 2 * 4 + e] = __bf16(float(nb >> (8 * e) & 1));
            }
            const bf16x8 v0 = fp8x8_to_bf16(x[0], x[1], vs), v1 = fp8x8_to_bf16(x[2], x[3], vs);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              bf16x8 sv[2];
#pragma unroll
              for (int e = 0; e < 16; ++e) sv[e / 8][e % 8] = __bf16(float(see[r] >> e & 1));
              v4f n = mfma_bf16(nv[0], sv[0], v4f{0, 0, 0, 0});
              n = mfma_bf16(nv[1], sv[1], n);
              o[r][d] = mfma_bf16(v0, p[r][0], o[r][d]);
              o[r][d] = mfma_bf16(v1, p[r][1], o[r][d]);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (n[e] > 0.0f) o[r][d][e] = __builtin_nanf("");
            }
          }
        }
        if (more) load_v(tn, pv);
      }

      // join the four waves
      __syncthreads();  // the last segment's use of the LDS
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        l[r] += __shfl_xor(l[r], 16, 64);
        l[r] += __shfl_xor(l[r], 32, 64);
        if (g == 0) lds.ml[wave][16 * r + c][0] = mx[r], lds.ml[wave][16 * r + c][1] = l[r];
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < AT_WAVES; ++w) m = fmaxf(m, lds.ml[w][16 * r + c][0]);
        const float ref = m == -INFINITY ? 0.0f : m, f = __builtin_amdgcn_exp2f(mx[r] - ref);
        l[r] = 0.0f;
#pragma unroll
        for (int w = 0; w < AT_WAVES; ++w)
          l[r] += lds.ml[w][16 * r + c][1] * __builtin_amdgcn_exp2f(lds.ml[w][16 * r + c][0] - ref);
        mx[r] = m;
#pragma unroll
        for (int d = 0; d < S::DT; ++d) o[r][d] *= f;
      }
      const auto put = [&](float* to) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int d = 0; d < S::DT; ++d)
            *reinterpret_cast<v4f*>(to + ((r * S::DT + d) * 64 + lane) * 4) = o[r][d];
      };
      const auto add = [&](const float* from) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int d = 0; d < S::DT; ++d)
            o[r][d] += *reinterpret_cast<const v4f*>(from + ((r * S::DT + d) * 64 + lane) * 4);
      };
      if (wave >= 2) put(lds.o[wave - 2]);
      __syncthreads();
      if (wave < 2) add(lds.o[wave]);
      __syncthreads();
      if (wave == 1) put(lds.o[0]);
      __syncthreads();
      if (wave == 0) {
        add(lds.o[0]);
        const bool whole = i0 == 0 && i1 == tiles.count;
        const size_t slot = size_t(blockIdx.x) * 2 + (i0 == 0 ? 1 : 0);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const int ri = row0 + 16 * r + c;
          if (whole) {
            if (ri >= nrows) continue;
            const int row = q.r0 + ri / a.group, hq = h * a.group + ri % a.group;
            const float inv = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
            bf16* y = a.out + size_t(row) * a.ldo + size_t(hq) * D + 4 * g;
#pragma unroll
            for (int d = 0; d < S::DT; ++d) {
              uint16_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = f32_to_bf16(l[r] == 0.0f ? 0.0f : o[r][d][e] * inv);
              *reinterpret_cast<uint2*>(y + 16 * d) =
                  make_uint2(uint32_t(w[0]) | uint32_t(w[1]) << 16, uint32_t(w[2]) | uint32_t(w[3]) << 16);
            }
            if (a.lse && g == 0)
              a.lse[size_t(row) * (a.group * a.c.heads) + hq] = l[r] == 0.0f ? -INFINITY : mx[r] * LN2 + logf(l[r]);
          } else {
            float* y = a.po + (slot * S::ROWS + 16 * r + c) * D + 4 * g;
#pragma unroll
            for (int d = 0; d < S::DT; ++d) *reinterpret_cast<v4f*>(y + 16 * d) = o[r][d];
            if (g == 0) {
              float* ml = a.pml + (slot * S::ROWS + 16 * r + c) * 2;
              ml[0] = mx[r];
              ml[1] = l[r];
            }
          }
        }
      }
    }
    base += in_b;
  }
}

// Rows of sequences without a tile: zero. Rows whose tiles went to several workgroups: their partial sums, in the order of the tiles. A workgroup per row and
// query head; D / 4 lanes hold a partial row, the 1024 / D groups of them take every such partial in turn.
template <int D, int ROWS>
__global__ __launch_bounds__(AT_NT) void kv_join_kernel(Attend a, int wgs) {
  __shared__ int64_t wsum[AT_WAVES];
  __shared__ int64_t at_b;
  constexpr int LANES = D / 4, GROUPS = AT_NT / LANES;
  __shared__ __align__(16) float red[GROUPS][D];
  __shared__ float redm[AT_WAVES], redl[GROUPS];
  const int tid = threadIdx.x, row = blockIdx.x, hq = blockIdx.y, h = hq / a.group;
  int lo = 0, hi = a.st.B;  // the sequence of this row: the first one that ends behind it
  while (lo < hi) {
    const int m = (lo + hi) / 2;
    if (a.st.cu[m + 1] <= row) lo = m + 1; else hi = m;
  }
  const int b = lo;
  if (b >= a.st.B) return;
  const Seq q = seq_of(a.st, b);
  if (row < q.r0 || row >= q.r1) return;
  const int tiles = tiles_of(a, q).count;
  bf16* y = a.out + size_t(row) * a.ldo + size_t(hq) * D;
  float* lse = a.lse ? a.lse + size_t(row) * (a.group * a.c.heads) + hq : nullptr;
  if (tiles == 0) {
    if (tid < D) y[tid] = 0;
    if (tid == 0 && lse) *lse = -INFINITY;
    return;
  }
  int64_t total = 0, sum;
  int rg;
  for (int b0 = 0; b0 < a.st.B; b0 += AT_NT) {
    const int64_t mine = b0 + tid < a.st.B ? units_of<ROWS>(a, b0 + tid, rg) : 0;
    const int64_t before = total + scan64(mine, wsum, sum);
    if (b0 + tid == b) at_b = before;
    total += sum;
  }
  __syncthreads();
  const int64_t share = share_of(total, wgs);
  const int ri = (row - q.r0) * a.group + hq % a.group;
  rg = row_groups((q.r1 - q.r0) * a.group, ROWS);
  const int64_t s0 = at_b + (int64_t(h) * rg + ri / ROWS) * tiles, s1 = s0 + tiles;
  const int w0 = int(s0 / share), w1 = int((s1 - 1) / share), n = w1 - w0 + 1;
  if (n == 1) return;  // written by the one workgroup that had them all
  // in the workgroup that begins these rows they are its range's last, in the others the first
  const auto slot = [&](int i) { return (size_t(w0 + i) * 2 + (i == 0)) * ROWS + ri % ROWS; };
  float m = -INFINITY;
  for (int i = tid; i < n; i += AT_NT) m = fmaxf(m, a.pml[slot(i) * 2]);
  m = wave_max(m);
  if ((tid & 63) == 0) redm[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(redm[0], redm[1]), fmaxf(redm[2], redm[3]));
  const float ref = m == -INFINITY ? 0.0f : m;
  const int grp = tid / LANES, d = tid % LANES * 4;
  v4f acc{0, 0, 0, 0};
  float l = 0.0f;
  for (int i = grp; i < n; i += GROUPS) {
    const size_t sl = slot(i);
    const float f = __builtin_amdgcn_exp2f(a.pml[sl * 2] - ref);
    l += f * a.pml[sl * 2 + 1];
    acc += f * *reinterpret_cast<const v4f*>(a.po + sl * D + d);
  }
  *reinterpret_cast<v4f*>(&red[grp][d]) = acc;
  if (tid % LANES == 0) redl[grp] = l;
  __syncthreads();
  if (tid >= LANES) return;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) {
    acc += *reinterpret_cast<const v4f*>(&red[i][d]);
    l += redl[i];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = f32_to_bf16(l == 0.0f ? 0.0f : acc[e] * inv);
  *reinterpret_cast<uint2*>(y + d) = make_uint2(uint32_t(w[0]) | uint32_t(w[1]) << 16, uint32_t(w[2]) | uint32_t(w[3]) << 16);
  if (tid == 0 && lse) *lse = l == 0.0f ? -INFINITY : m * LN2 + logf(l);
}

// The shape of a split launch: row tiles a wave, and as many workgroups as the chip holds at a time.
struct SplitShape {
  int rt, wgs;
  size_t slots() const { return size_t(wgs) * 2 * 16 * rt; }
};
SplitShape split_shape(int dim, int rows) {
  const int rt = rows <= 16 ? 1 : rows <= 32 || dim == 256 ? 2 : 4;
  return {rt, 256 * wgs_per_cu(dim, rt)};
}
int most_rows(int rows, int max_new, int group) {
  return int(std::min<int64_t>(int64_t(std::min(rows, max_new)) * group, INT32_MAX));
}

}  // namespace

size_t kv_attend_workspace(int rows, int max_new, int B, int Hq, int heads, int dim) {
  if (rows < 0 || max_new < 0 || B < 0 || heads < 1 || Hq < heads || dim < 1) return 0;
  return split_shape(dim, most_rows(rows, max_new, Hq / heads)).slots() * (size_t(dim) + 2) * sizeof(float);
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

  Attend a{q, out, lse, s, c, ldq, ldo, Hq / c.heads, 0, window, sinks, scale * LOG2E, nullptr, nullptr};
  while (1 << a.page_shift < c.page) ++a.page_shift;
  const SplitShape shape = split_shape(c.dim, most_rows(s.rows, s.max_new, a.group));
  a.po = static_cast<float*>(ws);
  a.pml = a.po + shape.slots() * c.dim;
  const auto go = [&]<int D, int RT>() {
    kv_split_kernel<D, RT><<<unsigned(shape.wgs), AT_NT, 0, st>>>(a);
    UH_CHECK_LAUNCH();
    kv_join_kernel<D, 16 * RT><<<dim3(unsigned(s.rows), unsigned(Hq)), AT_NT, 0, st>>>(a, shape.wgs);
    UH_CHECK_LAUNCH();
  };
  const auto by_rt = [&]<int D>() {
    if (shape.rt == 1) go.template operator()<D, 1>();
    else if (shape.rt == 2 || D == 256) go.template operator()<D, 2>();
    else if constexpr (D < 256) go.template operator()<D, 4>();
  };
  if (c.dim == 64) by_rt.template operator()<64>();
  else if (c.dim == 128) by_rt.template operator()<128>();
  else by_rt.template operator()<256>();
}

}  // namespace unholy::kernels
