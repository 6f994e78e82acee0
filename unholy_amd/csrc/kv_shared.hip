// Attention of sequences that begin alike over the 8-bit paged key / value cache: who shares what, and the attention that
// reads it once (include/unholy/kernels/kv_cache.hpp has the contracts).
#include "kv_attend_core.hpp"

namespace unholy::kernels {

using namespace uh;
using namespace kv;

namespace {

// ---- the plan ---------------------------------------------------------------------------------------------------------
// A wave a sequence finds the lowest sequence of its class (the same number, or first page) and how far their tables agree, 256
// entries at a time; the workgroup that finishes last makes the plan of what all have found: for each class the length that
// saves the most tiles' reads, then places and lists. Loops over all pairs of sequences go through LDS, up to SH_MOST sequences
// (through the plan past that). They take time with the square of how many there are (256 14 us, 1024 84, 2048 0.8 ms, 4096 2.9,
// and 8192 would take 11): sequences past the first SHARE_SEQS are in no group, and cost the plan a store each.
constexpr int SH_NT = 256;
constexpr int SH_MOST = 1024;
constexpr int SH_AHEAD = SHARE_AHEAD;
static_assert(SHARE_ROWS < 32);
constexpr int SH_KEYS = 2048;  // classes and first positions of sequences, in LDS at a time

// The class of sequence b, -1 if it is in none.
__device__ __forceinline__ int share_key(const int32_t* group, const KvStep& st, int pages, int page, int b, const Seq& q) {
  const int n = q.r1 - q.r0, key = group ? group[b] : page_of(st.table, st.max_blocks, pages, b, 0);
  const int64_t whole = int64_t(min(max(q.first, 0) / page, st.max_blocks)) * page;
  return n >= 1 && n <= SHARE_ROWS && !too_many(st, q) && whole >= SHARE_TILE && key >= 0 && (!group || key < st.B) ? key : -1;
}

template <bool LDS>
__global__ __launch_bounds__(SH_NT) void kv_share_kernel(const int32_t* __restrict__ group, KvStep st, int pages, int page,
                                                         Share sh) {
  __shared__ int2 wsum[SH_NT / 64];
  __shared__ union {
    int2 keys[SH_KEYS];
    struct {
      int4 found[LDS ? SH_MOST : 1];  // (a multiple of SH_AHEAD, as the plan's)
      unsigned long long best[LDS ? SH_MOST : 1];
      int2 sums[LDS ? SH_MOST : 1];
      alignas(16) uint32_t key[LDS ? SH_MOST : 4];  // what a loop over all compares, in one number: SH_MOST is 2^10
    } all;
  } lds;
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int B = LDS ? st.B : share_seqs(st.B);  // sequences that may be in a group

  if constexpr (!LDS)
    for (int b = B + int(blockIdx.x) * SH_NT + tid; b < st.B; b += int(gridDim.x) * SH_NT) sh.seqs[b] = ShareSeq{0, 0, 0, 0};
  for (int b0 = blockIdx.x * (SH_NT / 64); b0 < B; b0 += gridDim.x * (SH_NT / 64)) {
    const int b = b0 + wave;
    Seq q{};
    int key = -1, rep = -1, first = 0, same = 0;  // rep: the lowest of the class, first: the position of its first row
    if (b < B) {
      q = seq_of(st, b);
      key = share_key(group, st, pages, page, b, q);
    }
    for (int k0 = 0; k0 < min(b0 + SH_NT / 64, B); k0 += SH_KEYS) {
      __syncthreads();  // the keys' last use
      for (int i = tid; i < min(SH_KEYS, min(b0 + SH_NT / 64, B) - k0); i += SH_NT) {
        const Seq s = seq_of(st, k0 + i);
        lds.keys[i] = make_int2(share_key(group, st, pages, page, k0 + i, s), s.first);
      }
      __syncthreads();
      for (int i = 0; key >= 0 && rep < 0 && i < min(SH_KEYS, b + 1 - k0); i += 64) {
        const uint64_t hit = __ballot(i + lane < min(SH_KEYS, b + 1 - k0) && lds.keys[i + lane].x == key);
        if (hit) {
          const int at = i + __ffsll((unsigned long long)hit) - 1;
          rep = k0 + at;
          first = lds.keys[at].y;
        }
      }
    }
    if (rep >= 0) {
      const int most = min(min(q.first, first) / page, st.max_blocks);
      const int32_t *x = st.table + size_t(b) * st.max_blocks, *y = st.table + size_t(rep) * st.max_blocks;
      constexpr int AHEAD = 4;
      for (bool all = true; all && same < most;) {
        int u[AHEAD], v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const int j = min(same + k * 64 + lane, most - 1);
          u[k] = x[j], v[k] = y[j];
        }
        const int from = same;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const bool ok = from + k * 64 + lane < most && u[k] == v[k] && u[k] >= 0 && u[k] < pages;
          const uint64_t bad = ~__ballot(ok);
          if (all) same += bad ? __ffsll((unsigned long long)bad) - 1 : 64;
          all = all && !bad;
        }
      }
    }
    if (b < B && lane < 4) {
      const int tiles = int(int64_t(same) * page / SHARE_TILE);
      const int v = lane == 0 ? rep : lane == 1 ? tiles : lane == 2 ? q.r1 - q.r0 : q.first;
      __hip_atomic_store(&reinterpret_cast<int*>(sh.found + b)[lane], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  // (through to memory, as the attention's partial sums go; the last workgroup reads them from there)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0)
    last = __hip_atomic_fetch_add(&sh.head->done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;

  // f(i, the first two of what was found of sequence i), i < n, in order: SH_AHEAD reads on their way at a time
  const auto for_all = [&](const int4* found, int n, auto f) {
    for (int i0 = 0; i0 < n; i0 += SH_AHEAD) {
      int2 v[SH_AHEAD];
#pragma unroll
      for (int k = 0; k < SH_AHEAD; ++k) v[k] = *reinterpret_cast<const int2*>(found + i0 + k);
#pragma unroll
      for (int k = 0; k < SH_AHEAD; ++k) f(i0 + k, v[k].x, v[k].y);
    }
  };
  // The same of the keys in LDS, f(i, key), from i0 on (256 sequences: 14.3 us for the plan, 18.2 with two numbers to compare).
  const auto for_keys = [&](int i0, int n, auto f) {
    for (; i0 < n; i0 += SH_AHEAD) {
      uint4 v[SH_AHEAD / 4];
#pragma unroll
      for (int k = 0; k < SH_AHEAD / 4; ++k) v[k] = *reinterpret_cast<const uint4*>(lds.all.key + i0 + 4 * k);
#pragma unroll
      for (int k = 0; k < SH_AHEAD / 4; ++k)
        f(i0 + 4 * k, v[k].x), f(i0 + 4 * k + 1, v[k].y), f(i0 + 4 * k + 2, v[k].z), f(i0 + 4 * k + 3, v[k].w);
    }
  };
  constexpr int LONG = (1 << 21) - 1;  // tiles that a key has room for: 2^27 tokens
  const uint32_t none = ~0u;
  int4* found = LDS ? lds.all.found : sh.found;  // {lowest of the class, tiles in common with it, rows, position of the first}
  unsigned long long* best = LDS ? lds.all.best : sh.best;  // by the class's lowest: saved, then tiles (25 bits)
  int2* sums = LDS ? lds.all.sums : sh.sums;                // by the same: rows of the group, position of the first of them
  for (int b = tid; b < B; b += SH_NT) {
    int v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      v[k] = __hip_atomic_load(&reinterpret_cast<int*>(sh.found + b)[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if constexpr (LDS) {
      v[1] = min(v[1], LONG);
      lds.all.key[b] = v[0] < 0 ? none : uint32_t(v[0]) << 21 | uint32_t(v[1]);
    }
    found[b] = make_int4(v[0], v[1], v[2], v[3]);
    best[b] = 0;
    sums[b] = make_int2(0, INT32_MAX);
  }
  if (tid < SH_AHEAD && B + tid < (B + SH_AHEAD - 1) / SH_AHEAD * SH_AHEAD) {
    found[B + tid] = make_int4(-2, 0, 0, 0);
    if constexpr (LDS) lds.all.key[B + tid] = none;
  }
  __syncthreads();
  // what each length would save: the tiles of all but one of the sequences that are as long
  for (int b = tid; b < B; b += SH_NT) {
    const int r = found[b].x, t = found[b].y;
    if (r < 0 || t == 0) continue;
    int count = 0;
    if constexpr (LDS) {
      const uint32_t from = uint32_t(r) << 21 | uint32_t(t);
      for_keys(0, B, [&](int, uint32_t key) { count += int(key - from <= uint32_t(LONG - t)); });
    } else {
      for_all(found, B, [&](int, int rep, int tiles) { count += int(rep == r) & int(tiles >= t); });
    }
    if (count > 1) atomicMax(&best[r], (unsigned long long)min(int64_t(count - 1) * t, int64_t(1) << 38) << 25 | (unsigned long long)t);
  }
  __syncthreads();
  // who is in a group: found becomes {lowest of the group or -1, rows, position of the first, first row of the step}
  for (int b = tid; b < B; b += SH_NT) {
    const int4 f = found[b];
    const int t = f.x >= 0 ? int(best[f.x] & 0x1ffffff) : 0;
    const bool member = t > 0 && f.y >= t;
    if (member) {
      atomicAdd(&sums[f.x].x, f.z);
      atomicMin(&sums[f.x].y, f.w);
    }
    found[b] = make_int4(member ? f.x : -1, f.z, f.w, seq_of(st, b).r0);
    if constexpr (LDS) lds.all.key[b] = member ? uint32_t(f.x) << 5 | uint32_t(f.z) : none;  // (up to SHARE_ROWS rows)
  }
  __syncthreads();
  // the groups in the order of their lowest sequences
  int groups = 0, list = 0;
  for (int b0 = 0; b0 < B; b0 += SH_NT) {
    const int b = b0 + tid;
    const bool head = b < B && found[b].x == b;  // (the lowest of a class is as long as any of it)
    const int rows = head ? sums[b].x : 0;
    const uint32_t g = wave_scan(head), l = wave_scan(uint32_t(rows));
    __syncthreads();  // the last round's reads
    if (lane == 63) wsum[wave] = int2{int(g), int(l)};
    __syncthreads();
    int at = groups + int(g) - int(head), row0 = list + int(l) - rows;
#pragma unroll
    for (int i = 0; i < SH_NT / 64; ++i) {
      if (i < wave) at += wsum[i].x, row0 += wsum[i].y;
      groups += wsum[i].x;
      list += wsum[i].y;
    }
    if (head) {
      sh.groups[at] = ShareGroup{row0, rows, int(best[b] & 0x1ffffff), b, sums[b].y, {0, 0, 0}};
      sums[b] = make_int2(row0, at);
    }
  }
  // (A cu that does not ascend names rows more than once: where that is more than the list has room for, nobody is in a group.)
  const bool fits = list <= st.rows;
  if (!fits) groups = list = 0;
  __syncthreads();
  // the rows of a group in the order of the slots
  for (int b = tid; b < B; b += SH_NT) {
    const int4 f = found[b];
    if (f.x < 0 || !fits) {
      sh.seqs[b] = ShareSeq{0, 0, 0, 0};
      continue;
    }
    int at = 0;
    if constexpr (LDS) {
      const auto rows = [&](uint32_t key) {
        const uint32_t n = key - (uint32_t(f.x) << 5);
        return n < 32 ? int(n) : 0;
      };
      const int whole = b & -SH_AHEAD;
      for_keys(0, whole, [&](int, uint32_t key) { at += rows(key); });
      for_keys(whole, b, [&](int i, uint32_t key) { at += i < b ? rows(key) : 0; });
    } else {
      for_all(found, b, [&](int i, int rep, int rows) { at += int(rep == f.x) & int(i < b) ? rows : 0; });
    }
    const int2 to = sums[f.x];
    sh.seqs[b] = ShareSeq{int(best[f.x] & 0x1ffffff), at, to.x, to.y};
    for (int i = 0; i < f.y; ++i) sh.list[to.x + at + i] = make_int2(f.w + i, b);
  }
  if (tid == 0) {
    ShareHead& h = *sh.head;
    h.magic = SHARE_MAGIC, h.B = st.B, h.rows = st.rows, h.max_new = st.max_new, h.max_blocks = st.max_blocks, h.page = page;
    h.groups = groups, h.list = list;
    __hip_atomic_store(&h.done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // as it was found
  }
}

// ---- the attention -----------------------------------------------------------------------------------------------------
// Two launches. In the first, some workgroups take the groups' blocks of PR_ROWS rows over the tiles that their sequences have
// in common (kv_tiled_kernel: the rows of up to PR_ROWS / heads sequences share each tile's read and conversion), the others
// every sequence's own tiles (own_segments), side by side: the first are bound by the matrix and vector units, the second by
// memory and by loads that depend on each other. All leave partial sums, and the second launch joins them by sequence and head.
// (Where the blocks of 64 channels have many tiles, every workgroup takes own segments first and then a part of a block.)

// How the workgroups are dealt, worked out by each of them from what the device knows.
struct Deal {
  uint32_t common;  // workgroups of the groups' blocks; those behind them are the sequences'
  uint32_t share;   // tiles of a part at most
  bool single;      // whole blocks
  bool both;        // each workgroup takes own segments and then a part of a block
  Split own;
};
constexpr uint32_t NONE = 1u << 30;
// A block's tile, which its workgroup's waves take together, in sequences' tiles, of which each takes its own. (Where that
// decides: 3 rather than 6 for 4 x 16 sequences of up to 2000 tokens behind 3000, 128 channels: 41 us / 46; 128 of 500 behind
// 2000: 32 / 37; with 256 channels 8 x 8 of 900 behind 3000: 42 / 57; 128 of 500 behind 2000: 40 / 39. With 2, 2 x 32 of 3000
// behind 1500 and 256 channels 75 / 51.)
constexpr float COMMON_TILE = 3.0f;

// Of a group: blocks of rows, and tiles that its rows see.
struct GroupWork {
  uint32_t blocks, count;
};
__device__ __forceinline__ GroupWork group_work(const AttendShared& a, const ShareGroup& g, bool is) {
  GroupWork w{0, 0};
  if (is) {
    w.blocks = uint32_t(row_groups(g.rows * a.group, PR_ROWS));
    w.count = uint32_t(tiles_of(a, Seq{0, 0, g.tiles * TILE, g.first}).count);
  }
  return w;
}
__device__ __forceinline__ ShareGroup group_at(const AttendShared& a, int i) { return a.share.groups[min(i, a.st.B / 2)]; }
// Of sequence b: segments, and each one's tiles.
struct SeqWork {
  Seq q;
  Tiles t;
  uint32_t segs;
  int list;
};
__device__ __forceinline__ SeqWork seq_work(const AttendShared& a, int b, const ShareSeq& mine, const Seq& q, bool fits,
                                            bool& over) {
  SeqWork w{};
  if (b >= a.st.B) return w;
  w.q = q;
  over |= too_many(a.st, q);
  if (is_few(a, q)) {
    w.segs = uint32_t(segments_of(a, q));
    w.t = tiles_of(a, q, fits ? mine.tiles : 0);
    w.list = list_of(a, mine, q);
  }
  return w;
}
__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

struct FindLds {
  ShareGroup groups[64];  // the first of them
  uint32_t sums[AT_WAVES][2];
  int over[AT_WAVES];
  int found[AT_WAVES][12];
};

// The part `at` of the groups' blocks.
__device__ __forceinline__ bool find_common(const AttendShared& a, const Deal& deal, int n, const FindLds& lds, uint32_t at,
                                            BlockPart& p, int& sums) {
  const int lane = threadIdx.x & 63;
  const uint32_t heads = uint32_t(a.c.heads);
  uint32_t from = 0;
  for (int b0 = 0; b0 < n; b0 += 64) {
    const ShareGroup g = b0 ? group_at(a, b0 + lane) : lds.groups[lane];
    const GroupWork w = group_work(a, g, b0 + lane < n);
    const uint32_t parts = parts_of(w.count, deal.share), wgs = w.blocks * parts * heads, end = from + wave_scan(wgs);
    const uint64_t hit = __ballot(at < end);
    if (hit) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      const uint32_t in = at - lane_of(end - wgs, l), np = lane_of(parts, l);
      const int row0 = int(lane_of(g.row0, l)), block = int(in / heads / np);
      p.b = int(lane_of(g.seq, l));
      p.h = int(in % heads);
      p.index = int(in / heads % np);
      p.parts = int(np);
      p.row0 = block * PR_ROWS;
      p.q = Seq{row0, row0 + int(lane_of(g.rows, l)), int(lane_of(g.tiles, l)) * TILE, int(lane_of(g.first, l))};
      p.t = tiles_of(a, p.q);
      const int each = p.t.count / p.parts, more = p.t.count % p.parts;
      p.i0 = p.index * each + min(p.index, more);
      p.i1 = p.i0 + each + (p.index < more ? 1 : 0);
      // whole blocks: a head's rows follow each other in the order of the list; else a workgroup has PR_ROWS places of its own
      sums = deal.single ? (p.h * a.share.head->list + row0) * a.group + p.row0 : int(at) * PR_ROWS;
      if (threadIdx.x == 0 && p.index == 0)
        a.common[(size_t(row0) * a.group / PR_ROWS + (b0 + l) + block) * heads + p.h] = Common{sums, p.parts};
      return true;
    }
    from = lane_of(end, 63);
  }
  return false;
}

// The segments that hold the first units of the workgroup's waves, u of the first wave: a sequence a thread, found through LDS.
__device__ __forceinline__ bool find_own(const AttendShared& a, const Deal& deal, bool fits, SeqWork w, uint32_t u, FindLds& lds,
                                         Walk& k) {
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63;
  if (tid < AT_WAVES) lds.found[tid][0] = -1;
  uint32_t from = 0;
  for (int b0 = 0; b0 < a.st.B; b0 += AT_NT) {
    const int b = b0 + tid;
    bool over = false;
    if (a.st.B > AT_NT) w = seq_work(a, b, a.share.seqs[min(b, a.st.B - 1)], seq_of(a.st, min(b, a.st.B - 1)), fits, over);
    const uint32_t each = units_of(deal.own, uint32_t(w.t.count)), n = w.segs * each;
    uint32_t end = wave_scan(n);
    __syncthreads();  // the LDS' last use
    if (lane == 63) lds.sums[wave][0] = end;
    __syncthreads();
    uint32_t all = from;
#pragma unroll
    for (int i = 0; i < AT_WAVES; ++i) {
      end += i < wave ? lds.sums[i][0] : 0;
      all += lds.sums[i][0];
    }
    end += from;
#pragma unroll
    for (int i = 0; i < AT_WAVES; ++i) {
      const uint32_t ui = u + uint32_t(i) * deal.own.unit;
      if (ui >= end || ui < end - n) continue;
      int* f = lds.found[i];
      const uint32_t seg = (ui - (end - n)) / each;
      f[0] = b, f[1] = w.q.r0, f[2] = w.q.r1, f[3] = w.q.len, f[4] = w.q.first;
      f[5] = w.t.sink_tiles, f[6] = w.t.skip, f[7] = w.t.count, f[8] = w.t.from;
      f[9] = int(seg), f[10] = int(end - n + seg * each), f[11] = w.list;
    }
    from = all;
    if (u + (AT_WAVES - 1) * deal.own.unit < all) break;
  }
  __syncthreads();
  int f[12];
#pragma unroll
  for (int i = 0; i < 12; ++i) f[i] = uniform(lds.found[wave][i]);
  k.b = f[0];
  k.q = Seq{f[1], f[2], f[3], f[4]};
  k.t = Tiles{f[5], f[6], f[7], f[8]};
  k.h = f[9] % a.c.heads;
  k.part = f[9] / a.c.heads;
  k.at = uint32_t(f[10]);
  k.list = f[11];
  return k.b >= 0;
}

// A wave's segments, from w on (of the launch's waves for them, the wv-th): what a sequence has for itself is mostly a few
// tiles, which four waves would begin and join for a tile each. A sequence's rows, up to SHARE_ROWS times the query heads of a
// head, go FEW at a time; the tiles that its group has in common are left out, and sums that others belong to are left to
// kv_shared_join_kernel. (A second tile on its way all the time: no faster, with 128 channels 4 us slower for its registers.)
template <int D>
__device__ __forceinline__ void own_segments(const AttendShared& a, const Split& sp, Walk w, uint32_t wv) {
  using S = Shape<D>;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int mask = a.c.page - 1, sh = a.page_shift;
  Part pt = part_of(sp, w, wv * sp.unit, wv);
  uint4 kr[4][S::KL];
  uint32_t vr[S::DT][4];
  int ksb, vsb, pk, pv, pk1, pv1;
  const auto token = [&](int i) { return w.t.at(i) * TILE; };
  const auto lookup = [&](int t0, int& pk, int& pv) {  // the pages of this lane's key rows and of its values
    pk = page_of(a.st.table, a.st.max_blocks, a.c.pages, w.b, (t0 + 16 * (c >> 2)) >> sh);
    pv = page_of(a.st.table, a.st.max_blocks, a.c.pages, w.b, (t0 + 16 * g) >> sh);
  };
  const auto load_k = [&](int t0, int pk) {
    const size_t ph = size_t(max(pk, 0)) * a.c.heads + w.h;
    const uint8_t* p = a.c.k + ((ph << sh) + ((t0 + 16 * (c >> 2) + (c & 3)) & mask)) * D + 16 * g;
    ksb = a.c.ks[ph];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int m = 0; m < S::KL; ++m) kr[j][m] = ld16(p + 4 * j * D + 64 * m);
  };
  const auto load_v = [&](int t0, int pv) {
    const size_t ph = size_t(max(pv, 0)) * a.c.heads + w.h;
    const uint8_t* p = a.c.v + ((ph * D + c) << sh) + ((t0 + 16 * g) & mask);
    vsb = a.c.vs[ph];
#pragma unroll
    for (int d = 0; d < S::DT; ++d) {
      const uint4 x = ld16(p);
      p += 16 << sh;
      vr[d][0] = x.x, vr[d][1] = x.y, vr[d][2] = x.z, vr[d][3] = x.w;
    }
  };
  for (bool again = true; again;) {
    // the part's rows, and its first loads on their way
    const int row0 = w.part * FEW, rows = min((w.q.r1 - w.q.r0) * a.group - row0, FEW);
    int i = pt.i0;
    if (i < pt.i1) lookup(token(i), pk, pv);
    const int ri = row0 + min(c, rows - 1), r = ri / a.group;
    const int row = w.q.r0 + r, hq = w.h * a.group + ri - r * a.group;
    const FewRow fr{w.q.first + r, w.q.first, w.q.first + (w.q.r1 - w.q.r0) - 1, w.q.len};
    bf16x8 qf[2 * S::KL];
    const bf16* x = a.q + size_t(row) * a.ldq + size_t(hq) * D + 16 * g;
#pragma unroll
    for (int m = 0; m < S::KL; ++m) {
      qf[2 * m] = bf16x8_of(*reinterpret_cast<const uint4*>(x + 64 * m));
      qf[2 * m + 1] = bf16x8_of(*reinterpret_cast<const uint4*>(x + 64 * m + 8));
    }
    if (i < pt.i1) {
      load_k(token(i), pk);
      load_v(token(i), pv);
      if (i + 1 < pt.i1) lookup(token(i + 1), pk1, pv1);
    }
    v4f o[S::DT];
    float mx = -INFINITY, l = 0.0f;
#pragma unroll
    for (int d = 0; d < S::DT; ++d) o[d] = v4f{0, 0, 0, 0};
    for (; i < pt.i1; ++i) {
      const bool more = i + 1 < pt.i1;
      const int pvt = pv;
      few_tile<D>(a, kr, vr, qf, ksb, vsb, pvt, token(i), fr, g, o, mx, l, [&] {
        if (!more) return;
        pk = pk1, pv = pv1;
        load_k(token(i + 1), pk);
        if (i + 2 < pt.i1) lookup(token(i + 2), pk1, pv1);
      });
      if (more) load_v(token(i + 1), pv);
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const bool alone = pt.parts == 1;  // (a wave may begin many of these, but only one that others go on with)
    if (pt.index == 0 && lane == 0) a.own[own_at(a, w.b, w.part, w.h)] = Common{int(wv), pt.parts};
    if (c < rows && alone && w.t.from == 0) {
#pragma unroll
      for (int d = 0; d < S::DT; ++d) store_out<D>(a, row, hq, 16 * d + 4 * g, o[d], l, mx, d == 0 && g == 0);
    } else if (c < rows) {
      const size_t slot = alone ? list_row(a, w.list, w.h, row0 + c) : (size_t(wv) * 2 + (pt.index == 0 ? 1 : 0)) * FEW + c;
      float* to = (alone ? a.lo : a.po) + slot * D + 4 * g;
#pragma unroll
      for (int d = 0; d < S::DT; ++d) *reinterpret_cast<v4f*>(to + 16 * d) = o[d];
      if (g == 0) *reinterpret_cast<float2*>((alone ? a.lml : a.pml) + slot * 2) = make_float2(mx, l);
    }
    again = next_segment(a, sp, w, wv);
    if (again) pt = part_of(sp, w, w.at, wv);
  }
}

// A workgroup's part of a common block for the tiled kernel, or no part: then it goes through own segments.
struct FindShared {
  using Call = AttendShared;
  template <int D>
  static __device__ __forceinline__ bool find(const AttendShared& a, BlockPart& bp, int& sums) {
    __shared__ FindLds lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const uint32_t heads = uint32_t(a.c.heads);

    // all work: the groups' by every wave for itself, a group a lane; the sequences' by all, a sequence a thread. (Every load
    // that depends on no other is on its way before one is waited for.)
    const int b_in = min(tid, a.st.B - 1);
    ShareGroup g = group_at(a, lane);
    const ShareSeq mine = a.share.seqs[b_in];
    const Seq q = seq_of(a.st, b_in);
    const bool fits = share_fits(a.share.head, a.st, a.c.page);
    const int n = fits ? a.share.head->groups : 0;
    if (tid < 64) lds.groups[lane] = g;
    // (sum: of the blocks' tiles, where these are fewer than the chip takes; past that it may wrap)
    uint32_t blocks = 0, sum = 0;
    float common_tiles = 0.0f, rows = 0.0f;  // (rows: of the blocks)
    GroupWork gw{0, 0};
    for (int b0 = 0; b0 < n; b0 += 64) {
      if (b0) g = group_at(a, b0 + lane);
      gw = group_work(a, g, b0 + lane < n);
      blocks += lane_of(wave_scan(gw.blocks), 63) * heads;
      sum += lane_of(wave_scan(gw.blocks * heads * gw.count), 63);
      rows += wave_add(b0 + lane < n ? float(g.rows * a.group) * float(heads) : 0.0f);
      common_tiles += wave_add(float(gw.blocks * heads) * float(gw.count));
    }
    bool over = false;
    SeqWork s = seq_work(a, tid, mine, q, fits, over);
    uint32_t tiles = s.segs * (uint32_t(s.t.count) + START), segs = s.segs;
    for (int b = AT_NT + tid; b < a.st.B; b += AT_NT) {
      const SeqWork x = seq_work(a, b, a.share.seqs[b], seq_of(a.st, b), fits, over);
      tiles += x.segs * (uint32_t(x.t.count) + START);
      segs += x.segs;
    }
    tiles = lane_of(wave_scan(tiles), 63);
    segs = lane_of(wave_scan(segs), 63);
    over = __any(over);
    if (lane == 0) {
      lds.sums[wave][0] = tiles;
      lds.sums[wave][1] = segs;
      lds.over[wave] = over;
    }
    __syncthreads();
    tiles = segs = 0;
    over = false;
#pragma unroll
    for (int i = 0; i < AT_WAVES; ++i) {
      tiles += lds.sums[i][0];
      segs += lds.sums[i][1];
      over |= lds.over[i] != 0;
    }

    // workgroups in proportion, some for each
    Deal deal{};
    deal.share = NONE;
    uint32_t wgs = a.target;  // the sequences'
    if (blocks) {
      const float part = COMMON_TILE * common_tiles / (COMMON_TILE * common_tiles + float(tiles));
      // With up to 128 channels a CU has room for two workgroups. One of each kind there: a block's tile takes 1.6 us, and
      // where some CUs have two blocks, 2.4 to 2.9, which all wait for (64 sequences behind 8003 tokens: 256 workgroups for
      // blocks 27 us, 320 30, 384 29, 128 33; 256 behind 32768: 207, 237, 208, 356).
      // Two of the blocks' where there are tiles enough for as many parts and either the sequences have next to nothing (128
      // behind 131,072: 375 us / 319; with fewer tiles, 16 behind 16000: 25.7 / 29.8) or the blocks' rows are one wave's of
      // four, which leaves the others' units free (4 query heads a head, 16 x 4 behind 4000: 50 us / 40, 8 x 8 behind 6000: 43
      // / 36; with two waves' rows, 8 query heads: 27 / 28).
      // Many tiles of 64 channels: two blocks on every CU, and own segments before them (8 query heads a head, 256 sequences
      // behind 32768 tokens: 272 us / 223; 512 behind 8000: 152 / 141; 64 behind 16000: 44 / 44; behind 8003: 29.6 / 30.7).
      // With 128 channels a wave alone leaves its unit no more than a tenth: 256 behind 32768 201 / 225.
      const bool enough = common_tiles > 6.0f * float(a.target);
      const bool narrow = rows <= 32.0f * float(blocks), little = float(tiles) < 0.32f * common_tiles;
      deal.both = D == 64 && common_tiles > 16.0f * float(a.target) + 0.5f * float(tiles);
      const uint32_t half = a.target / 2, nearly = a.target - a.target / 8;
      const uint32_t most = deal.both ? a.target : D == 256 || (enough && (narrow || little)) ? nearly : half;
      const uint32_t want = deal.both ? most : min(max(uint32_t(part * float(a.target)), 1u), most);
      deal.single = blocks >= want;
      if (deal.single) {  // (where they are more than their share of the chip, one after the other)
        deal.common = blocks;
      } else {
        const uint32_t least = max(4u, root(0.2f, sum, blocks));
        if (n <= 64) deal.share = smallest_share(gw.blocks * heads, gw.count, sum, blocks, want, least);
        else deal.share = max((sum + want - blocks - 1) / (want - blocks), least);
        for (int b0 = 0; b0 < n; b0 += 64) {
          if (n > 64) gw = group_work(a, group_at(a, b0 + lane), b0 + lane < n);
          deal.common += lane_of(wave_scan(gw.blocks * parts_of(gw.count, deal.share)), 63) * heads;
        }
      }
      if (!deal.both) wgs = a.target - min(deal.common, most);
    }
    const uint32_t target = wgs * AT_WAVES;  // waves
    deal.own.whole = segs * 8 <= target;
    const uint32_t lo = 2;  // tiles that are worth a wave
    deal.own.share = deal.own.whole ? max((tiles - START * segs + target - segs - 1) / (target - segs), lo)
                                    : max((tiles + target - 1) / target, lo);
    deal.own.unit = deal.own.whole ? 1 : deal.own.share;

    const bool common = blockIdx.x < deal.common;
    const uint32_t wg = deal.both || common ? blockIdx.x : blockIdx.x - deal.common;
    if ((deal.both || !common) && wg < wgs) {
      if (__builtin_expect(over && !a.blocks, 0)) clear_rows(a, int(wg), int(wgs));  // (else the join's to do)
      Walk w;
      if (find_own(a, deal, fits, s, wg * AT_WAVES * deal.own.unit, lds, w))
        own_segments<D>(a, deal.own, w, wg * AT_WAVES + uint32_t(wave));
    }
    return common && find_common(a, deal, n, lds, blockIdx.x, bp, sums);
  }
};

// A workgroup per (sequence, FEW of its rows, head): its own parts and its group's, in that order, four channels of a row a
// thread, the parts dealt to groups of threads, five at a time (64 sequences behind 8003 tokens 6.4, 6.3, 6.1, 6.5, 6.5
// us with 3, 4, 5, 6 and 10; 256 behind 32768 8.3, 8.4, 8.5, 8.8, 10.9).
constexpr int SJ_FLIGHT = 5;
template <int D>
__global__ __launch_bounds__(AT_NT) void kv_shared_join_kernel(AttendShared a) {
  __shared__ v4f group_o[AT_NT];
  __shared__ float2 group_ml[AT_NT];
  constexpr int ROWS = std::min(AT_NT / (D / 4), FEW);  // of a workgroup: a row's four channels a thread
  const int tid = threadIdx.x, h = int(blockIdx.x % a.c.heads), part = int(blockIdx.x / a.c.heads % a.most_parts);
  const int b = int(blockIdx.x / a.c.heads / a.most_parts);
  const ShareSeq mine = a.share.seqs[b];
  const Common own = a.own[own_at(a, b, part, h)];
  const Seq q = seq_of(a.st, b);
  const bool fits = share_fits(a.share.head, a.st, a.c.page);
  const int in0 = int(blockIdx.y) * ROWS, row0 = part * FEW + in0, rows = min((q.r1 - q.r0) * a.group - row0, ROWS);
  if (!is_few(a, q) || rows <= 0) return;
  // the group's sums of these rows: as many parts for each, which begin at rows of one block or of the next
  int parts = own.parts, upto = 0, begin0 = 0, begin1 = 0;
  if (fits && tiles_of(a, q, mine.tiles).from) {
    const int list = mine.at * a.group + row0, block = list / PR_ROWS;
    const Common* k = a.common + (size_t(mine.row0) * a.group / PR_ROWS + mine.group + block) * a.c.heads + h;
    parts += min(max(k->parts, 0), int(a.target));  // (see list_of)
    begin0 = k->row + list % PR_ROWS;
    upto = (block + 1) * PR_ROWS - list;  // rows in that block
    begin1 = upto < rows ? k[a.c.heads].row - upto : 0;
  }
  if (parts == 1) return;  // written as it was made
  const int items = rows * (D / 4), groups = min(AT_NT / items, AT_WAVES), gi = tid / items, it = tid - gi * items;
  const int r = it / (D / 4), d = it % (D / 4) * 4;
  if (gi < groups) {
    float m = -INFINITY, sum = 0.0f;
    v4f acc{0, 0, 0, 0};
    for (int k0 = gi; k0 < parts; k0 += SJ_FLIGHT * groups) {
      v4f y[SJ_FLIGHT];
      float2 x[SJ_FLIGHT];
#pragma unroll
      for (int k = 0; k < SJ_FLIGHT; ++k) {
        const int p = k0 + k * groups;
        x[k] = make_float2(-INFINITY, 0.0f);
        y[k] = v4f{0, 0, 0, 0};
        if (p >= parts) continue;
        const float *ml = a.sml, *o = a.so;
        const int64_t slot = int64_t((r < upto ? begin0 : begin1) + r) + int64_t(p - own.parts) * a.c.heads * PR_ROWS;
        size_t at = size_t(max(min(slot, int64_t(a.sum_rows) - 1), int64_t(0)));
        if (p < own.parts) {
          const bool alone = own.parts == 1;
          at = alone ? list_row(a, list_of(a, mine, q), h, row0 + r) : size_t(((own.row + p) * 2 + (p == 0 ? 1 : 0)) * FEW + in0 + r);
          ml = alone ? a.lml : a.pml, o = alone ? a.lo : a.po;
        }
        x[k] = *reinterpret_cast<const float2*>(ml + at * 2);
        y[k] = *reinterpret_cast<const v4f*>(o + at * D + d);
      }
      float m1 = m;
#pragma unroll
      for (int k = 0; k < SJ_FLIGHT; ++k) m1 = fmaxf(m1, x[k].x);
      const float ref = m1 == -INFINITY ? 0.0f : m1, al = __builtin_amdgcn_exp2f(m - ref);
      m = m1;
      acc *= al;
      sum *= al;
#pragma unroll
      for (int k = 0; k < SJ_FLIGHT; ++k) {
        const float f = __builtin_amdgcn_exp2f(x[k].x - ref);
        sum += f * x[k].y;
        acc += f * y[k];
      }
    }
    if (groups == 1) {
      store_out<D>(a, q.r0 + (row0 + r) / a.group, h * a.group + (row0 + r) % a.group, d, acc, sum, m, d == 0);
    } else {
      group_o[tid] = acc;
      group_ml[tid] = make_float2(m, sum);
    }
  }
  if (groups == 1) return;
  __syncthreads();
  if (tid < items) {
    float m = -INFINITY, sum = 0.0f;
    v4f acc{0, 0, 0, 0};
    for (int k = 0; k < groups; ++k) m = fmaxf(m, group_ml[k * items + tid].x);
    const float ref = m == -INFINITY ? 0.0f : m;
    for (int k = 0; k < groups; ++k) {
      const float2 x = group_ml[k * items + tid];
      const float f = __builtin_amdgcn_exp2f(x.x - ref);
      sum += f * x.y;
      acc += f * group_o[k * items + tid];
    }
    store_out<D>(a, q.r0 + (row0 + r) / a.group, h * a.group + (row0 + r) % a.group, d, acc, sum, m, d == 0);
  }
}

// Whether a step's tables may name so much that it is worth two launches (13 to 15 us at least, 20 with 256 channels;
// kv_attend's one takes 8 and 12, and where all sequences share one prefix as long overall near 60 MB (16 x 1450 tokens of 8
// heads of 128, or twice as many of 64), and at 90 to 140 MB with 256 channels). Of what they name the launch knows no more
// than how wide they are.
bool worth_sharing(const KvStep& s, const KvCache& c) {
  const double bytes = 2.0 * s.B * s.max_blocks * c.page * c.heads * c.dim;
  return s.B > 1 && bytes > (c.dim <= 128 ? 64e6 : 128e6);
}
// Sequences of up to SHARE_ROWS rows, in a group or alone, are own_segments', the others the tiled kernel's.
Way shared_way(int rows, int max_new, int group) {
  return {SHARE_ROWS * group, true, std::min(rows, max_new) > SHARE_ROWS};
}
// The workspace: counters and blocks, the groups' and the sequences' records, the sequences' sums (those of one part, the
// others), the groups' (where the tiled kernel's lie: it is done before).
struct SharedWs {
  int64_t blocks;     // of the groups, times heads, at most
  int64_t sum_rows;   // of the groups' sums
  int64_t list_rows;  // of the groups, times query heads
  int64_t segments;   // of the sequences
  int most_parts;
  size_t common, own, list, split, bytes;  // offsets; all
};
SharedWs carve_shared(int rows, int max_new, int B, int Hq, int heads, int dim) {
  SharedWs w;
  const int64_t group = Hq / heads, list = std::min<int64_t>(rows, int64_t(SHARE_ROWS) * B);
  const int64_t most = std::min<int64_t>(std::min(rows, max_new), SHARE_ROWS);
  w.blocks = (list * group / PR_ROWS + share_seqs(B) / 2 + 1) * heads;
  w.list_rows = list * Hq;
  w.sum_rows = std::max<int64_t>(int64_t(target_of(dim)) * PR_ROWS, w.list_rows);
  w.most_parts = int((most * group + FEW - 1) / FEW);
  w.segments = int64_t(B) * heads * w.most_parts;
  const auto up = [](size_t n) { return (n + 15) / 16 * 16; };
  w.common = kHeadBytes;
  w.own = up(w.common + size_t(w.blocks) * sizeof(Common));
  const size_t row = (size_t(dim) + 2) * sizeof(float);
  w.list = up(w.own + size_t(w.segments) * sizeof(Common));
  w.split = up(w.list + size_t(w.list_rows) * row);
  w.bytes = w.split + size_t(target_of(dim)) * AT_WAVES * 2 * FEW * row + size_t(w.sum_rows) * row;
  return w;
}

}  // namespace

size_t kv_attend_shared_workspace(int rows, int max_new, int B, int Hq, int heads, int dim) {
  if (rows < 0 || max_new < 0 || B < 0 || heads < 1 || Hq < heads || dim < 1) return 0;
  return std::max(carve_shared(rows, max_new, B, Hq, heads, dim).bytes, kv_attend_workspace(rows, max_new, B, Hq, heads, dim));
}

void kv_attend_shared(const bf16* q, int ldq, const KvStep& s, const KvCache& c, int Hq, float scale, int window, int sinks,
                      bf16* out, int ldo, float* lse, const void* plan, size_t plan_bytes, void* ws, size_t ws_bytes,
                      hipStream_t st) {
  const char* who = "kv_attend_shared";
  const auto fail = [&](const char* what) { throw std::runtime_error(std::string(who) + ": " + what); };
  const size_t need = kv_attend_shared_workspace(s.rows, s.max_new, s.B, Hq, c.heads, c.dim);
  if (!check_attend(who, q, ldq, s, c, Hq, scale, sinks, out, ldo, ws, ws_bytes, need)) return;
  if (!plan) fail("null plan");
  if (!aligned16(plan)) fail("plan not 16-byte aligned");
  if (plan_bytes < kv_share_plan(s.B, s.rows)) fail("plan too small");
  const Way way = shared_way(s.rows, s.max_new, Hq / c.heads);
  AttendShared a{attend_of(q, ldq, s, c, Hq, scale, window, sinks, out, ldo, lse, way, ws)};
  const SharedWs w = carve_shared(s.rows, s.max_new, s.B, Hq, c.heads, c.dim);
  const int64_t tiles = std::max<int64_t>(cdiv(size_t(s.max_blocks) * c.page, TILE), 1);
  const int64_t blocks = (cdiv(size_t(s.rows) * a.group, PR_ROWS) + int64_t(s.B)) * c.heads;
  // (kv_attend counts fewer segments, and refuses what is too much for it)
  const bool too_large =
      w.segments * 8 > INT32_MAX || blocks > INT32_MAX || w.blocks > INT32_MAX || w.sum_rows > INT32_MAX ||
      std::max(w.segments, std::min<int64_t>(std::max(blocks, w.blocks), a.target)) * (tiles + START) > INT32_MAX;
  if (too_large || !worth_sharing(s, c))
    return kv_attend(q, ldq, s, c, Hq, scale, window, sinks, out, ldo, lse, ws, ws_bytes, st);
  a.share = carve_share(const_cast<void*>(plan), s.B, s.rows);
  a.most_parts = w.most_parts;
  a.lists = int(w.list_rows / Hq), a.sum_rows = int(w.sum_rows);
  char* base = static_cast<char*>(ws);
  a.common = reinterpret_cast<Common*>(base + w.common);
  a.own = reinterpret_cast<Common*>(base + w.own);
  a.lo = reinterpret_cast<float*>(base + w.list);
  a.lml = a.lo + size_t(w.list_rows) * c.dim;
  a.so = reinterpret_cast<float*>(base + w.split) + size_t(a.target) * AT_WAVES * 2 * FEW * (c.dim + 2);
  a.sml = a.so + size_t(w.sum_rows) * c.dim;
  if (way.tiled) {
    a.po = a.so;
    a.pml = a.po + size_t(a.target) * PR_ROWS * c.dim;
    launch_tiled(a, blocks, st);
  }
  a.po = reinterpret_cast<float*>(base + w.split);
  a.pml = a.po + size_t(a.target) * AT_WAVES * 2 * FEW * c.dim;
  // As many workgroups as the chip has room for, or more where there may be more blocks than half of that.
  const unsigned grid = unsigned(a.target + std::max<int64_t>(w.blocks - a.target / 2, 0));
  by_dim(c.dim, [&]<int D>() { kv_tiled_kernel<D, FindShared><<<grid, AT_NT, 0, st>>>(a); });
  const dim3 join(unsigned(w.segments), unsigned(FEW * c.dim / 4 / AT_NT));
  by_dim(c.dim, [&]<int D>() { kv_shared_join_kernel<D><<<join, AT_NT, 0, st>>>(a); });
}

size_t kv_share_plan(int B, int rows) { return B < 0 || rows < 0 ? 0 : carve_share(nullptr, B, rows).bytes; }

void kv_share(const int32_t* group, const KvStep& s, int pages, int page, void* plan, size_t plan_bytes, hipStream_t st) {
  const auto fail = [](const char* what) { throw std::runtime_error(std::string("kv_share: ") + what); };
  check_step("kv_share", s);
  check_pages("kv_share", pages);
  if (page != 16 && page != 32 && page != 64 && page != 128) fail("page must be 16, 32, 64 or 128");
  if (s.B > (1 << 24)) fail("B > 2^24");
  if (!plan) fail("null plan");
  if (!aligned16(plan)) fail("plan not 16-byte aligned");
  if (plan_bytes < kv_share_plan(s.B, s.rows)) fail("plan too small");
  if (s.B == 0 || s.rows == 0 || s.max_new == 0) return;
  const Share sh = carve_share(plan, s.B, s.rows);
  const unsigned grid = std::min(cdiv(s.B, SH_NT / 64), 256u);
  if (s.B <= SH_MOST) kv_share_kernel<true><<<grid, SH_NT, 0, st>>>(group, s, pages, page, sh);
  else kv_share_kernel<false><<<grid, SH_NT, 0, st>>>(group, s, pages, page, sh);
  UH_CHECK_LAUNCH();
}

}  // namespace unholy::kernels
