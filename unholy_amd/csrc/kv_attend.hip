// Attention of a step's rows over the 8-bit paged key / value cache (include/unholy/kernels/kv_cache.hpp has the layout
// and the contract).
#include "kv_attend_core.hpp"

namespace unholy::kernels {

using namespace uh;
using namespace kv;

namespace {

// The segment that holds the workgroup's first unit. Every wave for itself, a sequence a lane: no barriers, and for up to 64
// sequences one pass over registers. over: some sequence brings more than max_new rows.
__device__ __forceinline__ bool find_segment(const Attend& a, Split& s, Walk& w, bool& over) {
  const int lane = threadIdx.x & 63;
  uint32_t segs = 0;  // of this lane's sequence
  int rows = 0;
  const auto look = [&](int b) {
    segs = 0;
    rows = 0;
    w.t = Tiles{0, 0, 0, 0};
    if (b < a.st.B) {
      w.q = seq_of(a.st, b);
      rows = w.q.r1 - w.q.r0;
      if (is_few(a, w.q)) {
        segs = uint32_t(segments_of(a, w.q));
        w.t = tiles_of(a, w.q);
      }
    }
  };
  uint32_t tiles = 0, all = 0;
  over = false;
  for (int b0 = 0; b0 < a.st.B; b0 += 64) {
    look(b0 + lane);
    over |= __ballot(rows > a.st.max_new) != 0;
    tiles += lane_of(wave_scan(segs * (uint32_t(w.t.count) + START)), 63);
    all += lane_of(wave_scan(segs), 63);
  }
  s.whole = all * 8 <= a.target;
  // Equal parts have a tile a wave at least, and where segments are long so many that they (0.35 us each) balance the join by
  // one workgroup (0.014 us a part and row): 16 rows over 131,000 tokens take 45 us a call, in 512 parts of four tiles 99.
  const uint32_t lo = max(uint32_t(AT_WAVES), root(0.04f * float(min(min(a.st.max_new, FEW) * a.group, FEW)), tiles, all));
  if (!s.whole) s.share = max((tiles + a.target - 1) / a.target, uint32_t(AT_WAVES));
  else if (a.st.B <= 64) s.share = smallest_share(segs, uint32_t(w.t.count), tiles - START * all, all, a.target, lo);
  else s.share = max((tiles + a.target - all - 1) / (a.target - all), lo);  // one that is large enough
  s.unit = s.whole ? 1 : s.share;
  const uint32_t u = blockIdx.x * s.unit;
  uint32_t from = 0;
  for (int b0 = 0; b0 < a.st.B; b0 += 64) {
    if (a.st.B > 64) look(b0 + lane);
    const uint32_t each = units_of(s, uint32_t(w.t.count)), n = segs * each, end = from + wave_scan(n);
    const uint64_t hit = __ballot(u < end);
    if (hit) {
      const int l = __ffsll((unsigned long long)hit) - 1;  // (a lane of no segments ends where the one before it does)
      w.b = b0 + l;
      w.q = Seq{int(lane_of(w.q.r0, l)), int(lane_of(w.q.r1, l)), int(lane_of(w.q.len, l)), int(lane_of(w.q.first, l))};
      w.t = Tiles{int(lane_of(w.t.sink_tiles, l)), int(lane_of(w.t.skip, l)), int(lane_of(w.t.count, l)), 0};
      const uint32_t first = lane_of(end - n, l), size = lane_of(each, l);
      w.h = int((u - first) / size);
      w.at = first + uint32_t(w.h) * size;
      w.part = 0;
      return true;
    }
    from = lane_of(end, 63);
  }
  return false;
}

template <int D>
__global__ __launch_bounds__(AT_NT, D <= 128 ? 2 : 1) void kv_split_kernel(Attend a) {
  using S = Shape<D>;
  __shared__ __align__(16) typename S::Lds lds;
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), c = lane & 15, g = lane >> 4;
  const uint32_t wg = blockIdx.x;
  Split sp;
  Walk w;
  bool over;
  const bool some = find_segment(a, sp, w, over);
  if (__builtin_expect(over && !a.blocks, 0)) clear_rows(a, int(wg), int(gridDim.x));  // (else the join's to do)
  if (!some) return;
  Part pt = part_of(sp, w, wg * sp.unit, wg);

  const int mask = a.c.page - 1, sh = a.page_shift;
  uint4 kr[4][S::KL];
  uint32_t vr[S::DT][4];
  bf16x8 qf[2 * S::KL];
  int ksb, vsb;
  int pos, my_row, my_hq;     // this lane's row (the last one where there are fewer)
  int pos_lo, pos_hi, nrows;  // of all rows
  int i, pk, pv, pk1, pv1;
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
  const auto begin = [&] {  // a part: its rows, and its first loads on their way
    nrows = (w.q.r1 - w.q.r0) * a.group;
    i = pt.i0 + wave;
    if (i < pt.i1) lookup(token(i), pk, pv);
    const int ri = min(c, nrows - 1);
    my_row = w.q.r0 + ri / a.group, my_hq = w.h * a.group + ri % a.group;
    pos = w.q.first + ri / a.group;
    pos_lo = w.q.first;
    pos_hi = w.q.first + (w.q.r1 - w.q.r0) - 1;
    const bf16* x = a.q + size_t(my_row) * a.ldq + size_t(my_hq) * D + 16 * g;
#pragma unroll
    for (int m = 0; m < S::KL; ++m) {
      qf[2 * m] = bf16x8_of(*reinterpret_cast<const uint4*>(x + 64 * m));
      qf[2 * m + 1] = bf16x8_of(*reinterpret_cast<const uint4*>(x + 64 * m + 8));
    }
    if (i < pt.i1) {
      load_k(token(i), pk);
      load_v(token(i), pv);
      if (i + AT_WAVES < pt.i1) lookup(token(i + AT_WAVES), pk1, pv1);
    }
  };

  begin();
  for (bool again = true; again;) {
    v4f o[S::DT];
    float mx = -INFINITY, l = 0.0f;
#pragma unroll
    for (int d = 0; d < S::DT; ++d) o[d] = v4f{0, 0, 0, 0};
    for (; i < pt.i1; i += AT_WAVES) {
      const int t0 = token(i);
      const bool more = i + AT_WAVES < pt.i1;
      const int tn = token(more ? i + AT_WAVES : i);
      const int pvt = pv;
      few_tile<D>(a, kr, vr, qf, ksb, vsb, pvt, t0, FewRow{pos, pos_lo, pos_hi, w.q.len}, g, o, mx, l, [&] {
        if (more) {
          pk = pk1, pv = pv1;
          load_k(tn, pk);
          if (i + 2 * AT_WAVES < pt.i1) lookup(token(i + 2 * AT_WAVES), pk1, pv1);
        }
      });
      if (more) load_v(tn, pv);
    }

    // the part is summed: the next one's loads go out, then the waves' sums of this one are joined, four channels of a row
    // a thread
    const Part done = pt;
    const uint32_t w0 = wg - uint32_t(done.index);
    const int r0 = w.q.r0, h = w.h, rows = nrows;
    again = next_segment(a, sp, w, wg);
    if (again) {
      pt = part_of(sp, w, w.at, wg);
      begin();
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    pipe::lds_barrier();  // the last part's use of the LDS
#pragma unroll
    for (int d = 0; d < S::DT; ++d) lds.o[wave * S::QUADS + d * 64 + lane] = o[d];
    if (g == 0) lds.ml[wave][c] = make_float2(mx, l);
    pipe::lds_barrier();
#pragma unroll
    for (int e = 0; e < S::QUADS; e += AT_NT) {
      const int at = e + tid, r = at & 15, d = at / 64 * 16 + (at >> 4 & 3) * 4;
      if (r >= rows) continue;
      float2 ml[AT_WAVES];  // of the waves: maximum and sum
      float m = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int k = 0; k < AT_WAVES; ++k) {
        ml[k] = lds.ml[k][r];
        m = fmaxf(m, ml[k].x);
      }
      const float ref = m == -INFINITY ? 0.0f : m;
      v4f acc{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < AT_WAVES; ++k) {
        const float f = __builtin_amdgcn_exp2f(ml[k].x - ref);
        sum += f * ml[k].y;
        acc += f * lds.o[k * S::QUADS + at];
      }
      if (done.parts == 1) {
        store_out<D>(a, r0 + r / a.group, h * a.group + r % a.group, d, acc, sum, m, d == 0);
      } else {
        const int slot = int(wg * 2 + (done.index == 0 ? 1 : 0)) * FEW + r;
        put4(sums_of(a.po), slot * D + d, acc);
        if (d == 0) put2(sums_of(a.pml), slot * 2, m, sum);
      }
    }
    if (done.parts == 1) continue;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's sums have left
    __syncthreads();
    if (tid == 0)
      last = __hip_atomic_fetch_add(&a.counters[w0], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
             uint32_t(done.parts - 1);
    __syncthreads();
    if (!last) continue;
    if (tid == 0)  // as it was found
      __hip_atomic_store(&a.counters[w0], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // The parts are dealt to `groups` of threads, four channels of a row a thread, and the groups joined in LDS. What takes
    // time are the rounds of reads, about a microsecond each: as many in flight as the registers hold, but not ten where
    // there are two (sixteen layers of one token over 4097: 160 us; by a group of all threads, eight at a time, 183).
    const int items = rows * (D / 4), groups = min(max(AT_NT / items, 1), AT_WAVES), gi = tid / items;
    for (int it = gi < groups ? tid - gi * items : items; it < items; it += AT_NT) {
      const int r = it / (D / 4), d = it % (D / 4) * 4;
      float m = -INFINITY, sum = 0.0f;
      v4f acc{0, 0, 0, 0};
      const auto add = [&]<int N>(int k0) {  // parts k0, k0 + groups, ... (N of them)
        v4f y[N];
        float2 x[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int p = min(k0 + k * groups, done.parts - 1);
          const int at = (int(w0 + uint32_t(p)) * 2 + (p == 0 ? 1 : 0)) * FEW + r;
          x[k] = get2(sums_of(a.pml), at * 2);
          y[k] = get4(sums_of(a.po), at * D + d);
        }
        float m1 = m;
#pragma unroll
        for (int k = 0; k < N; ++k) m1 = fmaxf(m1, x[k].x);
        const float ref = m1 == -INFINITY ? 0.0f : m1, al = __builtin_amdgcn_exp2f(m - ref);
        m = m1;
        acc *= al;
        sum *= al;
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (k0 + k * groups < done.parts) {
            const float f = __builtin_amdgcn_exp2f(x[k].x - ref);
            sum += f * x[k].y;
            acc += f * y[k];
          }
      };
      if (done.parts <= 2 * groups) add.template operator()<2>(gi % groups);
      else
        for (int k0 = gi % groups; k0 < done.parts; k0 += FLIGHT * groups) add.template operator()<FLIGHT>(k0);
      if (groups == 1) {
        store_out<D>(a, r0 + r / a.group, h * a.group + r % a.group, d, acc, sum, m, d == 0);
      } else {
        lds.o[tid] = acc;  // (the waves' sums were read before the counter was)
        lds.group_ml[tid] = make_float2(m, sum);
      }
    }
    if (groups == 1) continue;
    pipe::lds_barrier();
    if (tid < items) {
      float m = -INFINITY, sum = 0.0f;
      v4f acc{0, 0, 0, 0};
      for (int k = 0; k < groups; ++k) m = fmaxf(m, lds.group_ml[k * items + tid].x);
      const float ref = m == -INFINITY ? 0.0f : m;
      for (int k = 0; k < groups; ++k) {
        const float2 x = lds.group_ml[k * items + tid];
        const float f = __builtin_amdgcn_exp2f(x.x - ref);
        sum += f * x.y;
        acc += f * lds.o[k * items + tid];
      }
      const int r = tid / (D / 4), d = tid % (D / 4) * 4;
      store_out<D>(a, r0 + r / a.group, h * a.group + r % a.group, d, acc, sum, m, d == 0);
    }
  }
}

__device__ __forceinline__ bool find_block(const Attend& a, BlockPart& p, bool& over) {
  constexpr uint32_t NONE = 1u << 30;
  const int lane = threadIdx.x & 63;
  const uint32_t heads = uint32_t(a.c.heads);
  Seq q{0, 0, 0, 0};
  uint32_t blocks = 0, most = 0, all = 0;  // of this lane's sequence, tiles of its last block; of all, times the heads
  int rows = 0;
  const auto look = [&](int b) {
    blocks = most = 0;
    rows = 0;
    if (b < a.st.B) {
      q = seq_of(a.st, b);
      rows = q.r1 - q.r0;
      if (rows * a.group > a.few && rows <= a.st.max_new) {
        blocks = uint32_t(row_groups(rows * a.group, PR_ROWS));
        most = uint32_t(block_tiles(a, q, int(blocks - 1) * PR_ROWS).count);
      }
    }
  };
  uint32_t tiles = 0;  // (a block's taken as the last one's; as long as the blocks are few)
  over = false;
  for (int b0 = 0; b0 < a.st.B; b0 += 64) {
    look(b0 + lane);
    over |= __ballot(rows > a.st.max_new) != 0;
    all += lane_of(wave_scan(blocks), 63) * heads;
    if (all < a.target) tiles += lane_of(wave_scan(blocks * most), 63) * heads;
  }
  // A part has 4 tiles at least, and where blocks see many so many that they (1.5 us each) balance the join (0.3 us a part):
  // 80 rows of 128 over 131,000 tokens take 63 us a call, in 512 parts of four tiles 164.
  const uint32_t least = max(4u, root(0.2f, tiles, all));
  uint32_t share = NONE;
  if (all < a.target && a.st.B <= 64) share = smallest_share(blocks * heads, most, tiles, all, a.target, least);
  else if (all < a.target) share = max((tiles + a.target - all - 1) / (a.target - all), least);  // one that is large enough
  uint32_t from = 0;
  for (int b0 = 0; b0 < a.st.B; b0 += 64) {
    if (a.st.B > 64) look(b0 + lane);
    const uint32_t parts = parts_of(most, share), n = blocks * parts * heads, end = from + wave_scan(n);
    const uint64_t hit = __ballot(blockIdx.x < end);
    if (hit) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      p.b = b0 + l;
      p.q = Seq{int(lane_of(q.r0, l)), int(lane_of(q.r1, l)), int(lane_of(q.len, l)), int(lane_of(q.first, l))};
      const uint32_t in = blockIdx.x - lane_of(end - n, l), np = lane_of(parts, l);
      p.h = int(in % heads);
      p.index = int(in / heads % np);
      const int block = int(lane_of(blocks, l) - 1 - in / heads / np);
      p.row0 = block * PR_ROWS;
      const Tiles t = block_tiles(a, p.q, p.row0);
      p.t = Tiles{uniform(t.sink_tiles), uniform(t.skip), uniform(t.count)};
      p.parts = int(min(parts_of(uint32_t(p.t.count), share), np));  // (under a window the last block may see fewer tiles)
      if (p.index >= p.parts) return false;  // a block that sees less than the sequence's last
      const int each = p.t.count / p.parts, more = p.t.count % p.parts;
      p.i0 = p.index * each + min(p.index, more);
      p.i1 = p.i0 + each + (p.index < more ? 1 : 0);
      return true;
    }
    from = lane_of(end, 63);
  }
  return false;
}

struct FindBlock {
  using Call = Attend;
  template <int D>
  static __device__ __forceinline__ bool find(const Attend& a, BlockPart& bp, int&) {
    bool over;
    const bool some = find_block(a, bp, over);
    if (threadIdx.x == 0 && blockIdx.x < a.target)
      a.blocks[blockIdx.x] = some && bp.index == 0
                                 ? Block{bp.parts, int(a.c.heads), bp.row0, min(PR_ROWS, (bp.q.r1 - bp.q.r0) * a.group - bp.row0),
                                         bp.q.r0, bp.h, over, 0}
                                 : Block{0, 0, 0, 0, 0, 0, over, 0};
    return some;
  }
};

// The parts of the tiled kernel's blocks, in order. A thread per row and four channels, JOIN parts at a time: few registers and
// many threads rather than many parts in flight (eight parts of two quads a thread: 5% more for a step of 256 blocks in two
// parts each, 1% for 64 blocks in 7 or 8 parts; 5% less for four blocks in 16). 64 blocks of 40 rows: 7 us; by the last
// workgroup of each block, as in the split kernel, 14.
constexpr int JOIN = 4;
template <int D>
__global__ __launch_bounds__(AT_NT) void kv_join_kernel(Attend a) {
  constexpr int WAVE_QUADS = D / 32 * 256;  // of 32 rows
  const Block k = a.blocks[blockIdx.x];
  if (__builtin_expect(k.over, 0)) clear_rows(a, int(blockIdx.x * gridDim.y + blockIdx.y), int(gridDim.x * gridDim.y));
  if (k.parts <= 1) return;
  const int at = blockIdx.y * AT_NT + threadIdx.x, r = at / WAVE_QUADS * 32 + (at & 31), rr = k.row0 + r;
  if (r >= k.rows) return;
  float m = -INFINITY, sum = 0.0f;
  v4f acc{0, 0, 0, 0};
  for (int p0 = 0; p0 < k.parts; p0 += JOIN) {
    v4f y[JOIN];
    float2 x[JOIN];
#pragma unroll
    for (int p = 0; p < JOIN; ++p) {
      x[p] = make_float2(-INFINITY, 0.0f), y[p] = v4f{0, 0, 0, 0};
      if (p0 + p >= k.parts) continue;
      const size_t slot = size_t(blockIdx.x) + size_t(p0 + p) * k.step;
      x[p] = *reinterpret_cast<const float2*>(a.pml + (slot * PR_ROWS + r) * 2);
      y[p] = *reinterpret_cast<const v4f*>(a.po + (slot * (PR_ROWS * D / 4) + at) * 4);
    }
    float m1 = m;
#pragma unroll
    for (int p = 0; p < JOIN; ++p) m1 = fmaxf(m1, x[p].x);
    const float ref = m1 == -INFINITY ? 0.0f : m1, al = __builtin_amdgcn_exp2f(m - ref);
    m = m1;
    acc *= al;
    sum *= al;
#pragma unroll
    for (int p = 0; p < JOIN; ++p) {
      const float f = __builtin_amdgcn_exp2f(x[p].x - ref);
      sum += f * x[p].y;
      acc += f * y[p];
    }
  }
  const int quad = at / 64 % (D / 8), d = quad / 4 * 32 + quad % 4 * 8 + (at & 32) / 8;
  store_out<D>(a, k.r0 + rr / a.group, k.h * a.group + rr % a.group, d, acc, sum, m, d == 0);
}

int most_rows(int rows, int max_new, int group) {
  return int(std::min<int64_t>(int64_t(std::min(rows, max_new)) * group, INT32_MAX));
}
// Which kernels a step takes: up to FEW rows a sequence (of a key / value head) the split kernel (64 sequences of one token
// 105 us, by the tiled one 161), past that the tiled one, and where the step's sequences may be of both kinds each its own
// (eight tokens and a chunk of 1000: 111 us, all by the tiled one 128). The second way costs launches, though, 8 us or so: not
// taken for a single sequence, where every sequence of the step is past FEW by its group alone, and, if none has more rows
// than one block, where they are past FEW on average (16 x 5 draft tokens, four layers: 129 us, with the launches 139) or few
// (31 tokens and a chunk of 30, 8 heads: 51 us and 62; 63 tokens and a chunk of 30: 113 and 90).
Way way_of(int rows, int max_new, int B, int group, int heads) {
  const int most = most_rows(rows, max_new, group);
  if (most <= FEW) return {FEW, true, false};
  if (B == 1 || group > FEW) return {0, false, true};
  if (most <= PR_ROWS && (int64_t(rows) * group > int64_t(FEW) * B || int64_t(B) * heads <= 256)) return {0, false, true};
  return {FEW, true, true};
}
// Partial sums of one launch: 2 target of FEW rows, or target of a row block.
size_t sum_rows(const Way& way, int dim) {
  return size_t(target_of(dim)) * (way.tiled ? PR_ROWS : 2 * FEW);
}

}  // namespace

size_t kv_attend_workspace(int rows, int max_new, int B, int Hq, int heads, int dim) {
  if (rows < 0 || max_new < 0 || B < 0 || heads < 1 || Hq < heads || dim < 1) return 0;
  return kHeadBytes + sum_rows(way_of(rows, max_new, B, Hq / heads, heads), dim) * (size_t(dim) + 2) * sizeof(float);
}

namespace kv {

bool check_attend(const char* who, const bf16* q, int ldq, const KvStep& s, const KvCache& c, int Hq, float scale, int sinks,
                  const bf16* out, int ldo, const void* ws, size_t ws_bytes, size_t need) {
  const auto fail = [&](const std::string& what) { throw std::runtime_error(std::string(who) + ": " + what); };
  check_cache(who, c);
  check_step(who, s);
  if (Hq < 1 || Hq % c.heads || Hq > 65535) fail("Hq must be a multiple of heads, up to 65535");
  if (sinks < 0) fail("sinks < 0");
  if (!std::isfinite(scale)) fail("scale is not finite");
  if (s.B == 0 || s.rows == 0 || s.max_new == 0) return false;
  if (!q || !out) fail("null operand");
  const int64_t width = int64_t(Hq) * c.dim;
  if (ldq < width || ldo < width || ldq % 8 || ldo % 8) fail("ldq / ldo >= Hq * dim, % 8");
  if (!aligned16(q) || !aligned16(out)) fail("rows not 16-byte aligned");
  if (int64_t(s.rows) * Hq > INT32_MAX) fail("rows * Hq past 31 bits");
  if (!ws) fail("null workspace");
  if (!aligned16(ws)) fail("workspace not 16-byte aligned");
  if (ws_bytes < need) fail("workspace of " + std::to_string(ws_bytes) + " bytes, " + std::to_string(need) + " needed");
  return true;
}
Attend attend_of(const bf16* q, int ldq, const KvStep& s, const KvCache& c, int Hq, float scale, int window, int sinks, bf16* out,
                 int ldo, float* lse, const Way& way, void* ws) {
  Attend a{};
  a.q = q, a.out = out, a.lse = lse, a.st = s, a.c = c, a.ldq = ldq, a.ldo = ldo, a.group = Hq / c.heads;
  a.window = window, a.sinks = sinks, a.scale2 = scale * LOG2E, a.few = way.few, a.target = unsigned(target_of(c.dim));
  while (1 << a.page_shift < c.page) ++a.page_shift;
  a.counters = static_cast<uint32_t*>(ws);
  if (way.tiled) a.blocks = reinterpret_cast<Block*>(a.counters + 512);
  return a;
}
void launch_tiled(const Attend& a, int64_t blocks, hipStream_t st) {
  const unsigned grid = std::max(unsigned(blocks), a.target);
  by_dim(a.c.dim, [&]<int D>() { kv_tiled_kernel<D, FindBlock><<<grid, AT_NT, 0, st>>>(a); });
  const dim3 join(a.target, unsigned(PR_ROWS * a.c.dim / 4 / AT_NT));
  by_dim(a.c.dim, [&]<int D>() { kv_join_kernel<D><<<join, AT_NT, 0, st>>>(a); });
}

}  // namespace kv

void kv_attend(const bf16* q, int ldq, const KvStep& s, const KvCache& c, int Hq, float scale, int window, int sinks,
               bf16* out, int ldo, float* lse, void* ws, size_t ws_bytes, hipStream_t st) {
  const size_t need = kv_attend_workspace(s.rows, s.max_new, s.B, Hq, c.heads, c.dim);
  if (!check_attend("kv_attend", q, ldq, s, c, Hq, scale, sinks, out, ldo, ws, ws_bytes, need)) return;
  const Way way = way_of(s.rows, s.max_new, s.B, Hq / c.heads, c.heads);
  Attend a = attend_of(q, ldq, s, c, Hq, scale, window, sinks, out, ldo, lse, way, ws);
  a.po = reinterpret_cast<float*>(static_cast<char*>(ws) + kHeadBytes);
  a.pml = a.po + sum_rows(way, c.dim) * c.dim;
  const int64_t segs = int64_t(s.B) * c.heads;
  const int64_t tiles = std::max<int64_t>(cdiv(size_t(s.max_blocks) * c.page, TILE), 1);
  const int64_t blocks = (cdiv(size_t(s.rows) * a.group, PR_ROWS) + int64_t(s.B)) * c.heads;  // at most
  if (segs * 8 > INT32_MAX || std::max(segs, std::min<int64_t>(blocks, a.target)) * (tiles + START) > INT32_MAX ||
      blocks > INT32_MAX)
    throw std::runtime_error("kv_attend: rows times blocks past 31 bits");
  if (way.tiled) launch_tiled(a, blocks, st);
  if (way.split) {
    const unsigned grid = unsigned(std::min<int64_t>(segs * cdiv(tiles + START, AT_WAVES), a.target));
    by_dim(c.dim, [&]<int D>() { kv_split_kernel<D><<<grid, AT_NT, 0, st>>>(a); });
  }
}

}  // namespace unholy::kernels
