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
        segs = uint32_t(segments_of<false>(a, w.q));
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
  __shared__ __align__(16) typename Shape<D>::Lds lds;
  __shared__ int last;
  Split sp;
  Walk w;
  bool over;
  const bool some = find_segment(a, sp, w, over);
  if (__builtin_expect(over && !a.blocks, 0)) clear_rows(a, int(blockIdx.x), int(gridDim.x));  // (else the join's to do)
  if (some) split_segments<D>(a, lds, last, sp, w, blockIdx.x);
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

template <int D>
__global__ __launch_bounds__(AT_NT, D == 64 ? 3 : D == 128 ? 2 : 1) void kv_tiled_kernel(Attend a) {
  __shared__ __align__(1024) typename Tiled<D>::Lds lds;
  BlockPart bp;
  bool over;
  const bool some = find_block(a, bp, over);
  if (threadIdx.x == 0 && blockIdx.x < a.target)
    a.blocks[blockIdx.x] = some && bp.index == 0
                               ? Block{bp.parts, int(a.c.heads), bp.row0, min(PR_ROWS, (bp.q.r1 - bp.q.r0) * a.group - bp.row0),
                                       bp.q.r0, bp.h, over, 0}
                               : Block{0, 0, 0, 0, 0, 0, over, 0};
  if (some) tiled_part<D, false>(a, lds, bp, 0, blockIdx.x);
}

// The parts of the tiled kernel's blocks, in order. A thread per row and four channels, JOIN parts at a time: few registers and
// many threads rather than many parts in flight (eight parts of two quads a thread: 5% more for a step of 256 blocks in two
// parts each, 1% for 64 blocks in 7 or 8 parts; 5% less for four blocks in 16). 64 blocks of 40 rows: 7 us; by the last workgroup
// of each block, as in the split kernel, 14.
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
  by_dim(a.c.dim, [&]<int D>() { kv_tiled_kernel<D><<<grid, AT_NT, 0, st>>>(a); });
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
