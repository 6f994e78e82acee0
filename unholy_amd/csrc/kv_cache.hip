// The 8-bit paged key / value cache: quantizing a step's tokens into it, and its pages' bookkeeping
// (include/unholy/kernels/kv_cache.hpp has the layout and the contracts).
#include <algorithm>

#include "kv_internal.hpp"
#include "numerics.hpp"

namespace unholy::kernels {

using namespace uh;
using namespace kv;

namespace {

// ---- append -----------------------------------------------------------------------------------------------------------
// A workgroup per (sequence, block that its new tokens reach, key / value head, keys or values): the block's new rows are
// read once into registers, their amax over the workgroup gives the scale, and the codes go straight to the cache. Keys: a
// thread takes 8 channels of a token, lanes along the rows. Values, whose tokens lie a byte apart: 8 channels of the four
// tokens of a dword, lanes along the tokens, so that a wave reads 64-byte pieces of 16 rows and writes whole 64-byte rows of
// channels (12,002 tokens of 8 heads of 128: 16.8 us, 4.4 TB/s; through an LDS tile of bytes 25.8). A step of few tokens is
// bound by its three dependent loads (lengths, page, scale): 6.3 us a layer, while no block's scale grows. Where one does, its
// earlier codes are read and written by the byte, one after the other, and the launch waits for that: 43 us a layer for 64
// tokens in full use, of whose blocks a sixth grow (prompts, which write whole blocks, lose some 5 us).
// A power-of-two scale, as everywhere in this library, so that a block whose scale grows keeps its codes: rne(c 2^-g) is
// exact unless the result is subnormal, and then off by at most 2^-10 of the new scale's unit. (A scale with a mantissa
// would round every code of the block again, each time that it grows.)
constexpr int kScaleTop = 246;  // 2^119: 448 2^119 is finite in bf16 and fp32

__device__ __forceinline__ uint8_t kv_code(float v, float inv) {
  if (v != v) return 0x7f;
  return e4m3_hw(clamp448(v * inv));
}
// A code under a scale 2^g times larger (f = 2^-g).
__device__ __forceinline__ uint8_t kv_move(uint8_t c, float f) {
  return (c & 0x7f) == 0x7f ? c : e4m3_hw(e4m3_to_f32(c) * f);
}
__device__ __forceinline__ float half_of(const uint4& v, int j) {  // value j of eight bf16
  const uint32_t w = j < 4 ? (j < 2 ? v.x : v.y) : (j < 6 ? v.z : v.w);
  return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
}
// Codes of four values; odd: there may be NaN among them.
__device__ __forceinline__ uint32_t kv_codes4(float a, float b, float c, float d, float inv, bool odd) {
  if (odd)
    return uint32_t(kv_code(a, inv)) | uint32_t(kv_code(b, inv)) << 8 | uint32_t(kv_code(c, inv)) << 16 |
           uint32_t(kv_code(d, inv)) << 24;
  return e4m3x4(clamp448(a * inv), clamp448(b * inv), clamp448(c * inv), clamp448(d * inv));
}

// Pieces of 8 channels x 4 tokens that a thread holds; a workgroup of one wave takes steps of few tokens.
constexpr int pieces_of(int dim, int page, int nt) { return nt == 64 ? 2 : std::max(1, page * dim / 32 / nt); }

template <int D, int PAGE, int NT>
__global__ __launch_bounds__(NT) void kv_append_kernel(const bf16* __restrict__ kx, int ldk, const bf16* __restrict__ vx,
                                                       int ldv, KvStep st, KvCache c, int nblk) {
  constexpr int CH = D / 8, Q = pieces_of(D, PAGE, NT);
  __shared__ float red[NT / 64];
  const int b = blockIdx.x / nblk, h = blockIdx.y, tid = threadIdx.x;
  const bool values = blockIdx.z != 0;
  const Seq q = seq_of(st, b);
  const int blk = max(q.first, 0) / PAGE + int(blockIdx.x % nblk), lo = blk * PAGE;
  if (lo >= q.len || blk >= st.max_blocks) return;
  const int p0 = max(max(q.first, lo), 0), s0 = p0 - lo, n = min(lo + PAGE, q.len) - p0, end = s0 + n;  // new: [s0, end)
  if (n <= 0 || too_many(st, q)) return;
  const int page = st.table[size_t(b) * st.max_blocks + blk];
  const int ld = values ? ldv : ldk;
  const bf16* x = (values ? vx : kx) + size_t(q.r0 + (p0 - q.first)) * ld + size_t(h) * D;

  uint4 raw[4 * Q];
  const int q0 = s0 / 4, nq = (end - 1) / 4 - q0 + 1;  // dwords of tokens
  const auto piece = [&](int i, int& u, int& d) {      // values: this thread's i-th dword of tokens and first channel
    const int at = tid + i * NT;
    u = q0 + at % nq;
    d = at / nq * 8;
    return d < D;
  };
#pragma unroll
  for (int i = 0; i < 4 * Q; ++i) raw[i] = make_uint4(0, 0, 0, 0);
  if (values) {
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      int u, d;
      if (!piece(i, u, d)) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = 4 * u + e - s0;
        if (t >= 0 && t < n) raw[4 * i + e] = *reinterpret_cast<const uint4*>(x + size_t(t) * ld + d);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4 * Q; ++i) {
      const int at = tid + i * NT;
      if (at < n * CH) raw[i] = *reinterpret_cast<const uint4*>(x + size_t(at / CH) * ld + at % CH * 8);
    }
  }
  if (page < 0 || page >= c.pages) return;
  const size_t ph = size_t(page) * c.heads + h;
  uint8_t* codes = (values ? c.v : c.k) + ph * (size_t(D) * PAGE);
  uint8_t* scale = (values ? c.vs : c.ks) + ph;
  const int old = s0 ? *scale : 0;

  float am = 0.0f;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4 * Q; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = fabsf(half_of(raw[i], j));
      const bool fine = a < INFINITY;
      am = fine ? fmaxf(am, a) : am;
      odd |= !fine;
    }
  am = wave_max(am);
  if constexpr (NT > 64) {
    if ((tid & 63) == 0) red[tid >> 6] = am;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) am = fmaxf(am, red[i]);
  }
  const int se = min(max(int(exact_fp8_scale(fmaxf(am, 1e-4f))), old), kScaleTop);
  const float inv = __uint_as_float(uint32_t(254 - se) << 23);
  if (values) {
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      int u, d;
      if (!piece(i, u, d)) continue;
      const bool whole = 4 * u >= s0 && 4 * u + 4 <= end;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t w = kv_codes4(half_of(raw[4 * i], j), half_of(raw[4 * i + 1], j), half_of(raw[4 * i + 2], j),
                                     half_of(raw[4 * i + 3], j), inv, odd);
        uint8_t* y = codes + size_t(d + j) * PAGE + 4 * u;
        if (whole) {
          *reinterpret_cast<uint32_t*>(y) = w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * u + e >= s0 && 4 * u + e < end) y[e] = uint8_t(w >> (8 * e));
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4 * Q; ++i) {
      const int at = tid + i * NT;
      if (at >= n * CH) continue;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = half_of(raw[i], j);
      *reinterpret_cast<uint2*>(codes + size_t(s0) * D + size_t(at) * 8) =
          make_uint2(kv_codes4(v[0], v[1], v[2], v[3], inv, odd), kv_codes4(v[4], v[5], v[6], v[7], inv, odd));
    }
  }
  if (s0 && se > old) {  // the codes of the tokens before, under the new scale
    const float f = ldexpf(1.0f, old - se);
    const int per = values ? (s0 + 3) / 4 : s0 * D / 4, rows = values ? D : 1, most = values ? s0 : s0 * D;
    for (int i = tid; i < rows * per; i += NT) {
      uint8_t* y = codes + size_t(i / per) * PAGE + i % per * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i % per * 4 + e < most) y[e] = kv_move(y[e], f);
    }
  }
  if (tid == 0 && se != old) *scale = uint8_t(se);
}

// ---- pages ------------------------------------------------------------------------------------------------------------
constexpr int PL_NT = 1024;

constexpr int kMany = 1 << 29;  // sums of pages stop here, past any pool
__device__ __forceinline__ int add_pages(int a, int b) { return min(a + b, kMany); }

// Exclusive prefix of v (0 .. kMany) over the workgroup's threads; total is their sum (wsum: PL_NT / 64 ints of LDS).
__device__ __forceinline__ int block_scan(int v, int* wsum, int& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x = add_pages(x, y);
  }
  int before = __shfl_up(x, 1, 64);
  if (lane == 0) before = 0;
  __syncthreads();  // the last call's reads of wsum
  if (lane == 63) wsum[w] = x;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int i = 0; i < PL_NT / 64; ++i) {
    before = add_pages(before, i < w ? wsum[i] : 0);
    total = add_pages(total, wsum[i]);
  }
  return before;
}

// Workspace of the page calls: a header, the copies to make and int lists.
struct PagesWs {
  int* n;         // [0] copies, [1] the pages below which a compaction leaves all (live)
  int2* pairs;    // {from, to}, up to max(B, pages)
  int *a, *b;     // B + pages each
  size_t bytes;
};
inline PagesWs carve_pages(void* ws, int B, int pages) {
  PagesWs w;
  char* p = static_cast<char*>(ws);
  w.n = reinterpret_cast<int*>(p);
  w.pairs = reinterpret_cast<int2*>(p + 64);
  w.a = reinterpret_cast<int*>(w.pairs + size_t(std::max(B, pages)));
  w.b = w.a + size_t(B) + pages;
  w.bytes = 64 + sizeof(int2) * size_t(std::max(B, pages)) + 2 * sizeof(int) * (size_t(B) + pages);
  return w;
}

// One workgroup: the sequences' needs (prefix over the slots), the free pages in order as far as they are needed, then the
// tables. a[b]: pages needed before sequence b; b[b]: its shared last page, or -1; a[B + i]: the i-th free page.
__global__ __launch_bounds__(PL_NT) void kv_reserve_kernel(KvSeqs s, const int32_t* __restrict__ grow, int32_t* refs,
                                                           int pages, int page, int32_t* __restrict__ ok, PagesWs w) {
  __shared__ int wsum[PL_NT / 64];
  __shared__ int copies;
  const int tid = threadIdx.x;
  if (tid == 0) copies = 0;
  int total = 0;
  for (int b0 = 0; b0 < s.B; b0 += PL_NT) {
    const int b = b0 + tid;
    int need = 0, src = -1;
    if (b < s.B) {
      const int64_t len = max(s.lens[b], 0), g = max(grow[b], 0);
      const int64_t held = (len + page - 1) / page, want = (len + g + page - 1) / page;
      if (want <= s.max_blocks) {
        if (g > 0 && len % page) {
          const int tail = page_of(s.table, s.max_blocks, pages, b, int(held) - 1);
          if (tail >= 0 && refs[tail] > 1) src = tail;
        }
        need = int(want - held) + (src >= 0);
      }
    }
    int sum;
    const int before = block_scan(need, wsum, sum);
    if (b < s.B) {
      w.a[b] = add_pages(total, before);
      w.b[b] = src;
    }
    total = add_pages(total, sum);
  }
  int found = 0;
  for (int p0 = 0; p0 < pages && found < total; p0 += PL_NT * 4) {
    int is[4], mine = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = p0 + tid * 4 + j;
      is[j] = p < pages && refs[p] == 0;
      mine += is[j];
    }
    int sum, at = found + block_scan(mine, wsum, sum);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (is[j]) w.a[s.B + at++] = p0 + tid * 4 + j;
    found += sum;
  }
  __syncthreads();  // every decision above is made on refs as they were
  const int lane = tid & 63;
  for (int b0 = tid & ~63; b0 < s.B; b0 += PL_NT) {  // a sequence a thread, and where it gets many pages its wave
    const int b = b0 + lane;
    int held = 0, count = 0, first = 0;
    if (b < s.B) {
      const int64_t len = max(s.lens[b], 0), g = max(grow[b], 0);
      const int64_t held64 = (len + page - 1) / page, want64 = (len + g + page - 1) / page;
      const int src = w.b[b], begin = w.a[b], extra = src >= 0;
      const bool fits = want64 <= s.max_blocks;
      const int more = fits ? int(want64 - held64) : 0;
      const bool served = fits && (more + extra == 0 || begin + more + extra <= found);
      ok[b] = served;
      if (served) {
        held = int(held64);
        count = more;
        first = begin + extra;
        if (g > 0) s.lens[b] = int(len + g);
        if (extra) {
          const int to = w.a[s.B + begin];
          s.table[size_t(b) * s.max_blocks + held - 1] = to;
          refs[to] = 1;
          atomicSub(&refs[src], 1);
          w.pairs[atomicAdd(&copies, 1)] = make_int2(src, to);  // in any order: they touch different pages
        }
      }
    }
    for (uint64_t some = __ballot(count > 0); some; some &= some - 1) {
      const int l = __ffsll((unsigned long long)some) - 1;
      const int c = __builtin_amdgcn_readlane(count, l), h = __builtin_amdgcn_readlane(held, l);
      const int* list = w.a + s.B + __builtin_amdgcn_readlane(first, l);
      for (int j = lane; j < c; j += 64) {
        const int p = list[j];
        s.table[size_t(b0 + l) * s.max_blocks + h + j] = p;
        refs[p] = 1;
      }
    }
  }
  __syncthreads();
  if (tid == 0) w.n[0] = copies;
}

// The copies of w.pairs in every layer, 16 KiB pieces of a page's keys or values over the grid; a page's scales go with its
// first piece. One read and one write of the data: bound by HBM (1.04 GB in all: 209 us, 4.9 TB/s, as fast as a large copy).
constexpr int CP_BYTES = 16384;
__global__ __launch_bounds__(256) void kv_copy_kernel(KvCache c, int layers, PagesWs w, const int32_t* table,
                                                      int32_t* table_out, size_t entries) {
  const int n = w.n[0];
  const size_t bytes = size_t(c.heads) * c.page * c.dim;
  const int per = int((bytes + CP_BYTES - 1) / CP_BYTES);
  const size_t items = size_t(n) * layers * 2 * per;
  for (size_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int part = int(it % per), which = int(it / per & 1);
    const size_t rest = it / per / 2;
    const int layer = int(rest % layers);
    const int2 pair = w.pairs[rest / layers];
    const size_t base = size_t(layer) * c.pages;
    uint8_t* data = which ? c.v : c.k;
    const uint4* src = reinterpret_cast<const uint4*>(data + (base + pair.x) * bytes + size_t(part) * CP_BYTES);
    uint4* dst = reinterpret_cast<uint4*>(data + (base + pair.y) * bytes + size_t(part) * CP_BYTES);
    const int vecs = int(min(bytes - size_t(part) * CP_BYTES, size_t(CP_BYTES)) / 16);
    if (vecs == CP_BYTES / 16) {
      const v4i *from = reinterpret_cast<const v4i*>(src) + threadIdx.x;
      v4i* to = reinterpret_cast<v4i*>(dst) + threadIdx.x;
      const v4i v0 = from[0], v1 = from[256], v2 = from[512], v3 = from[768];
      to[0] = v0, to[256] = v1, to[512] = v2, to[768] = v3;
    } else {
      for (int i = threadIdx.x; i < vecs; i += 256) dst[i] = src[i];
    }
    if (part == 0) {
      uint8_t* sc = which ? c.vs : c.ks;
      for (int h = threadIdx.x; h < c.heads; h += 256)
        sc[(base + pair.y) * c.heads + h] = sc[(base + pair.x) * c.heads + h];
    }
  }
  for (size_t i = blockIdx.x * size_t(256) + threadIdx.x; i < entries; i += size_t(gridDim.x) * 256) {  // a compaction's
    const int t = table[i];
    table_out[i] = t >= 0 && t < c.pages ? w.a[t] : -1;
  }
}

// One workgroup: the number of live pages, then in page order the used ones from there on and the free ones below.
// a[p]: where page p goes; b[i]: the i-th free number.
__global__ __launch_bounds__(PL_NT) void kv_compact_kernel(const int32_t* refs, int32_t* refs_out, int pages,
                                                           int32_t* live_out, PagesWs w) {
  __shared__ int wsum[PL_NT / 64];
  const int tid = threadIdx.x;
  int mine = 0, live;
  for (int p = tid; p < pages; p += PL_NT) mine += refs[p] > 0;
  block_scan(mine, wsum, live);
  int nsrc = 0, ndst = 0;
  for (int p0 = 0; p0 < pages; p0 += PL_NT) {
    const int p = p0 + tid;
    const int r = p < pages ? refs[p] : 0;
    const bool src = p < pages && r > 0 && p >= live, dst = p < live && r <= 0;
    int sum;
    const int at = block_scan(src | dst << 16, wsum, sum);
    if (src) w.pairs[nsrc + (at & 0xffff)].x = p;
    if (dst) w.pairs[ndst + (at >> 16)].y = p;
    if (p < pages) {
      w.a[p] = p;
      if (!src && !dst) refs_out[p] = r > 0 ? r : 0;
    }
    nsrc += sum & 0xffff;
    ndst += sum >> 16;
  }
  __syncthreads();
  for (int i = tid; i < nsrc; i += PL_NT) {  // as many free numbers below live as used ones from there on
    const int2 m = w.pairs[i];
    const int r = refs[m.x];
    w.a[m.x] = m.y;
    refs_out[m.y] = r;
    refs_out[m.x] = 0;
  }
  if (tid == 0) {
    w.n[0] = nsrc;
    if (live_out) *live_out = live;
  }
}

// A wave per slot. The lengths are written by the next launch: every slot decides on what they were.
__global__ __launch_bounds__(64) void kv_fork_kernel(KvSeqs s, const int32_t* __restrict__ from, int32_t* refs, int pages,
                                                     int page, int32_t* __restrict__ done) {
  const int b = blockIdx.x, src = from[b], lane = threadIdx.x;
  const bool doit = s.lens[b] == 0 && src >= 0 && src < s.B && src != b && s.lens[src] > 0;
  if (lane == 0) done[b] = doit;
  if (!doit) return;
  const int held = int(min((int64_t(s.lens[src]) + page - 1) / page, int64_t(s.max_blocks)));
  for (int j = lane; j < held; j += 64) {
    const int p = s.table[size_t(src) * s.max_blocks + j];
    s.table[size_t(b) * s.max_blocks + j] = p;
    if (p >= 0 && p < pages) atomicAdd(&refs[p], 1);
  }
}
__global__ __launch_bounds__(256) void kv_fork_lens_kernel(KvSeqs s, const int32_t* __restrict__ from,
                                                           const int32_t* __restrict__ done) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b < s.B && done[b]) s.lens[b] = s.lens[from[b]];  // (a source has tokens: it is no slot that is written here)
}

__global__ __launch_bounds__(64) void kv_free_kernel(KvSeqs s, const int32_t* __restrict__ keep, int32_t* refs, int pages,
                                                     int page) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const int len = s.lens[b], left = min(max(keep[b], 0), max(len, 0));
  const int64_t have = min((int64_t(max(len, 0)) + page - 1) / page, int64_t(s.max_blocks));
  for (int64_t j = (int64_t(left) + page - 1) / page + lane; j < have; j += 64) {
    int32_t* e = s.table + size_t(b) * s.max_blocks + j;
    const int p = *e;
    if (p >= 0 && p < pages) atomicSub(&refs[p], 1);
    *e = -1;
  }
  if (lane == 0 && left != len) s.lens[b] = left;
}

void check_seqs(const char* who, const KvSeqs& s, const int32_t* more, const int32_t* refs, int pages, int page) {
  const auto fail = [&](const char* what) { throw std::runtime_error(std::string(who) + ": " + what); };
  if (s.B < 0 || s.max_blocks < 0) fail("negative size");
  if (s.max_blocks > (1 << 23)) fail("max_blocks > 2^23");
  if (page != 16 && page != 32 && page != 64 && page != 128) fail("page must be 16, 32, 64 or 128");
  check_pages(who, pages);
  if ((!s.table && s.max_blocks) || !s.lens || !more || !refs) fail("null operand");
}
void check_ws(const char* who, const void* ws, size_t bytes, size_t need) {
  if (!ws) throw std::runtime_error(std::string(who) + ": null workspace");
  if (!aligned16(ws)) throw std::runtime_error(std::string(who) + ": workspace not 16-byte aligned");
  if (bytes < need)
    throw std::runtime_error(std::string(who) + ": workspace of " + std::to_string(bytes) + " bytes, " +
                             std::to_string(need) + " needed");
}

}  // namespace

void kv_append(const bf16* k, int ldk, const bf16* v, int ldv, const KvStep& s, const KvCache& c, hipStream_t st) {
  check_cache("kv_append", c);
  check_step("kv_append", s);
  if (s.B == 0 || s.rows == 0 || s.max_new == 0 || s.max_blocks == 0) return;
  if (!k || !v) throw std::runtime_error("kv_append: null operand");
  if (int64_t(ldk) < int64_t(c.heads) * c.dim || int64_t(ldv) < int64_t(c.heads) * c.dim || ldk % 8 || ldv % 8)
    throw std::runtime_error("kv_append: ldk / ldv >= heads * dim, % 8");
  if (!aligned16(k) || !aligned16(v)) throw std::runtime_error("kv_append: rows not 16-byte aligned");
  const int64_t most = std::min(s.max_new, s.rows);  // (up to 2^31 - 1)
  const int nblk = int(std::min<int64_t>((most - 1 + c.page - 1) / c.page + 1, s.max_blocks));  // that they can reach
  if (int64_t(s.B) * nblk > INT32_MAX) throw std::runtime_error("kv_append: B * blocks past 31 bits");
  const dim3 grid(unsigned(s.B) * unsigned(nblk), unsigned(c.heads), 2);
  // A wave holds 128 pieces of 8 channels x 4 tokens: enough for `most` tokens, wherever they begin, or a workgroup of four
  // (64 sequences of one token in eight layers: 50 us by waves, 59 by workgroups)
  const bool few = ((most + 2) / 4 + 1) * (c.dim / 8) <= 64 * pieces_of(c.dim, c.page, 64);
  const auto go = [&]<int D, int PAGE>() {
    if (few) kv_append_kernel<D, PAGE, 64><<<grid, 64, 0, st>>>(k, ldk, v, ldv, s, c, nblk);
    else kv_append_kernel<D, PAGE, 256><<<grid, 256, 0, st>>>(k, ldk, v, ldv, s, c, nblk);
  };
  const auto by_page = [&]<int D>() {
    switch (c.page) {
      case 16: return go.template operator()<D, 16>();
      case 32: return go.template operator()<D, 32>();
      case 64: return go.template operator()<D, 64>();
      default: return go.template operator()<D, 128>();
    }
  };
  if (c.dim == 64) by_page.template operator()<64>();
  else if (c.dim == 128) by_page.template operator()<128>();
  else by_page.template operator()<256>();
  UH_CHECK_LAUNCH();
}

size_t kv_pages_workspace(int B, int pages) { return B < 0 || pages < 0 ? 0 : carve_pages(nullptr, B, pages).bytes; }

// The copies, by at most `wgs` workgroups and no more than there can be pieces.
static void launch_copies(const KvCache& c, int layers, size_t most, const PagesWs& w, const int32_t* table,
                          int32_t* table_out, size_t entries, size_t wgs, hipStream_t st) {
  const size_t per = (size_t(c.heads) * c.page * c.dim + CP_BYTES - 1) / CP_BYTES;
  const size_t want = std::max(most * layers * 2 * per, (entries + 255) / 256);
  const unsigned grid = unsigned(std::clamp<size_t>(want, 1, wgs));
  kv_copy_kernel<<<grid, 256, 0, st>>>(c, layers, w, table, table_out, entries);
  UH_CHECK_LAUNCH();
}

void kv_reserve(const KvSeqs& s, const int32_t* grow, int32_t* refs, const KvCache& c, int layers, int32_t* ok, void* ws,
                size_t ws_bytes, hipStream_t st) {
  check_cache("kv_reserve", c);
  check_seqs("kv_reserve", s, grow, refs, c.pages, c.page);
  if (layers < 1) throw std::runtime_error("kv_reserve: layers < 1");
  if (!ok) throw std::runtime_error("kv_reserve: null operand");
  check_ws("kv_reserve", ws, ws_bytes, kv_pages_workspace(s.B, c.pages));
  if (s.B == 0) return;
  const PagesWs w = carve_pages(ws, s.B, c.pages);
  kv_reserve_kernel<<<1, PL_NT, 0, st>>>(s, grow, refs, c.pages, c.page, ok, w);
  UH_CHECK_LAUNCH();
  launch_copies(c, layers, size_t(s.B), w, nullptr, nullptr, 0, 2048, st);  // (most steps copy nothing)
}

void kv_fork(const KvSeqs& s, const int32_t* from, int32_t* refs, int pages, int page, int32_t* done, hipStream_t st) {
  check_seqs("kv_fork", s, from, refs, pages, page);
  if (!done) throw std::runtime_error("kv_fork: null operand");
  if (s.B == 0) return;
  kv_fork_kernel<<<unsigned(s.B), 64, 0, st>>>(s, from, refs, pages, page, done);
  UH_CHECK_LAUNCH();
  kv_fork_lens_kernel<<<cdiv(s.B, 256), 256, 0, st>>>(s, from, done);
  UH_CHECK_LAUNCH();
}

void kv_free(const KvSeqs& s, const int32_t* keep, int32_t* refs, int pages, int page, hipStream_t st) {
  check_seqs("kv_free", s, keep, refs, pages, page);
  if (s.B == 0) return;
  kv_free_kernel<<<unsigned(s.B), 64, 0, st>>>(s, keep, refs, pages, page);
  UH_CHECK_LAUNCH();
}

void kv_compact(const int32_t* table, int32_t* table_out, int max_blocks, int B, const int32_t* refs, int32_t* refs_out,
                const KvCache& c, int layers, int32_t* live, void* ws, size_t ws_bytes, hipStream_t st) {
  check_cache("kv_compact", c);
  if (B < 0 || max_blocks < 0) throw std::runtime_error("kv_compact: negative size");
  if (max_blocks > (1 << 23)) throw std::runtime_error("kv_compact: max_blocks > 2^23");
  const size_t entries = size_t(B) * max_blocks;
  if (layers < 1) throw std::runtime_error("kv_compact: layers < 1");
  if (!refs || !refs_out || (entries && (!table || !table_out))) throw std::runtime_error("kv_compact: null operand");
  check_ws("kv_compact", ws, ws_bytes, kv_pages_workspace(B, c.pages));
  const PagesWs w = carve_pages(ws, B, c.pages);
  kv_compact_kernel<<<1, PL_NT, 0, st>>>(refs, refs_out, c.pages, live, w);
  UH_CHECK_LAUNCH();
  launch_copies(c, layers, size_t(c.pages) / 2, w, table, table_out, entries, 8192, st);  // (2048: 3% longer)
}

}  // namespace unholy::kernels
