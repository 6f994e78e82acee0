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

__device__ __forceinline__ bool visible(int p, int t, int window, int sinks) {
  return t <= p && (window <= 0 || p - t < window || t < sinks);
}
// An e4m3 code, NaN for its NaN.
__device__ __forceinline__ float kv_value(uint8_t c) {
  return (c & 0x7f) == 0x7f ? __builtin_nanf("") : e4m3_to_f32(c);
}

// A wave per (row, query head): 64 tokens at a time, a token a lane for the products with the query, then a channel (or
// four) a lane for the values; running maximum and sum in fp32.
template <int D>
__global__ __launch_bounds__(64) void kv_attend_rows_kernel(const bf16* __restrict__ qx, int ldq, KvStep st, KvCache c,
                                                            int group, float scale, int window, int sinks,
                                                            bf16* __restrict__ out, int ldo, float* __restrict__ lse) {
  __shared__ float qs[D];
  __shared__ float ps[64];
  const int r = blockIdx.x, hq = blockIdx.y, h = hq / group, lane = threadIdx.x;
  int lo = 0, hi = st.B;  // the last sequence that begins at or before row r
  while (lo < hi) {
    const int m = (lo + hi) / 2;
    if (st.cu[m + 1] <= r) lo = m + 1; else hi = m;
  }
  const int b = lo;
  if (b >= st.B) return;
  const Seq q = seq_of(st, b);
  if (r < q.r0 || r >= q.r1) return;
  const int p = q.first + r - q.r0;
  for (int d = lane; d < D; d += 64) qs[d] = bf16_to_f32(qx[size_t(r) * ldq + size_t(hq) * D + d]);
  __syncthreads();
  float m = -INFINITY, l = 0.0f, acc[D / 64] = {};
  for (int t0 = 0; t0 <= p; t0 += 64) {
    const int t = t0 + lane;
    const int page = t <= p ? page_of(st.table, st.max_blocks, c.pages, b, t / c.page) : -1;
    const bool see = page >= 0 && visible(p, t, window, sinks);
    const size_t ph = size_t(max(page, 0)) * c.heads + h;
    float s = -INFINITY;
    if (see) {
      const uint8_t* k = c.k + (ph * c.page + t % c.page) * D;
      float a = 0.0f;
      for (int d = 0; d < D; ++d) a = fmaf(qs[d], kv_value(k[d]), a);
      s = a * e8m0_to_f32(c.ks[ph]) * scale;
    }
    const float mx = fmaxf(m, wave_max(s == s ? s : -INFINITY));
    const float base = mx == -INFINITY ? 0.0f : mx, w = see ? expf(s - base) : 0.0f, al = expf(m - base);
    l = l * al + wave_sum(w);
    m = mx;
    __syncthreads();
    ps[lane] = w;
    __syncthreads();
    for (int i = 0; i < D / 64; ++i) acc[i] *= al;
    for (int j = 0; j < 64 && t0 + j <= p; ++j) {
      const int pj = __shfl(page, j, 64);
      if (!__shfl(int(see), j, 64)) continue;
      const size_t phj = size_t(pj) * c.heads + h;
      const float f = ps[j] * e8m0_to_f32(c.vs[phj]);
      for (int i = 0; i < D / 64; ++i)
        acc[i] = fmaf(f, kv_value(c.v[(phj * D + lane + 64 * i) * c.page + (t0 + j) % c.page]), acc[i]);
    }
  }
  for (int i = 0; i < D / 64; ++i)
    out[size_t(r) * ldo + size_t(hq) * D + lane + 64 * i] = f32_to_bf16(l == 0.0f ? 0.0f : acc[i] / l);
  if (lse && lane == 0) lse[size_t(r) * (group * c.heads) + hq] = l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace

size_t kv_attend_workspace(int, int, int, int, int, int) { return 256; }

void kv_attend(const bf16* q, int ldq, const KvStep& s, const KvCache& c, int Hq, float scale, int window, int sinks,
               bf16* out, int ldo, float* lse, void* ws, size_t ws_bytes, hipStream_t st) {
  const auto fail = [](const std::string& what) { throw std::runtime_error("kv_attend: " + what); };
  check_cache("kv_attend", c);
  check_step("kv_attend", s);
  if (Hq < 1 || Hq % c.heads || Hq / c.heads > 1024) fail("Hq must be a multiple of heads, up to 1024 times it");
  if (sinks < 0) fail("sinks < 0");
  if (!std::isfinite(scale)) fail("scale is not finite");
  if (s.B == 0 || s.rows == 0 || s.max_new == 0) return;
  if (!q || !out) fail("null operand");
  const int64_t width = int64_t(Hq) * c.dim;
  if (ldq < width || ldo < width || ldq % 8 || ldo % 8) fail("ldq / ldo >= Hq * dim, % 8");
  if (!aligned16(q) || !aligned16(out)) fail("rows not 16-byte aligned");
  const size_t need = kv_attend_workspace(s.rows, s.max_new, s.B, Hq, c.heads, c.dim);
  if (!ws) fail("null workspace");
  if (!aligned16(ws)) fail("workspace not 16-byte aligned");
  if (ws_bytes < need) fail("workspace of " + std::to_string(ws_bytes) + " bytes, " + std::to_string(need) + " needed");
  const dim3 grid(unsigned(s.rows), unsigned(Hq));
  const auto go = [&](auto kernel) {
    kernel<<<grid, 64, 0, st>>>(q, ldq, s, c, Hq / c.heads, scale, window, sinks, out, ldo, lse);
  };
  if (c.dim == 64) go(kv_attend_rows_kernel<64>);
  else if (c.dim == 128) go(kv_attend_rows_kernel<128>);
  else go(kv_attend_rows_kernel<256>);
  UH_CHECK_LAUNCH();
}

}  // namespace unholy::kernels
