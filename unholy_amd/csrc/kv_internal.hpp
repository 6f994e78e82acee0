// What the kernels of the 8-bit paged cache share: the step's geometry, read on the device, and argument checks.
#pragma once

#include <stdexcept>
#include <string>

#include "common.hpp"
#include "unholy/kernels/kv_cache.hpp"

namespace unholy::kernels::kv {

// Sequence b's rows [r0, r1) of the step, kept inside the row arrays whatever cu holds, its length and the position of
// row r0 (below 0 where more rows come than tokens are counted).
struct Seq {
  int r0, r1, len, first;
};
__device__ __forceinline__ Seq seq_of(const KvStep& s, int b) {
  Seq q;
  q.r0 = min(max(s.cu[b], 0), s.rows);
  q.r1 = min(max(s.cu[b + 1], q.r0), s.rows);
  q.len = max(s.lens[b], 0);
  q.first = q.len - (q.r1 - q.r0);
  return q;
}

// A launch is sized for max_new rows of a sequence: one that has more is taken as one without rows, not as the first of them.
__device__ __forceinline__ bool too_many(const KvStep& s, const Seq& q) { return q.r1 - q.r0 > s.max_new; }

// The page of block blk of sequence b, or -1.
__device__ __forceinline__ int page_of(const int32_t* table, int max_blocks, int pages, int b, int blk) {
  if (blk < 0 || blk >= max_blocks) return -1;
  const int p = table[size_t(b) * max_blocks + blk];
  return p >= 0 && p < pages ? p : -1;
}

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

inline void check_pages(const char* who, int pages) {
  if (pages < 1 || pages > (1 << 28)) throw std::runtime_error(std::string(who) + ": pages must be in [1, 2^28]");
}
inline void check_cache(const char* who, const KvCache& c) {
  const auto fail = [&](const char* what) { throw std::runtime_error(std::string(who) + ": " + what); };
  if (c.page != 16 && c.page != 32 && c.page != 64 && c.page != 128) fail("page must be 16, 32, 64 or 128");
  if (c.dim != 64 && c.dim != 128 && c.dim != 256) fail("dim must be 64, 128 or 256");
  if (c.heads < 1 || c.heads > 1024) fail("heads must be in [1, 1024]");
  check_pages(who, c.pages);
  if (!c.k || !c.v || !c.ks || !c.vs) fail("null operand");
  if (!aligned16(c.k) || !aligned16(c.v)) fail("cache not 16-byte aligned");
}
inline void check_step(const char* who, const KvStep& s) {
  const auto fail = [&](const char* what) { throw std::runtime_error(std::string(who) + ": " + what); };
  if (s.B < 0 || s.rows < 0 || s.max_blocks < 0 || s.max_new < 0) fail("negative size");
  if (s.max_blocks > (1 << 23)) fail("max_blocks > 2^23");  // positions stay in 30 bits
  if (!s.cu || !s.lens || (!s.table && s.max_blocks)) fail("null operand");
}

}  // namespace unholy::kernels::kv
