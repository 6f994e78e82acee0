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

// What kv_share writes and kv_attend_shared reads (device). Sequences of a group read the first `tiles` tiles of SHARE_TILE
// tokens, whose pages they have in common, together: all rows of its sequences, in the order of the slots, are the group's
// list.
constexpr int SHARE_TILE = 64;
constexpr int SHARE_ROWS = 16;  // a sequence that brings more rows is left alone: they fill tiles of rows by themselves
constexpr int SHARE_SEQS = 4096;  // sequences past these are alone: the plan compares all pairs
__host__ __device__ inline int share_seqs(int B) { return B < SHARE_SEQS ? B : SHARE_SEQS; }
struct ShareHead {
  int magic, B, rows, max_new, max_blocks, page;
  int groups, list;  // their number, rows in the list
  int pad[7];
  unsigned done;     // kv_share's workgroups that are done; zero between launches
};
struct ShareSeq {
  int tiles;  // 0: alone
  int at;     // its first row, from the group's first on
  int row0, group;
};
struct ShareGroup {
  int row0, rows, tiles;
  int seq;    // whose table is read
  int first;  // the lowest position of its rows when the plan was made: no row has a lower one while sequences grow
  int pad[3];
};
struct Share {
  ShareHead* head;
  ShareSeq* seqs;      // [B]
  ShareGroup* groups;  // [B / 2 + 1]
  int2* list;          // [rows] {row of the step, its sequence}
  int4* found;         // [n = share_seqs(B), up to a multiple of SHARE_AHEAD] kv_share's own: what it knows of each sequence
  unsigned long long* best;  // [n] the same of each class
  int2* sums;                // [n]
  size_t bytes;
};
constexpr int SHARE_AHEAD = 16;
constexpr int SHARE_MAGIC = 0x5ea4ed01;
inline Share carve_share(void* plan, int B, int rows) {
  Share s;
  char* p = static_cast<char*>(plan);
  const size_t n = size_t(share_seqs(B));
  const auto take = [&](size_t bytes) {
    char* at = p;
    p += (bytes + 15) / 16 * 16;
    return at;
  };
  s.head = reinterpret_cast<ShareHead*>(take(sizeof(ShareHead)));
  s.seqs = reinterpret_cast<ShareSeq*>(take(sizeof(ShareSeq) * size_t(B)));
  s.groups = reinterpret_cast<ShareGroup*>(take(sizeof(ShareGroup) * (size_t(B) / 2 + 1)));
  s.list = reinterpret_cast<int2*>(take(sizeof(int2) * size_t(rows)));
  s.found = reinterpret_cast<int4*>(take(sizeof(int4) * ((n + SHARE_AHEAD - 1) / SHARE_AHEAD * SHARE_AHEAD)));
  s.best = reinterpret_cast<unsigned long long*>(take(sizeof(unsigned long long) * n));
  s.sums = reinterpret_cast<int2*>(take(sizeof(int2) * n));
  s.bytes = size_t(p - static_cast<char*>(plan));
  return s;
}
// Whether a plan was made for a step of these sizes: another one is not used.
__device__ __forceinline__ bool share_fits(const ShareHead* h, const KvStep& s, int page) {
  return h->magic == SHARE_MAGIC && h->B == s.B && h->rows == s.rows && h->max_new == s.max_new &&
         h->max_blocks == s.max_blocks && h->page == page;
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
