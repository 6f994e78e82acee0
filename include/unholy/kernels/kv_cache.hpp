// The 8-bit paged key / value cache of the attention between the projections: appending, attention, pages. No reference
// counterpart.
//
// One layer's cache is pages of `page` tokens (16, 32, 64 or 128), for each page and key / value head
//   k  e4m3 [page, dim], one row a token,
//   v  e4m3 [dim, page], transposed: consecutive tokens of a channel, as the value product's matrix operand wants them,
//   ks, vs  e8m0, the power-of-two scale of the block's keys and of its values (kv_append's are 2^119 at most; 255 is NaN,
//           and so are the keys or values of its block then),
// each array [pages, heads, ...] (pool-wide calls: [layers, pages, heads, ...]); dim 64, 128 or 256; k and v 16-byte
// aligned. Position t of sequence b lies in slot t % page of page table[b * max_blocks + t / page]; an entry that is no
// page number (-1) holds nothing.
//
// A step brings rows cu[b] .. cu[b + 1] of sequence b (cu [B + 1], ascending); lens[b] counts the sequence's tokens, the
// new ones included, so row i of its n is the token at position lens[b] - n + i. cu, lens and table are read on the
// device: a captured step replays with what they hold then. `rows` is how many rows the row arrays have, `max_new` at
// least the rows of any one sequence: a sequence that brings more all the same (a launch captured for fewer, say) is taken
// as one that brings none, none of its rows is appended, and their attention is what a row is given that sees nothing. Rows
// that no sequence has are left as they are. No sequences, no rows or max_new 0: nothing is launched.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace unholy::kernels {

using bf16 = uint16_t;

struct KvCache {
  uint8_t *k, *v, *ks, *vs;
  int pages, page, heads, dim;
};
struct KvStep {
  const int32_t *cu, *lens, *table;
  int B, max_blocks, rows, max_new;
};

// The new rows' keys and values k, v bf16 [rows, heads, dim] (row strides ldk, ldv >= heads * dim, % 8; 16-byte aligned)
// quantized into their slots. A block's scale is the smallest power of two 2^e, e <= 119, with amax <= 448 2^e over its
// new tokens' finite values (amax floored at 1e-4); where the block holds earlier tokens of the sequence it is at least
// the block's scale so far (kv_append's own: 2^119 at most), and if it grows their codes are rounded to the new one (a shift
// by a power of two: exact but for codes that become subnormal). Codes: round to nearest even, saturating at 448 2^e; a NaN
// stays one. Tokens at negative positions, past the table or without a page are skipped. A page that the step writes must
// belong to one sequence (kv_reserve sees to that). Nothing but the slots of the sequence's tokens and the block's scales
// is written.
void kv_append(const bf16* k, int ldk, const bf16* v, int ldv, const KvStep& step, const KvCache& cache,
               hipStream_t st);

// Causal attention of the step's rows over their sequences' cached tokens (the new ones among them: kv_append goes
// before). Query head h reads key / value head h / (Hq / heads). Row at position p sees token t <= p, with window > 0 only
// if p - t < window or t < sinks, and only if its page exists;
//   s = scale q . k,  out = sum softmax(s) v,  lse = ln(sum e^s) (may be null),
// out zero and lse -inf for a row whose visible tokens have no s above -inf. Values of tokens that a row does not see do
// not reach it, NaN among them, nor do the scales of blocks that it sees nothing of, whatever they hold.
// q bf16 [rows, Hq, dim] and out the same (row strides ldq, ldo >= Hq * dim, % 8; 16-byte aligned), lse fp32 [rows, Hq].
// ws: device workspace of kv_attend_workspace bytes, 16-byte aligned, zeroed before its first call (finished, or earlier on
// the same stream); a call leaves it as the next one, of any shape, needs it, and nothing else may write it meanwhile. Calls
// that may overlap need one each.
size_t kv_attend_workspace(int rows, int max_new, int B, int Hq, int heads, int dim);
void kv_attend(const bf16* q, int ldq, const KvStep& step, const KvCache& cache, int Hq, float scale, int window,
               int sinks, bf16* out, int ldo, float* lse, void* ws, size_t ws_bytes, hipStream_t st);

// ---- pages ------------------------------------------------------------------------------------------------------------
// The bookkeeping lives on the device: table [B, max_blocks], lens [B] and refs [pages], how many table entries name each
// page (0: free). A sequence holds ceil(lens[b] / page) entries, the others are -1. Every choice goes to the lowest page
// number, so results do not depend on timing. Calls that overlap on the same table or refs race.
struct KvSeqs {
  int32_t *table, *lens;
  int B, max_blocks;
};

// Pages for the next grow[b] tokens (negative: 0) of each sequence, and lens[b] += grow[b]. A last page that is shared
// (refs > 1) and not full is replaced by a copy in all `layers` of the cache, so that the sequence may append to it. Free
// pages go to the sequences in order, lowest first, the copy before the new ones; from the first sequence on whose pages
// no longer suffice, none that needs a page is served. ok[b] = 1: served; 0: untouched (no pages left, or more blocks than
// the table has): such a sequence must bring no rows to the step, they would take its last tokens' places. Pages that this
// call frees by copying them for every user are free afterwards. ws: kv_pages_workspace bytes, 16-byte aligned, any contents.
size_t kv_pages_workspace(int B, int pages);
void kv_reserve(const KvSeqs& seqs, const int32_t* grow, int32_t* refs, const KvCache& cache, int layers, int32_t* ok,
                void* ws, size_t ws_bytes, hipStream_t st);
// Slot b becomes a fork of sequence from[b]: the same pages (refs + 1) and length. done[b] = 1 where that is done; 0, and
// the slot untouched, where from[b] is no slot (-1), has no tokens or b is not empty (lens[b] != 0). All of it as the slots
// are before the call.
void kv_fork(const KvSeqs& seqs, const int32_t* from, int32_t* refs, int pages, int page, int32_t* done,
             hipStream_t st);
// Sequence b keeps its first keep[b] tokens (>= lens[b]: all; <= 0: none, the slot is free then) and gives up the pages
// behind them (refs - 1).
void kv_free(const KvSeqs& seqs, const int32_t* keep, int32_t* refs, int pages, int page, hipStream_t st);
// The `live` pages with refs > 0 moved to numbers below live: the i-th used page from there on, ascending, to the i-th free
// number below. table_out and refs_out (may be table and refs) are the table and the counts afterwards; a moved page's old
// place keeps its contents until the page is used again. *live (device; may be null): their number. ws as above.
void kv_compact(const int32_t* table, int32_t* table_out, int max_blocks, int B, const int32_t* refs, int32_t* refs_out,
                const KvCache& cache, int layers, int32_t* live, void* ws, size_t ws_bytes, hipStream_t st);

}  // namespace unholy::kernels
