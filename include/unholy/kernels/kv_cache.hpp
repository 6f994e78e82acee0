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

#include "unholy/kernels/rope.hpp"

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

// The step between the projections and the cache in one launch: queries q [rows, Hq, dim] and keys k [rows, heads, dim] of each
// row normalised by head (wq, wk bf16 [dim], eps; null: not) and rotated to the row's position, as qk_norm_rope (rope, where
// the weights are null) does it at positions lens[b] - n + i; the queries into qo, the keys, rounded to bf16, and the values v
// into the cache as kv_append does it: all results are those of the two calls, bit for bit. Hq 0: no queries. qo may be q (with
// its stride), otherwise they share no element. Rows that no sequence has, and those of one with more than max_new, are left as
// they are in qo; queries are also rotated where their token has no page. Strides and alignment as in kv_append (q, qo and the
// weights too); r.rot % 16, r.first % 8.
void kv_append_rope(const bf16* q, int ldq, bf16* qo, int ldqo, int Hq, const bf16* wq, const bf16* k, int ldk, const bf16* wk,
                    float eps, const bf16* v, int ldv, const KvStep& step, const Rope& r, const KvCache& cache,
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

// ---- sequences that begin alike ---------------------------------------------------------------------------------------
// Sequences whose tables begin with the same pages (forks, requests behind the same instructions) need those pages' tokens
// read and multiplied once for all of their rows. kv_share finds out which on the device, once for the layers of a step, and
// kv_attend_shared is kv_attend with that plan: the same results but for the order of sums and how far they are off. The common
// tokens go the way of kv_attend's prompts, whose weights are rounded to bf16 (for the product with the values only) relative to
// a maximum that lags by up to 2^8, so that the largest is rounded too: outputs are off by 2.0e-3 to 2.3e-3 of their norm, those
// of kv_attend's single tokens by 1.8e-3, and their rounding to bf16 alone is 1.65e-3.
//
// group [B] (device, may be null): sequences with the same number, in [0, B), may be taken together, others (-1) are alone;
// null: those with the same first page. Of such sequences those that bring 1 to 16 rows and have the same pages as the lowest
// of them for long enough (in whole pages before any new row, and in multiples of 64 tokens) become a group, as many of them
// and as long as saves the most; the others are alone, and so are all past the first 4096. A number has one group at most, and
// its lowest sequence decides with what the others are compared: where numbers are known, sequences of one prefix that others
// share only the beginning of should have their own. Wrong numbers cost time, never results: what is shared is read off the
// table.
// plan: kv_share_plan bytes, 16-byte aligned, zeroed before the first call that makes one in it. It holds for the step's cu,
// lens and table as they were when it was made, and stays valid, under a window too, for steps of the same cu while sequences
// only grow and none of its pages is changed, moved (kv_compact) or given up. (Under a window, common tiles that no row sees any
// more are read until the next plan.) One that does not hold for a step of the same sizes makes wrong results, but writes
// nothing outside of out, lse and the workspace.
size_t kv_share_plan(int B, int rows);
void kv_share(const int32_t* group, const KvStep& step, int pages, int page, void* plan, size_t plan_bytes, hipStream_t st);
// The operands are kv_attend's; the step's sizes (B, rows, max_new, max_blocks) and the page are those of kv_share's call,
// earlier on the same stream or finished: a plan of others is not used. Steps whose tables (B * max_blocks entries) can name
// no more than 64 MB of keys and values, 128 with dim 256, are kv_attend's without further ado (it is faster there), and so are
// those too large for the shared form's 31-bit counts. That goes by how wide the tables are, which is all that the launch knows:
// short sequences in wide tables, and sequences that share little, are faster by kv_attend. ws as kv_attend's (its own size; a
// workspace may serve both calls).
size_t kv_attend_shared_workspace(int rows, int max_new, int B, int Hq, int heads, int dim);
void kv_attend_shared(const bf16* q, int ldq, const KvStep& step, const KvCache& cache, int Hq, float scale, int window,
                      int sinks, bf16* out, int ldo, float* lse, const void* plan, size_t plan_bytes, void* ws,
                      size_t ws_bytes, hipStream_t st);

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
