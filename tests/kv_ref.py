"""The 8-bit paged key / value cache in plain numpy, 64 bits: what kv_append, kv_attend and the page calls compute."""
from __future__ import annotations

import numpy as np

from tests.helpers import from_bf16, to_bf16

NAN = 0x7F


def _e4m3_table():
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m / 512.0, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v = np.where((c & 127) == NAN, np.nan, v)
    return np.where(c & 128, -v, v)


E4M3 = _e4m3_table()
_POS = E4M3[:127]  # ascending, 0 .. 448


def encode(v):
    """Nearest e4m3 codes, ties to even, saturating; NaN -> 0x7f."""
    v = np.asarray(v, np.float64)
    a = np.minimum(np.abs(np.nan_to_num(v, nan=0.0, posinf=448.0, neginf=-448.0)), 448.0)
    hi = np.minimum(np.searchsorted(_POS, a), 126)
    lo = np.maximum(hi - 1, 0)
    up, down = _POS[hi] - a, a - _POS[lo]
    c = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    c = np.where(_POS[hi] == a, hi, c)
    c = c | np.where(np.signbit(v), 128, 0)
    return np.where(np.isnan(v), NAN, c).astype(np.uint8)


def scale_byte(amax):
    """Smallest e with amax <= 448 2^e, e8m0, capped at 119."""
    m, e = np.frexp(np.maximum(np.asarray(amax, np.float64), np.float64(np.float32(1e-4))))
    return (np.minimum(e - 9 + (m > 0.875), 119) + 127).astype(np.int64)


class Step:
    """A step over a cache of random contents: B sequences of `ctx[b]` tokens that bring `n[b]` rows each."""

    def __init__(self, rng, n, ctx, Hkv, D, page, spare_rows=0, spare_blocks=1, scale_bytes=(118, 124)):
        self.n, self.ctx, self.Hkv, self.D, self.page = list(n), list(ctx), Hkv, D, page
        self.B = len(self.n)
        self.lens = np.array([a + c for a, c in zip(self.n, self.ctx)], np.int32)
        self.cu = np.concatenate(([0], np.cumsum(self.n))).astype(np.int32)
        self.rows = int(self.cu[-1]) + spare_rows
        blocks = [-(-int(t) // page) for t in self.lens]
        self.max_blocks = max(blocks + [0]) + spare_blocks
        self.pages = sum(blocks) + 2
        take = rng.permutation(self.pages)[: sum(blocks)]
        self.table = np.full((self.B, self.max_blocks), -1, np.int32)
        at = 0
        for b, k in enumerate(blocks):
            self.table[b, :k] = take[at:at + k]
            at += k
        # every slot, the unused ones too, holds any code, NaN among them; tokens of the sequences hold numbers
        self.k = rng.integers(0, 256, (self.pages, Hkv, page, D), dtype=np.uint8)
        self.v = rng.integers(0, 256, (self.pages, Hkv, D, page), dtype=np.uint8)
        self.ks = rng.integers(*scale_bytes, (self.pages, Hkv), dtype=np.uint8)
        self.vs = rng.integers(*scale_bytes, (self.pages, Hkv), dtype=np.uint8)
        for b in range(self.B):
            for t in range(int(self.lens[b])):
                p, s = self.table[b, t // page], t % page
                self.k[p, :, s] = encode(rng.standard_normal((Hkv, D)) * 64)
                self.v[p, :, :, s] = encode(rng.standard_normal((Hkv, D)) * 64)

    def position(self, b, i):
        return int(self.lens[b]) - self.n[b] + i

    def gather(self, b, length=None):
        """Keys and values [T, Hkv, D] in 64 bits of sequence b's tokens, and which of them have a page."""
        T = int(self.lens[b]) if length is None else length
        k, v = np.zeros((T, self.Hkv, self.D)), np.zeros((T, self.Hkv, self.D))
        has = np.zeros(T, bool)
        for blk in range(-(-T // self.page)):
            if blk >= self.max_blocks or not 0 <= self.table[b, blk] < self.pages:
                continue
            p, lo = self.table[b, blk], blk * self.page
            hi = min(T, lo + self.page)
            ks, vs = (2.0 ** (s[p].astype(np.float64) - 127) for s in (self.ks, self.vs))
            k[lo:hi] = (E4M3[self.k[p]] * ks[:, None, None])[:, : hi - lo].transpose(1, 0, 2)
            v[lo:hi] = (E4M3[self.v[p]] * vs[:, None, None])[:, :, : hi - lo].transpose(2, 0, 1)
            has[lo:hi] = True
        return k, v, has


def attend(step, q, Hq, scale, window=0, sinks=0):
    """out and lse of q [rows, Hq, D] (64 bits), with how far a bf16 output and an fp32 lse may be off (see below); NaN
    where a row is no sequence's.

    Bounds: the output is rounded to bf16 (half a step: 2^-8 |out|); the weights are rounded to bf16 for the product with the
    values (2^-8 of each, so 2^-8 sum p |v| at most); a score is a sum of D products in fp32 and a few roundings more, off
    by at most (D + 16) 2^-24 sum |q k| scale, which moves a weight by that share twice (its exponential and the sum); sums
    over T tokens in fp32 add (T + 64) 2^-24. A weight, relative to the largest, that is below fp32's (and bf16's) smallest
    normal number 2^-126 may be taken as zero, and so may a product or an output: T + 2 times 2^-126 max(1, |v|) at most,
    absolute."""
    rows, G = q.shape[0], Hq // step.Hkv
    out, lse = np.full((rows, Hq, step.D), np.nan), np.full((rows, Hq), np.nan)
    tol, ltol = np.zeros((rows, Hq, step.D)), np.zeros((rows, Hq))
    for b in range(step.B):
        k, v, has = step.gather(b)
        t = np.arange(len(k))
        for i in range(step.n[b]):
            r, p = int(step.cu[b]) + i, step.position(b, i)
            see = has & (t <= p)
            if window > 0:
                see &= (p - t < window) | (t < sinks)
            for h in range(Hq):
                if not see.any():
                    out[r, h], lse[r, h] = 0.0, -np.inf
                    continue
                kk, vv = k[see, h // G], v[see, h // G]
                s = kk @ q[r, h] * scale
                m = s.max()
                w = np.exp(s - m)
                out[r, h], lse[r, h] = w @ vv / w.sum(), m + np.log(w.sum())
                ds = (step.D + 16) * 2.0 ** -24 * np.max(np.abs(kk) @ np.abs(q[r, h])) * abs(scale)
                few = (len(kk) + 64) * 2.0 ** -24
                a = w @ np.abs(vv) / w.sum()
                tol[r, h] = 2.0 ** -8 * np.abs(out[r, h]) + (2.0 ** -8 + 2 * ds + few) * 1.01 * a
                tol[r, h] += (len(kk) + 2) * 2.0 ** -126 * max(1.0, np.abs(vv).max())
                ltol[r, h] = ds + few + 2.0 ** -22 * abs(lse[r, h])
    return out, lse, tol, ltol


def append(step, knew, vnew):
    """The caches after the rows knew, vnew bf16 bits [rows, Hkv, D] went into them: k, v, ks, vs."""
    k, v, ks, vs = step.k.copy(), step.v.copy(), step.ks.copy(), step.vs.copy()
    for b in range(step.B):
        first = step.position(b, 0)
        for blk in range(max(first, 0) // step.page, -(-int(step.lens[b]) // step.page)):
            lo, p0 = blk * step.page, max(first, blk * step.page, 0)
            hi = min(lo + step.page, int(step.lens[b]))
            if hi <= p0 or blk >= step.max_blocks or not 0 <= step.table[b, blk] < step.pages:
                continue
            p, s0 = step.table[b, blk], p0 - lo
            r = int(step.cu[b]) + p0 - first
            for x, codes, scales in ((knew, k[p], ks[p]), (vnew, v[p].transpose(0, 2, 1), vs[p])):
                x = from_bf16(x[r:r + hi - p0]).astype(np.float64)  # [n, Hkv, D]
                for h in range(step.Hkv):
                    fine = np.abs(x[:, h])[np.isfinite(x[:, h])]
                    e, old = int(scale_byte(fine.max() if fine.size else 0.0)), int(scales[h])
                    if s0:
                        e = min(max(e, old), 246)
                        if e > old:
                            codes[h, :s0] = encode(E4M3[codes[h, :s0]] * 2.0 ** (old - e)) | (codes[h, :s0] & 128)
                    codes[h, s0:s0 + hi - p0] = encode(x[:, h] / 2.0 ** (e - 127))
                    scales[h] = e
    return k, v, ks, vs


def reserve(table, lens, refs, grow, page):
    """Returns table, lens, refs, ok, copies [(from, to)]."""
    table, lens, refs = table.copy(), lens.copy(), refs.copy()
    before, free, done, copies = refs.copy(), [int(p) for p in np.flatnonzero(refs == 0)], False, []
    ok = np.zeros(len(lens), np.int32)
    for b in range(len(lens)):
        g = max(int(grow[b]), 0)
        held, want = -(-int(lens[b]) // page), -(-(int(lens[b]) + g) // page)
        if want > table.shape[1]:
            continue
        tail = int(table[b, held - 1]) if g and lens[b] % page else -1
        split = tail >= 0 and before[tail] > 1
        need = want - held + split
        done |= need > len(free)
        if need and done:
            continue
        ok[b] = 1
        if split:
            to = free.pop(0)
            copies.append((tail, to))
            table[b, held - 1] = to
            refs[to] = 1
            refs[tail] -= 1
        for j in range(held, want):
            table[b, j] = free.pop(0)
            refs[table[b, j]] = 1
        lens[b] += g
    return table, lens, refs, ok, copies


def fork(table, lens, refs, src):
    table, lens, refs, was = table.copy(), lens.copy(), refs.copy(), lens.copy()
    old, done = table.copy(), np.zeros(len(lens), np.int32)
    for b, j in enumerate(src):
        if 0 <= j < len(lens) and was[b] == 0 and was[j] > 0:
            table[b], lens[b], done[b] = old[j], was[j], 1
            for p in old[j][old[j] >= 0]:
                refs[p] += 1
    return table, lens, refs, done


def free(table, lens, refs, keep, page):
    table, lens, refs = table.copy(), lens.copy(), refs.copy()
    for b in range(len(lens)):
        left = min(max(int(keep[b]), 0), int(lens[b]))
        for j in range(-(-left // page), -(-int(lens[b]) // page)):
            refs[table[b, j]] -= 1
            table[b, j] = -1
        lens[b] = left
    return table, lens, refs


def compact(table, refs):
    """table, refs, moves [(from, to)], live."""
    live = int((refs > 0).sum())
    src = [p for p in range(live, len(refs)) if refs[p] > 0]
    dst = [p for p in range(live) if refs[p] == 0]
    to, new = np.arange(len(refs)), refs.copy()
    for a, b in zip(src, dst):
        to[a], new[b], new[a] = b, refs[a], 0
    return np.where(table >= 0, to[np.maximum(table, 0)], -1).astype(np.int32), new, list(zip(src, dst)), live
