"""The 8-bit paged key / value cache on the GPU against the plain numpy reference (tests/kv_ref.py): codes, scales, tables
and copies exactly, the attention within bounds that count its roundings."""
import numpy as np
import pytest

from tests import kv_ref
from tests.helpers import from_bf16, randn_bf16, to_bf16
from unholy_amd import call
from unholy_amd.device import DeviceBuffer, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu

GUARD = 0xA5


def dev(a):
    return DeviceBuffer.from_array(np.ascontiguousarray(a))


class Cache:
    """A step's cache, tables and lengths on the device."""

    def __init__(self, step):
        self.step = step
        self.k, self.v, self.ks, self.vs = dev(step.k), dev(step.v), dev(step.ks), dev(step.vs)
        self.cu, self.lens, self.table = dev(step.cu), dev(step.lens), dev(step.table)

    def arrays(self):
        return self.k, self.v, self.ks, self.vs

    def down(self):
        s = self.step
        return (self.k.download(s.k.shape, np.uint8), self.v.download(s.v.shape, np.uint8),
                self.ks.download(s.ks.shape, np.uint8), self.vs.download(s.vs.shape, np.uint8))


def attend(c, q, Hq, scale, window=0, sinks=0, pad=0, max_new=None, stream=None, lse=True):
    """out bits [rows, Hq, D] and lse [rows, Hq] (NaN where not written); rows with `pad` values between them."""
    s = c.step
    rows, width = q.shape[0], Hq * s.D
    ld = width + pad
    x = np.full((rows, ld), 0x7FC0, np.uint16)
    x[:, :width] = q.reshape(rows, width)
    dq, out = dev(x), dev(np.full((rows, ld), 0x7FC1, np.uint16))
    dl = dev(np.full((rows, Hq), np.nan, np.float32))
    most = max(s.n + [0]) if max_new is None else max_new
    need = call("uh_kv_attend_workspace_size", rows, most, s.B, Hq, s.Hkv, s.D)
    ws = dev(np.concatenate([np.zeros(need, np.uint8), np.full(64, GUARD, np.uint8)]))
    call("uh_kv_attend", dq, ld, c.cu, rows, most, c.lens, c.table, s.max_blocks, s.B, *c.arrays(), s.pages, s.page, Hq,
         s.Hkv, s.D, scale, window, sinks, out, ld, dl if lse else None, ws, need, stream)
    synchronize()
    assert (ws.download(need + 64, np.uint8)[need:] == GUARD).all()
    got = out.download((rows, ld), np.uint16)
    assert (got[:, width:] == 0x7FC1).all()
    return got[:, :width].reshape(rows, Hq, s.D), dl.download((rows, Hq), np.float32)


def check_attend(step, Hq, scale=None, window=0, sinks=0, pad=0, seed=1, qscale=1.0, max_new=None):
    rng = np.random.default_rng(seed)
    scale = step.D ** -0.5 if scale is None else scale
    q = randn_bf16(rng, (step.rows, Hq, step.D), qscale)
    got, lse = attend(Cache(step), q, Hq, scale, window, sinks, pad, max_new)
    ref, rlse, tol, ltol = kv_ref.attend(step, from_bf16(q).astype(np.float64), Hq, scale, window, sinks)
    untouched = np.ones(step.rows, bool)
    for b in range(step.B):
        untouched[step.cu[b]:step.cu[b + 1]] = False
    assert (got[untouched] == 0x7FC1).all() and np.isnan(lse[untouched]).all()
    out, ref, rlse, tol, ltol = (x[~untouched] for x in (from_bf16(got).astype(np.float64), ref, rlse, tol, ltol))
    lse = lse[~untouched]
    assert np.array_equal(np.isnan(out), np.isnan(ref)) and np.array_equal(np.isnan(lse), np.isnan(rlse))
    fine, near = ~np.isnan(ref), np.isfinite(rlse)
    err = np.abs(out - ref)[fine]
    print(f"attend rows={step.rows} worst error {np.max(err / np.maximum(tol[fine], 1e-30), initial=0):.3f} of bound")
    assert (err <= tol[fine]).all()
    empty = np.isneginf(rlse)
    assert (np.isneginf(lse) == empty).all() and (out[empty] == 0).all()
    assert (np.abs(lse[near] - rlse[near]) <= ltol[near]).all()


# ---- attention -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 1), (6, 2)])
def test_decode(D, page, Hq, Hkv):
    """One token a sequence; contexts of nothing, under a page, page and tile borders, a few hundred."""
    rng = np.random.default_rng(D + page + Hq)
    ctx = [0, 1, 14, 15, 16, 62, 63, 64, 127, 128, 300, 511]
    check_attend(kv_ref.Step(rng, [1] * len(ctx), ctx, Hkv, D, page), Hq)


@pytest.mark.parametrize("Hq,Hkv", [(12, 1), (16, 1), (17, 1), (40, 2), (96, 8), (7, 7)])
@pytest.mark.parametrize("n", [1, 5])
def test_groups(Hq, Hkv, n):
    """Query heads per key / value head on both sides of a 16-row operand, alone and with draft tokens."""
    rng = np.random.default_rng(Hq + n)
    check_attend(kv_ref.Step(rng, [n, n, n], [3, 200, 77], Hkv, 128, 32), Hq)


@pytest.mark.parametrize("D,page,Hq,Hkv", [(64, 16, 8, 2), (128, 64, 4, 1), (128, 128, 3, 3), (256, 32, 8, 1)])
@pytest.mark.parametrize("n,ctx", [([300], [0]), ([257], [130]), ([64, 1, 190, 2], [0, 400, 65, 0]),
                                   ([129, 33], [7, 1000])])
def test_prompts(D, page, Hq, Hkv, n, ctx):
    rng = np.random.default_rng(sum(n) + D)
    check_attend(kv_ref.Step(rng, n, ctx, Hkv, D, page), Hq)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (5, 1), (64, 0), (64, 4), (100, 64), (100, 130), (5000, 3)])
@pytest.mark.parametrize("n,ctx", [([1, 1, 1, 1], [0, 63, 300, 901]), ([5, 2], [70, 611]), ([260, 1, 40], [0, 513, 200])])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (128, 128)])
def test_window_and_sinks(window, sinks, n, ctx, D, page):
    rng = np.random.default_rng(window + sinks + sum(n))
    check_attend(kv_ref.Step(rng, n, ctx, 2, D, page), 8, window=window, sinks=sinks)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_long_contexts(D):
    """Contexts that are split over many workgroups, next to short ones, and their joined rows."""
    rng = np.random.default_rng(D)
    check_attend(kv_ref.Step(rng, [1, 1, 1, 3, 1], [9000, 3, 2500, 4000, 0], 1, D, 64), 4)


@pytest.mark.parametrize("n,Hq", [(1, 1), (1, 16), (5, 16), (2, 40)])
@pytest.mark.parametrize("D", [64, 128])
def test_one_long_context(n, Hq, D):
    """One sequence and one key / value head, with as many parts as are worth their join."""
    rng = np.random.default_rng(n * Hq)
    check_attend(kv_ref.Step(rng, [n], [20000], 1, D, 64), Hq, max_new=max(n, 3) if Hq == 1 else 2 ** 31 - 1)


@pytest.mark.parametrize("n", [[0, 0], [0, 3, 0], [1, 0, 0, 150, 0, 1], [0, 200]])
def test_sequences_without_rows(n):
    rng = np.random.default_rng(len(n))
    check_attend(kv_ref.Step(rng, n, [20 * i for i in range(len(n))], 2, 64, 16, spare_rows=5), 4)


@pytest.mark.parametrize("pad", [0, 8, 4096])
def test_strided_rows_and_rows_behind_the_last_sequence(pad):
    rng = np.random.default_rng(pad)
    check_attend(kv_ref.Step(rng, [1, 6, 130], [50, 9, 0], 2, 64, 32, spare_rows=7), 4, pad=pad, max_new=140)


@pytest.mark.parametrize("n", [[1, 2], [100, 3]])
def test_rows_that_see_nothing(n):
    """More rows than tokens (positions below zero), and blocks without a page: zeros and -inf."""
    rng = np.random.default_rng(5)
    s = kv_ref.Step(rng, n, [200, 100], 2, 64, 16)
    s.lens = np.array([n[0] - 1, 60], np.int32)  # the first row of sequence 0 stands before its first token
    s.table[1, 0], s.table[1, 1], s.table[1, 2] = -1, s.pages, 1 << 30
    check_attend(s, 4)
    s.table[:] = -1
    check_attend(s, 4)
    check_attend(s, 4, window=3, sinks=1)


@pytest.mark.parametrize("n", [[1, 1], [150, 2]])
def test_lengths_past_the_table(n):
    """Tokens that the table has no entry for are not there."""
    rng = np.random.default_rng(6)
    s = kv_ref.Step(rng, n, [90, 33], 1, 128, 16, spare_blocks=0)
    s.lens = s.lens + 40
    check_attend(s, 4)


@pytest.mark.parametrize("scale,qscale", [(0.0, 1.0), (-0.1, 1.0), (1.0, 8.0), (30.0, 1.0)])
def test_scales(scale, qscale):
    """All weights alike, a negative scale, and scores so far apart that one token takes all."""
    rng = np.random.default_rng(9)
    check_attend(kv_ref.Step(rng, [1, 70, 4], [130, 60, 700], 2, 64, 32), 4, scale=scale, qscale=qscale)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("n", [1, 3, 140])
def test_nan_reaches_only_the_rows_that_see_it(n, page):
    """NaN codes fill every slot behind the last token. One value NaN and one key NaN of a visible token: the value's
    channel and the key's row, and from the token on only."""
    rng = np.random.default_rng(n)
    s = kv_ref.Step(rng, [n, n], [100, 40], 2, 64, page)
    for b in range(2):
        for t in range(int(s.lens[b]), -(-int(s.lens[b]) // page) * page):
            s.k[s.table[b, t // page], :, t % page] = 0xFF
            s.v[s.table[b, t // page], :, :, t % page] = 0x7F
    check_attend(s, 4)
    check_attend(s, 4, window=30, sinks=2)
    q = randn_bf16(rng, (s.rows, 4, 64))
    clean, _ = attend(Cache(s), q, 4, 0.1, 60, 2)
    tv, tk = 100 + n - 1, 40 + n // 2  # the last token of sequence 0; one of the new ones of sequence 1
    s.v[s.table[0, tv // page], 1, 5, tv % page] = 0x7F
    s.k[s.table[1, tk // page], 0, tk % page, 7] = 0xFF
    s.v[s.table[0, 0], 0, 9, 30 % page if page > 30 else 3] = 0xFF  # an early token: outside the window of late rows
    early = 30 if page > 30 else 3
    got, _ = attend(Cache(s), q, 4, 0.1, 60, 2)
    want = from_bf16(clean).copy()
    for i in range(n):
        if s.position(0, i) >= tv:
            want[i, 2:, 5] = np.nan
        if s.position(0, i) - early < 60:
            want[i, :2, 9] = np.nan
        if 0 <= s.position(1, i) - tk < 60:
            want[n + i, :2] = np.nan
    assert (np.isnan(from_bf16(got)) == np.isnan(want)).all()
    fine = ~np.isnan(want)
    assert np.array_equal(from_bf16(got)[fine], want[fine])


def spare_page_0(s):
    """Page 0 of a step changes places with a page that no sequence has; the pages that none has then, page 0 first."""
    free = np.setdiff1d(np.arange(s.pages), s.table)
    if free[0] != 0:
        s.table[s.table == 0] = free[0]
        for x in (s.k, s.v, s.ks, s.vs):
            x[free[0]] = x[0]
        free[0] = 0
    return free


@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
@pytest.mark.parametrize("D,page,n", [(64, 16, 1), (64, 64, 3), (128, 32, 5), (256, 128, 1), (64, 16, 140), (128, 64, 140),
                                      (256, 32, 140)])
def test_scales_of_pages_that_no_row_sees(D, page, n, window, sinks):
    """Not a number (byte 255): the scales of every page that holds no token of a sequence. One stands in the table behind
    each sequence's last token, and page 0 is one, next to blocks that have no page."""
    rng = np.random.default_rng(page + n)
    s = kv_ref.Step(rng, [n, n], [400, 130], 2, D, page, spare_blocks=4)
    free = spare_page_0(s)
    s.ks[free], s.vs[free] = 255, 255
    for b in range(2):
        blocks = -(-int(s.lens[b]) // page)
        s.table[b, blocks:blocks + 2] = free[1]
    s.table[0, 130 // page] = -1
    check_attend(s, 4, window=window, sinks=sinks)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("n", [1, 3, 140])
@pytest.mark.parametrize("side", ["ks", "vs"])
def test_a_scale_that_is_nan_reaches_only_the_rows_that_see_it(side, n, page):
    """Not a number (byte 255): the scale of sequence 0's first block and of sequence 1's third, of one head. Every value of
    it is NaN for the rows that see one of its tokens, and nothing for the others."""
    rng = np.random.default_rng(n + page)
    s = kv_ref.Step(rng, [n, n], [400, 130], 2, 64, page)
    q = randn_bf16(rng, (s.rows, 4, 64))
    for window in (0, 60):
        clean, clse = attend(Cache(s), q, 4, 0.1, window)
        kept = getattr(s, side).copy()
        getattr(s, side)[s.table[0, 0], 1] = getattr(s, side)[s.table[1, 2], 0] = 255
        got, lse = attend(Cache(s), q, 4, 0.1, window)
        setattr(s, side, kept)
        want, wlse = from_bf16(clean).copy(), clse.copy()
        for b, blk, heads in ((0, 0, slice(2, 4)), (1, 2, slice(0, 2))):
            for i in range(n):
                p = s.position(b, i)
                first, last = (max(p - window + 1, 0) if window else 0), p  # what the row sees
                if first < (blk + 1) * page and last >= blk * page:
                    want[b * n + i, heads] = np.nan
                    if side == "ks":
                        wlse[b * n + i, heads] = np.nan
        assert (np.isnan(from_bf16(got)) == np.isnan(want)).all()
        fine = ~np.isnan(want)
        assert np.array_equal(from_bf16(got)[fine], want[fine])
        assert np.array_equal(lse, wlse, equal_nan=True)


def test_attend_is_the_same_every_time_and_without_lse():
    rng = np.random.default_rng(3)
    s = kv_ref.Step(rng, [1, 1, 40, 1], [3000, 0, 500, 1500], 2, 128, 64)
    c, q = Cache(s), randn_bf16(rng, (s.rows, 8, 128))
    first, lse = attend(c, q, 8, 0.1)
    for _ in range(3):
        again, l2 = attend(c, q, 8, 0.1)
        assert np.array_equal(first, again) and np.array_equal(lse, l2)
    assert np.array_equal(first, attend(c, q, 8, 0.1, lse=False)[0])


@pytest.mark.parametrize("B,tokens", [(100, 256), (70, 128), (300, 64), (65, 448)])
def test_tables_that_are_full(B, tokens):
    """Many sequences as long as the table: every workgroup that the launch may have is needed."""
    rng = np.random.default_rng(B)
    check_attend(kv_ref.Step(rng, [1] * B, [tokens - 1] * B, 1, 64, 64, spare_blocks=0), 2)


@pytest.mark.parametrize("Hkv", [1, 2])
@pytest.mark.parametrize("n,ctx,window", [(129, 600, 190), (129, 600, 200), (300, 1000, 255), (257, 63, 130), (130, 800, 1)])
def test_last_rows_that_see_fewer_tiles(n, ctx, window, Hkv):
    """A window that is cut finer for a sequence's whole row blocks than for the few rows of its last."""
    rng = np.random.default_rng(n + window)
    check_attend(kv_ref.Step(rng, [n], [ctx], Hkv, 64, 32), Hkv, window=window, sinks=2)


@pytest.mark.parametrize("window", [0, 77])
@pytest.mark.parametrize("n", [[1, 2] * 65, [0] * 60 + [1, 3] + [0] * 70 + [2, 0], [20] * 70, [0] * 67 + [150, 18],
                               [1] * 50 + [19, 0] * 15 + [140] + [2] * 20])
def test_more_sequences_than_lanes(n, window):
    """Past 64 sequences the work is cut in several passes; some with rows for one kernel, some for both."""
    rng = np.random.default_rng(len(n))
    ctx = [int(x) for x in rng.integers(0, 400, len(n))]
    ctx[60], ctx[-2] = 3000, 1700
    check_attend(kv_ref.Step(rng, n, ctx, 1, 64, 64), 1, window=window, sinks=window // 20)


@pytest.mark.parametrize("n", [[1] * 39 + [60], [1] * 20 + [0] * 15 + [3, 17, 100, 0, 16], [20] * 33, [2] * 31 + [30]])
def test_few_and_many_rows_in_no_more_than_a_block(n):
    """Steps that the two kernels share, and steps that are the tiled one's, by rows on average and sequences."""
    rng = np.random.default_rng(sum(n))
    check_attend(kv_ref.Step(rng, n, rng.integers(0, 300, len(n)).tolist(), 8, 64, 64), 8)


@pytest.mark.parametrize("n", [[1, 1], [5, 130], [40]])
def test_windows_past_any_length(n):
    rng = np.random.default_rng(2)
    s = kv_ref.Step(rng, n, [300] * len(n), 1, 64, 16)
    check_attend(s, 4, window=2 ** 31 - 1)
    check_attend(s, 4, window=50, sinks=2 ** 31 - 1)
    check_attend(s, 4, window=-1, sinks=3)  # none


@pytest.mark.parametrize("D,page,Hq,Hkv", [(64, 16, 128, 8), (128, 64, 64, 4), (256, 128, 64, 4)])
@pytest.mark.parametrize("window", [0, 1500])
def test_many_rows_over_many_tiles(D, page, Hq, Hkv, window):
    """Enough row blocks to fill the chip, each over the tiles of a long context, a block without a page far into it; some
    rows of them, each against a sequence of its own that ends there."""
    rng = np.random.default_rng(D)
    n, ctx = 1100, 2000
    s = kv_ref.Step(rng, [n], [ctx], Hkv, D, page)
    s.table[0, 2300 // page] = -1
    q = randn_bf16(rng, (n, Hq, D))
    got, lse = attend(Cache(s), q, Hq, D ** -0.5, window, 3)
    rows = [0, 1, 127, 128, 300, 511, 777, n - 1]
    s.n, s.B, s.cu, s.rows = [1] * len(rows), len(rows), np.arange(len(rows) + 1), len(rows)
    s.lens, s.table = np.array([ctx + 1 + r for r in rows]), np.repeat(s.table, len(rows), 0)
    ref, rlse, tol, ltol = kv_ref.attend(s, from_bf16(q[rows]).astype(np.float64), Hq, D ** -0.5, window, 3)
    assert (np.abs(from_bf16(got[rows]) - ref) <= tol).all() and (np.abs(lse[rows] - rlse) <= ltol).all()


def test_one_workspace_for_calls_of_any_shape():
    """The workspace of the largest call serves the others in any order, and each gives what it gives with its own."""
    rng = np.random.default_rng(21)
    steps = [(kv_ref.Step(rng, n, ctx, Hkv, D, 32), Hq) for n, ctx, Hkv, D, Hq in
             [([1] * 3, [2000, 5, 900], 2, 128, 8), ([150, 1], [700, 90], 1, 64, 4), ([20, 18], [1500, 3], 2, 256, 2),
              ([1] * 90, [70] * 90, 1, 64, 1), ([40] * 3, [800, 0, 64], 2, 128, 4)]]
    calls = [(Cache(s), s, Hq, randn_bf16(rng, (s.rows, Hq, s.D))) for s, Hq in steps]
    want = [attend(c, q, Hq, 0.1)[0] for c, s, Hq, q in calls]
    need = max(call("uh_kv_attend_workspace_size", s.rows, max(s.n), s.B, Hq, s.Hkv, s.D) for s, Hq in steps)
    ws = dev(np.zeros(need, np.uint8))
    for i in [0, 1, 0, 2, 3, 4, 1, 3, 2, 0, 4]:
        c, s, Hq, q = calls[i]
        out = dev(np.zeros(q.shape, np.uint16))
        call("uh_kv_attend", dev(q), Hq * s.D, c.cu, s.rows, max(s.n), c.lens, c.table, s.max_blocks, s.B, *c.arrays(),
             s.pages, s.page, Hq, s.Hkv, s.D, 0.1, 0, 0, out, Hq * s.D, None, ws, need, None)
        synchronize()
        assert np.array_equal(out.download(q.shape, np.uint16), want[i]), i


def test_calls_on_two_streams_at_once():
    """A decode step and a prompt on streams of their own, with workspaces of their own, over the same cache."""
    rng = np.random.default_rng(22)
    s = kv_ref.Step(rng, [1, 1], [4000, 900], 2, 128, 64)
    t = kv_ref.Step.__new__(kv_ref.Step)
    t.__dict__.update(s.__dict__)
    t.n, t.rows, t.cu = [150, 33], 183, np.array([0, 150, 183], np.int32)
    calls = []
    for x in (s, t):
        c, q = Cache(x), randn_bf16(rng, (x.rows, 8, 128))
        need = call("uh_kv_attend_workspace_size", x.rows, max(x.n), 2, 8, 2, 128)
        calls.append((c, x, dev(q), dev(np.zeros(q.shape, np.uint16)), dev(np.zeros(need, np.uint8)), need, Stream(),
                      attend(c, q, 8, 0.1)[0]))
    for _ in range(20):
        for c, x, q, out, ws, need, st, _ in calls:
            call("uh_kv_attend", q, 1024, c.cu, x.rows, max(x.n), c.lens, c.table, x.max_blocks, 2, *c.arrays(), x.pages,
                 x.page, 8, 2, 128, 0.1, 0, 0, out, 1024, None, ws, need, st.handle)
    for c, x, q, out, ws, need, st, want in calls:
        st.synchronize()
        assert np.array_equal(out.download(want.shape, np.uint16), want)


@pytest.mark.parametrize("window,sinks", [(0, 0), (500, 4)])
def test_readers_of_one_cache_on_two_streams(window, sinks):
    """The device arrays of one cache, its tables and lengths read by a decode step, drafts and a prompt at once, each on a
    stream and with rows, output and workspace of its own."""
    rng = np.random.default_rng(23)
    s = kv_ref.Step(rng, [1, 1], [4000, 900], 2, 128, 64)
    c, calls = Cache(s), []
    for n in ([1, 1], [150, 33], [6, 5]):
        x = Cache.__new__(Cache)
        x.__dict__.update(c.__dict__)
        x.step = kv_ref.Step.__new__(kv_ref.Step)
        x.step.__dict__.update(s.__dict__)
        x.step.n, x.step.rows, x.step.cu = n, sum(n), np.concatenate(([0], np.cumsum(n))).astype(np.int32)
        x.cu = dev(x.step.cu)
        q = randn_bf16(rng, (sum(n), 8, 128))
        need = call("uh_kv_attend_workspace_size", sum(n), max(n), 2, 8, 2, 128)
        calls.append((x, n, dev(q), dev(np.zeros(q.shape, np.uint16)), dev(np.zeros(need, np.uint8)), need, Stream(),
                      attend(x, q, 8, 0.1, window, sinks)[0]))
    for _ in range(20):
        for x, n, q, out, ws, need, st, _ in calls:
            call("uh_kv_attend", q, 1024, x.cu, sum(n), max(n), c.lens, c.table, s.max_blocks, 2, *c.arrays(), s.pages,
                 s.page, 8, 2, 128, 0.1, window, sinks, out, 1024, None, ws, need, st.handle)
    for x, n, q, out, ws, need, st, want in calls:
        st.synchronize()
        assert np.array_equal(out.download(want.shape, np.uint16), want)
    for got, want in zip(c.down(), (s.k, s.v, s.ks, s.vs)):
        assert np.array_equal(got, want)


def test_large_page_numbers():
    """A pool past 4 GiB: pages whose bytes lie beyond 32-bit offsets."""
    rng = np.random.default_rng(8)
    s = kv_ref.Step(rng, [1, 9], [300, 100], 8, 256, 128)
    pages = (1 << 32) // (8 * 256 * 128) + 40
    per, base = 8 * 256 * 128, pages - s.pages
    big = Cache(s)
    k, v = DeviceBuffer(pages * per), DeviceBuffer(pages * per)
    ks, vs = DeviceBuffer(pages * 8), DeviceBuffer(pages * 8)
    for buf, a, unit in ((k, s.k, per), (v, s.v, per), (ks, s.ks, 8), (vs, s.vs, 8)):
        call("uh_memcpy_h2d", buf.ptr + base * unit, a.ctypes.data, a.nbytes)
    q = randn_bf16(rng, (s.rows, 8, 256))
    want, _ = attend(big, q, 8, 0.05)
    far = Cache(s)
    far.k, far.v, far.ks, far.vs = k, v, ks, vs
    far.table = dev(np.where(s.table >= 0, s.table + base, -1).astype(np.int32))
    s.pages, near = pages, s.pages
    got, _ = attend(far, q, 8, 0.05)
    assert np.array_equal(got, want)
    new = randn_bf16(rng, (s.rows, 8, 256), 3.0)
    s.pages = near
    run_append(big, new, new)
    s.pages = pages
    run_append(far, new, new)
    for buf, a, unit in zip((k, v, ks, vs), big.down(), (per, per, 8, 8)):
        assert np.array_equal(buf.download(a.shape, np.uint8, base * unit), a)


# ---- append ----------------------------------------------------------------------------------------------------------
def run_append(c, knew, vnew, pad=0, max_new=None, stream=None):
    s = c.step
    rows, width = knew.shape[0], s.Hkv * s.D
    bufs = []
    for x, extra in ((knew, pad), (vnew, 2 * pad)):
        a = np.full((rows, width + extra), 0x7F80, np.uint16)
        a[:, :width] = x.reshape(rows, width)
        bufs.append(dev(a))
    call("uh_kv_append", bufs[0], width + pad, bufs[1], width + 2 * pad, c.cu, rows, max(s.n + [0]) if max_new is None else
         max_new, c.lens, c.table, s.max_blocks, s.B, *c.arrays(), s.pages, s.page, s.Hkv, s.D, stream)
    synchronize()


def check_append(s, knew, vnew, **kw):
    c = Cache(s)
    run_append(c, knew, vnew, **kw)
    for name, got, want in zip(("k", "v", "ks", "vs"), c.down(), kv_ref.append(s, knew, vnew)):
        assert np.array_equal(got, want), name


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("n,ctx", [([1] * 6, [0, 1, 15, 16, 127, 200]), ([150, 0, 3, 17, 128], [0, 5, 14, 130, 1])])
def test_append(D, page, n, ctx):
    """Tokens whose size differs by 2^12: scales of blocks that are begun, kept and grown."""
    rng = np.random.default_rng(D + page + len(n))
    s = kv_ref.Step(rng, n, ctx, 3, D, page, spare_rows=2, spare_blocks=0)
    size = 2.0 ** rng.integers(-6, 7, (s.rows, 3, 1))
    knew, vnew = (to_bf16(rng.standard_normal((s.rows, 3, D)) * size) for _ in range(2))
    check_append(s, knew, vnew, pad=8, max_new=max(n) + 3)


def test_append_values_at_the_borders():
    """Zeros, the smallest and the largest numbers, infinities and NaN, and values halfway between codes."""
    rng = np.random.default_rng(1)
    s = kv_ref.Step(rng, [1] * 8, [0, 5] * 4, 1, 64, 16)
    x = np.zeros((8, 1, 64), np.uint16)
    x[1, 0, :2] = to_bf16([1e-38, -0.0])
    x[2, 0, :4] = [0x7F7F, 0xFF7F, 0x0001, 0x4000]
    x[3, 0, :4] = [0x7F80, 0xFF80, 0x3F80, 0x7FC0]
    x[4, 0, :3] = [0xFFC0, 0x7F80, 0x7F80]
    x[5, 0] = to_bf16(448 / 64 * np.linspace(-1, 1, 64))
    x[6, 0] = to_bf16(np.arange(64) / 16 + 1 / 32)
    x[7, 0] = randn_bf16(rng, (64,), 1e30)
    check_append(s, x, x[::-1].copy())


@pytest.mark.parametrize("rows", [2 ** 31 - 1, 2 ** 31 - 64, (1 << 29) - 3, (1 << 26) + 1])
@pytest.mark.parametrize("D", [64, 256])
def test_append_for_any_number_of_rows(D, rows):
    """A launch that is sized for as many rows as an int counts, of which the step brings a few hundred (none past them is
    read)."""
    rng = np.random.default_rng(7)
    s = kv_ref.Step(rng, [150, 1, 64], [5, 130, 0], 2, D, 64)
    c, width = Cache(s), 2 * D
    knew, vnew = (randn_bf16(rng, (s.rows, 2, D)) for _ in range(2))
    call("uh_kv_append", dev(knew), width, dev(vnew), width, c.cu, rows, rows, c.lens, c.table, s.max_blocks, s.B,
         *c.arrays(), s.pages, s.page, 2, D, None)
    synchronize()
    for got, want in zip(c.down(), kv_ref.append(s, knew, vnew)):
        assert np.array_equal(got, want)


def test_append_skips_what_has_no_slot():
    rng = np.random.default_rng(2)
    s = kv_ref.Step(rng, [5, 40, 3, 70], [0, 20, 30, 0], 2, 64, 16, spare_blocks=0)
    s.lens = np.array([3, 60, 33, 200], np.int32)  # two rows before the first token; tokens past the table
    s.table[1, 2], s.table[2, 2], s.table[3, 1:3] = -1, s.pages, -7
    new = randn_bf16(rng, (s.rows, 2, 64))
    check_append(s, new, new)


def test_append_then_attend_step_by_step():
    """A sequence built token by token: each step's attention over what the cache holds then."""
    rng = np.random.default_rng(4)
    s = kv_ref.Step(rng, [1, 1], [0, 13], 2, 64, 16, spare_blocks=4)
    s.table[0, :3], s.pages = [s.pages, s.pages + 1, s.pages + 2], s.pages + 3
    s.k, s.v = (np.concatenate([x, rng.integers(0, 256, (3,) + x.shape[1:], dtype=np.uint8)]) for x in (s.k, s.v))
    s.ks, s.vs = (np.concatenate([x, np.full((3, 2), 127, np.uint8)]) for x in (s.ks, s.vs))
    s.table[1, 1:3] = [s.table[0, 1], s.table[0, 2]]
    s.table[0, 1:3] = -1
    for step in range(14):
        new = [randn_bf16(rng, (2, 2, 64), 2.0 ** (step % 5)) for _ in range(2)]
        c = Cache(s)
        run_append(c, *new)
        want = kv_ref.append(s, *new)
        s.k, s.v, s.ks, s.vs = c.down()
        for got, ref in zip((s.k, s.v, s.ks, s.vs), want):
            assert np.array_equal(got, ref)
        check_attend(s, 4, seed=step)
        s.lens = s.lens + 1
        s.ctx = [x + 1 for x in s.ctx]


@pytest.mark.parametrize("Hq,max_new,n,mode", [
    (4, 1, [1, 3, 1, 0, 2], "few rows"), (2, 3, [4, 3, 0, 200], "few rows"), (1, 2, [1] * 70 + [3, 2, 9], "few rows"),
    (4, 20, [20, 30, 5], "many rows"), (40, 1, [1, 2, 1], "many rows"), (4, 40, [41], "many rows"),
    (4, 130, [1, 131, 130, 2], "both"), (2, 150, [1] * 66 + [151, 9, 700, 140], "both")])
def test_sequences_of_more_rows_than_max_new(Hq, max_new, n, mode):
    """Steps captured for max_new rows a sequence, replayed with more: the others' results are theirs, of these sequences
    nothing is appended, and their rows come back as rows that see nothing, not with what was there."""
    rng = np.random.default_rng(len(n))
    s = kv_ref.Step(rng, n, rng.integers(0, 150, len(n)).tolist(), 1, 64, 32, spare_rows=2)
    c, st, D = Cache(s), Stream(), 64
    q, new = randn_bf16(rng, (s.rows, Hq, D)), randn_bf16(rng, (s.rows, 1, D))
    dq, dn, out = dev(q), dev(new), dev(np.full(q.shape, 0x7FC1, np.uint16))
    lse = dev(np.full((s.rows, Hq), np.nan, np.float32))
    need = call("uh_kv_attend_workspace_size", s.rows, max_new, s.B, Hq, 1, D)
    ws = dev(np.zeros(need, np.uint8))
    c.cu.upload(np.zeros(s.B + 1, np.int32))  # captured, and run once, without rows

    def work():
        call("uh_kv_append", dn, D, dn, D, c.cu, s.rows, max_new, c.lens, c.table, s.max_blocks, s.B, *c.arrays(), s.pages,
             s.page, 1, D, st.handle)
        call("uh_kv_attend", dq, Hq * D, c.cu, s.rows, max_new, c.lens, c.table, s.max_blocks, s.B, *c.arrays(), s.pages,
             s.page, Hq, 1, D, 0.125, 0, 0, out, Hq * D, lse, ws, need, st.handle)

    synchronize()
    work()
    g = Graph(st, work)
    st.synchronize()
    c.cu.upload(s.cu)
    synchronize()
    taken = kv_ref.Step.__new__(kv_ref.Step)
    taken.__dict__.update(s.__dict__)
    taken.n = [k if k <= max_new else 0 for k in n]
    for _ in range(2):
        g.launch()
        st.synchronize()
        want = kv_ref.append(taken, new, new)
        for got, x in zip(c.down(), want):
            assert np.array_equal(got, x)
        taken.k, taken.v, taken.ks, taken.vs = want
        ref, rlse, tol, ltol = kv_ref.attend(taken, from_bf16(q).astype(np.float64), Hq, 0.125)
        got, gl = out.download(q.shape, np.uint16), lse.download((s.rows, Hq), np.float32)
        for b, k in enumerate(n):
            r = slice(int(s.cu[b]), int(s.cu[b]) + k)
            if k > max_new:
                assert (got[r] == 0).all() and np.isneginf(gl[r]).all(), b
            else:
                assert (np.abs(from_bf16(got[r]) - ref[r]) <= tol[r]).all() and (np.abs(gl[r] - rlse[r]) <= ltol[r]).all(), b
        assert (got[sum(n):] == 0x7FC1).all() and np.isnan(gl[sum(n):]).all()


# ---- pages -----------------------------------------------------------------------------------------------------------
class Pool:
    """Tables, lengths and reference counts of B slots over a pool, host and device."""

    def __init__(self, rng, lens, pages, page, width, layers=2, Hkv=3, D=64):
        self.page, self.pages, self.layers, self.Hkv, self.D, self.B = page, pages, layers, Hkv, D, len(lens)
        blocks = [-(-n // page) for n in lens]
        take = rng.permutation(pages)[: sum(blocks)].astype(np.int32)
        self.table, self.lens = np.full((self.B, width), -1, np.int32), np.array(lens, np.int32)
        for b, k in enumerate(blocks):
            self.table[b, :k], take = take[:k], take[k:]
        self.refs = np.bincount(self.table[self.table >= 0], minlength=pages).astype(np.int32)
        unit = Hkv * page * D
        self.data = [rng.integers(0, 256, (layers, pages, n), dtype=np.uint8) for n in (unit, unit, Hkv, Hkv)]
        self.up()

    def up(self):
        self.d = [dev(x) for x in (self.table, self.lens, self.refs)]
        self.caches = [dev(x) for x in self.data]
        n = call("uh_kv_pages_workspace_size", self.B, self.pages)
        self.ws, self.need = dev(np.full(n + 64, GUARD, np.uint8)), n

    def shape(self):
        return self.layers, self.pages, self.page, self.Hkv, self.D

    def reserve(self, grow, stream=None):
        ok = dev(np.full(self.B, -9, np.int32))
        t, n, r = self.d
        call("uh_kv_reserve", t, self.table.shape[1], n, dev(np.array(grow, np.int32)), self.B, r, *self.caches,
             *self.shape(), ok, self.ws, self.need, stream)
        synchronize()
        ref = kv_ref.reserve(self.table, self.lens, self.refs, grow, self.page)
        self.table, self.lens, self.refs, want, copies = ref
        for a, b in copies:
            for x in self.data:
                x[:, b] = x[:, a]
        self.check()
        assert ok.download(self.B, np.int32).tolist() == want.tolist()
        return want

    def fork(self, src):
        done = dev(np.full(self.B, -9, np.int32))
        t, n, r = self.d
        call("uh_kv_fork", t, self.table.shape[1], n, dev(np.array(src, np.int32)), self.B, r, self.pages, self.page, done,
             None)
        synchronize()
        self.table, self.lens, self.refs, want = kv_ref.fork(self.table, self.lens, self.refs, src)
        self.check()
        assert done.download(self.B, np.int32).tolist() == want.tolist()

    def free(self, keep):
        t, n, r = self.d
        call("uh_kv_free", t, self.table.shape[1], n, dev(np.array(keep, np.int32)), self.B, r, self.pages, self.page, None)
        synchronize()
        self.table, self.lens, self.refs = kv_ref.free(self.table, self.lens, self.refs, keep, self.page)
        self.check()

    def compact(self, in_place):
        t, n, r = self.d
        to, ro = (t, r) if in_place else (dev(np.full_like(self.table, -5)), dev(np.full_like(self.refs, -5)))
        live = dev(np.array([-5], np.int32))
        call("uh_kv_compact", t, to, self.table.shape[1], self.B, r, ro, *self.caches, *self.shape(), live, self.ws,
             self.need, None)
        synchronize()
        if not in_place:
            self.check()  # the tables that were there, and the pages that they name, are as before
        self.table, self.refs, moves, n = kv_ref.compact(self.table, self.refs)
        for a, b in moves:
            for x in self.data:
                x[:, b] = x[:, a]
        self.d = [to, self.d[1], ro]
        self.check()
        assert live.download(1, np.int32)[0] == n

    def check(self):
        for name, buf, want in zip(("table", "lens", "refs"), self.d, (self.table, self.lens, self.refs)):
            assert np.array_equal(buf.download(want.shape, np.int32), want), name
        if not hasattr(self, "lazy"):
            for i, (buf, x) in enumerate(zip(self.caches, self.data)):
                got, used = buf.download(x.shape, np.uint8), self.refs > 0
                assert np.array_equal(got[:, used], x[:, used]), i
        assert (self.ws.download(self.need + 64, np.uint8)[self.need:] == GUARD).all()


@pytest.mark.parametrize("page", [16, 64, 128])
def test_reserve_fork_free(page):
    """A life of a pool: growth, forks of forks, copies on the first growth of a shared page, pages given back."""
    rng = np.random.default_rng(page)
    p = Pool(rng, [0, 1, page, 3 * page + 5, 0, 2 * page, 0, 0], 40, page, 9)
    p.reserve([5, 0, 1, page, -3, 2 * page + 1, 0, 0])
    p.fork([-1, -1, -1, 1, 3, -1, 5, 4])  # slot 3 is not empty, slot 7's source is only now being forked
    p.fork([-1, 99, -1, -1, -1, -1, -1, 4])
    p.reserve([1, 1, 1, 1, 1, 1, 1, 1])
    p.free([0, 1, page - 1, 2 * page, 1 << 30, -1, page, 3])
    p.reserve([page] * 8)
    p.free([0] * 8)
    assert (p.refs == 0).all() and (p.table == -1).all()


def test_reserve_when_pages_run_out():
    rng = np.random.default_rng(1)
    p = Pool(rng, [20, 0, 40, 16, 0], 12, 16, 6)
    p.fork([-1, 0, -1, -1, -1])
    assert p.reserve([5, 0, 97, 30, 3]).tolist() == [1, 1, 0, 1, 1]  # 97 more are past the table's six blocks
    assert p.reserve([0, 1, 40, 1, 20]).tolist() == [1, 1, 1, 1, 0]  # two pages were left, and slot 2 takes both
    p.free([0, 0, 1 << 20, 1 << 20, 1 << 20])
    assert p.reserve([0, 0, 16, 0, 20]).tolist() == [1, 1, 1, 1, 1]


@pytest.mark.parametrize("B,pages", [(1500, 9000), (70, 20000)])
def test_many_sequences(B, pages):
    """More slots than the planning workgroup has threads, and free pages far up in the pool."""
    rng = np.random.default_rng(B)
    lens = rng.integers(0, 60, B).tolist()
    p = Pool(rng, lens, pages, 16, 8, layers=1, Hkv=1)
    p.reserve(rng.integers(0, 40, B).tolist())
    empty = np.flatnonzero(p.lens == 0)
    src = np.full(B, -1, np.int32)
    src[empty] = rng.integers(0, B, len(empty))
    p.fork(src.tolist())
    p.reserve(rng.integers(0, 3, B).tolist())
    p.free(np.where(rng.random(B) < 0.5, 0, p.lens - 1).tolist())
    p.compact(in_place=False)
    p.compact(in_place=True)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens", [[], [0, 0], [70, 3, 200], [16] * 30])
def test_compact(in_place, lens):
    rng = np.random.default_rng(len(lens))
    p = Pool(rng, lens, 61, 16, 14, layers=3)
    if len(lens) > 2:
        p.fork([-1] * len(lens))
        p.free([n if b % 2 else n // 2 for b, n in enumerate(lens)])
    p.compact(in_place)
    live = int((p.refs > 0).sum())
    assert (p.refs[:live] > 0).all() and (p.refs[live:] == 0).all()


# ---- together --------------------------------------------------------------------------------------------------------
def test_a_serving_loop():
    """Prompts, forks, decode steps, rollback and compaction as an engine runs them: reserve, append, attend on the device,
    with the reference following."""
    rng = np.random.default_rng(11)
    page, Hkv, Hq, D, B = 16, 2, 8, 64, 6
    p = Pool(rng, [0] * B, 48, page, 10, layers=1, Hkv=Hkv, D=D)
    p.lazy = True

    def step(n):
        s = kv_ref.Step.__new__(kv_ref.Step)
        s.n, s.B, s.Hkv, s.D, s.page, s.pages = list(n), B, Hkv, D, page, p.pages
        ok = p.reserve(n)
        assert ok.all()
        s.lens, s.table, s.max_blocks = p.lens, p.table, p.table.shape[1]
        s.cu = np.concatenate(([0], np.cumsum(n))).astype(np.int32)
        s.rows = int(s.cu[-1])
        shapes = ((p.pages, Hkv, page, D), (p.pages, Hkv, D, page), (p.pages, Hkv), (p.pages, Hkv))
        s.k, s.v, s.ks, s.vs = (b.download(x, np.uint8) for b, x in zip(p.caches, shapes))
        knew, vnew = (randn_bf16(rng, (s.rows, Hkv, D), 2.0 ** float(rng.integers(-2, 3))) for _ in range(2))
        want = kv_ref.append(s, knew, vnew)
        c = Cache.__new__(Cache)
        c.step, (c.k, c.v, c.ks, c.vs), c.cu, c.lens, c.table = s, p.caches, dev(s.cu), p.d[1], p.d[0]
        run_append(c, knew, vnew)
        s.k, s.v, s.ks, s.vs = c.down()
        used = p.refs > 0
        for got, ref in zip((s.k, s.v, s.ks, s.vs), want):
            assert np.array_equal(got[used], ref[used])
        p.data = [x.reshape(1, p.pages, -1) for x in (s.k, s.v, s.ks, s.vs)]
        q = randn_bf16(rng, (s.rows, Hq, D))
        for window, sinks in ((0, 0), (20, 2)):
            got, lse = attend(c, q, Hq, D ** -0.5, window, sinks)
            ref, rlse, tol, ltol = kv_ref.attend(s, from_bf16(q).astype(np.float64), Hq, D ** -0.5, window, sinks)
            assert (np.abs(from_bf16(got) - ref) <= tol).all() and (np.abs(lse - rlse) <= ltol).all()

    step([37, 5, 0, 0, 0, 1])
    p.fork([-1, -1, 0, 0, 1, -1])
    step([1, 1, 1, 3, 1, 1])
    step([1, 0, 1, 1, 2, 4])
    p.free([38, 0, 1 << 20, 37, 5, 3])
    p.compact(in_place=True)
    step([1, 20, 1, 1, 1, 1])


def test_captured_step_replays_with_new_lengths():
    """reserve, append and attend captured once: each replay takes the lengths, tables and rows that are there then."""
    rng = np.random.default_rng(12)
    s = kv_ref.Step(rng, [1, 1, 2], [1000, 3, 100], 2, 128, 64, spare_blocks=3)
    st, Hq = Stream(), 8
    q, new = dev(randn_bf16(rng, (4, Hq, 128))), dev(randn_bf16(rng, (4, 2, 128)))
    out, grow = dev(np.zeros((4, Hq, 128), np.uint16)), dev(np.array([1, 1, 2], np.int32))
    refs, ok = dev((np.bincount(s.table[s.table >= 0], minlength=s.pages + 8) > 0).astype(np.int32)), dev(np.zeros(3, np.int32))
    extra = 8
    s.pages += extra
    s.k, s.v = (np.concatenate([x, np.zeros((extra,) + x.shape[1:], np.uint8)]) for x in (s.k, s.v))
    s.ks, s.vs = (np.concatenate([x, np.zeros((extra, 2), np.uint8)]) for x in (s.ks, s.vs))
    before = s.lens - np.array(s.n, np.int32)
    s.lens = before
    c = Cache(s)
    wa = call("uh_kv_attend_workspace_size", 4, 2, 3, Hq, 2, 128)
    wp = call("uh_kv_pages_workspace_size", 3, s.pages)
    ws_a, ws_p = dev(np.zeros(wa, np.uint8)), DeviceBuffer(wp)

    def work():
        h = st.handle
        call("uh_kv_reserve", c.table, s.max_blocks, c.lens, grow, 3, refs, *c.arrays(), 1, s.pages, 64, 2, 128, ok, ws_p,
             wp, h)
        call("uh_kv_append", new, 256, new, 256, c.cu, 4, 2, c.lens, c.table, s.max_blocks, 3, *c.arrays(), s.pages, 64, 2,
             128, h)
        call("uh_kv_attend", q, Hq * 128, c.cu, 4, 2, c.lens, c.table, s.max_blocks, 3, *c.arrays(), s.pages, 64, Hq, 2, 128,
             0.09, 0, 0, out, Hq * 128, None, ws_a, wa, h)

    g = Graph(st, work)
    for i in range(5):
        x, y = randn_bf16(rng, (4, Hq, 128)), randn_bf16(rng, (4, 2, 128), 2.0 ** i)
        q.upload(x)
        new.upload(y)
        table, lens, r, _, _ = kv_ref.reserve(c.table.download(s.table.shape, np.int32), c.lens.download(3, np.int32),
                                              refs.download(s.pages, np.int32), [1, 1, 2], 64)
        s.table, s.lens = table, lens
        s.k, s.v, s.ks, s.vs = c.down()
        s.k, s.v, s.ks, s.vs = kv_ref.append(s, y, y)
        g.launch()
        st.synchronize()
        for got, want in zip(c.down(), (s.k, s.v, s.ks, s.vs)):
            assert np.array_equal(got, want)
        assert np.array_equal(c.table.download(table.shape, np.int32), table)
        ref, _, tol, _ = kv_ref.attend(s, from_bf16(x).astype(np.float64), Hq, 0.09)
        assert (np.abs(from_bf16(out.download((4, Hq, 128), np.uint16)) - ref) <= tol).all()
        synchronize()


def test_captured_prompts_replay_with_other_rows():
    """A step of prompts and decode rows captured once: each replay takes the rows and lengths that are there then, and leaves
    the workspace for the next."""
    rng = np.random.default_rng(13)
    s = kv_ref.Step(rng, [100, 100, 100], [400, 1500, 20], 2, 64, 32)
    st, Hq, rows, most = Stream(), 8, 300, 300
    c, q, out = Cache(s), dev(np.zeros((rows, Hq, 64), np.uint16)), dev(np.zeros((rows, Hq, 64), np.uint16))
    need = call("uh_kv_attend_workspace_size", rows, most, 3, Hq, 2, 64)
    ws = dev(np.zeros(need, np.uint8))
    g = Graph(st, lambda: call("uh_kv_attend", q, Hq * 64, c.cu, rows, most, c.lens, c.table, s.max_blocks, 3, *c.arrays(),
                               s.pages, 32, Hq, 2, 64, 0.125, 0, 0, out, Hq * 64, None, ws, need, st.handle))
    for n in ([100, 100, 100], [1, 298, 1], [0, 3, 5], [300, 0, 0], [2, 2, 2], [64, 1, 120], [0, 0, 0], [1, 298, 1]):
        s.n = n
        s.cu = np.concatenate(([0], np.cumsum(n))).astype(np.int32)
        s.lens = np.array([max(500, n[0]), 1600, max(120, n[2])], np.int32)
        x = randn_bf16(rng, (rows, Hq, 64))
        q.upload(x)
        c.cu.upload(s.cu)
        c.lens.upload(s.lens)
        out.upload(np.full((rows, Hq, 64), 0x7FC1, np.uint16))
        synchronize()
        g.launch()
        st.synchronize()
        got = out.download((rows, Hq, 64), np.uint16)
        ref, _, tol, _ = kv_ref.attend(s, from_bf16(x).astype(np.float64), Hq, 0.125)
        m = sum(n)
        assert (np.abs(from_bf16(got[:m]) - ref[:m]) <= tol[:m]).all() and (got[m:] == 0x7FC1).all()
        attend(c, x[:max(m, 1)], Hq, 0.125, max_new=300)  # eager work between the replays
