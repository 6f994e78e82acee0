"""Attention of sequences that begin alike on the GPU: the plan against a plain restatement, the attention against the 64-bit
reference within the bounds that hold for kv_attend (its products and roundings are the same; sums join in another order)."""
import numpy as np
import pytest

from tests import kv_ref, rope_ref
from tests.helpers import from_bf16, randn_bf16, to_bf16
from tests.test_gpu_kv import Cache, Pool, attend, dev
from unholy_amd import call
from unholy_amd.device import DeviceBuffer, Event, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu

GUARD = 0xA5


def wide(s):
    """The step with tables so wide that they could name more than what kv_attend takes by itself."""
    width = int(128e6 if s.D == 256 else 64e6) // (2 * s.B * s.page * s.Hkv * s.D) + 1
    if s.max_blocks < width:
        s.table = np.concatenate([s.table, np.full((s.B, width - s.max_blocks), -1, np.int32)], 1)
        s.max_blocks = width
    return s


def step_of(rng, groups, alone, Hkv, D, page, n=1, order=None, spare_rows=0):
    """A step of groups [(tokens that begin alike, [further tokens of each])] and sequences alone [tokens], n rows each (or a list
    in the order of the sequences), in slots by `order`; and each slot's group (-1: alone)."""
    ctx = [p + o for p, own in groups for o in own] + list(alone)
    label = [g for g, (_, own) in enumerate(groups) for _ in own] + [-1] * len(alone)
    ns = [n] * len(ctx) if isinstance(n, int) else list(n)
    order = np.arange(len(ctx)) if order is None else np.asarray(order)
    s = kv_ref.Step(rng, [ns[i] for i in order], [ctx[i] for i in order], Hkv, D, page, spare_rows=spare_rows)
    label = np.array([label[i] for i in order], np.int32)
    for g, (p, _) in enumerate(groups):
        slots = np.flatnonzero(label == g)
        s.table[slots, :p // page] = s.table[slots[0], :p // page]
    return wide(s), label


def share_ref(s, group=None, max_new=None):
    """tiles of each sequence, and the groups as [(tiles, slots)]."""
    most = max(s.n + [0]) if max_new is None else max_new
    limit = [min(max(int(s.lens[b]) - s.n[b], 0) // s.page, s.max_blocks) for b in range(s.B)]
    classes = {}
    for b in range(s.B):
        key = int(s.table[b, 0]) if group is None else int(group[b])
        ok = 0 <= key < (s.pages if group is None else s.B) and 1 <= s.n[b] <= min(16, most) and limit[b] * s.page >= 64
        if ok:
            classes.setdefault(key, []).append(b)
    tiles, groups = np.zeros(s.B, int), []
    for slots in classes.values():
        r, long = slots[0], {}
        for b in slots:
            k = 0
            while k < min(limit[b], limit[r]) and s.table[b, k] == s.table[r, k] and 0 <= s.table[b, k] < s.pages:
                k += 1
            long[b] = k * s.page // 64
        saved, t = max(((sum(x >= t for x in long.values()) - 1) * t, t) for t in long.values())
        if saved > 0:
            groups.append((t, [b for b in slots if long[b] >= t]))
    for t, slots in groups:
        tiles[slots] = t
    return tiles, sorted(groups, key=lambda g: g[1][0])


def plan_of(c, group=None, most=None, stream=None):
    s = c.step
    most = max(s.n + [0]) if most is None else most
    need = call("uh_kv_share_plan_size", s.B, s.rows)
    plan = dev(np.concatenate([np.zeros(need, np.uint8), np.full(64, GUARD, np.uint8)]))
    g = None if group is None else dev(np.asarray(group, np.int32))
    call("uh_kv_share", g, c.cu, s.rows, most, c.lens, c.table, s.max_blocks, s.B, s.pages, s.page, plan, need, stream)
    synchronize()
    assert (plan.download(need + 64, np.uint8)[need:] == GUARD).all()
    return plan, need


def check_plan(c, plan, group=None, most=None):
    s = c.step
    got = plan.download(16 + 4 * s.B, np.int32)
    tiles, groups = share_ref(s, group, most)
    head, seqs = got[:16], got[16:].reshape(s.B, 4)
    assert head[1:6].tolist() == [s.B, s.rows, max(s.n + [0]) if most is None else most, s.max_blocks, s.page]
    assert seqs[:, 0].tolist() == tiles.tolist()
    assert head[6:8].tolist() == [len(groups), sum(s.n[b] for _, slots in groups for b in slots)]
    row0 = 0
    for g, (_, slots) in enumerate(groups):
        at = 0
        for b in slots:
            assert seqs[b].tolist()[1:] == [at, row0, g]
            at += s.n[b]
        row0 += at
    return tiles, groups


def shared(c, q, Hq, scale, plan, need_plan, window=0, sinks=0, pad=0, most=None, stream=None, lse=True, ws=None):
    s = c.step
    rows, width = q.shape[0], Hq * s.D
    ld, most = width + pad, max(s.n + [0]) if most is None else most
    x = np.full((rows, ld), 0x7FC0, np.uint16)
    x[:, :width] = q.reshape(rows, width)
    dq, out = dev(x), dev(np.full((rows, ld), 0x7FC1, np.uint16))
    dl = dev(np.full((rows, Hq), np.nan, np.float32))
    need = call("uh_kv_attend_shared_workspace_size", rows, most, s.B, Hq, s.Hkv, s.D)
    if ws is None:
        ws = DeviceBuffer(need + 64)
        ws.zero()
        call("uh_memcpy_h2d", ws.ptr + need, np.full(64, GUARD, np.uint8).ctypes.data, 64)
    call("uh_kv_attend_shared", dq, ld, c.cu, rows, most, c.lens, c.table, s.max_blocks, s.B, *c.arrays(), s.pages, s.page, Hq,
         s.Hkv, s.D, scale, window, sinks, out, ld, dl if lse else None, plan, need_plan, ws, need, stream)
    synchronize()
    assert (ws.download(64, np.uint8, need) == GUARD).all()
    got = out.download((rows, ld), np.uint16)
    assert (got[:, width:] == 0x7FC1).all()
    return got[:, :width].reshape(rows, Hq, s.D), dl.download((rows, Hq), np.float32)


def check(s, Hq, group=None, window=0, sinks=0, pad=0, scale=None, qscale=1.0, most=None, seed=1, expect=None, gone=()):
    """gone: sequences with more rows than the launch is sized for."""
    c, scale = Cache(s), s.D ** -0.5 if scale is None else scale
    plan, need = plan_of(c, group, most)
    _, groups = check_plan(c, plan, group, most)
    if expect is not None:
        assert len(groups) == expect
    q = randn_bf16(np.random.default_rng(seed), (s.rows, Hq, s.D), qscale)
    got, lse = shared(c, q, Hq, scale, plan, need, window, sinks, pad, most)
    ref, rlse, tol, ltol = kv_ref.attend(s, from_bf16(q).astype(np.float64), Hq, scale, window, sinks)
    for b in gone:
        r = slice(int(s.cu[b]), int(s.cu[b + 1]))
        ref[r], rlse[r], tol[r], ltol[r] = 0.0, -np.inf, 0.0, 0.0
    untouched = np.ones(s.rows, bool)
    untouched[:s.cu[-1]] = False
    assert (got[untouched] == 0x7FC1).all() and np.isnan(lse[untouched]).all()
    out, ref, rlse, tol, ltol = (x[~untouched] for x in (from_bf16(got).astype(np.float64), ref, rlse, tol, ltol))
    lse = lse[~untouched]
    assert np.array_equal(np.isnan(out), np.isnan(ref)) and np.array_equal(np.isnan(lse), np.isnan(rlse))
    fine, near = ~np.isnan(ref), np.isfinite(rlse)
    err = np.abs(out - ref)[fine]
    print(f"shared rows={s.rows} worst error {np.max(err / np.maximum(tol[fine], 1e-30), initial=0):.3f} of bound")
    assert (err <= tol[fine]).all()
    assert (np.isneginf(lse) == np.isneginf(rlse)).all()
    assert (np.abs(lse[near] - rlse[near]) <= ltol[near]).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (8, 1), (6, 2)])
def test_decode(D, page, Hq, Hkv):
    """A group, one more, and sequences that share nothing."""
    rng = np.random.default_rng(D + page + Hq)
    s, label = step_of(rng, [(300, [0, 1, 65, 40]), (128, [10, 200])], [0, 5, 700], Hkv, D, page, order=rng.permutation(9))
    check(s, Hq, expect=2)
    check(s, Hq, label, expect=2)


@pytest.mark.parametrize("n", [2, 5, 16])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 1, 64, 16), (16, 1, 128, 64), (6, 2, 128, 32), (4, 2, 256, 128), (1, 1, 64, 64)])
def test_drafts(n, Hq, Hkv, D, page):
    """Several rows a sequence: parts of 16 of them, blocks of 128 that end inside a sequence."""
    rng = np.random.default_rng(n + Hq)
    s, _ = step_of(rng, [(400, [3, 90, 0, 17, 64])], [33], Hkv, D, page, n=n, spare_rows=3)
    check(s, Hq, expect=1, pad=8)


@pytest.mark.parametrize("n", [1, 3, 16])
@pytest.mark.parametrize("Hq,Hkv", [(17, 1), (40, 2), (130, 1)])
def test_more_query_heads_than_an_operand_has_rows(n, Hq, Hkv):
    """Parts of 16 rows and blocks of 128 that end inside a token's heads; beside a sequence alone."""
    rng = np.random.default_rng(n + Hq)
    s, _ = step_of(rng, [(200, [3, 90, 0]), (64, [1, 40])], [150], Hkv, 64, 32, n=n)
    check(s, Hq, expect=2)
    check(s, Hq, window=120, sinks=3, expect=2)


@pytest.mark.parametrize("n", [[1, 16, 17, 3, 1, 40], [5, 0, 1, 2, 0, 1], [200, 1, 1, 1, 1, 1], [17, 300, 20, 18, 30, 19]])
def test_steps_of_many_kinds(n):
    """Sequences with more than 16 rows, or none, among the others: they are in no group."""
    rng = np.random.default_rng(sum(n))
    s, label = step_of(rng, [(200, [5, 60, 9, 100])], [70, 0], 2, 64, 16, n=n, spare_rows=4)
    check(s, 6)
    check(s, 6, label, most=max(n) + 5)


@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 4), (100, 70), (150, 0), (400, 64), (5000, 3), (2 ** 31 - 1, 0), (90, 2 ** 31 - 1)])
@pytest.mark.parametrize("D,page,n", [(64, 16, 1), (128, 64, 3)])
def test_window_and_sinks(window, sinks, D, page, n):
    rng = np.random.default_rng(window % 1000 + sinks % 1000)
    s, _ = step_of(rng, [(330, [0, 40, 90, 300]), (128, [2, 5])], [450], 2, D, page, n=n)
    check(s, 4, window=window, sinks=sinks, expect=2)


@pytest.mark.parametrize("scale,qscale", [(0.0, 1.0), (-0.1, 1.0), (1.0, 8.0), (30.0, 1.0)])
def test_scales(scale, qscale):
    rng = np.random.default_rng(9)
    s, _ = step_of(rng, [(200, [5, 60, 9])], [70], 2, 64, 32, n=2)
    check(s, 4, scale=scale, qscale=qscale, expect=1)


@pytest.mark.parametrize("each,Hq", [(40, 4), (33, 8), (70, 16)])
def test_blocks_of_rows(each, Hq):
    """More rows than one block, the last of them not full."""
    rng = np.random.default_rng(each)
    s, _ = step_of(rng, [(256, [int(x) for x in rng.integers(0, 30, each)])], [], 1, 64, 64)
    check(s, Hq, expect=1)


@pytest.mark.parametrize("groups,each", [(70, 2), (3, 50), (130, 3)])
def test_more_sequences_than_lanes(groups, each):
    rng = np.random.default_rng(groups)
    s, label = step_of(rng, [(64 + 16 * int(rng.integers(0, 6)), rng.integers(0, 20, each).tolist()) for _ in range(groups)], [10, 100],
                       1, 64, 16, order=rng.permutation(groups * each + 2))
    check(s, 2, expect=groups)
    check(s, 2, label, expect=groups)


def test_more_sequences_than_the_plan_has_room_for_in_lds():
    rng = np.random.default_rng(17)
    s, label = step_of(rng, [(64, [1, 2])] * 500 + [(80, [0, 3, 1])] * 20, [10] * 5, 1, 64, 16, order=rng.permutation(1065))
    check(s, 1, expect=520)
    check_plan(Cache(s), plan_of(Cache(s), label)[0], label)


def test_more_sequences_than_the_plan_compares():
    """Of pairs that begin alike those among the first 4096 sequences are groups, the others alone; the attention of all."""
    rng = np.random.default_rng(19)
    B, page, Hkv, D = 4500, 64, 1, 64
    s = kv_ref.Step.__new__(kv_ref.Step)
    s.n, s.B, s.Hkv, s.D, s.page, s.rows, s.max_blocks = [1] * B, B, Hkv, D, page, B, 2
    s.cu, s.lens = np.arange(B + 1, dtype=np.int32), rng.integers(65, 100, B).astype(np.int32)
    s.pages = B // 2 + B
    order = rng.permutation(s.pages).astype(np.int32)
    s.table = np.stack([order[np.arange(B) // 2], order[B // 2 + np.arange(B)]], 1)
    s.k, s.v = (kv_ref.encode(rng.standard_normal(x) * 64) for x in ((s.pages, Hkv, page, D), (s.pages, Hkv, D, page)))
    s.ks, s.vs = (rng.integers(118, 124, (s.pages, Hkv), dtype=np.uint8) for _ in range(2))
    s = wide(s)
    c = Cache(s)
    plan, need = plan_of(c)
    got = plan.download(16 + 4 * B, np.int32)
    assert got[6:8].tolist() == [2048, 4096]
    assert (got[16:].reshape(B, 4)[:, 0] == (np.arange(B) < 4096)).all()
    q = randn_bf16(rng, (B, 2, D))
    out, lse = shared(c, q, 2, 0.1, plan, need)
    ref, rlse, tol, ltol = kv_ref.attend(s, from_bf16(q).astype(np.float64), 2, 0.1)
    assert (np.abs(from_bf16(out) - ref) <= tol).all() and (np.abs(lse - rlse) <= ltol).all()


def test_the_time_of_a_plan_does_not_grow_with_the_square_of_its_sequences():
    """A million of them, among which all pairs would be compared for minutes."""
    B, page = 1 << 20, 64
    cu, lens = dev(np.arange(B + 1, dtype=np.int32)), dev(np.full(B, 70, np.int32))
    table = dev(np.stack([np.arange(B, dtype=np.int32) // 2, np.full(B, -1, np.int32)], 1))
    need = call("uh_kv_share_plan_size", B, B)
    plan = dev(np.concatenate([np.zeros(need, np.uint8), np.full(64, GUARD, np.uint8)]))
    st, times = Stream(), []
    for _ in range(2):
        a, b = Event(), Event()
        a.record(st)
        call("uh_kv_share", None, cu, B, 1, lens, table, 2, B, B, page, plan, need, st.handle)
        b.record(st)
        st.synchronize()
        times.append(a.elapsed_ms(b))
    got = plan.download(need + 64, np.uint8)
    assert (got[need:] == GUARD).all()
    got = got[:64 + 16 * B].view(np.int32)
    assert got[6:8].tolist() == [2048, 4096] and (got[16:].reshape(B, 4)[:, 0] == (np.arange(B) < 4096)).all()
    print(f"{times} ms")
    assert min(times) < 100.0


def test_a_block_of_a_group_for_every_workgroup():
    """More blocks than the chip has places: none is cut."""
    rng = np.random.default_rng(70)
    s, _ = step_of(rng, [(64, [1, 2])] * 20, [], 32, 64, 64)
    check(s, 32, expect=20)


@pytest.mark.parametrize("D,parts", [(64, 9000), (128, 5000), (256, 3000)])
def test_long_common_parts(D, parts):
    """Contexts that are split over many workgroups, in two forms."""
    rng = np.random.default_rng(D)
    s, _ = step_of(rng, [(parts, [7, 700, 0])], [1500], 1, D, 64)
    check(s, 4, expect=1)


@pytest.mark.parametrize("groups,times,window", [(16, 42, 0), (70, 11, 0), (16, 42, 5000)])
def test_many_tiles_of_64_channels(groups, times, window):
    """So many common tiles that every workgroup takes own segments and then a part of a block; and more blocks than workgroups.
    (The same two pages over and over: a table may name a page as often as it likes.)"""
    rng = np.random.default_rng(groups)
    s, _ = step_of(rng, [(128, [int(x) for x in rng.integers(0, 40, 2)]) for _ in range(groups)], [], 8, 64, 64)
    s.table = np.concatenate([np.tile(s.table[:, :2], times - 1), s.table], 1)
    s.max_blocks += 2 * (times - 1)
    s.lens += 128 * (times - 1)
    check(s, 8, window=window, sinks=window // 1000, expect=groups)


@pytest.mark.parametrize("D,Hq,Hkv,groups,each,times,alone,window", [
    (128, 8, 8, 4, 2, 50, [20] * 40, 0), (128, 8, 8, 4, 2, 60, [20] * 40, 6600), (128, 4, 4, 2, 2, 200, [2000], 0),
    (128, 48, 8, 8, 6, 26, [], 0), (128, 8, 8, 60, 2, 4, [9] * 20, 0), (64, 8, 8, 16, 2, 16, [30] * 40, 0),
    (64, 8, 8, 16, 2, 30, [700], 2000), (64, 40, 8, 16, 7, 16, [], 0)])
def test_blocks_on_most_of_the_chip(D, Hq, Hkv, groups, each, times, alone, window):
    """So many common tiles, of few rows each or beside little else, that blocks take seven of eight workgroups: cut into parts, or
    (the fifth) whole; the sequences' own tiles share the rest, segment after segment or (the third) one in parts. (The same two
    pages over and over, as above.)"""
    rng = np.random.default_rng(groups * times + D)
    s, _ = step_of(rng, [(128, [int(x) for x in rng.integers(0, 40, each)]) for _ in range(groups)], [], Hkv, D, 64)
    blocks, tiles = groups * Hkv * -(-each * Hq // Hkv // 128), 2 * times  # of which some leave the window
    assert 6 * 512 < blocks * (min(tiles, window // 64) if window else tiles) and (D == 128 or blocks * tiles < 16 * 512)
    t, _ = step_of(rng, [], alone, Hkv, D, 64) if alone else (None, None)
    s.table = np.concatenate([np.tile(s.table[:, :2], times - 1), s.table], 1)
    s.lens += 128 * (times - 1)
    s.ctx = [x + 128 * (times - 1) for x in s.ctx]
    if alone:  # behind the others
        width = max(s.table.shape[1], t.table.shape[1])
        at = np.where(t.table >= 0, t.table + s.pages, -1)
        s.table = np.concatenate([np.pad(x, ((0, 0), (0, width - x.shape[1])), constant_values=-1) for x in (s.table, at)])
        s.k, s.v, s.ks, s.vs = (np.concatenate(x) for x in ((s.k, t.k), (s.v, t.v), (s.ks, t.ks), (s.vs, t.vs)))
        s.pages, s.n, s.ctx, s.lens = s.pages + t.pages, s.n + t.n, s.ctx + t.ctx, np.concatenate([s.lens, t.lens])
        s.B, s.rows, s.cu = len(s.n), s.rows + t.rows, np.arange(len(s.n) + 1, dtype=np.int32)
    s.max_blocks = s.table.shape[1]
    check(s, Hq, window=window, sinks=window // 1000, expect=groups)


def test_the_plan_takes_what_saves_most():
    """Three begin alike for long, six for a little: of 5 x 2 tiles and 2 x 9 the second; and with numbers that say so, both."""
    rng = np.random.default_rng(3)
    s, label = step_of(rng, [(640, [0, 5, 9]), (128, [300, 2, 70])], [], 1, 64, 64)
    s.table[3:, :2] = s.table[0, :2]
    plan = plan_of(Cache(s))[0]
    assert check_plan(Cache(s), plan)[1] == [(10, [0, 1, 2])]
    check(s, 2, expect=1)
    check(s, 2, label, expect=2)
    check(s, 2, [0, 1, 2, 3, 4, 5], expect=0)  # nobody with anybody
    check(s, 2, [0, 0, 9, -5, 6, 2 ** 31 - 1], expect=1)  # numbers out of range: alone
    check(s, 2, [4] * 6, expect=1)


def test_pages_that_are_missing_or_differ():
    """The common part ends where tables have no page, or not the same one."""
    rng = np.random.default_rng(4)
    s, label = step_of(rng, [(640, [0, 5, 9, 33])], [], 1, 64, 16)
    s.table[:, 25] = -1
    check(s, 2, expect=1)
    s.table[2, 13] = s.table[2, 39]
    check(s, 2, label, expect=1)
    s.table[:, 0] = s.pages + 3
    check(s, 2, label, expect=0)
    s.table[:] = -1
    check(s, 2, label, expect=0)


def test_lengths_that_end_the_common_part():
    """No tile of which a new row is a token, or comes before it, is common; nothing past the table is."""
    rng = np.random.default_rng(5)
    s, _ = step_of(rng, [(200, [0, 0, 0])], [], 1, 64, 16)
    s.table[1:] = s.table[0]  # the new tokens' page too
    for lens in ([201, 193, 129], [64, 65, 66], [1, 0, 200], [129, 129, 129], [500, 500, 500]):
        s.lens = np.array(lens, np.int32)
        check(s, 2)


@pytest.mark.parametrize("most", [4, 16])
def test_more_rows_than_the_launch_is_sized_for(most):
    rng = np.random.default_rng(6)
    n = [1, most + 1, 2, 3]
    s, label = step_of(rng, [(150, [0, 4, 8, 70])], [], 2, 64, 16, n=n, spare_rows=2)
    check(s, 4, label, most=most, expect=1, gone=[1])


def test_nan_reaches_the_rows_that_see_it():
    """A NaN in a common value: that channel of every row of the group; in a common key: every row; under a window, the rows
    that still see it. What follows the last tokens is NaN throughout."""
    rng = np.random.default_rng(7)
    s, _ = step_of(rng, [(256, [3, 60, 100])], [90], 2, 64, 64)
    for b in range(s.B):
        for t in range(int(s.lens[b]), -(-int(s.lens[b]) // 64) * 64):
            s.k[s.table[b, t // 64], :, t % 64] = 0xFF
            s.v[s.table[b, t // 64], :, :, t % 64] = 0x7F
    check(s, 4, expect=1)
    s.v[s.table[0, 1], 0, 5, 9] = 0x7F  # token 73
    s.k[s.table[0, 2], 1, 3, 7] = 0xFF  # token 131
    c = Cache(s)
    plan, need = plan_of(c)
    q = randn_bf16(rng, (s.rows, 4, 64))
    for window in (0, 240):
        got = np.isnan(from_bf16(shared(c, q, 4, 0.1, plan, need, window)[0]))
        want = np.isnan(from_bf16(attend(c, q, 4, 0.1, window)[0]))
        assert np.array_equal(got, want) and got[0, 0, 5] and got[0, 2:].all()


def test_scales_that_are_no_number():
    rng = np.random.default_rng(8)
    s, _ = step_of(rng, [(256, [3, 60, 100])], [90], 2, 64, 64)
    s.ks[s.table[0, 1], 0] = s.vs[s.table[0, 2], 1] = 255
    c = Cache(s)
    plan, need = plan_of(c)
    q = randn_bf16(rng, (s.rows, 4, 64))
    for window in (0, 150, 20):
        got, want = (np.isnan(from_bf16(x[0])) for x in (shared(c, q, 4, 0.1, plan, need, window), attend(c, q, 4, 0.1, window)))
        assert np.array_equal(got, want)


def test_a_plan_of_other_sizes_is_not_used():
    """Of a step with another number of rows, sequences or blocks, or of no step: every sequence reads its own."""
    rng = np.random.default_rng(10)
    s, _ = step_of(rng, [(300, [3, 60, 100])], [90], 2, 64, 64, n=2)
    t, _ = step_of(rng, [(300, [3, 60, 100])], [90, 5], 2, 64, 64, n=1)
    c, q = Cache(s), randn_bf16(rng, (s.rows, 4, 64))
    ref, _, tol, _ = kv_ref.attend(s, from_bf16(q).astype(np.float64), 4, 0.1)
    need = call("uh_kv_share_plan_size", s.B, s.rows)
    other, size = plan_of(Cache(t))
    for plan, n in ((other, max(size, need)), (dev(np.zeros(need, np.uint8)), need), (dev(np.full(need, 0xFF, np.uint8)), need)):
        if plan.nbytes < n:
            continue
        got, _ = shared(c, q, 4, 0.1, plan, n)
        assert (np.abs(from_bf16(got) - ref) <= tol).all()


@pytest.mark.parametrize("n", [[16, 1, 1, 1, 1, 1], [1, 1, 1, 1, 1, 16], [0, 9, 0, 9, 1, 2]])
def test_a_plan_of_other_rows_writes_nowhere_else(n):
    """The plan of a step of one row each and two more: what a step of the same sizes and other rows gets is undefined, but it
    stays within its arrays, and the next call with a plan of its own is right."""
    rng = np.random.default_rng(n[0] + 20)
    s, _ = step_of(rng, [(300, [20, 30, 40, 50, 60, 70])], [], 2, 64, 64, n=[4, 1, 4, 4, 4, 4])
    t, _ = step_of(rng, [(300, [20, 30, 40, 50, 60, 70])], [], 2, 64, 64, n=n)
    for x in ("table", "k", "v", "ks", "vs", "lens", "pages", "max_blocks", "rows"):
        setattr(t, x, getattr(s, x))
    q = randn_bf16(rng, (s.rows, 16, 64))
    a, b = Cache(s), Cache(t)
    plan, need = plan_of(a, most=16)
    got, _ = shared(b, q, 16, 0.1, plan, need, most=16)
    assert (got[t.cu[-1]:] == 0x7FC1).all()
    out, _ = shared(b, q, 16, 0.1, *plan_of(b, most=16), most=16)
    ref, _, tol, _ = kv_ref.attend(t, from_bf16(q).astype(np.float64), 16, 0.1)
    err = np.abs(from_bf16(out).astype(np.float64) - ref)[:t.cu[-1]]
    assert (err <= tol[:t.cu[-1]]).all()


def grown(s, q, Hq, by, window, sinks):
    """The attention of a step by the plan of a step before, when its sequences were `by` tokens shorter."""
    lens = s.lens.copy()
    s.lens = (lens - np.asarray(by)).astype(np.int32)
    c = Cache(s)
    plan, need = plan_of(c)
    _, groups = check_plan(c, plan)
    s.lens = lens
    c.lens.upload(lens)
    got, lse = shared(c, q, Hq, 0.1, plan, need, window, sinks)
    ref, rlse, tol, ltol = kv_ref.attend(s, from_bf16(q).astype(np.float64), Hq, 0.1, window, sinks)
    assert (np.abs(from_bf16(got) - ref) <= tol).all() and (np.abs(lse - rlse) <= ltol).all()
    return groups


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (100, 0), (170, 3), (250, 70), (420, 0), (2 ** 31 - 1, 0)])
@pytest.mark.parametrize("by", [0, 1, 3, 64, 130, [1, 0, 5, 200, 2, 70, 0]])
@pytest.mark.parametrize("D,page,Hq,n", [(64, 16, 4, 1), (128, 64, 16, 3), (256, 32, 2, 1)])
def test_a_plan_kept_while_sequences_grow(window, sinks, by, D, page, Hq, n):
    """The plan of an earlier step of the same rows: what a window hides moves on with the lengths. Windows that end in what the
    sequences share, in what they have for themselves, and that leave nothing of either."""
    rng = np.random.default_rng(window % 1000 + D)
    s, _ = step_of(rng, [(330, [200, 240, 290, 400]), (128, [202, 205])], [450], 2, D, page, n=n)
    assert len(grown(s, randn_bf16(rng, (s.rows, Hq, D)), Hq, by, window, sinks)) == 2


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [700, 2000])
def test_a_long_plan_kept_while_sequences_grow(D, window):
    """Blocks that are cut into parts, the first of which no row sees any more."""
    rng = np.random.default_rng(window + D)
    s, _ = step_of(rng, [(3000, [600, 800, 500])], [1500], 1, D, 64)
    for by in (5, 300, [1, 500, 0, 64]):
        assert len(grown(s, randn_bf16(rng, (s.rows, 4, D)), 4, by, window, 2)) == 1


@pytest.mark.parametrize("B", [40, 1100])
def test_a_cu_that_does_not_ascend_writes_nowhere_else(B):
    """Every other sequence names the same 16 rows: more than the plan's list has room for. Nobody is in a group then, and plan, rows
    and workspace end where they end. The next plan in the same place is right."""
    rng = np.random.default_rng(B)
    s, _ = step_of(rng, [(128, [int(x) for x in rng.integers(0, 30, B)])], [], 1, 64, 64)
    t = kv_ref.Step.__new__(kv_ref.Step)
    t.__dict__.update(s.__dict__, rows=16, lens=s.lens + 15)
    t.cu = (np.arange(B + 1) % 2 * 16).astype(np.int32)
    bad = Cache(t)
    plan, need = plan_of(bad, most=16)
    got = plan.download(16 + 4 * B, np.int32)
    assert got[6:8].tolist() == [0, 0] and (got[16:].reshape(B, 4)[:, 0] == 0).all()
    shared(bad, randn_bf16(rng, (16, 2, 64)), 2, 0.1, plan, need, most=16)
    t.cu = np.minimum(np.arange(B + 1), 16).astype(np.int32)
    t.n = np.diff(t.cu).tolist()
    bad.cu.upload(t.cu)
    call("uh_kv_share", None, bad.cu, 16, 16, bad.lens, bad.table, t.max_blocks, B, t.pages, 64, plan, need, None)
    synchronize()
    check_plan(bad, plan, most=16)


def test_the_same_every_time_and_without_lse():
    rng = np.random.default_rng(11)
    s, _ = step_of(rng, [(2000, [3, 700, 100, 0])], [900], 2, 128, 64)
    c, q = Cache(s), randn_bf16(rng, (s.rows, 8, 128))
    plan, need = plan_of(c)
    first, lse = shared(c, q, 8, 0.1, plan, need)
    for _ in range(3):
        again, l2 = shared(c, q, 8, 0.1, plan, need)
        assert np.array_equal(first, again) and np.array_equal(lse, l2)
    assert np.array_equal(first, shared(c, q, 8, 0.1, plan, need, lse=False)[0])


def test_two_streams_read_one_plan():
    """Layers on two streams at once, a workspace each, behind one plan."""
    rng = np.random.default_rng(22)
    s, _ = step_of(rng, [(1500, [3, 200, 100, 0])], [900], 2, 128, 64)
    c, st = Cache(s), (Stream(), Stream())
    plan, need_plan = plan_of(c)
    q = [randn_bf16(rng, (s.rows, 8, 128)) for _ in st]
    want = [shared(c, x, 8, 0.1, plan, need_plan)[0] for x in q]
    need = call("uh_kv_attend_shared_workspace_size", s.rows, 1, s.B, 8, 2, 128)
    dq, ws, out = [dev(x) for x in q], [dev(np.zeros(need, np.uint8)) for _ in st], [DeviceBuffer(q[0].nbytes) for _ in st]
    synchronize()
    for _ in range(20):
        for t, x, w, o in zip(st, dq, ws, out):
            call("uh_kv_attend_shared", x, 8 * 128, c.cu, s.rows, 1, c.lens, c.table, s.max_blocks, s.B, *c.arrays(), s.pages, s.page, 8,
                 2, 128, 0.1, 0, 0, o, 8 * 128, None, plan, need_plan, w, need, t.handle)
    for t, o, x in zip(st, out, want):
        t.synchronize()
        assert np.array_equal(o.download(x.shape, np.uint16), x)


def test_one_sequence():
    rng = np.random.default_rng(12)
    for n in (1, 20):
        check(kv_ref.Step(rng, [n], [300], 1, 64, 16), 4, expect=0)
        check(wide(kv_ref.Step(rng, [n], [300], 1, 64, 16)), 4, expect=0)


def test_tables_too_wide_for_the_shared_form():
    """A launch sized for 16 rows of each of 2048 sequences, over tables of a million tokens: more segments times tiles than 31 bits
    count. It is kv_attend's, which counts them by sequences."""
    rng = np.random.default_rng(21)
    B, page, Hkv, Hq, D = 2048, 128, 8, 64, 64
    s = kv_ref.Step.__new__(kv_ref.Step)
    s.n, s.B, s.Hkv, s.D, s.page, s.rows, s.max_blocks, s.pages = [1] * B, B, Hkv, D, page, B, 8192, 40
    s.cu, s.lens = np.arange(B + 1, dtype=np.int32), rng.integers(100, 300, B).astype(np.int32)
    s.table = np.full((B, s.max_blocks), -1, np.int32)
    s.table[:, :3] = rng.integers(0, s.pages, (B, 3))
    s.k, s.v = (kv_ref.encode(rng.standard_normal(x) * 64) for x in ((s.pages, Hkv, page, D), (s.pages, Hkv, D, page)))
    s.ks, s.vs = (rng.integers(118, 124, (s.pages, Hkv), dtype=np.uint8) for _ in range(2))
    c, q = Cache(s), randn_bf16(rng, (B, Hq, D))
    plan, need = plan_of(c, most=16)
    got, lse = shared(c, q, Hq, 0.1, plan, need, most=16)
    want, wlse = attend(c, q, Hq, 0.1, max_new=16)
    assert np.array_equal(got, want) and np.array_equal(lse, wlse)


@pytest.mark.parametrize("n", [1, 7])
def test_narrow_tables(n):
    """A step that the other kernels take, in the same workspace."""
    rng = np.random.default_rng(15)
    s, _ = step_of(rng, [(200, [3, 9])], [40], 2, 64, 16, n=n)
    narrow = kv_ref.Step.__new__(kv_ref.Step)
    narrow.__dict__.update(s.__dict__)
    narrow.max_blocks = 20
    narrow.table = np.ascontiguousarray(s.table[:, :20])
    check(narrow, 8, expect=1)
    c, d = Cache(s), Cache(narrow)
    q = randn_bf16(rng, (s.rows, 8, 64))
    need = call("uh_kv_attend_shared_workspace_size", s.rows, n, s.B, 8, 2, 64)
    ws = dev(np.concatenate([np.zeros(need, np.uint8), np.full(64, GUARD, np.uint8)]))
    ref, _, tol, _ = kv_ref.attend(s, from_bf16(q).astype(np.float64), 8, 0.1)
    for x in (c, d, c, d):
        got = shared(x, q, 8, 0.1, *plan_of(x), ws=ws)[0]
        assert (np.abs(from_bf16(got) - ref) <= tol).all()


def test_captured_steps_replay_with_other_tables():
    """The plan and two layers captured once, replayed with other rows, lengths and tables, eager work between; one workspace."""
    rng = np.random.default_rng(13)
    st, Hq, B, rows = Stream(), 8, 6, 8
    steps = []
    for groups, alone, n in (([(300, [0, 9, 40, 100])], [7, 200], [1, 1, 2, 1, 2, 1]), ([(128, [5, 5]), (400, [1, 2, 3])], [50], 1),
                             ([], [300, 0, 10, 500, 64, 70], 1), ([(450, [0, 1, 2, 3, 4, 5])], [], [2, 1, 1, 2, 1, 1])):
        s, _ = step_of(rng, groups, alone, 2, 128, 64, n=n)
        s.rows = rows
        steps.append(s)
    width, pages = max(s.max_blocks for s in steps), max(s.pages for s in steps)  # (wide ones)
    for s in steps:
        s.table = np.concatenate([s.table, np.full((B, width - s.max_blocks), -1, np.int32)], 1)
        extra = pages - s.pages
        s.k, s.v, s.ks, s.vs = (np.concatenate([x, np.zeros((extra,) + x.shape[1:], np.uint8)]) for x in (s.k, s.v, s.ks, s.vs))
        s.max_blocks, s.pages = width, pages
    c = Cache(steps[0])
    need_p = call("uh_kv_share_plan_size", B, rows)
    need = call("uh_kv_attend_shared_workspace_size", rows, 2, B, Hq, 2, 128)
    plan, ws = dev(np.zeros(need_p, np.uint8)), dev(np.zeros(need, np.uint8))
    q, out = [dev(np.zeros((rows, Hq, 128), np.uint16)) for _ in range(2)], [dev(np.zeros((rows, Hq, 128), np.uint16)) for _ in range(2)]

    def work():
        call("uh_kv_share", None, c.cu, rows, 2, c.lens, c.table, width, B, pages, 64, plan, need_p, st.handle)
        for a, b in zip(q, out):
            call("uh_kv_attend_shared", a, Hq * 128, c.cu, rows, 2, c.lens, c.table, width, B, *c.arrays(), pages, 64, Hq, 2, 128,
                 0.09, 0, 0, b, Hq * 128, None, plan, need_p, ws, need, st.handle)

    g = Graph(st, work)
    for s in steps + steps[:2]:
        for buf, a in zip((c.k, c.v, c.ks, c.vs, c.cu, c.lens, c.table), (s.k, s.v, s.ks, s.vs, s.cu, s.lens, s.table)):
            buf.upload(a)
        x = [randn_bf16(rng, (rows, Hq, 128)) for _ in range(2)]
        for a, b, o in zip(q, x, out):
            a.upload(b)
            o.upload(np.full((rows, Hq, 128), 0x7FC1, np.uint16))
        synchronize()
        g.launch()
        st.synchronize()
        c.step = s
        used = int(s.cu[-1])
        for b, o in zip(x, out):
            got = o.download((rows, Hq, 128), np.uint16)
            ref, _, tol, _ = kv_ref.attend(s, from_bf16(b).astype(np.float64), Hq, 0.09)
            assert (np.abs(from_bf16(got[:used]) - ref[:used]) <= tol[:used]).all() and (got[used:] == 0x7FC1).all()
        eager = plan_of(c, most=2)
        shared(c, x[0], Hq, 0.09, *eager, most=2)


def test_after_forks():
    """As an engine makes them: prompts, forks of them, pages for the next tokens, then the plan by the forks' sources."""
    rng = np.random.default_rng(14)
    page, Hkv, Hq, D, B = 16, 2, 8, 64, 7
    p = Pool(rng, [200, 0, 0, 0, 90, 0, 40], 80, page, 20, layers=1, Hkv=Hkv, D=D)
    p.fork([-1, 0, 0, 0, -1, 4, -1])
    assert p.reserve([1, 2, 1, 1, 1, 1, 1]).all()
    s = kv_ref.Step.__new__(kv_ref.Step)
    s.n, s.B, s.Hkv, s.D, s.page, s.pages = [1, 2, 1, 1, 1, 1, 1], B, Hkv, D, page, p.pages
    s.lens, s.table, s.max_blocks = p.lens, p.table, p.table.shape[1]
    s.cu = np.concatenate(([0], np.cumsum(s.n))).astype(np.int32)
    s.rows = int(s.cu[-1])
    shapes = ((p.pages, Hkv, page, D), (p.pages, Hkv, D, page))
    s = wide(s)
    s.k, s.v = (kv_ref.encode(rng.standard_normal(x) * 64) for x in shapes)
    s.ks, s.vs = (rng.integers(118, 124, (p.pages, Hkv), dtype=np.uint8) for _ in range(2))
    check(s, Hq, [0, 0, 0, 0, 4, 4, 6], expect=2)
    check(s, Hq, expect=2)


def test_a_serving_loop():
    """Prompts, forks and decode steps as an engine runs them: pages, norms, rotation and the append in one launch, the plan, the
    attention. The queries and the new keys against 64 bits, the attention against 64 bits over the cache as it is."""
    rng = np.random.default_rng(16)
    page, Hkv, Hq, D, B, rot = 16, 2, 8, 64, 7, 32
    width = int(64e6) // (2 * B * page * Hkv * D) + 1  # tables of what a long context takes
    p = Pool(rng, [0] * B, 200, page, width, layers=1, Hkv=Hkv, D=D)
    p.lazy = True
    freq = rope_ref.frequencies(rot, 10000.0, 2, 8.0, 1.0, 32.0, 4096.0)
    f, w = dev(freq), to_bf16(1 + 0.3 * rng.standard_normal((2, D)))
    dw, heads = [dev(x) for x in w], Hq + 2 * Hkv
    shapes = ((p.pages, Hkv, page, D), (p.pages, Hkv, D, page), (p.pages, Hkv), (p.pages, Hkv))

    def step(n, groups, group=None):
        assert p.reserve(n).all()
        s = kv_ref.Step.__new__(kv_ref.Step)
        s.n, s.B, s.Hkv, s.D, s.page, s.pages, s.lens, s.table, s.max_blocks = list(n), B, Hkv, D, page, p.pages, p.lens, p.table, width
        s.cu = np.concatenate(([0], np.cumsum(n))).astype(np.int32)
        s.rows = int(s.cu[-1])
        c = Cache.__new__(Cache)
        c.step, (c.k, c.v, c.ks, c.vs), c.cu, c.lens, c.table = s, p.caches, dev(s.cu), p.d[1], p.d[0]
        x = randn_bf16(rng, (s.rows, heads, D), 2.0 ** float(rng.integers(-2, 3)))
        qkv, q = dev(x), dev(np.zeros((s.rows, Hq, D), np.uint16))
        k = qkv.ptr + 2 * Hq * D
        call("uh_kv_append_rope", qkv, heads * D, q, Hq * D, Hq, dw[0], k, heads * D, dw[1], 1e-6, k + 2 * Hkv * D, heads * D, c.cu,
             s.rows, max(n), c.lens, c.table, width, B, f, 0, rot, 0, 1.2, *c.arrays(), p.pages, page, Hkv, D, None)
        synchronize()
        s.k, s.v, s.ks, s.vs = (b.download(z, np.uint8) for b, z in zip(p.caches, shapes))
        p.data = [z.reshape(1, p.pages, -1) for z in (s.k, s.v, s.ks, s.vs)]
        pos = np.concatenate([s.position(b, 0) + np.arange(s.n[b]) for b in range(B)])
        got = from_bf16(q.download((s.rows, Hq, D), np.uint16)).astype(np.float64)
        wide_x, wide_w = from_bf16(x).astype(np.float64), from_bf16(w).astype(np.float64)
        ref, tol = rope_ref.norm_rope(wide_x[:, :Hq], wide_w[0], 1e-6, pos, freq, 0, rot, False, 1.2)
        assert (np.abs(got - ref) <= tol).all()
        ref, tol = rope_ref.norm_rope(wide_x[:, Hq:Hq + Hkv], wide_w[1], 1e-6, pos, freq, 0, rot, False, 1.2)
        for b in range(B):
            rows = slice(int(s.cu[b]), int(s.cu[b + 1]))
            unit = 2.0 ** (s.ks[p.table[b, pos[rows] // page]].astype(np.float64) - 127)[..., None]
            off = np.abs(s.gather(b)[0][pos[rows]] - ref[rows])  # half a step of e4m3: 2^-4, of subnormal codes 2^-10 of the scale
            assert (off <= 1.01 * (2.0 ** -4 * np.abs(ref[rows]) + tol[rows] + 2.0 ** -10 * unit)).all()
        plan = plan_of(c, group)
        assert len(check_plan(c, plan[0], group)[1]) == groups
        bits = q.download((s.rows, Hq, D), np.uint16)
        for window, sinks in ((0, 0), (70, 2)):
            out, lse = shared(c, bits, Hq, D ** -0.5, *plan, window, sinks)
            ref, rlse, tol, ltol = kv_ref.attend(s, got, Hq, D ** -0.5, window, sinks)
            assert (np.abs(from_bf16(out) - ref) <= tol).all() and (np.abs(lse - rlse) <= ltol).all()

    step([150, 0, 0, 0, 90, 0, 20], 0)
    p.fork([-1, 0, 0, 0, -1, 4, -1])
    step([1, 1, 3, 1, 1, 1, 1], 2)
    step([1, 1, 1, 5, 2, 1, 1], 2, [0, 0, 0, 0, 4, 4, 6])
    p.free([1 << 20, 1 << 20, 0, 152, 1 << 20, 40, 3])
    p.compact(in_place=True)
    p.fork([-1, -1, 1, -1, -1, -1, -1])
    step([1, 1, 1, 1, 1, 1, 1], 1)
    step([2, 0, 1, 17, 1, 1, 1], 1, [0, 0, 0, 0, -1, -1, -1])
