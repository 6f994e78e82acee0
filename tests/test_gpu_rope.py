"""Rotary positions, the norms before them and both into the paged cache, on the GPU against plain numpy (tests/rope_ref.py),
within bounds that count the roundings; what is one launch against the calls that it stands for, bit for bit."""
from fractions import Fraction

import numpy as np
import pytest

from tests import kv_ref, rope_ref
from tests.helpers import from_bf16, randn_bf16, to_bf16
from tests.test_gpu_kv import Cache, dev, run_append
from unholy_amd import call
from unholy_amd.device import DeviceBuffer, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu

EMPTY = 0x7FC1


class Rows:
    """Rows [rows, heads, dim] on the device with `pad` values between them, `shift` values behind a 16-byte boundary; what is
    not theirs stays as it is."""

    def __init__(self, rows, heads, dim, pad=0, shift=0, data=None):
        self.shape, self.ld, self.shift = (rows, heads, dim), heads * dim + pad, shift
        self.host = np.full(shift + rows * self.ld + 24, EMPTY, np.uint16)
        if data is not None:
            self.view()[:] = data.reshape(rows, -1)
        self.buf = dev(self.host)
        self.ptr = self.buf.ptr + 2 * shift

    def view(self):
        rows, heads, dim = self.shape
        return self.host[self.shift:self.shift + rows * self.ld].reshape(rows, self.ld)[:, :heads * dim]

    def down(self):
        got = self.buf.download(self.host.shape, np.uint16)
        rows, heads, dim = self.shape
        mine = got[self.shift:self.shift + rows * self.ld].reshape(rows, self.ld)[:, :heads * dim].reshape(self.shape).copy()
        rest = got.copy()
        rest[self.shift:self.shift + rows * self.ld].reshape(rows, self.ld)[:, :heads * dim] = EMPTY
        assert (rest == EMPTY).all()
        return mine


def near(got, ref, tol, what=""):
    got = from_bf16(got).astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    fine = np.isfinite(ref)
    err = np.abs(got - ref)[fine]
    print(f"{what} worst error {np.max(err / tol[fine], initial=0):.3f} of bound")
    assert (err <= tol[fine]).all()


def turn(dim, first, rot, interleaved=False, mscale=1.0, base=10000.0):
    f = rope_ref.frequencies(rot, base)
    return f, dev(f), (first, rot, int(interleaved), mscale)


def rope(x, y, pos, f, t, inverse=False, stream=None):
    rows, heads, dim = x.shape
    call("uh_rope", x.ptr, x.ld, y.ptr, y.ld, pos, rows, heads, dim, f, *t, int(inverse), stream)
    synchronize()


SHAPES = [(1, 0, 0), (2, 0, 2), (7, 1, 6), (48, 36, 12), (64, 0, 64), (80, 60, 20), (80, 0, 32), (96, 48, 48), (128, 0, 128),
          (128, 32, 64), (192, 128, 64), (256, 0, 256), (255, 0, 254), (576, 512, 64), (513, 3, 510), (514, 2, 512), (516, 4, 512),
          (1024, 0, 1024), (1023, 1, 2), (1020, 0, 20)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,first,rot", SHAPES)
def test_rope(dim, first, rot, interleaved):
    """Heads of every width that takes another load, some of them rotated in part; few heads and more than a workgroup has."""
    rng = np.random.default_rng(dim + rot)
    f, df, t = turn(dim, first, rot, interleaved, 1.25)
    for rows, heads, pad, inverse in ((1, 1, 0, False), (5, 3, 8, True), (3, 300 if dim < 200 else 9, 5, False)):
        x = randn_bf16(rng, (rows, heads, dim))
        pos = rng.integers(0, 5000, rows).astype(np.int32)
        dx, dy = Rows(rows, heads, dim, pad, data=x), Rows(rows, heads, dim, 2 * pad)
        rope(dx, dy, dev(pos), df, t, inverse)
        got = dy.down()
        ref, tol = rope_ref.rope(from_bf16(x).astype(np.float64), pos, f, first, rot, interleaved, 1.25, inverse)
        near(got, ref, tol, f"rope {dim} {first} {rot}")
        rest = np.ones(dim, bool)
        rest[first:first + rot] = False
        assert np.array_equal(got[..., rest], x[..., rest])
        rope(dx, dx, dev(pos), df, t, inverse)  # in place: the same
        assert np.array_equal(dx.down(), got)


@pytest.mark.parametrize("shift", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("pad", [0, 1, 2, 4])
def test_strides_and_addresses(shift, pad):
    """Whatever loads they allow, the results are the same."""
    rng = np.random.default_rng(shift)
    f, df, t = turn(64, 16, 32)
    x, pos = randn_bf16(rng, (9, 5, 64)), dev(rng.integers(0, 99, 9).astype(np.int32))
    want = Rows(9, 5, 64)
    rope(Rows(9, 5, 64, data=x), want, pos, df, t)
    for a, b in ((shift, 0), (0, shift), (shift, shift)):
        y = Rows(9, 5, 64, 3 * pad, b)
        rope(Rows(9, 5, 64, pad, a, x), y, pos, df, t)
        assert np.array_equal(y.down(), want.down())


def test_far_positions_are_as_exact_as_near_ones():
    rng = np.random.default_rng(4)
    pos = np.array([0, 1, -1, 4095, 131071, 1 << 20, (1 << 24) + 1, 2 ** 31 - 1, -2 ** 31], np.int32)
    x = randn_bf16(rng, (len(pos), 2, 128))
    f, df, t = turn(128, 0, 128, base=500000.0)
    y = Rows(len(pos), 2, 128)
    rope(Rows(len(pos), 2, 128, data=x), y, dev(pos), df, t)
    ref, tol = rope_ref.rope(from_bf16(x).astype(np.float64), pos, f, 0, 128, False)
    near(y.down(), ref, tol, "far")


def exact_turn(pos, freq):
    """Cosine and sine of pos * freq, whole turns cut off in rational numbers (pi to 50 digits)."""
    turn = 2 * Fraction(314159265358979323846264338327950288419716939937511, 10 ** 50)
    angle = [float((p * Fraction(f)) % turn) for p in pos.tolist() for f in freq.tolist()]
    angle = np.array(angle).reshape(len(pos), len(freq))
    return np.cos(angle), np.sin(angle)


@pytest.mark.parametrize("far", [1000, 1 << 24, 1 << 28, 2 ** 31 - 1])
@pytest.mark.parametrize("interleaved", [False, True])
def test_the_error_of_an_angle_does_not_grow_with_the_position(far, interleaved):
    """Pairs that a rotation turns almost onto an axis: a cos - b sin is next to nothing, and shows by how much the factors are
    off. Bounds: each factor is rounded once (2^-25, its sine or cosine and angle another eighth of that), the product b sin
    is (2^-24 of it), the sum is (2^-24), and the result to bf16 (2^-8)."""
    rng = np.random.default_rng(far % 1000)
    rot, rows = 32, 400
    freq = rope_ref.frequencies(rot, 5.0)
    pos = rng.integers(far // 2, far + 1, rows).astype(np.int32)
    pos[::3] *= -1
    c, s = exact_turn(pos, freq)
    a, b = s[:, None], c[:, None]  # (a cos - b sin = 0, before a and b are bf16)
    x = np.stack([a, b], -1).reshape(rows, 1, rot) if interleaved else np.concatenate([a, b], -1)
    x = to_bf16(x.astype(np.float32))
    t = (0, rot, int(interleaved), 1.0)
    y = Rows(rows, 1, rot)
    rope(Rows(rows, 1, rot, data=x), y, dev(pos), dev(freq), t)
    ia, ib = rope_ref.pairs(rot, 0, rot, interleaved)
    wide, got = from_bf16(x).astype(np.float64)[:, 0], from_bf16(y.down()).astype(np.float64)[:, 0]
    for sign, u, v, out in ((-1, c, s, ia), (1, s, c, ib)):
        ref = wide[:, ia] * u + sign * wide[:, ib] * v
        tol = (np.abs(wide[:, ia]) + np.abs(wide[:, ib])) * 2.0 ** -25 * 1.125 + 2.0 ** -24 * (np.abs(wide[:, ib] * v) + np.abs(ref))
        tol += 2.0 ** -8 * np.abs(ref)
        err = np.abs(got[:, out] - ref)
        print(f"far {far} worst error {np.max(err / tol):.3f} of bound")
        assert (err <= tol).all()


def test_turning_back_undoes_it():
    rng = np.random.default_rng(6)
    x, pos = randn_bf16(rng, (40, 3, 64)), dev(rng.integers(0, 1 << 20, 40).astype(np.int32))
    f, df, t = turn(64, 0, 64, True)
    y, z = Rows(40, 3, 64), Rows(40, 3, 64)
    rope(Rows(40, 3, 64, data=x), y, pos, df, t)
    rope(y, z, pos, df, t, inverse=True)
    a = np.abs(from_bf16(x).reshape(40, 3, 32, 2)).sum(-1, keepdims=True).repeat(2, -1).reshape(x.shape)
    assert (np.abs(from_bf16(z.down()) - from_bf16(x)) <= (3 * 2.0 ** -8 + 2.0 ** -18) * a).all()  # three roundings to bf16


def norm_rope(q, k, qo, ko, wq, wk, eps, pos, f, t, stream=None):
    rows, _, dim = q.shape
    call("uh_qk_norm_rope", q.ptr, q.ld, qo.ptr, qo.ld, q.shape[1], wq, k.ptr, k.ld, ko.ptr, ko.ld, k.shape[1], wk, eps, pos,
         rows, dim, f, *t, stream)
    synchronize()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,first,rot", SHAPES)
def test_norm_rope(dim, first, rot, interleaved):
    rng = np.random.default_rng(dim + rot)
    f, df, t = turn(dim, first, rot, interleaved, 0.8)
    wq, wk = to_bf16(1 + 0.3 * rng.standard_normal(dim)), to_bf16(rng.standard_normal(dim))
    for rows, hq, hkv, pad, scale, eps in ((1, 4, 1, 0, 1.0, 1e-6), (6, 7, 3, 8, 2.0 ** -12, 1e-5), (3, 2, 0, 3, 100.0, 0.0),
                                           (2, 0, 40, 1, 1.0, 1e-6)):
        q, k = randn_bf16(rng, (rows, hq, dim), scale), randn_bf16(rng, (rows, hkv, dim), scale)
        pos = rng.integers(0, 5000, rows).astype(np.int32)
        a, b, c, d = Rows(rows, hq, dim, pad, data=q), Rows(rows, hkv, dim, pad, data=k), Rows(rows, hq, dim), Rows(rows, hkv, dim, pad)
        norm_rope(a, b, c, d, dev(wq), dev(wk), eps, dev(pos), df, t)
        for x, w, y in ((q, wq, c), (k, wk, d)):
            ref, tol = rope_ref.norm_rope(from_bf16(x).astype(np.float64), from_bf16(w).astype(np.float64), eps, pos, f, first,
                                          rot, interleaved, 0.8)
            near(y.down(), ref, tol, f"norm_rope {dim} {first} {rot}")
        want = c.down(), d.down()
        norm_rope(a, b, a, b, dev(wq), dev(wk), eps, dev(pos), df, t)  # in place
        assert np.array_equal(a.down(), want[0]) and np.array_equal(b.down(), want[1])


@pytest.mark.parametrize("rows,hq,hkv", [(1000, 5, 1), (1024, 40, 8), (2049, 1, 1), (300, 16, 2), (1500, 33, 0)])
def test_many_rows(rows, hq, hkv):
    """Queries and keys side by side in one projection's rows, in place."""
    rng = np.random.default_rng(rows)
    dim, heads = 128, hq + hkv
    f, df, t = turn(dim, 0, dim)
    x = randn_bf16(rng, (rows, heads, dim))
    wq, wk = to_bf16(1 + 0.3 * rng.standard_normal(dim)), to_bf16(1 + 0.3 * rng.standard_normal(dim))
    pos = np.arange(7, rows + 7, dtype=np.int32)
    b = Rows(rows, heads, dim, data=x)
    call("uh_qk_norm_rope", b.ptr, b.ld, b.ptr, b.ld, hq, dev(wq), b.ptr + 2 * hq * dim, b.ld, b.ptr + 2 * hq * dim, b.ld, hkv,
         dev(wk), 1e-6, dev(pos), rows, dim, df, *t, None)
    synchronize()
    w = np.concatenate((np.repeat(from_bf16(wq)[None], hq, 0), np.repeat(from_bf16(wk)[None], hkv, 0))).astype(np.float64)
    ref, tol = rope_ref.norm_rope(from_bf16(x).astype(np.float64), w, 1e-6, pos, f, 0, dim, False)
    near(b.down(), ref, tol, "many rows")


def test_what_is_no_number_stays_in_its_pair_or_head():
    rng = np.random.default_rng(8)
    x = randn_bf16(rng, (2, 3, 64))
    x[0, 1, 5], x[1, 2, 40] = 0x7FC0, 0x7F80  # NaN, infinity
    pos = dev(np.array([3, 9], np.int32))
    f, df, t = turn(64, 0, 64)
    y = Rows(2, 3, 64)
    rope(Rows(2, 3, 64, data=x), y, pos, df, t)
    bad = np.zeros((2, 3, 64), bool)
    bad[0, 1, [5, 37]] = bad[1, 2, [8, 40]] = True
    assert np.array_equal(~np.isfinite(from_bf16(y.down())), bad)
    w, qo, ko = dev(to_bf16(np.ones(64))), Rows(2, 3, 64), Rows(2, 3, 64)
    norm_rope(Rows(2, 3, 64, data=x), Rows(2, 3, 64, data=randn_bf16(rng, (2, 3, 64))), qo, ko, w, w, 1e-6, pos, df, t)
    got = np.isnan(from_bf16(qo.down()))
    assert got[0, 1].all() and got[1, 2].any() and not np.delete(got.reshape(6, 64), [1, 5], 0).any()
    assert np.isfinite(from_bf16(ko.down())).all()
    zero = Rows(2, 3, 64, data=np.zeros((2, 3, 64), np.uint16))
    norm_rope(zero, zero, qo, ko, w, w, 1e-6, pos, df, t)
    assert (from_bf16(qo.down()) == 0).all()


def test_rows_four_gigabytes_apart():
    rng = np.random.default_rng(9)
    ld, dim, heads = 2 ** 31 - 8, 64, 2
    buf = DeviceBuffer(2 * (ld + heads * dim))
    x, pos = randn_bf16(rng, (2, heads, dim)), np.array([11, 500], np.int32)
    for r in range(2):
        call("uh_memcpy_h2d", buf.ptr + 2 * r * ld, x[r].ctypes.data, x[r].nbytes)
    f, df, t = turn(dim, 0, dim)
    call("uh_rope", buf.ptr, ld, buf.ptr, ld, dev(pos), 2, heads, dim, df, *t, 0, None)
    synchronize()
    got = np.stack([buf.download((heads, dim), np.uint16, 2 * r * ld) for r in range(2)])
    ref, tol = rope_ref.rope(from_bf16(x).astype(np.float64), pos, f, 0, dim, False)
    near(got, ref, tol, "far apart")


# ---- into the cache --------------------------------------------------------------------------------------------------
def positions(s):
    """Of each row; -1 << 20 for rows that no sequence has."""
    p = np.full(s.rows, -1 << 20, np.int32)
    for b in range(s.B):
        p[s.cu[b]:s.cu[b + 1]] = int(s.lens[b]) - s.n[b] + np.arange(s.n[b])
    return p


def append_rope(c, qkv, qo, Hq, wq, wk, f, t, eps=1e-6, max_new=None, stream=None):
    """qkv: Rows of a projection's queries, keys and values."""
    s = c.step
    most = max(s.n + [0]) if max_new is None else max_new
    k = qkv.ptr + 2 * Hq * s.D
    call("uh_kv_append_rope", qkv.ptr if Hq else None, qkv.ld, qo.ptr if Hq else None, qo.ld, Hq, wq, k, qkv.ld, wk, eps,
         k + 2 * s.Hkv * s.D, qkv.ld, c.cu, s.rows, most, c.lens, c.table, s.max_blocks, s.B, f, *t, *c.arrays(), s.pages, s.page,
         s.Hkv, s.D, stream)


def check_append(s, Hq, first, rot, interleaved=False, normed=True, pad=0, seed=0, max_new=None, skip=()):
    """One launch against qk_norm_rope (or rope) and kv_append, bit for bit. skip: sequences whose rows are left alone."""
    rng = np.random.default_rng(seed)
    f, df, t = turn(s.D, first, rot, interleaved, 1.1)
    heads = Hq + 2 * s.Hkv
    x = randn_bf16(rng, (s.rows, heads, s.D), 2.0)
    wq, wk = (dev(to_bf16(1 + 0.3 * rng.standard_normal(s.D))) if normed else None for _ in range(2))
    q, k, v = x[:, :Hq], x[:, Hq:Hq + s.Hkv], x[:, Hq + s.Hkv:]
    qkv, qo, c = Rows(s.rows, heads, s.D, pad, data=x), Rows(s.rows, Hq, s.D, 2 * pad), Cache(s)
    append_rope(c, qkv, qo, Hq, wq, wk, df, t, max_new=max_new)
    synchronize()
    pos = positions(s)
    dq, dk = Rows(s.rows, Hq, s.D, data=q), Rows(s.rows, s.Hkv, s.D, data=k)
    if normed:
        norm_rope(dq, dk, dq, dk, wq, wk, 1e-6, dev(pos), df, t)
    else:
        for r in (dq, dk):
            rope(r, r, dev(pos), df, t)
    want = dq.down()
    want[pos == -1 << 20] = EMPTY
    for b in skip:
        want[s.cu[b]:s.cu[b + 1]] = EMPTY
    assert np.array_equal(qo.down(), want)
    plain = Cache(s)
    run_append(plain, dk.down(), v, max_new=max_new)
    for a, b in zip(c.down(), plain.down()):
        assert np.array_equal(a, b)
    return c, dk.down()


@pytest.mark.parametrize("D,page", [(64, 16), (64, 64), (128, 32), (128, 64), (128, 128), (256, 16), (256, 128)])
@pytest.mark.parametrize("n,ctx", [([1, 1, 1, 1], [0, 3, 63, 200]), ([5, 1, 20], [11, 0, 130]), ([150, 1, 70], [0, 77, 13])])
@pytest.mark.parametrize("interleaved,normed", [(False, True), (True, True), (False, False)])
def test_append_rope(D, page, n, ctx, interleaved, normed):
    rng = np.random.default_rng(D + page + sum(n))
    s = kv_ref.Step(rng, n, ctx, 2, D, page, spare_rows=3)
    check_append(s, 6, 0, D, interleaved, normed)


@pytest.mark.parametrize("first,rot", [(0, 0), (0, 16), (48, 16), (8, 32), (24, 96), (56, 64)])
@pytest.mark.parametrize("Hq,Hkv", [(0, 1), (1, 1), (3, 1), (40, 8)])
def test_append_rope_of_a_part(first, rot, Hq, Hkv):
    rng = np.random.default_rng(rot + Hq)
    s = kv_ref.Step(rng, [1, 4, 33], [5, 70, 0], Hkv, 128, 32)
    check_append(s, Hq, first, rot, pad=8)


@pytest.mark.parametrize("n,ctx", [([1, 1, 1], [0, 63, 200]), ([90, 1, 20], [0, 7, 33])])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("wq,wk", [(True, True), (True, False), (False, True)])
def test_append_rope_in_place(n, ctx, interleaved, wq, wk):
    """Queries rotated where they stand in the projection's rows, beside keys and values that stay; norms of one of the two."""
    rng = np.random.default_rng(sum(n))
    s = kv_ref.Step(rng, n, ctx, 2, 128, 64, spare_rows=2)
    f, df, t = turn(128, 32, 64, interleaved, 1.1)
    w = [dev(to_bf16(1 + 0.3 * rng.standard_normal(128))) if x else None for x in (wq, wk)]
    x = randn_bf16(rng, (s.rows, 9, 128))
    a, qo, b, c, d = Rows(s.rows, 9, 128, 8, data=x), Rows(s.rows, 5, 128), Rows(s.rows, 9, 128, 8, data=x), Cache(s), Cache(s)
    append_rope(c, a, qo, 5, *w, df, t)
    append_rope(d, b, b, 5, *w, df, t)
    synchronize()
    used, got = int(s.cu[-1]), b.down()
    assert np.array_equal(got[:used, :5], qo.down()[:used])
    assert np.array_equal(got[used:], x[used:]) and np.array_equal(got[:, 5:], x[:, 5:]) and np.array_equal(a.down(), x)
    for u, v in zip(c.down(), d.down()):
        assert np.array_equal(u, v)
    pos = positions(s)
    for heads, weight in ((slice(0, 5), w[0]), (slice(5, 7), w[1])):  # each as its own call does it
        one = Rows(s.rows, heads.stop - heads.start, 128, data=x[:, heads])
        if weight is None:
            rope(one, one, dev(pos), df, t)
        else:
            none = Rows(s.rows, 0, 128)
            norm_rope(one, none, one, none, weight, None, 1e-6, dev(pos), df, t)
        if heads.start == 0:
            assert np.array_equal(one.down()[:used], got[:used, :5])
        else:
            run_append(e := Cache(s), one.down(), x[:, 7:])
            for u, v in zip(c.down(), e.down()):
                assert np.array_equal(u, v)


def test_append_rope_against_64_bits():
    """Keys in the cache: the rounding to bf16 (2^-8 and what rope_ref counts), and half a step of e4m3 (2^-4, of subnormal
    codes 2^-10 of the scale)."""
    rng = np.random.default_rng(2)
    s = kv_ref.Step(rng, [100, 1], [0, 64], 2, 128, 64)
    f, df, t = turn(128, 0, 64)
    x, w = randn_bf16(rng, (101, 8, 128)), to_bf16(1 + 0.3 * rng.standard_normal(128))
    c, qo = Cache(s), Rows(101, 4, 128)
    append_rope(c, Rows(101, 8, 128, data=x), qo, 4, dev(w), dev(w), df, t)
    synchronize()
    s.k, s.v, s.ks, s.vs = c.down()
    pos, w = positions(s), from_bf16(w).astype(np.float64)
    ref, tol = rope_ref.norm_rope(from_bf16(x).astype(np.float64), w, 1e-6, pos, f, 0, 64, False)
    near(qo.down(), ref[:, :4], tol[:, :4], "queries")
    for b in range(2):
        k, v, _ = s.gather(b)
        rows = slice(int(s.cu[b]), int(s.cu[b + 1]))
        page = s.table[b, pos[rows] // 64]
        unit = 2.0 ** (s.ks[page].astype(np.float64) - 127)[..., None]
        off = np.abs(k[pos[rows]] - ref[rows, 4:6])
        assert (off <= 1.01 * (2.0 ** -4 * np.abs(ref[rows, 4:6]) + tol[rows, 4:6] + 2.0 ** -10 * unit)).all()


def test_append_rope_rows_that_are_left_alone():
    """Rows behind the last sequence, sequences without rows, with more than the launch is sized for, at negative positions,
    without a page, without a table."""
    rng = np.random.default_rng(3)
    s = kv_ref.Step(rng, [3, 0, 9, 1, 2], [20, 5, 40, 0, 50], 2, 64, 16, spare_rows=4)
    check_append(s, 4, 0, 64, max_new=4, skip=[2])
    s.lens = s.lens.copy()
    s.lens[0] = 1
    s.table[4, 3] = -1
    check_append(s, 4, 0, 64)
    s.table[:] = -1
    check_append(s, 4, 0, 64)
    t = kv_ref.Step(rng, [2, 1], [0, 0], 1, 64, 16)
    t.max_blocks, t.table = 0, np.zeros((2, 0), np.int32)
    check_append(t, 4, 0, 64)


@pytest.mark.parametrize("rows,n,max_new,Hq", [(66000, 1, 1, 2), (140000, 2, 3, 1), (20000, 1, 1, 64), (66000, 70, 70, 2)])
def test_append_rope_with_far_more_rows_than_sequences_have(rows, n, max_new, Hq):
    """Row arrays of a large batch for a sequence of it."""
    rng = np.random.default_rng(rows)
    check_append(kv_ref.Step(rng, [n], [5], 1, 64, 16, spare_rows=rows), Hq, 0, 64, max_new=max_new)


@pytest.mark.parametrize("B", [65, 200])
def test_append_rope_of_many_sequences(B):
    rng = np.random.default_rng(B)
    n = rng.integers(0, 3, B).tolist()
    check_append(kv_ref.Step(rng, n, rng.integers(0, 60, B).tolist(), 1, 64, 32, spare_rows=2), 3, 0, 32)


def test_captured_steps_replay_at_other_positions():
    """Rotation, norms and the append captured once, replayed with other rows and lengths between eager calls."""
    rng = np.random.default_rng(12)
    s = kv_ref.Step(rng, [1, 2], [100, 30], 2, 128, 64, spare_blocks=2)
    st, Hq = Stream(), 4
    f, df, t = turn(128, 0, 128)
    w = dev(to_bf16(1 + 0.3 * rng.standard_normal(128)))
    c, plain = Cache(s), Cache(s)
    qkv, qo, pos = Rows(3, Hq + 4, 128, data=randn_bf16(rng, (3, Hq + 4, 128))), Rows(3, Hq, 128), dev(np.zeros(3, np.int32))
    y = Rows(3, Hq + 4, 128)

    def work():
        append_rope(c, qkv, qo, Hq, w, w, df, t, stream=st.handle)
        call("uh_rope", qkv.ptr, qkv.ld, y.ptr, y.ld, pos, 3, Hq + 4, 128, df, *t, 0, st.handle)

    g = Graph(st, work)
    for i in range(4):
        x = randn_bf16(rng, (3, Hq + 4, 128), 2.0 ** i)
        s.lens = np.array([101 + 3 * i, 32 + i], np.int32)
        p = positions(s)
        for buf, a in ((qkv.buf, np.concatenate((x.reshape(-1), np.full(24, EMPTY, np.uint16)))), (pos, p), (c.lens, s.lens),
                       (plain.lens, s.lens)):
            buf.upload(a)
        synchronize()
        g.launch()
        st.synchronize()
        a, b = Rows(3, Hq, 128), Rows(3, Hq + 4, 128)
        append_rope(plain, qkv, a, Hq, w, w, df, t)
        rope(qkv, b, pos, df, t)
        assert np.array_equal(a.down(), qo.down()) and np.array_equal(b.down(), y.down())
        for u, v in zip(c.down(), plain.down()):
            assert np.array_equal(u, v)
