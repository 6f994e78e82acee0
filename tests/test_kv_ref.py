"""The paged cache on the CPU: what its calls refuse before they touch a device, and the plain reference that the GPU tests
compare with against simpler definitions."""
import numpy as np
import pytest

from tests import kv_ref
from unholy_amd import _lib

P = 4096  # an aligned address that nothing reads

APPEND = dict(k=P, ldk=1024, v=P, ldv=1024, cu=P, rows=4, max_new=2, lens=P, table=P, max_blocks=8, B=3, kc=P, vc=P, ks=P,
              vs=P, pages=16, page=64, Hkv=8, D=128, stream=None)
ATTEND = dict(q=P, ldq=4096, cu=P, rows=4, max_new=2, lens=P, table=P, max_blocks=8, B=3, kc=P, vc=P, ks=P, vs=P, pages=16,
              page=64, Hq=32, Hkv=8, D=128, scale=0.1, window=0, sinks=0, out=P, ldo=4096, lse=None, ws=P,
              ws_bytes=1 << 40, stream=None)
RESERVE = dict(table=P, max_blocks=8, lens=P, grow=P, B=3, refs=P, kc=P, vc=P, ks=P, vs=P, layers=2, pages=16, page=64,
               Hkv=8, D=128, ok=P, ws=P, ws_bytes=1 << 30, stream=None)
FORK = dict(table=P, max_blocks=8, lens=P, src=P, B=3, refs=P, pages=16, page=64, done=P, stream=None)
FREE = dict(table=P, max_blocks=8, lens=P, keep=P, B=3, refs=P, pages=16, page=64, stream=None)
COMPACT = dict(table=P, table_out=P, max_blocks=8, B=3, refs=P, refs_out=P, kc=P, vc=P, ks=P, vs=P, layers=2, pages=16,
               page=64, Hkv=8, D=128, live=P, ws=P, ws_bytes=1 << 30, stream=None)
CALLS = {"uh_kv_append": APPEND, "uh_kv_attend": ATTEND, "uh_kv_reserve": RESERVE, "uh_kv_fork": FORK,
         "uh_kv_free": FREE, "uh_kv_compact": COMPACT}

REFUSED = (
    [(c, {"page": p}, "page must be") for c in CALLS for p in (0, 8, 48, 256)]
    + [(c, {"pages": n}, "pages must be") for c in CALLS for n in (0, -1, (1 << 28) + 1)]
    + [(c, {"D": d}, "dim must be") for c in CALLS if "D" in CALLS[c] for d in (0, 96, 512)]
    + [(c, {"Hkv": 0, "Hq": 0} if "Hq" in CALLS[c] else {"Hkv": 0}, "heads must be") for c in CALLS if "Hkv" in CALLS[c]]
    + [(c, {f: None}, "null operand") for c in CALLS for f in ("kc", "vc", "ks", "vs", "lens", "table", "refs", "refs_out",
                                                               "table_out", "k", "v", "q", "out", "cu", "grow", "src",
                                                               "keep", "ok", "done") if f in CALLS[c]]
    + [(c, {f: P + 8}, "aligned") for c in CALLS for f in ("kc", "vc", "k", "v", "q", "out", "ws") if f in CALLS[c]]
    + [(c, {f: -1}, "negative") for c in CALLS for f in ("B", "rows", "max_new", "max_blocks") if f in CALLS[c]]
    + [(c, {"max_blocks": (1 << 24) + 1}, "max_blocks") for c in CALLS]
    + [(c, {"layers": 0}, "layers") for c in ("uh_kv_reserve", "uh_kv_compact")]
    + [(c, {"ws_bytes": 8}, "workspace") for c in CALLS if "ws" in CALLS[c]]
    + [(c, {"ws": None}, "null workspace") for c in CALLS if "ws" in CALLS[c]]
    + [("uh_kv_append", {f: n}, "ldk / ldv") for f in ("ldk", "ldv") for n in (1016, 1028, 0)]
    + [("uh_kv_attend", {f: n}, "ldq / ldo") for f in ("ldq", "ldo") for n in (4088, 4100, 0)]
    + [("uh_kv_attend", {"Hq": n}, "Hq must be") for n in (0, 12, -8, 1 << 16)]
    + [("uh_kv_attend", {"rows": (1 << 31) // 32, "max_new": 5}, "rows * Hq")]
    + [("uh_kv_attend", {"B": 1 << 20, "max_blocks": 1 << 12}, "31 bits")]
    + [("uh_kv_attend", {"B": 1, "Hkv": 1, "rows": 1 << 14, "max_new": 1 << 14, "max_blocks": 1 << 23, "ws_bytes": 1 << 40},
        "31 bits")]
    + [("uh_kv_attend", {"sinks": -1}, "sinks"), ("uh_kv_attend", {"scale": float("nan")}, "scale"),
       ("uh_kv_attend", {"scale": float("inf")}, "scale")]
)


@pytest.mark.parametrize("name,wrong,msg", REFUSED, ids=lambda x: str(x).replace("uh_kv_", ""))
def test_refusals(name, wrong, msg):
    args = {**CALLS[name], **wrong}
    assert list(args) == list(CALLS[name])
    rc = getattr(_lib.lib(), name)(*args.values())
    assert rc == -1 and msg in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("name,none", [("uh_kv_append", {"B": 0}), ("uh_kv_append", {"rows": 0, "k": None, "v": None}),
                                       ("uh_kv_append", {"max_new": 0}), ("uh_kv_append", {"max_blocks": 0, "table": None}),
                                       ("uh_kv_attend", {"B": 0}), ("uh_kv_attend", {"rows": 0, "q": None, "out": None}),
                                       ("uh_kv_attend", {"max_new": 0}), ("uh_kv_reserve", {"B": 0}),
                                       ("uh_kv_fork", {"B": 0}), ("uh_kv_free", {"B": 0})])
def test_nothing_to_do(name, none):
    """A step without sequences or rows launches nothing (there is no device here to launch on)."""
    assert getattr(_lib.lib(), name)(*{**CALLS[name], **none}.values()) == 0, _lib.last_error()


def test_codes_round_to_nearest_even():
    fine = np.flatnonzero((np.arange(256) & 127) != kv_ref.NAN)
    assert np.array_equal(kv_ref.encode(kv_ref.E4M3[fine]), np.where(fine == 128, 128, fine))
    for a, b in zip(range(0, 126), range(1, 127)):
        x, y = kv_ref.E4M3[a], kv_ref.E4M3[b]
        mid = (x + y) / 2
        assert kv_ref.encode(mid) == (a if a % 2 == 0 else b)
        assert kv_ref.encode(np.nextafter(mid, 0)) == a and kv_ref.encode(np.nextafter(mid, 1e9)) == b
    assert kv_ref.encode(1e30) == 126 and kv_ref.encode(-np.inf) == 254 and kv_ref.encode(np.nan) == kv_ref.NAN


@pytest.mark.parametrize("amax", [0.0, 1e-4, 1.75, 1.7500001, 448.0, 449.0, 3.0e38])
def test_scale_is_the_smallest_power_of_two(amax):
    e = int(kv_ref.scale_byte(amax)) - 127
    a = max(amax, float(np.float32(1e-4)))
    assert e == 119 or a <= 448 * 2.0 ** e
    assert a > 448 * 2.0 ** (e - 1)


def test_reserve_serves_in_order():
    """Four free pages; a copy of a shared last page counts as one; the first sequence that does not fit ends the service,
    but for those that need no page."""
    table = np.array([[0, -1, -1], [0, -1, -1], [1, -1, -1], [2, 3, -1], [4, -1, -1]], np.int32)
    lens = np.array([10, 10, 16, 20, 5], np.int32)
    refs = np.array([2, 1, 1, 1, 1, 0, 0, 0, 0], np.int32)
    t, n, r, ok, copies = kv_ref.reserve(table, lens, refs, [1, 0, 32, 17, 11], 16)
    assert ok.tolist() == [1, 1, 1, 1, 1] and copies == [(0, 5)]
    assert t.tolist() == [[5, -1, -1], [0, -1, -1], [1, 6, 7], [2, 3, 8], [4, -1, -1]]
    t, n, r, ok, copies = kv_ref.reserve(table, lens, refs, [30, 1, 32, 17, 11], 16)
    assert ok.tolist() == [1, 1, 0, 0, 1] and copies == [(0, 5), (0, 8)]
    assert r.tolist() == [0, 1, 1, 1, 1, 1, 1, 1, 1] and n.tolist() == [40, 11, 16, 20, 16]


def test_compact_moves_the_high_pages_down():
    table = np.array([[7, 2, -1], [7, 5, 4]], np.int32)
    t, r, moves, live = kv_ref.compact(table, np.array([0, 0, 1, 0, 1, 1, 0, 2], np.int32))
    assert live == 4 and moves == [(4, 0), (5, 1), (7, 3)]
    assert t.tolist() == [[3, 2, -1], [3, 1, 0]] and r.tolist() == [1, 1, 1, 2, 0, 0, 0, 0]
