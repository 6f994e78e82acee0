"""Rotary positions without a GPU: frequencies, the reference itself, and what the entry points refuse."""
import numpy as np
import pytest

from tests import rope_ref
from unholy_amd import UhError, _lib, call


def frequencies(rot, base, scaling=0, factor=1.0, low=1.0, high=32.0, trained=1.0):
    f = np.full(rot // 2 + 1, 7.0)
    call("uh_rope_frequencies", f.ctypes.data, rot, base, scaling, factor, low, high, trained)
    assert f[-1] == 7.0
    return f[:-1]


@pytest.mark.parametrize("rot", [0, 2, 6, 64, 128, 512])
@pytest.mark.parametrize("base", [1.5, 10000.0, 5e6])
@pytest.mark.parametrize("scaling,factor,low,high,trained", [(0, 9.0, 0, 0, 0), (1, 1.0, 0, 0, 0), (1, 8.0, 0, 0, 0),
                                                             (2, 8.0, 1, 4, 8192), (2, 40.0, 1, 32, 4096), (3, 40.0, 1, 32, 4096),
                                                             (3, 4.0, 1, 32, 10), (3, 2.0, 1e-9, 1e9, 4096), (2, 3.0, 0.5, 1, 1e-3)])
def test_frequencies(rot, base, scaling, factor, low, high, trained):
    """Within a few roundings of 64 bits: an exponential of a product, then three operations."""
    got, want = (f(rot, base, scaling, factor, low, high, trained) for f in (frequencies, rope_ref.frequencies))
    assert (np.abs(got - want) <= 64 * 2.0 ** -53 * want).all()


@pytest.mark.parametrize("bad", [{"rot": 3}, {"rot": -2}, {"base": 1.0}, {"base": 0.0}, {"base": float("nan")}, {"base": float("inf")},
                                 {"scaling": 4}, {"scaling": -1}, {"scaling": 1, "factor": 0.5}, {"scaling": 1, "factor": float("nan")},
                                 {"scaling": 2, "trained": 0.0}, {"scaling": 2, "low": 32.0}, {"scaling": 3, "low": 0.0},
                                 {"scaling": 3, "high": float("inf")}, {"scaling": 2, "trained": float("nan")}])
def test_frequencies_refused(bad):
    args = {"rot": 4, "base": 1e4, "scaling": 0, "factor": 2.0, "low": 1.0, "high": 32.0, "trained": 4096.0, **bad}
    with pytest.raises(UhError, match="rope_frequencies"):
        call("uh_rope_frequencies", np.zeros(8).ctypes.data, *args.values())
    with pytest.raises(UhError, match="null"):
        call("uh_rope_frequencies", None, 4, 1e4, 0, 1.0, 0.0, 0.0, 0.0)


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_inverse_is_the_gradient(interleaved):
    """The reference's transpose against differences of its rotation (which is linear: exact but for roundings)."""
    rng = np.random.default_rng(0)
    dim, first, rot, pos = 10, 2, 6, np.array([5, -3])
    f = rope_ref.frequencies(rot, 100.0)
    x, g = rng.standard_normal((2, 2, 1, dim))
    grad, _ = rope_ref.rope(g, pos, f, first, rot, interleaved, 1.3, inverse=True)
    for r in range(2):
        for d in range(dim):
            h = np.zeros_like(x)
            h[r, 0, d] = 0.5
            up, down = (rope_ref.rope(x + e, pos, f, first, rot, interleaved, 1.3)[0] for e in (h, -h))
            assert abs(((up - down) * g).sum() - grad[r, 0, d]) < 1e-13


P = 16  # an address that nothing reads: every call here is refused, or has nothing to do, before the device is touched
ROPE = {"x": P, "ldx": 64, "y": 4096, "ldy": 64, "pos": P, "rows": 2, "heads": 2, "dim": 32, "freq": P, "first": 0, "rot": 32,
        "interleaved": 0, "mscale": 1.0, "inverse": 0, "stream": None}
NORM = {"q": P, "ldq": 64, "qo": 4096, "ldqo": 64, "Hq": 2, "wq": P, "k": P, "ldk": 32, "ko": 4096, "ldko": 32, "Hkv": 1,
        "wk": P, "eps": 1e-6, "pos": P, "rows": 2, "dim": 32, "freq": P, "first": 0, "rot": 32, "interleaved": 0, "mscale": 1.0,
        "stream": None}
APPEND = {"q": P, "ldq": 256, "qo": 4096, "ldqo": 256, "Hq": 4, "wq": P, "k": P, "ldk": 128, "wk": P, "eps": 1e-6, "v": P,
          "ldv": 128, "cu": P, "rows": 3, "max_new": 2, "lens": P, "table": P, "max_blocks": 4, "B": 2, "freq": P, "first": 0,
          "rot": 64, "interleaved": 0, "mscale": 1.0, "kc": P, "vc": P, "ks": P, "vs": P, "pages": 9, "page": 16, "Hkv": 2,
          "D": 64, "stream": None}
CALLS = {"uh_rope": ROPE, "uh_qk_norm_rope": NORM, "uh_kv_append_rope": APPEND}


@pytest.mark.parametrize("name,bad,message", [
    ("uh_rope", {"rows": -1}, "rows"), ("uh_rope", {"heads": -1}, "heads"), ("uh_rope", {"heads": 65536, "ldx": 1 << 30}, "heads"),
    ("uh_rope", {"dim": 0}, "dim"), ("uh_rope", {"dim": 1025}, "dim"), ("uh_rope", {"rot": 31}, "rot even"),
    ("uh_rope", {"rot": -2}, "rot even"), ("uh_rope", {"rot": 34}, "rot even"), ("uh_rope", {"first": 2}, "rot even"),
    ("uh_rope", {"first": -2, "rot": 2}, "rot even"), ("uh_rope", {"first": 2 ** 31 - 1, "rot": 2}, "rot even"),
    ("uh_rope", {"freq": None}, "frequencies"), ("uh_rope", {"freq": 20}, "aligned"), ("uh_rope", {"mscale": float("nan")}, "mscale"),
    ("uh_rope", {"mscale": float("inf")}, "mscale"), ("uh_rope", {"x": None}, "null"), ("uh_rope", {"y": None}, "null"),
    ("uh_rope", {"pos": None}, "positions"), ("uh_rope", {"pos": 18}, "aligned"), ("uh_rope", {"x": 17}, "aligned"),
    ("uh_rope", {"y": 4097}, "aligned"), ("uh_rope", {"ldx": 63}, "strides"), ("uh_rope", {"ldy": 63}, "strides"),
    ("uh_rope", {"y": P, "ldy": 72}, "in place"),
    ("uh_qk_norm_rope", {"wq": None}, "null"), ("uh_qk_norm_rope", {"wk": None}, "null"), ("uh_qk_norm_rope", {"ko": None}, "null"),
    ("uh_qk_norm_rope", {"eps": -1e-9}, "eps"), ("uh_qk_norm_rope", {"eps": float("nan")}, "eps"),
    ("uh_qk_norm_rope", {"eps": float("inf")}, "eps"), ("uh_qk_norm_rope", {"ldk": 31}, "strides"),
    ("uh_qk_norm_rope", {"ldqo": 60}, "strides"), ("uh_qk_norm_rope", {"wk": 19}, "aligned"), ("uh_qk_norm_rope", {"Hkv": -1}, "heads"),
    ("uh_qk_norm_rope", {"rot": 33}, "rot even"), ("uh_qk_norm_rope", {"ko": P, "ldko": 40}, "in place"),
    ("uh_kv_append_rope", {"rot": 8}, "rot % 16"), ("uh_kv_append_rope", {"first": 4, "rot": 16}, "rot % 16"),
    ("uh_kv_append_rope", {"rot": 80}, "rot even"), ("uh_kv_append_rope", {"freq": None}, "frequencies"),
    ("uh_kv_append_rope", {"D": 96}, "dim"), ("uh_kv_append_rope", {"page": 8}, "page"), ("uh_kv_append_rope", {"k": None}, "null"),
    ("uh_kv_append_rope", {"v": None}, "null"), ("uh_kv_append_rope", {"q": None}, "null"), ("uh_kv_append_rope", {"qo": None}, "null"),
    ("uh_kv_append_rope", {"ldq": 248}, "ldq"), ("uh_kv_append_rope", {"ldqo": 257}, "ldq"), ("uh_kv_append_rope", {"ldk": 120}, "ldk"),
    ("uh_kv_append_rope", {"q": 18}, "aligned"), ("uh_kv_append_rope", {"wq": 18}, "aligned"), ("uh_kv_append_rope", {"k": 24}, "aligned"),
    ("uh_kv_append_rope", {"Hq": -1}, "Hq"), ("uh_kv_append_rope", {"Hq": 65536}, "Hq"), ("uh_kv_append_rope", {"eps": -1.0}, "eps"),
    ("uh_kv_append_rope", {"qo": P, "ldqo": 264}, "in place"), ("uh_kv_append_rope", {"cu": None}, "null"),
    ("uh_kv_append_rope", {"B": -1}, "negative"), ("uh_kv_append_rope", {"max_blocks": 1 << 24}, "max_blocks")])
def test_refusals(name, bad, message):
    args = {**CALLS[name], **bad}
    with pytest.raises(UhError, match=message):
        call(name, *args.values())


@pytest.mark.parametrize("name,none", [("uh_rope", {"rows": 0, "x": None, "pos": None}), ("uh_rope", {"heads": 0, "x": None}),
                                       ("uh_rope", {"y": P, "rot": 0, "freq": None}), ("uh_qk_norm_rope", {"rows": 0}),
                                       ("uh_qk_norm_rope", {"Hq": 0, "Hkv": 0, "q": None}), ("uh_kv_append_rope", {"B": 0}),
                                       ("uh_kv_append_rope", {"rows": 0, "k": None}), ("uh_kv_append_rope", {"max_new": 0})])
def test_nothing_to_do(name, none):
    """Nothing is launched (there is no device here to launch on)."""
    assert getattr(_lib.lib(), name)(*{**CALLS[name], **none}.values()) == 0, _lib.last_error()
