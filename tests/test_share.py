"""Attention of sequences that begin alike without a GPU: what the entry points refuse, and what needs no launch."""
import pytest

from unholy_amd import UhError, _lib, call

P = 16
SHARE = {"group": None, "cu": P, "rows": 3, "max_new": 2, "lens": P, "table": P, "max_blocks": 4, "B": 2, "pages": 9, "page": 16,
         "plan": P, "plan_bytes": 1 << 20, "stream": None}
ATTEND = {"q": P, "ldq": 256, "cu": P, "rows": 3, "max_new": 2, "lens": P, "table": P, "max_blocks": 4, "B": 2, "kc": P, "vc": P,
          "ks": P, "vs": P, "pages": 9, "page": 16, "Hq": 4, "Hkv": 2, "D": 64, "scale": 0.1, "window": 0, "sinks": 0, "out": P,
          "ldo": 256, "lse": None, "plan": P, "plan_bytes": 1 << 20, "ws": P, "ws_bytes": 1 << 30, "stream": None}
CALLS = {"uh_kv_share": SHARE, "uh_kv_attend_shared": ATTEND}


@pytest.mark.parametrize("name,bad,message", [
    ("uh_kv_share", {"page": 24}, "page"), ("uh_kv_share", {"pages": 0}, "pages"), ("uh_kv_share", {"B": -1}, "negative"),
    ("uh_kv_share", {"rows": -1}, "negative"), ("uh_kv_share", {"max_new": -1}, "negative"), ("uh_kv_share", {"B": (1 << 24) + 1}, "B >"),
    ("uh_kv_share", {"max_blocks": 1 << 24}, "max_blocks"), ("uh_kv_share", {"cu": None}, "null"), ("uh_kv_share", {"lens": None}, "null"),
    ("uh_kv_share", {"table": None}, "null"), ("uh_kv_share", {"plan": None}, "null plan"), ("uh_kv_share", {"plan": 24}, "aligned"),
    ("uh_kv_share", {"plan_bytes": 63}, "too small"),
    ("uh_kv_attend_shared", {"plan": None}, "null plan"), ("uh_kv_attend_shared", {"plan": 8}, "plan not"),
    ("uh_kv_attend_shared", {"plan_bytes": 63}, "too small"), ("uh_kv_attend_shared", {"ws": None}, "null workspace"),
    ("uh_kv_attend_shared", {"ws": 24}, "workspace not"), ("uh_kv_attend_shared", {"ws_bytes": 100}, "workspace of"),
    ("uh_kv_attend_shared", {"Hq": 3}, "Hq"), ("uh_kv_attend_shared", {"Hq": 0}, "Hq"), ("uh_kv_attend_shared", {"D": 96}, "dim"),
    ("uh_kv_attend_shared", {"Hkv": 0}, "heads"), ("uh_kv_attend_shared", {"page": 8}, "page"),
    ("uh_kv_attend_shared", {"scale": float("nan")}, "scale"), ("uh_kv_attend_shared", {"sinks": -1}, "sinks"),
    ("uh_kv_attend_shared", {"q": None}, "null"), ("uh_kv_attend_shared", {"out": None}, "null"), ("uh_kv_attend_shared", {"q": 24}, "aligned"),
    ("uh_kv_attend_shared", {"ldq": 255}, "ldq"), ("uh_kv_attend_shared", {"ldo": 248}, "ldq"), ("uh_kv_attend_shared", {"kc": 8}, "cache"),
    ("uh_kv_attend_shared", {"rows": 1 << 30, "max_new": 1, "plan_bytes": 1 << 60, "ws_bytes": 1 << 60}, "31 bits"),
    ("uh_kv_attend_shared", {"B": 1 << 23, "max_blocks": 1 << 20, "plan_bytes": 1 << 60, "ws_bytes": 1 << 60}, "31 bits")])
def test_refusals(name, bad, message):
    with pytest.raises(UhError, match=message):
        call(name, *{**CALLS[name], **bad}.values())


@pytest.mark.parametrize("name", ["uh_kv_share", "uh_kv_attend_shared"])
@pytest.mark.parametrize("none", [{"B": 0}, {"rows": 0}, {"max_new": 0}])
def test_nothing_to_do(name, none):
    assert getattr(_lib.lib(), name)(*{**CALLS[name], **none}.values()) == 0, _lib.last_error()


def test_sizes():
    """Workspaces serve both forms of the attention; sizes that make no sense have none."""
    for rows, most, B, hq, hkv, d in ((1, 1, 1, 1, 1, 64), (64, 1, 64, 32, 8, 128), (120, 5, 24, 32, 4, 128), (3000, 2000, 7, 96, 8, 256)):
        a = call("uh_kv_attend_workspace_size", rows, most, B, hq, hkv, d)
        assert call("uh_kv_attend_shared_workspace_size", rows, most, B, hq, hkv, d) >= a > 0
    assert call("uh_kv_attend_shared_workspace_size", -1, 1, 1, 1, 1, 64) == 0
    assert call("uh_kv_share_plan_size", -1, 1) == 0 and call("uh_kv_share_plan_size", 1, -1) == 0
    assert call("uh_kv_share_plan_size", 64, 64) < 1 << 14
