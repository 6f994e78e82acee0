"""The calls that perf/operators.py makes of the library: a step runs on torch's current stream, whether call by call or
replayed, in order with what writes its inputs and reads its results."""
import pathlib
import subprocess
import sys
import types

import pytest

torch = pytest.importorskip("torch")

SMALL = {"Hkv": 1, "D": 64, "page": 16, "layers": 2, "B": 2, "n": 1, "chunk": 0, "ctx_lo": 3, "ctx_hi": 9, "graph": True}


@pytest.mark.parametrize("op", ["attend", "append"])
@pytest.mark.parametrize("graph", [True, False])
def test_steps_are_launched_on_the_current_stream(monkeypatch, op, graph):
    """Three steps of a state, with the library's calls written down and not made."""
    import unholy_amd
    import unholy_amd.device
    from perf import operators

    now, other, seen, capturing = 0x70, 0x90, [], []

    class Stream:
        handle = other

    class Graph:
        handle = 0x50

        def __init__(self, stream, work):
            self.stream = stream
            capturing.append(True)
            work()
            capturing.pop()

        def launch(self):
            seen.append(("replay", self.stream.handle))

    def call(name, *args):
        if capturing:
            assert args[-1] == other
        else:
            seen.append(("replay" if name == "uh_graph_launch" else "call", args[-1]))

    monkeypatch.setattr(unholy_amd, "call", call)
    monkeypatch.setattr(unholy_amd.device, "Stream", Stream)
    monkeypatch.setattr(unholy_amd.device, "Graph", Graph)
    monkeypatch.setattr(operators, "_stream", None)
    monkeypatch.setattr(operators, "own", True)
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda: types.SimpleNamespace(cuda_stream=now, synchronize=lambda: None))
    case = {**SMALL, "op": op, "graph": graph, "Hq": 2, "window": 0, "sinks": 0}
    byte, half = (lambda *n: torch.zeros(n, dtype=torch.uint8)), (lambda *n: torch.zeros(n, dtype=torch.bfloat16))
    state = {"case": case, "graph": None, "pages": 4, "rows": 2, "most": 1, "cu": byte(3), "lens": byte(2),
             "table": byte(2, 2), "cache": {f: byte(2, 4, 1) for f in ("k", "v", "ks", "vs")}, "q": half(2, 2, 2, 64),
             "out": half(2, 2, 2, 64), "ws": byte(8), "knew": half(2, 2, 1, 64), "vnew": half(2, 2, 1, 64)}
    for _ in range(3):
        operators.run(state)
    once = [("call", now)] * case["layers"]
    assert seen == (once + [("replay", now)] * 2 if graph else once * 3)


ORDER = """
import torch
from perf import operators as o
x = torch.randn(4096, 4096, device="cuda")
for stream in (torch.cuda.default_stream(), torch.cuda.Stream()):
    with torch.cuda.stream(stream):
        for graph in (True, False):
            s = o.prepare({"op": "attend", "B": 3, "n": 1, "chunk": 0, "ctx_lo": 40, "ctx_hi": 300, "Hq": 8, "Hkv": 2,
                           "D": 64, "page": 16, "window": 0, "sinks": 0, "layers": 2, "graph": graph}, 1)
            for i in range(4):
                for _ in range(20):  # the stream is busy for a while; then come new rows, the step and a copy of its result
                    y = x @ x
                s["q"].copy_(torch.randn(s["q"].shape, device="cuda"))
                o.own = True
                got = o.run(s).clone()
                o.own = False
                want = o.run(s)
                # roundings to bf16, 2^-8 each, of the weights and of both outputs, where values are up to 448 2^-5
                assert (got.float() - want.float()).abs().max() <= 3.01 * 14 / 256, (graph, i)
                assert got.abs().max() > 0
torch.cuda.synchronize()
print("in order")
"""


@pytest.mark.gpu
def test_steps_run_in_order_with_torch():
    """Rows written by torch just before a step, and results read by torch just after it, without a wait of the host. (In a
    process of its own, where torch comes first and the library takes torch's HIP runtime.)"""
    done = subprocess.run([sys.executable, "-u", "-c", ORDER], cwd=pathlib.Path(__file__).resolve().parents[1],
                          capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "in order" in done.stdout, done.stderr[-2000:]
