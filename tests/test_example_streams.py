"""The example's order of streams, on the CPU: torch's streams and the library's calls are stand-ins that write down who waits
for whom."""
import contextlib
import importlib.util
import os

import torch

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "moe_decode.py")


def test_the_warm_up_waits_for_what_the_current_stream_makes(monkeypatch):
    spec = importlib.util.spec_from_file_location("moe_decode_streams", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    log, now = [], ["first"]

    class Stream:
        def wait_stream(self, other):
            log.append(("wait", other))

        def synchronize(self):
            log.append(("done", "side"))

    class Graph:
        def replay(self):
            log.append(("replay", now[0]))

    @contextlib.contextmanager
    def on(stream):
        before, now[0] = now[0], "side"
        yield
        now[0] = before

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "graph", lambda graph, stream=None: on(stream))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: now[0])
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: log.append(("all done", now[0])))

    def quantize(x, q=None, s=None, stream=None):
        log.append(("call", now[0]))
        return torch.zeros_like(x, dtype=torch.int8), torch.zeros(len(x))
    monkeypatch.setattr(example.dc, "quantize_i8", quantize)
    for name in ("rms_norm_i8", "mul_mat_i8", "moe_route", "moe_plan", "moe_gate_up_i8", "moe_down_i8"):
        monkeypatch.setattr(example.dc, name, lambda *a, **kw: log.append(("call", now[0])))
    monkeypatch.setattr(example, "reference", lambda layer, x, residual: (x + residual).double() + 1)

    example.main(device="cpu")
    made = log.index(("call", "first"))
    used = log.index(("call", "side"))
    assert made < used and ("wait", "first") in log[made:used]
    # and what replays after the warm-up has its end
    assert ("done", "side") in log[used:log.index(("replay", "first"))]
