"""perf/operators.py calls the library on the stream and the device that are current at each call,
wherever the process stands."""
import importlib.util
import os
import sys
import types

import pytest

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load():
    spec = importlib.util.spec_from_file_location("operators_file", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_the_handle_follows_stream_and_device(monkeypatch, tmp_path):
    """Against a fake of the package: one handle a (device, stream), made once."""
    made = []

    class Device:
        def __init__(self, ordinal):
            self.ordinal = ordinal

        def wrap_stream(self, raw):
            made.append((self.ordinal, raw))
            return (self.ordinal, raw)

    fake = types.ModuleType("qgemm")
    fake.Device = Device
    fake.QuantizedGemmOps = lambda st: types.SimpleNamespace(stream=st)
    for i, n in enumerate(("ACT_NONE", "ACT_RELU", "ACT_GELU", "ACT_GELU_TANH", "ACT_SILU", "F32", "BF16")):
        setattr(fake, n, i)
    monkeypatch.setitem(sys.modules, "qgemm", fake)
    now = [0, 11]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: types.SimpleNamespace(cuda_stream=now[1]))
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: now[1], raising=False)
    monkeypatch.chdir(tmp_path)
    m = load()
    for device, stream in ((0, 11), (0, 12), (0, 11), (1, 11), (1, 11), (0, 12)):
        now[:] = [device, stream]
        assert m._ops()[0].stream == (device, stream)
    assert made == [(0, 11), (0, 12), (1, 11)]


@pytest.mark.gpu
def test_a_case_on_two_streams_and_captured():
    m = load()
    case = {"op": "dispatch", "type": "bf16", "quantize": True, "T": 300, "E": 8, "k": 2, "K": 4096}
    s = m.prepare(case, 1)
    torch.cuda.synchronize()
    m.own = False
    want = {k: v.clone() for k, v in m.run(s).items()}
    m.own = True
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (torch.cuda.current_stream(), side, torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            s["q"].zero_()
            s["sq"].zero_()
            got = m.run(s)
        stream.synchronize()
        for k, v in want.items():
            assert torch.equal(got[k], v), k
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = m.run(s)
    for seed in (2, 3):
        t = m.prepare(case, seed)
        for k in ("x", "rows"):
            s[k].copy_(t[k])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        m.own = False
        want = m.run(t)
        m.own = True
        for k, v in want.items():
            assert torch.equal(got[k], v), k
    del graph
