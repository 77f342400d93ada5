"""perf/operators.py: the calls that its cases make through the package."""

import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")


def load():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")
    spec = importlib.util.spec_from_file_location("measured_cases", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_a_handle_for_each_device_and_stream(monkeypatch):
    """The calls queue where the caller's other work is queued at that moment, not where the first call found it."""
    from types import SimpleNamespace as Object

    from harp_amd import backend
    opened = []
    monkeypatch.setattr(backend, "HipDevice", lambda index, stream: opened.append((index, stream)) or (index, stream))
    cases, handles = load(), []
    for index, stream in ((0, 0), (0, 64), (1, 64), (0, 0), (1, 64)):
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i, s=stream: s, raising=False)
        handles.append(cases._device(Object(get_device=lambda i=index: i)))
    assert handles == [(0, 0), (0, 64), (1, 64), (0, 0), (1, 64)]
    assert opened == [(0, 0), (0, 64), (1, 64)]


@pytest.mark.gpu
def test_a_case_on_streams_of_its_own():
    """Behind work that is still under way on the same stream: nothing runs ahead of its inputs."""
    from harp_amd import backend as hb
    if hb.device_count() == 0:
        pytest.skip("no HIP device")
    cases = load()
    cases.own = True
    case = {"op": "score", "rows": 4, "vocab": 1000, "dtype": "f32", "top": 3, "masked": 0, "scale": 1.0}
    state = cases.prepare(case, 1)
    want = {k: v.clone() for k, v in cases.run(state).items()}
    torch.cuda.synchronize()
    logits = state["logits"].clone()
    big = torch.randn(4096, 4096, device="cuda")
    for _ in range(2):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            state["logits"].zero_()
            y = big
            for _ in range(20):
                y = (y @ big).mul_(1e-3)
            state["logits"].copy_(logits + 0.0 * y.flatten()[:4000].view(4, 1000).nan_to_num(0.0, 0.0, 0.0))
            got = {k: v.clone() for k, v in cases.run(state).items()}
        stream.synchronize()
        for k, v in want.items():
            assert torch.equal(got[k], v), k
