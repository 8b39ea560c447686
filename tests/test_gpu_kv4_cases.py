"""GPU test of the measured cases of the 4-bit cache (perf/operators.py): a pass through the
framework's calls stands in torch's order, without a synchronisation on either side."""
import importlib.util
import os

import pytest

from common import ROOT

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture
def cases(monkeypatch):
    monkeypatch.chdir(ROOT)
    spec = importlib.util.spec_from_file_location("kv4_cases", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    before = torch.cuda.current_stream()
    yield m
    torch.cuda.synchronize()
    torch.cuda.set_stream(before)


@pytest.mark.parametrize("name", ["decode 0.5B 17 ragged", "decode 1x300", "verify 7B 4x5"])
def test_a_pass_is_in_torchs_order(cases, name):
    """The query is written behind some milliseconds of torch's work, and the output read at
    once: both are seen in order."""
    case = next(c for c in cases.listed() if c["name"] == name)
    s = cases.prepare(case, 3)
    q = s["q"].clone()
    torch.cuda.synchronize()
    want = cases.run(s).clone()
    torch.cuda.synchronize()
    want = want.clone()
    w = torch.randn(4096, 4096, device="cuda")
    s["q"].zero_()
    s["out"].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        w = w @ w
    s["q"].copy_(q)
    got = cases.run(s).clone()
    s["q"].zero_()
    s["out"].zero_()
    torch.cuda.synchronize()
    assert torch.isfinite(want).all() and want.abs().max() > 0
    assert torch.equal(got, want)
