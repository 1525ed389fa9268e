"""When a PagedAttentionPlan's own workspace is cleared: before the plan can be
run from any stream or graph, or, for a plan made inside a capture, by whichever
run comes first.  The GPU is stood in for: what is asked of it is written down."""
from types import SimpleNamespace

import pytest
import torch

from zoomkv_revision_amd import paged


@pytest.fixture
def device(monkeypatch):
    """A stand-in device: `log` has what was done, `capturing` is set by the test."""
    d = SimpleNamespace(capturing=False, log=[])
    stub = SimpleNamespace(zkv_paged_attention_workspace_size=lambda n: 4096, zkv_paged_attention=None)
    stream = SimpleNamespace(synchronize=lambda: d.log.append("synchronize"))
    monkeypatch.setattr(paged, "lib", lambda: stub)
    monkeypatch.setattr(paged, "_capturing", lambda device: d.capturing)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: stream)
    monkeypatch.setattr(paged, "_attention_args", lambda *a, copies: (a, "out", a))

    def launch(fn, device, args):
        workspace = args[-1]
        assert d.capturing or not bool(workspace[:1024].any()), "an eager run on counts that are not clear"
        d.log.append("captured run" if d.capturing else "run")

    monkeypatch.setattr(paged, "_launch", launch)
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: empty(*a, **k).fill_(0xAB))     # whatever was there before
    return d


def _plan():
    q = SimpleNamespace(is_cuda=True, shape=(1, 1, 8, 128), device=torch.device("cpu"))
    return paged.PagedAttentionPlan(q, None, None, None, None)


def test_a_plan_is_clear_once_it_is_made(device):
    plan = _plan()
    assert device.log == ["synchronize"]
    device.capturing = True            # a first run that is captured, on whatever stream
    plan.run()
    device.capturing = False
    plan.run()                         # an eager one behind it
    assert device.log == ["synchronize", "captured run", "run"]


def test_a_plan_made_in_a_capture_clears_its_counts_wherever_it_runs_first(device):
    device.capturing = True
    plan = _plan()
    counts = plan._counts
    assert device.log == [] and bool(counts.all())         # nothing ran
    for _ in range(2):
        counts.fill_(7)                                    # (the graph's own clearing comes before the run's node)
        plan.run()
        assert not bool(counts.any())
    counts.fill_(7)
    device.capturing = False
    plan.run()                                             # eager, before any replay
    plan.run()
    counts.fill_(7)
    device.capturing = True
    plan.run()                                             # a later capture relies on what the eager run left
    assert bool(counts.all()) and device.log == ["captured run"] * 2 + ["run"] * 2 + ["captured run"]
