"""The calls that the measured cases (perf/operators.py) make of the kernels."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["gn_8x8x256", "rotary_step_b8", "attn_77_causal"])
def test_calls_follow_the_current_stream(name, monkeypatch):
    """A state that ran once on the default stream runs again inside a capture
    on another: its launches belong to the graph."""
    import torch
    import perf.operators as cases
    monkeypatch.setattr(cases, "own", True)
    case = next(c for c in cases.listed() if c["name"] == name)
    state = cases.prepare(case, 1)
    out = cases.run(state)
    out = out["o"] if isinstance(out, dict) else out
    want = out.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        cases.run(state)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
