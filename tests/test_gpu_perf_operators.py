"""The framework's calls of the performance cases (perf/operators.py): prepared states do not share what
a call writes."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SMALL = {"op": "delta", "seqs": 2, "rows_lo": 40, "rows_hi": 70, "hk": 2, "hv": 4, "dk": 64, "dv": 64, "checkpoints": False}
LARGE = dict(SMALL, seqs=4, rows_lo=1000, rows_hi=3000, hk=8, hv=16)
ATTEND = {"op": "attend", "format": "bf16", "seqs": 1, "rows_lo": 1, "rows_hi": 1, "ctx_lo": 4001, "ctx_hi": 4001,
          "page": 64, "hq": 16, "hkv": 2, "dim": 256}


@pytest.fixture()
def operators(q38, monkeypatch):
    monkeypatch.chdir(ROOT)
    spec = importlib.util.spec_from_file_location("perf_operators", os.path.join(ROOT, "perf", "operators.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.own = True
    return mod


def copy(result):
    return {k: v.clone() for k, v in result.items()}


@pytest.mark.parametrize("case", [SMALL, ATTEND])
def test_a_graph_outlives_larger_cases(operators, case):
    """A pass is captured, larger cases run and memory of the sizes that they might free is written over: the
    replays give the eager pass's bits."""
    s = operators.prepare(case, 1)
    want = copy(operators.run(s))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        operators._own(s)
    for i in range(3):
        operators.run(operators.prepare(LARGE, i))
        held = [torch.full((n,), 0xff, dtype=torch.uint8, device="cuda") for n in (1 << 20, 1 << 20, 1 << 21, 1 << 24)]
        s["out"].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(bool((h == 0xff).all()) for h in held), "a replay wrote into another allocation"
        assert torch.equal(s["out"], want["out"])


@pytest.mark.parametrize("cases", [(SMALL, LARGE), (ATTEND, ATTEND), (LARGE, ATTEND)])
def test_states_on_streams_of_their_own(operators, cases):
    states = [operators.prepare(c, i) for i, c in enumerate(cases)]
    want = [copy(operators.run(s)) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(4):
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                operators._own(s)
    torch.cuda.synchronize()
    for s, w in zip(states, want):
        assert torch.equal(s["out"], w["out"])
