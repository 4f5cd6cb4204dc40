"""The framework's calls on tensors of torch's: the engine has a stream of its own, so torch's is waited for first."""
import importlib.util
import os
import random

import pytest
import torch

import gorgonia_b200

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Recorder:
    """An engine that notes the names of its calls, and a stream that notes its waits."""

    def __init__(self, calls):
        self.calls = calls

    def __getattr__(self, name):
        return lambda *args, **kw: self.calls.append(name)


@pytest.fixture()
def operators(monkeypatch):
    spec = importlib.util.spec_from_file_location("operator_cases", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    m.calls = []
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Recorder(m.calls))
    monkeypatch.setattr(gorgonia_b200, "Engine", lambda *a, **kw: Recorder(m.calls))
    return m


def state(m, kind):
    case = next(c for c in m.listed() if c["kind"] == kind)
    f8, f32, i64 = torch.float8_e4m3fn, torch.float32, torch.int64
    names = {"quantize": {"x": f32, "q": f8, "scales": f32},
             "matmul": {"a": f8, "a_scales": f32, "b": f8, "b_scales": f32, "c": f32},
             "logprobs": dict({n: f32 for n in ("x", "logp", "entropy", "lse", "top_logp")}, targets=i64, top_index=i64),
             "diff": dict({n: f32 for n in ("x", "lse", "entropy", "grad_logp", "grad_entropy", "dx")}, targets=i64)}[kind]
    case = {**case, "format": "e4m3", "block": "row"}
    s = {n: torch.zeros((128, 1) if "scales" in n else (128, 128)).to(t) for n, t in names.items()}
    if kind == "matmul":
        case.update(a_block="row", b_block="row", layer=False)
        s["bias"] = None
    return {**s, "case": case}


@pytest.mark.parametrize("kind", ["quantize", "matmul", "logprobs", "diff"])
def test_inputs_are_waited_for_once(operators, kind):
    s = state(operators, kind)
    operators.run(s)
    assert operators.calls[0] == "synchronize" and len(operators.calls) == 2
    operators.run(s)
    assert operators.calls.count("synchronize") == 1 and len(operators.calls) == 3
    operators.run(state(operators, kind))        # another state: other inputs
    assert operators.calls.count("synchronize") == 2 and operators.calls[-2] == "synchronize"


def test_drawn_cases_are_of_the_listed_kinds(operators):
    kinds = {c["kind"] for c in operators.listed()}
    r = random.Random(5)
    assert {operators.draw(r)["kind"] for _ in range(200)} == kinds
