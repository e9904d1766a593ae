"""Steps and generations of a model run with its device as the current one,
whichever is current at the call: graphs are captured, and events recorded, on
the current device's streams.  On the host, with the devices faked."""

import pytest
import torch

from persona import ops
from persona.engine import StaticBatchEngine
from persona.mistral import MistralLoRAModel


class _Reached(Exception):
    pass


@pytest.fixture
def current(monkeypatch):
    """The devices made current, innermost last."""
    stack = []

    class device:
        def __init__(self, d):
            self.d = d

        def __enter__(self):
            stack.append(self.d)

        def __exit__(self, *a):
            stack.pop()

    monkeypatch.setattr(torch.cuda, "device", device)
    return stack


def _reach(current):
    def call(*args, **kwargs):
        raise _Reached(list(current))

    return call


@pytest.mark.parametrize("use_graph", [True, False])
@pytest.mark.parametrize("name", ["decode_step", "paged_step"])
def test_steps(current, monkeypatch, name, use_graph):
    model = MistralLoRAModel.__new__(MistralLoRAModel)
    model.device = torch.device("cuda", 1)
    monkeypatch.setattr(ops, "check_errors", lambda *a, **k: None)
    monkeypatch.setattr(model, "_decode_body", _reach(current), raising=False)
    monkeypatch.setattr(model, "_paged_step", _reach(current), raising=False)

    class State:
        graph = type("Graph", (), {"replay": staticmethod(_reach(current))})

    state = State()
    state.st = type("St", (), {"decode": state})
    with pytest.raises(_Reached) as at:
        getattr(model, name)(state, use_graph=use_graph)
    assert at.value.args[0] == [torch.device("cuda", 1)] and current == []


@pytest.mark.parametrize("name", ["run_static_generate", "run_ragged_generate"])
def test_generations(current, monkeypatch, name):
    eng = StaticBatchEngine.__new__(StaticBatchEngine)
    eng.device = torch.device("cuda", 1)
    monkeypatch.setattr(eng, "plan_batch", _reach(current), raising=False)
    with pytest.raises(_Reached) as at:
        getattr(eng, name)([])
    assert at.value.args[0] == [torch.device("cuda", 1)] and current == []
