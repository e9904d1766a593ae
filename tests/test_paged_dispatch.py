"""The paged operators and the draft verification are seen by fake tensors,
dispatch and function modes and the compiler, as the other operators are."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

from test_native_build import built  # noqa: F401  (fixture)

H = torch.float16


def _arguments():
    """Keyword-free argument lists by operator, made in the current mode."""
    dev = dict(device="cuda")
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, **dev)  # noqa: E731
    q, k = torch.zeros(4, 8, 128, dtype=H, **dev), torch.zeros(4, 2, 128, dtype=H, **dev)
    cache = [torch.zeros(9, 2, 16, 128, dtype=H, **dev) for _ in range(2)]
    index = [i32(4, 4), i32(5), i32(4)]
    i64 = lambda: torch.zeros(4, dtype=torch.int64, **dev)  # noqa: E731
    f32 = lambda: torch.zeros(4, **dev)  # noqa: E731
    return {"paged_rope_cache": (q, k, k.clone(), *cache, *index, 1e6),
            "paged_cache_read": (*cache, *index, k, k.clone()),
            "paged_attention": (q, *cache, *index, torch.zeros_like(q), 0.1),
            "verify_draft": (torch.zeros(4, 50, **dev), i64(), None, i32(5), f32(), f32(), i64(), i32(4))}


NAMES = ["paged_rope_cache", "paged_cache_read", "paged_attention", "verify_draft"]


class _Names(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if "persona" in str(func):
            self.names.append(str(func))
            return None
        return func(*args, **(kwargs or {}))  # (a fake tensor's device, say)


class _Functions(TorchFunctionMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_function__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func))
        return None if "persona" in str(func) else func(*args, **(kwargs or {}))


@pytest.mark.parametrize("name", NAMES)
def test_fake_tensors(built, name):  # noqa: F811
    from persona import ops

    with FakeTensorMode():
        getattr(ops, name)(*_arguments()[name])


@pytest.mark.parametrize("name", NAMES)
def test_modes_see_the_call(built, name):  # noqa: F811
    from persona import ops

    with FakeTensorMode():
        args = _arguments()[name]
    with _Names() as seen:
        getattr(ops, name)(*args)
    assert seen.names == [f"persona.{name}.default"]
    with FakeTensorMode(), _Functions() as seen:
        getattr(ops, name)(*args)
    assert any(f"persona.{name}" in n or f"persona::{name}" in n for n in seen.names), seen.names


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_compiled_calls(name):
    """Captured whole, and with the results of the plain calls."""
    from persona import ops

    a, b = _arguments()[name], _arguments()[name]
    for t in (*a, *b):
        if torch.is_tensor(t) and t.dtype == torch.int32 and t.shape == (5,):
            t.copy_(torch.arange(5))
        elif torch.is_tensor(t) and t.dtype == torch.int32 and t.shape == (4,):
            t.fill_(3)
        elif torch.is_tensor(t) and t.dtype == torch.int32:  # a page for each sequence
            t.copy_(torch.arange(4)[:, None].expand(4, 4))
    for x, y in zip(a, b):
        if torch.is_tensor(x) and x.is_floating_point():
            x.uniform_(generator=torch.Generator(device="cuda").manual_seed(x.numel()))
            y.copy_(x)
    getattr(ops, name)(*a)
    torch.compile(lambda *t: getattr(ops, name)(*t), fullgraph=True, backend="eager")(*b)
    ops.check_errors(torch.device("cuda", 0))
    assert all(torch.equal(x, y) for x, y in zip(a, b) if torch.is_tensor(x))
