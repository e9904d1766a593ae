"""CPU checks of step planning, block scales and sampling: statuses of the C
entry points (no call gets past its checks), and what modes and fake tensors
see."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from test_native_build import built  # noqa: F401  (fixture)
from test_paged import FAKE, _attend, _cache as _kv, lib  # noqa: F401
from test_paged_dispatch import _Names

OK, INVALID, SHAPE, DTYPE, ALIGN, OVERLAP = 0, 1, 2, 3, 4, 9
FAR = 1 << 40


def _p(i):
    """Places far from each other, never touched."""
    return FAR + (i << 30)


def _plan(lib, **change):  # noqa: F811
    a = dict(add=_p(0), keep=None, lengths=_p(1), B=4, table=_p(2), stride=8, width=8, free=_p(3), pool=32, num=_p(4),
             page=16, indptr=_p(5), places=_p(6), seq=None, row=None, rows=9)
    a.update(change)
    return lib.persona_paged_plan(a["add"], a["keep"], a["lengths"], a["B"], a["table"], a["stride"], a["width"], a["free"],
                                  a["pool"], a["num"], a["page"], a["indptr"], a["places"], a["seq"], a["row"], a["rows"],
                                  None, None)


@pytest.fixture(scope="module")
def step(lib):  # noqa: F811
    import ctypes

    p, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
    lib.persona_paged_plan.restype = lib.persona_sample_tokens.restype = i32
    lib.persona_paged_plan.argtypes = [p, p, p, i64, p, i64, i64, p, i64, p, i64, p, p, p, p, i64, p, p]
    lib.persona_sample_tokens.argtypes = [p, i64, i32, p, p, p, p, p, p, i64, i64, p]
    return lib


@pytest.mark.parametrize("change,want", [
    (dict(B=-1), SHAPE), (dict(B=8193), SHAPE), (dict(rows=-1), SHAPE), (dict(rows=2147483647), SHAPE),
    (dict(width=-1), SHAPE), (dict(stride=7), SHAPE), (dict(pool=-1), SHAPE), (dict(pool=2147483647), SHAPE),
    (dict(page=0), SHAPE), (dict(page=1 << 31), SHAPE), (dict(num=None), INVALID), (dict(indptr=None), INVALID),
    (dict(add=None), INVALID), (dict(lengths=None), INVALID), (dict(table=None), INVALID), (dict(free=None), INVALID),
    (dict(places=None), INVALID), (dict(row=_p(7)), INVALID), (dict(add=_p(0) + 2), ALIGN), (dict(places=_p(6) + 4), ALIGN),
    (dict(keep=_p(7) + 1), ALIGN), (dict(keep=_p(1)), OVERLAP), (dict(add=_p(1) + 12), OVERLAP),
    (dict(free=_p(2) + 4 * 31), OVERLAP), (dict(indptr=_p(6) + 8), OVERLAP), (dict(num=_p(3) + 4 * 31), OVERLAP),
    (dict(seq=_p(7), row=_p(6) + 64), OVERLAP), (dict(seq=_p(7), row=_p(7)), OVERLAP), (dict(num=_p(5) + 16), OVERLAP),
    (dict(lengths=_p(2) + 4 * 30), OVERLAP)])
def test_plan_statuses(step, change, want):
    assert _plan(step, **change) == want


def _sample(lib, **change):  # noqa: F811
    a = dict(x=_p(0), ld=100, type=0, u=_p(1), t=None, k=None, p=None, m=None, tokens=_p(2), B=4, V=100)
    a.update(change)
    return lib.persona_sample_tokens(a["x"], a["ld"], a["type"], a["u"], a["t"], a["k"], a["p"], a["m"], a["tokens"], a["B"],
                                     a["V"], None)


@pytest.mark.parametrize("change,want", [
    (dict(type=3), DTYPE), (dict(type=-1), DTYPE), (dict(B=-1), SHAPE), (dict(V=0), SHAPE), (dict(V=2097153, ld=2097153), SHAPE),
    (dict(ld=-1), SHAPE), (dict(B=1 << 30), SHAPE), (dict(x=None), INVALID), (dict(u=None), INVALID),
    (dict(tokens=None), INVALID), (dict(x=_p(0) + 1), ALIGN), (dict(x=_p(0) + 2, type=2), ALIGN), (dict(tokens=_p(2) + 4), ALIGN),
    (dict(t=_p(3) + 2), ALIGN), (dict(k=_p(3) + 1), ALIGN), (dict(tokens=_p(1) + 8), OVERLAP), (dict(tokens=_p(0) + 792), OVERLAP),
    (dict(t=_p(2)), OVERLAP), (dict(k=_p(2) + 28), OVERLAP), (dict(p=_p(2)), OVERLAP), (dict(m=_p(2) + 16), OVERLAP),
    (dict(B=0, x=None, u=None, tokens=None), OK)])
def test_sample_statuses(step, change, want):
    assert _sample(step, **change) == want


def test_block_scale_statuses(lib):  # noqa: F811
    kind = lambda n: 1 | n << 8  # noqa: E731  (PERSONA_PAGES_E4M3_BLOCK)
    with_scales = dict(k_scale=FAKE, v_scale=FAKE)
    for n, page, want in ((8, 256, DTYPE), (-1, 16, DTYPE), (5, 16, SHAPE), (4, 24, SHAPE), (7, 64, SHAPE)):
        assert _attend(lib, _kv(kind=kind(n), page_size=page, **with_scales)) == want, (n, page)
    assert _attend(lib, _kv(kind=kind(4))) == INVALID          # no scales
    assert _attend(lib, _kv(kind=2 | 4 << 8, **with_scales)) == DTYPE
    assert _attend(lib, _kv(kind=4 << 8)) == DTYPE             # blocks of 16-bit pages
    assert _attend(lib, _kv(kind=kind(4), **with_scales), ws=None) == 6  # gets to the workspace


def _arguments():
    dev = dict(device="cuda")
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, **dev)  # noqa: E731
    return {"paged_plan": (i32(4), i32(4), i32(4, 3), i32(12), i32(1), 16, i32(5), torch.zeros(7, dtype=torch.int64, **dev)),
            "sample_tokens": (torch.zeros(4, 50, **dev), torch.zeros(4, **dev), torch.zeros(4, dtype=torch.int64, **dev))}


@pytest.mark.parametrize("name", ["paged_plan", "sample_tokens"])
def test_modes_and_fake_tensors(built, name):  # noqa: F811
    from persona import ops

    with FakeTensorMode():
        args = _arguments()[name]
        getattr(ops, name)(*args)
    with _Names() as seen:
        getattr(ops, name)(*args)
    assert seen.names == [f"persona.{name}.default"]


def test_cpu_tensors_are_refused(built):  # noqa: F811
    from persona import ops

    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ops.paged_plan(i32(2), i32(2), i32(2, 2), i32(4), i32(1), 16, i32(3), torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="must be CUDA"):
        ops.sample_tokens(torch.zeros(2, 9), torch.zeros(2), torch.zeros(2, dtype=torch.int64))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["paged_plan", "sample_tokens"])
def test_compiled_calls(name):
    """Captured whole, and with the results of the plain calls."""
    from persona import ops

    a, b = _arguments()[name], _arguments()[name]
    for args in (a, b):
        if name == "paged_plan":
            args[0].fill_(1)
            args[3].copy_(torch.arange(12))
            args[4].fill_(12)
        else:
            args[0].uniform_(generator=torch.Generator(device="cuda").manual_seed(1))
            args[1].fill_(0.5)
    getattr(ops, name)(*a)
    torch.compile(lambda *t: getattr(ops, name)(*t), fullgraph=True, backend="eager")(*b)
    ops.check_errors(torch.device("cuda", 0))
    assert all(torch.equal(x, y) for x, y in zip(a, b) if torch.is_tensor(x))
    assert int(a[-1].sum()) != 0  # it did something
