"""verify_draft on the GPU against the definition on the host, token for token."""

import pytest
import torch

import paged_ref as R
from persona import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _run(p, d, q, indptr, ua, us):
    tokens = torch.full((p.shape[0],), 77, dtype=torch.int64, device=DEV)
    acc = torch.full((indptr.numel() - 1,), 77, dtype=torch.int32, device=DEV)
    ops.verify_draft(p, d, q, indptr, ua, us, tokens, acc)
    return tokens, acc


def _same(p, d, q, indptr, ua, us):
    tokens, acc = _run(p, d, q, indptr, ua, us)
    ops.check_errors(torch.device(DEV, 0))
    want, want_a = R.verify(p, d, q, indptr, ua, us)
    assert acc.tolist() == want_a
    assert tokens.tolist() == [77 if t is None else t for t in want]
    return acc


def _case(new, V, dtype, seed, pad=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows = sum(new) + pad
    z = torch.randn(rows, V, device=DEV, generator=g) * 2
    p = torch.softmax(z, -1)
    q = torch.softmax(z + 0.5 * torch.randn(rows, V, device=DEV, generator=g), -1)
    d = torch.multinomial(q, 1, generator=g)[:, 0]
    indptr = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    return (p.to(dtype), d, q.to(dtype), indptr, torch.rand(rows, device=DEV, generator=g),
            torch.rand(len(new), device=DEV, generator=g))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,V", [([1], 1), ([5] * 8, 32000), ([3, 0, 1, 8, 2, 40], 257), ([4] * 30, 50257),
                                   ([2, 3], 7), ([100], 50), ([6] * 5, 2048), ([2], 300001)])
def test_matches_the_definition(new, V, dtype):
    p, d, q, indptr, ua, us = _case(new, V, dtype, 3 + V, pad=2)
    a = _same(p, d, q, indptr, ua, us)
    b = _same(p, d, None, indptr, ua * 0.05, us)
    if len(new) > 7 and V > 1000:
        assert int(a.max()) > 0 and int(a.min()) < 4 and b is not None


def test_all_kept_all_rejected_and_ends_of_the_number():
    p, d, q, indptr, ua, us = _case([5] * 6, 1000, torch.float32, 1)
    assert _same(p, d, q, indptr, ua * 0, us).tolist() == [4] * 6
    big = torch.full_like(ua, 1e9)
    assert _same(p, d, q, indptr, big, us).tolist() == [0] * 6
    _same(p, d, q, indptr, ua, us * 0)                    # the first token with weight
    _same(p, d, q, indptr, big, torch.ones_like(us))      # a number of one: the last with weight
    one = torch.nextafter(torch.ones_like(us), torch.zeros_like(us))
    _same(p, d, q, indptr, big, one)


def test_weights_of_nothing():
    """p equal to q: the residual is empty and p itself is drawn from; a row
    without a positive weight draws no token; NaN and negative ones count as none."""
    p, d, q, indptr, ua, us = _case([3, 3, 2], 500, torch.float32, 2)
    _same(p, d, p.clone(), indptr, torch.full_like(ua, 2.0), us)
    p0 = p.clone()
    p0[0] = 0
    p0[3, ::2] = float("nan")
    p0[4, 5:] = -1
    _same(p0, d, q, indptr, torch.full_like(ua, 2.0), us)
    z = torch.zeros(1, 9, device=DEV)
    t, a = _run(z, d[:1], None, torch.tensor([0, 1], dtype=torch.int32, device=DEV), ua[:1], us[:1])
    assert t.tolist() == [-1] and a.tolist() == [0]


def test_single_tokens_and_strided_rows():
    """A draft that was certain of its token never draws it again; rows inside a wider buffer."""
    V = 333
    p, d, q, indptr, ua, us = _case([4] * 9, V, torch.float16, 5)
    wide = torch.zeros(p.shape[0], V + 7, dtype=p.dtype, device=DEV)
    wide[:, :V] = p
    wq = torch.zeros(p.shape[0], V + 30, dtype=p.dtype, device=DEV)
    wq[:, :V] = q
    acc = _same(wide[:, :V], d, wq[:, :V], indptr, ua, us)
    tokens, acc = _run(p, d, None, indptr, torch.full_like(ua, 2.0), us)
    first = indptr[:-1].long()
    assert acc.tolist() == [0] * 9 and not (tokens[first] == d[first]).any()


def test_frequencies():
    """Over many sequences the token behind no drafts follows p, and the first
    token of drafted ones does too (the point of the rule).  8192 draws: the
    bound is six standard deviations of a frequency."""
    g = torch.Generator(device=DEV).manual_seed(9)
    B, V = 8192, 11
    p1 = torch.softmax(torch.randn(V, device=DEV, generator=g), -1)
    q1 = torch.softmax(torch.randn(V, device=DEV, generator=g), -1)
    p, q = p1.expand(2 * B, V).contiguous(), q1.expand(2 * B, V).contiguous()
    d = torch.multinomial(q, 1, generator=g)[:, 0]
    indptr = torch.arange(0, 2 * B + 1, 2, dtype=torch.int32, device=DEV)
    tokens, acc = _run(p, d, q, indptr, torch.rand(2 * B, device=DEV, generator=g), torch.rand(B, device=DEV, generator=g))
    freq = torch.bincount(tokens[::2], minlength=V).double() / B
    assert torch.all((freq - p1).abs() <= 6 * (p1 * (1 - p1) / B).sqrt())


def test_bad_tokens_and_rows_are_flagged():
    p, d, q, indptr, ua, us = _case([3, 3], 100, torch.float32, 4)
    d[0] = 100
    tokens, acc = _run(p, d, q, indptr, ua * 0, us)
    with pytest.raises(RuntimeError, match="outside the vocabulary"):
        ops.check_errors(torch.device(DEV, 0))
    assert acc.tolist() == [0, 2]
    indptr[2] = 7
    tokens, acc = _run(p, d.clamp_max(99), q, indptr, ua * 0, us)
    with pytest.raises(RuntimeError, match="segment"):
        ops.check_errors(torch.device(DEV, 0))
    assert acc.tolist() == [2, 0] and torch.all(tokens[3:] == 77)


def test_captured():
    p, d, q, indptr, ua, us = _case([5] * 4, 3000, torch.float32, 6)
    tokens = torch.zeros(20, dtype=torch.int64, device=DEV)
    acc = torch.zeros(4, dtype=torch.int32, device=DEV)
    ops.verify_draft(p, d, q, indptr, ua, us, tokens, acc)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.verify_draft(p, d, q, indptr, ua, us, tokens, acc)
    for i in range(3):
        us.copy_(torch.rand(4, device=DEV))
        ua.copy_(torch.rand(20, device=DEV))
        g.replay()
        want, want_a = R.verify(p, d, q, indptr, ua, us)
        assert tokens.tolist() == want and acc.tolist() == want_a


def test_tokens_over_the_drafts_are_refused():
    p, d, q, indptr, ua, us = _case([3, 2], 50, torch.float32, 8)
    acc = torch.zeros(2, dtype=torch.int32, device=DEV)
    both = torch.cat([d, d])
    for tokens in (both[:5], both[1:6]):
        with pytest.raises(RuntimeError, match="must not overlap draft_tokens"):
            ops.verify_draft(p, both[:5], q, indptr, ua, us, tokens, acc)
    tokens, _ = ops.verify_draft(p, both[:5], q, indptr, ua, us, both[5:], acc)
    want, want_a = R.verify(p, d, q, indptr, ua, us)
    assert tokens.tolist() == want and acc.tolist() == want_a


@pytest.mark.parametrize("scale", [2.0 ** -20, 2.0 ** -3, 0.3, 1.0, 40.0, 60000.0])
@pytest.mark.parametrize("drafts", ["none", "certain", "given"])
def test_fp16_weights_of_any_size(scale, drafts):
    """Unnormalised fp16 weights, from subnormals to its largest values, whose
    sums of eight lie below, around and above 1.  Both sides sum them exactly
    (multiples of 2^-24 below 2^29), so the tokens are the same."""
    V, n = 5003, 4
    g = torch.Generator(device=DEV).manual_seed(31)
    p, q = ((torch.rand(n * 12, V, device=DEV, generator=g) * scale).half() for _ in range(2))
    p[:, ::97] = 2.0 ** -24
    p[5, 4000:4008] = 1.0
    d = torch.randint(0, V, (n * 12,), device=DEV, generator=g)
    new = [1] * 48 if drafts == "none" else [n] * 12
    indptr = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    ua = torch.full((n * 12,), 0.9, device=DEV)
    us = torch.rand(len(new), device=DEV, generator=g)
    _same(p, d, q if drafts == "given" else None, indptr, ua, us)
