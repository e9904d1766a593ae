"""verify_draft where its 32-bit indices, its random numbers and its division of
a sequence among CTAs reach their ends, against the definition on the host."""

import pytest
import torch

import paged_ref as R
from persona import ops
from test_verify_draft_gpu import DEV, _case, _run, _same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("token", [(1 << 32) + 5, -(1 << 32) + 5, (1 << 31) + 5, -1, 50])
def test_a_drafted_token_outside_the_vocabulary_takes_no_weight_from_another(token):
    """Such a token is rejected and was nobody's: every token of the row keeps
    its weight, also the one that the low 32 bits name (5, which has nearly all
    of it in the first sequence)."""
    p, d, _, indptr, ua, us = _case([2, 3], 50, torch.float32, 11)
    p[0] = 0.001
    p[0, 5] = 1
    us[0] = 0.5
    d[0] = d[2] = token
    tokens, acc = _run(p, d, None, indptr, ua * 0, us)
    with pytest.raises(RuntimeError, match="outside the vocabulary"):
        ops.check_errors(torch.device(DEV, 0))
    want, want_a = R.verify(p, d, None, indptr, ua * 0, us)
    assert acc.tolist() == want_a == [0, 0] and tokens.tolist() == want
    assert int(tokens[0]) == 5


@pytest.mark.parametrize("split", [1, 60])  # eight CTAs a sequence, and several sequences a wave
@pytest.mark.parametrize("number", [-1e-30, -0.25, float("-inf"), float("nan"), -0.0])
def test_a_number_below_zero_draws_as_zero_does(number, split):
    """The first token with weight, in every sequence; nothing is left unwritten."""
    p, d, q, indptr, ua, us = _case([2, 1, 3] * split, 3001, torch.float32, 12)
    p[:, :7] = 0  # tokens without weight before the first one with some
    q[:, :7] = 0
    reject = torch.full_like(ua, 1e9)
    for draft in (q, None):
        want, want_a = R.verify(p, d, draft, indptr, reject, us * 0)
        tokens, acc = _run(p, d, draft, indptr, reject, torch.full_like(us, number))
        ops.check_errors(torch.device(DEV, 0))
        assert acc.tolist() == want_a and tokens.tolist() == want


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("B", [74, 75, 100, 149, 200, 297, 400])
def test_every_number_of_ctas_a_sequence(B, dtype):
    """Eight CTAs to one, by the number of sequences, over several tiles a warp."""
    p, d, q, indptr, ua, us = _case([1 + b % 3 for b in range(B)], 5003, dtype, B, pad=1)
    _same(p, d, q, indptr, ua, us)
    _same(p, d, None, indptr, ua * 0.05, us)


@pytest.mark.parametrize("B,V", [(2, 2097152), (75, 1062912), (75, 1062913), (149, 531456), (149, 531457),
                                 (297, 265728), (297, 265729)])
def test_largest_vocabularies_of_each_division(B, V):
    """The most tokens that fewer CTAs a sequence may share, and one more; rows
    start off a 16-byte boundary, so that the tiles are as many as they can be.
    fp16 weights are multiples of 2^-24: sums of them are exact on both sides."""
    g = torch.Generator(device=DEV).manual_seed(V)
    wide = torch.zeros(B, V + 9, dtype=torch.float16, device=DEV)
    p = wide[:, 1:V + 1]
    p.copy_(torch.rand(B, V, device=DEV, generator=g))
    indptr = torch.arange(B + 1, dtype=torch.int32, device=DEV)
    d, ua = torch.zeros(B, dtype=torch.int64, device=DEV), torch.zeros(B, device=DEV)
    us = torch.rand(B, device=DEV, generator=g)
    us[0], us[-1] = 0.0, 1.0  # the ends: the first and the last token with weight
    tokens, acc = _run(p, d, None, indptr, ua, us)
    ops.check_errors(torch.device(DEV, 0))
    assert not acc.any()
    for b in range(B):
        cum = p[b].double().cumsum(0)
        want = int(torch.searchsorted(cum, us[b].double() * cum[-1], right=True))
        assert int(tokens[b]) == (want if want < V else int(p[b].nonzero()[-1])), b
