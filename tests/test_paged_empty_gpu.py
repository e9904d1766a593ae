"""Batches without sequences, without rows, and page tables without columns:
nothing to do, and nothing refused."""

import pytest
import torch

import paged_ref as R
from persona import ops

pytestmark = pytest.mark.gpu
H = torch.float16


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32, device="cuda")


def _call_all(bt, table, indptr, lengths, rows):
    """Every operator on `rows` rows, none of them a sequence's; what they
    write stays as it was but for attention's rows of a sequence (zeros)."""
    q, k = bt.randn(rows, 8, 128), bt.randn(rows, 2, 128)
    kv = (bt.k_cache, bt.v_cache, table, indptr, lengths)
    before = bt.k_cache.clone()
    q_out, ko, vo, out = torch.full_like(q, 3.0), torch.full_like(k, 3.0), torch.full_like(k, 3.0), torch.full_like(q, 3.0)
    ops.paged_rope_cache(q, k, k, *kv, 1e6, q_out=q_out, **bt.scales())
    ops.paged_cache_read(*kv, ko, vo, **bt.scales())
    for hint in (1, 100):
        ops.paged_attention(q, *kv, out, 0.1, max_new=hint, **bt.scales())
    ops.check_errors(q.device)
    assert torch.equal(bt.k_cache.view(torch.uint8), before.view(torch.uint8))
    for t in (q_out, ko, vo):
        assert torch.all(t == 3.0)
    return out


@pytest.mark.parametrize("rows", [0, 1, 70])
@pytest.mark.parametrize("e4m3", [False, True])
def test_no_sequences(e4m3, rows):
    bt = R.Batch([1], [3], 16, 2, 128, H, e4m3)
    for width in (0, 5):
        assert torch.all(_call_all(bt, _i32(0, width), _i32(1), _i32(0), rows) == 3.0)


@pytest.mark.parametrize("e4m3", [False, True])
def test_a_page_table_without_columns(e4m3):
    """Places of a padded batch alone: no new tokens, or one before position 0."""
    bt = R.Batch([1], [3], 16, 2, 128, H, e4m3)
    indptr = torch.tensor([0, 1, 1, 2], dtype=torch.int32, device="cuda")
    out = _call_all(bt, _i32(3, 0), indptr, _i32(3), 5)
    assert torch.all(out[:2] == 0) and torch.all(out[2:] == 3.0)


def test_verification_without_sequences_or_rows():
    i64, f32 = dict(dtype=torch.int64, device="cuda"), dict(device="cuda")
    for B in (0, 3):
        acc = torch.full((B,), 7, dtype=torch.int32, device="cuda")
        for draft in (None, torch.zeros(0, 50, **f32)):
            ops.verify_draft(torch.zeros(0, 50, **f32), torch.zeros(0, **i64), draft, _i32(B + 1), torch.zeros(0, **f32),
                             torch.rand(B, **f32), torch.zeros(0, **i64), acc)
        ops.check_errors(torch.device("cuda", 0))
        assert not acc.any()
