"""Buffers of the paged operators and of the draft verification that share
memory: what is refused, and layouts that look entangled and are not."""

import pytest
import torch

import paged_ref as R
from persona import ops
from test_paged_gpu import THETA, _attend, _check
from test_verify_draft_gpu import _case

pytestmark = pytest.mark.gpu
H = torch.float16


def _batch(e4m3=False, **more):
    bt = R.Batch([4, 3], [60, 9], 16, 2, 128, H, e4m3, pad=1, **more)
    bt.fill()
    return bt, bt.randn(bt.rows, 8, 128), bt.randn(bt.rows, 2, 128), bt.randn(bt.rows, 2, 128)


def _refused(f, *args, **kw):
    with pytest.raises(RuntimeError, match="overlap"):
        f(*args, **kw)


def test_one_cache_for_k_and_v_is_refused_for_writing():
    bt, q, k, v = _batch()
    kc, vc, *rest = bt.args()
    _refused(ops.paged_rope_cache, q, k, v, kc, kc, *rest, THETA)
    flat = kc.view(-1)
    _refused(ops.paged_rope_cache, q, k, v, kc[:-1], kc[1:], *rest, THETA)     # a page on
    tangled = flat.as_strided(kc.shape, (128, 16 * 128, 128, 1))               # every page a position on
    _refused(ops.paged_rope_cache, q, k, v, tangled, tangled, *rest, THETA)
    bt.v_cache = kc
    _attend(bt, q)                                                             # reading one cache as both is fine


def test_shared_scales_are_refused_for_writing():
    bt, q, k, v = _batch(e4m3=True)
    ks, vs = bt.k_scale, bt.v_scale
    one = torch.zeros(1, 1, 16, device=q.device)
    for a, b in ((ks, ks), (ks[:1].expand_as(ks), vs[:1].expand_as(vs)), (one.expand_as(ks), one.clone().expand_as(vs))):
        _refused(ops.paged_rope_cache, q, k, v, *bt.args(), THETA, k_scale=a, v_scale=b)


def test_outputs_inside_the_pages_are_refused():
    bt, q, k, v = _batch()
    kc, vc, table, indptr, lengths = bt.args()
    rows = vc.view(-1, 8, 128)[:bt.rows]
    _refused(ops.paged_attention, q, *bt.args(), rows, 0.1)
    _refused(ops.paged_rope_cache, q, k, v, *bt.args(), THETA, q_out=rows)
    few = kc.view(-1, 2, 128)[:bt.rows]
    _refused(ops.paged_cache_read, *bt.args(), k, few)
    _refused(ops.paged_rope_cache, q, few, v, *bt.args(), THETA)
    ints = torch.zeros(bt.rows * 8 * 128, dtype=H, device=q.device)
    ints.view(torch.int32)[:2] = lengths
    _refused(ops.paged_attention, q, kc, vc, table, indptr, ints.view(torch.int32)[:2], ints.view(bt.rows, 8, 128), 0.1)


def test_verification_outputs_over_inputs_are_refused():
    p, d, q, indptr, ua, us = _case([3, 2], 50, torch.float32, 8)
    tokens, acc = torch.zeros(5, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    _refused(ops.verify_draft, p, d, q, indptr, ua, us, tokens, indptr[1:])
    _refused(ops.verify_draft, p, d, q, indptr, ua, us, tokens, us.view(torch.int32))
    _refused(ops.verify_draft, p, d, q, indptr, ua, us, p.view(-1)[:10].view(torch.int64), acc)
    _refused(ops.verify_draft, p, d, q, indptr, ua, us, tokens, tokens.view(torch.int32)[1:3])


def _write_and_read(bt, q, k, v):
    """A write and its way back, against the plain rotation."""
    used = sum(bt.new)
    want_q, want_v = R.rotate(q[:used], _pos(bt), THETA), v[:used].clone()
    ops.paged_rope_cache(q, k, v, *bt.args(), THETA, **bt.scales())
    ko, vo = (torch.zeros(bt.rows, bt.Hkv, bt.D, dtype=H, device=q.device) for _ in range(2))
    ops.paged_cache_read(*bt.args(), ko, vo, **bt.scales())
    ops.check_errors(q.device)
    _check(q[:used], want_q, 2.0 ** -11 * want_q.abs() + 2.0 ** -20 * want_q.abs().amax(-1, keepdim=True))
    tol = want_v.double().abs().amax(-1, keepdim=True) * (2.0 ** -4 if bt.e4m3 else 0)
    _check(vo[:used], want_v.double(), tol + 0 * want_v.double())


def _pos(bt):
    return torch.cat([torch.arange(L - n, L) for n, L in zip(bt.new, bt.len)]).cuda()


def test_a_pool_of_codes_and_their_scales():
    """One byte pool per page and head: the codes of its positions, then their
    scales; k and v side by side."""
    bt, q, k, v = _batch(e4m3=True)
    page, D = bt.page, bt.D
    pool = torch.zeros(bt.num_pages, 2, 2, page * (D + 4), dtype=torch.uint8, device=q.device)
    codes = pool[..., :page * D].view(R.E4M3).unflatten(-1, (page, D))
    scales = pool[..., page * D:].view(torch.float32)
    bt.k_cache, bt.v_cache = codes[:, 0], codes[:, 1]
    bt.k_scale, bt.v_scale = scales[:, 0], scales[:, 1]
    bt.fill()
    _write_and_read(bt, q, k, v)
    _attend(bt, q)


def test_pools_of_every_order():
    """k and v of a position, of a head or of a page side by side."""
    for dim in (1, 2, 3):
        bt, q, k, v = _batch()
        shape = list(bt.k_cache.shape)
        shape.insert(dim, 2)
        pool = torch.zeros(shape, dtype=H, device=q.device)
        bt.k_cache, bt.v_cache = pool.select(dim, 0), pool.select(dim, 1)
        bt.fill()
        _write_and_read(bt, q, k, v)
        _attend(bt, q)


def test_a_fused_buffer_of_a_head_at_a_time():
    """q, k and v of every head side by side ([rows, heads, 3, D]): slices that
    share nothing, whatever their ranges."""
    bt = R.Batch([4, 3], [60, 9], 16, 8, 128, H, pad=1)
    bt.fill()
    qkv = bt.randn(bt.rows, 8, 4, 128)
    q, k, v, out = qkv.unbind(2)
    before = qkv.clone()
    _write_and_read(bt, q, k, v)
    assert torch.equal(qkv[:, :, 1:], before[:, :, 1:])
    rotated = q.clone()
    want, tol = R.attention(bt, rotated, 0.1)
    ops.paged_attention(q, *bt.args(), out, 0.1)
    ops.check_errors(q.device)
    _check(out[:7], want[:7], tol[:7])
    assert torch.equal(q, rotated) and torch.equal(qkv[:, :, 1:3], before[:, :, 1:3])
    ops.paged_cache_read(*bt.args(), k, v)
    assert torch.equal(q, rotated)
    for other in (qkv.view(bt.rows, 32, 128)[:, 1:9], qkv.view(bt.rows, 32, 128)[:, :32:4]):
        _refused(ops.paged_attention, q, *bt.args(), other, 0.1)
