"""8-bit pages with one scale per block of tokens and head: write, read back
and attention against the definition in 64 bits."""

import pytest
import torch

import block_ref as K
import paged_ref as R
from persona import ops

pytestmark = pytest.mark.gpu
THETA = 1e6
H, BF = torch.float16, torch.bfloat16


def _write(bt, Hq, pad_value=3.0, **kw):
    q, k, v = (bt.randn(bt.rows, h, bt.D) for h in (Hq, bt.Hkv, bt.Hkv))
    q_out = torch.full_like(q, pad_value)
    ops.paged_rope_cache(q, k, v, *bt.args(), THETA, q_out=q_out, **bt.scales(), **kw)
    return q, k, v, q_out


@pytest.mark.parametrize("dtype", [H, BF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page,block", [(16, 16), (32, 16), (64, 64), (128, 128), (24, 8), (8, 2), (48, 4)])
def test_write(dtype, D, page, block):
    # empty sequences, single tokens at, before and behind a block's border, chunks over several pages, far positions
    new = [1, 0, 1, 1, 5, 150, 2, 33, 1]
    ctx = [0, 9, block - 1, block, 3, 7, 2 * page - 1, 0, 100003]
    bt = K.BlockBatch(new, ctx, page, 3, D, dtype, block, pad=2, seed=page + D)
    # earlier tokens smaller (the scale grows), larger (it stays)
    bt.fill(scale=0.02, spread=4.0, upto=ctx, tail=3)
    before = K.state(bt)
    q, k, v, q_out = _write(bt, 6)
    ops.check_errors(q.device)
    K.check_write(bt, before, q, k, v, q_out, THETA)
    assert torch.all(q_out[sum(new):] == 3.0)


def test_write_grows_token_by_token():
    """A block filled one token a call, each twice as large as the one before,
    then much smaller ones: earlier codes move exactly until they leave the
    normal ones, and stay where nothing grows."""
    bt = K.BlockBatch([1], [0], 16, 2, 64, H, 16)
    for p in range(16):
        bt.len[0] = p + 1
        bt.lengths.fill_(p + 1)
        before = K.state(bt)
        q, k, v = (bt.randn(1, h, 64, scale=2.0 ** (p if p < 9 else -6)) for h in (2, 2, 2))
        q_out = torch.empty_like(q)
        ops.paged_rope_cache(q, k, v, *bt.args(), THETA, q_out=q_out, **bt.scales())
        K.check_write(bt, before, q, k, v, q_out, THETA)


def test_scale_borders():
    """Maxima on, just below and just above 448 times a power of two, zeros,
    and the smallest scale."""
    big = 448.0
    rows = [big, big - 0.25, big * (1 + 2.0 ** -10), 0.0, 2.0 ** -24, 1.0, 1.75, 1.751, 65504.0, 7.0, 7.004]
    n = len(rows)
    bt = K.BlockBatch([1] * n, [0] * n, 16, 1, 64, H, 16)
    v = torch.zeros(n, 1, 64, dtype=H, device="cuda")
    v[:, 0, 5] = torch.tensor(rows, device="cuda").half()
    k, q = torch.zeros_like(v), torch.zeros_like(v)
    before = K.state(bt)
    q_out = torch.empty_like(q)
    ops.paged_rope_cache(q, k, v, *bt.args(), THETA, q_out=q_out, **bt.scales())
    K.check_write(bt, before, q, k, v, q_out, THETA)
    assert float(bt.blocks["v"][bt.table[3, 0], 0, 0]) == 2.0 ** -40
    assert float(bt.blocks["v"][bt.table[0, 0], 0, 0]) == 1.0


def test_write_of_padded_and_negative_places():
    """Rows before position 0, sequences of length 0, wrong pages and padding
    rows are left alone; in place for q; slices of one buffer."""
    bt = K.BlockBatch([4, 1, 3, 2], [-2, -1, 5, 30], 16, 2, 128, BF, 16, pad=3)
    bt.fill(upto=[0, 0, 5, 30])
    fused = bt.randn(bt.rows, 4 + 2 + 2, 128)
    q, k, v = fused[:, :4], fused[:, 4:6], fused[:, 6:]
    copy = fused.clone()
    before = K.state(bt)
    ops.paged_rope_cache(q, k, v, *bt.args(), THETA, **bt.scales())
    ops.check_errors(q.device)
    K.check_write(bt, before, copy[:, :4], copy[:, 4:6], copy[:, 6:], q, THETA)
    assert torch.equal(q[:2], copy[:2, :4]) and torch.equal(q[10:], copy[10:, :4]) and torch.equal(q[4], copy[4, :4])
    assert torch.equal(k, copy[:, 4:6]) and torch.equal(v, copy[:, 6:])
    # a page outside of the cache: that sequence's rows alone
    bt.table[3, 1] = bt.num_pages
    before = K.state(bt)
    q_out = torch.full_like(q, 3.0)
    ops.paged_rope_cache(q.contiguous(), k, v, *bt.args(), THETA, q_out=q_out, **bt.scales())
    with pytest.raises(RuntimeError, match="outside the paged cache"):
        ops.check_errors(q.device)
    K.check_write(bt, before, q, k, v, q_out, THETA, skip=(3,))
    assert torch.all(q_out[8:10] == 3.0)


def test_indices_that_are_wrong():
    """indptr beyond the rows, decreasing or negative: no row outside of the activations is touched."""
    bt = K.BlockBatch([2, 2, 2], [5, 9, 30], 16, 2, 64, H, 16)
    bt.fill()
    for indptr in ([0, 2, 4, 900], [-50, 2, 4, 6], [0, 6, 2, 4], [6, 6, 6, 6], [4, 4, 4, 6]):
        bt.indptr.copy_(torch.tensor(indptr, dtype=torch.int32))
        _write(bt, 4)
        torch.cuda.synchronize()
    ops._load().take_device_error(0)


@pytest.mark.parametrize("dtype", [H, BF])
@pytest.mark.parametrize("page,block,D", [(16, 16, 128), (64, 16, 64), (24, 8, 128), (128, 128, 128)])
def test_read(dtype, page, block, D):
    bt = K.BlockBatch([5, 0, 70, 1], [0, 3, 20, 200], page, 3, D, dtype, block, pad=2)
    bt.fill(spread=3.0)
    ko, vo = (torch.full((bt.rows, 3, D), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    ops.paged_cache_read(*bt.args(), ko, vo, **bt.scales())
    r = 0
    for b, (n, L) in enumerate(zip(bt.new, bt.len)):
        for name, o in (("k", ko), ("v", vo)):
            assert torch.equal(o[r:r + n], bt.get(name, b, L - n, L).to(dtype))
        r += n
    assert torch.all(ko[r:] == 7.0) and torch.all(vo[r:] == 7.0)


def _check(out, want, tol):
    err = (out.double() - want).abs()
    assert torch.isfinite(out).all() and torch.all(err <= tol), float((err / tol).max())


@pytest.mark.parametrize("dtype", [H, BF])
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (4, 4, 64), (14, 2, 128), (8, 1, 64)])
@pytest.mark.parametrize("page,block", [(16, 16), (64, 16), (32, 32), (128, 128), (24, 8)])
@pytest.mark.parametrize("window", [0, 40])
def test_attention_few_rows(dtype, Hq, Hkv, D, page, block, window):
    bt = K.BlockBatch([1, 0, 1, 4, 1, 1, 2], [0, 9, 15, 60, 700, 2300, 127], page, Hkv, D, dtype, block, pad=2, seed=3)
    bt.fill(spread=1.0)
    q = bt.randn(bt.rows, Hq, D, scale=1.5)
    out = torch.full_like(q, 9.0)
    want, tol = R.attention(bt, q, D ** -0.5, window)
    n = sum(bt.new)
    for max_new in (1, 3, 4, 5, 8):  # a bound that is too small is still computed right
        ops.paged_attention(q, *bt.args(), out, D ** -0.5, window=window, max_new=max_new, **bt.scales())
        ops.check_errors(q.device)
        _check(out[:n], want[:n], tol[:n])
        assert torch.all(out[n:] == 9.0)
        out.fill_(9.0)


@pytest.mark.parametrize("dtype,Hq,Hkv,D", [(H, 32, 8, 128), (BF, 8, 2, 64), (BF, 6, 6, 128)])
@pytest.mark.parametrize("page,block", [(16, 16), (64, 64), (128, 8), (24, 8)])
def test_attention_many_rows(dtype, Hq, Hkv, D, page, block):
    bt = K.BlockBatch([300, 1, 129, 0, 40], [100, 333, 0, 5, 77], page, Hkv, D, dtype, block, pad=1, seed=4)
    bt.fill(spread=1.0)
    q = bt.randn(bt.rows, Hq, D, scale=1.5)
    for window in (0, 100):
        out = torch.zeros_like(q)
        ops.paged_attention(q, *bt.args(), out, D ** -0.5, window=window, **bt.scales())
        ops.check_errors(q.device)
        want, tol = R.attention(bt, q, D ** -0.5, window)
        n = sum(bt.new)
        _check(out[:n], want[:n], tol[:n])


@pytest.mark.parametrize("B,L", [(64, 3000), (3, 20000), (200, 90)])
def test_attention_batches(B, L):
    """Ranges that end inside tiles, clusters of every size."""
    ctx = [(L * (i + 1)) // B for i in range(B)]
    bt = K.BlockBatch([1] * B, ctx, 32, 2, 128, BF, 32, seed=5)
    bt.fill(spread=1.0)
    for Hq in (2, 8, 32):
        q = bt.randn(bt.rows, Hq, 128, scale=1.5)
        out = torch.zeros_like(q)
        ops.paged_attention(q, *bt.args(), out, 128 ** -0.5, **bt.scales())
        want, tol = R.attention(bt, q, 128 ** -0.5)
        _check(out, want, tol)
        again = torch.zeros_like(q)
        ops.paged_attention(q, *bt.args(), again, 128 ** -0.5, **bt.scales())
        assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", [H, BF])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (7, 1, 64), (5, 5, 128)])
@pytest.mark.parametrize("new,ctx", [([5, 3, 5], [40, 0, 200]), ([6] * 40, [31 * i % 700 for i in range(40)]),
                                     ([2, 9, 1, 4], [9000, 30, 4000, 0]), ([3] * 100, [17 * i for i in range(100)])])
def test_attention_of_drafts(dtype, Hq, Hkv, D, new, ctx):
    """17 to 64 rows per kv head: clusters, ranges that end inside tiles, more than one tile."""
    bt = K.BlockBatch(new, ctx, 64, Hkv, D, dtype, 32, pad=1, seed=15)
    bt.fill(spread=1.0)
    q = bt.randn(bt.rows, Hq, D, scale=1.5)
    for window in (0, 130):
        out = torch.full_like(q, 9.0)
        ops.paged_attention(q, *bt.args(), out, D ** -0.5, window=window, max_new=max(new), **bt.scales())
        ops.check_errors(q.device)
        want, tol = R.attention(bt, q, D ** -0.5, window)
        _check(out[:-1], want[:-1], tol[:-1])
        assert torch.all(out[-1] == 9.0)


def test_attention_leaves_other_contents_out():
    """NaN codes and scales behind a sequence's last block, in pages that it
    does not hold and before a window; NaN codes behind its last token."""
    bt = K.BlockBatch([1, 3, 1], [20, 70, 500], 16, 2, 128, H, 16, seed=6)
    bt.fill()
    q = bt.randn(bt.rows, 8, 128)
    want, tol = R.attention(bt, q, 0.09, 48)
    lo = (500 + 1 - 48) // 16  # the pages before the window of the last sequence
    for j in range(lo):
        pg = int(bt.table[2, j])
        bt.cache8("k")[pg] = bt.cache8("v")[pg] = 0x7f
        bt.blocks["k"][pg] = bt.blocks["v"][pg] = float("nan")
    bt.table[2, :lo] = -7
    out = torch.zeros_like(q)
    ops.paged_attention(q, *bt.args(), out, 0.09, window=48, **bt.scales())
    ops.check_errors(q.device)
    _check(out, want, tol)


def test_attention_scales_far_apart():
    """Blocks whose scales lie up to 2^60 apart, zeros among them: the weight of
    a block is not lost beside another one's scale."""
    bt = K.BlockBatch([1, 1], [63, 200], 16, 1, 64, H, 16, seed=8)
    bt.fill()
    for name in "v":
        for b in range(2):
            for j in range(bt.table.shape[1]):
                pg = int(bt.table[b, j])
                if 0 <= pg < bt.num_pages:
                    bt.blocks[name][pg] *= 2.0 ** ([-30, 0, -55, 3][j % 4])
    pg = int(bt.table[1, 2])
    bt.blocks["k"][pg] = 0.0
    q = bt.randn(2, 4, 64)
    out = torch.zeros(2, 4, 64, dtype=H, device="cuda")
    ops.paged_attention(q, *bt.args(), out, 0.125, **bt.scales())
    want, _ = R.attention(bt, q, 0.125)
    # weights are rounded to fp16 beside the largest p v_scale of a run of
    # positions: 2^-11 of a term, or 2^-25 of the largest term's weight; |v / v_scale| <= 448
    r = 0
    for b, L in enumerate(bt.len):
        k = bt.get("k", b, 0, L).repeat_interleave(4, 1)
        v = bt.get("v", b, 0, L).repeat_interleave(4, 1)
        pgs, at = bt.where(b, 0, L)
        vs = bt.v_scale[pgs, :, at].double().repeat_interleave(4, 1)
        p = torch.softmax(torch.einsum("hd,lhd->hl", q[r].double(), k) * 0.125, -1)
        bound = (2.0 ** -11 + 2.0 ** -17) * torch.einsum("hl,lhd->hd", p, v.abs()) + \
            (p * vs.t()).amax(-1, keepdim=True) * 2.0 ** -24 * L * 448 + 2.0 ** -11 * want[r].abs() + 2.0 ** -25
        assert torch.all((out[r].double() - want[r]).abs() <= bound)
        r += 1


def test_interleaved_pages_and_other_stream():
    bt = K.BlockBatch([1, 2, 60], [100, 40, 9], 32, 2, 128, H, 16, interleaved=True, seed=9)
    bt.fill()
    q = bt.randn(bt.rows, 8, 128)
    want, tol = R.attention(bt, q, 0.09)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = torch.zeros_like(q)
        ops.paged_attention(q, *bt.args(), out, 0.09, **bt.scales())
    s.synchronize()
    _check(out, want, tol)


@pytest.mark.parametrize("D", [64, 128])
def test_pages_with_gaps(D):
    """Positions further apart than a head is wide, heads and pages with gaps, scales in one pool."""
    bt = K.BlockBatch([1, 3, 40], [100, 20, 9], 32, 2, D, H, 16, seed=12)
    pools = [torch.full((bt.num_pages, 2, 34, D + 16), float("nan"), device="cuda").to(R.E4M3) for _ in range(2)]
    bt.k_cache, bt.v_cache = (p[:, :, 1:33, :D] for p in pools)
    scales = torch.full((bt.num_pages, 2, 2, 3), float("nan"), device="cuda")
    bt.blocks = {"k": scales[:, 0, :, :2], "v": scales[:, 1, :, :2]}
    bt.fill(upto=[100, 20, 9])
    before = K.state(bt)
    q, k, v, q_out = _write(bt, 8)
    K.check_write(bt, before, q, k, v, q_out, THETA)
    for max_new in (1, 40):
        out = torch.zeros_like(q)
        ops.paged_attention(q_out, *bt.args(), out, 0.09, max_new=max_new, **bt.scales())
        want, tol = R.attention(bt, q_out, 0.09)
        _check(out, want, tol)
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    ops.paged_cache_read(*bt.args(), ko, vo, **bt.scales())
    assert torch.equal(ko[4:], bt.get("k", 2, 9, 49).to(H)) and torch.equal(vo[:1], bt.get("v", 0, 100, 101).to(H))
    ops.check_errors(q.device)


def test_captured_into_two_graphs():
    """Write, attention and read back of two batches, replayed on two streams with changed lengths."""
    graphs, parts = [], []
    for i in range(2):
        bt = K.BlockBatch([1, 1, 2], [40, 200, 13], 32, 2, 128, H, 16, seed=20 + i, width=9)
        bt.fill(upto=[40, 200, 13])
        q, k, v = bt.randn(4, 8, 128), bt.randn(4, 2, 128), bt.randn(4, 2, 128)
        q_out, out = torch.zeros_like(q), torch.zeros_like(q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.paged_rope_cache(q, k, v, *bt.args(), THETA, q_out=q_out, **bt.scales())
            ops.paged_attention(q_out, *bt.args(), out, 0.09, max_new=2, **bt.scales())
        graphs.append(g)
        parts.append((bt, q, k, v, q_out, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for step in range(3):
        states = [K.state(p[0]) for p in parts]
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (bt, q, k, v, q_out, out), before in zip(parts, states):
            K.check_write(bt, before, q, k, v, q_out, THETA)
            want, tol = R.attention(bt, q_out, 0.09)
            _check(out, want, tol)
            for b in range(3):  # the next tokens, other rows
                bt.len[b] += bt.new[b]
            bt.lengths.copy_(torch.tensor(bt.len, dtype=torch.int32))
            for t in (q, k, v):
                t.copy_(bt.randn(*t.shape))
    ops.check_errors(torch.device("cuda", 0))


def test_refusals():
    bt = K.BlockBatch([1, 1], [20, 70], 48, 2, 128, H, 16)
    bt.fill()
    q, k = bt.randn(2, 8, 128), bt.randn(2, 2, 128)
    bad = lambda n: dict(k_scale=torch.zeros(bt.num_pages, 2, n, device="cuda"),  # noqa: E731
                         v_scale=torch.zeros(bt.num_pages, 2, n, device="cuda"))
    for n in (0, 1, 2, 4, 5, 16, 47, 49, 96):
        with pytest.raises(RuntimeError, match="a page has a scale per position, or per block"):
            ops.paged_attention(q, *bt.args(), torch.zeros_like(q), 0.1, **bad(n))
    with pytest.raises(RuntimeError, match="scales must be"):
        ops.paged_attention(q, *bt.args(), torch.zeros_like(q), 0.1, k_scale=bt.blocks["k"], v_scale=bad(6)["v_scale"])
    with pytest.raises(RuntimeError, match="overlap"):
        ops.paged_rope_cache(q, k, k.clone(), *bt.args(), THETA, k_scale=bt.blocks["k"], v_scale=bt.blocks["k"])
