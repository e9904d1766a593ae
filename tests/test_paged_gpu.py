"""The paged KV cache operators on the GPU against plain 64-bit forms: rotary
write and read back (16-bit and e4m3 pages), attention of ragged new tokens,
their masks, strides, odd pages and lengths, and a step of them together."""

import math

import pytest
import torch

import paged_ref as R
from persona import ops

pytestmark = pytest.mark.gpu
H, B16 = torch.float16, torch.bfloat16
THETA = 1e6


def _check(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((got.double() - want).abs() / tol).nan_to_num(9e9).max():.3g} x the bound"


def _attend(bt, q, scale=None, window=0, max_new=None, out=None):
    scale = 1 / math.sqrt(bt.D) if scale is None else scale
    out = torch.full_like(q, 7.0) if out is None else out
    ops.paged_attention(q, *bt.args(), out, scale, window=window, max_new=max_new, **bt.scales())
    ops.check_errors(q.device)
    want, tol = R.attention(bt, q, scale, window)
    used = int(bt.indptr[-1])
    _check(out[:used], want[:used], tol[:used])
    assert torch.all(out[used:] == 7.0)  # rows behind the last sequence
    return out


# ------------------------------------------------------------ write, read --
WRITES = [
    # new, ctx, page, Hkv, Hq, D, dtype, e4m3
    ([1], [0], 16, 8, 32, 128, H, False),
    ([1] * 8, [5, 0, 255, 16, 15, 31, 32, 100], 16, 8, 32, 128, H, False),
    ([3, 0, 7, 1], [0, 9, 30, 4000], 24, 2, 4, 64, B16, False),
    ([3, 0, 7, 1], [0, 9, 30, 4000], 7, 3, 3, 64, H, True),
    ([130, 1, 65], [100, 2, 63], 64, 8, 32, 128, B16, True),
    ([9] * 40, list(range(40)), 1, 1, 7, 128, H, True),
    ([1, 1], [1000000, 131071], 4096, 1, 2, 128, H, False),  # far positions
]


@pytest.mark.parametrize("new,ctx,page,Hkv,Hq,D,dtype,e4m3", WRITES)
def test_rope_write_and_read_back(new, ctx, page, Hkv, Hq, D, dtype, e4m3):
    bt = R.Batch(new, ctx, page, Hkv, D, dtype, e4m3, pad=3)
    q, k, v = bt.randn(bt.rows, Hq, D), bt.randn(bt.rows, Hkv, D), bt.randn(bt.rows, Hkv, D)
    k0, v0, before = k.clone(), v.clone(), (bt.k_cache.clone(), bt.v_cache.clone())
    q_out = torch.full_like(q, 3.0)
    ops.paged_rope_cache(q, k, v, *bt.args(), THETA, q_out=q_out, **bt.scales())
    ops.check_errors(q.device)
    used = bt.rows - 3
    pos = torch.cat([torch.arange(L - n, L) for n, L in zip(bt.new, bt.len)]).to(q.device)
    assert torch.equal(k, k0) and torch.equal(v, v0)
    half = torch.finfo(dtype).eps / 2

    def close16(got, want, x):  # half a step, plus fp32 products of sines good to 2^-22
        _check(got, want, half * want.abs() + 2.0 ** -20 * x.double().abs().amax(-1, keepdim=True))

    close16(q_out[:used], R.rotate(q[:used], pos, THETA), q[:used])
    assert torch.all(q_out[used:] == 3.0)
    kr = R.rotate(k[:used], pos, THETA)
    r = 0
    touched = torch.zeros(bt.num_pages, page, dtype=torch.bool, device=q.device)
    for b, (n, L) in enumerate(zip(bt.new, bt.len)):
        pg, at = bt.where(b, L - n, L)
        touched[pg, at] = True
        for name, want in (("k", kr[r:r + n]), ("v", v[r:r + n].double())):
            got = bt.get(name, b, L - n, L)
            if not e4m3:
                close16(got, want, want) if name == "k" else None
                assert name == "k" or torch.equal(got, want)
            else:
                s = getattr(bt, name + "_scale")[pg, :, at].double()
                want_s = want.abs().amax(-1) / 448
                _check(s, want_s, 2.0 ** -20 * want_s)
                # half a step of e4m3: 2^-4 of the value, or half its smallest step, 2^-10
                _check(got, want, (2.0 ** -4 * want.abs()).maximum(2.0 ** -10 * s[..., None]) + 2.0 ** -19 * want.abs().amax(-1, keepdim=True))
        r += n
    for now, old in zip((bt.k_cache, bt.v_cache), before):  # nothing else is written
        same = now.view(torch.uint8).reshape(bt.num_pages, Hkv, page, -1) == old.view(torch.uint8).reshape(bt.num_pages, Hkv, page, -1)
        assert same.transpose(1, 2)[~touched].all()
    # the way back
    ko, vo = (torch.full((bt.rows, Hkv, D), 5.0, dtype=dtype, device=q.device) for _ in range(2))
    ops.paged_cache_read(*bt.args(), ko, vo, **bt.scales())
    ops.check_errors(q.device)
    r = 0
    for b, (n, L) in enumerate(zip(bt.new, bt.len)):
        for got, name in ((ko, "k"), (vo, "v")):
            want = bt.get(name, b, L - n, L)
            _check(got[r:r + n], want, half * want.abs() * (1 + 2.0 ** -10) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps)
        r += n
    assert torch.all(ko[used:] == 5.0) and torch.all(vo[used:] == 5.0)


def test_rope_write_in_place_strided_and_tiny_values():
    """q rotated in place out of a fused q / k / v buffer; heads of zeros and of
    values far below one keep finite, exact scales."""
    bt = R.Batch([5, 2], [3, 60], 16, 2, 128, H, True, interleaved=True)
    qkv = bt.randn(bt.rows, 8 + 2 + 2, 128)
    qkv[0, 8:] = 0
    qkv[1, 8:] = 2.0 ** -24
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    ref = qkv.clone()
    got = ops.paged_rope_cache(q, k, v, *bt.args(), THETA, **bt.scales())
    ops.check_errors(q.device)
    assert got is q and torch.equal(qkv[:, 8:], ref[:, 8:])
    pos = torch.tensor([3, 4, 5, 6, 7, 60, 61], device=q.device)
    want = R.rotate(ref[:, :8], pos, THETA)
    _check(q, want, 2.0 ** -11 * want.abs() + 2.0 ** -20 * ref[:, :8].double().abs().amax(-1, keepdim=True))
    pg, at = bt.where(0, 3, 8)
    for name in "kv":
        s = getattr(bt, name + "_scale")[pg, :, at]
        assert torch.isfinite(s).all() and torch.all(s[0] == 2.0 ** -40)
        assert torch.all(bt.get(name, 0, 3, 4) == 0)
    assert torch.all(bt.get("v", 0, 4, 5) == 448 * bt.v_scale[pg[1], :, at[1]].double()[None, :, None])


def test_positions_before_the_start_and_bad_pages_leave_the_row_alone():
    bt = R.Batch([1, 2, 1], [4, 5, 6], 16, 2, 128, H)
    bt.lengths[0] = 0        # an idle place of a padded batch: its row is before position 0
    bt.table[2, 0] = -1      # no page
    q, k, v = bt.randn(4, 4, 128), bt.randn(4, 2, 128), bt.randn(4, 2, 128)
    q_out = torch.full_like(q, 3.0)
    ops.paged_rope_cache(q, k, v, *bt.args(), THETA, q_out=q_out)
    with pytest.raises(RuntimeError, match="outside the paged cache"):
        ops.check_errors(q.device)
    assert torch.all(q_out[0] == 3.0) and torch.all(q_out[3] == 3.0) and not (q_out[1:3] == 3.0).any()
    ko = torch.full_like(k, 5.0)
    bt.lengths[2] = 1 << 20  # behind the table
    ops.paged_cache_read(*bt.args(), ko, ko.clone())
    with pytest.raises(RuntimeError, match="outside the paged cache"):
        ops.check_errors(q.device)
    assert torch.all(ko[0] == 5.0) and torch.all(ko[3] == 5.0)


# -------------------------------------------------------------- attention --
SHAPES = [
    # new, ctx, page, Hkv, G, D
    ([1], [0], 16, 8, 4, 128),
    ([1] * 8, [127, 0, 255, 16, 15, 31, 32, 100], 16, 8, 4, 128),
    ([1, 0, 1, 1], [0, 0, 64, 63], 64, 2, 2, 64),
    ([1] * 5, [1000, 3, 2047, 511, 40], 24, 1, 8, 128),
    ([1] * 3, [200, 17, 1], 7, 3, 1, 64),
    ([1], [30000], 32, 4, 7, 128),
    ([1] * 150, [(37 * i) % 301 for i in range(150)], 16, 1, 4, 64),
    ([4] * 6, [100, 0, 1, 15, 16, 613], 16, 8, 4, 128),
    ([5, 1, 0, 8, 2], [0, 300, 5, 77, 129], 8, 2, 4, 128),
    ([9, 3], [4000, 0], 128, 1, 16, 64),
    ([70, 33], [0, 100], 16, 2, 4, 128),
    ([200, 1, 1, 17], [333, 1000, 0, 64], 64, 2, 2, 128),
    ([40], [20], 1, 1, 3, 64),
    ([2, 2], [6, 7], 16, 1, 40, 128),
]


@pytest.mark.parametrize("dtype,e4m3", [(H, False), (B16, False), (H, True), (B16, True)])
@pytest.mark.parametrize("new,ctx,page,Hkv,G,D", SHAPES)
def test_attention(new, ctx, page, Hkv, G, D, dtype, e4m3):
    bt = R.Batch(new, ctx, page, Hkv, D, dtype, e4m3, pad=2, seed=len(new))
    bt.fill()
    q = bt.randn(bt.rows, Hkv * G, D, scale=2.0)
    a = _attend(bt, q, max_new=max(new))
    if bt.rows < 400:
        _attend(bt, q)                    # the default choice
        _attend(bt, q, max_new=1)         # a hint that is too small changes nothing but speed
        b = _attend(bt, q, max_new=max(new))
        assert torch.equal(a, b)          # the same call, the same bits


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("window", [1, 5, 16, 64, 100, 5000])
def test_attention_window(window, e4m3):
    bt = R.Batch([1, 6, 40, 3], [300, 90, 33, 0], 16, 2, 128, B16, e4m3, seed=window)
    bt.fill()
    q = bt.randn(bt.rows, 8, 128)
    _attend(bt, q, window=window, max_new=40)
    _attend(bt, q, window=window, max_new=1)


def test_attention_rows_that_see_nothing_give_zeros():
    bt = R.Batch([1, 3, 1], [10, 20, 30], 16, 2, 128, H)
    bt.fill()
    q = bt.randn(5, 8, 128)
    bt.lengths[0], bt.lengths[1] = 0, 2   # no cache; the first of three rows is before position 0
    out = torch.full_like(q, 7.0)
    ops.paged_attention(q, *bt.args(), out, 0.1)
    ops.check_errors(q.device)
    assert torch.all(out[0] == 0) and torch.all(out[1] == 0)
    bt.len = [0, 2, 31]
    bt.new = [0, 2, 1]
    want, tol = R.attention(bt, q[2:], 0.1)
    _check(out[2:], want, tol)


def test_attention_large_scores_and_wide_scales():
    """Scores of a few hundred (one position takes all the weight) and v rows
    whose e4m3 scales lie 2^20 apart."""
    bt = R.Batch([1, 7], [500, 300], 16, 2, 128, H, True)
    bt.fill(v_spread=3.0)
    _attend(bt, bt.randn(8, 8, 128, scale=30.0))
    bt = R.Batch([1, 7], [500, 300], 16, 2, 128, B16, False)
    bt.fill(scale=8.0)
    _attend(bt, bt.randn(8, 8, 128, scale=8.0))


@pytest.mark.parametrize("n", [1, 6])
def test_attention_strided_views(n):
    bt = R.Batch([n, n], [100, 37], 16, 2, 128, H, interleaved=True)
    bt.fill()
    qkv = bt.randn(bt.rows, 12, 128)
    wide = torch.full((bt.rows, 10, 128), 7.0, dtype=H, device="cuda")
    _attend(bt, qkv[:, :8], out=wide[:, 1:9])
    assert torch.all(wide[:, 0] == 7.0) and torch.all(wide[:, 9] == 7.0)
    # heads before positions swapped: pages [pages, page size, heads, D]
    kt, vt = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (bt.k_cache, bt.v_cache))
    bt.k_cache, bt.v_cache = kt, vt
    _attend(bt, qkv[:, :8])


@pytest.mark.parametrize("e4m3", [False, True])
def test_offsets_past_32_bits(e4m3):
    """Pages whose first element lies behind 2^32."""
    page, Hkv, D = 64, 8, 128
    first = (1 << 32) // (page * Hkv * D)
    bt = R.Batch([3, 1], [130, 40], page, Hkv, D, H, e4m3)
    shape = (first + bt.num_pages, Hkv, page, D)
    bt.k_cache, bt.v_cache = (torch.empty(shape, dtype=R.E4M3 if e4m3 else H, device="cuda") for _ in range(2))
    if e4m3:
        bt.k_scale, bt.v_scale = (torch.empty(shape[:3], device="cuda") for _ in range(2))
    bt.table[bt.table < 1 << 30] += first
    bt.fill()
    q, k, v = bt.randn(4, 16, D), bt.randn(4, Hkv, D), bt.randn(4, Hkv, D)
    ops.paged_rope_cache(q, k, v, *bt.args(), THETA, **bt.scales())
    _attend(bt, q)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    ops.paged_cache_read(*bt.args(), ko, vo, **bt.scales())
    want = bt.get("v", 0, 130, 133)
    _check(vo[:3], want, 2.0 ** -11 * want.abs() + 2.0 ** -24)


def test_bad_tables_are_flagged():
    bt = R.Batch([1, 2], [100, 50], 16, 2, 128, H)
    bt.fill()
    q = bt.randn(3, 8, 128)
    out = torch.zeros_like(q)
    good = bt.table.clone()
    bt.table[0, 2] = bt.num_pages
    ops.paged_attention(q, *bt.args(), out, 0.1)
    with pytest.raises(RuntimeError, match="outside the paged cache"):
        ops.check_errors(q.device)
    want, tol = R.attention(R_only(bt, good, 1), q[1:], 0.1)
    _check(out[1:], want, tol)  # the other sequence is not affected
    bt.table = good
    bt.lengths[0] = 1 << 20
    ops.paged_attention(q, *bt.args(), out, 0.1)
    with pytest.raises(RuntimeError, match="outside the paged cache"):
        ops.check_errors(q.device)
    bt.lengths[0] = 101
    bt.indptr[2] = 9  # behind the rows
    ops.paged_attention(q, *bt.args(), out, 0.1)
    with pytest.raises(RuntimeError, match="segment"):
        ops.check_errors(q.device)


def R_only(bt, table, b):
    """The batch's sequence b alone."""
    import copy

    one = copy.copy(bt)
    one.new, one.len, one.table = [bt.new[b]], [bt.len[b]], table[b:b + 1]
    return one


def test_captured_calls_follow_the_device_arrays_and_share_no_state():
    """Two captured graphs of different batches, replayed in turn and after the
    lengths and pages changed, on another stream than the eager calls."""
    def make(seed, new, ctx, e4m3):
        bt = R.Batch(new, ctx, 16, 2, 128, H, e4m3, seed=seed, width=64)
        bt.fill()
        return bt, bt.randn(bt.rows, 8, 128)

    made = [make(1, [1] * 4, [700, 30, 0, 99], False), make(2, [3, 2], [500, 800], True)]
    graphs = []
    for bt, q in made:
        out = torch.zeros_like(q)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ops.paged_attention(q, *bt.args(), out, 0.1, **bt.scales())
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.paged_attention(q, *bt.args(), out, 0.1, **bt.scales())
        graphs.append((g, out))
    for turn in range(3):
        for (bt, q), (g, out) in zip(made, graphs):
            out.zero_()
            g.replay()
        for (bt, q), (g, out) in zip(made, graphs):
            want, tol = R.attention(bt, q, 0.1)
            _check(out, want, tol)
        for bt, q in made:  # shorter sequences next time
            bt.len = [max(n, L - 23) for n, L in zip(bt.new, bt.len)]
            bt.lengths.copy_(torch.tensor(bt.len, dtype=torch.int32))
            q.copy_(bt.randn(*q.shape))
    ops.check_errors(torch.device("cuda", 0))


def test_two_streams_at_once():
    made = []
    for seed in range(4):
        bt = R.Batch([1, 2], [900 + seed, 400], 16, 4, 128, H, seed=seed)
        bt.fill()
        made.append((bt, bt.randn(3, 16, 128), torch.zeros(3, 16, 128, dtype=H, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for bt, q, out, s in made:
            with torch.cuda.stream(s):
                ops.paged_attention(q, *bt.args(), out, 0.1)
    torch.cuda.synchronize()
    for bt, q, out, _ in made:
        want, tol = R.attention(bt, q, 0.1)
        _check(out, want, tol)


@pytest.mark.parametrize("e4m3", [False, True])
def test_a_speculative_step(e4m3):
    """A prompt in two chunks, then a chunk of drafted tokens: write, attend,
    verify, roll the lengths back to what was accepted, and go on.  The cache
    after the steps is that of the kept tokens alone."""
    Hkv, Hq, D, V = 2, 8, 128, 97
    bt = R.Batch([30, 12], [0, 0], 16, Hkv, D, H, e4m3, width=8, spare=16)
    bt.table.copy_(torch.randperm(16).view(2, 8).to(torch.int32))
    emb = {n: bt.randn(V, h, D) for n, h in (("q", Hq), ("k", Hkv), ("v", Hkv))}
    head = bt.randn(Hq * D, V, scale=0.1)
    seqs = [torch.randint(0, V, (30,)).tolist(), torch.randint(0, V, (12,)).tolist()]

    def feed(chunks):
        """One ragged call: the chunks' tokens through write and attention."""
        bt.new = [len(c) for c in chunks]
        bt.len = [L + n for L, n in zip(have, bt.new)]
        bt.indptr = torch.tensor([0, bt.new[0], sum(bt.new)], dtype=torch.int32, device="cuda")
        bt.lengths = torch.tensor(bt.len, dtype=torch.int32, device="cuda")
        tok = torch.tensor(sum(chunks, []), device="cuda")
        q, k, v = (emb[n][tok].clone() for n in "qkv")
        ops.paged_rope_cache(q, k, v, *bt.args(), THETA, **bt.scales())
        out = _attend(bt, q, max_new=max(bt.new))
        return torch.softmax((out.reshape(len(tok), -1) @ head).float(), dim=-1)

    have = [0, 0]
    feed([seqs[0][:20], seqs[1][:12]])
    have = [20, 12]
    feed([seqs[0][20:], []])
    have = [30, 12]
    last = [5, 6]  # the token each sequence feeds next
    g = torch.Generator(device="cuda").manual_seed(3)
    for step in range(4):
        drafts = [torch.randint(0, V, (3,)).tolist(), torch.randint(0, V, (2,)).tolist()]
        chunks = [[last[i]] + drafts[i] for i in range(2)]
        p = feed(chunks)
        rows = p.shape[0]
        qd = torch.softmax(torch.randn(rows, V, device="cuda", generator=g), dim=-1)
        judged = torch.tensor([t for i in range(2) for t in drafts[i] + [0]], device="cuda")
        ua, us = torch.rand(rows, device="cuda", generator=g), torch.rand(2, device="cuda", generator=g)
        tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
        acc = torch.zeros(2, dtype=torch.int32, device="cuda")
        ops.verify_draft(p, judged, qd, bt.indptr, ua, us, tokens, acc)
        want, want_a = R.verify(p, judged, qd, bt.indptr, ua, us)
        assert tokens.tolist() == want and acc.tolist() == want_a
        for i in range(2):
            a, r0 = int(acc[i]), int(bt.indptr[i])
            seqs[i] += chunks[i][:1 + a]
            have[i] += 1 + a
            last[i] = int(tokens[r0 + a])
    ops.check_errors(torch.device("cuda", 0))
    for i in range(2):
        tok = torch.tensor(seqs[i], device="cuda")
        assert have[i] == len(seqs[i])
        want = emb["v"][tok].double()
        got = bt.get("v", i, 0, have[i])
        _check(got, want, want.abs() * (2.0 ** -4 if e4m3 else 0) + (want.abs().amax(-1, keepdim=True) / 448 * 2.0 ** -9 if e4m3 else 0))


@pytest.mark.parametrize("e4m3", [False, True])
def test_short_and_wide_page_tables(e4m3):
    """The same sequences behind a page table of their own width and a wide one
    (another division of the work), and more new tokens than the hint says."""
    outs = []
    for width in (None, 4, 40, 600):
        bt = R.Batch([3, 1, 9, 0], [37, 2, 44, 5], 16, 2, 128, H, e4m3, seed=8, width=width)
        bt.fill()
        q = bt.randn(bt.rows, 8, 128)
        outs += [_attend(bt, q, max_new=n) for n in (1, 3, 9)]
        bt.lengths.zero_()  # nothing cached: all rows lie before the start
        out = torch.full_like(q, 7.0)
        ops.paged_attention(q, *bt.args(), out, 0.1, **bt.scales())
        assert torch.all(out == 0)
    ops.check_errors(torch.device("cuda", 0))


def test_long_step_of_many_rows_of_the_chunk_shape():
    """A prompt chunk over a long cache, beside decoding sequences."""
    bt = R.Batch([600, 1, 1, 129], [3000, 2500, 0, 1], 64, 2, 128, H, False)
    bt.fill()
    _attend(bt, bt.randn(bt.rows, 8, 128), max_new=600)


@pytest.mark.parametrize("page", [16, 7, 1])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("n", [1, 5, 150])
def test_pages_before_the_window_may_be_given_back(n, e4m3, page):
    """Table entries of the pages that the first new token's window does not
    reach point nowhere, and what is left of the last such page is NaN.  What
    is computed then is what it was with the pages still there."""
    window, ctx = 45, [400, 83, 20]
    bt = R.Batch([n] * 3, ctx, page, 2, 128, H, e4m3, seed=n)
    bt.fill()
    q = bt.randn(bt.rows, 8, 128)
    want, tol = R.attention(bt, q, 0.1, window)
    for b, c in enumerate(ctx):
        first = max(0, c + 1 - window)
        if first:
            pg, at = bt.where(b, 0, first)
            for x in (bt.k_cache, bt.v_cache):
                if e4m3:
                    x.view(torch.uint8)[pg, :, at] = 0x7F  # NaN
                else:
                    x[pg, :, at] = float("nan")
            if e4m3:
                bt.k_scale[pg, :, at] = bt.v_scale[pg, :, at] = float("nan")
            bt.table[b, :first // page] = -1
    out = torch.zeros_like(q)
    ops.paged_attention(q, *bt.args(), out, 0.1, window=window, max_new=n, **bt.scales())
    ops.check_errors(q.device)
    _check(out, want, tol)


@pytest.mark.parametrize("n", [1, 20])
def test_many_sequences(n):
    """More sequences than threads of a CTA, in both kernels."""
    B = 700
    bt = R.Batch([n if b % 3 else 0 for b in range(B)], [b * 7 % 90 for b in range(B)], 16, 1, 64, H, seed=2, pad=2)
    bt.fill()
    _attend(bt, bt.randn(bt.rows, 4, 64), max_new=n)


def test_captured_chunks_on_two_streams():
    """Prompt chunks captured on their own streams, both graphs under way at once."""
    made = []
    for seed in range(2):
        bt = R.Batch([300, 40], [200 + 50 * seed, 0], 16, 2, 128, H, seed=seed)
        bt.fill()
        q = bt.randn(bt.rows, 8, 128)
        out, s = torch.zeros_like(q), torch.cuda.Stream()
        ops.paged_attention(q, *bt.args(), out, 0.1, max_new=300)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.paged_attention(q, *bt.args(), out, 0.1, max_new=300)
        made.append((bt, q, out, s, g))
    for _ in range(4):
        for bt, q, out, s, g in made:
            out.zero_()
        torch.cuda.synchronize()
        for *_, s, g in made:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for bt, q, out, *_ in made:
            want, tol = R.attention(bt, q, 0.1)
            _check(out, want, tol)
    ops.check_errors(torch.device("cuda", 0))


def test_outputs_that_overlap_inputs_are_refused():
    bt = R.Batch([4, 3], [60, 9], 16, 2, 128, H, pad=1)
    bt.fill()
    fused = bt.randn(bt.rows, 24, 128)
    q, k, v = fused[:, :8], fused[:, 8:10], fused[:, 10:12]
    for out in (q, fused[:, 1:9], fused[:, 7:15]):
        with pytest.raises(RuntimeError, match="out must not overlap q"):
            ops.paged_attention(q, *bt.args(), out, 0.1)
    # q and out as slices of one buffer that share nothing
    want, tol = R.attention(bt, q, 0.1)
    out = fused[:, 16:24]
    ops.paged_attention(q, *bt.args(), out, 0.1)
    _check(out[:7], want[:7], tol[:7])
    with pytest.raises(RuntimeError, match="q_out must be q"):
        ops.paged_rope_cache(q, k, v, *bt.args(), THETA, q_out=fused[:, 1:9])
    with pytest.raises(RuntimeError, match="must not overlap k or v"):
        ops.paged_rope_cache(q, k, v, *bt.args(), THETA, q_out=fused[:, 9:17])
    with pytest.raises(RuntimeError, match="k_out and v_out"):
        ops.paged_cache_read(*bt.args(), fused[:, 8:10], fused[:, 9:11])
    ops.paged_cache_read(*bt.args(), k, v)
    want = bt.get("v", 1, 9, 12)
    _check(v[4:7], want, 0 * want)
    flat = bt.k_cache[0].expand_as(bt.k_cache)
    with pytest.raises(RuntimeError, match="overlap themselves"):
        ops.paged_rope_cache(q, k, v, flat, flat, *bt.args()[2:], THETA)
