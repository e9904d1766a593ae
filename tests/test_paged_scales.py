"""Attention over e4m3 pages whose v scales lie far apart (2^20 and more between
the largest and the smallest), within a bound that a wrong output does not meet.

The kernels put log2 of the v scale into the exponent: position j's weight for
the second product is w_j = p_j vs_j, relative to the largest, and the sum of
the p_j is taken of w_j / vs_j."""

import math

import pytest
import torch

import paged_ref as R

H, B16 = torch.float16, torch.bfloat16


def attention(bt, q, scale, window=0):
    """out [rows, Hq, D] in 64 bits, and a bound of the kernels' error:

    * the weights are rounded to fp16: half a step, 2^-11 of w_j, or half of its
      smallest one, 2^-25 of the largest w of the row (the unit they are in is
      never above it), times what they weigh, |code_j|;
    * a weight's own error, the same in the sum of the p_j: its exponent's, which
      is that of a score of D products and sums (the operands exact, but for a
      bf16 q in fp16: 2^-25 of the row's largest element), of the fp32 exponent
      and of a logarithm good to 2^-22 of its value; exponentials and reciprocals
      good to 2^-21;
    * both sums in fp32, and the result rounded once: half a step of its type,
      which below the smallest normal number is half of the smallest step
      (fp16: 2^-14 * 2^-10 / 2 = 2^-25, where outputs of 2e-6 were 2e-8 off)."""
    rows, Hq, D = q.shape
    G = Hq // bt.Hkv
    out = torch.zeros(rows, Hq, D, dtype=torch.float64, device=q.device)
    tol = torch.full_like(out, 1e-30)
    r = 0
    for b, (n, L) in enumerate(zip(bt.new, bt.len)):
        if n and L > 0:
            pg, at = bt.where(b, 0, L)
            k, v = (bt.get(x, b, 0, L).repeat_interleave(G, dim=1) for x in "kv")
            vs = bt.v_scale[pg, :, at].double().repeat_interleave(G, dim=1)  # [L, Hq]
            code = (v / vs[..., None]).abs()
            pos = torch.arange(L - n, L, device=q.device)[:, None]
            j = torch.arange(L, device=q.device)[None, :]
            gone = (j > pos) | ((j <= pos - window) if window else torch.zeros_like(j, dtype=torch.bool))
            qq = q[r:r + n].double()
            s = (torch.einsum("nhd,lhd->hnl", qq, k) * scale).masked_fill(gone, -math.inf)
            p = torch.softmax(s, dim=-1)
            o = torch.einsum("hnl,lhd->nhd", p, v)
            va = torch.einsum("hnl,lhd->nhd", p, v.abs())
            kept = (~gone).double()
            top = (p * vs.t()[:, None, :]).amax(-1)                       # largest w, [Hq, n]
            small = 2.0 ** -25 * top.t()[..., None] * torch.einsum("nl,lhd->nhd", kept, code)
            sabs = (torch.einsum("nhd,lhd->hnl", qq.abs(), k.abs()) * scale).masked_fill(gone, 0).amax(-1).t()[..., None]
            ds = sabs * (D / 4 + 4) * 2.0 ** -24
            if bt.dtype == B16:
                ksum = (k.abs().sum(-1).t()[:, None, :] * scale).masked_fill(gone, 0).amax(-1).t()[..., None]
                ds = ds + 2.0 ** -25 * qq.abs().amax(-1, keepdim=True) * ksum
            ds = ds + vs.log2().abs().amax() * 2.0 ** -22
            out[r:r + n] = o
            step = torch.finfo(bt.dtype).eps * o.abs().clamp_min(torch.finfo(bt.dtype).smallest_normal)
            tol[r:r + n] += step / 2 + va * (2.0 ** -11 + 2 * ds + 2.0 ** -20 + L * 2.0 ** -24) + small
        r += n
    return out, tol


CASES = [
    # new, ctx, page, Hkv, G, D, spread (standard deviation of log2 of a row's size), size of q
    ([1, 7], [500, 300], 16, 2, 4, 128, 3.0, 1.0),
    ([1, 7], [500, 300], 16, 2, 4, 128, 3.0, 30.0),
    ([1, 5, 1], [900, 40, 7], 24, 1, 4, 64, 6.0, 2.0),
    ([200, 1], [300, 100], 64, 2, 4, 128, 3.0, 2.0),
    ([70, 33], [0, 600], 7, 1, 8, 64, 6.0, 8.0),
]


def _batch(case, dtype, device):
    new, ctx, page, Hkv, G, D, spread, size = case
    bt = R.Batch(new, ctx, page, Hkv, D, dtype, True, pad=1, seed=len(new), device=device)
    bt.fill(v_spread=spread)
    return bt, bt.randn(bt.rows, Hkv * G, D, scale=size)


def _inside(got, want, tol):
    return ((got.double() - want).abs() <= tol).double().mean()


@pytest.mark.parametrize("case", CASES[:4], ids=str)
def test_the_bound_turns_wrong_outputs_away(case):
    """Zeros, an output without the scales, and one with each position's scale
    replaced by its neighbour's."""
    bt, q = _batch(case, H, "cpu")
    scale = 1 / math.sqrt(bt.D)
    want, tol = attention(bt, q, scale)
    n = sum(bt.new)
    want, tol = want[:n], tol[:n]
    assert float(bt.v_scale.nan_to_num(1).max() / bt.v_scale.nan_to_num(1).min()) > 2.0 ** 15
    assert _inside(want.half(), want, tol) == 1
    assert _inside(torch.zeros_like(want), want, tol) < 0.02
    true = bt.v_scale.clone()
    for wrong in (torch.ones_like(true), true.roll(1, 2).nan_to_num(1.0)):
        bt.v_scale = torch.where(true.isnan(), true, wrong)
        assert _inside(attention(bt, q, scale)[0][:n], want, tol) < 0.05


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B16])
@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention_over_scales_far_apart(case, window, dtype):
    """The kernels of few rows and, by the larger hint, of prompt chunks."""
    from persona import ops

    bt, q = _batch(case, dtype, "cuda")
    scale = 1 / math.sqrt(bt.D)
    want, tol = attention(bt, q, scale, window)
    n = sum(bt.new)
    for hint in (1, 200):
        out = torch.full_like(q, 7.0)
        ops.paged_attention(q, *bt.args(), out, scale, window=window, max_new=hint, **bt.scales())
        ops.check_errors(q.device)
        # a value of at least half a step above the type's largest rounds to infinity
        # (fp16: 65520; rows of 2^21 are in the widest case), one so near may
        limit = torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps / 4)
        over = out[:n].isinf() & (out[:n].sign() == want[:n].sign()) & (want[:n].abs() + tol[:n] >= limit)
        bad = ~(((out[:n].double() - want[:n]).abs() <= tol[:n]) | over)
        assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((out[:n].double() - want[:n]).abs() / tol[:n]).max():.3g} x the bound"
        assert torch.all(out[n:] == 7.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [H, B16])
@pytest.mark.parametrize("new", [[1, 6], [150, 40]])
def test_rows_of_zeros_that_take_most_of_the_weight(new, dtype):
    """Positions whose v is all zeros (the smallest scale, 2^-40) and whose
    scores stand far above the others': the sum of the weights is theirs, the
    output what little the others have."""
    from persona import ops

    bt = R.Batch(new, [300, 90], 16, 2, 128, dtype, True, device="cuda", seed=7)
    bt.fill()
    q = bt.randn(bt.rows, 8, 128)
    q += 1  # scores with the positions below: about 128 * 0.1 more than the others'
    for b in range(2):
        pg, at = bt.where(b, 0, 1)
        bt.put("k", pg, at, torch.ones(1, 2, 128, device="cuda"))
        bt.put("v", pg, at, torch.zeros(1, 2, 128, device="cuda"))
    assert float(bt.v_scale.nan_to_num(1).min()) == 2.0 ** -40
    want, tol = attention(bt, q, 0.1)
    for hint in (1, 200):
        out = ops.paged_attention(q, *bt.args(), torch.zeros_like(q), 0.1, max_new=hint, **bt.scales())
        ops.check_errors(q.device)
        assert ((out.double() - want).abs() <= tol).all()
