"""e4m3 codes that paged_rope_cache writes: those of value / scale, rounded to
the nearest code, ties to even, with no tolerance."""

import pytest
import torch

import paged_ref as R
from persona import ops

pytestmark = pytest.mark.gpu


def _codes(x, scale):
    return (x.float() / scale[..., None]).to(R.E4M3).float()


def _check(bt, name, x):
    """The codes and scales of one position per sequence, the last one."""
    pg, at = (torch.cat(t) for t in zip(*(bt.where(b, L - 1, L) for b, L in enumerate(bt.len))))
    scale = getattr(bt, name + "_scale")[pg, :, at]
    most = x.float().abs().amax(-1)
    want = (most / torch.full_like(most, 448.0)).clamp_min(2.0 ** -40)  # (a number's reciprocal would be multiplied)
    assert torch.equal(scale, want)
    got = getattr(bt, name + "_cache").view(torch.uint8)[pg, :, at].view(R.E4M3).float()
    assert torch.equal(got, _codes(x, want))  # (zeros of either sign: the rotation adds two of them)


def _write(bt, k, v):
    q = bt.randn(bt.rows, 2, bt.D)
    ops.paged_rope_cache(q, k, v, *bt.args(), 1e6, **bt.scales())
    ops.check_errors(q.device)


@pytest.mark.parametrize("D", [64, 128])
def test_codes_of_ties(D):
    """Heads whose largest value is 448 s and whose others lie half way between
    two codes times s, all exact in fp16, for odd s: the quotients are exact
    ties.  At position 0 the rotation leaves k as it is."""
    code = torch.arange(127, dtype=torch.uint8).view(R.E4M3).double()
    ties = (code[1:] + code[:-1]) / 2
    scales = [s for s in range(1, 147, 2) if 448 * s <= 65504]
    rows = []
    for s in scales:
        x = ties * s
        x = x[x.half().double() == x]
        for i in range(0, len(x), D - 1):
            row = torch.zeros(D, dtype=torch.float64)
            part = x[i:i + D - 1]
            row[:len(part)] = part * (1 - 2 * (torch.arange(len(part)) % 2))
            row[-1] = 448 * s
            rows.append(row)
    x = torch.stack(rows).half().cuda()[:, None, :].repeat(1, 2, 1)
    x[:, 1] = -x[:, 1]
    bt = R.Batch([1] * len(rows), [0] * len(rows), 16, 2, D, torch.float16, True)
    _write(bt, x, x)
    _check(bt, "k", x)
    _check(bt, "v", x)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [2.0 ** -20, 0.02, 1.0, 3.0, 900.0])
def test_codes_of_random_values(dtype, size):
    n = 600
    bt = R.Batch([1] * n, [0] * n, 16, 3, 128, dtype, True, seed=4)
    k, v = bt.randn(n, 3, 128, scale=size), bt.randn(n, 3, 128, scale=size)
    _write(bt, k, v)
    _check(bt, "k", k)
    _check(bt, "v", v)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_that_are_not_finite(dtype):
    """A NaN stays one and spoils no other value but, in k, the one it is rotated
    with; an infinity makes its head NaN; the other heads and tokens are as ever."""
    bt = R.Batch([3], [5], 16, 2, 128, dtype, True)
    k, v = bt.randn(3, 2, 128), bt.randn(3, 2, 128)
    k[0, 0, 10], v[0, 0, 10], k[1, 1, 70], v[1, 1, 70] = [float("nan")] * 2 + [float("inf")] * 2
    _write(bt, k, v)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    ops.paged_cache_read(*bt.args(), ko, vo, **bt.scales())
    want_k, want_v = torch.zeros_like(k, dtype=torch.bool), torch.zeros_like(v, dtype=torch.bool)
    want_k[0, 0, [10, 74]] = want_v[0, 0, 10] = True
    want_k[1, 1] = want_v[1, 1] = True
    assert torch.equal(ko.isnan(), want_k) and torch.equal(vo.isnan(), want_v)
