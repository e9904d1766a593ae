"""Batches over 8-bit pages with one scale per block, and what a write to them has to leave behind."""

import torch

import paged_ref as R

E4M3 = R.E4M3


def two_power(amax):
    """The smallest power of two s with amax <= 448 s, and 2^-40 at least (amax in 64 bits)."""
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e, -100)
    return torch.exp2((e - 9 + (m > 0.875)).clamp_min(-40).double()).float()


class BlockBatch(R.Batch):
    """A Batch whose scales are per block; ``k_scale`` / ``v_scale`` are those
    spread over the positions, for the plain forms, ``scales()`` the real ones."""

    def __init__(self, new, ctx, page, Hkv, D, dtype, block, **kw):
        super().__init__(new, ctx, page, Hkv, D, dtype, e4m3=True, **kw)
        assert page % block == 0
        self.block = block
        shape = (self.num_pages, Hkv, page // block)
        self.blocks = {n: torch.full(shape, float("nan"), device=self.device) for n in "kv"}

    @property
    def k_scale(self):
        return self.blocks["k"].repeat_interleave(self.block, dim=2) if "blocks" in self.__dict__ else None

    @property
    def v_scale(self):
        return self.blocks["v"].repeat_interleave(self.block, dim=2) if "blocks" in self.__dict__ else None

    @k_scale.setter
    def k_scale(self, _):
        pass

    @v_scale.setter
    def v_scale(self, _):
        pass

    def scales(self):
        return dict(k_scale=self.blocks["k"], v_scale=self.blocks["v"])

    def fill(self, scale=1.0, spread=0.0, upto=None, tail=None):
        """Random values at the first ``upto[b]`` positions (default: all), block by
        block; with ``tail`` only in that many blocks at their end."""
        for b, L in enumerate(upto or self.len):
            for lo in list(range(0, max(L, 0), self.block))[-tail if tail else 0:]:
                hi = min(lo + self.block, L)
                pg, at = self.where(b, lo, hi)
                for name in "kv":
                    x = self.randn(hi - lo, self.Hkv, self.D, scale=scale).float()
                    if spread:
                        x = x * torch.exp2(spread * torch.randn(1, self.Hkv, 1, generator=self.g).to(x.device))
                    s = two_power(x.abs().amax(dim=(0, 2)).double())
                    self.cache8(name)[pg, :, at] = (x / s[None, :, None]).to(E4M3).view(torch.uint8)
                    self.blocks[name][pg[0], :, int(at[0]) // self.block] = s

    def cache8(self, name):
        return getattr(self, name + "_cache").view(torch.uint8)


def check_write(bt, before, q, k, v, q_out, theta, skip=()):
    """The state of ``bt`` after a write of k and v, ``before`` = its codes and
    scales from before it, against the definition in 64 bits.

    A code is off by at most half a step (2^-4 of the value, 2^-10 of the scale
    below the normal ones); k also by the fp32 rotation: two products and a sum,
    2^-22 of |x1| + |x2| with the angle's rounding."""
    dev = bt.device
    codes = {n: c.clone() for n, c in before[0].items()}
    scales = {n: s.clone() for n, s in before[1].items()}
    r, blk = 0, bt.block
    half = torch.finfo(bt.dtype).eps / 2
    for b, (n, L) in enumerate(zip(bt.new, bt.len)):
        first = max(L - n, 0)
        if b not in skip and L > 0 and n > 0:
            rows = slice(r + (first - (L - n)), r + n)
            pos = torch.arange(first, L, device=dev)
            want = R.rotate(q[rows], pos, theta)
            tol = half * want.abs() + 2.0 ** -20 * R.rotate(q[rows].abs(), torch.zeros_like(pos), theta).abs().amax() + 1e-30
            assert torch.all((q_out[rows].double() - want).abs() <= tol), "q"
            for name, x in (("k", R.rotate(k[rows], pos, theta)), ("v", v[rows].double())):
                lo = first
                while lo < L:
                    start = lo // blk * blk
                    hi = min(start + blk, L)
                    pg, at = bt.where(b, start, hi)
                    page, i = int(pg[0]), int(at[0]) // blk
                    y = x[lo - first:hi - first]
                    amax = y.abs().amax(dim=(0, 2))
                    old = scales[name][page, :, i].clone()
                    s = two_power(amax)
                    if name == "k":  # within the rotation's rounding of the border either scale is right
                        got = bt.blocks[name][page, :, i]
                        near = ((two_power(amax * (1 - 2.0 ** -20)) == got) | (two_power(amax * (1 + 2.0 ** -20)) == got))
                        s = torch.where(near, got, s)
                    if lo > start:
                        s = torch.maximum(s, old)
                        e = codes[name][pg[:lo - start], :, at[:lo - start]].view(E4M3).float()
                        again = (e * (old / s)[None, :, None]).to(E4M3).view(torch.uint8)
                        codes[name][pg[:lo - start], :, at[:lo - start]] = again
                    scales[name][page, :, i] = s
                    got = bt.cache8(name)[pg[lo - start:], :, at[lo - start:]].clone()
                    if name == "v":
                        want8 = (v[rows][lo - first:hi - first].float() / s[None, :, None]).to(E4M3).view(torch.uint8)
                        assert torch.equal(got, want8), "v codes"
                    else:
                        sd = s.double()[None, :, None]
                        rot = 2.0 ** -22 * R.rotate(k[rows][lo - first:hi - first].abs(), torch.zeros(hi - lo, device=dev), theta).amax() * 2
                        err = (got.view(E4M3).double() * sd - y).abs()
                        assert torch.all(err <= 2.0 ** -4 * y.abs() + sd * 2.0 ** -10 + rot), "k codes"
                    codes[name][pg[lo - start:], :, at[lo - start:]] = got
                    lo = hi
        r += n
    for name in "kv":  # and nothing else has changed
        assert torch.equal(codes[name], bt.cache8(name)), name
        assert torch.equal(scales[name].view(torch.int32), bt.blocks[name].view(torch.int32)), name


def state(bt):
    return {n: bt.cache8(n).clone() for n in "kv"}, {n: bt.blocks[n].clone() for n in "kv"}
