"""Plain 64-bit forms of the paged cache operators and of the draft
verification, and the batches that their tests run on."""

import math

import torch

E4M3 = torch.float8_e4m3fn


class Batch:
    """A ragged batch over a pool of pages in shuffled order.  Unused table
    entries are far outside the pool, unused page contents NaN."""

    def __init__(self, new, ctx, page, Hkv, D, dtype, e4m3=False, device="cuda", seed=0, spare=2, interleaved=False,
                 pad=0, width=None):
        g = torch.Generator().manual_seed(seed)
        self.new, self.len = list(new), [n + c for n, c in zip(new, ctx)]
        self.B, self.page, self.Hkv, self.D, self.dtype, self.e4m3 = len(self.new), page, Hkv, D, dtype, e4m3
        self.device = torch.device(device)
        self.rows = sum(self.new) + pad
        starts = [0]
        for n in self.new:
            starts.append(starts[-1] + n)
        i32 = dict(dtype=torch.int32, device=self.device)
        self.indptr = torch.tensor(starts, **i32)
        self.lengths = torch.tensor(self.len, **i32)
        per = [max(0, -(-L // page)) for L in self.len]
        self.num_pages = sum(per) + spare
        perm = torch.randperm(self.num_pages, generator=g).tolist()
        table = torch.full((self.B, width or max(per + [1])), 1 << 30, dtype=torch.int32)
        at = 0
        for b, n in enumerate(per):
            table[b, :n] = torch.tensor(perm[at:at + n], dtype=torch.int32)
            at += n
        self.table = table.to(self.device)
        shape = (self.num_pages, Hkv, page, D)
        store = E4M3 if e4m3 else dtype
        if interleaved:  # k and v of a page side by side in one pool
            pool = torch.full((self.num_pages, 2, Hkv, page, D), float("nan"), device=self.device).to(store)
            self.k_cache, self.v_cache = pool[:, 0], pool[:, 1]
        else:
            self.k_cache, self.v_cache = (torch.full(shape, float("nan"), device=self.device).to(store) for _ in range(2))
        self.k_scale = self.v_scale = None
        if e4m3:
            self.k_scale, self.v_scale = (torch.full(shape[:3], float("nan"), device=self.device) for _ in range(2))
        self.g = g

    def randn(self, *shape, scale=1.0):
        return (torch.randn(*shape, generator=self.g) * scale).to(self.dtype).to(self.device)

    def where(self, b, lo, hi):
        """Pages and places of positions lo .. hi of sequence b."""
        p = torch.arange(lo, hi, device=self.device)
        return self.table[b].long()[p // self.page], p % self.page

    def fill(self, scale=1.0, v_spread=0.0):
        """Random values at every position of every sequence."""
        for b, L in enumerate(self.len):
            if L <= 0:
                continue
            pg, at = self.where(b, 0, L)
            for name in ("k", "v"):
                x = self.randn(L, self.Hkv, self.D, scale=scale).float()
                if name == "v" and v_spread:  # rows whose sizes differ by powers of two
                    x = x * torch.exp2(v_spread * torch.randn(L, self.Hkv, 1, generator=self.g).to(self.device))
                self.put(name, pg, at, x)

    def put(self, name, pg, at, x):
        cache = getattr(self, name + "_cache")
        if not self.e4m3:
            cache[pg, :, at] = x.to(self.dtype)
            return
        s = (x.abs().amax(-1) / 448).clamp_min(2.0 ** -40)
        cache.view(torch.uint8)[pg, :, at] = (x / s[..., None]).to(E4M3).view(torch.uint8)
        getattr(self, name + "_scale")[pg, :, at] = s

    def get(self, name, b, lo, hi):
        """Positions lo .. hi of sequence b in 64 bits: [hi - lo, Hkv, D]."""
        pg, at = self.where(b, lo, hi)
        cache = getattr(self, name + "_cache")
        if not self.e4m3:
            return cache[pg, :, at].double()
        return cache.view(torch.uint8)[pg, :, at].view(E4M3).double() * getattr(self, name + "_scale")[pg, :, at].double()[..., None]

    def args(self):
        return self.k_cache, self.v_cache, self.table, self.indptr, self.lengths

    def scales(self):
        return dict(k_scale=self.k_scale, v_scale=self.v_scale)


def rotate(x, pos, theta):
    """Rotate-half rotary embedding in 64 bits; x [rows, H, D], pos [rows]."""
    D = x.shape[-1]
    ang = pos.double()[:, None] * theta ** (-torch.arange(0, D, 2, dtype=torch.float64, device=x.device) / D)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    lo, hi = x[..., :D // 2].double(), x[..., D // 2:].double()
    return torch.cat([lo * c - hi * s, hi * c + lo * s], dim=-1)


def attention(batch, q, scale, window=0):
    """out [rows, Hq, D] in 64 bits (zeros in rows of no sequence), and a bound
    of the error that a kernel in the batch's types may make.

    The kernel rounds the probabilities to 16 bits for the second product
    (half a step of the products' type: bf16 for bf16 pages, else fp16; at
    least 2^-25, half of fp16's smallest step, of the largest weight p v_scale
    of a run of positions), works in fp32 elsewhere (scores: D products and
    sums; exponentials to 2^-21; the sums of the second product and of p) and
    rounds the result once."""
    rows, Hq, D = q.shape
    G = Hq // batch.Hkv
    out = torch.zeros(rows, Hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    half = torch.finfo(batch.dtype).eps / 2
    phalf = torch.finfo(torch.float16 if batch.e4m3 else batch.dtype).eps / 2
    r = 0
    for b, (n, L) in enumerate(zip(batch.new, batch.len)):
        if n and L > 0:
            k = batch.get("k", b, 0, L).repeat_interleave(G, dim=1)
            v = batch.get("v", b, 0, L).repeat_interleave(G, dim=1)
            pos = torch.arange(L - n, L, device=q.device)[:, None]
            j = torch.arange(L, device=q.device)[None, :]
            gone = (j > pos) | ((j <= pos - window) if window else torch.zeros_like(j, dtype=torch.bool))
            qq = q[r:r + n].double()
            s = torch.einsum("nhd,lhd->hnl", qq, k) * scale
            s = s.masked_fill(gone, -math.inf)
            p = torch.softmax(s, dim=-1).nan_to_num(0.0)
            o = torch.einsum("hnl,lhd->nhd", p, v)
            va = torch.einsum("hnl,lhd->nhd", p, v.abs())
            sabs = (torch.einsum("nhd,lhd->hnl", qq.abs(), k.abs()) * abs(scale)).masked_fill(gone, 0).amax(-1).t()[..., None]
            ds = sabs * (D / 4 + 4) * 2.0 ** -24
            # the largest e4m3 v scale against the smallest: how far a weight
            # can lie below the largest one of its run
            small = 2.0 ** -25 * v.abs().sum(0)
            if batch.e4m3:
                pg, at = batch.where(b, 0, L)
                vs = batch.v_scale[pg, :, at].double()
                small = small * (vs.amax() / vs.amin())
            out[r:r + n] = o
            tol[r:r + n] = half * o.abs() + va * (phalf + 2 * ds + 2.0 ** -20 + L * 2.0 ** -24) + small + 1e-30
        r += n
    return out, tol


def verify(p, d, q, indptr, ua, us):
    """Tokens [rows] and accepted [B] by the definition, on the host."""
    P, Q = p.double().cpu(), None if q is None else q.double().cpu()
    d, ua, us, indptr = d.tolist(), ua.double().tolist(), us.double().tolist(), indptr.tolist()
    V = P.shape[1]
    tokens, accepted = [None] * P.shape[0], []
    for b in range(len(indptr) - 1):
        r0, n = indptr[b], indptr[b + 1] - indptr[b]
        a = 0
        while a < n - 1 and 0 <= d[r0 + a] < V and ua[r0 + a] * (1.0 if Q is None else float(Q[r0 + a, d[r0 + a]])) < float(P[r0 + a, d[r0 + a]]):
            a += 1
        accepted.append(a)
        if n == 0:
            continue
        row = P[r0 + a].nan_to_num(0.0).clamp_min(0)
        w = row
        if a < n - 1:
            if Q is not None:
                w = (P[r0 + a] - Q[r0 + a]).nan_to_num(0.0).clamp_min(0)
            else:
                w = row.clone()
                if 0 <= d[r0 + a] < V:
                    w[d[r0 + a]] = 0
            if not float(w.sum()) > 0:
                w = row
        cum = w.cumsum(0)
        if float(cum[-1]) > 0:
            over = (cum > us[b] * float(cum[-1])).nonzero()
            t = int(over[0]) if len(over) else int((w > 0).nonzero()[-1])
        else:
            t = -1
        tokens[r0:r0 + n] = d[r0:r0 + a] + [t] + [-1] * (n - a - 1)
    return tokens, accepted
