"""The operators of speculative serving over a paged KV cache: what is timed, their plain forms and their 64-bit values.

* ``write``: rotary embedding of a ragged batch of new tokens and the write of their k and v to a paged cache, in the
  cache's own 16-bit type or as e4m3 with one scale per token and head (``ops.paged_rope_cache``).
* ``read``: cached positions back out of the pages as 16-bit rows (``ops.paged_cache_read``).
* ``attend``: causal attention of each sequence's new tokens over its pages (``ops.paged_attention``).
* ``verify``: acceptance of drafted tokens against the target's probabilities (``ops.verify_draft``).

Sequence b's new tokens are rows indptr[b] .. indptr[b + 1] and sit at its last positions, the last one at
lengths[b] - 1.  Caches are [pages, kv heads, page size, head dim], the scales of 8-bit ones [pages, kv heads, page size].
"""

import math
import random
import sys

import torch

own = False

THETA = 1e6  # rotary base of the model configuration
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -40


def _ops():
    if "multi-lora-llm-kernel_b200" not in sys.path:
        sys.path.insert(1, "multi-lora-llm-kernel_b200")
    from persona import ops
    return ops


# ---------------------------------------------------------------- cases ----

def _paged(name, op, **more):
    """A case over the cache; heads and head size are the model configuration's unless said."""
    c = {"name": name, "op": op, "dtype": "f16", "cache": "same", "batch": 8, "new_lo": 1, "new_hi": 1, "chunks": 0,
         "ctx_lo": 0, "ctx_hi": 0, "mix": 0, "hq": 32, "hkv": 8, "dim": 128, "page": 16, "window": 0, "pad": 0}
    c.update(more)
    return c


def _verify(name, **more):
    c = {"name": name, "op": "verify", "dtype": "f32", "batch": 8, "new_lo": 5, "new_hi": 5, "chunks": 0, "ctx_lo": 0,
         "ctx_hi": 0, "mix": 0, "vocab": 32000, "draft": "probs", "pad": 0}
    c.update(more)
    return c


def listed():
    return [
        # one decode step of the engine's batch of 8: all latency
        _paged("write step 8", "write", ctx_lo=128, ctx_hi=255, mix=1),
        # a verification step of 64 sequences, up to 8 fed tokens each, bf16, 8-bit pages, three rows of padding
        _paged("write drafts 64 e4m3", "write", dtype="bf16", cache="e4m3", batch=64, new_lo=2, new_hi=8, ctx_lo=100,
               ctx_hi=4000, mix=2, page=32, pad=3),
        # the prompts of a prefill batch: 32 of 512 tokens, 8-bit pages
        _paged("write prompts 32x512 e4m3", "write", cache="e4m3", batch=32, new_lo=512, new_hi=512, page=64),
        # one cached prefix handed back as dense rows, an odd length
        _paged("read prefix 1999", "read", batch=1, new_lo=1999, new_hi=1999, ctx_lo=7, ctx_hi=7),
        # 8-bit pages of 16 ragged sequences restored to 16 bits
        _paged("read 16 ragged e4m3", "read", dtype="bf16", cache="e4m3", batch=16, new_lo=500, new_hi=8000, mix=3,
               page=64),
        # the decode step of the engine's batch of 8 at its own lengths: all latency
        _paged("attend step 8", "attend", ctx_lo=128, ctx_hi=255, mix=1),
        # a decode step of a full server: 64 ragged sequences, up to 8192 tokens each
        _paged("attend step 64 long", "attend", dtype="bf16", batch=64, ctx_lo=500, ctx_hi=8191, mix=4, page=32),
        # verification of drafted tokens over 8-bit pages: 32 sequences, 5 fed tokens each
        _paged("attend drafts 32x5 e4m3", "attend", cache="e4m3", batch=32, new_lo=5, new_hi=5, ctx_lo=300, ctx_hi=6000,
               mix=5),
        # prompt chunks mixed with decoding sequences, 8-bit pages, a sliding window, padding rows
        _paged("attend mixed e4m3", "attend", dtype="bf16", cache="e4m3", batch=8, new_hi=1001, chunks=2, ctx_lo=700,
               ctx_hi=3000, mix=6, page=64, window=2048, pad=5),
        # a chunk of a long prompt: 4096 new tokens over 12288 cached ones
        _paged("attend chunk 4096 of 16384", "attend", batch=1, new_lo=4096, new_hi=4096, ctx_lo=12288, ctx_hi=12288,
               page=64),
        # 8 requests, 4 drafted tokens each
        _verify("verify 8x4"),
        # a full server, up to 7 drafted tokens, half-precision probabilities, a large vocabulary of odd size
        _verify("verify 256 ragged", dtype="f16", batch=256, new_lo=1, new_hi=8, mix=7, vocab=50257, pad=2),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "attend", "verify"])
    mix = rng.randrange(1 << 30)
    if op == "verify":
        c = _verify("", dtype=rng.choice(["f32", "f16", "bf16"]), batch=_log(rng, 1, 200), mix=mix,
                    vocab=_log(rng, 100, 60000), draft=rng.choice(["probs", "probs", "point"]), pad=rng.randrange(3),
                    new_lo=rng.randrange(3))
        c["new_hi"] = c["new_lo"] + rng.randint(1, 7)
    else:
        hkv, group = rng.choice([(8, 4), (8, 4), (2, 2), (1, 8), (4, 7), (16, 1), (5, 3)])
        c = _paged("", op, dtype=rng.choice(["f16", "bf16"]), cache=rng.choice(["same", "e4m3"]), mix=mix, hkv=hkv,
                   hq=hkv * group, dim=rng.choice([64, 128, 128]), page=rng.choice([16, 32, 64, 128, 8, 24]),
                   pad=rng.randrange(4))
        if op == "attend" and rng.random() < 0.4:  # prompt chunks, some with decoding sequences beside them
            c["batch"] = rng.randint(1, 6)
            c["new_lo"], c["new_hi"] = 1, _log(rng, 33, 1500)
            c["chunks"] = rng.randint(0, c["batch"])
            c["ctx_lo"], c["ctx_hi"] = 0, _log(rng, 1, 6000)
        elif op == "attend":  # decoding and drafted tokens
            c["batch"] = _log(rng, 1, 64)
            c["new_lo"] = rng.randint(0, 1)
            c["new_hi"] = rng.choice([1, 1, rng.randint(2, 9)])
            c["ctx_hi"] = _log(rng, 20, max(200, min(16000, 200000 // c["batch"])))
            c["ctx_lo"] = rng.choice([0, c["ctx_hi"] // 20, c["ctx_hi"] // 2])
        else:
            c["batch"] = _log(rng, 1, 48)
            c["new_hi"] = _log(rng, 1, max(2, 16000 // c["batch"]))
            c["new_lo"] = rng.choice([0, 1, (c["new_hi"] + 1) // 2])
            c["ctx_lo"], c["ctx_hi"] = 0, _log(rng, 1, 1000)
        if op == "attend" and rng.random() < 0.3:
            c["window"] = _log(rng, 5, 4096)
    del c["name"]
    return c


def _lens(c):
    """New tokens and total length of each sequence: the same for every seed.  The first `chunks` sequences have new_hi
    new tokens, the others of such a case one."""
    rng = random.Random(c["mix"])
    new, total = [], []
    for b in range(c["batch"]):
        if c["chunks"]:
            n = c["new_hi"] if b < c["chunks"] else 1
        else:
            n = rng.randint(c["new_lo"], c["new_hi"]) if c["new_hi"] < 16 * max(1, c["new_lo"]) else \
                _log(rng, max(1, c["new_lo"]), c["new_hi"])
        if b == 0:
            n = max(n, 1)
        new.append(n)
        total.append(n + (rng.randint(c["ctx_lo"], c["ctx_hi"]) if c["ctx_hi"] < 4 else
                          _log(rng, max(1, c["ctx_lo"]), c["ctx_hi"])))
    return new, total


def work(c):
    new, total = _lens(c)
    rows = sum(new)
    if c["op"] == "verify":
        e = 4 if c["dtype"] == "f32" else 2
        # every drafted token's two probabilities, one row of each distribution per sequence, the tokens and numbers
        rowbytes = c["vocab"] * e * (1 if c["draft"] == "point" else 2)
        return {"bytes": c["batch"] * (rowbytes + 16) + rows * (2 * e + 8 + 8 + 4), "flops": 3.0 * c["batch"] * c["vocab"]}
    e = 2 if c["cache"] == "same" else 1
    kv = c["hkv"] * (c["dim"] * e + (4 if e == 1 else 0)) * 2  # one position's k and v in the cache
    row = c["dim"] * 2
    if c["op"] == "write":
        return {"bytes": rows * (2 * c["hq"] * row + 2 * c["hkv"] * row + kv), "flops": 3.0 * rows * (c["hq"] + c["hkv"]) * c["dim"]}
    if c["op"] == "read":
        return {"bytes": rows * (kv + 2 * c["hkv"] * row), "flops": 0}
    pairs = seen = 0
    for n, L in zip(new, total):
        w = c["window"] or L
        first = L - n
        pairs += sum(min(p + 1, w) for p in range(first, L))
        seen += L - max(0, first + 1 - w) if n else 0
    return {"bytes": seen * kv + 2 * rows * c["hq"] * row, "flops": 4.0 * pairs * c["hq"] * c["dim"]}


# --------------------------------------------------------------- inputs ----

def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + c["mix"] % 1000003)
    new, total = _lens(c)
    B, rows = c["batch"], sum(new) + c["pad"]
    s = {"case": c, "max_new": max(max(new), 1), "rows": sum(new)}
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["indptr"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    dt = TYPES[c["dtype"]]
    if c["op"] == "verify":
        V = c["vocab"]
        # a target whose probabilities fall off as a language model's do, and a draft near it
        z = _randn(g, rows, V) * 3
        s["target"] = torch.softmax(z, dim=-1).to(dt)
        q = torch.softmax(z + 0.7 * _randn(g, rows, V), dim=-1)
        s["draft_tokens"] = torch.multinomial(q, 1, generator=g)[:, 0] if rows else torch.zeros(0, dtype=torch.int64, device=DEV)
        s["draft"] = q.to(dt) if c["draft"] == "probs" else None
        s["u_accept"] = torch.rand(rows, generator=g, device=DEV)
        s["u_sample"] = torch.rand(B, generator=g, device=DEV)
        s["tokens"] = torch.zeros(rows, dtype=torch.int64, device=DEV)
        s["accepted"] = torch.zeros(B, dtype=torch.int32, device=DEV)
        return s
    Hq, Hkv, D, ps = c["hq"], c["hkv"], c["dim"], c["page"]
    per = [-(-L // ps) for L in total]
    width = max(max(per), 1)
    pages = sum(per) + 3
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(B, width, dtype=torch.int32, device=DEV)
    at = torch.tensor(per, device=DEV)
    have = torch.arange(width, device=DEV)[None, :] < at[:, None]
    table[have] = perm[:sum(per)]
    s["table"] = table
    s["lengths"] = torch.tensor(total, dtype=torch.int32, device=DEV)
    s["k_scale"] = s["v_scale"] = None
    if c["op"] == "write":
        s["q"], s["k"], s["v"] = (_randn(g, rows, h, D, dtype=dt) for h in (Hq, Hkv, Hkv))
        s["q_out"] = torch.zeros_like(s["q"])
        if c["cache"] == "same":
            s["k_cache"], s["v_cache"] = (torch.zeros(pages, Hkv, ps, D, dtype=dt, device=DEV) for _ in range(2))
        else:
            s["k_cache"], s["v_cache"] = (torch.zeros(pages, Hkv, ps, D, dtype=torch.float8_e4m3fn, device=DEV) for _ in range(2))
            s["k_scale"], s["v_scale"] = (torch.zeros(pages, Hkv, ps, device=DEV) for _ in range(2))
        return s
    for name in ("k", "v"):
        x = _randn(g, pages, Hkv, ps, D, dtype=dt)
        if c["cache"] == "same":
            s[name + "_cache"] = x
        else:
            codes, scale = _quantise(x.float())
            s[name + "_cache"], s[name + "_scale"] = codes, scale
        del x
    if c["op"] == "read":
        s["k_out"], s["v_out"] = (torch.zeros(rows, Hkv, D, dtype=dt, device=DEV) for _ in range(2))
    else:
        s["q"] = (_randn(g, rows, Hq, D) * 1.5).to(dt)
        s["out"] = torch.zeros_like(s["q"])
    return s


# ----------------------------------------------------------- plain forms ----

def _quantise(x):
    """e4m3 codes and fp32 scales of the rows of x (fp32), one scale per row of the last axis."""
    scale = (x.abs().amax(dim=-1) / E4M3_MAX).clamp_min(MIN_SCALE)
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def _places(s):
    """For every new row: its sequence, position, page and place in the page."""
    n, rows = s["indptr"].diff().long(), s["rows"]
    b = torch.repeat_interleave(torch.arange(n.numel(), device=DEV), n, output_size=rows)
    pos = torch.arange(rows, device=DEV) - s["indptr"][b] + (s["lengths"][b] - n[b])
    ps = s["case"]["page"]
    return b, pos, s["table"][b, pos // ps].long(), pos % ps


def _rotate(x, pos, dtype):
    """Rotate-half rotary embedding: the angles in 64 bits, the products in `dtype`."""
    D = x.shape[-1]
    inv = THETA ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    ang = pos[:, None].double() * inv[None, :]
    cs, sn = ang.cos().to(dtype)[:, None, :], ang.sin().to(dtype)[:, None, :]
    lo, hi = x[..., :D // 2].to(dtype), x[..., D // 2:].to(dtype)
    return torch.cat([lo * cs - hi * sn, hi * cs + lo * sn], dim=-1)


def _plain_write(s):
    c = s["case"]
    b, pos, page, at = _places(s)
    R = pos.numel()
    s["q_out"][:R] = _rotate(s["q"][:R], pos, torch.float32).to(s["q"].dtype)
    k, v = _rotate(s["k"][:R], pos, torch.float32), s["v"][:R]
    if c["cache"] == "same":
        s["k_cache"][page, :, at] = k.to(s["k"].dtype)
        s["v_cache"][page, :, at] = v
        return s["q_out"], s["k_cache"], s["v_cache"]
    for x, name in ((k, "k"), (v.float(), "v")):
        codes, scale = _quantise(x)
        s[name + "_cache"].view(torch.uint8)[page, :, at] = codes.view(torch.uint8)
        s[name + "_scale"][page, :, at] = scale
    return s["q_out"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _plain_read(s):
    b, pos, page, at = _places(s)
    for name in ("k", "v"):
        x = s[name + "_cache"][page, :, at] if s[name + "_scale"] is None else \
            s[name + "_cache"].view(torch.uint8)[page, :, at].view(torch.float8_e4m3fn).float() * s[name + "_scale"][page, :, at][..., None]
        s[name + "_out"][:pos.numel()] = x.to(s[name + "_out"].dtype)
    return s["k_out"], s["v_out"]


def _dense(cache, scale, table):
    """The pages of every sequence side by side: [B, kv heads, positions, head dim] in fp32."""
    B, W = table.shape
    x = cache.view(torch.uint8)[table.long()].view(cache.dtype) if cache.dtype.itemsize == 1 else cache[table.long()]
    x = x.float()
    if scale is not None:
        x *= scale[table.long()][..., None]
    return x.transpose(1, 2).reshape(B, cache.shape[1], W * cache.shape[2], cache.shape[3])


def _plain_attend(s):
    c = s["case"]
    Hq, Hkv, D = c["hq"], c["hkv"], c["dim"]
    G, N, B = Hq // Hkv, s["max_new"], c["batch"]
    k, v = _dense(s["k_cache"], s["k_scale"], s["table"]), _dense(s["v_cache"], s["v_scale"], s["table"])
    L = k.shape[2]
    n = s["indptr"].diff().long()
    i = torch.arange(N, device=DEV)
    real = i[None, :] < n[:, None]                                     # [B, N]
    row = (s["indptr"][:-1, None] + i[None, :]).clamp_max(max(s["q"].shape[0] - 1, 0))
    pos = s["lengths"][:, None] - n[:, None] + i[None, :]
    q = s["q"].float()[row].view(B, N, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, N * G, D)
    w = torch.matmul(q, k.transpose(2, 3)).mul_(1 / math.sqrt(D)).view(B, Hkv, N, G, L)
    j = torch.arange(L, device=DEV)
    keep = (j <= pos[..., None]) & real[..., None]
    if c["window"]:
        keep &= j > pos[..., None] - c["window"]
    w.masked_fill_(~keep[:, None, :, None, :], -math.inf)
    w -= w.amax(dim=-1, keepdim=True).clamp_min(-1e30)
    w = w.exp_()
    total = w.sum(dim=-1, keepdim=True).clamp_min(1e-30)
    v = v.masked_fill((j[None, :] >= s["lengths"][:, None])[:, None, :, None], 0.0)
    o = torch.matmul(w.view(B, Hkv, N * G, L), v).view(B, Hkv, N, G, D) / total
    s["out"][row[real]] = o.permute(0, 2, 1, 3, 4).reshape(B, N, Hq, D)[real].to(s["out"].dtype)
    return s["out"]


def _plain_verify(s):
    c = s["case"]
    N, B, V = s["max_new"], c["batch"], c["vocab"]
    p, q, d = s["target"], s["draft"], s["draft_tokens"]
    rows = p.shape[0]
    r = torch.arange(rows, device=DEV)
    n = s["indptr"].diff().long()
    pd = p[r, d].double()
    qd = q[r, d].double() if q is not None else torch.ones_like(pd)
    ok = s["u_accept"].double() * qd < pd
    i = torch.arange(N, device=DEV)
    row = (s["indptr"][:-1, None] + i[None, :]).clamp_max(max(rows - 1, 0))  # [B, N]
    judged = i[None, :] < n[:, None] - 1
    a = (ok[row] & judged).cumprod(dim=1).sum(dim=1)
    last = row.gather(1, a[:, None].clamp_max(N - 1))[:, 0]
    x = p[last].double()
    rejected = (a < n - 1)[:, None]
    if q is not None:
        x_rej = (x - q[last].double()).clamp_min(0.0)
    else:
        x_rej = x.scatter(1, d[last][:, None], 0.0)
    rejected = rejected & (x_rej.sum(dim=1, keepdim=True) > 0)
    x = torch.where(rejected, x_rej, x)
    cum = x.cumsum(dim=1)
    over = cum > s["u_sample"].double()[:, None] * cum[:, -1:]
    # the first index past the number; the last one with weight where rounding leaves none
    final = torch.where(over.any(dim=1), over.to(torch.uint8).argmax(dim=1), V - 1 - (x > 0).flip(1).to(torch.uint8).argmax(dim=1))
    tok = torch.where(i[None, :] < a[:, None], d[row], torch.where(i[None, :] == a[:, None], final[:, None], -1))
    real = i[None, :] < n[:, None]
    s["tokens"][row[real]] = tok[real]
    s["accepted"].copy_(a)
    return s["tokens"], s["accepted"]


def run(s):
    c = s["case"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "verify": _plain_verify}[c["op"]](s)
    ops = _ops()
    if c["op"] == "write":
        ops.paged_rope_cache(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["indptr"], s["lengths"],
                             THETA, q_out=s["q_out"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        if s["k_scale"] is None:
            return s["q_out"], s["k_cache"], s["v_cache"]
        return s["q_out"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    if c["op"] == "read":
        ops.paged_cache_read(s["k_cache"], s["v_cache"], s["table"], s["indptr"], s["lengths"], s["k_out"], s["v_out"],
                             k_scale=s["k_scale"], v_scale=s["v_scale"])
        return s["k_out"], s["v_out"]
    if c["op"] == "attend":
        return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["indptr"], s["lengths"], s["out"],
                                   1 / math.sqrt(c["dim"]), window=c["window"], max_new=s["max_new"],
                                   k_scale=s["k_scale"], v_scale=s["v_scale"])
    return ops.verify_draft(s["target"], s["draft_tokens"], s["draft"], s["indptr"], s["u_accept"], s["u_sample"],
                            s["tokens"], s["accepted"])


# ------------------------------------------------------------- in 64 bits ----

def _rows64(s, name, b, lo, hi):
    """Positions lo .. hi of sequence b out of the pages, in 64 bits: [hi - lo, kv heads, head dim]."""
    ps = s["case"]["page"]
    where = torch.arange(lo, hi, device=DEV)
    page = s["table"][b].long()[where // ps]
    x = s[name + "_cache"]
    x = x.view(torch.uint8).transpose(1, 2)[page, where % ps].view(x.dtype).double() if x.dtype.itemsize == 1 else \
        x.transpose(1, 2)[page, where % ps].double()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"].double().transpose(1, 2)[page, where % ps][..., None]
    return x


def _exact_write(s):
    c = s["case"]
    new, total = _lens(c)
    D, ps, r = c["dim"], c["page"], 0
    q_out = s["q_out"].double()
    cache = {n: s[n + "_cache"].double() for n in "kv"}
    scale = {n: s[n + "_scale"].double() for n in "kv"} if c["cache"] != "same" else None
    turn = torch.exp(-math.log(THETA) * torch.arange(D // 2, device=DEV, dtype=torch.float64) * 2 / D)
    for b, (n, L) in enumerate(zip(new, total)):
        p = torch.arange(L - n, L, device=DEV)
        z = torch.polar(torch.ones_like(turn)[None].expand(n, -1), p[:, None].double() * turn)[:, None, :]
        def spin(x):
            y = torch.complex(x[..., :D // 2].double(), x[..., D // 2:].double()) * z
            return torch.cat([y.real, y.imag], dim=-1)
        q_out[r:r + n] = spin(s["q"][r:r + n])
        page, at = s["table"][b].long()[p // ps], p % ps
        for name, x in (("k", spin(s["k"][r:r + n])), ("v", s["v"][r:r + n].double())):
            if scale is not None:
                f = torch.clamp(x.abs().max(dim=-1).values / E4M3_MAX, min=MIN_SCALE)
                scale[name][page, :, at] = f
                x = (x / f[..., None]).float().to(torch.float8_e4m3fn).double()
            cache[name][page, :, at] = x
        r += n
    out = [q_out, cache["k"], cache["v"]]
    return out if scale is None else out + [scale["k"], scale["v"]]


def _exact_read(s):
    new, total = _lens(s["case"])
    out = []
    for name in "kv":
        x, r = s[name + "_out"].double(), 0
        for b, (n, L) in enumerate(zip(new, total)):
            x[r:r + n] = _rows64(s, name, b, L - n, L)
            r += n
        out.append(x)
    return out


def _exact_attend(s):
    c = s["case"]
    new, total = _lens(c)
    Hkv, D = c["hkv"], c["dim"]
    G, r = c["hq"] // Hkv, 0
    out = s["out"].double()
    for b, (n, L) in enumerate(zip(new, total)):
        if n:
            lo = max(0, L - n + 1 - c["window"]) if c["window"] else 0
            k, v = _rows64(s, "k", b, lo, L), _rows64(s, "v", b, lo, L)
            p, j = torch.arange(L - n, L, device=DEV)[:, None], torch.arange(lo, L, device=DEV)[None, :]
            gone = (j > p) | ((j <= p - c["window"]) if c["window"] else (j > p))
            for h in range(Hkv):
                q = s["q"][r:r + n, h * G:(h + 1) * G].double()
                x = torch.einsum("ngd,ld->gnl", q, k[:, h]) / math.sqrt(D)
                x = torch.softmax(x.masked_fill(gone, -math.inf), dim=-1)
                out[r:r + n, h * G:(h + 1) * G] = torch.einsum("gnl,ld->ngd", x, v[:, h])
        r += n
    return out


def _exact_verify(s):
    c = s["case"]
    new, _ = _lens(c)
    tokens, accepted, r = s["tokens"].tolist(), [], 0
    p_all, q_all = s["target"], s["draft"]
    d, ua, us = s["draft_tokens"].tolist(), s["u_accept"].tolist(), s["u_sample"].tolist()
    pd = p_all.gather(1, s["draft_tokens"][:, None])[:, 0].tolist() if len(d) else []
    qd = q_all.gather(1, s["draft_tokens"][:, None])[:, 0].tolist() if q_all is not None and len(d) else [1.0] * len(d)
    for b, n in enumerate(new):
        a = 0
        while a < n - 1 and ua[r + a] * qd[r + a] < pd[r + a]:
            a += 1
        accepted.append(a)
        if n:
            p = p_all[r + a].double()
            if a < n - 1:
                left = torch.relu(p - q_all[r + a].double()) if q_all is not None else p.clone()
                if q_all is None:
                    left[d[r + a]] = 0
                p = left if float(left.sum()) > 0 else p
            sums = torch.cumsum(p, dim=0)
            t = int(torch.searchsorted(sums, us[b] * sums[-1], right=True))
            t = t if t < c["vocab"] else int(p.nonzero()[-1])
            tokens[r:r + n] = d[r:r + a] + [t] + [-1] * (n - a - 1)
        r += n
    return torch.tensor(tokens, dtype=torch.int64, device=DEV), torch.tensor(accepted, dtype=torch.int32, device=DEV)


def exact(c, seed):
    s = prepare(c, seed)
    return {"write": _exact_write, "read": _exact_read, "attend": _exact_attend, "verify": _exact_verify}[c["op"]](s)
