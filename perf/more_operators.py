"""The operators of a decode step that stays on the GPU: what is timed, their plain forms and their 64-bit values.

* ``plan``: page tables, row offsets, cache places and adapter slots of the next step's ragged rows, built on the device
  from the sequences' lengths; cut back sequences give their pages back first (``ops.paged_plan``).
* ``write``: rotary embedding of the new rows and the write of their k and v to 8-bit pages with one scale per block of
  tokens and head, a power of two that grows with the block (``ops.paged_rope_cache``).
* ``attend``: causal attention of the new rows over such pages (``ops.paged_attention``).
* ``sample``: the next token of every sequence from its logits and a given random number, each sequence with its own
  temperature, top-k, top-p and min-p (``ops.sample_tokens``).

Sequence b's new tokens are rows indptr[b] .. indptr[b + 1] and sit at its last positions, the last one at
lengths[b] - 1.  Caches are [pages, kv heads, page size, head dim], their scales [pages, kv heads, blocks of a page].
"""

import math
import random
import sys

import torch

own = False

THETA = 1e6  # rotary base of the model configuration
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -40


def _ops():
    if "multi-lora-llm-kernel_b200" not in sys.path:
        sys.path.insert(1, "multi-lora-llm-kernel_b200")
    from persona import ops
    return ops


# ---------------------------------------------------------------- cases ----

def _plan(name, **more):
    """New tokens per sequence new_lo .. new_hi, up to `cut` of the cached ones given up first."""
    c = {"name": name, "op": "plan", "batch": 8, "new_lo": 1, "new_hi": 1, "chunks": 0, "ctx_lo": 0, "ctx_hi": 0, "cut": 0,
         "page": 16, "mix": 0, "pad": 0}
    c.update(more)
    return c


def _paged(name, op, **more):
    """A case over the cache; heads and head size are the model configuration's unless said."""
    c = {"name": name, "op": op, "dtype": "f16", "batch": 8, "new_lo": 1, "new_hi": 1, "chunks": 0, "ctx_lo": 0,
         "ctx_hi": 0, "mix": 0, "hq": 32, "hkv": 8, "dim": 128, "page": 16, "block": 16, "window": 0, "pad": 0}
    c.update(more)
    return c


def _sample(name, **more):
    """`rule`: "all" (temperature alone), "top_p", "top_k", "min_p", or "mixed": every sequence its own of these."""
    c = {"name": name, "op": "sample", "dtype": "f16", "batch": 8, "vocab": 32000, "rule": "top_p", "mix": 0}
    c.update(more)
    return c


def listed():
    return [
        # the step of a small batch: one token each, now and then a new page
        _plan("plan step 8", ctx_lo=128, ctx_hi=255, mix=11),
        # a server's verification step: 256 sequences give up rejected drafts and take up to 8 tokens, padded rows
        _plan("plan drafts 256", batch=256, new_lo=1, new_hi=8, ctx_lo=20, ctx_hi=4000, cut=7, page=32, mix=12, pad=40),
        # the prompts of a prefill batch: 32 of up to 512 tokens, and 16 sequences that decode
        _plan("plan prompts 32", batch=48, chunks=32, new_lo=400, new_hi=512, ctx_lo=10, ctx_hi=900, mix=13),
        # one decode step of 64 sequences, blocks of 16 partly filled, bf16
        _paged("write step 64", "write", dtype="bf16", batch=64, ctx_lo=100, ctx_hi=4000, page=64, mix=14, pad=2),
        # ragged prompts of a prefill batch, 9 to 10 thousand rows, pages of one block
        _paged("write prompts 20 ragged", "write", batch=20, new_lo=37, new_hi=1000, ctx_hi=90, page=32, block=32, mix=15),
        # the decode step of a small batch at short lengths: all latency
        _paged("attend step 8", "attend", ctx_lo=128, ctx_hi=255, mix=16),
        # a decode step of a full server: 64 ragged sequences of up to 8192 tokens
        _paged("attend step 64 long", "attend", dtype="bf16", batch=64, ctx_lo=500, ctx_hi=8191, page=32, block=32, mix=17),
        # verification of drafted tokens, 32 sequences of 5 fed tokens
        _paged("attend drafts 32x5", "attend", batch=32, new_lo=5, new_hi=5, ctx_lo=300, ctx_hi=6000, page=64, mix=18),
        # prompt chunks beside decoding sequences, a sliding window, padded rows
        _paged("attend mixed", "attend", dtype="bf16", batch=9, new_hi=1400, chunks=2, ctx_lo=700, ctx_hi=3500, page=64,
               block=64, window=2048, mix=19, pad=5),
        # 8 requests of the engine's batch, nucleus sampling over the model configuration's vocabulary
        _sample("sample 8 top-p"),
        # a full server, every request with its own parameters, a vocabulary of odd size
        _sample("sample 256 mixed", batch=256, vocab=50257, rule="mixed", mix=21),
        # fp32 logits of a large vocabulary, nothing cut: every token counts
        _sample("sample 64 all f32", dtype="f32", batch=64, vocab=130001, rule="all", mix=22),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "write", "attend", "attend", "sample", "sample"])
    mix = rng.randrange(1 << 30)
    if op == "plan":
        c = _plan("", batch=_log(rng, 1, 600), page=rng.choice([16, 32, 64, 24, 8, 1]), mix=mix, pad=rng.randrange(50))
        c["new_lo"] = rng.randint(0, 1)
        c["new_hi"] = _log(rng, 1, max(1, 24000 // c["batch"]))
        c["ctx_hi"] = _log(rng, 1, max(2, min(6000, 100000 * c["page"] // (16 * c["batch"]))))
        c["cut"] = rng.choice([0, 3, 40])
    elif op == "sample":
        c = _sample("", dtype=rng.choice(["f16", "bf16", "f32"]), batch=_log(rng, 1, 256), mix=mix,
                    rule=rng.choice(["all", "top_p", "top_k", "min_p", "mixed", "mixed"]))
        c["vocab"] = _log(rng, 50, min(150000, 8000000 // c["batch"]))
    else:
        hkv, group = rng.choice([(8, 4), (8, 4), (2, 2), (1, 8), (4, 7), (16, 1), (5, 3)])
        page = rng.choice([16, 32, 64, 128, 24, 48])
        c = _paged("", op, dtype=rng.choice(["f16", "bf16"]), mix=mix, hkv=hkv, hq=hkv * group,
                   dim=rng.choice([64, 128, 128]), page=page, pad=rng.randrange(4),
                   block=rng.choice([b for b in (8, 16, 32, 64, 128) if page % b == 0]))
        if op == "attend" and rng.random() < 0.3:  # prompt chunks, some with decoding sequences beside them
            c["batch"] = rng.randint(1, 6)
            c["new_lo"], c["new_hi"] = 1, _log(rng, 33, 1400)
            c["chunks"] = rng.randint(0, c["batch"])
            c["ctx_lo"], c["ctx_hi"] = 0, _log(rng, 1, 6000)
        elif op == "attend":  # decoding and drafted tokens
            c["batch"] = _log(rng, 1, 64)
            c["new_lo"] = rng.randint(0, 1)
            c["new_hi"] = rng.choice([1, 1, rng.randint(2, 9)])
            c["ctx_hi"] = _log(rng, 20, max(200, min(16000, 200000 // c["batch"])))
            c["ctx_lo"] = rng.choice([0, c["ctx_hi"] // 20, c["ctx_hi"] // 2])
        else:
            c["batch"] = _log(rng, 1, 64)
            c["new_hi"] = _log(rng, 1, max(2, 9000 // c["batch"]))
            c["new_lo"] = rng.choice([0, 1, (c["new_hi"] + 1) // 2])
            c["ctx_lo"], c["ctx_hi"] = 0, _log(rng, 1, 1000)
        if op == "attend" and rng.random() < 0.3:
            c["window"] = _log(rng, 5, 4096)
    del c["name"]
    return c


def _lens(c):
    """New tokens and cached ones of each sequence: the same for every seed.  Where `chunks` is not 0 that many sequences
    have many new tokens, the others one."""
    rng = random.Random(c["mix"])
    new, ctx = [], []
    for b in range(c["batch"]):
        if c["chunks"]:
            n = rng.randint(max(c["new_lo"], c["new_hi"] * 2 // 3), c["new_hi"]) if b < c["chunks"] else 1
        else:
            n = rng.randint(c["new_lo"], c["new_hi"]) if c["new_hi"] < 40 else _log(rng, max(1, c["new_lo"]), c["new_hi"])
        new.append(max(n, 1) if b == 0 else n)
        ctx.append(rng.randint(c["ctx_lo"], c["ctx_hi"]) if c["ctx_hi"] < 4 else _log(rng, max(1, c["ctx_lo"]), c["ctx_hi"]))
    return new, ctx


def work(c):
    if c["op"] == "sample":
        e = 4 if c["dtype"] == "f32" else 2
        n = c["batch"] * c["vocab"]
        return {"bytes": n * e + c["batch"] * (4 + 16 + 8), "flops": 4.0 * n}
    new, ctx = _lens(c)
    rows = sum(new)
    if c["op"] == "plan":
        ps = c["page"]
        pages = sum(-(-(n + L) // ps) - -(-L // ps) for n, L in zip(new, ctx))
        # new, keep, lengths in and out, row offsets, adapter slots; a place and a slot per row; a page in and out
        return {"bytes": c["batch"] * 24 + (rows + c["pad"]) * 12 + pages * 8, "flops": 0}
    kv = c["hkv"] * (c["dim"] + 4 / c["block"]) * 2  # one position's k and v in the cache, with its share of the scales
    row = c["dim"] * 2
    if c["op"] == "write":
        return {"bytes": rows * (2 * c["hq"] * row + 2 * c["hkv"] * row + kv), "flops": 3.0 * rows * (c["hq"] + c["hkv"]) * c["dim"]}
    pairs = seen = 0
    for n, first in zip(new, ctx):
        L = first + n
        w = c["window"] or L
        pairs += sum(min(p + 1, w) for p in range(first, L))
        seen += L - max(0, first + 1 - w) if n else 0
    return {"bytes": seen * kv + 2 * rows * c["hq"] * row, "flops": 4.0 * pairs * c["hq"] * c["dim"]}


# --------------------------------------------------------------- inputs ----

def _gen(c, seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + c["mix"] % 1000003)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _table(g, per, spare, width):
    """A page table whose sequences hold per[b] pages of a shuffled pool, and the pages that are left."""
    perm = torch.randperm(sum(per) + spare, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(per), width, dtype=torch.int32, device=DEV)
    have = torch.arange(width, device=DEV)[None, :] < torch.tensor(per, device=DEV)[:, None]
    table[have] = perm[:sum(per)]
    return table, perm[sum(per):]


def _prepare_plan(c, seed):
    g = _gen(c, seed)
    new, keep = _lens(c)
    ps, B = c["page"], c["batch"]
    rng = random.Random(int(seed) * 7 + 1)
    length = [k + rng.randint(0, c["cut"]) for k in keep]
    held = [-(-n // ps) for n in length]
    most = [-(-(k + max(n, c["cut"])) // ps) for k, n in zip(keep, new)]
    table, pool = _table(g, held, sum(most) + 5 - sum(held), max(most + [1]))
    free = pool.numel()
    pool = torch.cat([pool, pool.new_zeros(sum(held))])
    rows = sum(new) + c["pad"]
    return {"case": c, "new": _i32(new), "keep": _i32(keep), "lengths": _i32(length), "table": table, "free": pool,
            "num_free": _i32([free]), "indptr": torch.zeros(B + 1, dtype=torch.int32, device=DEV),
            "places": torch.zeros(rows, dtype=torch.int64, device=DEV),
            "row_slots": torch.zeros(rows, dtype=torch.int32, device=DEV),
            "seq_slots": torch.randint(-1, 8, (B,), generator=g, device=DEV, dtype=torch.int32)}


def _prepare_paged(c, seed):
    g = _gen(c, seed)
    new, ctx = _lens(c)
    total = [n + x for n, x in zip(new, ctx)]
    rows, ps, blk = sum(new) + c["pad"], c["page"], c["block"]
    Hq, Hkv, D, dt = c["hq"], c["hkv"], c["dim"], TYPES[c["dtype"]]
    per = [-(-L // ps) for L in total]
    table, free = _table(g, per, 3, max(max(per), 1))
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s = {"case": c, "max_new": max(max(new), 1), "rows": sum(new), "table": table, "indptr": _i32(starts), "lengths": _i32(total)}
    pages = sum(per) + free.numel()
    for name in ("k", "v"):
        x = torch.randn(pages, Hkv, ps, D, generator=g, device=DEV)
        # blocks of different size, so that new tokens outgrow some of them
        x *= torch.exp2(-torch.randint(0, 4, (pages, Hkv, ps // blk, 1, 1), generator=g, device=DEV).float()).expand(
            -1, -1, -1, blk, -1).reshape(pages, Hkv, ps, 1)
        scale = _two_power(x.view(pages, Hkv, ps // blk, -1).abs().amax(dim=-1))
        s[name + "_cache"] = (x / scale.repeat_interleave(blk, dim=2)[..., None]).to(E4M3)
        s[name + "_scale"] = scale
        del x
    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEV).to(dt)
    if c["op"] == "write":
        s["q"], s["k"], s["v"] = rand(rows, Hq, D), rand(rows, Hkv, D), rand(rows, Hkv, D)
        s["q_out"] = torch.zeros_like(s["q"])
    else:
        s["q"] = (torch.randn(rows, Hq, D, generator=g, device=DEV) * 1.5).to(dt)
        s["out"] = torch.zeros_like(s["q"])
    return s


def _prepare_sample(c, seed):
    g = _gen(c, seed)
    B, V = c["batch"], c["vocab"]
    # a model's logits: most tokens far below a few that fit
    z = torch.randn(B, V, generator=g, device=DEV) * 2.5
    best = torch.randint(0, V, (B, 24), generator=g, device=DEV)
    z.scatter_add_(1, best, 4 + 5 * torch.rand(B, 24, generator=g, device=DEV))
    rng = random.Random(int(seed) * 13 + c["mix"])
    t, k, p, m = [], [], [], []
    for _ in range(B):
        rule = rng.choice(["all", "top_p", "top_k", "min_p", "both", "greedy"]) if c["rule"] == "mixed" else c["rule"]
        t.append(0.0 if rule == "greedy" else rng.choice([0.6, 0.8, 1.0, 1.3]))
        k.append(rng.choice([1, 5, 20, 50, 300]) if rule in ("top_k", "both") else 0)
        p.append(rng.choice([0.5, 0.8, 0.9, 0.95, 0.99]) if rule in ("top_p", "both") else 1.0)
        m.append(rng.choice([0.01, 0.05, 0.2]) if rule in ("min_p", "both") else 0.0)
    def f32(v):
        return torch.tensor(v, dtype=torch.float32, device=DEV)
    return {"case": c, "logits": z.to(TYPES[c["dtype"]]), "u": torch.rand(B, generator=g, device=DEV), "temperature": f32(t),
            "top_k": _i32(k) if any(k) else None, "top_p": f32(p) if min(p) < 1 else None,
            "min_p": f32(m) if any(m) else None, "tokens": torch.zeros(B, dtype=torch.int64, device=DEV)}


def prepare(c, seed):
    return {"plan": _prepare_plan, "sample": _prepare_sample}.get(c["op"], _prepare_paged)(c, seed)


# ----------------------------------------------------------- plain forms ----

def _plain_plan(s):
    """A step that can be made (one that cannot changes nothing, and is not among the cases)."""
    ps, table, free = s["case"]["page"], s["table"], s["free"]
    B, W = table.shape
    keep, new = s["keep"].long(), s["new"].long()
    held, kept = (s["lengths"].long() + ps - 1) // ps, (keep + ps - 1) // ps
    length = keep + new
    need = (length + ps - 1) // ps
    j = torch.arange(W, device=DEV)[None, :]
    # pages given back: the last sequence's last page first, so that the pages are taken again in their old order
    back = (j >= kept[:, None]) & (j < held[:, None])
    order = back.flatten().flip(0).cumsum(0).flip(0) - 1
    spill = free.numel()  # an entry behind the pool takes what is not meant
    pool = torch.cat([free, free.new_zeros(1)])
    pool.scatter_(0, torch.where(back.flatten(), s["num_free"].long() + order, spill), table.flatten())
    top = s["num_free"].long() + back.sum()
    take = (j >= kept[:, None]) & (j < need[:, None])
    nth = take.flatten().cumsum(0) - 1
    got = pool[(top - 1 - nth).clamp(0, spill)].view(B, W)
    s["table"].copy_(torch.where(take, got, table))
    free.copy_(pool[:spill])
    s["num_free"].copy_(top - take.sum())
    s["lengths"].copy_(length)
    s["indptr"][1:] = new.cumsum(0)
    rows = s["places"].numel()
    r = torch.arange(rows, device=DEV)
    b = torch.searchsorted(s["indptr"][1:].long(), r, right=True)
    real = b < B
    b = b.clamp_max(B - 1)
    pos = length[b] - (s["indptr"][b + 1].long() - r)
    at = s["table"][b, (pos // ps).clamp(0, W - 1)].long() * ps + pos % ps
    s["places"].copy_(torch.where(real, at, -1))
    s["row_slots"].copy_(torch.where(real, s["seq_slots"][b].long(), -1))
    return _plan_out(s)


def _plan_out(s):
    return s["lengths"], s["table"], s["free"], s["num_free"], s["indptr"], s["places"], s["row_slots"]


def _two_power(amax):
    """The smallest power of two that brings amax to at most 448, and 2^-40 at least."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1)
    e = e - 9 + (m > 0.875)   # 448 = 0.875 * 2^9
    return torch.exp2(e.clamp_min(-40).to(amax.dtype))


def _places(s):
    """For every new row: its sequence, position, page and place in the page."""
    n, rows = s["indptr"].diff().long(), s["rows"]
    b = torch.repeat_interleave(torch.arange(n.numel(), device=DEV), n, output_size=rows)
    pos = torch.arange(rows, device=DEV) - s["indptr"][b] + (s["lengths"][b] - n[b])
    ps = s["case"]["page"]
    return b, pos, s["table"][b, pos // ps].long(), pos % ps


def _rotate(x, pos):
    """Rotate-half rotary embedding: the angles in 64 bits, the products in 32."""
    D = x.shape[-1]
    inv = THETA ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    ang = pos[:, None].double() * inv[None, :]
    cs, sn = ang.cos().float()[:, None, :], ang.sin().float()[:, None, :]
    lo, hi = x[..., :D // 2].float(), x[..., D // 2:].float()
    return torch.cat([lo * cs - hi * sn, hi * cs + lo * sn], dim=-1)


def _plain_write(s):
    c = s["case"]
    ps, blk, D = c["page"], c["block"], c["dim"]
    b, pos, page, at = _places(s)
    R = pos.numel()
    s["q_out"][:R] = _rotate(s["q"][:R], pos).to(s["q"].dtype)
    n = s["indptr"].diff().long()
    first = torch.maximum((s["lengths"].long() - n)[b], pos // blk * blk)  # the first new position of the row's block
    lead = pos == first                # one row for every block with new tokens
    nth = lead.cumsum(0) - 1
    pg, bl, older = page[lead], at[lead] // blk, first[lead] % blk  # `older` tokens of the block came before
    place = bl[:, None] * blk + torch.arange(blk, device=DEV)
    for x, name in ((_rotate(s["k"][:R], pos), "k"), (s["v"][:R].float(), "v")):
        cache, scale = s[name + "_cache"].view(torch.uint8), s[name + "_scale"]
        H, K = cache.shape[1], pg.numel()
        amax = torch.zeros(K, H, device=DEV).scatter_reduce_(0, nth[:, None].expand(-1, H), x.abs().amax(dim=-1), "amax")
        old = scale[pg, :, bl]
        now = torch.maximum(torch.where(older[:, None] > 0, old, 0.0), _two_power(amax))
        codes = cache[pg[:, None], :, place]  # [blocks, places, heads, head dim]
        again = (codes.view(E4M3).float() * (old / now)[:, None, :, None]).to(E4M3).view(torch.uint8)
        before = torch.arange(blk, device=DEV)[None, :] < older[:, None]
        cache[pg[:, None], :, place] = torch.where(before[:, :, None, None], again, codes)
        cache[page, :, at] = (x / now[nth][..., None]).to(E4M3).view(torch.uint8)
        scale[pg, :, bl] = now
    return s["q_out"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _dense(cache, scale, table, blk):
    """The pages of every sequence side by side: [B, kv heads, positions, head dim] in fp32."""
    B, W = table.shape
    x = cache.view(torch.uint8)[table.long()].view(E4M3).float()
    x *= scale[table.long()].repeat_interleave(blk, dim=-1)[..., None]
    return x.transpose(1, 2).reshape(B, cache.shape[1], W * cache.shape[2], cache.shape[3])


def _plain_attend(s):
    c = s["case"]
    Hq, Hkv, D = c["hq"], c["hkv"], c["dim"]
    G, N, B = Hq // Hkv, s["max_new"], c["batch"]
    k, v = (_dense(s[x + "_cache"], s[x + "_scale"], s["table"], c["block"]) for x in "kv")
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


def _plain_sample(s):
    """In 64 bits: the draw falls between two sums over the vocabulary."""
    x = s["logits"].double()
    B, V = x.shape
    i = torch.arange(V, device=DEV)[None, :]
    t = s["temperature"].double()[:, None]
    top = x.amax(dim=1, keepdim=True)
    w = ((x - top) / torch.where(t > 0, t, 1.0)).exp()
    if s["top_k"] is not None or s["top_p"] is not None:
        _, order = torch.sort(s["logits"], dim=1, descending=True, stable=True)
        ws = w.gather(1, order)
        keep = torch.ones_like(ws, dtype=torch.bool)
        if s["top_k"] is not None:
            k = s["top_k"].long()[:, None]
            keep = (i < k) | (k <= 0)
        if s["top_p"] is not None:
            p = s["top_p"].double()[:, None]
            ws = ws * keep
            upto = ws.cumsum(dim=1)
            keep &= (upto - ws <= p * upto[:, -1:]) | (p >= 1)
        w = w * torch.zeros_like(keep).scatter_(1, order, keep)
    if s["min_p"] is not None:
        w = w * (w >= s["min_p"].double()[:, None])
    cum = w.cumsum(dim=1)
    over = cum > s["u"].double()[:, None] * cum[:, -1:]
    draw = torch.where(over, i, V).amin(dim=1)
    last = torch.where(w > 0, i, -1).amax(dim=1)
    best = torch.where(x == top, i, V).amin(dim=1)
    s["tokens"].copy_(torch.where(t[:, 0] > 0, torch.where(draw < V, draw, last), best))
    return s["tokens"]


def run(s):
    c = s["case"]
    if not own:
        return {"plan": _plain_plan, "write": _plain_write, "attend": _plain_attend, "sample": _plain_sample}[c["op"]](s)
    ops = _ops()
    if c["op"] == "plan":
        ops.paged_plan(s["new"], s["lengths"], s["table"], s["free"], s["num_free"], c["page"], s["indptr"], s["places"],
                       keep=s["keep"], seq_slots=s["seq_slots"], row_slots=s["row_slots"])
        return _plan_out(s)
    if c["op"] == "write":
        ops.paged_rope_cache(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["indptr"], s["lengths"],
                             THETA, q_out=s["q_out"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return s["q_out"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    if c["op"] == "attend":
        return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["indptr"], s["lengths"], s["out"],
                                   1 / math.sqrt(c["dim"]), window=c["window"], max_new=s["max_new"],
                                   k_scale=s["k_scale"], v_scale=s["v_scale"])
    return ops.sample_tokens(s["logits"], s["u"], s["tokens"], temperature=s["temperature"], top_k=s["top_k"],
                             top_p=s["top_p"], min_p=s["min_p"])


# ------------------------------------------------------------- in 64 bits ----

def _exact_plan(s):
    ps = s["case"]["page"]
    new, keep, length, slots = (s[x].tolist() for x in ("new", "keep", "lengths", "seq_slots"))
    table, pool, free = s["table"].tolist(), s["free"].tolist(), int(s["num_free"])
    for b in reversed(range(len(new))):
        for j in reversed(range(-(-keep[b] // ps), -(-length[b] // ps))):
            pool[free] = table[b][j]
            free += 1
    indptr, places, row_slots = [0], [], []
    for b, n in enumerate(new):
        for j in range(-(-keep[b] // ps), -(-(keep[b] + n) // ps)):
            free -= 1
            table[b][j] = pool[free]
        length[b] = keep[b] + n
        indptr.append(indptr[-1] + n)
        places += [table[b][p // ps] * ps + p % ps for p in range(keep[b], length[b])]
        row_slots += [slots[b]] * n
    short = s["places"].numel() - len(places)
    return (_i32(length), _i32(table).view(s["table"].shape), _i32(pool), _i32([free]), _i32(indptr),
            torch.tensor(places + [-1] * short, dtype=torch.int64, device=DEV), _i32(row_slots + [-1] * short))


def _exact_write(s):
    c = s["case"]
    new, ctx = _lens(c)
    D, ps, blk, r = c["dim"], c["page"], c["block"], 0
    q_out = s["q_out"].double()
    cache = {n: s[n + "_cache"].double() for n in "kv"}
    scale = {n: s[n + "_scale"].double() for n in "kv"}
    turn = torch.exp(-math.log(THETA) * torch.arange(D // 2, device=DEV, dtype=torch.float64) * 2 / D)
    for b, (n, at0) in enumerate(zip(new, ctx)):
        p = torch.arange(at0, at0 + n, device=DEV)
        z = torch.polar(torch.ones_like(turn)[None].expand(n, -1), p[:, None].double() * turn)[:, None, :]
        def spin(x):
            y = torch.complex(x[..., :D // 2].double(), x[..., D // 2:].double()) * z
            return torch.cat([y.real, y.imag], dim=-1)
        q_out[r:r + n] = spin(s["q"][r:r + n])
        pages = s["table"][b].tolist()
        for name, x in (("k", spin(s["k"][r:r + n])), ("v", s["v"][r:r + n].double())):
            lo = at0
            while lo < at0 + n:  # block by block
                start = lo // blk * blk
                hi = min(start + blk, at0 + n)
                pg, i = pages[lo // ps], lo % ps
                y = x[lo - at0:hi - at0].transpose(0, 1)  # [kv heads, tokens, head dim]
                f = torch.exp2(torch.ceil(torch.log2(y.abs().amax(dim=(1, 2)) / E4M3_MAX))).clamp_min(MIN_SCALE)
                if lo > start:
                    f = torch.maximum(f, scale[name][pg, :, i // blk])
                    older = cache[name][pg, :, start % ps:i]
                    cache[name][pg, :, start % ps:i] = (older * (scale[name][pg, :, i // blk] / f)[:, None, None]).float().to(E4M3).double()
                scale[name][pg, :, i // blk] = f
                cache[name][pg, :, i:i + hi - lo] = (y / f[:, None, None]).float().to(E4M3).double()
                lo = hi
        r += n
    return q_out, cache["k"], cache["v"], scale["k"], scale["v"]


def _rows64(s, name, b, lo, hi):
    """Positions lo .. hi of sequence b out of the pages, in 64 bits: [hi - lo, kv heads, head dim]."""
    ps, blk = s["case"]["page"], s["case"]["block"]
    where = torch.arange(lo, hi, device=DEV)
    page = s["table"][b].long()[where // ps]
    x = s[name + "_cache"].view(torch.uint8).transpose(1, 2)[page, where % ps].view(E4M3).double()
    return x * s[name + "_scale"].double().transpose(1, 2)[page, where % ps // blk][..., None]


def _exact_attend(s):
    c = s["case"]
    new, ctx = _lens(c)
    Hkv, D = c["hkv"], c["dim"]
    G, r = c["hq"] // Hkv, 0
    out = s["out"].double()
    for b, (n, first) in enumerate(zip(new, ctx)):
        L = first + n
        if n:
            lo = max(0, first + 1 - c["window"]) if c["window"] else 0
            k, v = _rows64(s, "k", b, lo, L), _rows64(s, "v", b, lo, L)
            p, j = torch.arange(first, L, device=DEV)[:, None], torch.arange(lo, L, device=DEV)[None, :]
            gone = (j > p) | ((j <= p - c["window"]) if c["window"] else (j > p))
            for h in range(Hkv):
                q = s["q"][r:r + n, h * G:(h + 1) * G].double()
                x = torch.einsum("ngd,ld->gnl", q, k[:, h]) / math.sqrt(D)
                x = torch.softmax(x.masked_fill(gone, -math.inf), dim=-1)
                out[r:r + n, h * G:(h + 1) * G] = torch.einsum("gnl,ld->ngd", x, v[:, h])
        r += n
    return out


def _exact_sample(s):
    B, V = s["logits"].shape
    def of(name, none):
        return [none] * B if s[name] is None else s[name].double().tolist()
    t, k, p, m, u = of("temperature", 1.0), of("top_k", 0), of("top_p", 1.0), of("min_p", 0.0), s["u"].double().tolist()
    tokens = []
    for b in range(B):
        z = s["logits"][b].double()
        order = torch.argsort(-z, stable=True)  # the likeliest token first, equal ones by their index
        if not t[b] > 0:
            tokens.append(int(order[0]))
            continue
        if k[b] > 0:
            order = order[:int(k[b])]
        prob = torch.softmax(z[order] / t[b], dim=0)
        sums = torch.cumsum(prob, dim=0)
        n = order.numel()
        if p[b] < 1:
            n = 1 + int((sums[:-1] <= p[b] * sums[-1]).sum())
        n = min(n, int((prob >= m[b] * prob[0]).sum()))
        kept, _ = torch.sort(order[:n])
        weight = torch.zeros(V, dtype=torch.float64, device=DEV)
        weight[order[:n]] = prob[:n]
        sums = torch.cumsum(weight[kept], dim=0)
        tokens.append(int(kept[min(int(torch.searchsorted(sums, u[b] * sums[-1], right=True)), n - 1)]))
    return torch.tensor(tokens, dtype=torch.int64, device=DEV)


def exact(c, seed):
    s = prepare(c, seed)
    return {"plan": _exact_plan, "write": _exact_write, "attend": _exact_attend, "sample": _exact_sample}[c["op"]](s)
