"""A Mistral-7B-architecture decoder whose base linears are NF4 and whose
seven projections carry per-row LoRA adapters from an ``AdapterPool``: the
model the end-to-end mixed-adapter decode runs.

The reference loads the real Mistral-7B through Hugging Face with
bitsandbytes NF4 (reference ``bench/e2e.py:70-90``), patches the projections
with ``MultiLoRALinear`` (``persona/model_patch.py``) and decodes with
``model.generate`` (``persona/engine.py:101-107``).  Here the weights are
random (N(0, 0.02), as for a freshly initialised model; norms are ones), the
architecture is the same (RMSNorm, rotary embedding with base 1e6, grouped
query attention, SwiGLU MLP, untied fp16 LM head) and every step runs this
package's kernels:

* base projections: ``nf4.linear`` (one launch for q / k / v, one for gate /
  up, one each for o and down);
* LoRA: ``ops.bgmv_fused_multi`` on a plan computed once per batch at decode;
  ``ops.sgmv_fused`` over the request segments at prefill;
* ragged chunks over a paged cache (``extend``): ``ops.paged_rope_cache`` and
  ``ops.paged_attention``, LoRA over the sequences as segments; single tokens
  over it (``start_decode``, ``paged_step``) in a captured step that finds its
  pages by ``ops.paged_plan`` and its tokens by ``ops.sample_tokens``;
* the rest: ``ops.add_rmsnorm`` (residual add fused into the
  next norm), ``rope_cache`` (rotary embedding + KV-cache write) at prefill,
  ``rope_decode_attention`` (the same and the attention, one launch) at
  decode, ``silu_mul``; the LM head and the prefill attention are library
  calls (cuBLAS, scaled_dot_product_attention).

A decode step has fixed shapes and reads the position from device memory,
so it is captured once as a CUDA graph and replayed for every token.
"""

from __future__ import annotations

import functools
import math
from dataclasses import dataclass, field
from typing import List, Optional, Sequence

import torch
import torch.nn.functional as F

from persona import nf4, ops
from persona.adapter_pool import AdapterPool
from persona.sampling import BatchSampling

def on_its_device(method):
    """The method runs with ``self.device`` as the current device: graphs are
    captured and replayed, and events recorded, on the current device's streams."""

    @functools.wraps(method)
    def call(self, *args, **kwargs):
        with torch.cuda.device(self.device):
            return method(self, *args, **kwargs)

    return call


@dataclass
class MistralConfig:
    num_layers: int = 32
    hidden: int = 4096
    n_heads: int = 32
    n_kv_heads: int = 8
    head_dim: int = 128
    intermediate: int = 14336
    vocab: int = 32000
    rope_theta: float = 1e6
    rms_eps: float = 1e-5

    @property
    def q_dim(self) -> int:
        return self.n_heads * self.head_dim

    @property
    def kv_dim(self) -> int:
        return self.n_kv_heads * self.head_dim


@dataclass
class LayerWeights:
    in_norm: torch.Tensor
    post_norm: torch.Tensor
    q: nf4.NF4Weight
    k: nf4.NF4Weight
    v: nf4.NF4Weight
    o: nf4.NF4Weight
    gate: nf4.NF4Weight
    up: nf4.NF4Weight
    down: nf4.NF4Weight


@dataclass
class DecodeState:
    """Static buffers of one batch (CUDA-graph friendly)."""

    B: int
    max_seq: int
    tok: torch.Tensor             # [B] int64: the token each row feeds next
    pos: torch.Tensor             # [1] int32: its position
    length: torch.Tensor          # [1] int32: pos + 1
    slots: torch.Tensor           # [B] int32 adapter slot per row
    plan: torch.Tensor            # BGMV plan of ``slots``
    k_cache: List[torch.Tensor]   # per layer [B, Hkv, max_seq, 128]
    v_cache: List[torch.Tensor]
    bufs: dict = field(default_factory=dict)
    graph: Optional[torch.cuda.CUDAGraph] = None


@dataclass
class PagedState:
    """A batch over a paged KV cache: sequences of any lengths, which grow by
    chunks (prompt chunks, single tokens, drafted tokens)."""

    slots: torch.Tensor           # [B] int32 adapter slot per sequence
    page_size: int
    page_table: torch.Tensor      # [B, max_pages] int32
    k_cache: List[torch.Tensor]   # per layer [pages, Hkv, page_size, 128], fp16 or e4m3
    v_cache: List[torch.Tensor]
    k_scale: List[Optional[torch.Tensor]]  # per layer [pages, Hkv, page_size or blocks of a page], e4m3 only
    v_scale: List[Optional[torch.Tensor]]
    lengths: List[int]            # cached tokens per sequence
    pages: List[List[int]]        # pages held by each sequence
    free: List[int]
    decode: Optional["PagedDecode"] = field(default=None, repr=False, compare=False)  # while the device keeps the lengths and the pages

    def _host(self) -> None:
        if self.decode is not None:
            raise ValueError("the sequences are being decoded (finish_decode first)")

    def set_length(self, b: int, length: int) -> None:
        """Sequence b keeps its first ``length`` tokens (rejected drafts, or 0
        to start over); pages behind them are free again."""
        self._host()
        if not 0 <= length <= self.lengths[b]:
            raise ValueError("a sequence can only be cut back")
        keep = -(-length // self.page_size)
        self.free.extend(self.pages[b][keep:])
        del self.pages[b][keep:]
        self.lengths[b] = length

    def _back_to(self, lengths: Sequence[int], held: Sequence[int]) -> None:
        """The state of before a ``_grow``: lengths, and pages held by each sequence."""
        for b in reversed(range(len(held))):  # (in the order that takes them out alike again)
            self.free.extend(reversed(self.pages[b][held[b]:]))
            del self.pages[b][held[b]:]
        self.lengths[:] = lengths

    def _grow(self, new: Sequence[int]) -> None:
        """Pages for ``new`` more tokens per sequence; lengths are moved on."""
        want = [-(-(n + add) // self.page_size) for n, add in zip(self.lengths, new)]
        if any(w > self.page_table.shape[1] for w in want):
            raise ValueError("a sequence outgrows its page table")
        if sum(w - len(p) for w, p in zip(want, self.pages)) > len(self.free):
            raise ValueError("the paged cache has no free pages left")
        table = None
        for b, w in enumerate(want):
            while len(self.pages[b]) < w:
                self.pages[b].append(self.free.pop())
                table = True
            self.lengths[b] += new[b]
        if table:
            host = torch.zeros(self.page_table.shape, dtype=torch.int32)
            for b, p in enumerate(self.pages):
                host[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
            self.page_table.copy_(host)


@dataclass
class PagedDecode:
    """A ``PagedState`` whose next tokens are made one a step without the host:
    lengths, pages and free list are device arrays that the step itself moves on."""

    st: PagedState
    sampling: BatchSampling
    tok: torch.Tensor       # [B + 1] int64: the token that each sequence feeds next (and a place for padded rows)
    alive: torch.Tensor     # [B] int32: 1 gets a token a step; 0 has ended, its pages go back with the next step
                            # (so has one whose token is none of the vocabulary, -1 say: nothing could be drawn)
    u: torch.Tensor         # [B] fp32: the numbers that the next step draws with
    lengths: torch.Tensor   # [B] int32
    keep: torch.Tensor      # [B] int32
    free: torch.Tensor      # [pages] int32, the first num_free of them free
    num_free: torch.Tensor  # [1] int32
    indptr: torch.Tensor    # [B + 1] int32
    places: torch.Tensor    # [B] int64
    seqs: torch.Tensor      # [B] int32: 0 .. B - 1
    row_seq: torch.Tensor   # [B] int32: the sequence of each row, -1 behind the last
    out: torch.Tensor       # [B + 1] int64: what the last step drew by sequence (and a place for padded rows)
    bufs: dict = field(default_factory=dict)
    graph: Optional[torch.cuda.CUDAGraph] = None

    def _moved(self) -> list:
        """What a step moves on, beside the pages' contents behind the lengths."""
        return [self.tok, self.alive, self.lengths, self.st.page_table, self.free, self.num_free]


class MistralLoRAModel:
    """Random-init Mistral-architecture decoder with NF4 base weights."""

    def __init__(self, cfg: MistralConfig, pool: AdapterPool, device, seed: int = 0):
        if pool.num_layers != cfg.num_layers:
            raise ValueError("adapter pool and model disagree on the layer count")
        if cfg.head_dim != 128:
            raise ValueError("the decode kernels take head_dim 128")
        self.cfg = cfg
        self.pool = pool
        self.device = torch.device(device)
        g = torch.Generator(device=self.device)
        g.manual_seed(seed)
        h, d = cfg.hidden, self.device
        self.embed = (torch.randn(cfg.vocab, h, generator=g, device=d) * 0.02).half()
        self.layers: List[LayerWeights] = []
        for _ in range(cfg.num_layers):
            def q(n_out, n_in):
                w = (torch.randn(n_out, n_in, generator=g, device=d) * 0.02).half()
                return nf4.quantize(w)

            self.layers.append(LayerWeights(
                in_norm=torch.ones(h, dtype=torch.float16, device=d),
                post_norm=torch.ones(h, dtype=torch.float16, device=d),
                q=q(cfg.q_dim, h), k=q(cfg.kv_dim, h), v=q(cfg.kv_dim, h), o=q(h, cfg.q_dim),
                gate=q(cfg.intermediate, h), up=q(cfg.intermediate, h), down=q(h, cfg.intermediate)))
        self.final_norm = torch.ones(h, dtype=torch.float16, device=d)
        self.lm_head = (torch.randn(cfg.vocab, h, generator=g, device=d) * 0.02).half()
        self._lora = [self._lora_pools(i) for i in range(cfg.num_layers)]

    # ---- weights ---------------------------------------------------------
    def _lora_pools(self, layer: int):
        p = self.pool
        mods = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")
        return {m: (p.a_pool(layer, m), p.b_pool(layer, m)) for m in mods}

    def base_bytes(self) -> int:
        """HBM bytes of the weights one decode step streams (NF4 + head)."""
        n = sum(w.nbytes for lw in self.layers for w in (lw.q, lw.k, lw.v, lw.o, lw.gate, lw.up, lw.down))
        return n + self.lm_head.numel() * 2

    # ---- batch state -------------------------------------------------------
    def new_state(self, slots: torch.Tensor, max_seq: int) -> DecodeState:
        cfg, d = self.cfg, self.device
        B = int(slots.numel())
        slots = slots.to(d, torch.int32).contiguous()
        plan = ops.bgmv_plan(slots, self.pool.max_slots)
        kc = [torch.zeros(B, cfg.n_kv_heads, max_seq, 128, dtype=torch.float16, device=d)
              for _ in range(cfg.num_layers)]
        vc = [torch.zeros_like(t) for t in kc]
        st = DecodeState(B=B, max_seq=max_seq, tok=torch.zeros(B, dtype=torch.int64, device=d),
                         pos=torch.zeros(1, dtype=torch.int32, device=d),
                         length=torch.ones(1, dtype=torch.int32, device=d), slots=slots, plan=plan,
                         k_cache=kc, v_cache=vc)
        f16 = dict(dtype=torch.float16, device=d)
        st.bufs = dict(
            h=torch.empty(B, cfg.hidden, **f16), xn=torch.empty(B, cfg.hidden, **f16),
            q=torch.empty(B, cfg.q_dim, **f16), k=torch.empty(B, cfg.kv_dim, **f16),
            v=torch.empty(B, cfg.kv_dim, **f16), attn=torch.empty(B, cfg.q_dim, **f16),
            o=torch.empty(B, cfg.hidden, **f16), g=torch.empty(B, cfg.intermediate, **f16),
            u=torch.empty(B, cfg.intermediate, **f16), act=torch.empty(B, cfg.intermediate, **f16),
            d=torch.empty(B, cfg.hidden, **f16), logits=torch.empty(B, cfg.vocab, **f16))
        return st

    # ---- prefill -------------------------------------------------------------
    @torch.inference_mode()
    def prefill(self, st: DecodeState, tokens: torch.Tensor) -> torch.Tensor:
        """Run the prompts ([B, T] token ids, all of length T) through the
        model, fill the caches, and return the last position's logits [B, V]."""
        cfg = self.cfg
        B, T = tokens.shape
        if B != st.B or T > st.max_seq:
            raise ValueError("prompt batch does not fit the decode state")
        R = B * T
        rows = tokens.reshape(-1).to(self.device)
        h = self.embed.index_select(0, rows)
        xn = torch.empty_like(h)
        indptr = torch.arange(0, R + 1, T, dtype=torch.int32, device=self.device)
        start = torch.zeros(1, dtype=torch.int32, device=self.device)
        # LoRA over the request segments (one adapter per prompt): the
        # segmented kernel splits its work evenly over the SMs whatever the
        # number of prompts (the reference's caller expands the same segments
        # into per-token slots, persona/lora_layer.py:21-28).
        def lora_apply(x, lora, names, ys):
            for name, y in zip(names, ys):
                ops.sgmv_fused(x, *lora[name], indptr, st.slots, y)

        delta = None
        for li, lw in enumerate(self.layers):
            lora = self._lora[li]
            ops.add_rmsnorm(h, delta, lw.in_norm, xn, cfg.rms_eps)
            q, k, v = nf4.linear(xn, [lw.q, lw.k, lw.v])
            lora_apply(xn, lora, ("q_proj", "k_proj", "v_proj"), (q, k, v))
            q3, k3, v3 = (t.view(R, -1, 128) for t in (q, k, v))
            ops.rope_cache(q3, k3, v3, st.k_cache[li], st.v_cache[li], start, T, cfg.rope_theta)
            qa = q3.view(B, T, cfg.n_heads, 128).transpose(1, 2)
            ka = k3.view(B, T, cfg.n_kv_heads, 128).transpose(1, 2)
            va = v3.view(B, T, cfg.n_kv_heads, 128).transpose(1, 2)
            attn = F.scaled_dot_product_attention(qa, ka, va, is_causal=True, enable_gqa=True)
            attn = attn.transpose(1, 2).reshape(R, cfg.q_dim).contiguous()
            o = nf4.linear(attn, [lw.o])[0]
            lora_apply(attn, lora, ("o_proj",), (o,))
            ops.add_rmsnorm(h, o, lw.post_norm, xn, cfg.rms_eps)
            g_, u_ = nf4.linear(xn, [lw.gate, lw.up])
            lora_apply(xn, lora, ("gate_proj", "up_proj"), (g_, u_))
            act = torch.empty_like(g_)
            ops.silu_mul(g_, u_, act)
            dn = nf4.linear(act, [lw.down])[0]
            lora_apply(act, lora, ("down_proj",), (dn,))
            delta = dn
        ops.add_rmsnorm(h, delta, self.final_norm, xn, cfg.rms_eps)
        last = xn.view(B, T, cfg.hidden)[:, -1, :]
        logits = torch.matmul(last, self.lm_head.t())
        st.pos.fill_(T)
        st.length.fill_(T + 1)
        return logits

    # ---- ragged chunks over a paged cache --------------------------------------
    def new_paged_state(self, slots: torch.Tensor, num_pages: int, page_size: int = 16, max_seq: int = 4096,
                        kv_dtype: torch.dtype = torch.float16, kv_block: int = 1) -> PagedState:
        """Empty sequences, one per adapter slot of ``slots``, over ``num_pages``
        pages per layer; ``kv_dtype`` fp16, or float8_e4m3fn with one scale per
        ``kv_block`` tokens (1, 2, 4, ... 128, a divisor of the page) and head."""
        cfg, d = self.cfg, self.device
        e4m3 = kv_dtype == torch.float8_e4m3fn
        if not e4m3 and kv_dtype != torch.float16:
            raise ValueError("paged caches are float16 or float8_e4m3fn")
        if kv_block not in (1, 2, 4, 8, 16, 32, 64, 128) or page_size % kv_block or (kv_block > 1 and not e4m3):
            raise ValueError("kv_block is a power of two up to 128 that divides the page, for float8_e4m3fn caches")
        B = int(slots.numel())
        shape = (num_pages, cfg.n_kv_heads, page_size, 128)
        scales = (*shape[:2], page_size // kv_block)

        def per_layer(*size, dtype):
            return [torch.zeros(*size, dtype=dtype, device=d) for _ in range(cfg.num_layers)]

        none = [None] * cfg.num_layers
        return PagedState(slots=slots.to(d, torch.int32).contiguous(), page_size=page_size,
                          page_table=torch.zeros(B, -(-max_seq // page_size), dtype=torch.int32, device=d),
                          k_cache=per_layer(*shape, dtype=kv_dtype), v_cache=per_layer(*shape, dtype=kv_dtype),
                          k_scale=per_layer(*scales, dtype=torch.float32) if e4m3 else none,
                          v_scale=per_layer(*scales, dtype=torch.float32) if e4m3 else none,
                          lengths=[0] * B, pages=[[] for _ in range(B)], free=list(range(num_pages)))

    @torch.inference_mode()
    def extend(self, st: PagedState, chunks: Sequence[Sequence[int]]) -> tuple:
        """Feed every sequence its chunk of token ids (any length, also none).
        Returns the logits behind every fed token, [rows, V], and ``indptr``
        [B + 1] int32: sequence b's rows are indptr[b] .. indptr[b + 1] (what
        ``sampling.verify_drafts`` takes for chunks of a last token and drafts).
        A call that raises leaves the sequences as they were."""
        st._host()
        new = [len(c) for c in chunks]
        if len(new) != len(st.lengths):
            raise ValueError("one chunk per sequence")
        flat_ids = [t for c in chunks for t in c]
        # (the -1 behind a verified sequence's drawn token is not one to feed)
        if flat_ids and not 0 <= min(flat_ids) <= max(flat_ids) < self.cfg.vocab:
            raise ValueError("token id outside the vocabulary")
        lengths, held = list(st.lengths), [len(p) for p in st.pages]
        try:
            st._grow(new)
            return self._extend_rows(st, new, flat_ids)
        except BaseException:
            st._back_to(lengths, held)
            raise

    def _extend_rows(self, st: PagedState, new: List[int], flat_ids: List[int]) -> tuple:
        cfg, d = self.cfg, self.device
        R = sum(new)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        indptr = torch.tensor(starts, dtype=torch.int32, device=d)
        lengths = torch.tensor(st.lengths, dtype=torch.int32, device=d)
        tokens = torch.tensor(flat_ids, dtype=torch.int64, device=d)
        if R == 0:
            return torch.empty(0, cfg.vocab, dtype=torch.float16, device=d), indptr
        h = self.embed.index_select(0, tokens)
        xn = torch.empty_like(h)
        attn = torch.empty(R, cfg.n_heads, 128, dtype=torch.float16, device=d)
        scale, most = 1.0 / math.sqrt(128), max(new)

        def lora_apply(x, lora, names, ys):
            for name, y in zip(names, ys):
                ops.sgmv_fused(x, *lora[name], indptr, st.slots, y)

        delta = None
        for li, lw in enumerate(self.layers):
            lora = self._lora[li]
            kv = (st.k_cache[li], st.v_cache[li], st.page_table, indptr, lengths)
            scales = dict(k_scale=st.k_scale[li], v_scale=st.v_scale[li])
            ops.add_rmsnorm(h, delta, lw.in_norm, xn, cfg.rms_eps)
            q, k, v = nf4.linear(xn, [lw.q, lw.k, lw.v])
            lora_apply(xn, lora, ("q_proj", "k_proj", "v_proj"), (q, k, v))
            q3, k3, v3 = (t.view(R, -1, 128) for t in (q, k, v))
            ops.paged_rope_cache(q3, k3, v3, *kv, cfg.rope_theta, **scales)
            ops.paged_attention(q3, *kv, attn, scale, max_new=most, **scales)
            flat = attn.view(R, cfg.q_dim)
            o = nf4.linear(flat, [lw.o])[0]
            lora_apply(flat, lora, ("o_proj",), (o,))
            ops.add_rmsnorm(h, o, lw.post_norm, xn, cfg.rms_eps)
            g_, u_ = nf4.linear(xn, [lw.gate, lw.up])
            lora_apply(xn, lora, ("gate_proj", "up_proj"), (g_, u_))
            act = torch.empty_like(g_)
            ops.silu_mul(g_, u_, act)
            dn = nf4.linear(act, [lw.down])[0]
            lora_apply(act, lora, ("down_proj",), (dn,))
            delta = dn
        ops.add_rmsnorm(h, delta, self.final_norm, xn, cfg.rms_eps)
        return torch.matmul(xn, self.lm_head.t()), indptr

    # ---- single tokens over a paged cache, without the host ----------------------
    def start_decode(self, st: PagedState, tokens: torch.Tensor, sampling: BatchSampling) -> PagedDecode:
        """Hands the sequences of ``st`` over to the device: ``tokens`` [B] are
        what each feeds first, ``sampling`` how the next ones are drawn.  Until
        ``finish_decode`` only ``paged_step`` moves them.  A sequence whose token
        is -1, what ``sample_batch`` gives for a row without any, ends with the
        first step."""
        st._host()
        cfg, d = self.cfg, self.device
        B, pages = len(st.lengths), st.k_cache[0].shape[0]
        if tokens.shape != (B,) or sampling.temperature.shape != (B,):
            raise ValueError("one token and one set of parameters per sequence")
        if B and not -1 <= int(tokens.min()) <= int(tokens.max()) < cfg.vocab:
            raise ValueError("token id outside the vocabulary")
        i32 = dict(dtype=torch.int32, device=d)
        free = torch.zeros(pages, **i32)
        free[:len(st.free)] = torch.tensor(st.free, **i32)
        dec = PagedDecode(st=st, sampling=sampling, tok=torch.zeros(B + 1, dtype=torch.int64, device=d),
                          alive=torch.ones(B, **i32), u=torch.zeros(B, device=d),
                          lengths=torch.tensor(st.lengths, **i32), keep=torch.zeros(B, **i32), free=free,
                          num_free=torch.tensor([len(st.free)], **i32), indptr=torch.zeros(B + 1, **i32),
                          places=torch.zeros(B, dtype=torch.int64, device=d), seqs=torch.arange(B, **i32),
                          row_seq=torch.zeros(B, **i32), out=torch.zeros(B + 1, dtype=torch.int64, device=d))
        dec.tok[:B].copy_(tokens)
        f16 = dict(dtype=torch.float16, device=d)
        dec.bufs = {n: torch.zeros(B, w, **f16) for n, w in
                    dict(h=cfg.hidden, xn=cfg.hidden, q=cfg.q_dim, k=cfg.kv_dim, v=cfg.kv_dim, attn=cfg.q_dim,
                         o=cfg.hidden, g=cfg.intermediate, u=cfg.intermediate, act=cfg.intermediate, d=cfg.hidden,
                         logits=cfg.vocab).items()}
        st.decode = dec
        return dec

    def finish_decode(self, dec: PagedDecode) -> None:
        """The host has the sequences again (their lengths and pages are read
        back).  A step that found no free page raises here, if no ``paged_step``
        has; it has changed nothing."""
        st = dec.st
        if st.decode is not dec:
            raise ValueError("this decode is not the sequences' own")
        torch.cuda.synchronize(self.device)
        lengths, table, free = dec.lengths.tolist(), st.page_table.tolist(), dec.free[:int(dec.num_free)].tolist()
        st.lengths[:] = lengths
        st.pages[:] = [table[b][:-(-n // st.page_size)] for b, n in enumerate(lengths)]
        st.free[:] = free
        st.decode = None
        ops.check_errors(self.device)

    def _paged_body(self, dec: PagedDecode) -> None:
        cfg, st, b = self.cfg, dec.st, dec.bufs
        B = len(dec.seqs)
        # A token outside of the vocabulary is not one to feed: its sequence has ended.
        dec.alive.mul_((dec.tok[:B] >= 0) & (dec.tok[:B] < cfg.vocab))
        # ended sequences give their pages back, the others get a row and, where they need one, a page
        torch.mul(dec.lengths, dec.alive, out=dec.keep)
        ops.paged_plan(dec.alive, dec.lengths, st.page_table, dec.free, dec.num_free, st.page_size, dec.indptr, dec.places,
                       keep=dec.keep, seq_slots=dec.seqs, row_slots=dec.row_seq)
        seq = dec.row_seq.clamp_min(0)
        slots = torch.where(dec.row_seq < 0, dec.row_seq, st.slots.index_select(0, seq))
        plan = ops.bgmv_plan(slots, self.pool.max_slots)
        # (rows of no sequence look a token up too, be it one that ended its sequence)
        torch.index_select(self.embed, 0, dec.tok.index_select(0, seq).clamp_(0, cfg.vocab - 1), out=b["h"])
        scale = 1.0 / math.sqrt(128)
        delta = None
        for li, lw in enumerate(self.layers):
            lora = self._lora[li]
            kv = (st.k_cache[li], st.v_cache[li], st.page_table, dec.indptr, dec.lengths)
            scales = dict(k_scale=st.k_scale[li], v_scale=st.v_scale[li])
            ops.add_rmsnorm(b["h"], delta, lw.in_norm, b["xn"], cfg.rms_eps)
            nf4.linear(b["xn"], [lw.q, lw.k, lw.v], outs=[b["q"], b["k"], b["v"]])
            ops.bgmv_fused_multi([b["xn"]] * 3, [lora[m][0] for m in ("q_proj", "k_proj", "v_proj")],
                                 [lora[m][1] for m in ("q_proj", "k_proj", "v_proj")], slots,
                                 [b["q"], b["k"], b["v"]], plan=plan)
            q, k, v, attn = (b[n].view(B, -1, 128) for n in ("q", "k", "v", "attn"))
            ops.paged_rope_cache(q, k, v, *kv, cfg.rope_theta, **scales)
            ops.paged_attention(q, *kv, attn, scale, max_new=1, **scales)
            nf4.linear(b["attn"], [lw.o], outs=[b["o"]])
            ops.bgmv_fused(b["attn"], *lora["o_proj"], slots, b["o"], plan=plan)
            ops.add_rmsnorm(b["h"], b["o"], lw.post_norm, b["xn"], cfg.rms_eps)
            nf4.linear(b["xn"], [lw.gate, lw.up], outs=[b["g"], b["u"]])
            ops.bgmv_fused_multi([b["xn"]] * 2, [lora[m][0] for m in ("gate_proj", "up_proj")],
                                 [lora[m][1] for m in ("gate_proj", "up_proj")], slots, [b["g"], b["u"]], plan=plan)
            ops.silu_mul(b["g"], b["u"], b["act"])
            nf4.linear(b["act"], [lw.down], outs=[b["d"]])
            ops.bgmv_fused(b["act"], *lora["down_proj"], slots, b["d"], plan=plan)
            delta = b["d"]
        ops.add_rmsnorm(b["h"], delta, self.final_norm, b["xn"], cfg.rms_eps)
        torch.matmul(b["xn"], self.lm_head.t(), out=b["logits"])
        drawn = torch.empty(B, dtype=torch.int64, device=self.device)
        ops.sample_tokens(b["logits"], dec.u.index_select(0, seq), drawn, **dec.sampling.rows(seq))
        place = torch.where(dec.row_seq < 0, B, dec.row_seq).long()
        dec.tok.index_copy_(0, place, drawn)
        # nothing for those alive whose step could not be made
        dec.out[:B].copy_(torch.where(dec.alive > 0, -1, dec.tok[:B]))
        dec.out.index_copy_(0, place, drawn)

    @on_its_device
    @torch.inference_mode()
    def paged_step(self, dec: PagedDecode, use_graph: bool = True,
                   generator: Optional[torch.Generator] = None) -> torch.Tensor:
        """Every sequence that is alive feeds its token and draws the next one,
        with numbers from ``generator`` (by sequence, whoever else is alive).
        Returns the tokens [B] on the device (``dec.out``; an ended sequence's
        stays what it was).  A row whose logits leave nothing to draw (all NaN or
        -infinity) gives -1, and its sequence ends with the next step.  A step
        that finds no page for some sequence is made for none and gives -1 for
        all that are alive; the next call that sees it raises (an eager step may
        see it itself), and the one behind that tries again (with some sequences
        ended, say).  A call that raises leaves the sequences as they were."""
        if dec.st.decode is not dec:  # its lengths and pages are others' now
            raise ValueError("this decode is not the sequences' own")
        try:
            ops.check_errors(self.device, synchronize=False)
            return self._paged_step(dec, use_graph, generator)
        except RuntimeError as error:
            # Steps that were on their way behind the one at fault have failed like it:
            # nothing of them stays pending for other calls.
            try:
                ops.check_errors(self.device)
            except RuntimeError as more:
                raise error from more
            raise

    def _paged_step(self, dec: PagedDecode, use_graph: bool, generator: Optional[torch.Generator]) -> torch.Tensor:
        dec.u.uniform_(generator=generator)
        B = len(dec.seqs)
        if not use_graph:
            was = [t.clone() for t in dec._moved()]
            try:
                self._paged_body(dec)
            except BaseException:
                for to, t in zip(dec._moved(), was):
                    to.copy_(t)
                raise
            return dec.out[:B]
        if dec.graph is None:
            # Warmed up on a side stream by a step in which nobody is alive; what it
            # moves is put back (nothing else is written but the padded rows' own buffers).
            was = [t.clone() for t in dec._moved()]
            s = torch.cuda.Stream(self.device)
            try:
                dec.alive.zero_()
                s.wait_stream(torch.cuda.current_stream(self.device))
                with torch.cuda.stream(s):
                    self._paged_body(dec)
            finally:
                torch.cuda.current_stream(self.device).wait_stream(s)
                for to, t in zip(dec._moved(), was):
                    to.copy_(t)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):  # (the default one is of the device that captured first)
                self._paged_body(dec)
            dec.graph = g
        dec.graph.replay()
        return dec.out[:B]

    # ---- decode --------------------------------------------------------------
    def _decode_body(self, st: DecodeState) -> None:
        cfg, b = self.cfg, st.bufs
        B = st.B
        torch.index_select(self.embed, 0, st.tok, out=b["h"])
        scale = 1.0 / math.sqrt(128)
        delta = None
        for li, lw in enumerate(self.layers):
            lora = self._lora[li]
            ops.add_rmsnorm(b["h"], delta, lw.in_norm, b["xn"], cfg.rms_eps)
            nf4.linear(b["xn"], [lw.q, lw.k, lw.v], outs=[b["q"], b["k"], b["v"]])
            ops.bgmv_fused_multi([b["xn"]] * 3, [lora[m][0] for m in ("q_proj", "k_proj", "v_proj")],
                                 [lora[m][1] for m in ("q_proj", "k_proj", "v_proj")], st.slots,
                                 [b["q"], b["k"], b["v"]], plan=st.plan)
            # rotary embedding, cache write and attention in one launch
            ops.rope_decode_attention(b["q"].view(B, cfg.n_heads, 128), b["k"].view(B, cfg.n_kv_heads, 128),
                                      b["v"].view(B, cfg.n_kv_heads, 128), st.k_cache[li], st.v_cache[li], st.pos,
                                      st.length, b["attn"].view(B, cfg.n_heads, 128), cfg.rope_theta, scale)
            nf4.linear(b["attn"], [lw.o], outs=[b["o"]])
            ops.bgmv_fused(b["attn"], *lora["o_proj"], st.slots, b["o"], plan=st.plan)
            ops.add_rmsnorm(b["h"], b["o"], lw.post_norm, b["xn"], cfg.rms_eps)
            nf4.linear(b["xn"], [lw.gate, lw.up], outs=[b["g"], b["u"]])
            ops.bgmv_fused_multi([b["xn"]] * 2, [lora[m][0] for m in ("gate_proj", "up_proj")],
                                 [lora[m][1] for m in ("gate_proj", "up_proj")], st.slots, [b["g"], b["u"]],
                                 plan=st.plan)
            ops.silu_mul(b["g"], b["u"], b["act"])
            nf4.linear(b["act"], [lw.down], outs=[b["d"]])
            ops.bgmv_fused(b["act"], *lora["down_proj"], st.slots, b["d"], plan=st.plan)
            delta = b["d"]
        ops.add_rmsnorm(b["h"], delta, self.final_norm, b["xn"], cfg.rms_eps)
        torch.matmul(b["xn"], self.lm_head.t(), out=b["logits"])
        st.tok.copy_(torch.argmax(b["logits"], dim=-1))
        st.pos.add_(1)
        st.length.add_(1)

    @on_its_device
    @torch.inference_mode()
    def decode_step(self, st: DecodeState, use_graph: bool = True) -> torch.Tensor:
        """Feed ``st.tok`` at ``st.pos``; greedy next tokens land in
        ``st.tok`` (returned) and the position advances."""
        if not use_graph:
            self._decode_body(st)
            return st.tok
        if st.graph is None:
            # warm up on a side stream (the first calls make the workspaces),
            # then capture; the warm-up step is undone by rewinding pos.
            pos0, tok0 = st.pos.clone(), st.tok.clone()
            s = torch.cuda.Stream(self.device)
            s.wait_stream(torch.cuda.current_stream(self.device))
            with torch.cuda.stream(s):
                self._decode_body(st)
            torch.cuda.current_stream(self.device).wait_stream(s)
            st.pos.copy_(pos0)
            st.length.copy_(pos0 + 1)
            st.tok.copy_(tok0)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):  # (the default one is of the device that captured first)
                self._decode_body(st)
            st.graph = g
            # capture does not run the body: run it now
        st.graph.replay()
        return st.tok
