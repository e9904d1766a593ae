"""BGMV op entry points on B200 (drop-in for the reference's ``persona/ops.py``).

``bgmv_shrink`` / ``bgmv_expand`` keep the reference's signatures and return
conventions (``persona/ops.py:71-90``): shrink allocates and returns the fp32
``v``; expand updates ``y`` in place and returns it.  Both dispatch to the
``torch.ops.persona`` ops registered by the in-tree extension, which this
module loads itself (the reference left that import to the caller, so its
"CUDA" path silently ran the fp32 fallback when nobody imported
``persona._C``).

There is no CPU fallback: CPU tensors, or a missing extension, raise.  The
reference's fp32 functions ``bgmv_*_ref`` are test infrastructure here and
live in the repository's ``oracle`` package.

New in this build:

* ``bgmv_fused`` -- shrink->expand in one launch, rank-R intermediate kept on
  chip (the reference's fused kernel is a stub, ``docs/BENCHMARKS.md:238``).
* ``bgmv_fused_multi`` -- the fused op for up to 8 projections of a layer
  that share the slots, in one launch.
* ``bgmv_plan`` -- groups a batch's rows by adapter slot once on the device;
  pass the result as ``plan=`` to every shrink/expand/fused call that uses
  the same slots (a decode step's 7 projections x 32 layers share one).
* ``paged_rope_cache`` / ``paged_cache_read`` / ``paged_attention`` -- a
  ragged batch of new tokens (single ones, drafted ones, prompt chunks) over a
  paged KV cache with 16-bit or e4m3 pages; ``verify_draft`` -- acceptance of
  drafted tokens.
* ``check_errors`` -- out-of-range slots are detected on the device (no
  per-row host sync); the next op on that device, or this function, raises.
"""

from __future__ import annotations

from typing import Optional

import torch

_EXT = None
_MODULE = type(torch)
_compiling = torch.compiler.is_dynamo_compiling


def _load():
    """Import the native extension once; raise loudly if it is unavailable."""
    global _EXT
    if _EXT is None:
        try:
            from persona import _C  # registers torch.ops.persona.*
        except ImportError as e:  # pragma: no cover - depends on the build
            _EXT = e
        else:
            _EXT = _C
    if isinstance(_EXT, Exception):
        raise RuntimeError(
            "persona: the native BGMV extension is not built or cannot be loaded "
            "(run multi-lora-llm-kernel_b200/build.py)") from _EXT
    return _EXT


def has_cuda_ops() -> bool:
    """True when the B200 BGMV ops are registered (reference ``ops.py:8-9``)."""
    try:
        _load()
    except RuntimeError:
        return False
    return hasattr(torch.ops, "persona") and hasattr(torch.ops.persona, "bgmv_shrink")


def _require_cuda(op: str, *tensors: torch.Tensor) -> None:
    _load()
    if not all(t.is_cuda for t in tensors):
        raise RuntimeError(f"{op}: all tensors must be CUDA (this build has no CPU fallback)")


def bgmv_plan(slots: torch.Tensor, num_slots: int) -> torch.Tensor:
    """Device-side row grouping of ``slots`` for a pool of ``num_slots`` slots."""
    _require_cuda("bgmv_plan", slots)
    return torch.ops.persona.bgmv_plan(slots, int(num_slots))


def bgmv_shrink(x: torch.Tensor, a_pool: torch.Tensor, slots: torch.Tensor,
                plan: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``v[t] = A[slots[t]] @ x[t]`` in fp32; rows with slot -1 give zeros."""
    _require_cuda("bgmv_shrink", x, a_pool, slots)
    v = torch.empty((x.shape[0], a_pool.shape[1]), dtype=torch.float32, device=x.device)
    if plan is None:
        torch.ops.persona.bgmv_shrink(x.contiguous(), a_pool, slots, v)
    else:
        torch.ops.persona.bgmv_shrink_with_plan(x.contiguous(), a_pool, slots, plan, v)
    return v


def bgmv_expand(v: torch.Tensor, b_pool: torch.Tensor, slots: torch.Tensor, y: torch.Tensor,
                plan: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[t] += B[slots[t]] @ v[t]`` in place (fp32 sum, one rounding)."""
    _require_cuda("bgmv_expand", v, b_pool, slots, y)
    if plan is None:
        torch.ops.persona.bgmv_expand(v, b_pool, slots, y)
    else:
        torch.ops.persona.bgmv_expand_with_plan(v, b_pool, slots, plan, y)
    return y


def bgmv_fused(x: torch.Tensor, a_pool: torch.Tensor, b_pool: torch.Tensor, slots: torch.Tensor,
               y: torch.Tensor, plan: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[t] += B[s] @ (A[s] @ x[t])`` in one launch; returns ``y``.

    Equal, within fp32 summation order, to ``bgmv_expand(bgmv_shrink(x))``.
    """
    _require_cuda("bgmv_fused", x, a_pool, b_pool, slots, y)
    if plan is None:
        torch.ops.persona.bgmv_fused(x, a_pool, b_pool, slots, y)
    else:
        torch.ops.persona.bgmv_fused_with_plan(x, a_pool, b_pool, slots, plan, y)
    return y


def bgmv_fused_multi(xs, a_pools, b_pools, slots: torch.Tensor, ys,
                     plan: Optional[torch.Tensor] = None):
    """``ys[i] += B_i[s] @ (A_i[s] @ xs[i])`` for up to 8 projections that
    share ``slots`` (one decoder layer), in one launch; returns ``ys``.

    Each result equals ``bgmv_fused`` on that projection.  All pools share
    the rank and the slot count.
    """
    xs, a_pools, b_pools, ys = list(xs), list(a_pools), list(b_pools), list(ys)
    _require_cuda("bgmv_fused_multi", *xs, *a_pools, *b_pools, slots, *ys)
    torch.ops.persona.bgmv_fused_multi(xs, a_pools, b_pools, slots, ys, plan)
    return ys


def sgmv_shrink(x: torch.Tensor, a_pool: torch.Tensor, seg_indptr: torch.Tensor,
                seg_slots: torch.Tensor) -> torch.Tensor:
    """Segmented shrink: rows ``[seg_indptr[i], seg_indptr[i+1])`` use slot
    ``seg_slots[i]``; rows outside every segment get zeros.  Equals
    ``bgmv_shrink`` on the per-row slots the segments imply."""
    _require_cuda("sgmv_shrink", x, a_pool, seg_indptr, seg_slots)
    v = torch.empty((x.shape[0], a_pool.shape[1]), dtype=torch.float32, device=x.device)
    torch.ops.persona.sgmv_shrink(x.contiguous(), a_pool, seg_indptr, seg_slots, v)
    return v


def sgmv_expand(v: torch.Tensor, b_pool: torch.Tensor, seg_indptr: torch.Tensor,
                seg_slots: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """Segmented expand, in place on ``y``; rows outside the segments untouched."""
    _require_cuda("sgmv_expand", v, b_pool, seg_indptr, seg_slots, y)
    torch.ops.persona.sgmv_expand(v, b_pool, seg_indptr, seg_slots, y)
    return y


def sgmv_fused(x: torch.Tensor, a_pool: torch.Tensor, b_pool: torch.Tensor, seg_indptr: torch.Tensor,
               seg_slots: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """Segmented shrink->expand in place on ``y``."""
    _require_cuda("sgmv_fused", x, a_pool, b_pool, seg_indptr, seg_slots, y)
    torch.ops.persona.sgmv_fused(x, a_pool, b_pool, seg_indptr, seg_slots, y)
    return y


def gemv_fp16(x: torch.Tensor, W: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """Warm-up GEMV kept from the reference (``csrc/gemv_fp16.cu``)."""
    _require_cuda("gemv_fp16", x, W, y)
    torch.ops.persona.gemv_fp16(x, W, y)
    return y


def check_errors(device: Optional[torch.device] = None, synchronize: bool = True) -> None:
    """Raise RuntimeError if a kernel on ``device`` flagged an error.

    With ``synchronize`` the device is synchronised first, so every op
    enqueued before this call has been checked.
    """
    ext = _load()
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    device = torch.device(device)
    if synchronize:
        torch.cuda.synchronize(device)
    bits = ext.take_device_error(device.index or 0)
    if bits:
        what = []
        if bits & 1:
            what.append("slot out of range")
        if bits & 2:
            what.append("device wait timed out")
        if bits & 4:
            what.append("invalid segment table")
        if bits & 8:
            what.append("reused plan does not match the call")
        if bits & 16:
            what.append("page or position outside the paged cache")
        if bits & 32:
            what.append("drafted token outside the vocabulary")
        raise RuntimeError(f"persona: device error 0x{bits:x}: {', '.join(what)}")


# ---- fused steps of the end-to-end decode (persona_add_rmsnorm & co.) ------
def add_rmsnorm(h: torch.Tensor, delta: Optional[torch.Tensor], w: torch.Tensor, out: torch.Tensor,
                eps: float) -> torch.Tensor:
    """``h += delta`` (if given) and ``out = w * fp16(h / rms(h))`` per row."""
    _require_cuda("add_rmsnorm", h, w, out)
    torch.ops.persona.add_rmsnorm(h, delta, w, out, float(eps))
    return out


def rope_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
               start: torch.Tensor, per_seq: int, theta: float) -> None:
    """Rotary embedding of q and k in place and the k / v cache write."""
    _require_cuda("rope_cache", q, k, v, k_cache, v_cache, start)
    torch.ops.persona.rope_cache(q, k, v, k_cache, v_cache, start, int(per_seq), float(theta))


def silu_mul(g: torch.Tensor, u: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    _require_cuda("silu_mul", g, u, out)
    torch.ops.persona.silu_mul(g, u, out)
    return out


def decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, length: torch.Tensor,
                     out: torch.Tensor, scale: float) -> torch.Tensor:
    """One new token per sequence over the first ``length`` cache positions."""
    _require_cuda("decode_attention", q, k_cache, v_cache, length, out)
    torch.ops.persona.decode_attention(q, k_cache, v_cache, length, out, float(scale))
    return out


def rope_decode_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                          v_cache: torch.Tensor, pos: torch.Tensor, length: torch.Tensor, out: torch.Tensor,
                          theta: float, scale: float) -> torch.Tensor:
    """``rope_cache`` (one token per sequence at ``pos``) and
    ``decode_attention`` in one launch, with the same results."""
    _require_cuda("rope_decode_attention", q, k, v, k_cache, v_cache, pos, length, out)
    torch.ops.persona.rope_decode_attention(q, k, v, k_cache, v_cache, pos, length, out, float(theta), float(scale))
    return out


def bgmv_lora_delta_multi(xs, a_pools, b_pools, slots: torch.Tensor, deltas):
    """``deltas[i][t] = B_i[s] @ (A_i[s] @ xs[i][t])`` in fp32 (0 for rows
    without adapter), at most 64 rows: the LoRA term alone, for a base
    projection that adds it (``nf4.linear(..., addends=...)``)."""
    _require_cuda("bgmv_lora_delta_multi", slots, *xs, *a_pools, *b_pools, *deltas)
    torch.ops.persona.bgmv_lora_delta_multi(list(xs), list(a_pools), list(b_pools), slots, list(deltas))
    return deltas


# ---- paged KV cache and drafted tokens ---------------------------------------
# These calls are short enough for the host's time to count: they go straight
# to the extension's functions, which check every tensor themselves (and pass
# the call on to torch.ops.persona.* where a mode or a tensor subclass has to
# see it).  A compiler traces the operators.
def _paged(op: str, first: torch.Tensor):
    if not first.is_cuda:
        _require_cuda(op, first)
    ext = _load() if type(_EXT) is not _MODULE else _EXT
    return torch.ops.persona if _compiling() else ext


def paged_rope_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     page_table: torch.Tensor, indptr: torch.Tensor, lengths: torch.Tensor, theta: float,
                     q_out: Optional[torch.Tensor] = None, k_scale: Optional[torch.Tensor] = None,
                     v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary embedding of a ragged batch of new tokens and the write of their
    k and v to a paged cache; returns the rotated q (``q_out``, by default
    ``q`` itself; k and v are left as they are).

    ``q`` [rows, Hq, D], ``k`` / ``v`` [rows, Hkv, D] (fp16 or bf16, D 64 or
    128, views with unit inner stride).  Rows ``indptr[b]`` to ``indptr[b+1]``
    are sequence b's new tokens, at its last positions: the last one is at
    ``lengths[b] - 1``.  Caches [pages, Hkv, page size, D]; position p of
    sequence b is in page ``page_table[b, p // page_size]``.  Caches of
    ``float8_e4m3fn`` take fp32 scales [pages, Hkv, page size]: one per token
    and head, ``max|x| / 448``.  Rows of no sequence are left alone.  ``theta``
    is taken as an fp32 number.  What is written must not overlap itself or
    another argument, but for ``q_out``, which may be ``q``."""
    q_out = q if q_out is None else q_out
    _paged("paged_rope_cache", q).paged_rope_cache(q, k, v, q_out, k_cache, v_cache, page_table, indptr, lengths, theta,
                                                   k_scale, v_scale)
    return q_out


def paged_cache_read(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, indptr: torch.Tensor,
                     lengths: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor,
                     k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None) -> None:
    """k and v of the last ``indptr[b+1] - indptr[b]`` positions of each
    sequence, out of the pages into ``k_out`` / ``v_out`` [rows, Hkv, D]
    (e4m3 pages: code times scale)."""
    _paged("paged_cache_read", k_cache).paged_cache_read(k_cache, v_cache, page_table, indptr, lengths, k_out, v_out,
                                                         k_scale, v_scale)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    indptr: torch.Tensor, lengths: torch.Tensor, out: torch.Tensor, scale: float, window: int = 0,
                    max_new: Optional[int] = None, k_scale: Optional[torch.Tensor] = None,
                    v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of each sequence's new tokens over its pages, theirs
    included (write them first; ``out`` must not overlap ``q``); with ``window`` over the last ``window``
    positions only (pages that no new token's window reaches may be given
    back: their table entries and contents are not used).  Layouts as in ``paged_rope_cache``; ``out`` like ``q``.
    A row that sees no position gives zeros; ``scale`` is positive.

    ``max_new``: an upper bound of the new tokens of one sequence, which
    chooses the kernel (default: what ``rows`` allows if every sequence has
    a token); it never changes what is computed."""
    ext = _paged("paged_attention", q)
    if max_new is None:
        max_new = max(1, q.shape[0] - lengths.shape[0] + 1)
    ext.paged_attention(q, k_cache, v_cache, page_table, indptr, lengths, out, scale, window, max_new, k_scale, v_scale)
    return out


def verify_draft(target_probs: torch.Tensor, draft_tokens: torch.Tensor, draft_probs: Optional[torch.Tensor],
                 indptr: torch.Tensor, u_accept: torch.Tensor, u_sample: torch.Tensor, tokens: torch.Tensor,
                 accepted: torch.Tensor):
    """Speculative sampling from given uniform numbers; returns ``tokens`` and
    ``accepted``.

    Row ``indptr[b] + i`` of ``target_probs`` [rows, V] is the target's
    distribution behind the i-th token fed for sequence b; all rows but the
    sequence's last judge the drafted token ``draft_tokens[row]``, drawn from
    ``draft_probs[row]`` (None: a draft without probabilities, certain of its
    token).  Drafts are kept while ``u_accept[row] * q < p``.  Then one token
    is drawn with ``u_sample[b]``: from ``max(p - q, 0)`` where a draft was
    rejected, else from the last row.  ``tokens`` [rows] int64: the kept
    drafts, the drawn token, then -1; ``accepted`` [B] int32: how many (buffers
    apart from each other and from the inputs).  ``u_sample`` lies in [0, 1): a
    smaller number or NaN counts as 0, a larger one draws the last token with
    weight."""
    _paged("verify_draft", target_probs).verify_draft(target_probs, draft_tokens, draft_probs, indptr, u_accept,
                                                      u_sample, tokens, accepted)
    return tokens, accepted
