"""Per-request sampling parameters and next-token choice.

The parameter set is the reference's (``persona/sampling.py:8-13``:
temperature, top-p, a token budget) with top-k and min-p beside it.  The choice
of ``sample_next_token`` is written around
the Gumbel-max identity instead of an explicit draw from a renormalised
distribution: ``argmax(z + G)`` with ``G`` i.i.d. standard Gumbel noise picks
index ``i`` with probability ``softmax(z)_i``.  That needs no renormalisation,
no ``multinomial`` and no host round trip, and a top-p cut becomes a mask on
``z`` (a per-row log-probability threshold), so every row of a batch is
handled in one set of tensor ops on the device.  Rows with parameters of their
own, top-k or min-p go to ``ops.sample_tokens``, which draws from given uniform
numbers (``sample_batch``).
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch


@dataclass
class SamplingParams:
    temperature: float = 0.0
    top_p: float = 1.0
    max_tokens: int = 128
    top_k: int = 0      # 0: all
    min_p: float = 0.0  # 0: off


class BatchSampling:
    """The parameters of a batch's rows as tensors on ``device``, what
    ``ops.sample_tokens`` takes (None where no row uses one)."""

    def __init__(self, params: Sequence[SamplingParams], device):
        def column(name, dtype, used):
            values = [getattr(p, name) for p in params]
            return torch.tensor(values, dtype=dtype, device=device) if any(used(v) for v in values) else None

        self.temperature = torch.tensor([p.temperature for p in params], dtype=torch.float32, device=device)
        self.top_k = column("top_k", torch.int32, lambda k: k > 0)
        self.top_p = column("top_p", torch.float32, lambda p: p < 1.0)
        self.min_p = column("min_p", torch.float32, lambda m: m > 0)

    def rows(self, index: Optional[torch.Tensor] = None) -> dict:
        """Keyword arguments of ``ops.sample_tokens``, for the rows ``index`` of the batch."""
        columns = dict(temperature=self.temperature, top_k=self.top_k, top_p=self.top_p, min_p=self.min_p)
        return {n: c if c is None or index is None else c.index_select(0, index) for n, c in columns.items()}


def sample_batch(logits: torch.Tensor, params, generator: Optional[torch.Generator] = None,
                 u: Optional[torch.Tensor] = None) -> torch.Tensor:
    """logits [batch, vocab] on the GPU -> next token ids [batch] (int64), each
    row by its own parameters (a ``BatchSampling`` or one ``SamplingParams`` per
    row); -1 for a row of NaN or -infinity alone.  ``u`` [batch] fp32 are the uniform numbers the tokens are drawn with;
    drawn from ``generator`` if not given."""
    from persona import ops

    if not isinstance(params, BatchSampling):
        params = BatchSampling(params, logits.device)
    B = logits.shape[0]
    if u is None:
        u = torch.rand(B, device=logits.device, generator=generator)
    tokens = torch.empty(B, dtype=torch.int64, device=logits.device)
    return ops.sample_tokens(logits, u, tokens, **params.rows())


def _nucleus_mask(z: torch.Tensor, top_p: float) -> torch.Tensor:
    """``z`` with every token outside the top-p nucleus set to -inf.

    The nucleus of a row is the most probable tokens, taken in order of
    probability while the mass of the tokens before them is at most
    ``top_p`` (so the most probable token always stays).  It is applied as a
    threshold on the log-probability of the last token kept; tokens tied
    with that one stay as well.
    """
    lp = torch.log_softmax(z, dim=-1)
    lp_sorted = torch.sort(lp, dim=-1, descending=True).values
    p_sorted = lp_sorted.exp()
    mass_before = torch.cumsum(p_sorted, dim=-1) - p_sorted
    keep = (mass_before <= top_p).sum(dim=-1, keepdim=True).clamp_(min=1)
    threshold = lp_sorted.gather(-1, keep - 1)
    return z.masked_fill(lp < threshold, float("-inf"))


def sample_next_token(logits: torch.Tensor, params: SamplingParams,
                      generator: Optional[torch.Generator] = None) -> torch.Tensor:
    """logits [batch, vocab] -> next token ids [batch] (int64).

    Temperature 0 (or below) is greedy.  Otherwise the logits are divided by
    the temperature, cut to the top-p nucleus when ``top_p < 1``, and one
    token per row is drawn by Gumbel-max.  With top-k or min-p: ``sample_batch``,
    but a row of NaN or -infinity alone gives its ``argmax``, as without them.
    """
    if params.temperature <= 0:
        return logits.argmax(dim=-1)
    if params.top_k > 0 or params.min_p > 0:
        token = sample_batch(logits, [params] * logits.shape[0], generator=generator)
        return torch.where(token < 0, logits.argmax(dim=-1), token)  # (callers feed it: always a token of the vocabulary)
    z = logits.float() / params.temperature
    if params.top_p < 1.0:
        z = _nucleus_mask(z, params.top_p)
    u = torch.rand(z.shape, device=z.device, generator=generator)
    gumbel = -torch.log(-torch.log(u.clamp_(min=torch.finfo(torch.float32).tiny)))
    return (z + gumbel).argmax(dim=-1)


def verify_drafts(target_logits: torch.Tensor, draft_tokens: torch.Tensor, draft_probs: Optional[torch.Tensor],
                  indptr: torch.Tensor, params: SamplingParams, generator: Optional[torch.Generator] = None):
    """Which drafted tokens of each sequence to keep, and the token behind them.

    ``target_logits`` [rows, V] are the model's behind every token of the fed
    chunks (a sequence's last token, then its drafts; rows ``indptr[b]`` to
    ``indptr[b+1]``), ``draft_tokens`` [rows] the token that the draft put
    behind each row's (ignored at a sequence's last row), ``draft_probs``
    [rows, V] fp32 its distributions under the same ``params``, or None for
    drafts without probabilities.  Returns ``(tokens [rows], accepted [B])``
    as ``ops.verify_draft``.  Temperature 0 keeps a draft while it is the
    most probable token."""
    from persona import ops

    if params.temperature > 0 and (params.top_k > 0 or params.min_p > 0):
        raise ValueError("drafts are verified by temperature and top_p")
    rows, dev = target_logits.shape[0], target_logits.device
    B = indptr.numel() - 1
    if params.temperature <= 0:
        best = target_logits.argmax(dim=-1, keepdim=True)
        p = torch.zeros(target_logits.shape, dtype=torch.float32, device=dev).scatter_(1, best, 1.0)
        draft_probs = None
    else:
        z = target_logits.float() / params.temperature
        if params.top_p < 1.0:
            z = _nucleus_mask(z, params.top_p)
        p = torch.softmax(z, dim=-1)
    u_accept = torch.rand(rows, device=dev, generator=generator)
    u_sample = torch.rand(B, device=dev, generator=generator)
    tokens = torch.empty(rows, dtype=torch.int64, device=dev)
    accepted = torch.empty(B, dtype=torch.int32, device=dev)
    return ops.verify_draft(p, draft_tokens, draft_probs, indptr, u_accept, u_sample, tokens, accepted)
