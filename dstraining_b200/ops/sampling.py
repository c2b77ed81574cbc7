"""The next token from logits, on the device, from given random numbers.

:func:`sample_tokens` scales by the temperature, keeps the tokens that top-k,
top-p and min-p leave and takes the maximum of ``t + gumbel`` over them, which
draws from their renormalised softmax if ``gumbel`` are independent standard
Gumbel numbers (:func:`gumbel_noise`). Nothing is copied to the host, and the
same numbers give the same tokens.

With ``t = logits / temperature`` and the tokens ordered by ``t`` descending,
equal values by index:

* top-k keeps the first ``top_k`` (0: all);
* top-p keeps of those the shortest prefix whose share of their mass reaches
  ``top_p`` (1: all);
* min-p keeps of those the ones at least ``min_p`` times as probable as the first;
* the first token always stays and a logit of -inf never does; ``temperature`` 0
  takes the first (logprob at temperature 1).

A temperature below the smallest normal fp32 number counts as 0, one above the
largest as the largest; a ``t`` below the smallest normal number is 0.

NaN logits count as -inf. A row with no token above -inf gives token -1 and
logprob -inf. CUDA logits in bf16 or fp32 run the kernel of ``csrc/sampling.cu``
(one CTA per row; a row of up to 52224 entries is read once, a longer one in each
of the kernel's passes); anything else PyTorch.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import native

Setting = Union[float, int, torch.Tensor]


def gumbel_noise(batch: int, vocab: int, device=None, generator: Optional[torch.Generator] = None) -> torch.Tensor:
    """Standard Gumbel numbers, fp32 [batch, vocab]."""
    u = torch.empty(batch, vocab, dtype=torch.float32, device=device).exponential_(generator=generator)
    return u.log_().neg_()


def _row_values(x: Setting, batch: int, dtype: torch.dtype, name: str):
    """(number, None) or (0, tensor [batch])."""
    if not isinstance(x, torch.Tensor):
        return x, None
    if x.shape != (batch,):
        raise ValueError(f"{name} must be a number or a tensor [{batch}], got {list(x.shape)}")
    return 0, x.to(dtype).contiguous()


def sample_tokens(logits: torch.Tensor, gumbel: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0,
                  top_p: Setting = 1.0, min_p: Setting = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """logits [B, V], gumbel fp32 [B, V]; each setting a number or a tensor [B]
    -> tokens int64 [B] and their log-probabilities fp32 [B] (under the softmax
    of ``t`` over the whole row)."""
    if logits.dim() != 2 or gumbel.shape != logits.shape or gumbel.dtype != torch.float32:
        raise ValueError(f"logits [B, V] and fp32 gumbel of the same shape required, got {list(logits.shape)} and "
                         f"{gumbel.dtype} {list(gumbel.shape)}")
    if gumbel.device != logits.device:
        raise ValueError(f"logits on {logits.device}, gumbel on {gumbel.device}")
    if logits.shape[1] == 0:
        raise ValueError("no vocabulary to sample from")
    for name, x in (("temperature", temperature), ("min_p", min_p)):
        if not isinstance(x, torch.Tensor) and not x >= 0:
            raise ValueError(f"{name} must not be negative, got {x}")
    b = logits.shape[0]
    if b == 0:
        return (torch.empty(0, dtype=torch.int64, device=logits.device),
                torch.empty(0, dtype=torch.float32, device=logits.device))
    settings = [_row_values(x, b, dtype, name) for name, x, dtype in (
        ("temperature", temperature, torch.float32), ("top_k", top_k, torch.int64),
        ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32))]
    if logits.is_cuda and logits.dtype in (torch.bfloat16, torch.float32) and native.enabled():
        logits, gumbel = (x if x.stride(1) == 1 else x.contiguous() for x in (logits, gumbel))
        return tuple(native.lib().sample_tokens(logits, gumbel, *(n for n, _ in settings), *(t for _, t in settings)))
    return _plain(logits, gumbel, *(torch.full((b, 1), n, dtype=d, device=logits.device) if t is None else t[:, None]
                                    for (n, t), d in zip(settings, (torch.float32, torch.int64, torch.float32, torch.float32))))


def _plain(logits, gumbel, temperature, top_k, top_p, min_p):
    fp32 = torch.finfo(torch.float32)
    greedy = ~(temperature >= fp32.tiny)
    t = logits.float() / torch.where(greedy, torch.ones_like(temperature), temperature.clamp(max=fp32.max))
    t = torch.where(t.isnan(), torch.full_like(t, float("-inf")), t)
    t = torch.where(t.abs() < fp32.tiny, torch.zeros_like(t), t)
    ranked, order = torch.sort(t, dim=-1, descending=True, stable=True)
    top = ranked[:, :1]
    gap = torch.where(ranked == top, torch.zeros_like(ranked), ranked - top)
    mass = torch.exp(gap)
    rank = torch.arange(t.shape[1], device=t.device)[None, :]
    keep = (top_k <= 0) | (rank < top_k)
    among = torch.where(keep, mass, torch.zeros_like(mass)).double()
    keep = keep & ((top_p >= 1) | (among.cumsum(dim=-1) - among < top_p * among.sum(dim=-1, keepdim=True)))
    keep = keep & (mass >= min_p) & (ranked > float("-inf")) & ~greedy | (rank == 0)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    score = t + gumbel
    score = torch.where(score.isnan(), torch.full_like(score, float("-inf")), score)
    # a kept token wins over every other one, also with a score of -inf
    score = torch.where(kept, score.clamp(min=fp32.min), torch.full_like(score, float("-inf")))
    token = score.argmax(dim=-1, keepdim=True)
    t_token = t.gather(1, token)
    logprob = torch.where(t_token == top, torch.zeros_like(top), t_token - top) - torch.log(mass.sum(dim=-1, keepdim=True))
    empty = top == float("-inf")
    return (torch.where(empty, torch.full_like(token, -1), token)[:, 0],
            torch.where(empty, torch.full_like(logprob, float("-inf")), logprob)[:, 0])
