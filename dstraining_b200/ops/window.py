"""Sliding-window attention with sinks.

Key ``j`` is visible to query ``i`` iff ``j <= i`` and (``i - j < window`` or
``j < sinks``): each query sees its last ``window`` tokens and the first
``sinks`` tokens of the sequence, so time and traffic grow with
``T * (window + sinks)`` instead of ``T^2``, and decoding needs a cache of only
``sinks + window`` slots (:mod:`dstraining_b200.ops.kv_cache`).

* CUDA bf16: the tcgen05 kernels of ``csrc/attn_window_*.cu``. Head sizes are
  multiples of 8 up to 128; any sequence length runs as it is (no padding);
  query heads may share key heads; operands are read where they lie if their
  strides are multiples of 16 bytes (copied otherwise). Backward recomputes the
  probabilities from the saved log-sum-exp and uses no atomics, so repeated
  runs give the same bits. The gradients have no derivative of their own:
  differentiating them (``create_graph``) raises.
* otherwise: :func:`core_window_attention`, the materialised algorithm.

A token's own key is always visible, so no row is empty. As in any tiled
attention, a masked key contributes its value times an exact zero: infinities
or NaN in the values of masked tokens reach the rows of the same key block.
"""

from __future__ import annotations

import math

import torch

from . import native


def window_mask(t: int, window: int, sinks: int, device=None) -> torch.Tensor:
    """[t, t] bool, True where key j (columns) is visible to query i (rows)."""
    i = torch.arange(t, device=device)[:, None]
    j = torch.arange(t, device=device)[None, :]
    return (j <= i) & ((i - j < window) | (j < sinks))


def core_window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int) -> torch.Tensor:
    """The scores materialised. q [B, T, H, D], k and v [B, T, Hk, D] -> [B, T, H, D]."""
    q, k, v = (x.transpose(1, 2) for x in (q, k, v))
    if k.shape[1] != q.shape[1]:
        k, v = (x.repeat_interleave(q.shape[1] // x.shape[1], dim=1) for x in (k, v))
    scores = (q @ k.transpose(-2, -1)) / math.sqrt(q.shape[-1])
    scores = scores.masked_fill(~window_mask(q.shape[2], window, sinks, q.device), float("-inf"))
    return (torch.softmax(scores, dim=-1) @ v).transpose(1, 2)


def _check(window: int, sinks: int) -> None:
    if window < 1:
        raise ValueError(f"window must be at least 1, got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")


def _split(qkv: torch.Tensor, n_head: int, head_dim: int):
    b, t, _ = qkv.shape
    return qkv.view(b, t, n_head, 3, head_dim).unbind(dim=3)


def window_attention(qkv: torch.Tensor, n_head: int, head_dim: int, window: int, sinks: int = 0) -> torch.Tensor:
    """qkv [B, T, n_head * 3 * head_dim] (head-major q|k|v, as the fused
    projection writes it) -> [B, T, n_head * head_dim]."""
    _check(window, sinks)
    if qkv.dim() != 3 or qkv.shape[2] != 3 * n_head * head_dim:
        raise ValueError(f"qkv must be [B, T, {3 * n_head * head_dim}], got {tuple(qkv.shape)}")
    b, t, _ = qkv.shape
    if native.active(qkv) and b and t:
        return native.lib().window_attention(qkv, n_head, head_dim, window, sinks)
    return core_window_attention(*_split(qkv.contiguous(), n_head, head_dim), window, sinks).reshape(b, t, n_head * head_dim)


def window_attention_qkv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0) -> torch.Tensor:
    """q [B, T, H, D], k and v [B, T, Hk, D] with Hk dividing H (query head h
    reads key head ``h // (H / Hk)``), any strides -> [B, T, H, D]."""
    _check(window, sinks)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
        raise ValueError(f"q [B, T, H, D] and k, v [B, T, Hk, D] required, got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    if not k.shape[2] or q.shape[2] % k.shape[2]:
        raise ValueError(f"{q.shape[2]} query heads cannot share {k.shape[2]} key heads evenly")
    if native.active(q, k, v) and q.numel():
        return native.lib().window_attention_qkv(q, k, v, window, sinks)
    return core_window_attention(q, k, v, window, sinks)
