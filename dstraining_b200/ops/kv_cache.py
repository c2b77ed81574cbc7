"""Rolling key/value cache of windowed attention with sinks, in bf16 or 4 bits.

One :class:`WindowCache` holds the keys and values of one layer: ``sinks +
window`` slots per (sequence, key head). Token ``p`` lies in slot ``p`` while
``p < sinks`` and in ``sinks + (p - sinks) % window`` after, so a new token
takes the slot of the one that leaves the window and the memory of a sequence
never grows. With ``window`` as long as the context it is an ordinary cache.

* :meth:`WindowCache.fill` writes the visible tokens of prompts (ragged lengths);
* :meth:`WindowCache.step` stores one token per sequence and attends over the
  cache with it, in one kernel (a long cache is split over the GPU and joined in
  the same launch) for given positions; the cache's own positions are advanced by
  two small launches more;
* :meth:`WindowCache.read` returns the held rows.

``bits=4`` stores, for each 32 channels of a row, ``step = bf16((max - min) /
15)``, ``low = min`` and 4-bit codes ``clamp(rint((x - low) / step), 0, 15)``;
a channel stands for ``low + code * step``: 20 bytes per 32 channels instead of
64. A group with an infinity or NaN stands for NaN.

CUDA bf16 runs the kernels of ``csrc/kv_cache.cu`` (head sizes multiples of 8 up
to 128, of 32 for 4 bits); anything else the PyTorch form of the same definition.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import native

GROUP = 32  # channels that share a step


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """[..., D] -> codes uint8 [..., D / 32, 32], step and low bf16 [..., D / 32, 1]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    low, high = g.amin(dim=-1, keepdim=True), g.amax(dim=-1, keepdim=True)
    step = ((high - low) / torch.full_like(high, 15.0)).to(torch.bfloat16)
    code = torch.where(step > 0, (g - low) / step.float(), torch.zeros((), device=x.device))
    code = code.round().nan_to_num(0.0).clamp(0, 15)
    return code.to(torch.uint8), step, low.to(torch.bfloat16)


def dequantize_rows(code: torch.Tensor, step: torch.Tensor, low: torch.Tensor) -> torch.Tensor:
    """What the codes stand for, fp32 [..., D]."""
    return (code.float() * step.float() + low.float()).flatten(-2)


class WindowCache:
    """Keys and values of one layer for ``batch`` sequences.

    ``pos`` [batch] int64 is the number of tokens each sequence has seen. It may
    be shared by the caches of several layers (``pos=``): :meth:`step` with
    explicit positions does not change it.

    Calls on one cache must be ordered (one stream, or streams that wait for one
    another): they share its rows and workspace. The caller owns the tensors of
    a call until the stream has passed it."""

    def __init__(self, batch: int, n_kv_head: int, head_dim: int, window: int, sinks: int = 0, *, bits: int = 16,
                 device=None, dtype: torch.dtype = torch.bfloat16, pos: Optional[torch.Tensor] = None):
        if batch < 1 or n_kv_head < 1 or head_dim < 1:
            raise ValueError("batch, n_kv_head and head_dim must be positive")
        if window < 1 or sinks < 0:
            raise ValueError(f"window >= 1 and sinks >= 0 required, got {window} and {sinks}")
        if bits not in (4, 16):
            raise ValueError(f"bits must be 4 or 16, got {bits}")
        if bits == 4 and head_dim % GROUP:
            raise ValueError(f"4-bit rows need a head_dim that is a multiple of {GROUP}, got {head_dim}")
        device = torch.device(device if device is not None else "cpu")
        self.batch, self.n_kv_head, self.head_dim = batch, n_kv_head, head_dim
        self.window, self.sinks, self.bits, self.dtype = window, sinks, bits, dtype
        self.slots = window + sinks
        self.device = device
        self.native = device.type == "cuda" and dtype == torch.bfloat16 and native.enabled()
        self.pos = pos if pos is not None else torch.zeros(batch, dtype=torch.int64, device=device)
        if self.pos.shape != (batch,) or self.pos.dtype != torch.int64:
            raise ValueError(f"pos must be an int64 tensor [{batch}]")
        if self.native:
            self._cache = native.lib().KVCache(batch, n_kv_head, head_dim, window, sinks, bits, self.pos)
            self._rows, self._params = self._cache.rows(), self._cache.params()
        elif bits == 16:
            rows = (batch, n_kv_head, self.slots, head_dim)
            self._rows = tuple(torch.zeros(rows, dtype=dtype, device=device) for _ in range(2))
        else:
            groups = (batch, n_kv_head, self.slots, head_dim // GROUP)
            self._rows = tuple(
                (torch.zeros(*groups, GROUP, dtype=torch.uint8, device=device),
                 torch.zeros(*groups, 1, dtype=torch.bfloat16, device=device),
                 torch.zeros(*groups, 1, dtype=torch.bfloat16, device=device)) for _ in range(2))

    # ------------------------------------------------------------- the rows
    @property
    def keys(self) -> torch.Tensor:
        """The slots' keys [B, Hk, slots, D] (a view; 16 bits)."""
        return self._buffer(0)

    @property
    def values(self) -> torch.Tensor:
        """The slots' values [B, Hk, slots, D] (a view; 16 bits)."""
        return self._buffer(1)

    def _buffer(self, i: int) -> torch.Tensor:
        if self.bits != 16:
            raise ValueError("4-bit rows have no bf16 buffer: use read()")
        return self._rows[i][:, :, : self.slots, : self.head_dim]

    def slot_of(self, pos: torch.Tensor) -> torch.Tensor:
        return torch.where(pos < self.sinks, pos, self.sinks + (pos - self.sinks) % self.window)

    def _check(self, x: torch.Tensor, shape, name: str) -> None:
        if tuple(x.shape) != tuple(shape):
            raise ValueError(f"{name} must be {list(shape)}, got {list(x.shape)}")
        if x.dtype != self.dtype or x.device.type != self.device.type:
            raise ValueError(f"{name} must be {self.dtype} on {self.device.type}, got {x.dtype} on {x.device.type}")

    def _positions(self, x: torch.Tensor, name: str) -> torch.Tensor:
        if tuple(x.shape) != (self.batch,) or x.dtype != torch.int64 or x.device.type != self.device.type:
            raise ValueError(f"{name} must be an int64 tensor [{self.batch}] on {self.device.type}")
        return x.contiguous()

    # ----------------------------------------------------------------- fill
    @torch.no_grad()
    def fill(self, k: torch.Tensor, v: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> None:
        """Start over with prompts k, v [B, T, Hk, D] (any strides) of which the
        first ``lengths`` [B] tokens count (default: all); ``pos`` becomes the
        lengths. Lengths outside 0..T are clamped and set the status word."""
        if self.native:
            self._cache.fill(k, v, lengths)
            return
        if k.dim() != 4:
            raise ValueError(f"k must be [B, T, Hk, D], got {list(k.shape)}")
        t = k.shape[1]
        self._check(k, (self.batch, t, self.n_kv_head, self.head_dim), "k")
        self._check(v, k.shape, "v")
        if lengths is not None:
            lengths = self._positions(lengths, "lengths")
        if t == 0:
            self.pos.zero_()
            return
        n = torch.full_like(self.pos, t) if lengths is None else lengths.clamp(0, t)
        s = torch.arange(self.slots, device=self.device)[None, :]
        wraps = torch.div(n[:, None] - 1 - s, self.window, rounding_mode="floor").clamp(min=0)
        token = torch.where(s < self.sinks, s, s + self.window * wraps)
        there = token < n[:, None]
        index = token.clamp(max=t - 1)[:, :, None, None].expand(-1, -1, self.n_kv_head, self.head_dim)
        for buffer, x in zip(self._rows, (k, v)):
            rows = torch.gather(x, 1, index).transpose(1, 2)
            self._put(buffer, rows, there[:, None, :, None].expand_as(rows))
        self.pos.copy_(n)

    def _put(self, buffer, rows: torch.Tensor, there: torch.Tensor) -> None:
        if self.bits == 16:
            buffer.copy_(torch.where(there, rows, buffer))
            return
        for held, new in zip(buffer, quantize_rows(rows)):
            held.copy_(torch.where(there[..., :1, None], new, held))

    # ----------------------------------------------------------------- read
    def read(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys and values [B, Hk, slots, D] in slot order, 0 where no token is:
        the cache's dtype, or fp32 for 4 bits."""
        if self.native:
            return tuple(self._cache.read())
        seen = torch.arange(self.slots, device=self.device)[None, :] < self.pos[:, None]
        rows = (x if self.bits == 16 else dequantize_rows(*x) for x in self._rows)
        return tuple(torch.where(seen[:, None, :, None], x, torch.zeros((), dtype=x.dtype, device=x.device))
                     for x in rows)

    # ----------------------------------------------------------------- step
    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pos: Optional[torch.Tensor] = None,
             return_stored: bool = False):
        """One token per sequence: q [B, H, D], k and v [B, Hk, D] (any strides;
        query head h reads key head ``h // (H / Hk)``). The token's key and value
        enter the cache, then its query attends over it -> [B, H, D].

        ``pos`` [B] int64: the tokens' positions, -1 for an idle sequence (stores
        nothing, result 0). By default the cache's own ``pos``, which advances.
        ``return_stored`` also returns what the stored key and value stand for
        (fp32 [B, Hk, D], 0 for idle sequences)."""
        at = self.pos if pos is None else pos
        if self.native:
            result = self._cache.step(q, k, v, at, return_stored)
        else:
            if q.dim() != 3 or q.shape[1] % self.n_kv_head or not q.shape[1]:
                raise ValueError(f"q must be [B, H, D] with H a multiple of {self.n_kv_head}, got {list(q.shape)}")
            self._check(q, (self.batch, q.shape[1], self.head_dim), "q")
            self._check(k, (self.batch, self.n_kv_head, self.head_dim), "k")
            self._check(v, k.shape, "v")
            result = self._plain_step(q, k, v, self._positions(at, "pos"), return_stored)
        if pos is None:
            self.pos += (self.pos >= 0)
        return tuple(result) if return_stored else result[0]

    @torch.no_grad()
    def _plain_step(self, q, k, v, pos, return_stored):
        on = (pos >= 0)[:, None, None]
        which = torch.arange(self.slots, device=self.device)[None, :] == self.slot_of(pos)[:, None]
        there = (which & (pos >= 0)[:, None])[:, None, :, None]
        for buffer, x in zip(self._rows, (k, v)):
            rows = x[:, :, None, :].expand(-1, -1, self.slots, -1)
            self._put(buffer, rows, there.expand_as(rows))
        keys, values = (x if self.bits == 16 else dequantize_rows(*x) for x in self._rows)
        groups = q.shape[1] // self.n_kv_head
        qg = q.to(keys.dtype).unflatten(1, (self.n_kv_head, groups))
        scores = (qg @ keys.transpose(-2, -1)) / math.sqrt(self.head_dim)
        seen = torch.arange(self.slots, device=self.device)[None, :] < (pos + 1)[:, None]
        scores = scores.masked_fill(~seen[:, None, None, :], float("-inf"))
        values = torch.where(seen[:, None, :, None], values, torch.zeros((), dtype=values.dtype, device=self.device))
        probs = torch.where(on[..., None], torch.softmax(scores, dim=-1), torch.zeros((), device=self.device, dtype=scores.dtype))
        out = (probs @ values).flatten(1, 2).to(q.dtype)
        if not return_stored:
            return (out,)
        stored = (x.float() if self.bits == 16 else dequantize_rows(*quantize_rows(x)) for x in (k, v))
        return (out, *(torch.where(on, x, torch.zeros((), device=self.device)) for x in stored))
