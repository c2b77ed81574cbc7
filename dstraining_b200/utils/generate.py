"""Sampling from a trained model.

    python -m dstraining_b200.utils.generate --ckpt ckpt/ --text "hello" --tokenizer bytes \
        --max-new-tokens 64 [--temperature 0.8 --top-k 40 --seed 0]

``generate(model, idx, ...)`` extends ``idx`` [B, T] token by token.
``temperature == 0`` is greedy decoding; otherwise tokens are sampled,
optionally from the ``top_k`` most probable and / or the nucleus of
probability ``top_p``. With ``device_sampling`` (or ``min_p``) the tokens are
drawn on the model's device by :func:`~dstraining_b200.ops.sampling.sample_tokens`
and nothing is copied to the host per token. Logits that leave no token to draw
(NaN throughout) raise ``RuntimeError``: at their token on the host's path, after
the last one with ``device_sampling``.

* With ``use_cache=True`` (the default) the prompt is run once and every
  later token costs one row per layer: its key and value are appended to a
  per-layer cache and its query attends over the cache (under tensor
  parallelism each rank caches its own heads; every rank of the group must
  call it with the same inputs and generator state).
  Positions are learned and absolute, so once the sequence outgrows
  ``block_size`` the window slides and every step re-runs the whole window,
  exactly as without a cache. Runs on the model's own parameters with
  PyTorch ops (fp32 on CPU, the model's dtype on CUDA).
* A model with an attention window, or ``cache_bits`` 16 or 4, decodes through
  :class:`~dstraining_b200.ops.kv_cache.WindowCache`: ``sinks + window`` slots
  per layer (the whole block without a window) in bf16 or 4 bits, appended to and
  attended over in one kernel per layer on CUDA bf16.
* Otherwise every step runs the model's full-context forward pass on the
  last ``block_size`` tokens, right-padded to a multiple of ``pad_to`` (the
  native causal attention kernels' 128-row tiles, so the sequence-parallel
  and fused tensor-parallel layers see whole tiles too) - under causal
  attention the padding never influences the positions before it. Every TP
  rank must call it with the same inputs and generator state; pipeline
  stages are not supported.

The CLI loads a sharded checkpoint (any layout) into a single-process model.
The reference has no sampling code.
"""

from __future__ import annotations

import argparse
import json
import os
from typing import Optional

import torch
import torch.distributed as dist
import torch.nn.functional as F

from ..models.gpt import GPT, GPTConfig
from ..ops.kv_cache import WindowCache
from ..ops.sampling import gumbel_noise, sample_tokens
from ..ops.window import window_attention
from ..parallel.comm import all_gather_dim
from ..parallel.topology import SINGLE


class KVCache:
    """Keys and values of every layer for the tokens seen so far, in
    preallocated ``[B, H, block_size, D]`` buffers, and the decoding step of
    a :class:`GPT` over them (PyTorch ops on the model's parameters). Under
    tensor parallelism each rank caches its own heads; the row-parallel
    outputs are summed over the group (bias added once, after the sum) and the
    vocabulary-sharded logits gathered, so every rank sees the same logits -
    every rank of the group must make the same calls.

    With ``bits`` (or a model that has an attention window) the rows live in one
    rolling :class:`WindowCache` per layer instead, and attention runs over it."""

    def __init__(self, model: GPT, batch: int, bits: Optional[int] = None):
        cfg = model.config
        self.model = model
        self.tp = model.tp
        p = model.wte.weight
        self.H, self.D = cfg.n_head // self.tp.world, cfg.n_embd // cfg.n_head
        self.len = 0
        self.window = min(cfg.attention_window or cfg.block_size, cfg.block_size)
        self.layers = None
        if bits is not None or cfg.attention_window:
            self.pos = torch.zeros(batch, dtype=torch.int64, device=p.device)  # shared by the layers
            self.layers = [WindowCache(batch, self.H, self.D, self.window, cfg.attention_sinks, bits=bits or 16,
                                       device=p.device, dtype=p.dtype, pos=self.pos) for _ in range(cfg.n_layer)]
            return
        shape = (batch, self.H, cfg.block_size, self.D)
        self.k = [torch.empty(shape, dtype=p.dtype, device=p.device) for _ in range(cfg.n_layer)]
        self.v = [torch.empty(shape, dtype=p.dtype, device=p.device) for _ in range(cfg.n_layer)]

    def _attend(self, i: int, qkv: torch.Tensor, p0: int) -> torch.Tensor:
        """Layer i's attention of qkv [B, t, H, 3, D] at positions p0.., its
        keys and values appended -> [B, t, H * D]."""
        b, t = qkv.shape[:2]
        if self.layers is not None:
            q, k, v = qkv.unbind(dim=3)
            if p0 == 0:
                self.layers[i].fill(k, v)
                return window_attention(qkv.reshape(b, t, -1), self.H, self.D, self.window, self.layers[i].sinks)
            return self.layers[i].step(q[:, 0], k[:, 0], v[:, 0], self.pos).reshape(b, t, -1)
        q, k, v = (qkv[:, :, :, j].transpose(1, 2) for j in range(3))
        self.k[i][:, :, p0 : p0 + t] = k
        self.v[i][:, :, p0 : p0 + t] = v
        keys, vals = self.k[i][:, :, : p0 + t], self.v[i][:, :, : p0 + t]
        # the window's first pass is causal; a single new token sees every cached one
        y = F.scaled_dot_product_attention(q, keys, vals, is_causal=p0 == 0 and t > 1)
        return y.transpose(1, 2).reshape(b, t, self.H * self.D)

    @staticmethod
    def _ln(ln, x):
        return F.layer_norm(x, ln.normalized_shape, ln.weight, ln.bias, ln.eps)

    def _row(self, x: torch.Tensor, layer) -> torch.Tensor:
        """Row-parallel linear: local partial product, sum over the group, then the full bias."""
        y = F.linear(x, layer.weight)
        if self.tp.enabled:
            dist.all_reduce(y, group=self.tp.group)
        return y + layer.bias if layer.bias is not None else y

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        """Run ``tokens`` [B, t] at positions ``len .. len + t - 1`` (the whole
        window when the cache is empty, else one token), append their keys and
        values, and return the logits [B, vocab] of the last one."""
        m, cfg = self.model, self.model.config
        b, t = tokens.shape
        p0 = self.len
        if p0 + t > cfg.block_size or (p0 > 0 and t != 1):
            raise ValueError("KVCache.forward: a full window first, then one token at a time")
        pos = torch.arange(p0, p0 + t, device=tokens.device)
        x = F.embedding(tokens, m.wte.weight) + F.embedding(pos, m.wpe.weight)[None]
        for i, blk in enumerate(m.blocks):
            a = blk.attn
            qkv = F.linear(self._ln(blk.ln_1, x), a.qkv.weight, a.qkv.bias).view(b, t, self.H, 3, self.D)
            x = x + self._row(self._attend(i, qkv, p0), a.proj)
            h = F.gelu(F.linear(self._ln(blk.ln_2, x), blk.mlp.c_fc.weight, blk.mlp.c_fc.bias), approximate="tanh")
            x = x + self._row(h, blk.mlp.c_proj)
        self.len = p0 + t
        if self.layers is not None and p0:
            self.pos += 1
        x = self._ln(m.ln_f, x[:, -1])
        logits = F.linear(x, m.lm_head.weight)  # this rank's vocabulary shard
        if self.tp.enabled:
            logits = all_gather_dim(logits, self.tp, 1)
        return logits[:, : cfg.vocab_size]


def _sample(logits: torch.Tensor, temperature: float, top_k: Optional[int], generator,
            top_p: Optional[float] = None) -> torch.Tensor:
    logits = logits.float()
    if temperature <= 0:
        return logits.argmax(dim=-1, keepdim=True)
    logits = logits / temperature
    if top_k is not None and top_k < logits.shape[-1]:
        kth = torch.topk(logits, top_k, dim=-1).values[:, -1:]
        logits = logits.masked_fill(logits < kth, float("-inf"))
    probs = torch.softmax(logits, dim=-1)
    if top_p is not None and top_p < 1.0:
        # nucleus: the most probable tokens whose probabilities sum to top_p (at least one)
        sorted_p, order = probs.sort(dim=-1, descending=True)
        drop = sorted_p.cumsum(dim=-1) - sorted_p >= top_p
        sorted_p = sorted_p.masked_fill(drop, 0.0)
        probs = torch.zeros_like(probs).scatter_(-1, order, sorted_p)
        probs = probs / probs.sum(dim=-1, keepdim=True)
    return torch.multinomial(probs.cpu(), 1, generator=generator).to(logits.device)


def _full_context_logits(model: GPT, idx: torch.Tensor, pad_to: int) -> torch.Tensor:
    cfg = model.config
    ctx = idx[:, -cfg.block_size:]
    n = ctx.shape[1]
    padded = min(cfg.block_size, -(-n // pad_to) * pad_to) if pad_to > 1 else n
    if padded > n:
        ctx = torch.cat([ctx, ctx.new_zeros(ctx.shape[0], padded - n)], dim=1)
    logits, _ = model(ctx)
    return logits[:, n - 1, : cfg.vocab_size]


@torch.no_grad()
def generate(model: GPT, idx: torch.Tensor, max_new_tokens: int, temperature: float = 1.0,
             top_k: Optional[int] = None, generator: Optional[torch.Generator] = None, pad_to: int = 128,
             use_cache: bool = True, top_p: Optional[float] = None, cache_bits: Optional[int] = None,
             min_p: Optional[float] = None, device_sampling: bool = False) -> torch.Tensor:
    cfg = model.config
    cache = KVCache(model, idx.shape[0], cache_bits) if use_cache else None
    was_training = model.training
    model.eval()
    least = None  # least token drawn on the device so far, per row: -1 where the logits left none
    try:
        for _ in range(max_new_tokens):
            if cache is None or idx.shape[1] > cfg.block_size:
                logits = _full_context_logits(model, idx, pad_to)  # window slides: positions shift
            elif cache.len == 0:
                logits = cache.forward(idx)
            else:
                logits = cache.forward(idx[:, -1:])
            if device_sampling or min_p:
                noise = gumbel_noise(*logits.shape, generator.device if generator is not None else logits.device, generator)
                nxt = sample_tokens(logits, noise.to(logits.device), max(temperature, 0.0), top_k or 0,
                                    1.0 if top_p is None else top_p, min_p or 0.0)[0][:, None]
                # -1 must not reach the embedding; the error waits for the end, where one copy to the host tells
                least = nxt if least is None else torch.minimum(least, nxt)
                nxt = nxt.clamp(min=0)
            else:
                nxt = _sample(logits, temperature, top_k, generator, top_p)
            idx = torch.cat([idx, nxt.to(idx.dtype)], dim=1)
    finally:
        model.train(was_training)
    if least is not None and (least < 0).any().item():
        raise RuntimeError("generate: a row of logits is NaN or -inf throughout, there is no token to draw")
    return idx


def load_model(ckpt: str, device: str = "cpu", dtype: torch.dtype = torch.float32) -> GPT:
    """A single-process GPT holding the weights of a sharded checkpoint (a step
    directory, or a root whose latest complete checkpoint is used)."""
    from . import checkpoint

    path = ckpt if os.path.exists(os.path.join(ckpt, "manifest.json")) else checkpoint.latest(ckpt)
    if path is None:
        raise FileNotFoundError(f"no complete checkpoint under {ckpt}")
    with open(os.path.join(path, "manifest.json")) as f:
        conf = json.load(f)["config"]
    fields = set(GPTConfig.__dataclass_fields__)
    cfg = GPTConfig(**{k: v for k, v in conf.items() if k in fields and k != "sequence_parallel"})
    model = GPT(cfg, SINGLE, seed=0)
    checkpoint.load(path, model, None, SINGLE)
    return model.to(device).to(dtype)


def main(argv=None) -> None:
    ap = argparse.ArgumentParser(description="sample from a trained checkpoint")
    ap.add_argument("--ckpt", required=True)
    ap.add_argument("--text", default=None, help="prompt text (needs --tokenizer)")
    ap.add_argument("--tokens", default=None, help="prompt as comma-separated token ids")
    ap.add_argument("--tokenizer", default="bytes", help="'bytes' or a tokenizer.json path")
    ap.add_argument("--max-new-tokens", type=int, default=64)
    ap.add_argument("--temperature", type=float, default=1.0)
    ap.add_argument("--top-k", type=int, default=None)
    ap.add_argument("--top-p", type=float, default=None, help="nucleus sampling")
    ap.add_argument("--min-p", type=float, default=None,
                    help="keep tokens at least this times as probable as the most probable (on the device)")
    ap.add_argument("--cache-bits", type=int, choices=(16, 4), default=None,
                    help="decode through the rolling key/value cache in bf16 or 4 bits")
    ap.add_argument("--device-sampling", action="store_true", help="draw tokens on the model's device")
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    a = ap.parse_args(argv)
    dtype = torch.bfloat16 if a.device.startswith("cuda") else torch.float32
    model = load_model(a.ckpt, a.device, dtype)
    if a.tokens:
        ids = [int(t) for t in a.tokens.split(",")]
        decode = None
    else:
        from .prepare_data import make_tokenizer

        tok = make_tokenizer(a.tokenizer)
        ids = tok.encode(a.text or "")
        if not ids:
            ids = [tok.eot]
        decode = (lambda out: bytes(t for t in out if t < 256).decode("utf-8", "replace")) if a.tokenizer == "bytes" \
            else (lambda out: tok.tok.decode(out))
    idx = torch.tensor([ids], dtype=torch.long, device=a.device)
    on_device = a.device_sampling or bool(a.min_p)
    g = torch.Generator(device=a.device if on_device else "cpu").manual_seed(a.seed)
    out = generate(model, idx, a.max_new_tokens, a.temperature, a.top_k, g, top_p=a.top_p, cache_bits=a.cache_bits,
                   min_p=a.min_p, device_sampling=a.device_sampling)[0].tolist()
    print(decode(out) if decode else ",".join(map(str, out)))


if __name__ == "__main__":
    main()
