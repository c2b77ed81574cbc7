"""Sliding-window attention with sinks, the rolling key/value cache and device
sampling (new; the reference has none of them)."""

from dstraining_b200.ops.kv_cache import WindowCache  # noqa: F401
from dstraining_b200.ops.sampling import gumbel_noise, sample_tokens  # noqa: F401
from dstraining_b200.ops.window import window_attention, window_attention_qkv  # noqa: F401
