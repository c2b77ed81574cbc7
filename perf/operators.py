"""Workloads of the windowed-attention and sampling operators.

Four operators of a GPT whose attention sees a sliding window and a few first
tokens (sinks), in the order in which a model uses them:

* ``train``    attention of whole sequences and its gradients;
* ``prefill``  attention of a prompt, and the key/value cache written from it;
* ``step``     one decoded token per sequence: its key and value enter the cache
  (bf16 or 4 bits), its query attends over the cache;
* ``sample``   the next token from logits and given Gumbel noise.

Key ``j`` is visible to query ``i`` iff ``j <= i`` and (``i - j < window`` or
``j < sinks``). The cache holds ``sinks + window`` slots: token ``p`` lies in
slot ``p`` while ``p < sinks`` and in ``sinks + (p - sinks) % window`` after.

``run`` computes the operators in elementary torch operations (``own`` false) or
through the framework (``own`` true); ``exact`` in 64 bits.
"""

import math

import torch

own = False

DEVICE = "cuda"
VOCAB, PADDED_VOCAB = 50257, 50304  # GPT-2's, padded as the LM head pads it


# ---------------------------------------------------------------- the cases
def listed():
    def attn(name, op, batch, length, heads, kv_heads, dim, window, sinks, **more):
        return dict(name=name, op=op, batch=batch, length=length, heads=heads, kv_heads=kv_heads, dim=dim,
                    window=window, sinks=sinks, **more)

    return [
        # fine-tuning on short texts: a length and batch that fill no tile
        attn("train_short_odd", "train", 2, 333, 12, 12, 64, 128, 4, fused=True),
        # the GPT-2 small layer of the benchmark with a quarter-length window
        attn("train_gpt2", "train", 8, 1024, 12, 12, 64, 256, 4, fused=True),
        # long-context training of a 16-head, 2048-wide layer
        attn("train_long", "train", 1, 8192, 16, 16, 128, 1024, 4, fused=True),
        # the first pass of an interactive prompt: latency counts
        attn("prefill_prompt", "prefill", 1, 45, 12, 12, 64, 1020, 4, bits=16),
        # ragged long prompts with shared key heads into a 4-bit cache
        attn("prefill_shared_4bit", "prefill", 2, 4001, 16, 4, 128, 1000, 8, bits=4),
        # a single user's token: latency counts
        attn("step_one", "step", 1, 701, 12, 12, 64, 1020, 4, bits=16),
        # a full serving batch, ragged, some slots idle
        attn("step_batch", "step", 64, 6000, 16, 16, 128, 4092, 4, bits=16),
        # a single user's long context in 4 bits
        attn("step_long_4bit", "step", 1, 50000, 12, 12, 64, 32764, 4, bits=4),
        # the serving batch in 4 bits
        attn("step_batch_4bit", "step", 64, 6000, 16, 16, 128, 4092, 4, bits=4),
        # shared key heads over a long window in 4 bits
        attn("step_shared_4bit", "step", 16, 20011, 16, 2, 128, 16380, 4, bits=4),
        # one user's next token from bf16 logits, the same settings every call
        dict(name="sample_one", op="sample", batch=1, vocab=VOCAB, dtype="bfloat16", per_row=False),
        # a serving batch whose requests each have their own settings
        dict(name="sample_batch", op="sample", batch=128, vocab=VOCAB, dtype="float32", per_row=True),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["train", "prefill", "step", "step", "sample"])
    if op == "sample":
        return dict(op=op, batch=_log_uniform(rng, 1, 128), vocab=_log_uniform(rng, 300, VOCAB),
                    dtype=rng.choice(["bfloat16", "float32"]), per_row=rng.random() < 0.5)
    dim = rng.choice([64, 128])
    heads = rng.choice([12, 16] if op == "train" else [8, 12, 16])
    kv_heads = rng.choice([heads, heads, heads // 4 if op != "step" else heads // 2, 2])
    sinks = rng.choice([0, 1, 4, rng.randint(2, 150)])
    case = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, sinks=sinks)
    if op == "step":
        window = _log_uniform(rng, 64, 32764)
        # no more cached tokens in all than the largest listed batch holds
        batch = _log_uniform(rng, 1, max(1, min(64, 64 * 16 * 4096 * 128 // (kv_heads * (window + sinks) * dim))))
        return dict(case, batch=batch, length=_log_uniform(rng, 2, 2 * window), window=window,
                    bits=rng.choice([16, 4]))
    length = _log_uniform(rng, 40, 8192)
    window = _log_uniform(rng, min(32, length), length)
    # no more scores in all than the largest listed sequence has
    batch = _log_uniform(rng, 1, max(1, min(8, 16 * 8192 * 8192 // (heads * length * length))))
    case.update(batch=batch, length=length, window=window)
    if op == "train":
        return dict(case, fused=kv_heads == heads and rng.random() < 0.5)
    return dict(case, bits=rng.choice([16, 4]))


def _visible_pairs(length, window, sinks):
    total = 0
    for i in range(length):
        low = max(0, i - window + 1)
        total += i + 1 - low + min(sinks, low)
    return total


def work(case):
    if case["op"] == "sample":
        # each logit once; the noise of the few tokens that stay, and the answer, are nothing beside it
        size = 2 if case["dtype"] == "bfloat16" else 4
        n = case["batch"] * case["vocab"]
        return {"bytes": n * size + 16 * case["batch"], "flops": 3 * n}
    b, h, g, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "step":
        slots = case["window"] + case["sinks"]
        held = sum(min(p + 1, slots) for p in _positions(case))
        row = 2 * d if case["bits"] == 16 else d // 2 + d // 32 * 4
        active = sum(p >= 0 for p in _positions(case))
        return {"bytes": 2 * held * g * row + active * (2 * 2 * g * d + 2 * 2 * h * d), "flops": 4 * held * h * d}
    t = case["length"]
    pairs = b * h * _visible_pairs(t, case["window"], case["sinks"])
    q, kv = b * t * h * d * 2, b * t * g * d * 2
    if case["op"] == "train":
        return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * d}  # out and dout, q and dq; k, v and theirs
    # the cache comes back whole: as it is (16 bits) or in 32 bits
    slots = b * g * (case["window"] + case["sinks"])
    out = 2 * slots * d * (2 if case["bits"] == 16 else 4)
    held = 0 if case["bits"] == 16 else 2 * 2 * slots * (d // 2 + d // 32 * 4)
    return {"bytes": 2 * q + 2 * kv + out + held, "flops": 4 * pairs * d}


# ---------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, device=DEVICE, generator=g, dtype=torch.float32)


def _keys(g, *shape):
    """Keys with the few strong channels that trained models have."""
    channel = 1.0 + 3.0 * (torch.rand(shape[-1], device=DEVICE, generator=g) > 0.95)
    return (_normal(g, *shape) * channel).to(torch.bfloat16)


def _positions(case):
    """The position of each sequence's new token; ragged in a batch, -1 where the batch slot is idle."""
    b, last = case["batch"], case["length"] - 1
    if b == 1:
        return [last]
    return [-1 if i % 16 == 7 else last - (last * i * 7 // (8 * b)) for i in range(b)]


def _prepare_sample(case, g):
    b, v = case["batch"], case["vocab"]
    padded = v + PADDED_VOCAB - VOCAB
    dtype = torch.bfloat16 if case["dtype"] == "bfloat16" else torch.float32
    logits = (2.5 * _normal(g, b, padded)).to(dtype)[:, :v]  # the real columns of the padded vocabulary
    gumbel = -torch.log(torch.empty(b, v, device=DEVICE).exponential_(generator=g))
    if not case["per_row"]:
        return dict(case=case, logits=logits, gumbel=gumbel,
                    settings=dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.02))
    pick = lambda values: torch.tensor(values, device=DEVICE)[  # noqa: E731
        torch.randint(len(values), (b,), device=DEVICE, generator=g)]
    return dict(case=case, logits=logits, gumbel=gumbel,
                settings=dict(temperature=pick([0.0, 0.6, 0.8, 1.0, 1.3]), top_k=pick([0, 0, 20, 50, 1000]),
                              top_p=pick([1.0, 0.95, 0.9, 0.5]), min_p=pick([0.0, 0.0, 0.02, 0.1])))


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "sample":
        return _prepare_sample(case, g)
    b, t, h, kvh, d = case["batch"], case["length"], case["heads"], case["kv_heads"], case["dim"]
    state = dict(case=case)
    if case["op"] == "train":
        q, k, v = _normal(g, b, t, h, d).to(torch.bfloat16), _keys(g, b, t, kvh, d), _normal(g, b, t, kvh, d).to(torch.bfloat16)
        if case["fused"]:  # one buffer, head by head q | k | v, as the layer's projection writes it
            state["qkv"] = torch.stack([q, k, v], dim=3).reshape(b, t, 3 * h * d).requires_grad_()
        else:
            state["q"], state["k"], state["v"] = (x.requires_grad_() for x in (q, k, v))
        state["dout"] = _normal(g, b, t, h, d).to(torch.bfloat16)
        return state
    slots = case["window"] + case["sinks"]
    if case["op"] == "prefill":
        state["q"] = _normal(g, b, t, h, d).to(torch.bfloat16)
        state["k"], state["v"] = _keys(g, b, t, kvh, d), _normal(g, b, t, kvh, d).to(torch.bfloat16)
        state["lengths"] = torch.tensor([t - t * i // (3 * b) for i in range(b)], device=DEVICE)
        held_k = held_v = held_lengths = None
    else:
        pos = torch.tensor(_positions(case), device=DEVICE)
        state["pos"] = pos
        state["q"] = _normal(g, b, h, d).to(torch.bfloat16)
        state["k"], state["v"] = _keys(g, b, kvh, d), _normal(g, b, kvh, d).to(torch.bfloat16)
        # what the slots hold is as good as random wherever the window stands
        n = min(slots, max(1, case["length"]))
        held_k, held_v = _keys(g, b, n, kvh, d), _normal(g, b, n, kvh, d).to(torch.bfloat16)
        held_lengths = pos.clamp(0, n)
    if own:
        from dstraining_b200.ops.kv_cache import WindowCache

        state["cache"] = WindowCache(b, kvh, d, case["window"], case["sinks"], bits=case["bits"], device=DEVICE)
        if held_k is not None:
            state["cache"].fill(held_k, held_v, held_lengths)
        return state
    if held_k is None:
        return state
    for name, x in (("cache_k", held_k), ("cache_v", held_v)):
        state[name] = _plain_fill(x, held_lengths, case, slots)
        if case["bits"] == 4:
            state[name] = _plain_pack(state[name])
    return state


# ---------------------------------------------------------------- the plain form
def _mask(length, window, sinks):
    i = torch.arange(length, device=DEVICE)[:, None]
    j = torch.arange(length, device=DEVICE)[None, :]
    return (j <= i) & ((i - j < window) | (j < sinks))


def _plain_probs(q, k, case):
    """q, k: [B, H, T, D] in 32 bits -> probabilities."""
    s = (q @ k.transpose(-2, -1)) / math.sqrt(q.shape[-1])
    s = s.masked_fill_(~_mask(q.shape[2], case["window"], case["sinks"]), float("-inf"))
    p = torch.exp(s - s.amax(dim=-1, keepdim=True))
    return p / p.sum(dim=-1, keepdim=True)


def _heads_first(x, heads):
    """[B, T, H', D] of any type -> [B, heads, T, D] in 32 bits, shared heads repeated."""
    return x.float().transpose(1, 2).repeat_interleave(heads // x.shape[2], dim=1)


def _plain_train(state):
    case = state["case"]
    b, t, h, kvh, d = case["batch"], case["length"], case["heads"], case["kv_heads"], case["dim"]
    if case["fused"]:
        q, k, v = state["qkv"].detach().view(b, t, h, 3, d).unbind(dim=3)
    else:
        q, k, v = state["q"].detach(), state["k"].detach(), state["v"].detach()
    q, k, v, dout = (_heads_first(x, h) for x in (q, k, v, state["dout"]))
    p = _plain_probs(q, k, case)
    out = p @ v
    dv = p.transpose(-2, -1) @ dout
    dp = dout @ v.transpose(-2, -1)
    ds = p * (dp - (p * dp).sum(dim=-1, keepdim=True)) / math.sqrt(d)
    dq, dk = ds @ k, ds.transpose(-2, -1) @ q
    dk, dv = (x.view(b, kvh, h // kvh, t, d).sum(dim=2) for x in (dk, dv))
    out, dq, dk, dv = (x.transpose(1, 2).to(torch.bfloat16) for x in (out, dq, dk, dv))
    if case["fused"]:
        return out.reshape(b, t, h * d), torch.stack([dq, dk, dv], dim=3).reshape(b, t, 3 * h * d)
    return out, dq, dk, dv


def _plain_fill(x, lengths, case, slots):
    """x: [B, T, H, D] -> what the slots [B, H, slots, D] hold after the first `lengths` tokens (0 where nothing is)."""
    s = torch.arange(slots, device=DEVICE)[None, :]
    n = lengths[:, None]
    wraps = torch.div(n - 1 - s, case["window"], rounding_mode="floor").clamp(min=0)
    token = torch.where(s < case["sinks"], s, s + case["window"] * wraps)
    there = token < n
    rows = torch.gather(x, 1, token.clamp(max=x.shape[1] - 1)[:, :, None, None].expand(-1, -1, *x.shape[2:]))
    return rows.masked_fill(~there[:, :, None, None], 0).transpose(1, 2).contiguous()


def _plain_pack(x):
    """[..., D] bf16 -> 4-bit codes with a bf16 step and least value for each 32 channels."""
    groups = x.float().unflatten(-1, (-1, 32))
    low, high = groups.amin(dim=-1, keepdim=True), groups.amax(dim=-1, keepdim=True)
    step = ((high - low) / torch.full_like(high, 15.0)).to(torch.bfloat16).float()
    code = torch.where(step > 0, (groups - low) / step, 0.0).round().clamp(0, 15)
    return code.to(torch.uint8), step.to(torch.bfloat16), low.to(torch.bfloat16)


def _plain_unpack(packed):
    code, step, low = packed
    return (code.float() * step.float() + low.float()).flatten(-2)


def _plain_prefill(state):
    case = state["case"]
    h = case["heads"]
    q, k, v = (_heads_first(state[x], h) for x in ("q", "k", "v"))
    out = (_plain_probs(q, k, case) @ v).transpose(1, 2).to(torch.bfloat16)
    slots = case["window"] + case["sinks"]
    held = [_plain_fill(state[x], state["lengths"], case, slots) for x in ("k", "v")]
    if case["bits"] == 4:
        held = [_plain_unpack(_plain_pack(x)) for x in held]
    return out, held[0], held[1]


def _plain_step(state):
    case = state["case"]
    b, h, kvh, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    slots, pos = case["window"] + case["sinks"], state["pos"]
    rows = torch.arange(b, device=DEVICE)
    active = pos >= 0
    slot = torch.where(pos < case["sinks"], pos, case["sinks"] + (pos - case["sinks"]) % case["window"]).clamp(min=0)
    on = active[:, None, None]

    def put(buffer, new):  # idle sequences keep what they have
        keep = buffer[rows, :, slot]
        buffer[rows, :, slot] = torch.where(on.view(b, *[1] * (keep.dim() - 1)), new, keep)

    if case["bits"] == 16:
        put(state["cache_k"], state["k"])
        put(state["cache_v"], state["v"])
        k, v = state["cache_k"].float(), state["cache_v"].float()
        after = (state["cache_k"], state["cache_v"])
    else:
        new_k, new_v = _plain_pack(state["k"]), _plain_pack(state["v"])
        put(state["cache_k"][0], new_k[0]), put(state["cache_k"][1], new_k[1]), put(state["cache_k"][2], new_k[2])
        put(state["cache_v"][0], new_v[0]), put(state["cache_v"][1], new_v[1]), put(state["cache_v"][2], new_v[2])
        k, v = _plain_unpack(state["cache_k"]), _plain_unpack(state["cache_v"])
        after = tuple(torch.where(on, _plain_unpack(x), 0.0) for x in (new_k, new_v))
    q = state["q"].float().view(b, kvh, h // kvh, d)
    s = (q @ k.transpose(-2, -1)) / math.sqrt(d)
    seen = torch.arange(slots, device=DEVICE)[None, :] < (pos + 1).clamp(max=slots)[:, None]
    s = s.masked_fill(~seen[:, None, None, :], float("-inf"))
    p = torch.exp(s - s.amax(dim=-1, keepdim=True).clamp(min=-3e38))
    out = (p @ v) / p.sum(dim=-1, keepdim=True).clamp(min=1e-30)  # a sequence that sees nothing gets 0
    return (out.view(b, h, d).to(torch.bfloat16),) + after


def _columns(settings, batch):
    """Each setting as a [B, 1] column."""
    kinds = dict(temperature=torch.float32, top_k=torch.int64, top_p=torch.float32, min_p=torch.float32)
    return {n: torch.as_tensor(settings[n], device=DEVICE).to(kinds[n]).expand(batch)[:, None] for n in kinds}


def _plain_sample(state):
    logits, gumbel = state["logits"].float(), state["gumbel"]
    b, v = logits.shape
    s = _columns(state["settings"], b)
    greedy = s["temperature"] <= 0
    t = logits / torch.where(greedy, 1.0, s["temperature"])
    ranked, order = torch.sort(t, dim=-1, descending=True, stable=True)  # equal logits by index
    mass = torch.exp(ranked - ranked[:, :1])
    rank = torch.arange(v, device=DEVICE)[None, :]
    keep = (s["top_k"] <= 0) | (rank < s["top_k"])
    among = torch.where(keep, mass, 0.0)
    keep &= (s["top_p"] >= 1) | (among.cumsum(dim=-1) - among < s["top_p"] * among.sum(dim=-1, keepdim=True))
    keep &= mass >= s["min_p"]
    keep = torch.where(greedy, rank == 0, keep)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    token = torch.where(kept, t + gumbel, float("-inf")).argmax(dim=-1)
    log_total = ranked[:, 0] + torch.log(mass.sum(dim=-1))
    return token, t.gather(1, token[:, None])[:, 0] - log_total


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if not own:
        plain = dict(train=_plain_train, prefill=_plain_prefill, step=_plain_step, sample=_plain_sample)
        return plain[case["op"]](state)
    if case["op"] == "sample":
        from dstraining_b200.ops.sampling import sample_tokens

        return sample_tokens(state["logits"], state["gumbel"], **state["settings"])
    if case["op"] == "step":
        cache = state["cache"]
        if case["bits"] == 16:
            return cache.step(state["q"], state["k"], state["v"], state["pos"]), cache.keys, cache.values
        return cache.step(state["q"], state["k"], state["v"], state["pos"], return_stored=True)
    from dstraining_b200.ops.window import window_attention, window_attention_qkv

    if case["op"] == "prefill":
        out = window_attention_qkv(state["q"], state["k"], state["v"], case["window"], case["sinks"])
        state["cache"].fill(state["k"], state["v"], state["lengths"])
        return (out,) + tuple(state["cache"].read())
    if case["fused"]:
        out = window_attention(state["qkv"], case["heads"], case["dim"], case["window"], case["sinks"])
        return (out.detach(),) + torch.autograd.grad(out, state["qkv"], state["dout"].view_as(out))
    x = (state["q"], state["k"], state["v"])
    out = window_attention_qkv(*x, case["window"], case["sinks"])
    return (out.detach(),) + torch.autograd.grad(out, x, state["dout"])


# ---------------------------------------------------------------- 64 bits
def _exact_attention(q, k, v, case, dout=None):
    """One head, in blocks of queries over the keys that the block sees: q, k, v [T, D] in 64 bits."""
    t, d = q.shape
    w, s = case["window"], case["sinks"]
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i0 in range(0, t, 512):
        i = torch.arange(i0, min(t, i0 + 512), device=DEVICE)
        low = max(0, i0 - w + 1)
        j = torch.cat([torch.arange(0, min(s, low), device=DEVICE), torch.arange(low, int(i[-1]) + 1, device=DEVICE)])
        gap = i[:, None] - j[None, :]
        seen = (gap >= 0) & ((gap < w) | (j[None, :] < s))
        x = torch.einsum("id,jd->ij", q[i], k[j]) * d ** -0.5
        p = torch.softmax(x.masked_fill(~seen, float("-inf")), dim=1)
        out[i] = torch.einsum("ij,jd->id", p, v[j])
        if dout is not None:
            dp = torch.einsum("id,jd->ij", dout[i], v[j])
            ds = p * (dp - (out[i] * dout[i]).sum(dim=1, keepdim=True)) * d ** -0.5
            dq[i] = torch.einsum("ij,jd->id", ds, k[j])
            dk.index_add_(0, j, torch.einsum("ij,id->jd", ds, q[i]))
            dv.index_add_(0, j, torch.einsum("ij,id->jd", p, dout[i]))
    return out, dq, dk, dv


def _exact_stored(x):
    """What 4 bits stand for, for bf16 x [..., D]: least + code * step, the code from steps as the cache keeps them."""
    x = x.float().reshape(*x.shape[:-1], -1, 32)
    low = x.min(dim=-1, keepdim=True).values
    step = ((x.max(dim=-1, keepdim=True).values - low) / x.new_full((), 15.0).expand_as(low)).bfloat16().float()
    code = torch.where(step == 0, torch.zeros_like(x), torch.round((x - low) / step)).clamp_(0, 15)
    return (low.double() + code.double() * step.double()).flatten(-2)


def _exact_slots(x, lengths, case):
    """x [B, T, H, D] -> [B, H, slots, D], token by token of each slot."""
    b, t, h, d = x.shape
    w, s = case["window"], case["sinks"]
    out = x.new_zeros(b, h, w + s, d)
    for n, length in enumerate(lengths.tolist()):
        first = torch.arange(0, min(s, length), device=DEVICE)
        rest = torch.arange(max(s, length - w), length, device=DEVICE)
        out[n][:, first] = x[n, first].transpose(0, 1)
        if len(rest):
            out[n][:, s + (rest - s) % w] = x[n, rest].transpose(0, 1)
    return out


def _exact_step(case, seed):
    global own
    before, own = own, False  # the inputs as the plain form gets them
    try:
        state = prepare(case, seed)
    finally:
        own = before
    b, h, kvh, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    w, s = case["window"], case["sinks"]
    out = torch.zeros(b, h, d, dtype=torch.float64, device=DEVICE)
    new = [state[n] if case["bits"] == 16 else _exact_stored(state[n]) for n in ("k", "v")]
    stored = [torch.zeros(b, kvh, d, dtype=torch.float64, device=DEVICE) for _ in range(2)]
    for n, p in enumerate(state["pos"].tolist()):
        if p < 0:
            continue
        slot = p if p < s else s + (p - s) % w
        kv = []
        for i, name in enumerate(("cache_k", "cache_v")):
            if case["bits"] == 16:
                state[name][n, :, slot] = new[i][n]
                rows = state[name][n].double()
            else:
                code, step, low = (x[n].double() for x in state[name])
                rows = (low + code * step).flatten(-2)
                rows[:, slot] = stored[i][n] = new[i][n]
            kv.append(rows[:, : min(p + 1, w + s)])
        q = state["q"][n].double().view(kvh, h // kvh, d)
        p_ = torch.softmax(torch.einsum("gqd,gkd->gqk", q, kv[0]) * d ** -0.5, dim=-1)
        out[n] = torch.einsum("gqk,gkd->gqd", p_, kv[1]).reshape(h, d)
    if case["bits"] == 16:
        return out, state["cache_k"], state["cache_v"]
    return out, stored[0], stored[1]


def _exact_sample(case, seed):
    state = prepare(case, seed)
    b, v = state["logits"].shape
    s = {n: x[:, 0].tolist() for n, x in _columns(state["settings"], b).items()}
    token = torch.zeros(b, dtype=torch.int64, device=DEVICE)
    logprob = torch.zeros(b, dtype=torch.float64, device=DEVICE)
    for n in range(b):
        warm = s["temperature"][n]
        t = state["logits"][n].double() / (warm if warm > 0 else 1.0)
        p = torch.softmax(t, dim=0)
        order = torch.argsort(t, descending=True, stable=True)
        if warm <= 0:
            order = order[:1]
        if s["top_k"][n] > 0:
            order = order[: s["top_k"][n]]
        if s["top_p"][n] < 1:
            c = torch.cumsum(p[order], dim=0)
            order = order[: int((c - p[order] < s["top_p"][n] * c[-1]).sum())]
        order = order[p[order] >= s["min_p"][n] * p.max()]
        token[n] = order[(t[order] + state["gumbel"][n, order].double()).argmax()]
        logprob[n] = t[token[n]] - torch.logsumexp(t, dim=0)
    return token, logprob


def exact(case, seed):
    if case["op"] == "sample":
        return _exact_sample(case, seed)
    if case["op"] == "step":
        return _exact_step(case, seed)
    state = prepare(case, seed)
    b, t, h, kvh, d = case["batch"], case["length"], case["heads"], case["kv_heads"], case["dim"]
    fused = case["op"] == "train" and case["fused"]
    if fused:
        q, k, v = state["qkv"].detach().view(b, t, h, 3, d).unbind(dim=3)
    else:
        q, k, v = (state[n].detach() for n in ("q", "k", "v"))
    dout = state["dout"] if case["op"] == "train" else None
    out, dq = (torch.zeros(b, t, h, d, dtype=torch.float64, device=DEVICE) for _ in range(2))
    dk, dv = (torch.zeros(b, t, kvh, d, dtype=torch.float64, device=DEVICE) for _ in range(2))
    for n in range(b):
        for i in range(h):
            g = i * kvh // h
            got = _exact_attention(q[n, :, i].double(), k[n, :, g].double(), v[n, :, g].double(), case,
                                   None if dout is None else dout[n, :, i].double())
            out[n, :, i], dq[n, :, i] = got[0], got[1]
            dk[n, :, g] += got[2]
            dv[n, :, g] += got[3]
    if case["op"] == "prefill":
        held = [_exact_slots(state[n], state["lengths"], case) for n in ("k", "v")]
        if case["bits"] == 4:
            held = [_exact_stored(x) for x in held]
        return out, held[0], held[1]
    if fused:
        return out.reshape(b, t, h * d), torch.stack([dq, dk, dv], dim=3).reshape(b, t, 3 * h * d)
    return out, dq, dk, dv
