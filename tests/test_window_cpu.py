"""Windowed attention, the rolling cache and device sampling in their PyTorch
form, and the model and the decoder that use them."""

import math

import pytest
import torch

from dstraining_b200.models.gpt import GPT, GPTConfig
from dstraining_b200.ops.kv_cache import WindowCache, dequantize_rows, quantize_rows
from dstraining_b200.ops.sampling import gumbel_noise, sample_tokens
from dstraining_b200.ops.window import window_attention, window_attention_qkv, window_mask
from dstraining_b200.parallel.topology import SINGLE
from dstraining_b200.utils.export_hf import hf_config
from dstraining_b200.utils.generate import KVCache, generate


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def test_mask():
    m = window_mask(6, 2, 1)
    assert m.int().tolist() == [[1, 0, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0], [1, 1, 1, 0, 0, 0], [1, 0, 1, 1, 0, 0],
                                [1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 1]]
    assert torch.equal(window_mask(5, 5, 0), torch.ones(5, 5, dtype=torch.bool).tril())


def test_gradients_against_differences():
    x = [torch.randn(1, 9, h, 4, generator=_gen(h), dtype=torch.double).requires_grad_() for h in (4, 2, 2)]
    assert torch.autograd.gradcheck(lambda *t: window_attention_qkv(*t, 3, 2), x)


def test_fused_buffer_and_refusals():
    qkv = torch.randn(2, 7, 3 * 2 * 4, generator=_gen(0))
    q, k, v = qkv.view(2, 7, 2, 3, 4).unbind(dim=3)
    assert torch.equal(window_attention(qkv, 2, 4, 3, 1), window_attention_qkv(q, k, v, 3, 1).reshape(2, 7, 8))
    with pytest.raises(ValueError, match="window"):
        window_attention(qkv, 2, 4, 0)
    with pytest.raises(ValueError, match="qkv"):
        window_attention(qkv, 2, 8, 3)


@pytest.mark.parametrize("bits", [16, 4])
def test_cache_is_attention_over_the_window(bits):
    """Prompt, then tokens one by one: the rows of whole-sequence attention (over
    what the stored rows stand for), also long after the ring has wrapped."""
    B, T, n, H, Hk, D, W, S = 2, 40, 17, 4, 2, 32, 9, 3
    q, k, v = (torch.randn(B, T, h, D, generator=_gen(h + i)) for i, h in enumerate((H, Hk, Hk)))
    cache = WindowCache(B, Hk, D, W, S, bits=bits, dtype=torch.float32)
    cache.fill(k[:, :n], v[:, :n])
    kk, vv = (k, v) if bits == 16 else (dequantize_rows(*quantize_rows(x)) for x in (k, v))
    want = window_attention_qkv(q, kk, vv, W, S)
    for t in range(n, T):
        out = cache.step(q[:, t], k[:, t], v[:, t])
        torch.testing.assert_close(out, want[:, t], atol=1e-5, rtol=1e-5)
    assert cache.pos.tolist() == [T, T]


def test_cache_ragged_idle_and_empty():
    cache = WindowCache(3, 1, 8, 4, 2, dtype=torch.float32)
    k = torch.randn(3, 9, 1, 8, generator=_gen(1))
    cache.fill(k, k, torch.tensor([9, 1, 0]))
    held, _ = cache.read()
    # sinks 0, 1, then the ring: tokens 5..8 at 2 + (p - 2) % 4
    assert torch.equal(held[0, 0], k[0, [0, 1, 6, 7, 8, 5], 0])
    assert torch.equal(held[1, 0, 0], k[1, 0, 0]) and not held[1, 0, 1:].any() and not held[2].any()
    new = torch.randn(3, 1, 8, generator=_gen(2))
    out, ks, _ = cache.step(new, new, new, torch.tensor([9, -1, 0]), return_stored=True)
    assert not out[1].any() and not ks[1].any()
    assert torch.equal(out[2], new[2])
    assert torch.equal(cache.keys[0, 0, 2 + (9 - 2) % 4], new[0, 0])
    assert torch.equal(cache.keys[1, 0, 0], k[1, 0, 0])
    assert cache.pos.tolist() == [9, 1, 0]  # explicit positions leave it alone


def test_cache_refusals():
    for kw, what in ((dict(bits=8), "bits"), (dict(window=0), "window"), (dict(sinks=-1), "sinks"),
                     (dict(bits=4, head_dim=24), "multiple of 32"), (dict(batch=0), "positive"),
                     (dict(pos=torch.zeros(3, dtype=torch.int64)), "pos")):
        args = dict(batch=1, n_kv_head=1, head_dim=32, window=4, sinks=0, dtype=torch.float32)
        args.update(kw)
        with pytest.raises(ValueError, match=what):
            WindowCache(**args)
    cache = WindowCache(1, 1, 32, 4, bits=4, dtype=torch.float32)
    with pytest.raises(ValueError, match="read"):
        cache.keys


def test_quantization_bounds():
    """Each value within half a step, up to the rounding of the step (2^-9) over 15 steps."""
    x = torch.randn(50, 64, generator=_gen(3)).to(torch.bfloat16)
    code, step, low = quantize_rows(x)
    err = (dequantize_rows(code, step, low) - x.float()).abs().unflatten(-1, (-1, 32))
    assert (err <= step.float() * (0.5 + 15 * 2.0**-8)).all()
    assert torch.isnan(dequantize_rows(*quantize_rows(torch.tensor([[float("nan")] + [0.0] * 31])))).all()


def test_sampling_keeps_the_right_tokens():
    x = torch.log(torch.tensor([[0.05, 0.4, 0.1, 0.3, 0.15]]))
    flat = torch.zeros(1, 5)
    def kept(**kw):  # a token is kept iff noise can make it win
        out = set()
        for i in range(5):
            g = flat.clone()
            g[0, i] = 100.0
            out.add(sample_tokens(x, g, **kw)[0].item())
        return out
    assert kept() == {0, 1, 2, 3, 4}
    assert kept(top_k=2) == {1, 3}
    assert kept(top_p=0.6) == {1, 3}
    assert kept(top_p=0.75) == {1, 3, 4}
    assert kept(top_k=3, top_p=0.45) == {1}  # 0.4 of 0.85 is not enough: 0.47
    assert kept(min_p=0.3) == {1, 3, 4}
    assert kept(temperature=0.0) == {1} == kept(top_p=0.0) == kept(min_p=2.0)
    token, logprob = sample_tokens(x, flat, temperature=0.0)
    assert token.item() == 1 and abs(logprob.item() - math.log(0.4)) < 1e-6


def test_sampling_broken_rows_and_refusals():
    inf = float("inf")
    x = torch.tensor([[-inf, -inf, -inf], [float("nan"), 1.0, -inf], [0.0, inf, inf], [2.0, 2.0, 2.0]])
    token, logprob = sample_tokens(x, torch.zeros(4, 3))
    assert token.tolist() == [-1, 1, 1, 0]
    assert logprob[0] == -inf and logprob[1] == 0 and abs(logprob[2].item() + math.log(2)) < 1e-6
    # all scores -inf: equal, so the lowest index of the kept
    assert sample_tokens(x, torch.full((4, 3), -inf))[0].tolist() == [-1, 1, 0, 0]
    with pytest.raises(ValueError, match="gumbel"):
        sample_tokens(x, torch.zeros(4, 2))
    with pytest.raises(ValueError, match="temperature"):
        sample_tokens(x, torch.zeros(4, 3), temperature=-1)
    with pytest.raises(ValueError, match="top_p"):
        sample_tokens(x, torch.zeros(4, 3), top_p=torch.ones(3))


CFG = dict(vocab_size=300, block_size=64, n_layer=2, n_head=2, n_embd=64)


def test_model_with_a_window():
    """A window of the whole block changes nothing; a short one only late positions."""
    idx = torch.randint(0, 300, (2, 40), generator=_gen(4))
    full, _ = GPT(GPTConfig(**CFG), SINGLE, seed=3)(idx)
    same, _ = GPT(GPTConfig(**CFG, attention_window=64), SINGLE, seed=3)(idx)
    torch.testing.assert_close(full, same, atol=1e-5, rtol=1e-5)
    short, _ = GPT(GPTConfig(**CFG, attention_window=8, attention_sinks=2), SINGLE, seed=3)(idx)
    torch.testing.assert_close(full[:, :8], short[:, :8], atol=1e-5, rtol=1e-5)
    assert (full[:, 30:] - short[:, 30:]).abs().max() > 1e-4
    model = GPT(GPTConfig(**CFG, attention_window=8, recompute_attention=True), SINGLE, seed=3)
    _, loss = model(idx, idx)
    loss.backward()
    other = GPT(GPTConfig(**CFG, attention_window=8), SINGLE, seed=3)
    _, loss2 = other(idx, idx)
    loss2.backward()
    for a, b in zip(model.parameters(), other.parameters()):
        torch.testing.assert_close(a.grad, b.grad)


def test_window_configuration_refusals():
    with pytest.raises(ValueError, match="attention_sinks"):
        GPTConfig(**CFG, attention_sinks=4)
    with pytest.raises(ValueError, match="negative"):
        GPTConfig(**CFG, attention_window=-1)
    with pytest.raises(ValueError, match="sliding-window"):
        hf_config(GPT(GPTConfig(**CFG, attention_window=8), SINGLE, seed=0))


@pytest.mark.parametrize("window,sinks,bits", [(0, 0, 16), (8, 2, None), (64, 0, 16)])
def test_decoder_over_the_rolling_cache(window, sinks, bits):
    m = GPT(GPTConfig(**CFG, attention_window=window, attention_sinks=sinks), SINGLE, seed=7).eval()
    seq = torch.randint(0, 300, (3, 40), generator=_gen(2))
    cache = KVCache(m, 3, bits)
    with torch.no_grad():
        got = [cache.forward(seq[:, :9])] + [cache.forward(seq[:, t : t + 1]) for t in range(9, 40)]
        full, _ = m(seq)
    torch.testing.assert_close(torch.stack(got, dim=1), full[:, 8:, :300], atol=2e-5, rtol=1e-5)
    a = generate(m, seq[:, :5], 70, temperature=0.0, cache_bits=bits)  # past block_size
    b = generate(m, seq[:, :5], 70, temperature=0.0, use_cache=False, pad_to=1)
    assert torch.equal(a, b)


def test_decoder_in_4_bits_and_device_sampling():
    m = GPT(GPTConfig(**CFG, attention_window=16, attention_sinks=1), SINGLE, seed=7).eval()
    seq = torch.randint(0, 300, (2, 30), generator=_gen(2))
    exact, coarse = KVCache(m, 2), KVCache(m, 2, 4)
    with torch.no_grad():
        for t0, t1 in [(0, 20)] + [(t, t + 1) for t in range(20, 30)]:
            a, b = exact.forward(seq[:, t0:t1]), coarse.forward(seq[:, t0:t1])
    assert (a - b).norm() < 0.1 * a.norm() and not torch.equal(a, b)
    kw = dict(temperature=0.8, top_k=20, top_p=0.9, min_p=0.05, cache_bits=4)
    s1, s2 = (generate(m, seq, 10, generator=_gen(5), **kw) for _ in range(2))
    assert torch.equal(s1, s2) and s1.shape == (2, 40)
    greedy = generate(m, seq, 10, temperature=0.0, device_sampling=True)
    assert torch.equal(greedy, generate(m, seq, 10, temperature=0.0))


def test_gumbel_noise_is_standard():
    g = gumbel_noise(200, 1000, generator=_gen(6)).double()
    # mean 0.5772, standard deviation pi / sqrt(6); 5 standard errors of 200000 numbers
    assert abs(g.mean() - 0.57722) < 5 * 1.2825 / math.sqrt(2e5)
    assert abs(g.std() - 1.2825) < 0.02


@pytest.mark.parametrize("use_cache", [True, False])
@pytest.mark.parametrize("tokens", [1, 4])
@pytest.mark.parametrize("kw", [dict(device_sampling=True), dict(min_p=0.1), dict(device_sampling=True, temperature=0.0)])
def test_logits_without_a_token_raise(kw, tokens, use_cache):
    """A model that returns NaN: a clear error, no token of -1 fed back or returned."""
    m = GPT(GPTConfig(**CFG, attention_window=16), SINGLE, seed=7).eval()
    seq = torch.randint(0, 300, (2, 30), generator=_gen(2))
    with torch.no_grad():
        m.lm_head.weight.fill_(float("nan"))
    with pytest.raises(RuntimeError, match="no token to draw"):
        generate(m, seq, tokens, use_cache=use_cache, **kw)


def test_nothing_to_generate():
    m = GPT(GPTConfig(**CFG), SINGLE, seed=7).eval()
    seq = torch.randint(0, 300, (2, 30), generator=_gen(2))
    assert torch.equal(generate(m, seq, 0, device_sampling=True), seq)


@pytest.mark.parametrize("temperature", [float("inf"), 3.4e38])
def test_sampling_at_temperatures_without_bound(temperature):
    """Every finite logit weighs the same, a masked one nothing; below the smallest normal number it is greedy."""
    inf = float("inf")
    x = torch.tensor([[0.5, -1.0, 2.0, -inf, 0.0], [-inf, 3.0, -inf, -inf, 1.0]])
    g = torch.tensor([[0.1, 0.9, 0.3, 5.0, 0.2], [5.0, 0.1, 5.0, 5.0, 0.2]])
    token, logprob = sample_tokens(x, g, temperature)
    assert token.tolist() == [1, 4]
    torch.testing.assert_close(logprob, -torch.tensor([4.0, 2.0]).log())
    assert sample_tokens(x, g, temperature, top_k=1)[0].tolist() == [0, 1]  # all equal: the lowest index
    assert sample_tokens(x, g, 1e-40)[0].tolist() == [2, 1]
