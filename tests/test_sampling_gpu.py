"""The sampling kernel against the definition in 64 bits. Tokens have to be equal
(the noise is random, so no two scores are within rounding of one another);
log-probabilities are fp32 sums: 1e-5 absolute for values up to some tens."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status(cuda):
    from dstraining_b200.ops import native

    native.lib().read_status(True)
    yield
    assert native.lib().read_status(True) == 0


def exact(logits, gumbel, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row, on the CPU, by sorting."""
    if temperature > 0:  # t is an fp32 number of the definition
        t = (logits.float() / torch.full_like(logits, temperature, dtype=torch.float32)).double()
    else:
        t = logits.double()
    t = torch.where(t.isnan(), torch.full_like(t, -math.inf), t)
    if t.max() == -math.inf:
        return -1, -math.inf
    gap = torch.where(t == t.max(), torch.zeros_like(t), t - t.max())
    order = torch.argsort(t, descending=True, stable=True)
    n = len(order) if temperature > 0 else 1
    if top_k > 0:
        n = min(n, top_k)
    kept = order[:n]
    if top_p < 1 and temperature > 0:
        mass = gap[kept].exp()
        before = mass.cumsum(0) - mass
        kept = kept[: max(1, int((before < top_p * mass.sum()).sum()))]
    kept = kept[: max(1, int((gap[kept].exp() >= min_p).sum()))]
    score = (t[kept].float() + gumbel[kept]).double()
    score = torch.where(score.isnan(), torch.full_like(score, -math.inf), score)
    best = kept[score == score.max()].min().item()
    return best, (gap[best] - gap.exp().sum().log()).item()


def check(logits, gumbel, **settings):
    from dstraining_b200.ops.sampling import sample_tokens

    token, logprob = sample_tokens(logits, gumbel, **settings)
    x, g = logits.cpu(), gumbel.cpu()
    for b in range(len(x)):
        one = {n: (v[b].item() if isinstance(v, torch.Tensor) else v) for n, v in settings.items()}
        t, l = exact(x[b], g[b], **one)
        assert token[b].item() == t, (b, one)
        assert logprob[b].item() == l or abs(logprob[b].item() - l) < 1e-5, (b, one)


def _logits(B, V, dtype, seed, scale=2.5, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(B, V + pad, device="cuda", generator=g) * scale).to(dtype)[:, :V]


def _noise(B, V, seed):
    from dstraining_b200.ops.sampling import gumbel_noise

    return gumbel_noise(B, V, "cuda", torch.Generator(device="cuda").manual_seed(seed))


SETTINGS = [
    dict(),
    dict(temperature=0.0),
    dict(temperature=0.7, top_k=40),
    dict(top_k=1),
    dict(top_k=1024, top_p=0.9),
    dict(top_k=1500, top_p=0.3),
    dict(top_p=0.9),
    dict(top_p=0.05, temperature=1.7),
    dict(top_p=0.0),
    dict(min_p=0.1),
    dict(min_p=1.5),
    dict(temperature=0.8, top_k=50, top_p=0.95, min_p=0.02),
    dict(top_k=10**9, top_p=0.999),
]


@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: "-".join(f"{k}{v}" for k, v in s.items()) or "plain")
@pytest.mark.parametrize("B,V,dtype,pad", [(6, 50257, torch.bfloat16, 47), (3, 50257, torch.float32, 47),
                                           (4, 1, torch.float32, 0), (5, 17, torch.bfloat16, 2),
                                           (4, 1025, torch.float32, 3), (2, 70001, torch.bfloat16, 0)])
def test_settings_and_sizes(settings, B, V, dtype, pad):
    check(_logits(B, V, dtype, 1, pad=pad), _noise(B, V, 2), **settings)


def test_settings_per_row():
    B, V = 40, 3001
    g = torch.Generator(device="cuda").manual_seed(5)
    pick = lambda v: torch.tensor(v, device="cuda")[torch.randint(len(v), (B,), device="cuda", generator=g)]  # noqa: E731
    check(_logits(B, V, torch.float32, 3), _noise(B, V, 4), temperature=pick([0.0, 0.5, 1.0, 2.0]),
          top_k=pick([0, 1, 30, 2000]), top_p=pick([1.0, 0.9, 0.2]), min_p=pick([0.0, 0.05]))


@pytest.mark.parametrize("settings", [dict(top_k=7), dict(top_k=1100), dict(top_p=0.4), dict(top_k=900, top_p=0.5), dict(temperature=0.0)])
@pytest.mark.parametrize("values", [1, 3, 20])
def test_ties(settings, values):
    """Few distinct logits: the cuts fall among equal ones, lowest index first."""
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randint(values, (5, 5003), device="cuda", generator=g).float()
    check(x, _noise(5, 5003, 8), **settings)
    check(-x, _noise(5, 5003, 9), **settings)  # -0 and +0 are one value


@pytest.mark.parametrize("settings", [dict(), dict(top_k=5), dict(top_k=2000, top_p=0.9), dict(top_p=0.5), dict(min_p=0.2), dict(temperature=0.0)])
def test_masked_and_broken_logits(settings):
    V = 3000
    x = _logits(8, V, torch.float32, 11)
    x[0] = -math.inf
    x[1, 5:] = -math.inf
    x[2, ::2] = math.nan
    x[3] = math.nan
    x[4, [7, 90, 2000]] = math.inf
    x[5] = torch.finfo(torch.float32).min
    x[6, 3:] = torch.finfo(torch.float32).min
    x[7, 0] = 3e38
    check(x, _noise(8, V, 12), **settings)


def test_noise_may_be_infinite():
    x, g = _logits(4, 500, torch.float32, 13), _noise(4, 500, 14)
    g[0, 100] = math.inf
    g[1] = -math.inf
    g[2, ::3] = math.nan
    g[3] = 0.0  # no noise: the most probable token
    check(x, g, top_p=0.9)
    check(x, g, top_k=20)


def test_noise_that_always_asks_for_the_least_probable():
    """Every winner is refused until the first tokens are reached: still right, and in bounded time."""
    x = _logits(2, 20000, torch.float32, 15)
    check(x, -50 * x, top_p=0.3)
    flat = torch.zeros(2, 20000, device="cuda")
    check(flat, torch.arange(20000, device="cuda").float().expand(2, -1).contiguous(), top_p=0.01)


def test_draws_follow_the_distribution():
    """Frequencies over 20000 rows within 5 standard deviations of the kept softmax."""
    from dstraining_b200.ops.sampling import sample_tokens

    n = 20000
    x = torch.tensor([2.0, 1.0, 0.5, 0.0, -1.0, -5.0], device="cuda").expand(n, -1)
    token, _ = sample_tokens(x, _noise(n, 6, 16), top_k=4)
    want = torch.softmax(x[0, :4].double(), dim=0)
    got = torch.bincount(token, minlength=6)
    assert got[4:].sum() == 0
    for c, p in zip(got[:4].tolist(), want.tolist()):
        assert abs(c - n * p) < 5 * math.sqrt(n * p * (1 - p))


def test_repeatable_captured_and_on_another_stream():
    from dstraining_b200.ops.sampling import sample_tokens

    x, g = _logits(9, 50257, torch.bfloat16, 17), _noise(9, 50257, 18)
    a = sample_tokens(x, g, 0.9, 1000, 0.7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            b = sample_tokens(x, g, 0.9, 1000, 0.7)
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_strided_and_empty():
    from dstraining_b200.ops.sampling import sample_tokens

    x, g = _logits(3, 200, torch.float32, 19), _noise(3, 200, 20)
    a = sample_tokens(x.t().contiguous().t(), g.t().contiguous().t(), top_k=9)
    b = sample_tokens(x, g, top_k=9)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert sample_tokens(x[:0], g[:0])[0].shape == (0,)


def test_refusals():
    from dstraining_b200.ops.sampling import sample_tokens

    x, g = _logits(3, 20, torch.float32, 21), _noise(3, 20, 22)
    for bad in (g[:2], g.double(), g[:, :10]):
        with pytest.raises(ValueError, match="gumbel"):
            sample_tokens(x, bad)
    with pytest.raises(ValueError, match="gumbel on"):
        sample_tokens(x, g.cpu())
    with pytest.raises(ValueError, match="temperature"):
        sample_tokens(x, g, temperature=-1.0)
    with pytest.raises(ValueError, match="min_p"):
        sample_tokens(x, g, min_p=float("nan"))
    with pytest.raises(ValueError, match="top_k"):
        sample_tokens(x, g, top_k=torch.tensor([1, 2], device="cuda"))
    with pytest.raises(RuntimeError, match="per row"):
        sample_tokens(x, g, top_p=torch.tensor([0.5, 0.5, 0.5]))


@pytest.mark.parametrize("settings", [dict(), dict(top_p=0.4), dict(top_k=40), dict(top_k=600), dict(top_k=1500),
                                      dict(top_k=1500, top_p=0.5), dict(min_p=0.5)])
@pytest.mark.parametrize("temperature", [1e38, math.inf])
def test_temperatures_without_bound(temperature, settings):
    """Every t is 0 (below the smallest normal number): the tokens weigh the same, the lowest index first, and
    masked ones still never are."""
    from dstraining_b200.ops.sampling import sample_tokens

    V = 3001
    x = _logits(4, V, torch.float32, 33).clamp(-1, 1)
    x[1] = 0.75
    x[2, :10] = 0.0
    x[3, ::2] = -math.inf  # fewer tokens than top_k asks for
    g = _noise(4, V, 34)
    zeros = torch.where(x > -math.inf, torch.zeros_like(x), x)
    token, logprob = sample_tokens(x, g, temperature, **settings)
    for b in range(4):
        t, l = exact(zeros[b].cpu(), g[b].cpu(), **settings)
        assert token[b].item() == t and abs(logprob[b].item() - l) < 1e-5, b


@pytest.mark.parametrize("settings", [dict(), dict(top_k=7), dict(top_k=1500), dict(top_p=0.4), dict(top_p=0.9, top_k=400),
                                      dict(min_p=0.5)])
def test_quotients_that_overflow(settings):
    """t = x / temperature may be infinite where x is not: those tokens are equal, the lowest index first."""
    V = 3000
    x = _logits(5, V, torch.float32, 31)
    x[1] = x[1].abs() + 1
    x[2] = -x[2].abs() - 100  # every t is -inf: nothing to draw
    x[3, [70, 90, 2000]] = torch.tensor([3.0, 200.0, 100.0], device="cuda") * 1e36
    x[4, 11] = math.inf
    x[4, 5] = 1e36
    check(x, _noise(5, V, 32), temperature=2.0**-125, **settings)


@pytest.mark.parametrize("name", ["temperature", "top_p", "min_p"])
@pytest.mark.parametrize("more", [dict(), dict(top_k=30), dict(top_k=1500)])
def test_a_setting_that_is_nan_keeps_the_first_token(name, more):
    """As in the PyTorch form: no comparison with NaN holds."""
    from dstraining_b200.ops.sampling import sample_tokens

    x, g = _logits(3, 2000, torch.float32, 35), _noise(3, 2000, 36)
    rows = torch.tensor([math.nan, 0.5, math.nan], device="cuda")
    token, logprob = sample_tokens(x, g, **{name: rows}, **more)
    want, want_logprob = sample_tokens(x.cpu(), g.cpu(), **{name: rows.cpu()}, **more)
    assert torch.equal(token.cpu(), want) and token[0] == x[0].argmax() and token[2] == x[2].argmax()
    torch.testing.assert_close(logprob.cpu(), want_logprob, atol=1e-5, rtol=0)
