"""Sliding-window attention kernels against the definition in 64 bits.

Tolerances are norms of the error over norms of the result. One rounding to bf16
is at most u = 2^-9 relative. Output: P and the result are rounded (2 u). dV: the
same. dQ and dK: P or dS, the result, and the output that enters rowsum(dO * O)
(3 u, and 1 u for that sum's weight in dS).
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-9


@pytest.fixture(autouse=True)
def _status(cuda):
    from dstraining_b200.ops import native

    native.lib().read_status(True)
    yield
    assert native.lib().read_status(True) == 0


def _rand(*shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(torch.bfloat16)


def _err(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


def _exact(q, k, v, window, sinks, dout=None):
    from dstraining_b200.ops.window import core_window_attention

    x = [t.detach().double().requires_grad_() for t in (q, k, v)]
    out = core_window_attention(*x, window, sinks)
    return (out.detach(), *(torch.autograd.grad(out, x, dout.double()) if dout is not None else ()))


CASES = [
    # B, T, H, Hk, D, window, sinks
    (1, 2, 1, 1, 64, 2, 0),
    (2, 63, 3, 3, 64, 7, 1),
    (1, 64, 2, 2, 64, 64, 0),
    (2, 65, 2, 2, 128, 64, 0),
    (1, 128, 2, 1, 64, 1, 3),
    (2, 129, 4, 2, 128, 128, 4),
    (1, 257, 2, 2, 64, 1000, 0),  # a window longer than the sequence: causal
    (1, 333, 12, 12, 64, 128, 4),
    (2, 400, 6, 3, 40, 33, 70),  # sinks that end inside the second key block
    (1, 500, 8, 1, 8, 100, 128),
    (1, 513, 2, 2, 96, 130, 500),  # sinks past most windows
    (1, 700, 4, 2, 128, 65, 64),
    (1, 1025, 2, 2, 64, 256, 2000),  # every key a sink
    (1, 2300, 2, 1, 64, 511, 5),
]


@pytest.mark.parametrize("B,T,H,Hk,D,W,S", CASES)
def test_forward_and_gradients(B, T, H, Hk, D, W, S):
    from dstraining_b200.ops.window import window_attention_qkv

    q, k, v = _rand(B, T, H, D, seed=1), _rand(B, T, Hk, D, seed=2), _rand(B, T, Hk, D, seed=3)
    dout = _rand(B, T, H, D, seed=4)
    x = [t.requires_grad_() for t in (q, k, v)]
    out = window_attention_qkv(*x, W, S)
    got = (out.detach(), *torch.autograd.grad(out, x, dout))
    want = _exact(q, k, v, W, S, dout)
    for name, a, b, tol in zip(("out", "dq", "dk", "dv"), got, want, (2 * U, 4 * U, 4 * U, 2 * U)):
        assert a.shape == b.shape and a.dtype == torch.bfloat16
        assert _err(a, b) < tol, name


@pytest.mark.parametrize("T,W,S", [(1, 1, 0), (1, 5, 3), (300, 1, 0)])
def test_rows_that_see_themselves_only(T, W, S):
    """The output is V exactly and the scores have no gradient."""
    from dstraining_b200.ops.window import window_attention_qkv

    x = [_rand(1, T, 2, 64, seed=i).requires_grad_() for i in range(3)]
    dout = _rand(1, T, 2, 64, seed=5)
    out = window_attention_qkv(*x, W, S)
    dq, dk, dv = torch.autograd.grad(out, x, dout)
    assert torch.equal(out, x[2])
    assert torch.equal(dv, dout)
    # dP and rowsum(dO O) are the same 64-term sum, each off by at most 64 * 2^-23 of the terms' norm
    bound = 64 * 2.0**-22 * (dout.float().norm(dim=-1) * x[2].float().norm(dim=-1)).max() * 8
    assert dq.abs().max() <= bound and dk.abs().max() <= bound


@pytest.mark.parametrize("T,D,W,S", [(200, 64, 50, 4), (128, 128, 128, 0), (77, 24, 30, 2)])
def test_fused_buffer_equals_separate_operands(T, D, W, S):
    from dstraining_b200.ops.window import window_attention, window_attention_qkv

    H = 4
    qkv = _rand(2, T, 3 * H * D, seed=7).requires_grad_()
    dout = _rand(2, T, H * D, seed=8)
    out = window_attention(qkv, H, D, W, S)
    (dqkv,) = torch.autograd.grad(out, qkv, dout)
    x = [t.clone().requires_grad_() for t in qkv.detach().view(2, T, H, 3, D).unbind(dim=3)]
    out2 = window_attention_qkv(*x, W, S)
    grads = torch.autograd.grad(out2, x, dout.view(2, T, H, D))
    assert torch.equal(out.view_as(out2), out2)
    assert torch.equal(dqkv.view(2, T, H, 3, D), torch.stack(grads, dim=3))


def test_full_window_equals_causal_attention():
    """With every key in the window this is the framework's causal attention (both round P: 4 u)."""
    from dstraining_b200.ops.flash import flash_attention
    from dstraining_b200.ops.window import window_attention

    qkv = _rand(2, 384, 3 * 4 * 64, seed=9)
    a, b = window_attention(qkv, 4, 64, 384), flash_attention(qkv, 4, 64)
    assert _err(a, b.double()) < 4 * U


@pytest.mark.parametrize("layout", ["heads_first", "sliced", "misaligned", "expanded"])
def test_operand_layouts(layout):
    from dstraining_b200.ops.window import window_attention_qkv

    B, T, H, D, W, S = 2, 150, 4, 64, 40, 3
    def make(seed):
        if layout == "heads_first":
            return _rand(B, H, T, D, seed=seed).transpose(1, 2)
        if layout == "sliced":
            return _rand(B, T, H + 1, D + 8, seed=seed)[:, :, 1:, 8:]
        if layout == "misaligned":
            return _rand(B, T, H, D + 1, seed=seed)[..., 1:]
        return _rand(1, T, 1, D, seed=seed).expand(B, T, H, D)

    x = [make(i) for i in range(3)]
    dense = [t.clone(memory_format=torch.contiguous_format).requires_grad_() for t in x]
    dout = _rand(B, H, T, D, seed=11).transpose(1, 2)  # not contiguous either
    x = [t.detach().requires_grad_() for t in x]
    a, b = window_attention_qkv(*x, W, S), window_attention_qkv(*dense, W, S)
    assert torch.equal(a, b)
    for g, w in zip(torch.autograd.grad(a, x, dout), torch.autograd.grad(b, dense, dout)):
        assert torch.equal(g, w)


def test_neighbours_never_leak():
    """Infinities in the next sequence and past the window's key blocks leave a sequence untouched."""
    from dstraining_b200.ops.window import window_attention_qkv

    T, W = 700, 64
    x = [_rand(2, T, 2, 64, seed=i) for i in range(3)]
    clean = window_attention_qkv(*x, W, 0)
    for t in x:
        t[1] = float("inf")
        t[0, :64] = float("nan")  # a whole key block that queries from 128 on cannot see
    dirty = window_attention_qkv(*x, W, 0)
    assert torch.equal(clean[0, 128:], dirty[0, 128:])


def test_masked_scores_may_be_anything():
    """Huge keys outside the mask change neither output nor gradients of q."""
    from dstraining_b200.ops.window import window_attention_qkv

    T = 128
    q, k, v = (_rand(1, T, 1, 64, seed=i) for i in range(3))
    k2 = k.clone()
    k2[:, 100:] = 3e38  # finite, but their scores overflow
    dout = _rand(1, T, 1, 64, seed=5)
    dout[:, 100:] = 0
    outs = []
    for keys in (k, k2):
        x = q.clone().requires_grad_()
        out = window_attention_qkv(x, keys, v, 20, 2)
        (g,) = torch.autograd.grad(out[:, :100], x, dout[:, :100])
        outs.append((out[:, :100].detach(), g[:, :100]))
    assert torch.equal(outs[0][0], outs[1][0])
    assert torch.equal(outs[0][1], outs[1][1])


def test_gradient_against_differences():
    """<grad, h> against central differences of the 64-bit definition along random h."""
    from dstraining_b200.ops.window import core_window_attention, window_attention_qkv

    W, S = 37, 5
    x = [_rand(1, 190, h, 64, seed=i).requires_grad_() for i, h in enumerate((4, 2, 2))]
    dout = _rand(1, 190, 4, 64, seed=9)
    grads = torch.autograd.grad(window_attention_qkv(*x, W, S), x, dout)
    eps = 1e-4  # third-order term ~ eps^2, rounding ~ 1e-16 / eps
    for i, g in enumerate(grads):
        h = g.double() + g.double().norm() / g.numel() ** 0.5 * _rand(*g.shape, seed=20 + i).double()
        h = h / h.norm()
        def f(t):
            y = [p.detach().double() for p in x]
            y[i] = y[i] + t * h
            return (core_window_attention(*y, W, S) * dout.double()).sum()
        slope = (f(eps) - f(-eps)) / (2 * eps)
        assert abs((g.double() * h).sum() - slope) < 4 * U * slope.abs()


def test_repeatable_and_on_another_stream():
    from dstraining_b200.ops.window import window_attention

    qkv = _rand(2, 500, 3 * 4 * 64, seed=3).requires_grad_()
    dout = _rand(2, 500, 4 * 64, seed=4)
    def once():
        out = window_attention(qkv, 4, 64, 100, 4)
        return out.detach(), torch.autograd.grad(out, qkv, dout)[0]
    a = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = once()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("D", [64, 128])
def test_long_sequences_repeat_exactly(D):
    """Enough tiles and blocks that waves of CTAs overlap in many ways: the same bits every time, and right."""
    from dstraining_b200.ops.window import window_attention_qkv

    W, S = 700, 5
    q, k, v = _rand(1, 4001, 16, D, seed=1), _rand(1, 4001, 4, D, seed=2), _rand(1, 4001, 4, D, seed=3)
    dout = _rand(1, 4001, 16, D, seed=4)
    x = [t.requires_grad_() for t in (q, k, v)]

    def once():
        out = window_attention_qkv(*x, W, S)
        return (out.detach(), *torch.autograd.grad(out, x, dout))

    runs = [once() for _ in range(8)]
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))
    for h in (0, 7):  # two query heads, and the key head of each
        one = [t.detach()[:, :, i:i + 1] for t, i in ((q, h), (k, h // 4), (v, h // 4))]
        want = _exact(*one, W, S)[0]
        assert _err(runs[0][0][:, :, h:h + 1], want) < 2 * U


def test_graph_capture():
    from dstraining_b200.ops.window import window_attention

    qkv = _rand(1, 300, 3 * 2 * 64, seed=3)
    window_attention(qkv, 2, 64, 50, 4)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = window_attention(qkv, 2, 64, 50, 4)
    qkv.copy_(_rand(1, 300, 3 * 2 * 64, seed=5))
    g.replay()
    assert torch.equal(out, window_attention(qkv, 2, 64, 50, 4))


@pytest.mark.parametrize("shape", [(0, 5, 2, 64), (2, 0, 2, 64)])
def test_nothing_to_do(shape):
    from dstraining_b200.ops.window import window_attention_qkv

    x = [torch.zeros(shape, device="cuda", dtype=torch.bfloat16).requires_grad_() for _ in range(3)]
    out = window_attention_qkv(*x, 4, 1)
    assert out.shape == shape
    out.sum().backward()
    assert x[0].grad.shape == shape


def test_model_trains_and_decodes():
    """A GPT with a window: loss as in fp32 on the CPU (both layers round activations, loss ~ 5.6: a few u
    relative), decoding over the rolling cache as the full forward pass (activations rounded at other
    places: 16 u of the logits' norm; 4-bit rows: a step is 1/15 of a group's range)."""
    from dstraining_b200.models.gpt import GPT, GPTConfig
    from dstraining_b200.parallel.topology import SINGLE
    from dstraining_b200.utils.generate import KVCache, generate

    cfg = GPTConfig(vocab_size=257, block_size=256, n_layer=2, n_head=2, n_embd=128, attention_window=40,
                    attention_sinks=2)
    idx = torch.randint(0, 257, (2, 200), generator=torch.Generator().manual_seed(1))
    model, oracle = GPT(cfg, SINGLE, seed=3).cuda().to(torch.bfloat16), GPT(cfg, SINGLE, seed=3)
    _, loss = model(idx.cuda(), idx.cuda())
    _, want = oracle(idx, idx)
    loss.backward()
    want.backward()
    assert abs(loss.item() - want.item()) < 8 * U * want.item()
    for (name, a), b in zip(model.named_parameters(), oracle.parameters()):
        if b.grad.norm() > 1e-3:
            assert _err(a.grad.cpu(), b.grad.double()) < 32 * U, name
    model.eval()
    seq = idx.cuda()
    with torch.no_grad():
        full = model(seq)[0][:, 100:, :257].double()
        for bits, tol in ((16, 16 * U), (4, 0.2)):
            cache = KVCache(model, 2, bits)
            got = [cache.forward(seq[:, :101])] + [cache.forward(seq[:, t:t + 1]) for t in range(101, 200)]
            assert _err(torch.stack(got, dim=1), full) < tol
    g = lambda: torch.Generator(device="cuda").manual_seed(4)  # noqa: E731
    a, b = (generate(model, seq[:, :50], 30, 0.8, 20, g(), top_p=0.9, min_p=0.01, cache_bits=4, device_sampling=True)
            for _ in range(2))
    assert a.shape == (2, 80) and torch.equal(a, b)


def test_refusals():
    from dstraining_b200.ops import native
    from dstraining_b200.ops.window import window_attention, window_attention_qkv

    x = [_rand(1, 8, 2, 64, seed=i) for i in range(3)]
    with pytest.raises(ValueError, match="window"):
        window_attention_qkv(*x, 0)
    with pytest.raises(ValueError, match="sinks"):
        window_attention_qkv(*x, 4, -1)
    with pytest.raises(ValueError, match="share"):
        window_attention_qkv(_rand(1, 8, 3, 64, seed=0), x[1], x[2], 4)
    with pytest.raises(ValueError, match="required"):
        window_attention_qkv(x[0], x[1], x[2][:, :7], 4)
    with pytest.raises(ValueError, match="qkv"):
        window_attention(_rand(1, 8, 100, seed=0), 2, 64, 4)
    for d in (12, 136):
        with pytest.raises(RuntimeError, match="head_dim"):
            window_attention_qkv(*[_rand(1, 8, 2, d, seed=i) for i in range(3)], 4)
    lib = native.lib()
    with pytest.raises(RuntimeError, match="must be a CUDA bf16"):
        lib.window_attention_qkv(x[0].float(), x[1], x[2], 4, 0)
    with pytest.raises(RuntimeError, match="agree"):
        lib.window_attention_qkv(x[0], x[1][:, :7], x[2][:, :7], 4, 0)
    with pytest.raises(RuntimeError, match="window >= 1"):
        lib.window_attention(_rand(1, 8, 3 * 128, seed=0), 2, 64, 0, 0)


@pytest.mark.parametrize("T,S", [(4096, 4096), (8192, 8192), (8192, 1500)])
def test_workspace_stays_linear(T, S):
    """Many sinks: beside its results the backward pass holds no more than twice dK and dV in fp32 (and the row sums)."""
    from dstraining_b200.ops.window import window_attention_qkv

    H, D, W = 2, 128, 100
    x = [_rand(1, T, H, D, seed=i).requires_grad_() for i in range(3)]
    dout = _rand(1, T, H, D, seed=5)
    out = window_attention_qkv(*x, W, S)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    grads = torch.autograd.grad(out, x, dout)
    torch.cuda.synchronize()
    elements = T * H * D
    assert torch.cuda.max_memory_allocated() - before <= 3 * 2 * elements + 2 * 2 * 4 * elements + 4 * T * H + 2**16
    del grads


SINK_CHUNKS = [
    # B, T, H, Hk, D, window, sinks: three or more chunks of far queries a sink block
    (1, 3000, 2, 1, 128, 64, 5),
    (1, 2500, 4, 2, 128, 100, 1),
    (2, 2049, 2, 2, 128, 30, 130),
    (1, 2700, 3, 1, 64, 64, 260),
    (1, 4001, 2, 2, 96, 700, 3),
    (1, 2200, 2, 1, 128, 40, 1100),
    (1, 1500, 2, 1, 64, 20, 1500),
]


@pytest.mark.parametrize("B,T,H,Hk,D,W,S", SINK_CHUNKS)
def test_gradients_of_sinks_over_many_chunks(B, T, H, Hk, D, W, S):
    from dstraining_b200.ops.window import window_attention_qkv

    q, k, v = _rand(B, T, H, D, seed=1), _rand(B, T, Hk, D, seed=2), _rand(B, T, Hk, D, seed=3)
    dout = _rand(B, T, H, D, seed=4)
    x = [t.requires_grad_() for t in (q, k, v)]
    out = window_attention_qkv(*x, W, S)
    got = (out.detach(), *torch.autograd.grad(out, x, dout))
    want = _exact(q, k, v, W, S, dout)
    for name, a, b, tol in zip(("out", "dq", "dk", "dv"), got, want, (2 * U, 4 * U, 4 * U, 2 * U)):
        assert _err(a, b) < tol, name
    for name, a, b, tol in (("dk", got[2], want[2], 4 * U), ("dv", got[3], want[3], 2 * U)):  # of the sinks alone
        assert _err(a[:, :S], b[:, :S]) < tol, name


@pytest.mark.parametrize("fused", [True, False])
def test_a_second_derivative_is_refused(fused):
    """The gradients have no derivative of their own: asking for one is an error, not a silent zero."""
    from dstraining_b200.ops.window import window_attention, window_attention_qkv

    if fused:
        x = [_rand(1, 20, 3 * 2 * 64, seed=1).requires_grad_()]
        out = window_attention(x[0], 2, 64, 5, 1)
    else:
        x = [_rand(1, 20, 2, 64, seed=i).requires_grad_() for i in range(3)]
        out = window_attention_qkv(*x, 5, 1)
    once = torch.autograd.grad(out.sum(), x, retain_graph=True)
    grads = torch.autograd.grad(out.sum(), x, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(once, grads))
    penalty = sum((g.float() ** 2).sum() for g in grads)
    with pytest.raises(RuntimeError, match="second derivative"):
        (out.float().sum() + penalty).backward()


def test_training_pass_in_a_graph():
    """Forward and backward captured together: replays on new inputs give what the calls give."""
    from dstraining_b200.ops.window import window_attention

    qkv, dout = _rand(1, 700, 3 * 2 * 64, seed=3).requires_grad_(), _rand(1, 700, 2 * 64, seed=4)

    def once():
        out = window_attention(qkv, 2, 64, 50, 4)
        return out.detach(), torch.autograd.grad(out, qkv, dout)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            captured = once()
    torch.cuda.current_stream().wait_stream(side)
    with torch.no_grad():
        qkv.copy_(_rand(1, 700, 3 * 2 * 64, seed=5))
        dout.copy_(_rand(1, 700, 2 * 64, seed=6))
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(captured, once()))
