"""The rolling key/value cache on the GPU against its definition in 64 bits.

The stored rows have to be what the definition says bit by bit. The attention
over them is computed with fp32 scores and sums and probabilities good to 2^-17,
so its result is off by its own rounding to bf16, at most u = 2^-9 of each
element, and by far less from the rest: norm of the error under 1.1 u."""

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


def _stands_for(x, bits):
    """The definition, in 64 bits where it leaves the choice."""
    if bits == 16:
        return x
    g = x.float().unflatten(-1, (-1, 32))
    low = g.min(dim=-1, keepdim=True).values
    step = ((g.max(dim=-1, keepdim=True).values - low) / g.new_full(low.shape, 15.0)).bfloat16().float()
    code = torch.where(step > 0, torch.round((g - low) / step), torch.zeros_like(g)).clamp(0, 15)
    return (low.double() + code.double() * step.double()).flatten(-2).float()


class Oracle:
    """Token lists: what each slot holds, and attention over them in 64 bits."""

    def __init__(self, batch, window, sinks, bits):
        self.rows = [{} for _ in range(batch)]
        self.W, self.S, self.bits = window, sinks, bits

    def put(self, b, p, k, v):
        slot = p if p < self.S else self.S + (p - self.S) % self.W
        self.rows[b][slot] = (_stands_for(k, self.bits), _stands_for(v, self.bits))

    def fill(self, k, v, lengths):
        for b, n in enumerate(lengths):
            self.rows[b] = {}
            for p in sorted({*range(min(self.S, n)), *range(max(0, n - self.W), n)}):
                self.put(b, p, k[b, p], v[b, p])

    def held(self, heads, dim, slots, dtype):
        out = [torch.zeros(len(self.rows), heads, slots, dim, device="cuda", dtype=dtype) for _ in range(2)]
        for b, rows in enumerate(self.rows):
            for s, kv in rows.items():
                for o, x in zip(out, kv):
                    o[b, :, s] = x
        return out

    def attend(self, b, q):
        k, v = (torch.stack([kv[i] for kv in self.rows[b].values()], dim=1).double() for i in range(2))
        g = q.shape[0] // k.shape[0]
        k, v = k.repeat_interleave(g, dim=0), v.repeat_interleave(g, dim=0)
        p = torch.softmax((k @ q.double()[:, :, None])[..., 0] * q.shape[-1] ** -0.5, dim=-1)
        return (p[:, None] @ v)[:, 0]


CASES = [
    # B, H, Hk, D, window, sinks, T, bits
    (2, 4, 4, 64, 50, 3, 40, 16),
    (2, 4, 4, 64, 50, 3, 40, 4),
    (3, 8, 2, 128, 100, 0, 333, 16),
    (3, 8, 2, 128, 100, 5, 333, 4),
    (2, 3, 3, 40, 9, 2, 30, 16),
    (2, 3, 3, 96, 63, 2, 30, 4),
    (1, 2, 2, 32, 1, 0, 5, 4),
    (1, 2, 1, 8, 1, 1, 5, 16),
    (1, 20, 2, 64, 64, 64, 200, 4),  # ten query heads a key head: two CTAs
    (1, 18, 1, 128, 129, 1, 200, 16),
    (1, 2, 2, 64, 700, 4, 690, 16),  # split over CTAs, and joined
    (1, 2, 2, 128, 700, 4, 690, 4),
    (1, 4, 2, 64, 5000, 4, 4990, 4),  # over more splits than are joined at once
    (1, 8, 1, 128, 5000, 4, 4990, 4),
    (1, 8, 1, 64, 5000, 1, 4000, 16),
]


@pytest.mark.parametrize("B,H,Hk,D,W,S,T,bits", CASES)
def test_fill_and_steps(B, H, Hk, D, W, S, T, bits):
    from dstraining_b200.ops.kv_cache import WindowCache

    cache, oracle = WindowCache(B, Hk, D, W, S, bits=bits, device="cuda"), Oracle(B, W, S, bits)
    k, v = _rand(B, T, Hk, D, seed=1), _rand(B, T, Hk, D, seed=2)
    lengths = [T - i * T // B for i in range(B)]
    cache.fill(k, v, torch.tensor(lengths, device="cuda"))
    oracle.fill(k, v, lengths)
    assert cache.pos.tolist() == lengths
    dtype = torch.bfloat16 if bits == 16 else torch.float32
    for a, b in zip(cache.read(), oracle.held(Hk, D, W + S, dtype)):
        assert a.dtype == dtype and torch.equal(a, b)
    for step in range(3):
        q, k1, v1 = _rand(B, H, D, seed=10 + step), _rand(B, Hk, D, seed=20 + step), _rand(B, Hk, D, seed=30 + step)
        out, ks, vs = cache.step(q, k1, v1, return_stored=True)
        for b in range(B):
            oracle.put(b, lengths[b] + step, k1[b], v1[b])
            want = oracle.attend(b, q[b])
            assert ((out[b].double() - want).norm() / want.norm()).item() < 1.1 * U
        assert torch.equal(ks, _stands_for(k1, bits).float()) and torch.equal(vs, _stands_for(v1, bits).float())
        for a, b in zip(cache.read(), oracle.held(Hk, D, W + S, dtype)):
            assert torch.equal(a, b)
    assert cache.pos.tolist() == [n + 3 for n in lengths]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("D", [64, 128])
def test_from_an_empty_cache(bits, D):
    """Lengths of zero: the first token sees itself alone and comes back as it is stored."""
    from dstraining_b200.ops.kv_cache import WindowCache

    cache = WindowCache(2, 2, D, 5, 1, bits=bits, device="cuda")
    q, k, v = (_rand(2, 2, D, seed=i) for i in range(3))
    out = cache.step(q, k, v)
    assert torch.equal(out, _stands_for(v, bits).to(torch.bfloat16))
    cache.fill(k[:, None][:, :0], v[:, None][:, :0])
    assert cache.pos.tolist() == [0, 0]
    assert not cache.read()[0].any()


@pytest.mark.parametrize("bits", [16, 4])
def test_idle_sequences(bits):
    from dstraining_b200.ops.kv_cache import WindowCache

    cache = WindowCache(3, 2, 64, 20, 2, bits=bits, device="cuda")
    cache.fill(_rand(3, 30, 2, 64, seed=1), _rand(3, 30, 2, 64, seed=2))
    before = cache.read()
    q, k, v = _rand(3, 4, 64, seed=3), _rand(3, 2, 64, seed=4), _rand(3, 2, 64, seed=5)
    out, ks, _ = cache.step(q, k, v, torch.tensor([30, -1, 30], device="cuda"), return_stored=True)
    after = cache.read()
    assert not out[1].any() and not ks[1].any() and out[0].any() and out[2].any()
    for a, b in zip(before, after):
        assert torch.equal(a[1], b[1]) and not torch.equal(a[0], b[0])


@pytest.mark.parametrize("bits", [16, 4])
def test_what_left_the_window_is_gone(bits):
    """Infinities and NaN in evicted, replaced or never written rows touch nothing."""
    from dstraining_b200.ops.kv_cache import WindowCache

    def run(poison):
        cache = WindowCache(1, 1, 64, 40, 0, bits=bits, device="cuda")
        k, v = _rand(1, 60, 1, 64, seed=1), _rand(1, 60, 1, 64, seed=2)
        if poison:
            k[:, 20], v[:, 20] = float("nan"), float("inf")  # the row that the next token replaces
            for x in cache._rows:
                if bits == 16:
                    x[:, :, 40:] = float("nan")
            for x in cache._params:
                if x is not None:
                    x[:, :, 40:] = -1  # NaN steps
        cache.fill(k, v)
        return cache.step(*(_rand(1, 1, 64, seed=i) for i in (3, 4, 5)))

    a, b = run(False), run(True)
    assert torch.isfinite(a).all() and torch.equal(a, b)


def test_a_visible_nan_shows():
    from dstraining_b200.ops.kv_cache import WindowCache

    for bits in (16, 4):
        cache = WindowCache(1, 1, 64, 40, 0, bits=bits, device="cuda")
        k, v = _rand(1, 30, 1, 64, seed=1), _rand(1, 30, 1, 64, seed=2)
        v[0, 5, 0, 3] = float("nan")
        cache.fill(k, v)
        out = cache.step(*(_rand(1, 1, 64, seed=i) for i in (3, 4, 5)))
        assert out[..., 3].isnan().all()
        assert torch.isfinite(out[..., 32:]).all()  # another group of 32


def test_constant_and_extreme_groups():
    """Groups without a range, and of the smallest and largest ranges, keep their values."""
    from dstraining_b200.ops.kv_cache import WindowCache

    k = torch.zeros(1, 5, 1, 64, device="cuda", dtype=torch.bfloat16)
    k[:, 0] = 3.0
    k[:, 1, :, ::2] = 1e30
    k[:, 2, :, ::2] = 1e-30
    k[:, 3] = -7.25
    k[:, 4, :, :32] = torch.arange(32, device="cuda").to(torch.bfloat16)
    cache = WindowCache(1, 1, 64, 8, 0, bits=4, device="cuda")
    cache.fill(k, k)
    for x in cache.read():
        assert torch.equal(x[:, :, :5].transpose(1, 2), _stands_for(k, 4))


def test_positions_beyond_32_bits():
    from dstraining_b200.ops.kv_cache import WindowCache

    p, W, S = 2**33 + 5, 37, 3
    cache = WindowCache(1, 1, 64, W, S, device="cuda")
    k, v = _rand(1, 40, 1, 64, seed=1), _rand(1, 40, 1, 64, seed=2)
    cache.fill(k, v)
    new = _rand(1, 1, 64, seed=4)
    out = cache.step(_rand(1, 1, 64, seed=3), new, new, torch.tensor([p], device="cuda"))
    slot = S + (p - S) % W
    assert torch.equal(cache.keys[0, 0, slot], new[0, 0])
    rest = torch.arange(40, device="cuda") != slot
    assert torch.equal(cache.keys[0, 0, rest], k[0, rest, 0])
    vals = cache.values[0, 0].double()
    s = torch.softmax(cache.keys[0, 0].double() @ _rand(1, 1, 64, seed=3)[0, 0].double() / 8, dim=0)
    want = s @ vals
    assert ((out[0, 0].double() - want).norm() / want.norm()).item() < 1.1 * U


def test_rows_beyond_32_bit_offsets():
    """A cache of more than 2^32 bytes per operand: the last rows are found."""
    from dstraining_b200.ops.kv_cache import WindowCache

    W = 2**24 + 70
    cache = WindowCache(1, 1, 128, W, 0, device="cuda")
    x = _rand(1, 100, 1, 128, seed=1)
    cache.keys[0, 0, W - 100:] = x[0, :, 0]
    cache.values[0, 0, W - 100:] = x[0, :, 0]
    cache.keys[0, 0, :W - 100, 0] = -300.0  # next to no weight for the query below
    q = torch.zeros(1, 1, 128, device="cuda", dtype=torch.bfloat16)
    q[..., 0] = 20.0
    new = _rand(1, 1, 128, seed=3)
    out = cache.step(q, new, new, torch.tensor([W - 1], device="cuda"))
    rows = torch.cat([x[0, :99, 0], new[0]]).double()
    want = torch.softmax(rows[:, 0] * 20 / 128**0.5, dim=0) @ rows
    assert ((out[0, 0].double() - want).norm() / want.norm()).item() < 1.1 * U


@pytest.mark.parametrize("bits", [16, 4])
def test_repeatable_strided_and_captured(bits):
    """Operands of one fused buffer; the same bits from every launch, also from a graph on another stream."""
    from dstraining_b200.ops.kv_cache import WindowCache

    H, D = 4, 64
    cache = WindowCache(1, H, D, 3000, 4, bits=bits, device="cuda")
    cache.fill(_rand(1, 3200, H, D, seed=1), _rand(1, 3200, H, D, seed=2))
    qkv = _rand(1, H, 3, D, seed=3)
    q, k, v = qkv.unbind(dim=2)
    pos = torch.tensor([3200], device="cuda")
    a = cache.step(q, k, v, pos)
    b = cache.step(q.contiguous(), k.contiguous(), v.contiguous(), pos)
    assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            c = cache.step(q, k, v, pos)
        for _ in range(3):
            g.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, c)


def test_lengths_out_of_range_are_reported():
    from dstraining_b200.ops import native
    from dstraining_b200.ops.kv_cache import WindowCache

    cache = WindowCache(2, 1, 64, 8, 0, device="cuda")
    k = _rand(2, 5, 1, 64, seed=1)
    cache.fill(k, k, torch.tensor([9, -3], device="cuda"))
    assert cache.pos.tolist() == [5, 0]
    assert native.lib().read_status(True) == 6  # bad argument


def test_refusals():
    from dstraining_b200.ops.kv_cache import WindowCache

    with pytest.raises(ValueError, match="head size"):
        WindowCache(1, 1, 200, 8, device="cuda")
    cache = WindowCache(2, 2, 64, 8, device="cuda")
    q, k = _rand(2, 4, 64, seed=1), _rand(2, 2, 64, seed=2)
    for bad in (_rand(2, 3, 64, seed=1), q.float(), q.cpu(), q[:1]):
        with pytest.raises(ValueError, match="q must"):
            cache.step(bad, k, k)
    with pytest.raises(ValueError, match="k must"):
        cache.step(q, k[:, :1], k)
    with pytest.raises(ValueError, match="pos must"):
        cache.step(q, k, k, torch.tensor([1, 2], device="cuda", dtype=torch.int32))
    with pytest.raises(ValueError, match="pos must"):
        cache.step(q, k, k, torch.tensor([1, 2]))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [1, 3, 8, 20])
@pytest.mark.parametrize("new", [False, True])
def test_a_nan_stays_in_its_group_however_many_heads_share_it(G, D, new):
    """One NaN channel: its 32 channels stand for NaN, in a held row as in the new one; the others stay finite."""
    from dstraining_b200.ops.kv_cache import WindowCache

    cache = WindowCache(1, 1, D, 40, 0, bits=4, device="cuda")
    k, v = _rand(1, 30, 1, D, seed=1), _rand(1, 30, 1, D, seed=2)
    q, k1, v1 = _rand(1, G, D, seed=3), _rand(1, 1, D, seed=4), _rand(1, 1, D, seed=5)
    (v1[0, 0] if new else v[0, 5, 0])[3] = float("nan")
    cache.fill(k, v)
    out = cache.step(q, k1, v1)
    assert out[..., :32].isnan().all()
    assert torch.isfinite(out[..., 32:]).all()


@pytest.mark.parametrize("G", [1, 8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bits", [16, 4])
def test_one_cta_adds_up_a_long_cache(bits, D, G):
    """More (sequence, key head) pairs than CTAs fit on the GPU: each CTA holds a whole cache, a warp adds up 8192
    keys, and the error is still that of rounding the result. One set of rows serves all key heads."""
    from dstraining_b200.ops.kv_cache import WindowCache

    Hk, W, S = 608, 32764, 4  # 4 CTAs an SM: 592
    T = W + S - 2
    cache = WindowCache(1, Hk, D, W, S, bits=bits, device="cuda")
    k, v = _rand(1, T, 1, D, seed=1), _rand(1, T, 1, D, seed=2)
    cache.fill(k.expand(-1, -1, Hk, -1), v.expand(-1, -1, Hk, -1))
    q, k1, v1 = _rand(1, Hk * G, D, seed=3), _rand(1, 1, D, seed=4), _rand(1, 1, D, seed=5)
    out = cache.step(q, k1.expand(-1, Hk, -1), v1.expand(-1, Hk, -1))
    keys, values = (torch.cat([_stands_for(x[0, :, 0], bits), _stands_for(y[0], bits)]).double()
                    for x, y in ((k, k1), (v, v1)))
    some = torch.arange(0, Hk * G, G * Hk // 304, device="cuda")
    want = torch.softmax(q[0, some].double() @ keys.T * D**-0.5, dim=-1) @ values
    assert ((out[0, some].double() - want).norm() / want.norm()).item() < 1.1 * U


@pytest.mark.parametrize("G", [1, 8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("large", [8.0, 30.0])
def test_one_cta_adds_up_values_beside_a_large_channel(large, D, G):
    """One channel of each group is large and of one sign, so the others' codes are far from the middle: their sums
    cancel, and still are as good as their rounding."""
    from dstraining_b200.ops.kv_cache import WindowCache

    Hk, T = 608, 32766
    k, v = _rand(1, T, 1, D, seed=1), _rand(1, T, 1, D, seed=2)
    q, k1, v1 = _rand(1, Hk * G, D, seed=3), _rand(1, 1, D, seed=4), _rand(1, 1, D, seed=5)
    for x in (v, v1):
        x[..., 7::32] = large + x[..., 7::32].abs()
    cache = WindowCache(1, Hk, D, T + 2, 0, bits=4, device="cuda")
    cache.fill(k.expand(-1, -1, Hk, -1), v.expand(-1, -1, Hk, -1))
    out = cache.step(q, k1.expand(-1, Hk, -1), v1.expand(-1, Hk, -1))
    keys, values = (torch.cat([_stands_for(x[0, :, 0], 4), _stands_for(y[0], 4)]).double() for x, y in ((k, k1), (v, v1)))
    some = torch.arange(0, Hk * G, G * Hk // 304, device="cuda")
    want = torch.softmax(q[0, some].double() @ keys.T * D**-0.5, dim=-1) @ values
    for part in (slice(7, None, 32), slice(8, None, 32), slice(31, None, 32)):
        assert ((out[0, some, part].double() - want[:, part]).norm() / want[:, part].norm()).item() < 1.2 * U


@pytest.mark.parametrize("bits", [16, 4])
def test_first_step_under_capture(bits):
    """A cache whose first step is captured: steps outside the graph are right before and after its replays."""
    from dstraining_b200.ops.kv_cache import WindowCache

    H, D = 2, 64
    k, v = _rand(1, 3000, H, D, seed=1), _rand(1, 3000, H, D, seed=2)
    q, k1, v1 = (_rand(1, H, D, seed=i) for i in (3, 4, 5))
    pos = torch.tensor([3000], device="cuda")

    def make():
        cache = WindowCache(1, H, D, 4000, 4, bits=bits, device="cuda")
        cache.fill(k, v)
        return cache

    want = make().step(q, k1, v1, pos)
    cache = make()
    # the graphs' memory holds sevens
    pool, g0 = torch.cuda.graph_pool_handle(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g0, pool=pool):
        dirt = [torch.full((2**17,), 7, dtype=torch.int32, device="cuda") for _ in range(16)]
    g0.replay()
    del dirt
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, pool=pool):
        captured = cache.step(q, k1, v1, pos)
    for _ in range(2):
        got = torch.full_like(want, float("nan"))  # where the next result may land
        del got
        assert torch.equal(cache.step(q, k1, v1, pos), want)
    g.replay()
    assert torch.equal(captured, want)
    assert torch.equal(cache.step(q, k1, v1, pos), want)


@pytest.mark.parametrize("D,G1,G2", [(128, 2, 8), (64, 4, 8)])
def test_steps_of_one_cache_do_not_depend_on_earlier_ones(D, G1, G2):
    """Calls with other numbers of query heads leave no trace: the same bits as from a cache of its own."""
    from dstraining_b200.ops.kv_cache import WindowCache

    B, n = 33, 3000
    k, v = _rand(B, n, 1, D, seed=1), _rand(B, n, 1, D, seed=2)
    k1, v1 = _rand(B, 1, D, seed=4), _rand(B, 1, D, seed=5)
    pos = torch.full((B,), n, device="cuda")

    def make():
        cache = WindowCache(B, 1, D, n + 100, 0, bits=4, device="cuda")
        cache.fill(k, v)
        return cache

    used = make()
    for G in (G1, G2, G1):
        q = _rand(B, G, D, seed=6 + G)
        assert torch.equal(used.step(q, k1, v1, pos), make().step(q, k1, v1, pos))


@pytest.mark.parametrize("bits", [16, 4])
def test_positions_of_any_stride(bits):
    """Positions and lengths as columns of larger tables, also the cache's own."""
    from dstraining_b200.ops.kv_cache import WindowCache

    table = torch.tensor([[12, 30, -7], [40, 3, -7], [41, 0, -7]], device="cuda")
    own = torch.zeros(3, 2, dtype=torch.int64, device="cuda")
    k, v = _rand(3, 40, 2, 64, seed=1), _rand(3, 40, 2, 64, seed=2)
    q, k1, v1 = _rand(3, 4, 64, seed=3), _rand(3, 2, 64, seed=4), _rand(3, 2, 64, seed=5)
    a = WindowCache(3, 2, 64, 20, 2, bits=bits, device="cuda", pos=own[:, 1])
    b = WindowCache(3, 2, 64, 20, 2, bits=bits, device="cuda")
    a.fill(k, v, table[:, 1])
    b.fill(k, v, table[:, 1].contiguous())
    assert own.tolist() == [[0, 30], [0, 3], [0, 0]]
    assert all(torch.equal(x, y) for x, y in zip(a.read(), b.read()))
    assert torch.equal(a.step(q, k1, v1, table[:, 0]), b.step(q, k1, v1, table[:, 0].contiguous()))
    assert torch.equal(a.step(q, k1, v1), b.step(q, k1, v1))
    assert own.tolist() == [[0, 31], [0, 4], [0, 1]] and b.pos.tolist() == [31, 4, 1]
    assert all(torch.equal(x, y) for x, y in zip(a.read(), b.read()))
