"""Log probabilities, entropy and alternatives against 64 bits.

A logit less the maximum is rounded once (2^-24 of it), a power is 2^-22 of itself off, and a thread adds up to 200 of them (2^-24 each), in parts that are joined in some tens of steps: the sum is within
2^-15 of itself in the worst case, and its logarithm within 2^-15.  Entropy's second sum holds products with numbers up to 200 that have died down to e^-200 (x e^x is at most 1 / e): 2^-15 of
its terms' magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def ops():
    import lia_b200
    from lia_b200 import ops
    return ops


def reference(x, tokens, top):
    y = x.double()
    y = y - y.amax(-1, keepdim=True)
    logp = y - torch.log(torch.exp(y).sum(-1, keepdim=True))
    p = torch.exp(logp)
    entropy = -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(-1)
    ranked = torch.where(torch.isnan(x), torch.full_like(x, -INF), x).float()
    ids = torch.sort(ranked, dim=-1, descending=True, stable=True)[1][:, :top]
    given = None
    if tokens is not None:
        t = tokens.view(len(x), -1)
        inside = (t >= 0) & (t < x.shape[1])
        given = torch.where(inside, logp.gather(1, t.clamp(0, x.shape[1] - 1)), torch.full_like(t, NAN, dtype=torch.float64)).view(tokens.shape)
    return given, entropy, logp.gather(1, ids), ids


def close(a, b, what):
    assert a.shape == b.shape, what
    assert torch.equal(torch.isnan(a), torch.isnan(b)), (what, a, b)
    inf = torch.isinf(b)
    assert torch.equal(a[inf].double(), b[inf]), what
    fine = torch.isfinite(b)
    off = (a[fine].double() - b[fine]).abs()
    assert (off <= 2.0 ** -15 + 2.0 ** -21 * b[fine].abs()).all(), (what, off.max())


def check(ops, x, tokens, top):
    got, want = ops.token_logprobs(x, tokens, top), reference(x, tokens, top)
    if tokens is not None:
        close(got[0], want[0], "given")
    else:
        assert got[0] is None
    close(got[1], want[1], "entropy")
    close(got[2], want[2], "alternatives")
    assert got[3].dtype == torch.int64 and torch.equal(got[3], want[3]), "ids"
    return got


def rnd(M, V, seed=0, std=2.5, dtype=F32):
    return (torch.randn(M, V, generator=torch.Generator("cuda").manual_seed(seed), device="cuda") * std).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,V,n,top", [(1, 1, 1, 1), (3, 2, 2, 2), (2, 31, 1, 31), (2, 33, 1, 32), (5, 511, 1, 5), (5, 512, 3, 20), (4, 513, 0, 32), (3, 4095, 1, 1), (3, 4097, 1, 0),
                                       (1, 50272, 1, 20), (4, 50265, 2, 5), (77, 50265, 1, 8), (300, 8193, 1, 32), (700, 1000, 40, 20), (1300, 513, 1, 7)])
def test_sizes(ops, dtype, M, V, n, top):
    x = rnd(M, V, seed=M + V, dtype=dtype)
    tokens = torch.randint(0, V, (M, n), generator=torch.Generator("cuda").manual_seed(1), device="cuda") if n else None
    check(ops, x, tokens, top)
    if n == 1:
        got = ops.token_logprobs(x, tokens.view(M), top)
        assert got[0].shape == (M,) and torch.equal(got[0], ops.token_logprobs(x, tokens, top)[0][:, 0])        # and the same bits each time


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shift,extra", [(0, 1), (1, 0), (3, 2), (5, 7)])
def test_rows_off_16_byte_boundaries(ops, dtype, shift, extra):
    """Column slices: what lies beside a row is larger than anything in it."""
    M, V = 6, 5003
    wide = torch.full((M, V + shift + extra), 1e4, dtype=dtype, device="cuda")
    wide[:, shift:shift + V] = rnd(M, V, seed=2, dtype=dtype)
    check(ops, wide[:, shift:shift + V], torch.arange(M, device="cuda").view(M, 1) * 7, 9)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [40, 3000, 20001])
def test_orders_and_ties(ops, dtype, V):
    up = torch.linspace(-9, 9, V, device="cuda")
    rows = [up, up.flip(0), torch.zeros(V, device="cuda"), (torch.arange(V, device="cuda") % 3).float(), torch.where(torch.arange(V, device="cuda") % 2 == 0, 0.0, -0.0),
            (torch.arange(V, device="cuda") == V - 1).float() * 60, (torch.arange(V, device="cuda") % 512 == 511).float()]
    check(ops, torch.stack(rows).to(dtype), torch.full((len(rows), 1), V - 1, device="cuda"), 32)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [37, 9000])
def test_infinities_and_nan(ops, dtype, V):
    x = rnd(8, V, seed=5, dtype=dtype)
    x[0] = -INF
    x[1, : V - 3] = -INF                                   # fewer tokens that can be than alternatives asked for
    x[2, 5] = NAN
    x[3, V - 1] = INF
    x[4] = NAN
    x[5] = -INF
    x[5, 7] = 3.0                                          # one token alone
    x[6, ::2] = -INF
    x[7] = 1e30 if dtype == F32 else 1e30
    x[7, 3] = -1e30
    got = check(ops, x, torch.tensor([[1, V - 1]] * 8, device="cuda"), 10)
    assert got[1][5] == 0 and got[2][5, 0] == 0


def test_ids_outside_the_vocabulary(ops):
    x = rnd(4, 100)
    check(ops, x, torch.tensor([-1, 100, -(1 << 40), 99], device="cuda"), 3)


def test_nothing_to_do(ops):
    got = ops.token_logprobs(torch.empty(0, 100, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), 3)
    assert [tuple(t.shape) for t in got] == [(0,), (0,), (0, 3), (0, 3)]


def test_replayed_and_on_another_stream(ops):
    x, t = rnd(3, 30011, seed=1), torch.tensor([1, 2, 3], device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        first = ops.token_logprobs(x, t, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.token_logprobs(x, t, 4)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, got))
    x.copy_(rnd(3, 30011, seed=2))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ops.token_logprobs(x, t, 4), got))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("fill,most", [(None, 5.0), (-1e37, 5.0), (-3e38, 3e38)], ids=["least", "1e37", "3e38"])
@pytest.mark.parametrize("M,V", [(1, 40), (2, 600), (3, 9000), (4, 50265), (700, 4100)])
def test_finite_masks(ops, dtype, fill, most, M, V):
    """Banned tokens with the type's least number, or another far below the rest, instead of -inf: before the others, behind them, around them, all but one, in every second place, all of them.
    Their distances to the maximum, and those distances times their number, leave 32 bits; a distance that does is minus infinity in the results too."""
    fill = torch.finfo(dtype).min if fill is None else fill
    i = torch.arange(V, device="cuda")
    masks = [i < V // 2, i >= V // 3, (i < V // 3) | (i >= V // 2), i != V - 1, i != 0, i % 2 == 0, (i // 16) % 2 == 0, i >= 0]
    x = rnd(M * len(masks), V, seed=V, dtype=dtype)
    x[:, V - 1], x[:, 0] = most, most
    x = torch.where(torch.stack(masks).repeat(M, 1), torch.full_like(x, fill), x)
    tokens = torch.tensor([[V - 1, 0, V // 2]] * len(x), device="cuda")
    got, want = ops.token_logprobs(x, tokens, 5), reference(x, tokens, 5)
    for a, b, what in zip(got, want, ("given", "entropy", "alternatives")):
        close(a, b.float().double(), what)
    assert torch.isfinite(got[1]).all() and torch.equal(got[3], want[3])
