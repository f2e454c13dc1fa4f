"""Projections in 8-bit integers: tokens' codes against the definition in 64 bits, products against whole numbers.

Sums are exact, and what follows is three roundings that are the same anywhere -- the sum to 32 bits, times the token's scale, times the channel's -- and one to the output's type: outputs are equal, bit
by bit.  Codes of bf16 numbers are exact (tests/test_gpu_kv_8bit.py); of fp32 ones they may be the neighbouring code where the exact quotient is within 2^-20 of a border."""
import pytest
import torch

from test_gpu_wait_limits import given_up, nowait  # noqa: F401

pytestmark = pytest.mark.gpu
BF16, F32, F64, I8 = torch.bfloat16, torch.float32, torch.float64, torch.int8
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def ops():
    import lia_b200  # noqa: F401
    from lia_b200 import ops
    return ops


def codes(rows, K, seed, ld=None, lo=-127):
    c = torch.randint(lo, 128, (rows, K), generator=torch.Generator("cuda").manual_seed(seed), device="cuda", dtype=torch.int16).to(I8)
    out = torch.zeros(rows, ld or (K + 15) // 16 * 16, dtype=I8, device="cuda")[:, :K]
    out.copy_(c)
    return out


def scales(n, seed):
    return torch.rand(n, generator=torch.Generator("cuda").manual_seed(seed), device="cuda") * 0.02 + 1e-3


def want(x, sx, w, sw, out):
    return ((x.double() @ w.double().t()).float() * sx[:, None] * sw).to(out)


@pytest.mark.parametrize("act", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 8), (3, 17), (5, 64), (2, 1001), (7, 2560), (4, 8192), (3, 8200), (2, 28672), (300, 130), (1, 40001)])
def test_tokens_codes(ops, act, M, K):
    x = (torch.randn(M, K, generator=torch.Generator("cuda").manual_seed(K), device="cuda") * 1.7).to(act)
    x[:, ::11] *= 30
    c, s = ops.quantize_rows(x)
    a = x.double().abs().amax(1, keepdim=True).clamp(min=2.0 ** -100)
    assert c.shape == (M, K) and c.stride(0) % 16 == 0 and ((s.double() - a[:, 0] / 127).abs() <= 2.0 ** -24 * s.double()).all()
    y = x.double() * 127 / a
    if act == BF16:
        assert torch.equal(c.double(), torch.round(y))
    else:
        lo, hi = torch.round(y - y.abs() * 2.0 ** -20), torch.round(y + y.abs() * 2.0 ** -20)
        assert ((c.double() >= lo) & (c.double() <= hi)).all()


def test_tokens_codes_at_the_edges(ops):
    """Zeros, ties, extreme sizes, infinities and NaN; columns of something wider on an odd boundary, codes of a buffer of the caller's."""
    x = torch.randn(10, 50, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(BF16)
    x[0] = 0
    x[1, 3], x[2, 4], x[3, 5] = INF, -INF, NAN
    x[4] = (x[4].float() * 2.0 ** -120).to(BF16)
    x[5] = (x[5].float() / x[5].float().abs().max() * 3.3e38).to(BF16)
    x[6] = 0
    x[6, :3] = torch.tensor([1.0, 0.5, -0.5], dtype=BF16)                     # 63.5 goes to the even 64
    wide = torch.zeros(10, 61, dtype=BF16, device="cuda")
    wide[:, 3:53] = x
    buffer = torch.full((10, 80), 7, dtype=I8, device="cuda")
    c, s = ops.quantize_rows(wide[:, 3:53], codes=buffer[:, 8:58])
    assert (buffer[:, :8] == 7).all() and (buffer[:, 58:] == 7).all()
    assert torch.isnan(s[1:4]).all() and (c[1:4] == 0).all() and torch.isfinite(s[[0, 4, 5, 6, 7]]).all()
    assert (c[0] == 0).all() and c[6, :4].tolist() == [127, 64, -64, 0]
    for r in (4, 5, 7, 8, 9):
        a = x[r].double().abs().max().clamp(min=2.0 ** -100)
        assert torch.equal(c[r].double(), torch.round(x[r].double() * 127 / a))
    assert ops.quantize_rows(x[:0])[0].shape == (0, 50)


def test_rows_that_share_their_place_are_refused(ops):
    from lia_b200._lib import LiaError
    x = torch.randn(1, 64, device="cuda")
    w, sw = ops.quantize_rows(torch.randn(16, 64, device="cuda"))
    for call in (lambda: ops.quantize_rows(x.expand(5, 64)), lambda: ops.quantize_rows(x.view(64).as_strided((3, 32), (8, 1))), lambda: ops.linear_int8(x.expand(5, 64), w, sw),
                 lambda: ops.linear_int8(x, w[:1].expand(4, 64), sw[:4])):
        with pytest.raises(LiaError, match="sizes"):
            call()
    assert torch.equal(ops.quantize_rows(x.expand(1, 64))[0], ops.quantize_rows(x)[0])


@pytest.mark.parametrize("out", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [
    (1, 1, 1), (1, 2560, 2560), (2, 7, 15), (3, 130, 16), (16, 128, 128), (17, 1000, 129), (33, 129, 1000), (64, 4096, 512), (65, 300, 4096), (100, 257, 777), (128, 1024, 1024), (1, 300, 16384),
    (4, 20000, 640), (129, 64, 64), (130, 1, 300), (200, 1001, 1000), (300, 2560, 2560), (513, 130, 16), (700, 1000, 520), (1030, 2100, 1300), (2049, 515, 257), (1500, 6000, 384)])
def test_products_of_codes(ops, out, M, N, K):
    x, w, sx, sw = codes(M, K, 1), codes(N, K, 2), scales(M, 3), scales(N, 4)
    guard = torch.full((M * N + 64,), 77.0, dtype=out, device="cuda")
    y = ops.linear_int8(x, w, sw, out=guard[32:32 + M * N].view(M, N), x_scale=sx)
    assert torch.equal(y, want(x, sx, w, sw, out))
    assert (guard[:32] == 77).all() and (guard[-32:] == 77).all()


@pytest.mark.parametrize("M", [2, 40, 300])
def test_longest_sums(ops, M):
    """131071 products of the largest codes: just inside 32 bits; one more is refused."""
    K, N = 131071, 5
    x, w = codes(M, K, 1), codes(N, K, 2)
    x[0], w[0], w[1] = -128, -128, 127
    sx, sw = scales(M, 3), scales(N, 4)
    assert torch.equal(ops.linear_int8(x, w, sw, x_scale=sx, out=torch.empty(M, N, device="cuda")), want(x, sx, w, sw, F32))
    from lia_b200._lib import LiaError
    with pytest.raises(LiaError, match="131071"):
        ops.linear_int8(codes(M, K + 1, 1), codes(N, K + 1, 2), sw, x_scale=sx)


@pytest.mark.parametrize("act", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("M", [1, 5, 64, 128, 129, 600])
def test_from_activations(ops, act, M):
    """Tokens that are quantised on the way, from columns of something wider: what quantize_rows and the product of its codes give, and NaN for a token that is not finite."""
    N, K = 515, 1003
    wide = torch.randn(M, K + 9, generator=torch.Generator("cuda").manual_seed(2), device="cuda").to(act)
    x = wide[:, 5:5 + K]
    if M > 4:
        x[1] = 0
        x[3, 77] = INF
    w, sw = ops.quantize_rows(torch.randn(N, K, generator=torch.Generator("cuda").manual_seed(3), device="cuda") * K ** -0.5)
    y = ops.linear_int8(x, w, sw)
    assert y.dtype == act
    c, s = ops.quantize_rows(x)
    assert torch.equal(torch.nan_to_num(y.float(), nan=-5.0), torch.nan_to_num(want(c, s, w, sw, act).float(), nan=-5.0))
    if M > 4:
        assert torch.isnan(y[3]).all() and (y[1] == 0).all() and torch.isfinite(y[4]).all()


@pytest.mark.parametrize("M", [1, 3])
def test_weights_quantised_right_before(ops, M):
    """A product begins to bring its weights while the tokens are quantised: not before the kernel that wrote them has ended."""
    N, K = 8192, 4096
    x = torch.randn(M, K, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(BF16)
    c, s = ops.quantize_rows(x)
    buffer, sw = torch.empty(N, K, dtype=I8, device="cuda"), torch.empty(N, device="cuda")
    for i in range(6):
        real = torch.randn(N, K, generator=torch.Generator("cuda").manual_seed(10 + i), device="cuda").to(BF16)
        torch.cuda.synchronize()
        ops.quantize_rows(real, codes=buffer, scale=sw)
        one = ops.linear_int8(x, buffer, sw) if i % 2 else ops.linear_int8(c, buffer, sw, x_scale=s)
        assert torch.equal(one, want(c, s, buffer, sw, BF16)), i


@pytest.mark.parametrize("M", [1, 3, 64, 700])
def test_streams_and_graphs(ops, M):
    """Two streams at once, a captured call with other tokens in it, and two captured graphs that are replayed at the same time: each has its own workspace."""
    N, K = 2560, 2560
    w, sw = ops.quantize_rows(torch.randn(N, K, generator=torch.Generator("cuda").manual_seed(1), device="cuda"))
    xs = [torch.randn(M, K, generator=torch.Generator("cuda").manual_seed(5 + i), device="cuda").to(BF16) for i in range(2)]
    wants = [want(*ops.quantize_rows(x), w, sw, BF16) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(25):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(ops.linear_int8(xs[i], w, sw))
    torch.cuda.synchronize()
    assert all(torch.equal(y, wants[i]) for i in range(2) for y in outs[i])
    graphs = []
    for i, s in enumerate(streams):
        g, y = torch.cuda.CUDAGraph(), torch.empty(M, N, dtype=BF16, device="cuda")
        with torch.cuda.graph(g, stream=s):
            ops.linear_int8(xs[i], w, sw, out=y)
        graphs.append((g, y))
    xs[0].mul_(-3.0)
    torch.cuda.synchronize()
    for _ in range(10):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want(*ops.quantize_rows(xs[0]), w, sw, BF16)) and torch.equal(graphs[1][1], wants[1])


@pytest.mark.parametrize("act", [BF16, F32, I8], ids=["bf16", "f32", "codes"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 256), (2, 1, 255), (2, 3, 257), (1, 300, 511), (2, 1001, 513), (1, 129, 1543), (2, 515, 7000), (1, 7, 32768), (1, 7, 32769), (2, 33, 16384), (2, 33, 16385),
                                   (1, 200001, 300), (2, 120001, 270), (1, 64, 28673), (2, 2561, 2561), (1, 16384, 4096), (1, 16385, 4096)])
def test_a_token_or_two(ops, act, M, N, K):
    """Both sides of the borders of the form in one launch: its last channels' last codes lie at the very end of the weights, tokens are columns of something wider."""
    ld = (K + 15) // 16 * 16
    flat = codes(N, K, 2, ld).as_strided((N * ld,), (1,))[:(N - 1) * ld + K].clone()
    w, sw = flat.as_strided((N, K), (ld, 1)), scales(N, 4)
    guard = torch.full((M * N + 64,), 77.0, dtype=F32, device="cuda")
    y = guard[32:32 + M * N].view(M, N)
    if act == I8:
        x, sx = codes(M, K, 1, ld + 16), scales(M, 3)
        ops.linear_int8(x, w, sw, out=y, x_scale=sx)
    else:
        x = torch.randn(M, K + 9, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(act)[:, 5:5 + K]
        ops.linear_int8(x, w, sw, out=y)
        x, sx = ops.quantize_rows(x)
    assert torch.equal(y, want(x, sx, w, sw, F32)) and (guard[:32] == 77).all() and (guard[-32:] == 77).all()
    assert torch.equal(ops.linear_int8(x, w, sw, x_scale=sx), want(x, sx, w, sw, BF16))
    if act != I8:
        bad = torch.randn(M, K, device="cuda").to(act)
        bad[M - 1, K - 1] = NAN
        out = ops.linear_int8(bad, w, sw)
        assert torch.isnan(out[M - 1]).all() and torch.isfinite(out[:M - 1]).all()


def test_a_tokens_outputs_do_not_depend_on_the_others(ops):
    N, K = 1536, 2048
    w, sw = ops.quantize_rows(torch.randn(N, K, generator=torch.Generator("cuda").manual_seed(1), device="cuda"))
    x = torch.randn(1100, K, generator=torch.Generator("cuda").manual_seed(2), device="cuda").to(BF16)
    all_rows = ops.linear_int8(x, w, sw)
    for n in (1, 5, 31, 64, 128, 129, 400, 800):
        assert torch.equal(ops.linear_int8(x[:n], w, sw), all_rows[:n])


@pytest.mark.parametrize("M,N,K", [(3, 2560, 2560), (40, 700, 1000), (128, 300, 4096), (200, 500, 300), (700, 1000, 256)])
@pytest.mark.parametrize("given", [False, True])
def test_waits_that_run_out(nowait, monkeypatch, ops, M, N, K, given):  # noqa: F811
    """With a limit of 0 every wait gives up: the launch ends, every output is NaN and nothing else is written, its blocks are counted; the next launch is right."""
    x = torch.randn(M, K, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(BF16)
    w, sw = ops.quantize_rows(torch.randn(N, K, generator=torch.Generator("cuda").manual_seed(2), device="cuda"))
    c, s = ops.quantize_rows(x)
    guard = torch.full((M * N + 64,), 7.0, device="cuda")
    y = guard[32:32 + M * N].view(M, N)
    call = lambda: ops.linear_int8(c if given else x, w, sw, out=y, x_scale=s if given else None)  # noqa: E731
    seen = nowait.lia_moe_timeouts_seen()
    assert given_up(nowait, monkeypatch, call) >= 1
    assert nowait.lia_moe_timeouts_seen() > seen and torch.isnan(y).all() and (guard[:32] == 7).all() and (guard[-32:] == 7).all()
    call()
    assert torch.equal(y, want(c, s, w, sw, F32))
