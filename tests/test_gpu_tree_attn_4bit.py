"""Attention over caches of 4 bits, against 64 bits.

Tolerances are those of attention over 8-bit caches (tests/test_gpu_tree_attn.py): weights in fp16, 2^-11 of A; with more than 32 rows of a key head values are multiplied by their group's scale in
fp16 as well, 2^-11 for the factor and 2^-11 for the product.  There keys are multiplied by their group's scale, relative to the key's largest, in the same way: 2^-10 of every product, so that a score
is off by up to 2^-10 B more.

Up to two rows of a key head: the sums of 16 keys, of codes + 8 times weights, begin with -8 times the weights' sum W.  That is 5 products of up to 17 additions, each at least as exact as fp32 cut off
(2^-23) and none of more than 15 W in codes: 5 * 17 * 2^-23 * 15 W, and over all keys as much of the weighted sum of the channel's scales, where A is the weighted sum of its numbers."""
import pytest
import torch

from cache4 import numbers, packed
from test_gpu_tree_attn import DIMS, Case, family, rnd
from test_gpu_wait_limits import given_up, nowait  # noqa: F401

pytestmark = pytest.mark.gpu
BF16, F32, F64, U8 = torch.bfloat16, torch.float32, torch.float64, torch.uint8
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def ops():
    import lia_b200  # noqa: F401
    from lia_b200 import ops
    return ops


class Case4(Case):
    def __init__(self, *args, **kw):
        super().__init__(*args, "int4", **kw)

    def codes(self, x, kind, seed):
        y = x.float().unflatten(-1, (-1, 32))
        s = (y.abs().amax(-1) * (1 + torch.rand(y.shape[:-1], generator=torch.Generator("cuda").manual_seed(seed), device="cuda")) / 7).to(BF16)
        c = torch.round(y / s.float()[..., None]).flatten(-2)
        slots_first = x.shape[0] == self.slots and x.shape[1] == self.cap
        return packed(c), (s.permute(0, 2, 1, 3) if slots_first else s.permute(1, 2, 0, 3)).contiguous()

    def check(self, out):
        """Every row against 64 bits; rows of no portion untouched."""
        touched = torch.zeros(self.M, dtype=torch.bool, device="cuda")
        kc, vc = (x.view(x.shape[0], x.shape[1], self.G, -1) if x.dim() == 3 else x for x in (self.kc, self.vc))
        many = max(s[3] for s in self.segs) * (self.H // self.G) > 32
        for z, (s, p0, r, n) in enumerate(self.segs):
            touched[r:r + n] = True
            if n == 0:
                continue
            see = self.visible(z)
            for h in range(self.H):
                g = h // (self.H // self.G)
                k, v = numbers(kc[s, :p0 + n, g], self.ks[s, g, :p0 + n], self.dim), numbers(vc[s, :p0 + n, g], self.vs[s, g, :p0 + n], self.vdim)
                q = self.q[r:r + n, h * self.dim:(h + 1) * self.dim].double()
                f = self.scale * (float(self.temp[h]) if self.temp is not None else 1.0)
                x, B = q @ k.t() * f, torch.where(see, q.abs() @ k.abs().t() * abs(f), 0.0).amax(1, keepdim=True)
                if self.softcap:
                    x = self.softcap * torch.tanh(x / self.softcap)
                S = torch.where(see, x.abs(), torch.zeros_like(x)).amax(1, keepdim=True)
                x = x.masked_fill(~see, -INF)
                p = torch.where(see.any(1, keepdim=True), torch.softmax(x, -1), torch.zeros_like(x))
                o, A = p @ v, p @ v.abs()
                if max(s[3] for s in self.segs) * (self.H // self.G) <= 2:
                    A = A + 2.0 ** 11 * 5 * 17 * 15 * 2.0 ** -23 * (p @ self.vs[s, g, :p0 + n].double().nan_to_num().repeat_interleave(32, -1))
                d = (self.dim * 2.0 ** -24 + (2.0 ** -10 if many else 0)) * B + 2.0 ** -21 * (S + self.softcap) + 2.0 ** -20
                tol = 2.0 ** -8 * o.abs() + ((3 if many else 1) * 2.0 ** -11 + 2 * d) * A + 1e-30
                got = out[r:r + n, h * self.vdim:(h + 1) * self.vdim].double()
                bad = ((got - o).abs() > tol) | torch.isnan(got)
                assert not bad.any(), (z, h, bad.nonzero()[:4].tolist(), (got - o).abs().max().item(), ((got - o).abs() / tol).max().item())
        assert (out[~touched] == 77).all(), "rows of no portion"


@pytest.mark.parametrize("dim,vdim", DIMS)
@pytest.mark.parametrize("H,G", [(4, 4), (6, 2), (16, 1)])
def test_single_tokens(ops, dim, vdim, H, G):
    c = Case4([(i, p0, 1) for i, p0 in enumerate((0, 1, 14, 15, 16, 17, 63, 64, 255, 256, 1000))], H, G, dim, vdim)
    c.check(c.run(ops))


@pytest.mark.parametrize("H,G,n", [(3, 3, 2), (4, 4, 16), (4, 4, 17), (2, 2, 33), (2, 2, 64), (8, 2, 5), (8, 2, 29), (5, 1, 13), (32, 2, 9)])
def test_chains_behind_ragged_histories(ops, H, G, n):
    c = Case4([(2, 700, n), (0, 0, n), (1, 37, max(1, n - 1)), (3, 16, 1)], H, G, 128, 128, gap=2)
    c.check(c.run(ops))


@pytest.mark.parametrize("dim,vdim", DIMS)
@pytest.mark.parametrize("n,branch", [(2, 1), (7, 2), (29, 2), (40, 3), (64, 3), (65, 2), (130, 4)])
def test_trees(ops, dim, vdim, n, branch):
    parents = lambda i: (i - 1) // branch if i else -1  # noqa: E731
    c = Case4([(0, 333, n), (2, 0, n), (1, 48, max(1, n // 2))], 4, 2, dim, vdim, mask=[family(n, parents), family(n, parents), family(max(1, n // 2), parents)], softcap=20.0, temp=True)
    c.check(c.run(ops))


@pytest.mark.parametrize("window", [1, 2, 16, 100, 5000])
@pytest.mark.parametrize("masked", [False, True])
def test_windows(ops, window, masked):
    n = 21
    tree = family(n, lambda i: (i - 1) // 2 if i else -1)
    deep = [int(tree[i].sum()) - 1 for i in range(n)]
    c = Case4([(1, 500, n), (0, 3, n), (2, 0, 5)], 6, 3, 128, 128, mask=[tree, tree, tree[:5, :5]] if masked else None, depth=[deep, deep, deep] if masked else None, window=window)
    c.check(c.run(ops))


@pytest.mark.parametrize("dim,vdim", DIMS)
@pytest.mark.parametrize("window", [0, 90])
def test_portions_of_prompts(ops, dim, vdim, window):
    c = Case4([(1, 130, 301), (0, 0, 257), (2, 64, 1)], 4, 2, dim, vdim, window=window)
    c.check(c.run(ops))


def test_any_mask_and_rows_that_see_nothing(ops):
    g = torch.Generator().manual_seed(3)
    masks = [torch.rand(n, n, generator=g) < 0.3 for n in (11, 70, 1, 3)]
    masks[0][4] = False
    masks[1][69] = False
    masks[2][0] = False
    c = Case4([(0, 0, 11), (1, 0, 70), (2, 0, 1), (3, 20, 3)], 4, 4, 64, 64, mask=masks, words=3)
    c.mask[:, 2] = -1
    c.mask[c.segs[0][2]:c.segs[0][2] + 11, 0] |= -1 << 11
    out = c.run(ops)
    c.check(out)
    assert (out[c.segs[0][2] + 4] == 0).all() and (out[c.segs[2][2]] == 0).all()


@pytest.mark.parametrize("n", [12, 40])
@pytest.mark.parametrize("what", ["behind", "other slots", "value scales", "one value scale", "one key scale", "infinite"])
def test_what_a_row_does_not_see_has_no_effect(ops, n, what):
    """Scales of NaN and infinity of tokens that some rows see and others do not, behind the portions and in other slots; one group's scale spoils its own channels alone where it is a value's."""
    p0, H, G, bad = 40, 4, 2, 5                                             # seen by itself and what descends from it
    tree = family(n, lambda i: (i - 1) // 2 if i else -1)
    make = lambda: Case4([(1, p0, n)], H, G, 128, 128, mask=[tree], slots=3, cap=p0 + n + 20)  # noqa: E731
    clean = make().run(ops).clone()
    c = make()
    hit = [i for i in range(n) if tree[i, bad]]
    if what == "behind":
        c.kc[1, p0 + n:], c.vc[1, p0 + n:], hit = 0xff, 0xff, []
        c.ks[1, :, p0 + n:], c.vs[1, :, p0 + n:] = NAN, NAN
    elif what == "other slots":
        for s in (0, 2):
            c.ks[s], c.vs[s] = NAN, INF
        hit = []
    elif what == "value scales":
        c.vs[1, :, p0 + bad] = NAN
    elif what == "one value scale":
        c.vs[1, :, p0 + bad, 2] = NAN
    elif what == "one key scale":
        c.ks[1, :, p0 + bad, 3] = NAN
    else:
        c.vs[1, :, p0 + bad, 1] = INF
        c.vc[1, p0 + bad] = 0xaa                                            # codes of 2
    out = c.run(ops)
    rest = [i for i in range(n) if i not in hit]
    near = lambda a, b: (a.double() - b.double()).abs() <= 2.0 ** -7 * b.double().abs() + 2.0 ** -9  # noqa: E731 (formed key by key: rounded elsewhere)
    assert near(out[rest], clean[rest]).all()
    if hit:
        heads = out[hit].view(len(hit), H, 4, 32).float()
        if what == "one value scale":
            assert torch.isnan(heads[:, :, 2]).all() and near(out[hit].view(len(hit), H, 4, 32)[:, :, [0, 1, 3]], clean[hit].view(len(hit), H, 4, 32)[:, :, [0, 1, 3]]).all()
        elif what == "infinite":
            assert (heads[:, :, 1] == INF).all() and torch.isfinite(heads[:, :, [0, 2, 3]]).all()
        else:
            assert torch.isnan(heads).all()


@pytest.mark.parametrize("layout", ["slots", "time"])
def test_layouts_strides_and_splits(ops, layout):
    c = Case4([(2, 1500, 4), (0, 900, 3)], 6, 3, 128, 64, layout=layout, gap=1)
    wide = torch.zeros(c.M, c.q.shape[1] + 24, dtype=BF16, device="cuda")
    wide[:, 4:4 + c.q.shape[1]] = c.q
    c.q = wide[:, 4:4 + 6 * 128]
    if layout == "slots":
        c.kc = torch.stack((c.kc, c.kc), 3)[:, :, :, 1]                     # every second head of a cache of twice as many
    large = torch.zeros(3, 5, c.cap, 2, dtype=BF16, device="cuda")[:, 1:4]  # scales that are part of something larger
    large.copy_(c.vs)
    c.vs = large
    for max_ctx in (0, 1, 600, 1504, 100000):
        c.check(c.run(ops, max_ctx=max_ctx, out=torch.full_like(c.out, 77.0)))


@pytest.mark.parametrize("n", [3, 50])
def test_caches_past_32_bits(ops, n):
    """Slots whose rows lie more than 2^32 bytes into the cache, and a history whose last positions do."""
    G, dim, cap, slots, p0 = 8, 128, 4_300_000, 2, 70
    kc, vc = (torch.empty(slots, cap, G * dim // 2, dtype=U8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(slots, G, cap, 4, dtype=BF16, device="cuda") for _ in range(2))
    small = Case4([(0, p0, n)], 16, G, dim, dim, slots=1)
    at = cap - p0 - n - 1
    for big, little in ((kc, small.kc), (vc, small.vc)):
        big[1, :p0 + n] = big[1, at:at + p0 + n] = little[0, :p0 + n].reshape(p0 + n, -1)
    for big, little in ((ks, small.ks), (vs, small.vs)):
        big[1, :, :p0 + n] = big[1, :, at:at + p0 + n] = little[0, :, :p0 + n]
    want = small.run(ops)
    small.check(want)
    out = torch.empty_like(want)
    ops.tree_attn(small.q, kc, vc, torch.tensor([(1, p0, 0, n)], dtype=torch.int32, device="cuda"), out, 16, G, dim, dim, small.scale, rows=n, max_ctx=p0 + n, k_scale=ks, v_scale=vs)
    assert torch.equal(out, want)
    ops.tree_attn(small.q, kc, vc, torch.tensor([(1, at + p0, 0, n)], dtype=torch.int32, device="cuda"), out, 16, G, dim, dim, small.scale, rows=n, max_ctx=at + p0 + n, window=60, k_scale=ks,
                  v_scale=vs)
    small.window = 60
    small.check(out)


def test_portions_that_do_not_fit(ops):
    for max_ctx in (0, 100000):
        c = Case4([(0, 30, 2), (1, 20, 3), (0, 5, 4)], 4, 2, 128, 128, slots=2, cap=600, gap=1)
        segs = list(c.segs)
        for change in ((2, 20, segs[1][2], 3), (-1, 20, segs[1][2], 3), (1, 598, segs[1][2], 3), (1, -1, segs[1][2], 3), (1, 2 ** 31 - 2, segs[1][2], 3)):
            c.segs = [segs[0], change, segs[2]]
            out = c.run(ops, max_ctx=max_ctx, out=torch.full_like(c.out, 77.0))
            assert torch.isnan(out[change[2]:change[2] + 3].float()).all()
            out[change[2]:change[2] + 3] = 77
            c.segs = [segs[0], segs[2]]
            c.check(out)


@pytest.mark.parametrize("n", [6, 40])
def test_replayed_on_another_stream_and_the_same_bits(ops, n):
    c = Case4([(2, 1700, n), (0, 800, n), (1, 0, n)], 8, 2, 128, 128)
    first = c.run(ops).clone()
    assert torch.equal(first, c.run(ops, out=torch.empty_like(first)))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = c.run(ops, out=torch.empty_like(first))
    torch.cuda.synchronize()
    assert torch.equal(first, second)
    segs, out = torch.tensor(c.segs, dtype=torch.int32, device="cuda"), torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.tree_attn(c.q, c.kc, c.vc, segs, out, 8, 2, 128, 128, c.scale, rows=n, max_ctx=1700 + n, k_scale=c.ks, v_scale=c.vs)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, out)
    c.segs = [(1, 1234, 0, n), (2, 5, n, n - 2), (0, 40, 2 * n - 2, n)]     # other lengths and slots in the captured call
    segs.copy_(torch.tensor(c.segs, dtype=torch.int32))
    c.q.copy_(rnd(*c.q.shape, seed=99))
    out.fill_(77.0)
    graph.replay()
    torch.cuda.synchronize()
    c.check(out)


@pytest.mark.parametrize("n", [5, 40])
def test_scales_of_any_size(ops, n):
    """Scales far apart from token to token, zeros among them, and queries and keys of extreme sizes."""
    c = Case4([(0, 300, n)], 4, 2, 128, 128)
    f = 2.0 ** torch.linspace(-60, 20, c.cap, device="cuda")
    c.vs.copy_(c.vs.float() * f[torch.randperm(c.cap, generator=torch.Generator("cuda").manual_seed(1), device="cuda")][None, None, :, None])
    c.vs[0, :, 3::7] = 0
    c.ks[0, :, ::9] *= 2.0 ** -30
    c.q[1] *= 2.0 ** -90
    c.ks[0, 1] *= 2.0 ** 40
    c.q[:, 256:] = (c.q[:, 256:].float() * 2.0 ** -40).to(BF16)
    c.check(c.run(ops))


@pytest.mark.parametrize("n", [5, 40])
def test_groups_of_unequal_scales(ops, n):
    """A group's scale may be 2^-9 of its head's largest, or nothing, and its channels are as exact as the others."""
    c = Case4([(0, 300, n)], 4, 2, 128, 64)
    c.vs[..., 1] *= 2.0 ** -9
    c.ks[..., 0] *= 2.0 ** -7
    c.ks[0, :, 7::5, 3] = 0
    c.vs[0, :, 2::5, 0] = 0
    c.check(c.run(ops))


@pytest.mark.parametrize("n,G,past", [(33, 56, 280), (130, 16, 200)])
def test_many_blocks_and_no_wait_runs_out(ops, n, G, past):
    seqs = 64
    kc, vc = (torch.randint(0, 256, (seqs, past + n, G * 64), dtype=torch.int16, generator=torch.Generator("cuda").manual_seed(s), device="cuda").to(U8) for s in (1, 2))
    ks, vs = ((torch.rand(seqs, G, past + n, 4, generator=torch.Generator("cuda").manual_seed(s), device="cuda") * 0.1 + 0.01).to(BF16) for s in (3, 4))
    q = rnd(seqs * n, G * 128, seed=5)
    segs = torch.tensor([(i, past - i, i * n, n) for i in range(seqs)], dtype=torch.int32, device="cuda")
    from lia_b200 import _lib
    before = _lib.load().lia_moe_timeouts()
    outs = [ops.tree_attn(q, kc, vc, segs, torch.empty_like(q), G, G, 128, 128, 128 ** -0.5, rows=n, max_ctx=past + n, k_scale=ks, v_scale=vs) for _ in range(12)]
    assert _lib.load().lia_moe_timeouts() == before
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("nseg", [9, 12, 18, 37])
def test_blocks_that_share_a_history(ops, nseg):
    c = Case4([(i, 2500 - 61 * (i % 30), 0 if i == 5 else 2) for i in range(nseg)], 16, 8, 64, 64)
    c.check(c.run(ops))


def test_many_zeros_before_the_first_value(ops):
    """Groups of zeros are stored with scales near 2^-103: sums of weights over scales stay finite, and values behind 40000 such tokens count."""
    z = 40000
    c = Case4([(0, z, 40)] * 150, 1, 1, 64, 64)
    c.q.zero_()
    c.vc[0, :z] = 0x88
    c.vs[0, 0, :z] = 2.0 ** -103
    out = c.run(ops)
    c.check(out)
    assert (out.float().abs().amax(1) > 0).all()


@pytest.mark.parametrize("dim,vdim", DIMS)
@pytest.mark.parametrize("n,past,max_ctx", [(1, 90, 91), (40, 30, 70), (40, 30, 100000), (200, 70, 270), (20, 1500, 1520)])
def test_outputs_on_8_byte_boundaries(ops, dim, vdim, n, past, max_ctx):
    c = Case4([(0, past, n), (1, past // 2, max(1, n - 3))], 4, 2, dim, vdim)
    want = c.run(ops, max_ctx=max_ctx).clone()
    c.check(want)
    buffer = torch.full((4 + want.numel() + 4,), 77.0, dtype=BF16, device="cuda")
    out = buffer[4:4 + want.numel()].view(want.shape)
    assert torch.equal(c.run(ops, max_ctx=max_ctx, out=out), want)
    assert (buffer[:4] == 77).all() and (buffer[-4:] == 77).all()


@pytest.mark.parametrize("H", [4, 8])
@pytest.mark.parametrize("max_ctx", [364, 100000])
def test_waits_that_run_out(nowait, monkeypatch, ops, H, max_ctx):  # noqa: F811
    """With a limit of 0 every wait gives up: launches end and are counted, and rows, formed key by key, are right all the same."""
    sizes = (64, 40, 33)
    c = Case4([(0, 300, sizes[0]), (1, 70, sizes[1]), (2, 5, sizes[2])], H, 2, 128, 64, mask=[family(n, lambda i: (i - 1) // 2 if i else -1) for n in sizes], gap=1)
    again = torch.full_like(c.out, 77.0)
    assert given_up(nowait, monkeypatch, lambda: c.run(ops, out=again, max_ctx=max_ctx)) >= 3 * 2
    torch.cuda.synchronize()
    c.check(again)
    c.check(c.run(ops, max_ctx=max_ctx))


@pytest.mark.parametrize("dim,vdim", DIMS)
@pytest.mark.parametrize("H,G,n,masked,window", [(8, 8, 1, False, 0), (16, 8, 1, False, 0), (32, 8, 2, False, 0), (8, 8, 8, True, 0), (16, 8, 4, True, 700), (24, 8, 1, False, 1500), (56, 56, 1, False, 0)])
def test_histories_of_unequal_lengths_in_equal_spans(ops, dim, vdim, H, G, n, masked, window):
    """Long histories of up to eight rows are cut into equal spans over all requests: spans that end one history and begin the next, portions of no tokens, a slot that is not there, histories of nothing,
    rows that see nothing; and the same bits again, and from a graph with other lengths in it."""
    past = [7003, 0, 64, 2000, 1, 12345, 63, 65, 300, 4097, 0]
    portions = [(i, p, 0 if i == 6 else max(1, n - i % 3)) for i, p in enumerate(past)]
    tree = lambda m: family(m, lambda i: (i - 1) // 2 if i else -1)  # noqa: E731
    deep = [[int(tree(m)[i].sum()) - 1 for i in range(m)] for _, _, m in portions] if masked else None
    c = Case4(portions, H, G, dim, vdim, mask=[tree(m) for _, _, m in portions] if masked else None, depth=deep, window=window, gap=1)
    if masked:
        c.mask[c.segs[10][2]] = 0                                           # without history: this row sees nothing
        c.sees[10][0] = False
    long = 3_000_000 // (G * len(portions)) * 2                             # enough for spans, whatever is there
    from lia_b200 import _lib
    assert _lib.load().lia_tree_attn_plan(len(portions), n, long, H, G, window, 3) >> 30 or window
    out = c.run(ops, rows=n, max_ctx=long).clone()
    c.check(out)
    assert torch.equal(out, c.run(ops, rows=n, max_ctx=long, out=torch.full_like(out, 77.0)))
    lost = c.segs[3]
    c.segs[3] = (99, *lost[1:])
    gone = c.run(ops, rows=n, max_ctx=long, out=torch.full_like(out, 77.0))
    assert torch.isnan(gone[lost[2]:lost[2] + lost[3]].float()).all()
    gone[lost[2]:lost[2] + lost[3]] = out[lost[2]:lost[2] + lost[3]]
    c.segs[3] = lost
    c.check(gone)
    segs, again = torch.tensor(c.segs, dtype=torch.int32, device="cuda"), torch.full_like(out, 77.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.tree_attn(c.q, c.kc, c.vc, segs, again, H, G, dim, vdim, c.scale, rows=n, max_ctx=long, mask=c.mask, depth=c.depth, window=window, k_scale=c.ks, v_scale=c.vs)
    order = torch.randperm(len(portions), generator=torch.Generator().manual_seed(1)).tolist()
    segs.copy_(torch.tensor([c.segs[i] for i in order], dtype=torch.int32))  # (in another order, spans are others: sums of the same numbers)
    graph.replay()
    torch.cuda.synchronize()
    c.check(again)
    segs.copy_(torch.tensor([(s, 0, r, 0) for s, _, r, _ in c.segs], dtype=torch.int32))      # nothing at all
    again.fill_(77.0)
    graph.replay()
    torch.cuda.synchronize()
    assert (again == 77).all()


@pytest.mark.parametrize("n", [1, 4])
def test_weights_that_average_out(ops, n):
    """40000 keys of nearly equal weight: what their values average out to is a hundredth of the values, and as exact."""
    c = Case4([(0, 40000, n), (1, 39000, n)], 4, 2, 128, 128)
    c.q *= 0.02
    c.check(c.run(ops))
    c.check(c.run(ops, max_ctx=4_000_000))
