"""Attention of drafted tokens behind a history, against 64 bits.

How far an output may be off, for a row whose weights p give o = sum p v and A = sum p |v|: the output's own rounding, 2^-8 of it (bf16); weights in fp16 (8-bit caches), 2^-11 of A, or
in two bf16 parts, 2^-16 of A; more than 32 rows of a key head also have values of 8 bits multiplied by their scales in fp16, 2^-11 for the factor and 2^-11 for the product; and a score that is off by d puts a weight, and the sum of weights, off by d of itself: 2 d of A.  A score's sum of products of `dim` numbers is off by at most
dim 2^-24 of B, its largest sum of magnitudes; factors, the cap and the two powers' approximations add 2^-21 of the score's size S and 2^-20."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
KINDS = {"bf16": BF16, "int8": torch.int8, "e4m3": E4M3}
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def ops():
    import lia_b200
    from lia_b200 import ops
    return ops


def rnd(*shape, seed=0, std=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda") * std).to(dtype)


class Case:
    """Portions (slot, p0, n) over caches whose other rows hold numbers of their own; masks by token: the tokens of the portion that it sees."""

    def __init__(self, portions, H, G, dim, vdim, kind, slots=None, cap=None, layout="slots", mask=None, depth=None, window=0, softcap=0.0, temp=False, gap=0, seed=0, words=None):
        self.H, self.G, self.dim, self.vdim, self.window, self.softcap = H, G, dim, vdim, window, softcap
        self.slots, self.cap = slots or max(p[0] for p in portions) + 1, cap or max(p[1] + p[2] for p in portions) + 3
        self.segs, row = [], gap
        for s, p0, n in portions:
            self.segs.append((s, p0, row, n))
            row += n + gap
        self.M = row
        self.q = rnd(self.M, H * dim, seed=seed + 1, std=1.4)
        lay = (self.cap, self.slots) if layout == "time" else (self.slots, self.cap)
        k, v = rnd(*lay, G, dim, seed=seed + 2), rnd(*lay, G, vdim, seed=seed + 3)
        self.ks = self.vs = None
        if kind == "bf16":
            self.kc, self.vc = k, v
        else:
            self.kc, self.ks = self.codes(k, kind, seed + 4)
            self.vc, self.vs = self.codes(v, kind, seed + 5)
        if layout == "time":
            self.kc, self.vc = self.kc.permute(1, 0, 2, 3), self.vc.permute(1, 0, 2, 3)
        self.temp = rnd(H, seed=seed + 6, std=0.2, dtype=F32) + 1 if temp else None
        self.scale = dim ** -0.5
        self.sees = mask                                                    # per portion: bool [n, n], or None
        self.mask = None
        if mask is not None:
            words = words or max((n + 63) // 64 for _, _, n in portions) or 1
            self.mask = torch.zeros(self.M, words, dtype=torch.int64)
            for (s, p0, r, n), m in zip(self.segs, mask):
                for i in range(n):
                    for j in range(n):
                        if m[i, j]:
                            self.mask[r + i, j >> 6] |= 1 << (j & 63) if j & 63 != 63 else -(1 << 63)
            self.mask = self.mask.cuda()
        self.depth = None
        if depth is not None:
            self.depth = torch.zeros(self.M, dtype=torch.int32)
            for (s, p0, r, n), d in zip(self.segs, depth):
                self.depth[r:r + n] = torch.tensor(d[:n], dtype=torch.int32)
            self.depth = self.depth.cuda()
        self.out = torch.full((self.M, H * vdim), 77.0, dtype=BF16, device="cuda")

    def codes(self, x, kind, seed):
        a = x.float().abs().amax(-1) * (1 + torch.rand(x.shape[:-1], generator=torch.Generator("cuda").manual_seed(seed), device="cuda"))
        s = a / (127 if kind == "int8" else 448)
        c = x.float() / s[..., None]
        c = torch.round(c).to(torch.int8) if kind == "int8" else c.to(E4M3)
        # scales [slots, G, capacity] from [.., .., G]
        return c, (s.permute(0, 2, 1) if c.shape[0] == self.slots and c.shape[1] == self.cap else s.permute(1, 2, 0)).contiguous()

    def run(self, ops, max_ctx=None, rows=None, out=None):
        out = self.out if out is None else out
        return ops.tree_attn(self.q, self.kc, self.vc, torch.tensor(self.segs, dtype=torch.int32, device="cuda"), out, self.H, self.G, self.dim, self.vdim, self.scale,
                             rows=max(s[3] for s in self.segs) if rows is None else rows, max_ctx=max(s[1] + s[3] for s in self.segs) if max_ctx is None else max_ctx, mask=self.mask,
                             depth=self.depth, temp=self.temp, window=self.window, softcap=self.softcap, k_scale=self.ks, v_scale=self.vs)

    def visible(self, z):
        s, p0, r, n = self.segs[z]
        t, i = torch.arange(p0 + n, device="cuda"), torch.arange(n, device="cuda")
        d = self.depth[r:r + n].long() if self.depth is not None else i
        near = t[None] > (p0 + d)[:, None] - (self.window if self.window > 0 else 1 << 40)
        if self.sees is None:
            return (t[None] <= p0 + i[:, None]) & near
        see = near.clone()
        see[:, p0:] = self.sees[z].cuda()
        return see

    def check(self, out, kind):
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
                k, v = kc[s, :p0 + n, g].double(), vc[s, :p0 + n, g].double()
                if self.ks is not None:
                    k, v = k * self.ks[s, g, :p0 + n, None].double(), v * self.vs[s, g, :p0 + n, None].double()
                q = self.q[r:r + n, h * self.dim:(h + 1) * self.dim].double()
                f = self.scale * (float(self.temp[h]) if self.temp is not None else 1.0)
                x, size = q @ k.t() * f, q.abs() @ k.abs().t() * abs(f)
                if self.softcap:
                    x = self.softcap * torch.tanh(x / self.softcap)
                x = x.masked_fill(~see, -INF)
                some = see.any(1, keepdim=True)
                p = torch.where(some, torch.softmax(x, -1), torch.zeros_like(x))
                vz = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
                o, A = p @ vz, p @ vz.abs()
                seen = torch.where(see, size, torch.zeros_like(size))
                B = torch.nan_to_num(seen, 0, 0, 0).amax(1, keepdim=True)
                S = torch.where(see, torch.nan_to_num(x, 0, 0, 0).abs(), torch.zeros_like(x)).amax(1, keepdim=True)
                d = self.dim * 2.0 ** -24 * B + 2.0 ** -21 * (S + self.softcap) + 2.0 ** -20
                tol = 2.0 ** -8 * o.abs() + ((2.0 ** -16 if kind == "bf16" else 3 * 2.0 ** -11 if many else 2.0 ** -11) + 2 * d) * A + 1e-30
                got = out[r:r + n, h * self.vdim:(h + 1) * self.vdim].double()
                bad = ((got - o).abs() > tol) | torch.isnan(got)
                assert not bad.any(), (z, h, bad.nonzero()[:4].tolist(), (got - o).abs().max().item(), ((got - o).abs() / tol).max().item())
        assert (out[~touched] == 77).all(), "rows of no portion"


def family(n, parents):
    m = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        j = i
        while j >= 0:
            m[i, j] = True
            j = parents(j)
    return m


DIMS = [(128, 128), (64, 64), (128, 64), (64, 128)]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dim,vdim", DIMS)
@pytest.mark.parametrize("H,G", [(4, 4), (6, 2), (16, 1)])
def test_single_tokens(ops, kind, dim, vdim, H, G):
    """Histories from none to several blocks of keys, around their borders."""
    portions = [(i, p0, 1) for i, p0 in enumerate((0, 1, 14, 15, 16, 17, 63, 64, 255, 256, 1000))]
    c = Case(portions, H, G, dim, vdim, kind)
    c.check(c.run(ops), kind)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("H,G,n", [(3, 3, 2), (4, 4, 16), (4, 4, 17), (2, 2, 33), (2, 2, 64), (8, 2, 5), (8, 2, 29), (5, 1, 13), (32, 2, 9)])
def test_chains_behind_ragged_histories(ops, kind, H, G, n):
    c = Case([(2, 700, n), (0, 0, n), (1, 37, max(1, n - 1)), (3, 16, 1)], H, G, 128, 128, kind, gap=2)
    c.check(c.run(ops), kind)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dim,vdim", DIMS)
@pytest.mark.parametrize("n,branch", [(2, 1), (7, 2), (29, 2), (40, 3), (64, 3), (65, 2), (130, 4)])
def test_trees(ops, kind, dim, vdim, n, branch):
    parents = lambda i: (i - 1) // branch if i else -1  # noqa: E731
    c = Case([(0, 333, n), (2, 0, n), (1, 48, max(1, n // 2))], 4, 2, dim, vdim, kind, mask=[family(n, parents), family(n, parents), family(max(1, n // 2), parents)], softcap=20.0, temp=True)
    c.check(c.run(ops), kind)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("window", [1, 2, 16, 100, 5000])
@pytest.mark.parametrize("masked", [False, True])
def test_windows(ops, kind, window, masked):
    n = 21
    tree = family(n, lambda i: (i - 1) // 2 if i else -1)
    deep = [int(tree[i].sum()) - 1 for i in range(n)]
    c = Case([(1, 500, n), (0, 3, n), (2, 0, 5)], 6, 3, 128, 128, kind, mask=[tree, tree, tree[:5, :5]] if masked else None, depth=[deep, deep, deep] if masked else None, window=window)
    c.check(c.run(ops), kind)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("window", [0, 90])
def test_portions_of_prompts(ops, kind, window):
    c = Case([(1, 130, 301), (0, 0, 257), (2, 64, 1)], 4, 2, 128, 128, kind, window=window)
    c.check(c.run(ops), kind)


@pytest.mark.parametrize("kind", list(KINDS))
def test_any_mask_and_rows_that_see_nothing(ops, kind):
    """Masks need not be trees: a token may not see itself, or sees later ones; without history a row may see nothing at all.  Bits behind a portion's tokens mean nothing."""
    g = torch.Generator().manual_seed(3)
    masks = [torch.rand(n, n, generator=g) < 0.3 for n in (11, 70, 1, 3)]
    masks[0][4] = False
    masks[1][69] = False
    masks[2][0] = False
    c = Case([(0, 0, 11), (1, 0, 70), (2, 0, 1), (3, 20, 3)], 4, 4, 64, 64, kind, mask=masks, words=3)
    c.mask[:, 2] = -1
    c.mask[c.segs[0][2]:c.segs[0][2] + 11, 0] |= -1 << 11
    out = c.run(ops)
    c.check(out, kind)
    assert (out[c.segs[0][2] + 4] == 0).all() and (out[c.segs[2][2]] == 0).all()


@pytest.mark.parametrize("kind", list(KINDS))
def test_what_a_row_does_not_see_has_no_effect(ops, kind):
    """Infinities and NaN in keys, values and scales of tokens that some rows see and others do not, in rows of the cache behind the portions and in other slots."""
    n, p0, H, G = 12, 40, 4, 2
    tree = family(n, lambda i: (i - 1) // 2 if i else -1)
    c = Case([(1, p0, n)], H, G, 128, 128, kind, mask=[tree], slots=3, cap=p0 + n + 20)
    clean = c.run(ops).clone()
    c.check(clean, kind)
    for what in ("behind", "other slots", "value NaN", "value inf", "key NaN", "scale"):
        spoiled = Case([(1, p0, n)], H, G, 128, 128, kind, mask=[tree], slots=3, cap=p0 + n + 20)
        bad = 5                                                             # seen by itself and its children 11, (12)
        hit = [i for i in range(n) if tree[i, bad]]
        kc, vc = spoiled.kc.view(torch.uint8) if kind != "bf16" else spoiled.kc, spoiled.vc.view(torch.uint8) if kind != "bf16" else spoiled.vc
        nan = 0x7f if kind == "e4m3" else 1 if kind == "int8" else NAN
        if what == "behind":
            kc[1, p0 + n:], vc[1, p0 + n:] = nan, nan
            if kind != "bf16":
                spoiled.ks[1, :, p0 + n:], spoiled.vs[1, :, p0 + n:] = NAN, NAN
            hit = []
        elif what == "other slots":
            for s in (0, 2):
                kc[s], vc[s] = nan, nan
                if kind != "bf16":
                    spoiled.ks[s], spoiled.vs[s] = NAN, INF
            hit = []
        elif what == "scale":
            if kind == "bf16":
                continue
            spoiled.vs[1, :, p0 + bad], spoiled.ks[1, :, p0 + bad] = NAN, INF
        elif kind == "int8":
            continue                                                        # (its codes are finite)
        elif what == "value NaN":
            vc[1, p0 + bad] = nan
        elif what == "value inf":
            if kind == "e4m3":
                spoiled.vs[1, :, p0 + bad] = INF
            else:
                vc[1, p0 + bad] = INF
        else:
            kc[1, p0 + bad] = nan
        out = spoiled.run(ops)
        rest = [i for i in range(n) if i not in hit]
        # rows formed key by key are rounded elsewhere: a step of bf16 at most, and a hair
        assert ((out[rest].double() - clean[rest].double()).abs() <= 2.0 ** -7 * clean[rest].double().abs() + 2.0 ** -9).all(), what
        assert not torch.isfinite(out[hit].float()).any(1).any() if hit and what != "value inf" else torch.isfinite(out[rest].float()).all(), what


def test_scores_of_minus_infinity(ops):
    """Keys of -inf are of no weight; a row that sees nothing else is NaN, as the formula is."""
    c = Case([(0, 10, 1), (1, 3, 1)], 2, 2, 64, 64, "bf16")
    c.q.abs_()
    c.kc[0, 4:8] = -INF
    c.kc[1] = -INF
    out = c.run(ops)
    assert torch.isnan(out[1].float()).all()
    c.segs = c.segs[:1]
    k = c.kc.clone()
    keep = [t for t in range(11) if not 4 <= t < 8]
    c.kc[0, :len(keep)], c.vc[0, :len(keep)] = k[0, keep], c.vc[0, keep].clone()
    c.segs = [(0, 6, 0, 1)]
    again = c.run(ops, out=torch.full_like(c.out, 77.0))
    assert ((again[0].double() - out[0].double()).abs() <= 2.0 ** -7 * out[0].double().abs() + 2.0 ** -12).all()


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("layout", ["slots", "time"])
def test_layouts_strides_and_splits(ops, kind, layout):
    """Time-major caches (seen request by request), a head stride of its own, queries that are columns of something wider; however many blocks share a history, the result is right."""
    c = Case([(2, 1500, 4), (0, 900, 3)], 6, 3, 128, 64, kind, layout=layout, gap=1)
    wide = torch.zeros(c.M, c.q.shape[1] + 24, dtype=BF16, device="cuda")
    wide[:, 4:4 + c.q.shape[1]] = c.q
    c.q = wide[:, 4:4 + 6 * 128]
    if layout == "slots":                                                   # every second head of a cache of twice as many
        both = torch.stack((c.kc, c.kc), 3) if c.kc.dtype != E4M3 else torch.stack((c.kc.view(torch.uint8),) * 2, 3).view(E4M3)
        c.kc = both[:, :, :, 1]
    for max_ctx in (0, 1, 600, 1504, 100000):
        out = c.run(ops, max_ctx=max_ctx, out=torch.full_like(c.out, 77.0))
        c.check(out, kind)


@pytest.mark.parametrize("kind", ["int8", "bf16"])
def test_caches_past_32_bits(ops, kind):
    """Slots whose rows lie more than 2^32 bytes into the cache."""
    G, dim, cap, slots, p0, n = 8, 128, (2_200_000 if kind == "int8" else 1_100_000), 2, 70, 3
    kc, vc = (torch.empty(slots, cap, G * dim, dtype=KINDS[kind], device="cuda") for _ in range(2))
    small = Case([(0, p0, n)], 16, G, dim, dim, kind, slots=1)
    at = cap - p0 - n - 1
    ks = vs = None
    kc[1, :p0 + n], vc[1, :p0 + n] = small.kc[0, :p0 + n].view(p0 + n, -1), small.vc[0, :p0 + n].view(p0 + n, -1)
    if kind == "int8":
        ks, vs = torch.empty(slots, G, cap, device="cuda"), torch.empty(slots, G, cap, device="cuda")
        ks[1, :, :p0 + n], vs[1, :, :p0 + n] = small.ks[0, :, :p0 + n], small.vs[0, :, :p0 + n]
    want = small.run(ops)
    small.check(want, kind)
    out = torch.empty_like(want)
    segs = torch.tensor([(1, p0, 0, n)], dtype=torch.int32, device="cuda")
    ops.tree_attn(small.q, kc, vc, segs, out, 16, G, dim, dim, small.scale, rows=n, max_ctx=p0 + n, k_scale=ks, v_scale=vs)
    assert torch.equal(out, want)
    # and a history whose own last positions lie there, seen through a window
    kc[1, at:at + p0 + n], vc[1, at:at + p0 + n] = kc[1, :p0 + n].clone(), vc[1, :p0 + n].clone()
    if kind == "int8":
        ks[1, :, at:at + p0 + n], vs[1, :, at:at + p0 + n] = ks[1, :, :p0 + n].clone(), vs[1, :, :p0 + n].clone()
    segs = torch.tensor([(1, at + p0, 0, n)], dtype=torch.int32, device="cuda")
    ops.tree_attn(small.q, kc, vc, segs, out, 16, G, dim, dim, small.scale, rows=n, max_ctx=at + p0 + n, window=60, k_scale=ks, v_scale=vs)
    small.window = 60
    small.check(out, kind)


@pytest.mark.parametrize("kind", list(KINDS))
def test_portions_that_do_not_fit(ops, kind):
    """A slot that is not there, positions past the capacity, more tokens than the launch was told of: NaN rows, and the others are right."""
    for max_ctx in (0, 100000):
        c = Case([(0, 30, 2), (1, 20, 3), (0, 5, 4)], 4, 2, 128, 128, kind, slots=2, cap=600, gap=1)
        segs = list(c.segs)
        for z, change in ((1, (2, 20, segs[1][2], 3)), (1, (-1, 20, segs[1][2], 3)), (1, (1, 598, segs[1][2], 3)), (1, (1, -1, segs[1][2], 3)), (1, (1, 2 ** 31 - 2, segs[1][2], 3))):
            bad = list(segs)
            bad[z] = change
            c.segs = bad
            out = c.run(ops, max_ctx=max_ctx, out=torch.full_like(c.out, 77.0))
            r, n = change[2], change[3]
            assert torch.isnan(out[r:r + n].float()).all()
            kept = out.clone()
            kept[r:r + n] = 77
            c.segs = [s for i, s in enumerate(segs) if i != z]
            c.check(kept, kind)
        c.segs = segs
        out = c.run(ops, rows=3, max_ctx=max_ctx, out=torch.full_like(c.out, 77.0))      # the third has four
        assert torch.isnan(out[segs[2][2]:segs[2][2] + 4].float()).all() and torch.isfinite(out[segs[1][2]:segs[1][2] + 3].float()).all()
        c.segs = segs[:2] + [(0, 5, c.M - 2, 4)]                                         # rows that are not there
        out = c.run(ops, max_ctx=max_ctx, out=torch.full_like(c.out, 77.0))
        assert torch.isnan(out[c.M - 2:].float()).all()


def test_nothing_to_do(ops):
    c = Case([(0, 5, 2), (1, 3, 0)], 2, 2, 64, 64, "int8")
    c.check(c.run(ops), "int8")                                             # a portion of no tokens
    out = ops.tree_attn(c.q[:0], c.kc, c.vc, torch.empty(0, 4, dtype=torch.int32, device="cuda"), c.out[:0], 2, 2, 64, 64, 1.0, rows=0, max_ctx=0, k_scale=c.ks, v_scale=c.vs)
    assert out.shape == (0, 128)


@pytest.mark.parametrize("kind", list(KINDS))
def test_replayed_on_another_stream_and_the_same_bits(ops, kind):
    c = Case([(2, 1700, 6), (0, 800, 6), (1, 0, 6)], 8, 2, 128, 128, kind)
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
        ops.tree_attn(c.q, c.kc, c.vc, segs, out, 8, 2, 128, 128, c.scale, rows=6, max_ctx=1706, k_scale=c.ks, v_scale=c.vs)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, out)
    c.segs = [(1, 1234, 0, 6), (2, 5, 6, 4), (0, 40, 10, 6)]               # other lengths and slots in the captured call
    segs.copy_(torch.tensor(c.segs, dtype=torch.int32))
    c.q.copy_(rnd(*c.q.shape, seed=99))
    out.fill_(77.0)
    graph.replay()
    torch.cuda.synchronize()
    c.check(out, kind)


def test_portions_anywhere_in_a_buffer(ops):
    """The engine's portions lie in one buffer with ids and positions, on 4-byte boundaries."""
    c = Case([(1, 100, 3), (0, 50, 2)], 4, 2, 64, 128, "int8")
    want = c.run(ops).clone()
    buffer = torch.zeros(11, dtype=torch.int32, device="cuda")
    segs = buffer[3:11].view(2, 4)
    segs.copy_(torch.tensor(c.segs, dtype=torch.int32))
    out = ops.tree_attn(c.q, c.kc, c.vc, segs, torch.empty_like(want), 4, 2, 64, 128, c.scale, rows=3, max_ctx=103, k_scale=c.ks, v_scale=c.vs)
    assert torch.equal(want, out)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_scales_of_any_size(ops, kind):
    """Scales far apart, zeros among them (a value of nothing still takes its share of the weights), and queries and keys of extreme sizes."""
    c = Case([(0, 300, 5)], 4, 2, 128, 128, kind)
    f = 2.0 ** torch.linspace(-60, 20, c.cap, device="cuda")
    c.vs *= f[torch.randperm(c.cap, generator=torch.Generator("cuda").manual_seed(1), device="cuda")]
    c.vs[0, :, 3::7] = 0
    c.ks[0, :, ::9] *= 2.0 ** -30
    c.q[1] *= 2.0 ** -90
    c.ks[0, 1] *= 2.0 ** 40
    c.q[:, 256:] = (c.q[:, 256:].float() * 2.0 ** -40).to(BF16)
    c.check(c.run(ops), kind)


def test_a_drafted_tree_from_store_to_acceptance(ops):
    """The operators as they are used: a prompt goes into an 8-bit cache, a tree of drafted tokens behind it, one attention verifies them, their logits are scored; the accepted path's rows move
    up and the next single token sees what it would have seen without drafting."""
    H, G, dim, V, p0, n = 8, 2, 64, 997, 150, 12
    for kind in ("int8", "e4m3"):
        kc, vc = (torch.zeros(2, 256, G * dim, dtype=torch.uint8, device="cuda").view(KINDS[kind]) for _ in range(2))
        ks, vs = (torch.zeros(2, G, 256, device="cuda") for _ in range(2))
        k, v = rnd(p0 + n, G * dim, seed=1), rnd(p0 + n, G * dim, seed=2)
        meta = torch.tensor([(1, t) for t in range(p0 + n)], dtype=torch.int32, device="cuda")
        ops.kv_store_8bit(k[:p0], v[:p0], meta[:p0], kc, vc, ks, vs, G, dim, dim)                     # the prompt
        ops.kv_store_8bit(k[p0:], v[p0:], meta[p0:], kc, vc, ks, vs, G, dim, dim)                     # the drafted tree
        tree = family(n, lambda i: (i - 1) // 2 if i else -1)
        c = Case([(1, p0, n)], H, G, dim, dim, kind, slots=2, cap=256, mask=[tree])
        c.kc, c.vc, c.ks, c.vs = kc, vc, ks, vs
        out = c.run(ops)
        c.check(out, kind)
        logits = out.float() @ rnd(H * dim, V, seed=4, std=0.1, dtype=F32)
        tokens = torch.randint(0, V, (n, 2), generator=torch.Generator("cuda").manual_seed(5), device="cuda")
        logp, entropy, best, ids = ops.token_logprobs(logits, tokens, top=4)
        want = torch.log_softmax(logits.double(), -1)
        assert ((logp - want.gather(1, tokens)).abs() < 2.0 ** -14).all() and torch.equal(ids[:, 0], logits.argmax(-1))
        path = [0, 2, 5, 11]                                                                          # accepted: moved up behind the history
        for t in (kc, vc):
            t.view(torch.uint8)[1, p0:p0 + 4] = t.view(torch.uint8)[1, [p0 + j for j in path]]
        for t in (ks, vs):
            t[1, :, p0:p0 + 4] = t[1, :, [p0 + j for j in path]]
        q = rnd(1, H * dim, seed=9)
        one = ops.tree_attn(q, kc, vc, torch.tensor([(1, p0 + 3, 0, 1)], dtype=torch.int32, device="cuda"), torch.empty(1, H * dim, dtype=BF16, device="cuda"), H, G, dim, dim, dim ** -0.5,
                            rows=1, max_ctx=p0 + 4, k_scale=ks, v_scale=vs)
        plain = [torch.zeros_like(x) for x in (kc.view(torch.uint8), vc.view(torch.uint8))]
        pk, pv = (x.view(KINDS[kind]) for x in plain)
        pks, pvs = torch.zeros_like(ks), torch.zeros_like(vs)
        rows = list(range(p0)) + [p0 + j for j in path]
        ops.kv_store_8bit(k[rows], v[rows], meta[:p0 + 4], pk, pv, pks, pvs, G, dim, dim)
        two = ops.tree_attn(q, pk, pv, torch.tensor([(1, p0 + 3, 0, 1)], dtype=torch.int32, device="cuda"), torch.empty(1, H * dim, dtype=BF16, device="cuda"), H, G, dim, dim, dim ** -0.5,
                            rows=1, max_ctx=p0 + 4, k_scale=pks, v_scale=pvs)
        assert torch.equal(one, two)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("n,G,past", [(33, 56, 280), (130, 16, 200)])
def test_many_blocks_and_no_wait_runs_out(ops, kind, n, G, past):
    """Thousands of blocks of few steps each, over and over: every hand-over between a block's warps happens, the same bits come out, and no bounded wait has run out (a row whose block gave
    one up is formed key by key, so that the result alone would not tell)."""
    seqs = 64
    kc, vc = (rnd(seqs, past + n, G, 128, seed=s) for s in (1, 2))
    ks = vs = None
    if kind != "bf16":
        kc, vc = ((x.float() * 20).to(torch.int8) if kind == "int8" else x.to(E4M3) for x in (kc, vc))
        ks, vs = (torch.rand(seqs, G, past + n, generator=torch.Generator("cuda").manual_seed(s), device="cuda") * 0.1 + 0.01 for s in (3, 4))
    q = rnd(seqs * n, G * 128, seed=5)
    segs = torch.tensor([(i, past - i, i * n, n) for i in range(seqs)], dtype=torch.int32, device="cuda")
    from lia_b200 import _lib
    before = _lib.load().lia_moe_timeouts()
    outs = [ops.tree_attn(q, kc, vc, segs, torch.empty_like(q), G, G, 128, 128, 128 ** -0.5, rows=n, max_ctx=past + n, k_scale=ks, v_scale=vs) for _ in range(12)]
    assert _lib.load().lia_moe_timeouts() == before
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("nseg", [9, 10, 12, 14, 18, 24, 37, 75])
def test_blocks_that_share_a_history(ops, kind, nseg):
    """One to eight blocks of a cluster, whichever the number of requests leaves room for, with portions of no tokens and of slots that are not there among them."""
    portions = [(i, 2500 - 61 * (i % 30), 0 if i == 5 else 2) for i in range(nseg)]
    c = Case(portions, 16, 8, 64, 64, kind)
    c.check(c.run(ops), kind)
    lost = c.segs[3]
    c.segs[3] = (nseg + 7, *lost[1:])
    out = c.run(ops, out=torch.full_like(c.out, 77.0))
    assert torch.isnan(out[lost[2]:lost[2] + 2].float()).all()
    out[lost[2]:lost[2] + 2] = 77.0
    del c.segs[3]
    c.check(out, kind)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_many_zeros_before_the_first_value(ops, kind):
    """A head of zeros is stored with a scale near 2^-107: sums of weights over scales stay finite, and values behind 40000 such tokens count."""
    z = 40000
    c = Case([(0, z, 40)] * 150, 1, 1, 64, 64, kind)
    c.q.zero_()
    c.vc.view(torch.uint8)[0, :z] = 0
    c.vs[0, 0, :z] = 2.0 ** -107
    out = c.run(ops)
    c.check(out, kind)
    assert (out.float().abs().amax(1) > 0).all()


def test_a_capacity_whose_positions_do_not_fit(ops):
    from lia_b200._lib import LiaError
    far = torch.zeros(1, 1, 64, dtype=BF16, device="cuda").expand(1, (1 << 29) + 1, 64)
    q = torch.zeros(1, 64, dtype=BF16, device="cuda")
    with pytest.raises(LiaError):
        ops.tree_attn(q, far, far, torch.zeros(1, 4, dtype=torch.int32, device="cuda"), torch.empty_like(q), 1, 1, 64, 64, 1.0, rows=1, max_ctx=1)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("H,n", [(2, 1), (2, 9), (2, 40), (8, 40)])
def test_depths_behind_the_window(ops, kind, H, n):
    """Without a mask, tokens whose depth is so far behind that their window ends before the keys do see nothing, whether or not others of the call see something."""
    c = Case([(0, 4000, n), (1, 300, n), (0, 10, n)], H, 2, 64, 128, kind, depth=[[1000 + i for i in range(n)], list(range(n)), [60 + 2 * i for i in range(n)]], window=50)
    out = c.run(ops)
    c.check(out, kind)
    assert (out[:n] == 0).all()


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dim,vdim", DIMS)
@pytest.mark.parametrize("n,past,max_ctx", [(1, 90, 91), (40, 30, 70), (40, 30, 100000), (200, 70, 270), (20, 1500, 1520)])
def test_outputs_on_8_byte_boundaries(ops, kind, dim, vdim, n, past, max_ctx):
    """Part of a buffer that begins four numbers into it: the same bits, and nothing beside them, whichever kernel takes the rows."""
    c = Case([(0, past, n), (1, past // 2, max(1, n - 3))], 4, 2, dim, vdim, kind)
    want = c.run(ops, max_ctx=max_ctx).clone()
    c.check(want, kind)
    buffer = torch.full((4 + want.numel() + 4,), 77.0, dtype=BF16, device="cuda")
    out = buffer[4:4 + want.numel()].view(want.shape)
    assert out.data_ptr() % 16 == 8
    assert torch.equal(c.run(ops, max_ctx=max_ctx, out=out), want)
    assert (buffer[:4] == 77).all() and (buffer[-4:] == 77).all()
