"""Keys and values in 8 bits: codes and scales against the definition in 64 bits, and what is read back.

bf16 numbers make the definition exact: 127 x and the powers of two are, and a quotient of two numbers of 8 and 15 bits is either a tie or further than 2^-20 of itself from one, so
the correctly rounded 32-bit quotient rounds as the exact one does.  Codes of fp32 numbers may differ where the exact quotient is within 2^-20 of a border, codes of normed values too.

A normed value: a lane's 8 squares and five steps that join the lanes are 13 roundings of the sum, of which the root takes half (6.5 times 2^-24); the mean and eps are two more (1); the root, its
inverse, the product and the scale's quotient four (4): 11.5 times 2^-24 of itself, below 2^-20."""
import pytest
import torch

pytestmark = pytest.mark.gpu
E4M3, BF16, F32, F64 = torch.float8_e4m3fn, torch.bfloat16, torch.float32, torch.float64
LEAST = 2.0 ** -100


@pytest.fixture(scope="module")
def ops():
    import lia_b200
    from lia_b200 import ops
    return ops


def rnd(*shape, seed=0, std=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda") * std).to(dtype)


def codes_of(x, kind):
    """x [rows, heads, dim] float64 -> (the number that a code is before it is rounded, scale in 64 bits); none of e4m3 becomes 2^128"""
    a = x.abs().amax(-1, keepdim=True).clamp(min=LEAST)
    if kind == torch.int8:
        return x * 127 / a, (a / 127)[..., 0]
    m, e = torch.frexp(a)
    scale = torch.ldexp(torch.ones_like(a), e - 9 + (m > 0.875).to(e.dtype))
    most = torch.where(scale == 2.0 ** 120, 240.0, 448.0)
    return torch.minimum(torch.maximum(x / scale, -most), most), scale[..., 0]


def rounded(y, kind):
    if kind == torch.int8:
        return torch.round(y)
    grain = torch.ldexp(torch.ones_like(y), torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
    return torch.round(y / grain) * grain


def caches(slots, cap, G, dim, kind, layout="slots"):
    if layout == "time":
        c = torch.full((cap, slots, G, dim), 7, dtype=torch.uint8, device="cuda").view(kind).permute(1, 0, 2, 3)
    else:
        c = torch.full((slots, cap, G * dim), 7, dtype=torch.uint8, device="cuda").view(kind)
    return c, torch.full((slots, G, cap), -3.0, device="cuda")


def check_codes(cache, scale, x, meta, G, kind, exact, what, normed=False):
    y, s = codes_of(x, kind)
    slot, pos = meta.long().unbind(1)
    got = cache.view(torch.uint8)[slot, pos].view(kind).double().view(len(meta), G, -1)
    got_s = scale[slot, :, pos].double()
    if kind == E4M3:
        same = got_s == s
        assert same.all() if exact else same.double().mean() > 0.999, what            # (the largest may lie within 2^-20 of 448 times a power of two)
        y = y * (s / got_s)[..., None]
    else:
        assert ((got_s - s).abs() <= (2.0 ** -20 if normed else 2.0 ** -24) * s).all(), what
    want = rounded(y, kind)
    if exact:
        assert torch.equal(got, want), (what, (got != want).sum())
        return
    off = got != want
    border = torch.minimum((rounded(y * (1 + 2.0 ** -20), kind) - want).abs(), torch.ones_like(y) * 1e9) + (rounded(y * (1 - 2.0 ** -20), kind) - want).abs()
    assert (border[off] > 0).all(), (what, off.sum())


@pytest.mark.parametrize("kind", [torch.int8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("act,M,G,dim,vdim,layout,norm", [
    (BF16, 1, 1, 128, 128, "slots", False), (BF16, 37, 8, 128, 64, "time", False), (F32, 37, 3, 64, 128, "slots", False), (BF16, 5, 2, 8, 40, "slots", False),
    (BF16, 9, 3, 256, 264, "slots", False), (F32, 9, 2, 1024, 520, "time", False), (BF16, 130, 8, 128, 128, "slots", True), (F32, 70, 5, 72, 96, "time", True)])
def test_store_and_load(ops, kind, act, M, G, dim, vdim, layout, norm):
    slots, cap, eps = 3, M + 11, 1e-6
    g = torch.Generator().manual_seed(M)
    place = torch.randperm(slots * cap, generator=g)[:M]
    meta = torch.stack((place // cap, place % cap), 1).to(torch.int32).cuda()
    k, v = rnd(M, G * dim, seed=1, std=1.7, dtype=act), rnd(M, G * vdim, seed=2, std=0.3, dtype=act)
    k[:, ::5] *= 20
    kc, ks = caches(slots, cap, G, dim, kind, layout)
    vc, vs = caches(slots, cap, G, vdim, kind, layout)
    before = [x.clone() for x in (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)]
    ops.kv_store_8bit(k, v, meta, kc, vc, ks, vs, G, dim, vdim, eps=eps, norm_values=norm)
    x = v.double().view(M, G, vdim)
    check_codes(kc, ks, k.double().view(M, G, dim), meta, G, kind, act == BF16, "keys")
    check_codes(vc, vs, x / (x.square().mean(-1, keepdim=True) + eps).sqrt() if norm else x, meta, G, kind, act == BF16 and not norm, "values", norm)
    # no other place has changed
    used = torch.zeros(slots, cap, dtype=torch.bool, device="cuda")
    used[meta[:, 0].long(), meta[:, 1].long()] = True
    for now, old in zip((kc.view(torch.uint8), vc.view(torch.uint8)), before[:2]):
        assert torch.equal(now[~used], old[~used])
    for now, old in zip((ks, vs), before[2:]):
        assert torch.equal(now.transpose(1, 2)[~used], old.transpose(1, 2)[~used])
    # read back: code * scale, rounded once
    for out in (BF16, F32):
        ko, vo = torch.empty(M, G * dim, dtype=out, device="cuda"), torch.empty(M, G * vdim, dtype=out, device="cuda")
        ops.kv_load_8bit(meta, kc, vc, ks, vs, ko, vo, G, dim, vdim)
        for o, c, s in ((ko, kc, ks), (vo, vc, vs)):
            slot, pos = meta.long().unbind(1)
            want = c.view(torch.uint8)[slot, pos].view(kind).float().view(M, G, -1) * s[slot, :, pos][..., None]
            assert torch.equal(o, want.view(M, -1).to(out))


@pytest.mark.parametrize("kind", [torch.int8, E4M3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("act", [BF16, F32], ids=["bf16", "f32"])
def test_numbers_at_the_edges(ops, kind, act):
    """Zeros, ties, the largest and smallest numbers, infinities and NaN: a head of each."""
    dim, heads = 64, []
    base = rnd(dim, seed=3, dtype=F32).to(BF16).float()
    for a in (1.0, 1.75, 1.7578125, 3.0, 127.0, 254.0, 448.0, 449.0, 0.0078125, 3.3e38, 2.0 ** 126, 2.0 ** -95, 2.0 ** -100, 2.0 ** -110, 1e-40, 0.0):
        h = (base / base.abs().max()).to(BF16).float() * a
        h[0], h[1], h[2], h[3] = a, a / 2, -a / 2, a * (2.0 ** -9)
        heads.append(h.to(BF16).float())
    for bad in (float("inf"), float("-inf"), float("nan")):
        h = base.clone()
        h[11] = bad
        heads.append(h)
    x = torch.stack(heads).to(act).cuda()                                               # every row one head
    M = x.shape[0]
    meta = torch.stack((torch.zeros(M), torch.arange(M)), 1).to(torch.int32).cuda()
    kc, ks = caches(1, M, 1, dim, kind)
    vc, vs = caches(1, M, 1, dim, kind)
    ops.kv_store_8bit(x, x, meta, kc, vc, ks, vs, 1, dim, dim)
    fine = slice(0, M - 3)
    y, s = codes_of(x[fine].double().view(-1, 1, dim), kind)
    assert torch.equal(kc[0, fine].double(), rounded(y, kind)[:, 0])
    assert torch.equal(vc.view(torch.uint8), kc.view(torch.uint8)) and torch.equal(ks, vs) or torch.isnan(ks).any()
    assert ((ks[0, 0, fine].double() - s[:, 0]).abs() <= 2.0 ** -24 * s[:, 0]).all()
    assert torch.isnan(ks[0, 0, M - 3:]).all() and (kc[0, M - 3:].view(torch.uint8) == 0).all()
    out = torch.empty(M, dim, device="cuda")
    ops.kv_load_8bit(meta, kc, vc, ks, vs, out, out.clone(), 1, dim, dim)
    assert torch.isnan(out[M - 3:]).all() and torch.isfinite(out[fine]).all()
    assert (out[fine].double() - x[fine].double()).abs().max(1)[0].le(torch.maximum(x[fine].double().abs().max(1)[0], torch.tensor(LEAST, device="cuda")) * (0.5 / 127 + 2.0 ** -20 if kind == torch.int8 else 2.0 ** -4)).all()


@pytest.mark.parametrize("kind", [torch.int8, E4M3], ids=["int8", "e4m3"])
def test_strided_rows_and_places_that_are_not_there(ops, kind):
    """Column slices whose rows begin off 16-byte boundaries; slots and positions outside the caches are left out, and read as NaN."""
    M, G, dim, vdim, slots, cap = 21, 3, 64, 128, 2, 16
    for shift, wide in ((0, 8), (3, 5), (8, 0)):
        y = rnd(M, G * (dim + vdim) + shift + wide, seed=9)
        k, v = y[:, shift:shift + G * dim], y[:, shift + G * dim:shift + G * (dim + vdim)]
        meta = torch.tensor([(i % 4 - 1, (i * 5) % 21 - 2) for i in range(M)], dtype=torch.int32, device="cuda")
        there = (meta[:, 0] >= 0) & (meta[:, 0] < slots) & (meta[:, 1] >= 0) & (meta[:, 1] < cap)
        assert 0 < there.sum() < M and len({tuple(m) for m in meta[there].tolist()}) == there.sum()
        (kc, ks), (vc, vs) = caches(slots, cap, G, dim, kind), caches(slots, cap, G, vdim, kind)
        k2, v2 = caches(slots, cap, G, dim, kind), caches(slots, cap, G, vdim, kind)
        ops.kv_store_8bit(k, v, meta, kc, vc, ks, vs, G, dim, vdim)
        ops.kv_store_8bit(k[there].contiguous(), v[there].contiguous(), meta[there].contiguous(), k2[0], v2[0], k2[1], v2[1], G, dim, vdim)
        for a, b in ((kc, k2[0]), (vc, v2[0])):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(ks, k2[1]) and torch.equal(vs, v2[1])
        o = torch.full((M, G * (dim + vdim) + shift + wide), 5.0, dtype=BF16, device="cuda")
        ko, vo = o[:, shift:shift + G * dim], o[:, shift + G * dim:shift + G * (dim + vdim)]
        ops.kv_load_8bit(meta, kc, vc, ks, vs, ko, vo, G, dim, vdim)
        assert torch.isnan(ko[~there]).all() and torch.isnan(vo[~there]).all() and torch.isfinite(ko[there]).all() and torch.isfinite(vo[there]).all()
        assert (o[:, :shift] == 5).all() and (o[:, shift + G * (dim + vdim):] == 5).all()
        check_codes(kc, ks, k[there].double().view(-1, G, dim), meta[there], G, kind, True, "keys")


def test_rows_at_offsets_past_32_bits(ops):
    """A cache of more than 2^32 numbers."""
    G, dim, cap = 8, 128, 2_200_000
    kc = torch.empty(2, cap, G * dim, dtype=torch.int8, device="cuda")
    vc = torch.empty(2, cap, G * 64, dtype=torch.int8, device="cuda")
    ks, vs = (torch.empty(2, G, cap, device="cuda") for _ in range(2))
    meta = torch.tensor([(1, cap - 1), (1, cap - 200_000), (0, 0), (0, cap - 1)], dtype=torch.int32, device="cuda")
    k, v = rnd(4, G * dim, seed=4), rnd(4, G * 64, seed=5)
    ops.kv_store_8bit(k, v, meta, kc, vc, ks, vs, G, dim, 64)
    check_codes(kc, ks, k.double().view(4, G, dim), meta, G, torch.int8, True, "keys")
    check_codes(vc, vs, v.double().view(4, G, 64), meta, G, torch.int8, True, "values")


def test_replayed_on_another_stream(ops):
    G, dim, M = 4, 128, 6
    (kc, ks), (vc, vs) = caches(2, 32, G, dim, E4M3), caches(2, 32, G, dim, E4M3)
    meta = torch.tensor([(i % 2, 3 * i) for i in range(M)], dtype=torch.int32, device="cuda")
    k, v = rnd(M, G * dim, seed=1), rnd(M, G * dim, seed=2)
    ko, vo = torch.empty_like(k), torch.empty_like(v)

    def both():
        ops.kv_store_8bit(k, v, meta, kc, vc, ks, vs, G, dim, dim)
        ops.kv_load_8bit(meta, kc, vc, ks, vs, ko, vo, G, dim, dim)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    k.copy_(rnd(M, G * dim, seed=7)); v.copy_(rnd(M, G * dim, seed=8)); meta[:, 1] += 1
    graph.replay()
    torch.cuda.synchronize()
    got = ko.clone(), vo.clone()
    both()
    assert torch.equal(got[0], ko) and torch.equal(got[1], vo)
    check_codes(kc, ks, k.double().view(M, G, dim), meta, G, E4M3, True, "keys")


@pytest.mark.parametrize("kind", [torch.int8, E4M3], ids=["int8", "e4m3"])
def test_no_rows(ops, kind):
    """A step without tokens stores and reads nothing (an empty tensor has no address)."""
    (kc, ks), (vc, vs) = caches(2, 8, 3, 64, kind), caches(2, 8, 3, 128, kind)
    before = [x.clone() for x in (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)]
    k, v, meta = torch.empty(0, 3 * 64, dtype=BF16, device="cuda"), torch.empty(0, 3 * 128, dtype=BF16, device="cuda"), torch.empty(0, 2, dtype=torch.int32, device="cuda")
    ops.kv_store_8bit(k, v, meta, kc, vc, ks, vs, 3, 64, 128)
    ops.kv_load_8bit(meta, kc, vc, ks, vs, k, v, 3, 64, 128)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)))
