"""Keys and values in 4 bits: codes and scales against the definition in 64 bits, and what is read back.

A code is the rounded exact quotient, whatever the activations' type, so that codes and scales are equal -- but for normed values, which are rounded to 32 bits after a sum of squares that is off by
up to 11.5 * 2^-24 of itself (tests/test_gpu_kv_8bit.py), below 2^-20: a scale may be the neighbouring bf16 number where a / 7 is within 2^-20 of a border, a code the neighbouring one where the quotient is."""
import pytest
import torch

from cache4 import codes_of, numbers, packed, quantised

pytestmark = pytest.mark.gpu
BF16, F32, F64, U8 = torch.bfloat16, torch.float32, torch.float64, torch.uint8
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def ops():
    import lia_b200  # noqa: F401
    from lia_b200 import ops
    return ops


def rnd(*shape, seed=0, std=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda") * std).to(dtype)


def caches(slots, cap, G, dim, layout="slots"):
    lay = (cap, slots) if layout == "time" else (slots, cap)
    c = torch.full((*lay, G, dim // 2), 0x5a, dtype=U8, device="cuda")
    c = c.permute(1, 0, 2, 3) if layout == "time" else c.view(slots, cap, -1)
    return c, torch.full((slots, G, cap, dim // 32), -3.0, dtype=BF16, device="cuda")


def heads(c, G):
    return c if c.dim() == 4 else c.view(c.shape[0], c.shape[1], G, -1)


def check_codes(cache, scale, x, meta, G, normed, what):
    dim = x.shape[-1]
    slot, pos = meta.long().unbind(1)
    got, got_s = codes_of(heads(cache, G)[slot, pos], dim).double(), scale[slot, :, pos].double()
    y, s = quantised(x)
    if not normed:
        assert torch.equal(got_s, s), what
        assert torch.equal(got, torch.round(y)), (what, (got != torch.round(y)).sum())
        return
    near = [quantised(x * (1 + e))[1] for e in (-2.0 ** -20, 2.0 ** -20)]
    assert ((got_s >= near[0]) & (got_s <= near[1])).all(), what
    y = x / got_s.repeat_interleave(32, -1)
    lo, hi = torch.round(y * (1 - 2.0 ** -20)), torch.round(y * (1 + 2.0 ** -20))
    assert ((got >= torch.minimum(lo, hi)) & (got <= torch.maximum(lo, hi))).all(), what


@pytest.mark.parametrize("act,M,G,dim,vdim,layout,norm", [
    (BF16, 1, 1, 128, 128, "slots", False), (BF16, 37, 8, 128, 64, "time", False), (F32, 37, 3, 64, 128, "slots", False), (BF16, 5, 2, 32, 96, "slots", False),
    (BF16, 9, 3, 256, 288, "slots", False), (F32, 9, 2, 1024, 512, "time", False), (BF16, 130, 8, 128, 128, "slots", True), (F32, 70, 5, 96, 192, "time", True),
    (F32, 700, 8, 128, 128, "slots", False), (BF16, 7, 1, 160, 1024, "slots", True)])
def test_store_and_load(ops, act, M, G, dim, vdim, layout, norm):
    slots, cap, eps = 3, M + 11, 1e-6
    g = torch.Generator().manual_seed(M)
    place = torch.randperm(slots * cap, generator=g)[:M]
    meta = torch.stack((place // cap, place % cap), 1).to(torch.int32).cuda()
    k, v = rnd(M, G * dim, seed=1, std=1.7, dtype=act), rnd(M, G * vdim, seed=2, std=0.3, dtype=act)
    k[:, ::5] *= 20
    kc, ks = caches(slots, cap, G, dim, layout)
    vc, vs = caches(slots, cap, G, vdim, layout)
    before = [x.clone() for x in (kc, vc, ks, vs)]
    ops.kv_store_4bit(k, v, meta, kc, vc, ks, vs, G, dim, vdim, eps=eps, norm_values=norm)
    x = v.double().view(M, G, vdim)
    check_codes(kc, ks, k.double().view(M, G, dim), meta, G, False, "keys")
    check_codes(vc, vs, x / (x.square().mean(-1, keepdim=True) + eps).sqrt() if norm else x, meta, G, norm, "values")
    used = torch.zeros(slots, cap, dtype=torch.bool, device="cuda")          # no other place has changed
    used[meta[:, 0].long(), meta[:, 1].long()] = True
    for now, old in zip((kc, vc), before[:2]):
        assert torch.equal(now[~used], old[~used])
    for now, old in zip((ks, vs), before[2:]):
        assert torch.equal(now.transpose(1, 2)[~used], old.transpose(1, 2)[~used])
    for out in (BF16, F32):                                                   # read back: code * scale, rounded once
        ko, vo = torch.empty(M, G * dim, dtype=out, device="cuda"), torch.empty(M, G * vdim, dtype=out, device="cuda")
        ops.kv_load_4bit(meta, kc, vc, ks, vs, ko, vo, G, dim, vdim)
        for o, c, s, d in ((ko, kc, ks, dim), (vo, vc, vs, vdim)):
            slot, pos = meta.long().unbind(1)
            assert torch.equal(o, numbers(heads(c, G)[slot, pos], s[slot, :, pos], d).to(out).view(M, -1))


@pytest.mark.parametrize("act", [BF16, F32], ids=["bf16", "f32"])
def test_numbers_at_the_edges(ops, act):
    """Zeros, ties, the largest and smallest numbers, infinities and NaN: a group of each, beside groups that must not notice."""
    dim, groups = 128, []
    base = rnd(32, seed=3, dtype=F32).to(BF16).float()
    for a in (1.0, 1.75, 7.0, 3.0, 14.0, 0.0078125, 3.3e38, 2.0 ** 126, 2.0 ** -95, 2.0 ** -100, 2.0 ** -110, 1e-40, 0.0):
        h = base / base.abs().max() * a
        for i, f in enumerate((1.0, 0.5 / 7, -1.5 / 7, 2.5 / 7, -3.5 / 7, 4.5 / 7, 5.5 / 7, -6.5 / 7)):
            h[i] = a * f
        groups.append(h.to(act).float())
    for bad in (INF, -INF, NAN):
        h = base.clone()
        h[11] = bad
        groups.append(h)
    x = torch.stack(groups)
    order = torch.randperm(len(x), generator=torch.Generator().manual_seed(1))
    x = x[order.to(x.device)].reshape(len(x) // 4, dim).to(act)
    M = x.shape[0]
    meta = torch.tensor([(0, i) for i in range(M)], dtype=torch.int32, device="cuda")
    (kc, ks), (vc, vs) = caches(1, M, 1, dim), caches(1, M, 1, dim)
    ops.kv_store_4bit(x, x, meta, kc, vc, ks, vs, 1, dim, dim)
    y, s = quantised(x.double().view(M, 1, dim))
    want = torch.where(torch.isnan(s).repeat_interleave(32, -1), torch.zeros_like(y), torch.round(y))
    for c, got_s in ((kc, ks), (vc, vs)):
        assert torch.equal(codes_of(heads(c, 1)[0], dim).double(), want)
        assert torch.equal(torch.nan_to_num(got_s[0].transpose(0, 1).double(), nan=-1.0), torch.nan_to_num(s, nan=-1.0))
    o = [torch.empty(M, dim, dtype=F32, device="cuda") for _ in range(2)]
    ops.kv_load_4bit(meta, kc, vc, ks, vs, *o, 1, dim, dim)
    bad = torch.isnan(s).repeat_interleave(32, -1).view(M, dim)
    assert torch.isnan(o[0][bad]).all() and torch.isfinite(o[0][~bad]).all() and torch.equal(torch.nan_to_num(o[0]), torch.nan_to_num(o[1]))


def test_fp32_quotients_next_to_a_border(ops):
    """32-bit numbers whose quotient rounds to a tie in 32 bits but is none: the exact quotient decides."""
    scale, rows = torch.tensor(1.0078125 / 8, dtype=F64), []
    for k in range(-7, 7):
        tie = ((k + 0.5) * scale).to(F32)
        rows += [torch.nextafter(tie, torch.tensor(INF)), tie, torch.nextafter(tie, torch.tensor(-INF))]
    x = torch.zeros(2, 32, dtype=F32)
    x[0, :21], x[1, :21] = torch.stack(rows[:21]), torch.stack(rows[21:])
    x[:, 31] = 7 * scale
    x = x.cuda()
    meta = torch.tensor([(0, 0), (0, 1)], dtype=torch.int32, device="cuda")
    (kc, ks), (vc, vs) = caches(1, 2, 1, 32), caches(1, 2, 1, 32)
    ops.kv_store_4bit(x, x, meta, kc, vc, ks, vs, 1, 32, 32)
    check_codes(kc, ks, x.double().view(2, 1, 32), meta, 1, False, "borders")


def test_places_that_are_not_there(ops):
    """Rows outside the caches are left out by the store and read back as NaN; no rows are no work."""
    G, dim = 2, 64
    k, v = rnd(5, G * dim, seed=1), rnd(5, G * dim, seed=2)
    (kc, ks), (vc, vs) = caches(2, 4, G, dim), caches(2, 4, G, dim)
    meta = torch.tensor([(0, 1), (2, 0), (-1, 0), (1, 4), (1, -1)], dtype=torch.int32, device="cuda")
    old = kc.clone()
    ops.kv_store_4bit(k, v, meta, kc, vc, ks, vs, G, dim, dim)
    assert not torch.equal(kc[0, 1], old[0, 1])
    kc[0, 1] = old[0, 1]
    assert torch.equal(kc, old)
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    ops.kv_load_4bit(meta, kc, vc, ks, vs, ko, vo, G, dim, dim)
    assert torch.isnan(ko[1:]).all() and torch.isnan(vo[1:]).all() and torch.isfinite(ko[0]).all()
    ops.kv_store_4bit(k[:0], v[:0], meta[:0], kc, vc, ks, vs, G, dim, dim)
    ops.kv_load_4bit(meta[:0], kc, vc, ks, vs, ko[:0], vo[:0], G, dim, dim)


@pytest.mark.parametrize("act", [BF16, F32], ids=["bf16", "f32"])
def test_strides_and_another_stream(ops, act):
    """Columns of something wider on odd boundaries, caches with a head stride of their own, scales that are part of something larger, a captured call with other rows in it."""
    M, G, dim, vdim = 33, 3, 128, 64
    wide = rnd(M, G * (dim + vdim) + 7, seed=4, dtype=act)
    k, v = wide[:, 1:1 + G * dim], wide[:, 3 + G * dim:3 + G * (dim + vdim)]
    meta = torch.tensor([(i % 2, 3 * (i // 2)) for i in range(M)], dtype=torch.int32, device="cuda")
    cap = 64
    kc = torch.zeros(2, cap, G, 2, dim // 2, dtype=U8, device="cuda")[:, :, :, 1]
    vc = torch.zeros(2, cap + 5, G * vdim // 2, dtype=U8, device="cuda")[:, 5:]
    ks, vs = torch.zeros(2, 2 * G, cap, dim // 32, dtype=BF16, device="cuda")[:, G:], torch.zeros(2, G, cap, vdim // 32, dtype=BF16, device="cuda")
    ko = torch.zeros(M, G * dim + 5, dtype=act, device="cuda")[:, 5:]
    vo = torch.zeros(M, G * vdim, dtype=act, device="cuda")
    ops.kv_store_4bit(k, v, meta, kc, vc, ks, vs, G, dim, vdim)            # (loads the kernels before they are captured)
    ops.kv_load_4bit(meta, kc, vc, ks, vs, ko, vo, G, dim, vdim)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.kv_store_4bit(k, v, meta, kc, vc, ks, vs, G, dim, vdim)
        ops.kv_load_4bit(meta, kc, vc, ks, vs, ko, vo, G, dim, vdim)
    wide.copy_(rnd(*wide.shape, seed=5, dtype=act))
    meta[:, 0] = 1 - meta[:, 0]
    graph.replay()
    torch.cuda.synchronize()
    slot, pos = meta.long().unbind(1)
    for x, c, s, o, d in ((k, kc, ks, ko, dim), (v, vc, vs, vo, vdim)):
        check_codes(c, s, x.double().reshape(M, G, d), meta, G, False, "replayed")
        assert torch.equal(o.reshape(M, G, d), numbers(heads(c, G)[slot, pos], s[slot, :, pos], d).to(act))


def test_caches_past_32_bits(ops):
    G, dim, cap = 8, 128, 4_300_000
    kc, vc = (torch.empty(2, cap, G * dim // 2, dtype=U8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(2, G, cap, dim // 32, dtype=BF16, device="cuda") for _ in range(2))
    meta = torch.tensor([(1, cap - 1), (0, cap - 1), (1, 0)], dtype=torch.int32, device="cuda")
    k, v = rnd(3, G * dim, seed=1), rnd(3, G * dim, seed=2)
    ops.kv_store_4bit(k, v, meta, kc, vc, ks, vs, G, dim, dim)
    slot, pos = meta.long().unbind(1)
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        y, want = quantised(x.double().view(3, G, dim))
        assert torch.equal(s[slot, :, pos].double(), want) and torch.equal(codes_of(c[slot, pos].view(3, G, -1), dim).double(), torch.round(y))
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    ops.kv_load_4bit(meta, kc, vc, ks, vs, ko, vo, G, dim, dim)
    assert torch.equal(ko.view(3, G, dim), numbers(kc[slot, pos].view(3, G, -1), ks[slot, :, pos], dim).to(BF16))


def test_packing_is_its_own_reverse():
    c = torch.randint(-8, 8, (5, 3, 96), generator=torch.Generator().manual_seed(1))
    assert torch.equal(codes_of(packed(c), 96), c)
