"""4-bit caches, weights of 8 bits, forks and scores of choices through the model and the engine."""
import json

import pytest
import torch

import lia_b200  # noqa: F401
from lia_b200 import ops, registry
from lia_b200.checkpoint import write_safetensors
from lia_b200.engine import Engine
from lia_b200.modeling_bebulorn import BebulornConfig, BebulornForCausalLM
from lia_b200.seq_layers import Linear, StepBatch, WindowAttentionMixer
from lia_b200.seq_state import SlotError, SlotState

from bebulorn_cases import CASES, attention, config, delta, dense, lightning, moe
from test_gpu_drafted_serving import _weights, tokens

pytestmark = pytest.mark.gpu
BF16, F32, F64, I8, I4 = torch.bfloat16, torch.float32, torch.float64, torch.int8, torch.int4


def small(seed=0, cache_dtype=None, weight_dtype=None, window=40):
    c = BebulornConfig.from_dict(config([attention(4, 2, 64, 128, window, mlp=dense(96)), lightning(2, 32, 32, mlp=moe(4, 2, 48, shared=56)), delta(4, 2, 32, 32, 3),
                                         attention(8, 2, 64, 64, 1000, softcap=0.0, mlp=dense(96))], vocab=331, width=128))
    return BebulornForCausalLM(c, "cuda", BF16, cache_dtype, weight_dtype).init_weights(seed)


def test_mixer_with_a_4_bit_cache():
    """Prompts, portions and single tokens: the attention of what the caches hold, against 64 bits.  As with 8 bits (tests/test_gpu_drafted_serving.py); portions of more than 16 tokens have their keys
    multiplied by their groups' scales in fp16 (tests/test_gpu_tree_attn_4bit.py), a score off by up to 2^-10 B, which puts a row off by 2^-9 B of its values' weighted magnitudes."""
    H, G, dim, vdim, W, window, T = 4, 2, 64, 128, 128, 50, 150
    g = torch.Generator().manual_seed(1)
    w = {"q": torch.randn(H * dim, W, generator=g) * W ** -0.5, "k": torch.randn(G * dim, W, generator=g) * W ** -0.5, "v": torch.randn(G * vdim, W, generator=g) * W ** -0.5,
         "temp": 1 + 0.1 * torch.randn(H, generator=g), "o": (torch.randn(W, H * vdim, generator=g) * (H * vdim) ** -0.5).to(BF16).float()}
    mixer = WindowAttentionMixer(w, H, G, dim, vdim, window, dim ** -0.5, 30.0, 1e-5, BF16, "cuda", cache_dtype=I4)
    slots = SlotState(3, T + 5, "cuda")
    state = mixer.new_state(slots)
    h = torch.randn(T, W, generator=g).to(BF16).cuda()
    at, outs = 0, []
    for n in (70, 1, 1, 33, 2, 43):
        batch = StepBatch(n, torch.tensor([(2, at, 0, n)], dtype=torch.int32, device="cuda"), torch.tensor([(2, at + i) for i in range(n)], dtype=torch.int32, device="cuda"), at + n,
                          portions=[(2, at, 0, n)] if n != 33 else None)
        outs.append(mixer(h[at:at + n].contiguous(), batch, state))
        at += n
    got = torch.cat(outs).double()
    kc, ks, vc, vs = state
    assert kc.shape == (3, T + 5, G * dim // 2) and vs.shape == (3, G, T + 5, vdim // 32)
    meta = torch.tensor([(2, i) for i in range(T)], dtype=torch.int32, device="cuda")
    k, v = torch.empty(T, G * dim, device="cuda"), torch.empty(T, G * vdim, device="cuda")
    ops.kv_load_4bit(meta, kc, vc, ks, vs, k, v, G, dim, vdim)
    y = mixer.proj(h)
    near = mixer.proj.part(y, 1).double() - k.double()                        # half a step of the largest's seventh, and what the scale's 8 bits leave of seven steps
    assert (near.abs().view(T, G, -1, 32) <= (0.5 / 7 + 2.0 ** -8) * 1.01 * mixer.proj.part(y, 1).double().abs().view(T, G, -1, 32).amax(-1, keepdim=True)).all()
    q = mixer.proj.part(y, 0).double().view(T, H, dim)
    k, v = k.double().view(T, G, dim).repeat_interleave(H // G, 1), v.double().view(T, G, vdim).repeat_interleave(H // G, 1)
    f = dim ** -0.5 * mixer.temp.double()[:, None, None]
    x, B = torch.einsum("ihd,jhd->hij", q, k) * f, torch.einsum("ihd,jhd->hij", q.abs(), k.abs()) * f
    x = 30 * torch.tanh(x / 30)
    i, j = torch.arange(T, device="cuda")[:, None], torch.arange(T, device="cuda")
    hidden = (j > i) | (j <= i - window)
    p = torch.softmax(x.masked_fill(hidden, float("-inf")), -1)
    B = B.masked_fill(hidden, 0).amax(-1).t().repeat_interleave(vdim, 1)       # [T, H * vdim]
    o, A = torch.einsum("hij,jhd->ihd", p, v).reshape(T, -1), torch.einsum("hij,jhd->ihd", p, v.abs()).reshape(T, -1)
    wo = w["o"].double().cuda()
    want = o @ wo.t()
    tol = (2.0 ** -8 * o.abs() + (3 * 2.0 ** -11 + 2.0 ** -10 + 2.0 ** -9 * B) * A) @ wo.abs().t() + 2.0 ** -8 * want.abs() + 2.0 ** -14 * (o.abs() @ wo.abs().t())
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


@pytest.mark.parametrize("cache_dtype,weight_dtype", [(I4, None), (None, I8), (I4, I8), (I8, I8)], ids=["cache", "weights", "both", "8 bits"])
def test_engine_in_fewer_bits(cache_dtype, weight_dtype, tmp_path):
    """Decoding from graphs and without them picks the same tokens; portions of prompts are as good as whole ones; a checkpoint is loaded in the same way; fewer bytes."""
    m = small(3, cache_dtype, weight_dtype)
    prompts = [tokens(n, n) for n in (90, 1, 37)]
    with_graphs = Engine(m, 160, max_requests=3).generate(prompts, 24)
    assert with_graphs == Engine(m, 160, max_requests=3, graphs=False).generate(prompts, 24)
    whole = Engine(m, 160).step([{"id": 0, "tokens": prompts[0], "want": [89]}])
    eng = Engine(m, 160)
    eng.step([{"id": 0, "tokens": prompts[0][:41], "want": []}])
    parts = eng.step([{"id": 0, "tokens": prompts[0][41:], "want": [48]}])
    assert torch.isfinite(whole).all() and (whole - parts).abs().max() <= 0.1 * whole.abs().max()
    write_safetensors(str(tmp_path / "model.safetensors"), {n: t.to(BF16) for n, t in _weights(m.config, 3).items()})
    (tmp_path / "config.json").write_text(json.dumps(m.config.to_dict()))
    loaded = registry.load_model(str(tmp_path), cache_dtype=cache_dtype, weight_dtype=weight_dtype)
    assert Engine(loaded, 160, max_requests=3).generate(prompts, 24) == with_graphs
    bytes_of = lambda e: sum(t.numel() * t.element_size() for t in e.slots.rows)  # noqa: E731
    if cache_dtype == I4:
        assert bytes_of(Engine(m, 160)) < 0.29 * bytes_of(Engine(small(3), 160))


def test_weights_of_8_bits_by_their_formula(monkeypatch):
    """Every projection of mixers, dense feed-forwards and shared experts goes through the operator, and a step's logits are, bit by bit, those of its formula in 64 bits."""
    m, calls = small(4, weight_dtype=I8), []
    text = tokens(70, 1)
    run = lambda: Engine(m, 80, graphs=False).step([{"id": 0, "tokens": text, "want": [3, 69]}])  # noqa: E731
    got = run()

    def plain(x, w, w_scale, out=None, x_scale=None):
        calls.append(tuple(w.shape))
        a = x.float().abs().amax(1, keepdim=True).clamp(min=2.0 ** -100)
        codes = torch.round(127 * x.float() / a)
        return out.copy_((codes.double() @ w.double().t()).float() * (a / 127) * w_scale)
    monkeypatch.setattr(ops, "linear_int8", plain)
    want = run()
    assert len(calls) == 2 + 2 + 2 + 2 + 2 + 2 + 2 and torch.equal(got, want)         # two a mixer, two a dense feed-forward, two a shared expert
    held = [x for l in m.layers for part in (l.mixer, l.mlp, getattr(l.mlp, "shared", None)) if part is not None for x in vars(part).values() if isinstance(x, Linear)]
    assert all(x.weight.dtype == I8 and x.scale.shape == (x.N,) for x in held) and m.head.weight.dtype == BF16


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_odd_projections_of_8_bits(dtype):
    """Sizes that nothing divides: rows of codes are padded, columns of blocks begin where they did."""
    c = BebulornConfig.from_dict(json.loads(json.dumps(CASES["odd"])))
    m = BebulornForCausalLM(c, "cuda", dtype, weight_dtype=I8).init_weights(2)
    ref = BebulornForCausalLM(c, "cuda", dtype).init_weights(2)
    text = [t % 61 for t in tokens(33, 7)]
    a, b = (Engine(x, 64).step([{"id": 0, "tokens": text, "want": [32]}]) for x in (m, ref))
    assert torch.isfinite(a).all() and (a - b).norm() < 0.25 * b.norm()               # (codes of 8 bits through seven layers: some per cent)
    assert Engine(m, 64, max_requests=2).generate([text, text[:5]], 6) == Engine(m, 64, max_requests=2, graphs=False).generate([text, text[:5]], 6)


@pytest.mark.parametrize("cache_dtype", [None, I8, torch.float8_e4m3fn, I4], ids=["bf16", "int8", "e4m3", "int4"])
def test_a_fork_goes_on_as_its_request_would(cache_dtype):
    """Logits of forks are, bit by bit, those of a request that was never forked; the request itself goes on, and forks fork."""
    m = small(8, cache_dtype)
    text, ways = tokens(50, 3), [tokens(6, 20 + i) for i in range(4)]
    alone = []
    for way in ways:
        eng = Engine(m, 80, max_requests=5, graphs=False)
        eng.step([{"id": 0, "tokens": text}])
        alone.append([eng.step([{"id": 0, "tokens": [t], "want": [0]}]) for t in way])
    for graphs in (False, True):
        eng = Engine(m, 80, max_requests=5, graphs=graphs)
        eng.step([{"id": "other", "tokens": tokens(9, 1)}])                            # (so that slots are not the numbers they were)
        eng.step([{"id": "a", "tokens": text}])
        eng.fork("a", ["b", "c"])
        first = eng.step([{"id": "c", "tokens": ways[2][:1], "want": [0]}])
        assert torch.equal(first, alone[2][0])
        eng.fork("c", ["d"])
        for rid, k, at in (("a", 0, 0), ("b", 1, 0), ("c", 2, 1)):
            for i in range(at, 6):
                assert torch.equal(eng.step([{"id": rid, "tokens": [ways[k][i]], "want": [0]}]), alone[k][i]), (rid, i)
        assert torch.equal(eng.step([{"id": "d", "tokens": ways[2][1:2], "want": [0]}]), alone[2][1])
        with pytest.raises(SlotError):
            eng.fork("a", ["e"])                                                       # all slots are taken
        with pytest.raises(SlotError):
            eng.fork("nobody", ["e"])
        eng.step([], end=["d"])
        with pytest.raises(SlotError):
            eng.fork("a", ["b"])                                                       # b is there already
        eng.fork("a", [])
        assert eng.slots.slot_of("e") is None and eng.slots.owner.count(None) == 1


def test_forks_of_slots_take_tensors_that_come_later_and_are_all_or_none(monkeypatch):
    from lia_b200.seq_state import SlotState
    s = SlotState(4, 9, "cuda")
    a = s.add_rows(16, torch.bfloat16)
    s.alloc("x")
    s.reserve(0, 5)
    a[0] = 1
    assert s.fork("x", ["y"]) == [1]
    b = s.add_rows(8, torch.float32)
    b[0] = 2
    assert s.fork("x", ["z"]) == [2] and (a[2, :5] == 1).all() and (b[2, :5] == 2).all() and (b[2, 5:] == 0).all() and (b[1] == 0).all()

    def broken(*args, **kw):
        raise RuntimeError("no launch")
    monkeypatch.setattr(s._set, "fork", broken)
    with pytest.raises(RuntimeError, match="no launch"):
        s.fork("x", ["w"])
    assert s.owner == ["x", "y", "z", None] and s.length == [5, 5, 5, 0] and s.slot_of("w") is None


@pytest.mark.parametrize("requests", [8, 3, 2])
def test_scores_of_choices(requests):
    """As scores of the prompt with each choice behind it, whose last tokens they are; all slots are free afterwards."""
    m = small(9, I4)
    prompt, choices = tokens(40, 1), [tokens(n, 30 + n) for n in (5, 1, 9, 3)]
    eng = Engine(m, 64, max_requests=requests)
    got = eng.score_choices(prompt, choices, top=3)
    assert eng.slots.live_tokens == 0 and len(got) == 4
    ref = Engine(m, 64, max_requests=1)
    for c, g in zip(choices, got):
        want = ref.score([prompt + c], top=3)[0]
        n = len(c)
        assert len(g["logp"]) == len(g["entropy"]) == len(g["alternatives"]) == n
        # rows of other requests in a step, and portions, change sums' order: a step of bf16 here and there (tests/test_gpu_drafted_serving.py)
        assert (torch.tensor(g["logp"]) - torch.tensor(want["logp"][-n:])).abs().max() < 0.1 and (torch.tensor(g["entropy"]) - torch.tensor(want["entropy"][-n:])).abs().max() < 0.1
    assert eng.score_choices(prompt[:1], choices[:2])[0]["logp"] and eng.score_choices(prompt, []) == []
    for bad in ((prompt, [[1], []]), ([], [[1]])):
        with pytest.raises(ValueError):
            eng.score_choices(*bad)
    assert eng.slots.live_tokens == 0


def test_a_drafted_round_over_4_bits():
    """The operators as they are used: a prompt goes into a 4-bit cache, is forked, a tree of drafted tokens behind it in each, one attention over both; the accepted paths move up by compaction, and
    the next single tokens see what they would have seen without drafting."""
    H, G, dim, p0, n = 8, 2, 64, 150, 12
    slots = SlotState(3, 256, "cuda")
    (kc, ks), (vc, vs) = slots.add_rows_4bit(G, dim), slots.add_rows_4bit(G, dim)
    slots.alloc("a")
    slots.reserve(0, p0)
    gen = torch.Generator("cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(BF16)  # noqa: E731
    on = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    k, v = rnd(p0, G * dim), rnd(p0, G * dim)
    ops.kv_store_4bit(k, v, on([(0, t) for t in range(p0)]), kc, vc, ks, vs, G, dim, dim)
    assert slots.fork("a", ["b"]) == [1] and slots.length[:2] == [p0, p0]
    dk, dv = rnd(2 * n, G * dim), rnd(2 * n, G * dim)
    segs = on([(0, p0, 0, n), (1, p0, n, n)])
    ops.kv_store_4bit(dk, dv, on([(s, p0 + t) for s in range(2) for t in range(n)]), kc, vc, ks, vs, G, dim, dim)
    parent = lambda i: (i - 1) // 2 if i else -1  # noqa: E731
    seen = []
    for i in range(n):
        seen.append(1 << i | (seen[parent(i)] if i else 0))
    mask = torch.tensor(seen * 2, dtype=torch.int64, device="cuda").view(-1, 1)
    out = ops.tree_attn(rnd(2 * n, H * dim), kc, vc, segs, torch.empty(2 * n, H * dim, dtype=BF16, device="cuda"), H, G, dim, dim, dim ** -0.5, rows=n, max_ctx=p0 + n, mask=mask, k_scale=ks,
                        v_scale=vs)
    assert torch.isfinite(out).all()
    paths = [[0, 2, 5, 11], [0, 1]]
    ops.CacheSet(slots.positioned).compact(segs, on([p + [-1] * (5 - len(p)) for p in paths]))
    q = rnd(2, H * dim)
    one = ops.tree_attn(q, kc, vc, on([(0, p0 + 3, 0, 1), (1, p0 + 1, 1, 1)]), torch.empty_like(q), H, G, dim, dim, dim ** -0.5, rows=1, max_ctx=p0 + 4, k_scale=ks, v_scale=vs)
    plain = SlotState(3, 256, "cuda")
    (pk, pks), (pv, pvs) = plain.add_rows_4bit(G, dim), plain.add_rows_4bit(G, dim)
    for s, path in enumerate(paths):
        rows = torch.tensor([n * s + j for j in path], device="cuda")
        ops.kv_store_4bit(torch.cat((k, dk[rows])), torch.cat((v, dv[rows])), on([(s, t) for t in range(p0 + len(path))]), pk, pv, pks, pvs, G, dim, dim)
    two = ops.tree_attn(q, pk, pv, on([(0, p0 + 3, 0, 1), (1, p0 + 1, 1, 1)]), torch.empty_like(q), H, G, dim, dim, dim ** -0.5, rows=1, max_ctx=p0 + 4, k_scale=pks, v_scale=pvs)
    assert torch.equal(one, two)
