"""8-bit caches and scores through the model and the engine."""
import ctypes
import os
import subprocess

import pytest
import torch

import lia_b200  # noqa: F401
from lia_b200 import _lib, ops, registry
from lia_b200.checkpoint import write_safetensors
from lia_b200.engine import Engine
from lia_b200.modeling_bebulorn import BebulornConfig, BebulornForCausalLM
from lia_b200.seq_layers import StepBatch, WindowAttentionMixer
from lia_b200.seq_state import SlotState

from bebulorn_cases import attention, config, dense, lightning

pytestmark = pytest.mark.gpu
BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn


def small(seed=0, cache_dtype=None, window=40):
    c = BebulornConfig.from_dict(config([attention(4, 2, 64, 128, window, mlp=dense(96)), lightning(2, 32, 32, mlp=dense(96)), attention(8, 2, 64, 64, 1000, softcap=0.0, mlp=dense(96))],
                                        vocab=331, width=128))
    return BebulornForCausalLM(c, "cuda", BF16, cache_dtype).init_weights(seed)


def tokens(n, seed):
    return torch.randint(0, 331, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("cache_dtype", [torch.int8, E4M3], ids=["int8", "e4m3"])
def test_mixer_with_an_8_bit_cache(cache_dtype):
    """Prompts, portions and single tokens: the attention of what the caches hold, against 64 bits.  Before the output projection a row is off by 2^-8 of itself and 3 * 2^-11 + 2^-10 of its
    values' weighted magnitudes (tests/test_gpu_tree_attn.py; scores below 60 with 64 products are within 2^-12), and is then rounded: the projection takes both through its magnitudes, sums in
    32 bits and rounds once more."""
    H, G, dim, vdim, W, window, T = 4, 2, 64, 128, 128, 50, 150
    g = torch.Generator().manual_seed(1)
    w = {"q": torch.randn(H * dim, W, generator=g) * W ** -0.5, "k": torch.randn(G * dim, W, generator=g) * W ** -0.5, "v": torch.randn(G * vdim, W, generator=g) * W ** -0.5,
         "temp": 1 + 0.1 * torch.randn(H, generator=g), "o": (torch.randn(W, H * vdim, generator=g) * (H * vdim) ** -0.5).to(BF16).float()}
    mixer = WindowAttentionMixer(w, H, G, dim, vdim, window, dim ** -0.5, 30.0, 1e-5, BF16, "cuda", cache_dtype=cache_dtype)
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
    assert kc.dtype == vc.dtype == cache_dtype
    meta = torch.tensor([(2, i) for i in range(T)], dtype=torch.int32, device="cuda")
    k, v = torch.empty(T, G * dim, device="cuda"), torch.empty(T, G * vdim, device="cuda")
    ops.kv_load_8bit(meta, kc, vc, ks, vs, k, v, G, dim, vdim)
    q = mixer.proj.part(mixer.proj(h), 0).double().view(T, H, dim)
    k, v = k.double().view(T, G, dim).repeat_interleave(H // G, 1), v.double().view(T, G, vdim).repeat_interleave(H // G, 1)
    x = torch.einsum("ihd,jhd->hij", q, k) * dim ** -0.5 * mixer.temp.double()[:, None, None]
    x = 30 * torch.tanh(x / 30)
    i, j = torch.arange(T, device="cuda")[:, None], torch.arange(T, device="cuda")
    p = torch.softmax(x.masked_fill((j > i) | (j <= i - window), float("-inf")), -1)
    o, A = torch.einsum("hij,jhd->ihd", p, v).reshape(T, -1), torch.einsum("hij,jhd->ihd", p, v.abs()).reshape(T, -1)
    wo = w["o"].double().cuda()
    want = o @ wo.t()
    tol = (2.0 ** -8 * o.abs() + (3 * 2.0 ** -11 + 2.0 ** -10) * A) @ wo.abs().t() + 2.0 ** -8 * want.abs() + 2.0 ** -14 * (o.abs() @ wo.abs().t())
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


@pytest.mark.parametrize("cache_dtype", [torch.int8, E4M3], ids=["int8", "e4m3"])
def test_engine_with_8_bit_caches(cache_dtype, tmp_path):
    """Decoding from graphs and without them picks the same tokens; portions of prompts are as good as whole ones; a checkpoint is loaded with the same caches; half the bytes of a bf16 cache."""
    m = small(3, cache_dtype)
    prompts = [tokens(n, n) for n in (90, 1, 37)]
    with_graphs = Engine(m, 160, max_requests=3).generate(prompts, 24)
    assert with_graphs == Engine(m, 160, max_requests=3, graphs=False).generate(prompts, 24)
    whole = Engine(m, 160).step([{"id": 0, "tokens": prompts[0], "want": [89]}])
    eng = Engine(m, 160)
    eng.step([{"id": 0, "tokens": prompts[0][:41], "want": []}])
    parts = eng.step([{"id": 0, "tokens": prompts[0][41:], "want": [48]}])
    assert (whole - parts).abs().max() <= 0.05 * whole.abs().max()          # (the same numbers in other sums, through three layers in bf16)
    write_safetensors(str(tmp_path / "model.safetensors"), {n: t.to(BF16) for n, t in _weights(m.config, 3).items()})
    import json
    (tmp_path / "config.json").write_text(json.dumps(m.config.to_dict()))
    loaded = registry.load_model(str(tmp_path), cache_dtype=cache_dtype)
    assert Engine(loaded, 160, max_requests=3).generate(prompts, 24) == with_graphs
    bytes_of = lambda e: sum(t.numel() * t.element_size() for t in e.slots.rows)  # noqa: E731
    assert bytes_of(Engine(m, 160)) < 0.54 * bytes_of(Engine(small(3), 160))


def _weights(cfg, seed):
    """What ``init_weights`` makes."""
    got = {}

    class Keep(BebulornForCausalLM):
        def load_weights(self, get):
            got.update({n: get(n) for n in self.config.tensor_shapes()})
            return self
    m = Keep(cfg, "cuda")
    m.load_weights = lambda get: BebulornForCausalLM.load_weights(m, lambda n: got.setdefault(n, get(n)))
    m.init_weights(seed)
    return got


def test_8_bit_caches_are_refused_where_they_do_not_fit():
    c = BebulornConfig.from_dict(config([attention(4, 2, 64, 64, 40)], vocab=50, width=64))
    with pytest.raises(ValueError, match="8 bits"):
        BebulornForCausalLM(c, "cuda", F32, torch.int8).init_weights(0)
    with pytest.raises(ValueError, match="8 bits"):
        BebulornForCausalLM(c, "cuda", BF16, torch.float16).init_weights(0)
    odd = BebulornConfig.from_dict(config([attention(4, 2, 48, 64, 40)], vocab=50, width=64))
    with pytest.raises(ValueError, match="8 bits"):
        BebulornForCausalLM(odd, "cuda", BF16, torch.int8).init_weights(0)


@pytest.mark.parametrize("chunk", [None, 1, 7])
@pytest.mark.parametrize("max_rows", [4096, 50])
def test_scores(chunk, max_rows):
    """Against the logarithm of the softmax of the step's own logits, in 64 bits."""
    m = small(5)
    texts = [tokens(n, n + 1) for n in (33, 2, 1, 20, 0)]
    eng = Engine(m, 64, max_requests=5, max_rows=max_rows)
    got = eng.score(texts, top=4, chunk=chunk)
    assert eng.slots.live_tokens == 0
    for text, g in zip(texts, got):
        n = max(0, len(text) - 1)
        assert len(g["logp"]) == len(g["entropy"]) == len(g["alternatives"]) == n
        if not n:
            continue
        ref = Engine(m, 64)
        portion = chunk or max(1, max_rows // len(texts))
        rows = [ref.step([{"id": 0, "tokens": text[a:a + portion], "want": list(range(len(text[a:a + portion])))}]) for a in range(0, len(text), portion)]
        logp = torch.log_softmax(torch.cat(rows)[:n].double(), -1)
        want = logp.gather(1, torch.tensor(text[1:], device="cuda").view(-1, 1))[:, 0]
        # other requests' rows in a step may change a projection's form, by a step of bf16 in a row of it: logits of up to 5 are off by some hundredths
        assert (torch.tensor(g["logp"], dtype=F64, device="cuda") - want).abs().max() < 0.1
        assert (torch.tensor(g["entropy"], dtype=F64, device="cuda") + (logp.exp() * logp).sum(-1)).abs().max() < 0.1
        assert all(len(a) == 4 and all(x[1] >= y[1] for x, y in zip(a, a[1:])) for a in g["alternatives"])


def test_scores_of_one_request_are_its_logits(monkeypatch):
    """Alone in the step, the scores are those of the very logits that the step returned."""
    m, seen = small(6), []
    text = tokens(30, 9)
    eng = Engine(m, 64)
    step = eng.step
    monkeypatch.setattr(eng, "step", lambda e: seen.append(step(e)) or seen[-1])
    got = eng.score([text], top=2)[0]
    logp = torch.log_softmax(seen[0].double(), -1)
    assert (torch.tensor(got["logp"], dtype=F64, device="cuda") - logp.gather(1, torch.tensor(text[1:], device="cuda").view(-1, 1))[:, 0]).abs().max() < 2.0 ** -14
    assert [a[0][0] for a in got["alternatives"]] == seen[0].argmax(-1).tolist()


@pytest.fixture(scope="module")
def nowait():
    _lib.load()
    csrc = os.path.join(os.path.dirname(_lib.__file__), "csrc")
    subprocess.run(["make", "-C", csrc, "-j", str(os.cpu_count() or 4), "nowait"], check=True, capture_output=True, timeout=900)
    lib = ctypes.CDLL(os.path.join(csrc, "build", "nowait", "libliab200_nowait.so"))
    for name, (res, args) in _lib._PROTOTYPES.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    return lib


@pytest.mark.parametrize("kind", [BF16, torch.int8], ids=["bf16", "int8"])
@pytest.mark.parametrize("n,past,splits", [(50, 100, 1), (150, 100, 1), (40, 3000, 2)])
def test_waits_that_run_out(nowait, monkeypatch, kind, n, past, splits):
    """Built with a limit of 0, so that every bounded wait gives up at once: the launch ends, its blocks are counted, and its rows, formed key by key, are right all the same."""
    G, dim = 3, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF16)  # noqa: E731
    q, kc, vc, ks, vs = rnd(n, G * dim), rnd(1, past + n, G * dim), rnd(1, past + n, G * dim), None, None
    if kind == torch.int8:
        kc, vc = ((x.float() * 20).to(torch.int8) for x in (kc, vc))
        ks, vs = (torch.rand(1, G, past + n, generator=g, device="cuda") * 0.1 + 0.01 for _ in range(2))
    segs = torch.tensor([(0, past, 0, n)], dtype=torch.int32, device="cuda")

    def call():
        return ops.tree_attn(q, kc, vc, segs, torch.empty_like(q), G, G, dim, dim, dim ** -0.5, rows=n, max_ctx=past + n, k_scale=ks, v_scale=vs)
    want = call().double()
    with monkeypatch.context() as c:
        c.setattr(_lib, "_lib", nowait)
        before = nowait.lia_moe_timeouts()
        got = call().double()
        gave_up = nowait.lia_moe_timeouts() - before
    assert gave_up >= G * splits
    # both are within 2^-8 of themselves, and of 3 * 2^-11 + 2^-10 of weighted magnitudes below 2 (int8: below 2.6 times the scale's 0.11 * 127 / 2.6)
    assert ((got - want).abs() <= 2.0 ** -7 * want.abs() + (0.006 if kind == BF16 else 0.03)).all(), (got - want).abs().max()
    assert torch.equal(call().double(), want)


@pytest.mark.parametrize("cache_dtype", [torch.int8, E4M3], ids=["int8", "e4m3"])
def test_graphs_launch_what_a_step_would(cache_dtype):
    """A step that is replayed from a graph gives the bits of one that is launched, wherever the number of blocks that share a history changes: 256 positions, and far behind 2048."""
    m = small(11, cache_dtype, window=5000)
    text = tokens(3600, 5)
    launched, replayed = (Engine(m, 3600, max_requests=1, graphs=g) for g in (False, True))
    for n in (256, 256, 256, 257, 300, 2100, 2100, 2100, 2600, 3600):
        got = []
        for e in (launched, replayed):
            e.step([{"id": 0, "tokens": text[:n - 1], "want": []}])
            got.append(e.step([{"id": 0, "tokens": text[n - 1:n], "want": [0]}], end=[0]))
        assert torch.equal(*got), n
