"""What the operators of drafted tokens refuse, and their state's shapes: no GPU, no launch."""
import ctypes

import pytest
import torch

BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as g
    g.build()
    import lia_b200
    from lia_b200 import _lib
    return _lib


def view(_lib, **change):
    v = dict(data=1 << 20, scale=1 << 21, slot_stride=1 << 16, pos_stride=1024, head_stride=128, scale_slot_stride=512, scale_head_stride=64, slots=2, capacity=64, type=_lib.CACHE_INT8, dim=128)
    return _lib.LiaCacheView(**(v | change))


def test_view_layout(lib):
    assert ctypes.sizeof(lib.LiaCacheView) == 72 and lib.LiaCacheView.slots.offset == 56


@pytest.mark.parametrize("change,message", [
    ({"data": None}, "null cache"), ({"scale": None}, "scales"), ({"type": 7}, "type"), ({"type": 0, "scale": None}, "int8"), ({"slots": 0}, "empty"), ({"capacity": 0}, "empty"),
    ({"data": (1 << 20) + 4}, "vectors"), ({"pos_stride": 1028}, "vectors"), ({"head_stride": 132}, "vectors"), ({"dim": 100}, "multiples of 8"), ({"dim": 2048}, "1024"),
    ({"capacity": 65}, "different sizes"), ({"type": 2}, "both")])
def test_store_and_load_refuse(lib, change, message):
    L = lib.load()
    good, bad = view(lib), view(lib, **change)
    for kc, vc in ((bad, good), (good, bad)):
        assert L.lia_kv_store_8bit(16, 1024, 16, 1024, 0, 16, kc, vc, 4, 8, 0.0, 0, None) == -1 and message in lib.last_error()
        assert L.lia_kv_load_8bit(16, kc, vc, 16, 1024, 16, 1024, 0, 4, 8, None) == -1 and message in lib.last_error()


def test_store_refuses_short_rows_and_null_pointers(lib):
    L, v = lib.load(), view(lib)
    assert L.lia_kv_store_8bit(16, 1023, 16, 1024, 0, 16, v, v, 4, 8, 0.0, 0, None) == -1 and "shorter" in lib.last_error()
    assert L.lia_kv_store_8bit(None, 1024, 16, 1024, 0, 16, v, v, 4, 8, 0.0, 0, None) == -1
    assert L.lia_kv_store_8bit(16, 1024, 16, 1024, 0, None, v, v, 4, 8, 0.0, 0, None) == -1
    assert L.lia_kv_store_8bit(16, 1024, 16, 1024, 0, 16, v, v, -1, 8, 0.0, 0, None) == -1
    assert L.lia_kv_store_8bit(16, 1 << 20, 16, 1 << 20, 0, 16, v, v, 1 << 28, 8, 0.0, 0, None) == -1 and "too many" in lib.last_error()
    assert L.lia_kv_store_8bit(16, 1024, 16, 1024, 0, 16, v, v, 0, 8, 0.0, 0, None) == 0           # no rows, no launch


def attn(lib, kc, vc, q=256, ldq=2048, segs=256, nseg=2, mask=None, words=0, out=256, ws=None, floats=0, M=8, H=16, G=8, rows=4, max_ctx=40, window=0):
    return lib.load().lia_tree_attn(q, ldq, kc, vc, segs, nseg, mask, words, None, None, out, ws, floats, M, H, G, rows, max_ctx, window, 1.0, 0.0, None)


@pytest.mark.parametrize("change,message", [
    ({"data": (1 << 20) + 8}, "vectors"), ({"dim": 96}, "64 or 128"), ({"dim": 256}, "64 or 128"), ({"type": 2}, "different types"), ({"slots": 3}, "different types or sizes"),
    ({"scale": None}, "scales")])
def test_attention_refuses_caches(lib, change, message):
    good, bad = view(lib), view(lib, **change)
    assert attn(lib, bad, good) == -1 and message in lib.last_error()
    assert attn(lib, good, bad) == -1 and message in lib.last_error()


@pytest.mark.parametrize("change,message", [
    ({"q": None}, "null"), ({"segs": None}, "null"), ({"out": None}, "null"), ({"H": 15}, "sizes"), ({"G": 0}, "sizes"), ({"M": -1}, "sizes"), ({"ldq": 2047}, "vectors"), ({"ldq": 1024}, "vectors"),
    ({"q": 260}, "vectors"), ({"mask": 256, "words": 0}, "null"), ({"mask": 256, "words": 1, "rows": 65}, "words"), ({"nseg": 70000}, "too many"),
    ({"max_ctx": 100000, "nseg": 1}, "workspace"), ({"max_ctx": 100000, "nseg": 1, "ws": 256, "floats": 10}, "workspace")])
def test_attention_refuses(lib, change, message):
    v = view(lib)
    assert attn(lib, v, v, **change) == -1 and message in lib.last_error()


def test_attention_of_nothing(lib):
    v = view(lib)
    assert attn(lib, v, v, nseg=0) == attn(lib, v, v, M=0) == attn(lib, v, v, rows=0) == 0
    assert lib.load().lia_tree_attn_workspace_floats(0, 4, 40, 8, 16, 8, 128, 128, 0, 1) == 0
    assert lib.load().lia_tree_attn_workspace_floats(1, 4, 100000, 8, 16, 8, 128, 128, 0, 1) % (8 * 16 * 130) == 0


@pytest.mark.parametrize("args,message", [
    (dict(V=0), "sizes"), (dict(top=33), "sizes"), (dict(V=4, top=5), "sizes"), (dict(ld=99), "sizes"), (dict(n=-1), "sizes"), (dict(logits=None), "null"), (dict(logits=2), "misaligned"),
    (dict(top=3, ids=None), "null"), (dict(n=1, tokens=None), "null")])
def test_logprobs_refuse(lib, args, message):
    a = dict(logits=16, f32=1, ld=100, M=2, V=100, tokens=16, n=1, logp=16, entropy=16, top=0, best=16, ids=16) | args
    rc = lib.load().lia_token_logprobs(a["logits"], a["f32"], a["ld"], a["M"], a["V"], a["tokens"], a["n"], a["logp"], a["entropy"], a["top"], a["best"], a["ids"], None)
    assert rc == -1 and message in lib.last_error()


def test_wrappers_refuse(lib):
    """Tensors of the wrong shape, type or place raise before anything is launched."""
    from lia_b200 import ops
    E = lib.LiaError
    z = torch.zeros
    with pytest.raises(E):
        ops.kv_store_8bit(z(2, 128, dtype=BF16), z(2, 128, dtype=BF16), z(2, 2, dtype=torch.int32), z(1, 4, 128, dtype=torch.int8), z(1, 4, 128, dtype=torch.int8), z(1, 1, 4), z(1, 1, 4), 1, 128, 128)
    with pytest.raises(E):
        ops.tree_attn(z(2, 128, dtype=BF16), z(1, 4, 128, dtype=BF16), z(1, 4, 128, dtype=BF16), z(1, 4, dtype=torch.int32), z(2, 128, dtype=BF16), 1, 1, 128, 128, 1.0, rows=2, max_ctx=2)
    with pytest.raises(E):
        ops.token_logprobs(z(2, 10))
    with pytest.raises(E, match="float8_e4m3fn"):
        ops._cache_view("x", z(1, 4, 128), None, 1, 128, -1)


def test_slots_of_8_bit_rows():
    from lia_b200.seq_state import SlotState
    s = SlotState(3, 17, "cpu")
    for dtype in (torch.int8, E4M3):
        codes, scales = s.add_rows_8bit(4, 64, dtype)
        assert codes.shape == (3, 17, 256) and codes.dtype == dtype and scales.shape == (3, 4, 17) and scales.dtype == F32
    with pytest.raises(ValueError):
        s.add_rows_8bit(4, 64, BF16)


def test_scores_are_put_together(lib, monkeypatch):
    """Engine.score's bookkeeping on a stand-in for a model: the distribution after a token depends on the token and its place alone."""
    from lia_b200 import ops
    from lia_b200.engine import Engine
    from lia_b200.seq_state import SlotState

    class Model:
        device = torch.device("cpu")
        config = type("C", (), {"vocab": 11})

        def new_state(self, n, cap):
            return SlotState(n, cap, "cpu")

        def graph_class(self, n):
            return n

        def forward_rows(self, ids, batch, want, slots, trace=None):
            rows = torch.stack([self.logits(int(t), int(p)) for t, (_, p) in zip(ids, batch.meta.tolist())])
            return None if want is None else rows[want.long()]

        def logits(self, token, place):
            return torch.sin(torch.arange(11.0) * (token + 2) + place)

    def plain(logits, given, top=0):
        logp = torch.log_softmax(logits, -1)
        best, ids = logp.sort(dim=-1, descending=True, stable=True)
        return logp.gather(1, given.view(-1, 1))[:, 0], -(logp.exp() * logp).sum(-1), best[:, :top], ids[:, :top]
    monkeypatch.setattr(ops, "token_logprobs", plain)
    m = Model()
    texts = [[1, 2, 3, 4, 5, 6, 7], [9], [], [3, 3]]
    for chunk, rows in ((None, 4096), (2, 4096), (3, 4), (None, 3)):
        got = Engine(m, 16, max_requests=4, max_rows=rows).score(texts, top=2, chunk=chunk)
        for text, g in zip(texts, got):
            want = [torch.log_softmax(m.logits(t, i), -1) for i, t in enumerate(text[:-1])]
            assert g["logp"] == pytest.approx([float(w[t]) for w, t in zip(want, text[1:])])
            assert [a[0][0] for a in g["alternatives"]] == [int(w.argmax()) for w in want] and all(len(a) == 2 for a in g["alternatives"])
            assert g["entropy"] == pytest.approx([float(-(w.exp() * w).sum()) for w in want])


def test_no_rows_have_no_addresses(lib):
    """What an empty tensor is at the C ABI: a null pointer and no rows; caches and sizes are checked all the same."""
    L, v = lib.load(), view(lib)
    assert L.lia_kv_store_8bit(None, 1024, None, 1024, 0, None, v, v, 0, 8, 0.0, 0, None) == 0
    assert L.lia_kv_load_8bit(None, v, v, None, 1024, None, 1024, 0, 0, 8, None) == 0
    assert L.lia_kv_store_8bit(None, 1024, None, 1024, 0, None, view(lib, data=None), v, 0, 8, 0.0, 0, None) == -1 and "null cache" in lib.last_error()
    assert L.lia_kv_load_8bit(None, v, v, None, 1024, None, 1024, 0, 1, 8, None) == -1 and "null pointer" in lib.last_error()


@pytest.mark.parametrize("cache_dtype", [torch.int8, E4M3], ids=["int8", "e4m3"])
def test_graphs_of_decode_steps_go_by_what_is_launched(lib, cache_dtype):
    """The engine's key of a step of single tokens over 8-bit caches: another one wherever the number of blocks that share a history is another, however long the history, and no other."""
    import types

    from lia_b200.engine import Engine
    from lia_b200.modeling_bebulorn import BebulornForCausalLM
    from lia_b200.seq_layers import WindowAttentionMixer
    H, G, dim, L = 4, 2, 64, lib.load()

    def key(requests, max_ctx, windows):
        m = object.__new__(BebulornForCausalLM)
        m.cache_dtype, m.layers = cache_dtype, []
        for w in windows:
            x = object.__new__(WindowAttentionMixer)
            x.H, x.G, x.dim, x.vdim, x.window, x.cache_dtype = H, G, dim, dim, w, cache_dtype
            m.layers.append(types.SimpleNamespace(mixer=x))
        e = object.__new__(Engine)
        e.model, e.graphs = m, True
        return e._graph_key([(i, [1], []) for i in range(requests)], [(i, max_ctx - 1, i, 1) for i in range(requests)], [])

    def splits(requests, max_ctx, window):
        floats = lambda M: L.lia_tree_attn_workspace_floats(requests, 1, max_ctx, M, H, G, dim, dim, window, 1 if cache_dtype == torch.int8 else 2)  # noqa: E731
        return floats(requests) // (requests * H * (dim + 2))       # (0 up to eight blocks)
    for requests, windows in ((1, [1 << 20]), (3, [1 << 20, 900]), (30, [6000]), (200, [1 << 20])):
        lengths = [1, 255, 256, 257, 512, 513, 2048, 2049, 2304, 2305, 4000, 9000, 20000, 60000]
        for a, b in zip(lengths, lengths[1:]):
            if any(splits(requests, a, w) != splits(requests, b, w) for w in windows):
                assert key(requests, a, windows) != key(requests, b, windows), (requests, a, b)
        assert key(requests, 1, windows) == key(requests, 256, windows) and key(requests, 2049, windows) == key(requests, 2304, windows)
    assert key(1, 256, [5000]) != key(1, 257, [5000]) and key(1, 256, [100]) == key(1, 257, [100]) == key(1, 60000, [100])
    assert key(1, 3000, [1 << 20]) != key(1, 60000, [1 << 20]) and key(200, 3000, [1 << 20]) == key(200, 60000, [1 << 20])


@pytest.mark.parametrize("words,rows", [(0, 1), (0, 3), (1, 65), (2, 129)])
def test_masks_that_hold_too_few_tokens(lib, words, rows):
    """A mask of no words, whose tensor has no address, is not taken for no mask."""
    from lia_b200 import ops
    z, kv = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype), torch.zeros(1, 200, 128, dtype=BF16)  # noqa: E731
    with pytest.raises(lib.LiaError, match=f"{words} words"):
        ops.tree_attn(z(rows, 128), kv, kv, z(1, 4, dtype=torch.int32), z(rows, 128), 1, 1, 128, 128, 1.0, rows=rows, max_ctx=rows, mask=z(rows, words, dtype=torch.int64))


@pytest.mark.parametrize("name", ["OPTForCausalLM", "Davasun", "Bizetar", "Zatusun", "Pazivik", "Sekenex"])
def test_models_without_8_bit_caches_say_so(lib, tmp_path, name):
    """Asked for a cache of 8 bits, a model that has none refuses, before it reads anything; None asks for nothing."""
    import json

    from lia_b200 import registry
    (tmp_path / "config.json").write_text(json.dumps({"architecture": name}))
    with pytest.raises(ValueError, match="no caches of torch.int8"):
        registry.load_model(str(tmp_path), device="cpu", cache_dtype=torch.int8)
    with pytest.raises(ValueError, match="no caches of torch.float8_e4m3fn"):
        registry.model_class(str(tmp_path)).from_pretrained("nowhere", cache_dtype=E4M3)
    with pytest.raises(Exception) as e:                             # (there is no checkpoint to read)
        registry.load_model(str(tmp_path), device="cpu", cache_dtype=None)
    assert "caches of" not in str(e.value)


def test_soft_caps_end_where_scores_would_be_lost(lib):
    """A capped score is off by up to 2^-21 of the cap, whatever the score: of a cap of 10^8 nothing is left of scores of 8, and all would weigh the same."""
    from lia_b200.seq_layers import WindowAttentionMixer
    L, v = lib.load(), view(lib)
    attend = lambda softcap, M: L.lia_tree_attn(256, 2048, v, v, 256, 2, None, 0, None, None, 256, None, 0, M, 16, 8, 4, 40, 0, 1.0, softcap, None)  # noqa: E731
    for softcap in (1025.0, 1e8, float("inf")):
        assert attend(softcap, 8) == -1 and "soft cap" in lib.last_error()
    assert attend(1024.0, 0) == attend(0.0, 0) == attend(-1.0, 0) == 0
    with pytest.raises(ValueError, match="1024"):
        WindowAttentionMixer({}, 4, 2, 64, 64, 40, 0.1, 2000.0, 1e-5, BF16, "cpu", cache_dtype=torch.int8)


def test_scores_of_portions_of_less_than_nothing(lib):
    """A negative portion is refused: no step would be made, and every text would be scored as one without tokens."""
    import types

    from lia_b200.engine import Engine
    from lia_b200.seq_state import SlotState
    m = types.SimpleNamespace(device=torch.device("cpu"), config=types.SimpleNamespace(vocab=11), new_state=lambda n, cap: SlotState(n, cap, "cpu"))
    with pytest.raises(ValueError, match="-2"):
        Engine(m, 16).score([[1, 2, 3]], chunk=-2)
