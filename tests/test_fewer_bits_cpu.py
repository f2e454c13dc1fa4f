"""What the operators of serving in fewer bits refuse, and their state's shapes: no GPU, no launch."""
import pytest
import torch

BF16, F32, U8 = torch.bfloat16, torch.float32, torch.uint8


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as g
    g.build()
    import lia_b200  # noqa: F401
    from lia_b200 import _lib
    return _lib


def view(_lib, **change):
    v = dict(data=1 << 20, scale=1 << 21, slot_stride=1 << 15, pos_stride=512, head_stride=64, scale_slot_stride=2048, scale_head_stride=256, slots=2, capacity=64, type=_lib.CACHE_INT4, dim=128)
    return _lib.LiaCacheView(**(v | change))


@pytest.mark.parametrize("change,message", [
    ({"data": None}, "null cache"), ({"scale": None}, "scales"), ({"type": 7}, "type"), ({"type": 1}, "4 bits"), ({"slots": 0}, "empty"), ({"capacity": 0}, "empty"),
    ({"data": (1 << 20) + 4}, "vectors"), ({"pos_stride": 516}, "vectors"), ({"head_stride": 68}, "vectors"), ({"dim": 100}, "multiples of 32"), ({"dim": 2048}, "1024"),
    ({"capacity": 65}, "different sizes"), ({"scale": (1 << 21) + 2}, "scales"), ({"scale_head_stride": 258}, "scales"), ({"scale_slot_stride": 2049}, "scales")])
def test_store_and_load_of_4_bits_refuse(lib, change, message):
    L = lib.load()
    good, bad = view(lib), view(lib, **change)
    for kc, vc in ((bad, good), (good, bad)):
        assert L.lia_kv_store_4bit(16, 1024, 16, 1024, 0, 16, kc, vc, 4, 8, 0.0, 0, None) == -1 and message in lib.last_error()
        assert L.lia_kv_load_4bit(16, kc, vc, 16, 1024, 16, 1024, 0, 4, 8, None) == -1 and message in lib.last_error()


def test_store_of_4_bits_refuses_short_rows_and_null_pointers(lib):
    L, v = lib.load(), view(lib)
    assert L.lia_kv_store_4bit(16, 1023, 16, 1024, 0, 16, v, v, 4, 8, 0.0, 0, None) == -1 and "shorter" in lib.last_error()
    assert L.lia_kv_store_4bit(None, 1024, 16, 1024, 0, 16, v, v, 4, 8, 0.0, 0, None) == -1
    assert L.lia_kv_store_4bit(16, 1024, 16, 1024, 0, None, v, v, 4, 8, 0.0, 0, None) == -1
    assert L.lia_kv_store_4bit(16, 1024, 16, 1024, 0, 16, v, v, -1, 8, 0.0, 0, None) == -1
    assert L.lia_kv_store_4bit(16, 1 << 20, 16, 1 << 20, 0, 16, v, v, 1 << 28, 8, 0.0, 0, None) == -1 and "too many" in lib.last_error()
    assert L.lia_kv_store_4bit(None, 1024, None, 1024, 0, None, v, v, 0, 8, 0.0, 0, None) == 0     # no rows, no launch
    assert L.lia_kv_store_8bit(16, 1024, 16, 1024, 0, 16, v, v, 4, 8, 0.0, 0, None) == -1 and "int8" in lib.last_error()


@pytest.mark.parametrize("change,message", [({"data": (1 << 20) + 8}, "vectors"), ({"dim": 96}, "64 or 128"), ({"dim": 256}, "64 or 128"), ({"type": 1}, "different types"),
                                            ({"slots": 3}, "different types or sizes"), ({"scale": None}, "scales"), ({"scale": (1 << 21) + 4}, "scales")])
def test_attention_refuses_caches_of_4_bits(lib, change, message):
    good, bad = view(lib), view(lib, **change)
    for kc, vc in ((bad, good), (good, bad)):
        assert lib.load().lia_tree_attn(256, 2048, kc, vc, 256, 2, None, 0, None, None, 256, None, 0, 8, 16, 8, 4, 40, 0, 1.0, 0.0, None) == -1 and message in lib.last_error()


def test_views_of_4_bit_caches(lib):
    """Tensors of the wrong shape, type, strides or place raise before anything is launched."""
    from lia_b200 import ops
    z, E = torch.zeros, lib.LiaError
    c, s = z(2, 9, 3 * 64, dtype=U8), z(2, 3, 9, 4, dtype=BF16)
    v = ops._cache_view("x", c, s, 3, 128, -1)
    assert (v.type, v.dim, v.head_stride, v.pos_stride, v.slot_stride) == (lib.CACHE_INT4, 128, 64, 192, 9 * 192) and (v.scale_slot_stride, v.scale_head_stride) == (108, 36)
    v = ops._cache_view("x", z(2, 9, 3, 2, 64, dtype=U8)[:, :, :, 1], s, 3, 128, -1)
    assert (v.head_stride, v.pos_stride) == (128, 384)
    for cache, scale, dim, message in ((z(2, 9, 3 * 128, dtype=U8), s, 128, "bytes"), (c, None, 128, "bf16 scales"), (c, s.float(), 128, "bf16 scales"), (c, z(2, 3, 9, dtype=BF16), 128, "bf16 scales"),
                                       (c, z(2, 3, 9, 8, dtype=BF16)[..., ::2], 128, "neighbours"), (c, z(2, 3, 4, 9, dtype=BF16).transpose(2, 3), 128, "neighbours"),
                                       (z(2, 9, 3 * 24, dtype=U8), s, 48, "multiples of 32"), (z(2, 9, 3 * 128, dtype=U8)[..., ::2], s, 128, "neighbours")):
        with pytest.raises(E, match=message):
            ops._cache_view("x", cache, scale, 3, dim, -1)
    with pytest.raises(E):
        ops.kv_store_4bit(z(2, 128, dtype=BF16), z(2, 128, dtype=BF16), z(2, 2, dtype=torch.int32), z(1, 4, 64, dtype=U8), z(1, 4, 64, dtype=U8), z(1, 1, 4, 4), z(1, 1, 4, 4), 1, 128, 128)


def test_slots_of_4_bit_rows():
    from lia_b200.seq_state import SlotState
    s = SlotState(3, 17, "cpu")
    codes, scales = s.add_rows_4bit(4, 64)
    assert codes.shape == (3, 17, 128) and codes.dtype == U8 and scales.shape == (3, 4, 17, 2) and scales.dtype == BF16
    with pytest.raises(ValueError):
        s.add_rows_4bit(4, 48)


@pytest.mark.parametrize("change,message", [
    ({"x_type": 3}, "type"), ({"x_type": -1}, "type"), ({"M": -1}, "sizes"), ({"N": 0}, "sizes"), ({"K": 0}, "sizes"), ({"ldx": 99}, "sizes"), ({"ldw": 99}, "sizes"),
    ({"K": 131072, "ldx": 131072, "ldw": 131072}, "131071"), ({"x": None}, "null"), ({"w": None}, "null"), ({"w_scale": None}, "null"), ({"out": None}, "null"), ({"x_scale": None}, "null"),
    ({"x_type": 0}, "not codes"), ({"w": 264}, "vectors"), ({"ldw": 120}, "vectors"), ({"x": 264}, "vectors"), ({"ldx": 120}, "vectors"),
    ({"x_type": 0, "x_scale": None, "ws": None}, "workspace"), ({"x_type": 0, "x_scale": None, "bytes": 400}, "workspace"), ({"x_type": 1, "x_scale": None, "ws": 264}, "workspace"),
    ({"N": 1 << 30, "K": 131071, "ldx": 131072, "ldw": 131072}, "too large"),
    ({"M": 1 << 30, "N": 1 << 30}, "too large")])
def test_products_refuse(lib, change, message):
    a = dict(x=256, x_type=2, ldx=112, x_scale=256, w=256, ldw=112, w_scale=256, out=256, f32=0, M=4, N=64, K=100, ws=256, bytes=1 << 30) | change
    rc = lib.load().lia_linear_int8(a["x"], a["x_type"], a["ldx"], a["x_scale"], a["w"], a["ldw"], a["w_scale"], a["out"], a["f32"], a["M"], a["N"], a["K"], a["ws"], a["bytes"], None)
    assert rc == -1 and message in lib.last_error()


def test_products_of_no_tokens_and_their_workspace(lib):
    L = lib.load()
    assert L.lia_linear_int8(None, 0, 100, None, 256, 112, 256, None, 0, 0, 64, 100, None, 0, None) == 0
    assert L.lia_linear_int8_workspace_bytes(0, 0, 64, 100) == L.lia_linear_int8_workspace_bytes(0, 4, 64, 131072) == 0
    assert L.lia_linear_int8_workspace_bytes(0, 300, 64, 100) >= 300 * (112 + 4) and L.lia_linear_int8_workspace_bytes(2, 300, 64, 100) == 0
    assert L.lia_quantize_rows(None, 0, 8, None, 8, None, 0, 8, None) == 0
    for args, message in (((16, 0, 7, 16, 8, 16, 2, 8), "sizes"), ((16, 0, 8, 16, 7, 16, 2, 8), "sizes"), ((None, 0, 8, 16, 8, 16, 2, 8), "null"), ((16, 0, 8, 20, 8, 16, 2, 8), "vectors"),
                          ((16, 0, 12, 16, 12, 16, 2, 8), "vectors"), ((16, 0, 8, 16, 8, None, 2, 8), "null")):
        assert L.lia_quantize_rows(*args, None) == -1 and message in lib.last_error()


def test_wrappers_of_products_refuse(lib):
    from lia_b200 import ops
    z, E = torch.zeros, lib.LiaError
    with pytest.raises(E):
        ops.quantize_rows(z(2, 8, dtype=BF16))                                # not on a GPU
    with pytest.raises(E):
        ops.linear_int8(z(2, 8, dtype=BF16), z(4, 8, dtype=torch.int8), z(4))


def test_models_say_which_weights_they_can_hold(lib, tmp_path):
    from lia_b200.checkpoint import no_cache_dtype
    from lia_b200.modeling_bebulorn import BebulornConfig, BebulornForCausalLM
    with pytest.raises(ValueError, match="weight_dtype"):
        BebulornForCausalLM(BebulornConfig(), "cpu", BF16, weight_dtype=torch.float8_e4m3fn)
    for cls in (BebulornForCausalLM, str):
        with pytest.raises(ValueError, match="weight_dtype"):
            no_cache_dtype(cls, {"weight_dtype": torch.int8})


def test_forks_of_host_resident_state():
    from lia_b200.seq_state import SlotError, SlotState
    s = SlotState(4, 9, "cpu")
    r, (c, a) = s.add_recurrent((2, 3)), s.add_rows_8bit(2, 16, torch.int8)
    rows, (c4, a4) = s.add_rows(5, F32), s.add_rows_4bit(3, 32)
    assert s.alloc("x") == 0 and s.alloc("y") == 1 and s.reserve(1, 4) == 0
    for t in (r, c, a, rows, c4, a4):
        t[1] = torch.randint(1, 9, t.shape[1:], generator=torch.Generator().manual_seed(1)).to(t.dtype)
    s.free("x")
    assert s.fork("y", ["p", "q"]) == [0, 2] and s.length == [4, 4, 4, 0] and s.slot_of("q") == 2
    for t, axis in ((c, 0), (a, 1), (rows, 0), (c4, 0), (a4, 1)):
        for to in (0, 2):
            assert torch.equal(t[to].narrow(axis, 0, 4), t[1].narrow(axis, 0, 4)) and (t[to].narrow(axis, 4, 5) == 0).all()
    assert torch.equal(r[0], r[1]) and torch.equal(r[2], r[1]) and (r[3] == 0).all()
    for who, ids in (("z", ["u"]), ("y", ["p"]), ("y", ["u", "u"]), ("y", ["u", "v"])):
        with pytest.raises(SlotError):
            s.fork(who, ids)
    assert s.owner == ["p", "y", "q", None] and s.length == [4, 4, 4, 0]                # nothing of them was done
    assert s.reserve(2, 5) == 4 and s.fork("q", ["w"]) == [3] and s.length == [4, 4, 9, 9]


def rows(_lib, **change):
    return (_lib.LiaCacheRows * 1)(_lib.LiaCacheRows(**(dict(data=1 << 20, slot_stride=4096, pos_stride=64, piece_stride=0, piece_bytes=64, pieces=1, state=0) | change)))


@pytest.mark.parametrize("change,message", [({"data": None}, "null"), ({"pieces": 0}, "bytes"), ({"piece_bytes": 0}, "bytes"), ({"piece_bytes": 1 << 31}, "bytes"), ({"slot_stride": -64}, "share"),
                                            ({"slot_stride": 0}, "share"), ({"pos_stride": 0}, "share"), ({"pos_stride": 63}, "share"), ({"pieces": 2, "piece_bytes": 32, "piece_stride": 16}, "share"), ({"state": 1, "pieces": 2}, "pieces")])
def test_moves_refuse_tensors(lib, change, message):
    L = lib.load()
    assert L.lia_cache_fork(rows(lib, **change), 1, 4, 64, 16, 1, 1, None) == -1 and message in lib.last_error()
    assert L.lia_cache_compact(rows(lib, **change), 1, 4, 64, 16, 1, 16, 1, None) == -1 and message in lib.last_error()


def test_moves_refuse_sizes_and_null_pointers(lib):
    L, r = lib.load(), rows(lib)
    for args in ((r, -1, 4, 64, 16, 1, 1), (r, 1, 0, 64, 16, 1, 1), (r, 1, 4, 0, 16, 1, 1), (r, 1, 4, 64, 16, -1, 1), (None, 1, 4, 64, 16, 1, 1), (r, 1, 4, 64, None, 1, 1)):
        assert L.lia_cache_fork(*args, None) == -1
    for args in ((r, -1, 4, 64, 16, 1, 16, 1), (r, 1, 4, 64, 16, -1, 16, 1), (r, 1, 4, 64, 16, 1, 16, -1), (r, 1, 4, 64, None, 1, 16, 1), (r, 1, 4, 64, 16, 1, None, 1), (r, 1, 4, 64, 16, 70000, 16, 1)):
        assert L.lia_cache_compact(*args, None) == -1
    assert L.lia_cache_compact(rows(lib, state=1), 1, 4, 64, 16, 1, 16, 1, None) == -1 and "state" in lib.last_error()
    assert L.lia_cache_fork(None, 0, 4, 64, None, 0, 0, None) == L.lia_cache_compact(None, 0, 4, 64, None, 0, None, 0, None) == 0


def test_choices_are_put_together(lib, monkeypatch):
    """Engine.score_choices' bookkeeping on a stand-in for a model whose distribution after a token depends on all tokens before it: what a fork carries on is a recurrent sum."""
    from lia_b200 import ops
    from lia_b200.engine import Engine
    from lia_b200.seq_state import SlotState

    class Model:
        device = torch.device("cpu")
        config = type("C", (), {"vocab": 11})
        steps = 0

        def new_state(self, n, cap):
            s = SlotState(n, cap, "cpu")
            s.sums = s.add_recurrent(())
            return s

        def forward_rows(self, ids, batch, want, slots, trace=None):
            self.steps += len(ids)
            out = []
            for t, (slot, _) in zip(ids.tolist(), batch.meta.tolist()):
                slots.sums[slot] = slots.sums[slot] * 0.5 + t
                out.append(self.logits(slots.sums[slot]))
            return None if want is None else torch.stack(out)[want.long()]

        def logits(self, x):
            return torch.sin(torch.arange(11.0) * (x + 2))

    def plain(logits, given, top=0):
        logp = torch.log_softmax(logits, -1)
        best, ids = logp.sort(dim=-1, descending=True, stable=True)
        return logp.gather(1, given.view(-1, 1))[:, 0], -(logp.exp() * logp).sum(-1), best[:, :top], ids[:, :top]
    monkeypatch.setattr(ops, "token_logprobs", plain)
    choices = [[1, 2, 3], [9], [3, 3], [4, 5, 6, 7]]
    for prompt in ([8, 1, 5, 2], [6]):
        for requests in (1, 2, 3, 9) if len(prompt) == 1 else (2, 3, 9):
            m = Model()
            e = Engine(m, 16, max_requests=requests)
            got = e.score_choices(prompt, choices, top=2)
            assert e.slots.live_tokens == 0 and m.steps == len(prompt) - 1 + sum(len(c) for c in choices)      # the prompt once
            for c, g in zip(choices, got):
                x = torch.zeros(())
                logps = []
                for t in prompt + c[:-1]:
                    x = x * 0.5 + t
                    logps.append(torch.log_softmax(m.logits(x), -1))
                want = [float(w[t]) for w, t in zip(logps[-len(c):], c)]
                assert g["logp"] == pytest.approx(want) and all(len(a) == 2 for a in g["alternatives"])
    from lia_b200.seq_state import SlotError
    with pytest.raises(SlotError):
        Engine(Model(), 16, max_requests=1).score_choices([8, 1], choices)


def test_costs_of_the_operators():
    """What the comparison benchmark counts for them: bytes of codes and scales, half the operations of a product in 8 bits (which run at twice the rate)."""
    from lia_b200 import bench_compare
    e = lambda *s, dt=BF16: torch.empty(*s, dtype=dt)  # noqa: E731
    cost = bench_compare._cost
    assert cost("kv_store_4bit", (e(10, 256), e(10, 128)), {}) == (0.0, 10 * 384 * 2.5625, "mem") and cost("quantize_rows", (e(3, 64, dt=F32),), {}) == (0.0, 3 * (64 * 5 + 4), "mem")
    assert cost("linear_int8", (e(5, 64), e(7, 64, dt=torch.int8)), {"out": e(5, 7, dt=F32)}) == (5 * 7 * 64, 7 * 64 + 28 + 5 * 64 * 2 + 5 * 7 * 4, "tc")
    q, cache = e(4, 8 * 64), e(2, 100, 2 * 32, dt=U8)
    assert cost("tree_attn", (q, cache, cache, None, q, 8, 2, 64, 64), {"_wkeys": 50, "_wctx": 50}) == (2 * 50 * 8 * 128, 2 * 4 * 512 * 2 + 50 * 2 * 72, "tc")
