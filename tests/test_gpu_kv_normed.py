"""Values normed on their way into caches of 4 and 8 bits: heads of any size, and groups far below their heads."""
import pytest
import torch

from cache4 import codes_of
from test_gpu_kv_4bit import caches, check_codes, heads
from test_gpu_kv_8bit import caches as caches8

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    import lia_b200  # noqa: F401
    from lia_b200 import ops
    return ops


def normed(x, eps):
    """x [M, G, dim], 64 bits"""
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt()


@pytest.mark.parametrize("act", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("size", [0, -30, -60])
@pytest.mark.parametrize("dim", [128, 288])
def test_groups_of_nothing_in_small_heads(ops, act, size, dim):
    """A group of zeros, or of numbers far below the others', has codes of its own size however small the head is."""
    G, M = 2, 40
    x = torch.randint(-255, 256, (M, G, dim), generator=torch.Generator("cuda").manual_seed(3), device="cuda").float()
    x[::2, :, 32:64] = 0
    x[1::2, :, 64:96] *= 2.0 ** -60
    x = (x * 2.0 ** size).to(act)
    meta = torch.tensor([(0, i) for i in range(M)], dtype=torch.int32, device="cuda")
    (kc, ks), (vc, vs) = caches(1, M, G, dim), caches(1, M, G, dim)
    ops.kv_store_4bit(x.view(M, -1), x.view(M, -1), meta, kc, vc, ks, vs, G, dim, dim, norm_values=True)
    check_codes(vc, vs, normed(x.double(), 0.0), meta, G, True, "values")
    assert (codes_of(heads(vc, G)[0], dim)[::2, :, 32:64] == 0).all()


@pytest.mark.parametrize("act", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("kind", ["int4", torch.int8, torch.float8_e4m3fn], ids=str)
def test_heads_at_the_edges_of_32_bits(ops, act, kind):
    """Squares are summed in 32 bits, as by every norm here: heads up to 2^60 are what they are; larger ones, whose root is infinite, are zeros, and finite; an infinity or NaN makes NaN of its group or head;
    heads of zeros, or of numbers whose squares are nothing, have no root without eps, and are zeros with it.  Each beside heads that must not notice."""
    G, dim, M = 1, 128, 64
    x = torch.randn(M, G, dim, generator=torch.Generator("cuda").manual_seed(5), device="cuda").clamp(-4, 4)
    x[1::8] *= 2.0 ** 58
    x[2::8] *= 2.0 ** 90
    x[3::8] = 3e38
    x[4::8, :, 7] = float("inf")
    x[5::8, :, 7] = float("nan")
    x[6::8] = 0
    x[7::8] *= 2.0 ** -90
    x = x.to(act)
    meta = torch.tensor([(0, i) for i in range(M)], dtype=torch.int32, device="cuda")
    make = (lambda: caches(1, M, G, dim)) if kind == "int4" else (lambda: caches8(1, M, G, dim, kind))
    store, load = (ops.kv_store_4bit, ops.kv_load_4bit) if kind == "int4" else (ops.kv_store_8bit, ops.kv_load_8bit)
    for eps in (0.0, 1e-6):
        (kc, ks), (vc, vs) = make(), make()
        store(x.view(M, -1), x.view(M, -1), meta, kc, vc, ks, vs, G, dim, dim, eps=eps, norm_values=True)
        k, v = torch.empty(M, dim, device="cuda"), torch.empty(M, dim, device="cuda")
        load(meta, kc, vc, ks, vs, k, v, G, dim, dim)
        want = normed(x.double(), eps).view(M, dim)
        for i in (0, 1):                                                    # half a step of a group's or head's largest, and a scale of 8 bits for 7 steps
            step = 0.5 / 7 + 2.0 ** -8 if kind == "int4" else 0.5 / 127 if kind == torch.int8 else 2.0 ** -4
            assert ((v[i::8].double() - want[i::8]).abs() <= step * 1.01 * want[i::8].abs().amax(-1, keepdim=True)).all()
        assert (v[2::8] == 0).all() and (v[3::8] == 0).all()
        spoilt = slice(0, 32) if kind == "int4" else slice(0, dim)
        assert torch.isnan(v[4::8, spoilt]).all() and torch.isnan(v[5::8]).all()
        if kind == "int4":
            assert (v[4::8, 32:] == 0).all()
        assert (torch.isnan(v[6::8]) if eps == 0 else v[6::8] == 0).all()
        assert (torch.isnan(v[7::8]) if eps == 0 else v[7::8].abs() <= 2.0 ** -75).all()
