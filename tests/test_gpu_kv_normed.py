"""Values normed on their way into caches of 4 bits: heads of any size, and groups far below their heads."""
import pytest
import torch

from cache4 import codes_of
from test_gpu_kv_4bit import caches, check_codes, heads

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
