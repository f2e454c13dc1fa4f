"""Attention over 4-bit caches with windows where all histories are cut into equal spans: histories that begin inside a unit of 64 keys, shorter and longer than the window, masks and depths over them.
Every case here takes spans (its plan says so).  Tolerances: tests/test_gpu_tree_attn_4bit.py."""
import pytest
import torch

from test_gpu_tree_attn import DIMS, family
from test_gpu_tree_attn_4bit import Case4

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import lia_b200  # noqa: F401
    from lia_b200 import ops
    return ops


@pytest.mark.parametrize("dim,vdim", DIMS)
@pytest.mark.parametrize("H,G,n,masked,window,most", [(8, 8, 1, False, 20500, 30000), (16, 8, 4, True, 21000, 24000), (8, 8, 8, True, 20400, 20390), (24, 8, 1, False, 32000, 40000), (4, 1, 2, True, 450000, 9000)])
def test_windows_over_equal_spans(ops, dim, vdim, H, G, n, masked, window, most):
    past = [most, window - 1, window, window + 1, 0, 63, 12345 % most, window + 77, 1, most // 2, 300] if most > 20000 else [most, 0, 700, 5000]
    past = [min(p, most) for p in past]
    portions = [(i, p, max(1, n - i % 3)) for i, p in enumerate(past)]
    tree = lambda m: family(m, lambda i: (i - 1) // 2 if i else -1)  # noqa: E731
    deep = [[int(tree(m)[i].sum()) - 1 for i in range(m)] for _, _, m in portions] if masked else None
    c = Case4(portions, H, G, dim, vdim, mask=[tree(m) for _, _, m in portions] if masked else None, depth=deep, window=window, gap=1)
    rows, long = max(s[3] for s in c.segs), most + n
    while not lib_plan(len(portions), rows, long, H, G, window) >> 30 and long < 1 << 24:      # (how long a history is said to be decides the plan, not what is read)
        long *= 2
    assert lib_plan(len(portions), rows, long, H, G, window) >> 30
    out = c.run(ops, rows=rows, max_ctx=long).clone()
    c.check(out)
    assert torch.equal(out, c.run(ops, rows=rows, max_ctx=long, out=torch.full_like(out, 77.0)))


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("window", [530, 700])
def test_short_windows_of_many_requests(ops, masked, window):
    """Windows of a few units, most of them cut at both ends: 64 requests of 56 key heads."""
    n = 5
    tree = family(n, lambda i: (i - 1) // 2 if i else -1)
    past = [(37 * i * i) % 1500 for i in range(64)]
    past[:6] = [0, 1, window - 1, window, window + 1, 1499]
    deep = [int(tree[i].sum()) - 1 for i in range(n)]
    c = Case4([(i % 8, p, n if i % 5 else 1) for i, p in enumerate(past)], 56, 56, 64, 64, mask=[tree if i % 5 else tree[:1, :1] for i in range(64)] if masked else None,
              depth=[deep] * 64 if masked else None, window=window, cap=1600)
    assert lib_plan(64, n, 1510, 56, 56, window) >> 30
    c.check(c.run(ops, rows=n, max_ctx=1510))


def lib_plan(nseg, rows, max_ctx, H, G, window):
    from lia_b200 import _lib
    return _lib.load().lia_tree_attn_plan(nseg, rows, max_ctx, H, G, window, 3)
