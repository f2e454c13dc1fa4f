"""Attention of drafted tokens on tcgen05 (csrc/tree_attn_sm100.cu) whose waits run out at once: a launch ends and counts its blocks, and every row is formed again from the keys that it sees, so that
results are right all the same."""
import pytest
import torch

from test_gpu_tree_attn import Case, KINDS, family
from test_gpu_wait_limits import given_up, nowait  # noqa: F401
from lia_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("H", [4, 8])                               # rows of a key head: 128, 80 and 66, or twice as many
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("max_ctx", [364, 100000])                  # how many blocks share a history, and with which rows, goes by it
def test_rows_are_formed_again(nowait, monkeypatch, kind, H, masked, max_ctx):  # noqa: F811
    sizes = (64, 40, 33)
    mask = [family(n, lambda i: (i - 1) // 2 if i else -1) for n in sizes] if masked else None
    c = Case([(0, 300, sizes[0]), (1, 70, sizes[1]), (2, 5, sizes[2])], H, 2, 128, 64, kind, mask=mask, gap=1)
    again = torch.full_like(c.out, 77.0)
    assert given_up(nowait, monkeypatch, lambda: c.run(ops, out=again, max_ctx=max_ctx)) >= 3 * 2      # a block at least for each portion and key head
    torch.cuda.synchronize()
    c.check(again, kind)
    c.check(c.run(ops, max_ctx=max_ctx), kind)


def test_rows_that_are_right_raise_nothing(nowait, monkeypatch):  # noqa: F811
    """What the engine asks about are waits that left NaN: those of drafted tokens leave rows that are right, and are counted apart."""
    c = Case([(0, 300, 64)], 4, 2, 128, 64, "int8")
    seen = nowait.lia_moe_timeouts_seen()
    assert given_up(nowait, monkeypatch, lambda: c.run(ops)) >= 2
    c.check(c.out, "int8")
    assert nowait.lia_moe_timeouts_seen() == seen
