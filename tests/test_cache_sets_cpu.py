"""Which tensors a set of caches takes: slots, positions and runs of bytes in any order, as long as no two share a byte.  No GPU, no launch."""
import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as g
    g.build()
    import lia_b200  # noqa: F401
    from lia_b200 import _lib
    return _lib


def on(shape, strides):
    """A tensor of these strides in a storage that has just the room for it"""
    return torch.zeros(1 + sum((n - 1) * s for n, s in zip(shape, strides))).as_strided(shape, strides)


@pytest.mark.parametrize("shape,strides", [
    ((2, 8, 8), (8, 8, 1)), ((2, 8, 8), (56, 8, 1)), ((3, 8, 8), (60, 8, 1)),            # slots inside one another
    ((2, 8, 4, 8), (512, 8, 32, 1)), ((2, 8, 4, 8), (512, 16, 24, 1)),                    # positions inside the next piece's
    ((4, 6, 8), (8, 16, 1)), ((4, 6, 8), (0, 8, 1)), ((4, 6, 8), (48, 0, 1)), ((4, 6, 8), (48, 4, 1))])
def test_rows_that_share_bytes_are_refused(lib, shape, strides):
    from lia_b200 import ops
    with pytest.raises(lib.LiaError, match="share"):
        ops.CacheSet([on(shape, strides)])
    size = 4
    pieces = shape[2] if len(shape) == 4 else 1
    r = (lib.LiaCacheRows * 1)(lib.LiaCacheRows(1 << 20, strides[0] * size, strides[1] * size, strides[2] * size if pieces > 1 else 0, shape[-1] * size, pieces, 0))
    L = lib.load()
    assert L.lia_cache_fork(r, 1, shape[0], shape[1], 16, 1, 1, None) == -1 and "share" in lib.last_error()
    assert L.lia_cache_compact(r, 1, shape[0], shape[1], 16, 1, 16, 1, None) == -1 and "share" in lib.last_error()


def test_states_that_share_bytes_are_refused(lib):
    from lia_b200 import ops
    for shape, strides in (((2, 8), (4, 1)), ((3, 4, 4), (8, 4, 1)), ((2, 8), (0, 1))):
        with pytest.raises(lib.LiaError, match="share"):
            ops.CacheSet([], [on(shape, strides)])
    r = (lib.LiaCacheRows * 1)(lib.LiaCacheRows(1 << 20, 16, 0, 0, 32, 1, 1))
    assert lib.load().lia_cache_fork(r, 1, 2, 8, 16, 1, 1, None) == -1 and "share" in lib.last_error()


def test_a_tensor_twice_is_refused(lib):
    """Two blocks would move the same rows at their own pace, the second what the first has moved already."""
    from lia_b200 import ops
    a, b = torch.zeros(3, 20, 8), torch.zeros(3, 20, 8)
    ops.CacheSet([a, b])
    for rows, states in (([a, b, a], []), ([a, a.view(3, 20, 2, 4)], []), ([a], [a])):
        with pytest.raises(lib.LiaError, match="twice"):
            ops.CacheSet(rows, states)


@pytest.mark.parametrize("t", [torch.zeros(3, 20, 8), torch.zeros(20, 3, 8).transpose(0, 1), torch.zeros(3, 4, 20).transpose(1, 2), torch.zeros(3, 4, 20, 2, dtype=BF16).transpose(1, 2),
                               torch.zeros(4, 20, 3, 8).permute(2, 1, 0, 3), torch.zeros(3, 20, 2, 8)[:, :, 1], torch.zeros(1, 20, 8).expand(1, 20, 8), torch.zeros(3, 1, 4, 8)[:, :, 1:3],
                               torch.zeros(1, 1, 5), torch.zeros(3, 40, 8)[:, ::2], torch.zeros(3, 20)])
def test_rows_in_any_order_are_taken(lib, t):
    from lia_b200 import ops
    s = ops.CacheSet([t])
    r = s._rows[0]
    at = lambda slot, pos, piece: slot * r.slot_stride + pos * r.pos_stride + piece * r.piece_stride  # noqa: E731
    places = {at(a, b, c) + d for a in range(s.slots) for b in range(s.capacity) for c in range(r.pieces) for d in range(r.piece_bytes)}
    assert len(places) == t.numel() * t.element_size()
