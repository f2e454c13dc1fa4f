"""Rows of caches copied to other slots, and moved inside one: bytes are bytes, so that everything is equal, and nothing else has changed."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32, U8, I8 = torch.bfloat16, torch.float32, torch.uint8, torch.int8


@pytest.fixture(scope="module")
def ops():
    import lia_b200  # noqa: F401
    from lia_b200 import ops
    return ops


def rnd(*shape, seed=0, dtype=BF16):
    g = torch.Generator("cuda").manual_seed(seed)
    if dtype in (BF16, F32):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)
    return torch.randint(0, 100, shape, generator=g, device="cuda", dtype=torch.int16).to(dtype)


def tensors(slots, cap, seed=0):
    """Rows of every kind: [slots, capacity, ..], and states"""
    rows = [rnd(slots, cap, 1024, seed=seed), rnd(slots, cap, 96, seed=seed + 1, dtype=I8), rnd(slots, 4, cap, seed=seed + 2, dtype=F32).transpose(1, 2),
            rnd(slots, 3, cap, 4, seed=seed + 3).transpose(1, 2), rnd(slots, 3, cap, 1, seed=seed + 4).transpose(1, 2), rnd(cap, slots, 2, 64, seed=seed + 5).transpose(0, 1),
            rnd(slots, cap, 3, 40, seed=seed + 6)[:, :, :, 8:24], rnd(slots, cap, 1, seed=seed + 7, dtype=torch.int32), rnd(slots, cap, 7, seed=seed + 8, dtype=U8),
            rnd(slots, cap + 3, 33, seed=seed + 9)[:, 2:2 + cap], rnd(slots, cap, 2, 3, 64, seed=seed + 10, dtype=U8), rnd(slots, cap, 9000, seed=seed + 11)]
    states = [rnd(slots, 3, 64, 40, seed=seed + 20, dtype=F32), rnd(slots, 5, seed=seed + 21), rnd(slots, 1, seed=seed + 22, dtype=U8), rnd(slots, 2, 70000, seed=seed + 23, dtype=F32)]
    return rows, states


def on_gpu(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def forked(rows, states, copies):
    rows, states = [t.clone() for t in rows], [t.clone() for t in states]
    for a, b, n in copies:
        for t in rows:
            t[b, :n] = t[a, :n].clone()
        for t in states:
            t[b] = t[a].clone()
    return rows, states


@pytest.mark.parametrize("slots,cap,copies,max_count", [
    (4, 50, [(1, 3, 37)], 37), (4, 50, [(1, 3, 37), (1, 0, 50), (1, 2, 1)], 50), (6, 33, [(0, 1, 0), (2, 3, 33), (2, 4, 9)], 1), (3, 2100, [(2, 0, 2077), (2, 1, 13)], 0), (2, 1, [(0, 1, 1)], 5),
    (12, 20, [(11, i, 3 + i) for i in range(11)], 100), (5, 700, [(0, 3, 700), (1, 2, 699)], 64)])
def test_forks(ops, slots, cap, copies, max_count):
    rows, states = tensors(slots, cap)
    want_rows, want_states = forked(rows, states, copies)
    ops.CacheSet(rows, states).fork(on_gpu(copies), max_count=max_count)
    for i, (a, b) in enumerate(zip(rows + states, want_rows + want_states)):
        assert torch.equal(a, b), i


def test_copies_that_are_left_out(ops):
    """Slots that are not there, a slot to itself, counts beyond the capacity or below nothing."""
    rows, states = tensors(4, 20)
    want = forked(rows, states, [(0, 1, 20)])
    for t, s in zip(want[1], states):
        t[2] = s[0].clone()                                                   # (a state goes over whatever the count is)
    ops.CacheSet(rows, states).fork(on_gpu([(0, 1, 1000), (4, 2, 5), (-1, 2, 5), (0, 4, 5), (0, -3, 5), (3, 3, 5), (0, 2, -4), (2 ** 31 - 1, 2, 3), (1 << 20, 1 << 20, 3)]))
    for a, b in zip(rows + states, want[0] + want[1]):
        assert torch.equal(a, b)
    before = [t.clone() for t in rows]
    ops.CacheSet(rows).fork(torch.empty(0, 3, dtype=torch.int32, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(rows, before))


def test_more_tensors_than_a_launch_takes(ops):
    rows = [rnd(3, 40, 8 * (1 + i % 5), seed=i) for i in range(70)]
    states = [rnd(3, 17 + i, seed=100 + i) for i in range(70)]
    want = forked(rows, states, [(2, 0, 31)])
    ops.CacheSet(rows, states).fork(on_gpu([(2, 0, 31)]), max_count=31)
    assert all(torch.equal(a, b) for a, b in zip(rows + states, want[0] + want[1]))
    kept = [[1, 4, 6, -1]]
    want = compacted(rows, [(1, 7, 0, 9)], kept)
    ops.CacheSet(rows).compact(on_gpu([(1, 7, 0, 9)]), on_gpu(kept))
    assert all(torch.equal(a, b) for a, b in zip(rows, want))


def compacted(rows, segs, kept):
    rows = [t.clone() for t in rows]
    for (slot, p0, _, n), list_ in zip(segs, kept):
        last, places = -1, []
        for k in list_:
            if k <= last or k >= n:
                break
            places.append(k)
            last = k
        for t in rows:
            t[slot, p0:p0 + len(places)] = t[slot, [p0 + k for k in places]].clone() if places else t[slot, p0:p0]
    return rows


@pytest.mark.parametrize("slots,cap,segs,kept", [
    (3, 60, [(1, 20, 0, 12)], [[0, 2, 5, 11]]), (3, 60, [(2, 0, 0, 30), (0, 30, 30, 30)], [[0, 1, 2, 3, 4, 29, -1], [3, 7, 8, 9, 20, 21, 22]]),
    (2, 80, [(0, 10, 0, 64)], [list(range(1, 64, 2))]), (2, 80, [(1, 10, 0, 64)], [[0, 1, 2] + list(range(20, 51))]), (2, 9, [(1, 8, 0, 1)], [[0]]),
    (4, 40, [(0, 1, 0, 0), (1, 5, 0, 9), (2, 5, 9, 9), (3, 31, 0, 9)], [[0, 1], [-1, 4], [8, 3], [2, 9]])])
def test_compactions(ops, slots, cap, segs, kept):
    rows, _ = tensors(slots, cap)
    want = compacted(rows, segs, kept)
    ops.CacheSet(rows).compact(on_gpu(segs), on_gpu(kept))
    for i, (a, b) in enumerate(zip(rows, want)):
        assert torch.equal(a, b), i


def test_portions_that_do_not_fit_are_left_out(ops):
    rows, _ = tensors(3, 30)
    before = [t.clone() for t in rows]
    for seg in ((3, 5, 0, 4), (-1, 5, 0, 4), (0, 27, 0, 4), (0, -1, 0, 4), (0, 5, 0, -4), (0, 2 ** 31 - 2, 0, 4), (0, 5, 0, 2 ** 31 - 1)):
        ops.CacheSet(rows).compact(on_gpu([seg]), on_gpu([[1, 3]]))
    assert all(torch.equal(a, b) for a, b in zip(rows, before))
    ops.CacheSet(rows).compact(on_gpu([(0, 5, 0, 4)]), torch.empty(1, 0, dtype=torch.int32, device="cuda"))
    ops.CacheSet(rows).compact(torch.empty(0, 4, dtype=torch.int32, device="cuda"), torch.empty(0, 3, dtype=torch.int32, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(rows, before))


def test_caches_past_32_bits(ops):
    """Slots and positions more than 2^32 bytes into a tensor."""
    cap = 2_200_000
    rows = [torch.empty(2, cap, 1024, dtype=BF16, device="cuda"), torch.empty(2, 8, cap, dtype=F32, device="cuda").transpose(1, 2)]
    for i, t in enumerate(rows):
        t[0, :50], t[0, cap - 30:] = rnd(50, *t.shape[2:], seed=i, dtype=t.dtype), rnd(30, *t.shape[2:], seed=9 + i, dtype=t.dtype)
    tail = [t[0, cap - 30:].clone() for t in rows]
    ops.CacheSet(rows).compact(on_gpu([(0, cap - 30, 0, 30)]), on_gpu([[3, 9, 29]]))
    for t, old in zip(rows, tail):
        assert torch.equal(t[0, cap - 30:cap - 27], old[[3, 9, 29]]) and torch.equal(t[0, cap - 27:], old[3:])
    ops.CacheSet(rows).fork(on_gpu([(0, 1, cap)]), max_count=cap)
    for t in rows:
        assert torch.equal(t[0, :50], t[1, :50]) and torch.equal(t[0, cap - 30:], t[1, cap - 30:])


def test_captured_and_on_another_stream(ops):
    rows, states = tensors(4, 60)
    copies, segs, kept = on_gpu([(0, 1, 20), (0, 2, 30)]), on_gpu([(0, 10, 0, 20)]), on_gpu([[0, 4, 7]])
    both, only = ops.CacheSet(rows, states), ops.CacheSet(rows)
    both.fork(copies)                                                         # (loads the kernels before they are captured)
    only.compact(segs, kept)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        only.compact(segs, kept)
        both.fork(copies, max_count=30)
    copies.copy_(on_gpu([(3, 0, 55), (2, 1, 7)]))
    segs.copy_(on_gpu([(3, 40, 0, 15)]))
    kept.copy_(on_gpu([[2, 14, -1]]))
    want = forked(compacted(rows, [(3, 40, 0, 15)], [[2, 14, -1]]), states, [(3, 0, 55), (2, 1, 7)])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(rows + states, want[0] + want[1]))


def test_sets_that_are_refused(ops):
    from lia_b200._lib import LiaError
    a = rnd(3, 20, 8)
    for rows, states in (([], []), ([a, rnd(2, 20, 8)], []), ([a, rnd(3, 21, 8)], []), ([a, a.cpu()], []), ([a[:, :, :0]], []), ([rnd(3, 1, 8).expand(3, 20, 8)], []), ([rnd(1, 20, 8).expand(3, 20, 8)], []),
                         ([rnd(3, 20, 4, 9, 8)[:, :, :, :3, :5]], []), ([a], [rnd(3, 8, 8).transpose(1, 2)]), ([rnd(3, 20, 1).expand(3, 20, 8)], []), ([rnd(3, 200).as_strided((3, 20, 8), (200, 4, 1))], [])):
        with pytest.raises(LiaError):
            ops.CacheSet(rows, states)
    s = ops.CacheSet([a], [rnd(3, 4)])
    for copies in (on_gpu([(0, 1)]), torch.zeros(1, 3, dtype=torch.int64, device="cuda"), torch.zeros(1, 3, dtype=torch.int32)):
        with pytest.raises(LiaError):
            s.fork(copies)
    with pytest.raises(LiaError, match="state"):
        s.compact(on_gpu([(0, 1, 0, 3)]), on_gpu([[1]]))
    for segs, kept in ((on_gpu([(0, 1, 0, 3)]), on_gpu([[1], [2]])), (on_gpu([(0, 1, 3)]), on_gpu([[1]])), (on_gpu([(0, 1, 0, 3)]), torch.zeros(1, 1, dtype=torch.int64, device="cuda"))):
        with pytest.raises(LiaError):
            ops.CacheSet([a]).compact(segs, kept)
