"""One round of serving with a drafted tree, operators together: the tree's keys and values are stored behind the histories, its nodes attend, their children's log probabilities are looked up, and the
path that is kept moves to where its tokens belong, where the next token attends to it.  Beside it a second cache, in which the path was written as a chain from the start: the same codes at other
places.

An output is off by at most 2^-8 of itself, and 3 * 2^-11 + 2^-10 of the weighted magnitudes (scores below 2^5 in size, whose error of 2^-12 counts twice at most): two such ones by 2 (2^-8 + 2^-8) of the
largest value.  A row moved by way of fp32 reads back as it was.  e4m3: a number is a code times a power of two, exactly; where the head's largest, 224 to 232 of its scale, was rounded to 224, the
least scale that holds it is half of that, and codes of up to 224 double exactly.  int8: the largest code is 127, so a is 127 scale rounded once, the new scale a / 127 rounded once more, and code *
scale * 127 / a within 2^-21 of the old code, which is thus the new one; so numbers are within 2^-22 of themselves."""
import pytest
import torch

import lia_b200  # noqa: F401
from lia_b200 import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn], ids=["int8", "e4m3"])
@pytest.mark.parametrize("H,G,n,branch", [(4, 2, 13, 2), (8, 1, 29, 2), (4, 4, 64, 3)])
def test_round(kind, H, G, n, branch):
    D, V, past, cap = 128, 503, (37, 300), 400
    g = torch.Generator(device="cuda").manual_seed(n)
    rnd = lambda *s, std=1.0: torch.randn(*s, generator=g, device="cuda") * std  # noqa: E731
    ints = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device="cuda")  # noqa: E731

    def cache():
        codes = [torch.zeros(2, cap, G * D, dtype=torch.uint8, device="cuda").view(kind) for _ in range(2)]
        return codes + [torch.zeros(2, G, cap, device="cuda") for _ in range(2)]

    def store(c, k, v, places):
        ops.kv_store_8bit(k, v, ints(places), *c, G, D, D)

    def attend(c, q, segs, **kw):
        out = torch.empty(q.shape[0], H * D, dtype=BF16, device="cuda")
        return ops.tree_attn(q, c[0], c[1], ints(segs), out, H, G, D, D, D ** -0.5, rows=max(s[3] for s in segs), max_ctx=cap, k_scale=c[2], v_scale=c[3], **kw)

    parent = [(j - 1) // branch if j else -1 for j in range(n)]
    path = [n - 1]
    while parent[path[0]] >= 0:
        path.insert(0, parent[path[0]])
    deep, bits = [0] * n, [0] * n
    for j in range(n):
        deep[j], bits[j] = (deep[parent[j]] + 1, bits[parent[j]]) if j else (0, 0)
        bits[j] |= 1 << j
    bits = [b - (1 << 64) if b >> 63 else b for b in bits]
    tree, chain = cache(), cache()
    for s, p in enumerate(past):
        k, v = rnd(p, G * D).to(BF16), rnd(p, G * D).to(BF16)
        for c in (tree, chain):
            store(c, k, v, [(s, t) for t in range(p)])
    q, k, v = rnd(2 * n, H * D).to(BF16), rnd(2 * n, G * D).to(BF16), rnd(2 * n, G * D).to(BF16)
    kept = ints([s * n + j for s in range(2) for j in path], torch.int64)
    most = v.abs().max().item()                                     # (histories' values are of the same size)
    near = lambda a, b: ((a.float() - b.float()).abs() <= 2.0 ** -6 * most).all()  # noqa: E731

    # the tree's nodes attend, as the chain's tokens do
    store(tree, k, v, [(s, p + j) for s, p in enumerate(past) for j in range(n)])
    got = attend(tree, q, [(s, p, s * n, n) for s, p in enumerate(past)], mask=ints(bits * 2, torch.int64)[:, None], depth=ints(deep * 2))
    belong = [(s, p + i) for s, p in enumerate(past) for i in range(len(path))]
    store(chain, k[kept], v[kept], belong)
    want = attend(chain, q[kept], [(s, p, s * len(path), len(path)) for s, p in enumerate(past)])
    assert near(got[kept], want)

    # how likely each node's children are, from its logits
    logits = rnd(2 * n, V, std=3.0).to(BF16)
    children = torch.randint(0, V, (2 * n, branch), generator=g, device="cuda")
    logp, entropy, best, ids = ops.token_logprobs(logits, children, top=branch)
    exact = torch.log_softmax(logits.double(), -1)
    assert (logp - exact.gather(1, children)).abs().max() < 2e-5 and (entropy + (exact.exp() * exact).sum(-1)).abs().max() < 1e-4
    assert torch.equal(exact.gather(1, ids), exact.topk(branch).values) and (best - exact.gather(1, ids)).abs().max() < 2e-5

    # the kept path moves to where it belongs
    moved = torch.empty(len(kept), G * D, device="cuda"), torch.empty(len(kept), G * D, device="cuda")
    ops.kv_load_8bit(ints([(s, p + j) for s, p in enumerate(past) for j in path]), *tree, *moved, G, D, D)
    store(tree, *moved, belong)
    for s, p in enumerate(past):
        end = p + len(path)
        for a, ka, b, kb in ((tree[0], tree[2], chain[0], chain[2]), (tree[1], tree[3], chain[1], chain[3])):
            x, y = (c[s, :end].float().view(end, G, D) * f[s, :, :end].t()[..., None] for c, f in ((a, ka), (b, kb)))
            assert ((x - y).abs() <= (2.0 ** -22 if kind == torch.int8 else 0.0) * y.abs()).all()

    # and the next token attends to it
    k, v, q = rnd(2, G * D).to(BF16), rnd(2, G * D).to(BF16), rnd(2, H * D).to(BF16)
    for c in (tree, chain):
        store(c, k, v, [(s, p + len(path)) for s, p in enumerate(past)])
    segs = [(s, p + len(path), s, 1) for s, p in enumerate(past)]
    assert near(attend(tree, q, segs), attend(chain, q, segs))
