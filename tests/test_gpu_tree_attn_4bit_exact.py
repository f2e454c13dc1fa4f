"""Attention over caches of 4 bits where many rows take tcgen05: codes times their groups' scales are exact there, as with few rows.

A bf16 scale has 8 bits and a code 3 (-8 is a sign and a shift), so that their product relative to a power of two has 11, which is what fp16 holds.  What is left of the tolerances in
tests/test_gpu_tree_attn.py is then, with more than 32 rows too: the output's own rounding, 2^-8 of it; weights in fp16, 2^-11 of A; a score's sum of products, dim 2^-24 of B; 2^-21 of its size and
2^-20 for factors and powers; and 2^-24 of A for each of the weighted values' sums (a product adds 16 keys and its halves are cut off: 2^-23 for every 16 keys, and as much where it begins).

Weights that are small beside a row's largest: that one is 2^7 to 2^15 in fp16, whose numbers below 2^-14 are 2^-24 apart, so that such a weight is off by 2^-25, which is 2^-32 of the largest at most.  A
channel of which the largest weights' keys have a code of 0 is made of these: 2^-32 of the row's largest p for every key, times that key's value.  (Scales are within a factor of 64, so that the values' part of
the weights is one power of two for all.  Where a test has them further apart, a position's part z of the weights is a power of two within a factor of 2 of its largest scale y: then it is 2^-32 of the row's
largest p z, over z, for every key: 4 times that with y.)

Groups below 2^-23 of their position's largest scale y: that one's power of two is 2^6 in fp16, so that such a group's scale is below 2^-16 there and is off by up to half of 2^-24 for its factor, times a code
of 8, and as much for the product: 9 * 2^-25, which is 9 * 2^-31 of y for each of the position's channels in that group."""
import pytest
import torch

from cache4 import numbers, packed
from test_gpu_tree_attn import INF, rnd
from test_gpu_tree_attn_4bit import Case4

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    import lia_b200  # noqa: F401
    from lia_b200 import ops
    return ops


class Exact(Case4):
    apart = False                                                           # values' scales further apart than a factor of 64, each position's weights with its own part

    def check(self, out):
        for z, (s, p0, r, n) in enumerate(self.segs):
            see = self.visible(z)
            for h in range(self.H):
                g = h // (self.H // self.G)
                k, v = numbers(self.kc[s, :p0 + n, g], self.ks[s, g, :p0 + n], self.dim), numbers(self.vc[s, :p0 + n, g], self.vs[s, g, :p0 + n], self.vdim)
                q = self.q[r:r + n, h * self.dim:(h + 1) * self.dim].double()
                x, B = q @ k.t() * self.scale, torch.where(see, q.abs() @ k.abs().t() * self.scale, 0.0).amax(1, keepdim=True)
                if self.softcap:
                    x = self.softcap * torch.tanh(x / self.softcap)
                S = torch.where(see, x.abs(), torch.zeros_like(x)).amax(1, keepdim=True)
                p = torch.softmax(x.masked_fill(~see, -INF), -1)
                o, A = p @ v, p @ v.abs()
                d = self.dim * 2.0 ** -24 * B + 2.0 ** -21 * (S + self.softcap) + 2.0 ** -20
                y = 2 * self.vs[s, g, :p0 + n].double().amax(-1) if self.apart else torch.ones(p0 + n, dtype=torch.float64, device="cuda")
                small = 2.0 ** -32 * (p * y).amax(1, keepdim=True) * (see.double() @ (v.abs() * (4 / y if self.apart else y)[:, None]))
                groups, most = self.vs[s, g, :p0 + n].double(), self.vs[s, g, :p0 + n].double().amax(-1, keepdim=True)
                far = p @ torch.where(groups < 2.0 ** -23 * most, 9 * 2.0 ** -31 * most, 0.0).repeat_interleave(32, -1)
                tol = 2.0 ** -8 * o.abs() + (2.0 ** -11 + 2 * d + (p0 + n + 32) * 2.0 ** -24) * A + small + far + 1e-30
                off = ((out[r:r + n, h * self.vdim:(h + 1) * self.vdim].double() - o).abs() / tol)
                assert not torch.isnan(off).any() and off.max() <= 1, (z, h, off.max().item(), off.argmax().item())


def far_from_fp16():
    """Two scales of 8 bits, larger and smaller, whose quotient in fp16, times 7 and rounded again, is further from itself than that of any others."""
    m = torch.arange(128, 256, dtype=torch.float64) / 128
    f = (m[None] / m[:, None])
    y = ((f.half() * 7).double() - 7 * f) / (7 * f)
    y = torch.where(f < 1, y, torch.zeros_like(y))
    at = int(y.argmax())
    return float(m[at // 128]), float(m[at % 128])


@pytest.mark.parametrize("n,H,G,softcap", [(40, 2, 2, 0.0), (70, 4, 2, 0.0), (130, 4, 1, 0.0), (40, 2, 2, 200.0)])
def test_keys_scores_are_exact(ops, n, H, G, softcap):
    """Scores of 60 of keys that differ in nothing but their scales, with values of both signs: what an output is, is what a hundredth of a score decides."""
    large, small = far_from_fp16()
    c = Exact([(0, 300, n), (1, 200, n)], H, G, 128, 128, softcap=softcap)
    signs = torch.where(rnd(128, seed=8) > 0, 1, -1)
    s = torch.full((300, 4), float(torch.tensor((large + 3 * small) / 4).to(BF16)))
    s[::2] = torch.tensor([large, small, small, small])
    v = torch.where(torch.arange(300) % 2 == 0, 7, -7)[:, None, None].expand(300, G, 128)
    for slot, past in ((0, 300), (1, 200)):
        c.kc[slot, :past] = packed((7 * signs).expand(past, G, 128))
        c.ks[slot, :, :past] = s[:past].cuda().to(BF16)
        c.vc[slot, :past] = packed(v[:past].cuda())
        c.vs[slot, :, :past] = 0.125
    c.q = (signs.float() * 60 / (7 * 32 * (large + 3 * small) * c.scale)).to(BF16).repeat(c.M, H)
    c.check(c.run(ops))


@pytest.mark.parametrize("n,H,G", [(40, 2, 2), (66, 4, 2), (300, 4, 2)])
def test_large_scores_of_any_keys(ops, n, H, G):
    c = Exact([(1, 400, n), (0, 77, n)], H, G, 128, 64)
    c.q *= 8
    c.ks[..., 2] *= 2.0 ** -13                                              # and what such a group is asked for by
    c.q.view(c.M, H, 4, 32)[:, :, 2] *= 2.0 ** 10
    c.check(c.run(ops))


@pytest.mark.parametrize("n", [5, 40])
def test_codes_of_minus_eight(ops, n):
    """Stores give -7 to 7; a code of -8 is a number like the others."""
    c = Exact([(0, 200, n)], 2, 2, 64, 128)
    c.kc.copy_(torch.randint(0, 256, c.kc.shape, dtype=torch.int16, generator=torch.Generator("cuda").manual_seed(3), device="cuda").to(torch.uint8))
    c.vc.copy_(torch.randint(0, 256, c.vc.shape, dtype=torch.int16, generator=torch.Generator("cuda").manual_seed(4), device="cuda").to(torch.uint8))
    c.ks.copy_((c.ks.float() * 0 + 1.9921875).to(BF16))
    c.vs.copy_((c.vs.float() * 0 + 1.9921875).to(BF16))
    c.q *= 0.1
    c.check(c.run(ops))


@pytest.mark.parametrize("n,H,G,softcap", [(40, 4, 2, 0.0), (130, 4, 2, 0.0), (40, 2, 2, 30.0)])
@pytest.mark.parametrize("up", [5, 12])
@pytest.mark.parametrize("down", [9, 14, 17, 20])
def test_small_groups_of_values(ops, n, H, G, softcap, up, down):
    """A large value among the first 64 positions, whose scale the others' go by as long as they are near it, and a group of channels far below the others: its channels are as exact as theirs."""
    c = Exact([(0, 300, n), (1, 64, n)], H, G, 128, 128, softcap=softcap)
    c.apart = up > 6
    c.vs[:, :, 5, 0] *= 2.0 ** up
    c.vs[:, :, 5, 2:] *= 2.0 ** up
    c.vs[:, :, :, 1] *= 2.0 ** -down
    c.check(c.run(ops))


@pytest.mark.parametrize("n", [40, 130])
def test_groups_of_nothing_beside_others(ops, n):
    """Groups of zeros have scales near 2^-103 or of 0: the position's other channels, and its rows' sums, are what they are."""
    c = Exact([(0, 300, n)], 4, 2, 128, 64)
    c.vs[:, :, ::3, 0] = 2.0 ** -103
    c.vs[:, :, 1::3, 1] = 0
    c.vs[:, :, 2::9] = 0
    c.ks[:, :, ::4, 3] = 2.0 ** -103
    c.ks[:, :, 1::4, 2] = 0
    c.check(c.run(ops))
