"""Caches of 4 bits by their definition, in torch: where a head's codes lie, and what they stand for (used by the tests of 4-bit caches)."""
import torch

LEAST, GROUP = 2.0 ** -100, 32


def byte_of(dim):
    """The byte of a head's dim / 2 that holds channel c, and how far up in it the code + 8 is."""
    c = torch.arange(dim)
    return 2 * ((c % GROUP // 4) * (dim // GROUP) + c // GROUP) + c % 4 // 2, 4 * (c % 2)


def codes_of(raw, dim):
    """bytes [.., dim / 2] -> codes int64 [.., dim]"""
    at, up = (t.to(raw.device) for t in byte_of(dim))
    return ((raw[..., at].to(torch.int64) >> up) & 15) - 8


def packed(codes):
    """codes [.., dim] -> bytes [.., dim / 2]"""
    at, up = (t.to(codes.device) for t in byte_of(codes.shape[-1]))
    raw = torch.zeros(*codes.shape[:-1], codes.shape[-1] // 2, dtype=torch.int64, device=codes.device)
    raw.index_add_(-1, at, (codes.to(torch.int64) + 8) << up)
    return raw.to(torch.uint8)


def numbers(raw, scales, dim):
    """bytes [.., dim / 2] and scales [.., dim / 32] -> float64 [.., dim]"""
    return codes_of(raw, dim).double() * scales.double().repeat_interleave(GROUP, -1)


def quantised(x):
    """x float64 [.., dim] -> (quotients before rounding, scales float64 [.., dim / 32]); a group with a number that is not finite: NaN"""
    y = x.unflatten(-1, (-1, GROUP))
    a = y.abs().amax(-1)
    s = (a.clamp(min=LEAST) / 7).to(torch.float32).to(torch.bfloat16).double()
    s = torch.where(torch.isfinite(a), s, torch.full_like(s, float("nan")))
    return (y / s[..., None]).flatten(-2), s
