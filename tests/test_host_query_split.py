"""How far two 8-bit values are from a bf16 query (the tensor-core kernels over
the E4M3 cache hold a query so), over every significand and binade.

A row is scaled by a power of two that puts its largest magnitude into (224,
448]. hi is the nearest E4M3 value and lo the nearest E5M2 value of what hi
leaves. From 2^-6 on hi has four significant bits, so it leaves a whole number
of at most 8 units in the last of bf16's eight: that has three bits (or is 8)
and E5M2 holds it. Below, hi leaves at most 2^-10, which E5M2 holds to half
its step of 2^-13.
"""
import torch

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def split(x):
    hi = x.clamp(-448, 448).to(E4M3).float()
    lo = (x - hi).to(E5M2).float()
    return hi, lo


def _values():
    m = torch.arange(128, 256).float() / 128
    e = torch.arange(-24, 9).float()
    x = (m[None] * torch.exp2(e)[:, None]).flatten()
    x = x[x <= 448]
    assert torch.equal(x, x.bfloat16().float())
    return torch.cat([x, -x])


def test_pieces_hold_every_bf16_value_above_2_to_the_minus_6():
    x = _values()
    hi, lo = split(x)
    big = x.abs() >= 2.0 ** -6
    assert torch.equal((hi + lo)[big], x[big])


def test_pieces_below_are_off_by_at_most_2_to_the_minus_14():
    x = _values()
    hi, lo = split(x)
    err = ((hi.double() + lo.double()) - x.double()).abs()
    assert float(err.max()) == 2.0 ** -14
    # and what hi does not see keeps three bits
    tiny = (x.abs() < 2.0 ** -10) & (x.abs() >= 2.0 ** -14)
    assert bool((err[tiny] <= x[tiny].abs().double() / 8).all())


def test_two_e4m3_pieces_would_lose_more():
    """The reason for the two formats: with E4M3 for both, steps stay at 2^-9."""
    x = _values()
    hi = x.to(E4M3).float()
    err = ((hi + (x - hi).to(E4M3).float()) - x).abs()
    assert float(err.max()) == 2.0 ** -10
