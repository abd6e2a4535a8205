"""Rotated positions in 64 bits, with the bound that GPU results are held to.

With u half a step of the type: a sine or cosine is off by 5 * 2^-24 at most (three roundings of an angle of at most pi / 4, one of the result, 2^-29 of the series and 2^-33 of a turn of the angle beside
them), so a turned element by 5 * 2^-24 (|a| + |b|), and by 2 * 2^-24 (|a| + |b|) for the product's and the sum's rounding; it is rounded to the type once more."""
import math
from fractions import Fraction

import torch

TWO_PI = Fraction(628318530717958647692528676655900576839433879875021164194988918461563281257, 10 ** 74)


def angles(positions, frequencies):
    """[.., pairs] in 64 bits, less whole turns: exact before the last rounding"""
    flat = [[float((Fraction(f) * p / TWO_PI) % 1) * (2 * math.pi) for f in frequencies] for p in positions.flatten().tolist()]
    return torch.tensor(flat, dtype=torch.float64).reshape(tuple(positions.shape) + (len(frequencies),))


def turned(x, angle, neighbours, back=False):
    """(value, bound) of x [.., D] turned by angle, which broadcasts against [.., pairs]"""
    u = torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float64 else 0.
    tiny = 2. ** -25 if x.dtype == torch.float16 else 2. ** -126
    x = x.detach().double().cpu()
    n = angle.size(-1)
    one, two = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if neighbours else (slice(0, n), slice(n, 2 * n))
    cos, sin = torch.cos(angle), torch.sin(angle) * (-1 if back else 1)
    value, size = x.clone(), torch.zeros_like(x)
    value[..., one], value[..., two] = x[..., one] * cos - x[..., two] * sin, x[..., one] * sin + x[..., two] * cos
    size[..., one] = size[..., two] = x[..., one].abs() + x[..., two].abs()
    return value, torch.where(size > 0, u * value.abs() + 8 * 2. ** -24 * size + tiny, 0.)


def check(got, want, what):
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    bad = ~((got - value).abs() <= bound)
    assert not bool(bad.any()), '%s: %d of %d outside their bound, first at %s: got %g, is %g' % (
        what, int(bad.sum()), bad.numel(), torch.nonzero(bad)[0].tolist(), got[bad][0], value[bad][0])
