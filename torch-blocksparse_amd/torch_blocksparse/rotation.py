"""Rotated positions: pairs of elements turned by an angle that grows with the position.

`Rotation(frequencies)(q, k, positions=positions)` turns pair p of the row at position t by the angle t * frequencies[p], in queries and keys with one
launch, so that the product of two of them depends on how far apart they are:

    (a, b) -> (a cos - b sin, a sin + b cos)

A pair is elements p and pairs + p of a head, or, with neighbours=True, elements 2 p and 2 p + 1; elements from 2 * pairs on stay as they are.  No table of positions: a
frequency is kept as a fraction of a turn with 64 bits, with which any position of 32 bits gives an angle that is off by at most 2^-34 of a turn.  The gradient is
the turn back.  Sines, cosines and products are fp32, rounded once to the operands' type.

The caches take a rotation where keys are written to them (`KeyValueCache.write`, `LatentCache.write`)."""
import math
import struct
from fractions import Fraction

import torch

from . import _lib

_TWO_PI = Fraction(628318530717958647692528676655900576839433879875021164194988918461563281257, 10 ** 74)
_STRIDES = struct.Struct('@6q')      # of batch, head and position: x, y


def _fraction_of_a_turn(f):
    """f radians, less its whole turns, in units of 2^-64 of a turn (as a signed number of 64 bits)"""
    n = round(Fraction(f) / _TWO_PI * (1 << 64)) % (1 << 64)
    return n - (1 << 64) if n >> 63 else n


def _operand(t):
    """(t, or a copy that the kernel can address; its strides of batch, head and position); t [batch, heads, length, dim] or [tokens, heads, dim]"""
    for again in (False, True):
        at = (0,) + (t.stride(1), t.stride(0)) if t.dim() == 3 else t.stride()[:3]
        sizes = (1, t.size(1), t.size(0)) if t.dim() == 3 else t.shape[:3]
        at = tuple(s if n > 1 else 0 for s, n in zip(at, sizes))
        if again or (t.stride(-1) == 1 and not (at[0] | at[1] | at[2]) * t.element_size() % 16 and not t.data_ptr() % 16):
            return t, at
        t = t.clone(memory_format=torch.contiguous_format)


class _turn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, rotation, positions, back, *tensors):
        ctx.save_for_backward(positions)
        ctx.rotation, ctx.back = rotation, back
        ctx.set_materialize_grads(False)
        out = rotation._launch(tensors, positions, back)
        return out if len(out) > 1 else out[0]

    @staticmethod
    def backward(ctx, *grads):
        positions, = ctx.saved_tensors
        given = [g for g in grads if g is not None]
        if not given:
            return (None,) * (3 + len(grads))
        with _lib.on_device(given[0].device):
            turned = _turn.apply(ctx.rotation, positions, not ctx.back, *given)
        turned = iter(turned if len(given) > 1 else (turned,))
        return (None, None, None) + tuple(next(turned) if g is not None else None for g in grads)


class Rotation:
    """Turns pairs of elements by position times frequency.

    frequencies  radians a position, one for each pair: a multiple of 8 numbers (a list, or a vector; constants)
    neighbours   pairs of neighbouring elements, not of the two halves of what is turned

    Called with one or two tensors (queries and keys: of one type, float16, bfloat16 or float32, and alike but for their number of heads) of shape [batch,
    heads, length, dim] with positions [length] or [batch, length], or [tokens, heads, dim] with positions [tokens]: int32, on the tensors'
    device; without positions they are 0 .. length - 1.  dim is a multiple of 8, 2 * pairs at least.  Returns the turned tensors (one: not in a tuple), contiguous; differentiable
    in them, any number of times.

    A copy of the frequencies is made at the first call on a device, so a call that is captured into a graph needs one on its device before."""

    def __init__(self, frequencies, neighbours=False):
        f = [float(x) for x in (frequencies.detach().double().flatten().tolist() if isinstance(frequencies, torch.Tensor) else frequencies)]
        if isinstance(frequencies, torch.Tensor) and frequencies.dim() != 1:
            raise ValueError('frequencies must be a vector (got %s)' % list(frequencies.shape))
        if not f or len(f) % 8:
            raise ValueError('the number of pairs must be a multiple of 8 (got %d)' % len(f))
        if not all(math.isfinite(x) and abs(x) < 2. ** 64 for x in f):
            raise ValueError('frequencies must be finite numbers below 2^64')
        self.frequencies, self.pairs, self.neighbours = torch.tensor(f, dtype=torch.float64, device='cpu'), len(f), bool(neighbours)
        self._fractions = dict()

    @classmethod
    def of_base(cls, dim, base=10000., neighbours=False):
        """the frequencies base ** (-2 p / dim) for the dim / 2 pairs of dim elements"""
        if dim <= 0 or dim % 16:
            raise ValueError('dim must be a multiple of 16 (got %s)' % (dim,))
        return cls([float(base) ** (-2. * p / dim) for p in range(dim // 2)], neighbours)

    def __getstate__(self):
        return dict(self.__dict__, _fractions=dict())

    def fractions(self, device):
        """the frequencies as the kernels read them, noted as read by the current stream"""
        made = self._fractions.get(device)
        if made is None:
            table = torch.tensor([_fraction_of_a_turn(f) for f in self.frequencies.tolist()], dtype=torch.int64, device='cpu').to(device)
            made = self._fractions[device] = (table, _lib.Readers())
            made[1].table(table)
        made[1].read(device)
        return made[0]

    def check_positions(self, positions, shapes, device):
        if positions is not None and (positions.dtype != torch.int32 or positions.device != device or tuple(positions.shape) not in shapes):
            raise ValueError('positions must be int32 %s on %s (got %s %s on %s)' % (' or '.join(str(list(s)) for s in shapes), device, positions.dtype, list(positions.shape), positions.device))

    def _check(self, tensors, positions):
        if len(tensors) not in (1, 2):
            raise ValueError('a call takes one tensor or two (got %d)' % len(tensors))
        x = tensors[0]
        for t in tensors:
            _lib.require_gpu_tensor(t, 'a rotated tensor')
            if t.dim() not in (3, 4):
                raise ValueError('rotated tensors have shape [batch, heads, length, dim] or [tokens, heads, dim] (got %s)' % list(t.shape))
            if t.dtype not in _lib.DTYPES:
                raise ValueError('Rotation supports float16, bfloat16 and float32 (got %s)' % t.dtype)
            if t.dtype != x.dtype or t.device != x.device or t.dim() != x.dim() or t.shape[:1] + t.shape[2:] != x.shape[:1] + x.shape[2:]:
                raise ValueError('the tensors of a call must be alike but for their number of heads (got %s %s and %s %s)' % (x.dtype, list(x.shape), t.dtype, list(t.shape)))
        D = x.size(-1)
        if D % 8 or D < 2 * self.pairs:
            raise ValueError('heads must have a multiple of 8 elements, at least %d for %d pairs (got %d)' % (2 * self.pairs, self.pairs, D))
        if x.dim() == 3:
            self.check_positions(positions, ((x.size(0),),), x.device)
        else:
            self.check_positions(positions, ((x.size(2),), (x.size(0), x.size(2))), x.device)
        tokens = x.size(0) if x.dim() == 3 else x.size(0) * x.size(2)
        if tokens * D >= 1 << 32:
            raise ValueError('a call takes fewer than 2^32 elements of a head (got %d positions of %d)' % (tokens, D))

    def _launch(self, tensors, positions, back):
        x, device = tensors[0], tensors[0].device
        Z, L, D = (1, x.size(0), x.size(2)) if x.dim() == 3 else (x.size(0), x.size(2), x.size(3))
        out, args = [], []
        for t in tensors:
            y = torch.empty(t.shape, dtype=t.dtype, device=device)
            t, at = _operand(t)
            out.append(y)
            args.append((t, y, t.size(1), _STRIDES.pack(*at, *_operand(y)[1])))
        live = [a for a in args if a[0].numel()]
        if live:
            (x0, y0, H0, s0), (x1, y1, H1, s1) = live[0], live[1] if len(live) > 1 else (None, None, 0, None)
            p_z, p_l = (0, 0) if positions is None else (positions.stride(0) if positions.dim() == 2 else 0, positions.stride(-1))
            rc = _lib.load().bsp_rotate(_lib.DTYPES[x.dtype], Z, L, D, self.pairs, self.neighbours, back, self.fractions(device).data_ptr(), positions.data_ptr() if positions is not None else None,
                                        p_z, p_l, x0.data_ptr(), y0.data_ptr(), H0, s0, x1.data_ptr() if H1 else None, y1.data_ptr() if H1 else None, H1, s1, _lib.raw_stream(device))
            if rc:
                _lib.check(rc, 'bsp_rotate')
        return tuple(out)

    def __call__(self, *tensors, positions=None):
        self._check(tensors, positions)
        with _lib.on_device(tensors[0].device):
            if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
                return _turn.apply(self, positions, False, *tensors)
            out = self._launch(tensors, positions, False)
        return out if len(out) > 1 else out[0]
