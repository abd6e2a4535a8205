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
from torch.autograd import forward_ad

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
        stride, shape = t.stride(), t.shape
        z, h, l = (0, stride[1], stride[0]) if len(stride) == 3 else stride[:3]      # noqa: E741
        if shape[0] == 1:
            z, l = 0, l if len(stride) == 4 else 0                                   # noqa: E741
        if shape[1] == 1:
            h = 0
        if len(stride) == 4 and shape[2] == 1:
            l = 0                                                                    # noqa: E741
        if again or (stride[-1] == 1 and not (z | h | l) * t.element_size() % 16 and not t.data_ptr() % 16):
            return t, (z, h, l)
        t = t.clone(memory_format=torch.contiguous_format)


class _turn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, rotation, positions, back, *tensors):
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        ctx.rotation, ctx.back, ctx.shapes = rotation, back, [t.shape for t in tensors]
        ctx.set_materialize_grads(False)
        out = rotation._launch(tensors, positions, back)
        return out if len(out) > 1 else out[0]

    @staticmethod
    def backward(ctx, *grads):
        positions, = ctx.saved_tensors
        given = [g for g in grads if g is not None]
        if not given:
            return (None,) * (3 + len(grads))
        turned = iter(ctx.rotation._turned(given, positions, not ctx.back))
        return (None, None, None) + tuple(next(turned) if g is not None else None for g in grads)

    @staticmethod
    def jvp(ctx, _, __, ___, *tangents):                  # the turn is linear: the same of the tangents
        positions, = ctx.saved_tensors
        given = [t for t in tangents if t is not None]
        turned = iter(ctx.rotation._turned(given, positions, ctx.back))
        turned = tuple(next(turned) if t is not None else given[0].new_zeros(shape) for t, shape in zip(tangents, ctx.shapes))     # (an output has to have one)
        return turned if len(turned) > 1 else turned[0]


class Rotation:
    """Turns pairs of elements by position times frequency.

    frequencies  radians a position, one for each pair: a multiple of 8 numbers (a list, or a vector; constants)
    neighbours   pairs of neighbouring elements, not of the two halves of what is turned

    Called with one or two tensors (queries and keys: of one type, float16, bfloat16 or float32, and alike but for their number of heads) of shape [batch,
    heads, length, dim] with positions [length] or [batch, length], or [tokens, heads, dim] with positions [tokens]: int32, on the tensors'
    device; without positions they are 0 .. length - 1.  dim is a multiple of 8, 2 * pairs at least.  Returns the turned tensors (one: not in a tuple), contiguous; differentiable
    in them, any number of times, backward and in forward mode.

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
        self._turns = self._as_turns()

    def _as_turns(self):
        return torch.tensor([_fraction_of_a_turn(f) for f in self.frequencies.tolist()], dtype=torch.int64, device='cpu')

    @classmethod
    def of_base(cls, dim, base=10000., neighbours=False):
        """the frequencies base ** (-2 p / dim) for the dim / 2 pairs of dim elements"""
        if dim <= 0 or dim % 16:
            raise ValueError('dim must be a multiple of 16 (got %s)' % (dim,))
        return cls([float(base) ** (-2. * p / dim) for p in range(dim // 2)], neighbours)

    def __getstate__(self):
        state = dict(self.__dict__, _fractions=dict())
        state.pop('_turns', None)
        return state

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._turns = self._as_turns()

    def fractions(self, device):
        """the frequencies as the kernels read them, noted as read by the current stream"""
        made = self._fractions.get(device)
        if made is None:
            made = (self._turns.to(device), _lib.Readers())
            made[1].table(made[0])
            made = self._fractions.setdefault(device, made)      # (another thread's, which a call may be on its way to read, stays)
        if _lib.raw_stream(device) not in made[1].streams:
            made[1].read(device)
        return made[0]

    def check_positions(self, positions, shapes, device):
        if positions is not None and (positions.dtype != torch.int32 or positions.shape not in shapes or positions.device != device):
            raise ValueError('positions must be int32 %s on %s (got %s %s on %s)' % (' or '.join(str(list(s)) for s in shapes), device, positions.dtype, list(positions.shape), positions.device))

    def _check(self, tensors, positions):
        if len(tensors) not in (1, 2):
            raise ValueError('a call takes one tensor or two (got %d)' % len(tensors))
        x = tensors[0]
        shape, device = x.shape, x.device
        for t in tensors:
            if not t.is_cuda:
                _lib.require_gpu_tensor(t, 'a rotated tensor')
        if len(shape) not in (3, 4):
            raise ValueError('rotated tensors have shape [batch, heads, length, dim] or [tokens, heads, dim] (got %s)' % list(shape))
        if x.dtype not in _lib.DTYPES:
            raise ValueError('Rotation supports float16, bfloat16 and float32 (got %s)' % x.dtype)
        if len(tensors) == 2:
            y = tensors[1]
            if y.dtype != x.dtype or y.device != device or y.dim() != len(shape) or y.shape[0] != shape[0] or y.shape[2:] != shape[2:]:
                raise ValueError('the tensors of a call must be alike but for their number of heads (got %s %s and %s %s)' % (x.dtype, list(shape), y.dtype, list(y.shape)))
        D, L = shape[-1], shape[0] if len(shape) == 3 else shape[2]
        if D % 8 or D < 2 * self.pairs:
            raise ValueError('heads must have a multiple of 8 elements, at least %d for %d pairs (got %d)' % (2 * self.pairs, self.pairs, D))
        if positions is not None:
            self.check_positions(positions, ((L,),) if len(shape) == 3 else ((L,), (shape[0], L)), device)
        if (L if len(shape) == 3 else shape[0] * L) * D >= 1 << 32:
            raise ValueError('a call takes fewer than 2^32 elements of a head (got %s)' % list(shape))

    def _launch(self, tensors, positions, back):
        x = tensors[0]
        shape, device = x.shape, x.device
        Z, L, D = (1, shape[0], shape[2]) if len(shape) == 3 else (shape[0], shape[2], shape[3])
        out, args, live = [], [], 0
        for t in tensors:
            y = torch.empty_like(t, memory_format=torch.contiguous_format)
            out.append(y)
            if t.numel():
                H = t.shape[1]
                t, at = _operand(t)
                own = (0, D, H * D) if len(shape) == 3 else (H * L * D, L * D, D)
                args += [t, y, H, _STRIDES.pack(*at, *own)]
                live += 1
        if live:
            x0, y0, H0, s0 = args[:4]
            x1, y1, H1, s1 = args[4:] if live == 2 else (None, None, 0, None)
            p_z, p_l, p = 0, 0, None
            if positions is not None:
                p, p_l = positions.data_ptr(), positions.stride(-1)
                if positions.dim() == 2:
                    p_z = positions.stride(0)
            rc = _lib.load().bsp_rotate(_lib.DTYPES[x.dtype], Z, L, D, self.pairs, self.neighbours, back, self.fractions(device).data_ptr(), p, p_z, p_l, x0.data_ptr(), y0.data_ptr(), H0, s0,
                                        x1.data_ptr() if H1 else None, y1.data_ptr() if H1 else None, H1, s1, _lib.raw_stream(device))
            if rc:
                _lib.check(rc, 'bsp_rotate')
        return tuple(out)

    def _turned(self, tensors, positions, back):
        """the turned tensors; through autograd where a derivative may be wanted: a tensor that requires a gradient, or a forward-mode level that is open (whose tensors do not require one)"""
        with _lib.on_device(tensors[0].device):
            if (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)) or forward_ad._current_level >= 0:
                out = _turn.apply(self, positions, back, *tensors)
                return out if len(tensors) > 1 else (out,)
            return self._launch(tensors, positions, back)

    def __call__(self, *tensors, positions=None):
        self._check(tensors, positions)
        out = self._turned(tensors, positions, False)
        return out if len(out) > 1 else out[0]
