"""CPU: what Rotation and rotated writes refuse, and the fractions of a turn that they keep."""
import copy
import math
import pickle
from fractions import Fraction

import pytest
import torch

import rotation_oracle as R
import torch_blocksparse as tb
from torch_blocksparse import _lib, cache, rotation

ERR_ARG, UNSUPPORTED = -1, -2


def test_frequencies():
    for bad in ([], [1.] * 7, [1.] * 9, [math.inf] + [1.] * 7, [math.nan] + [1.] * 7, [2. ** 64] + [1.] * 7, torch.ones(2, 8)):
        with pytest.raises(ValueError):
            tb.Rotation(bad)
    for dim in (0, -16, 8, 40):
        with pytest.raises(ValueError):
            tb.Rotation.of_base(dim)
    op = tb.Rotation(torch.linspace(0, 1, 16, dtype=torch.float64), neighbours=1)
    assert op.pairs == 16 and op.neighbours is True and op.frequencies.tolist() == torch.linspace(0, 1, 16, dtype=torch.float64).tolist()
    assert tb.Rotation.of_base(64, 500.).frequencies.tolist() == [500. ** (-2. * p / 64) for p in range(32)]


@pytest.mark.parametrize('f', [0., 1., -1., 1e-30, 0.1, 1e18, 6.283185307179586, -3.7e12])
def test_fractions_of_a_turn(f):
    n = rotation._fraction_of_a_turn(f)
    assert -2 ** 63 <= n < 2 ** 63
    off = (Fraction(n, 2 ** 64) - Fraction(f) / R.TWO_PI) % 1
    assert min(off, 1 - off) <= Fraction(1, 2 ** 65) + Fraction(1, 2 ** 100)


def test_kept_without_its_tables():
    op = tb.Rotation.of_base(32)
    op._fractions[torch.device('cuda', 0)] = ('table', None)
    for other in (copy.deepcopy(op), pickle.loads(pickle.dumps(op))):
        assert other._fractions == {} and other.frequencies.tolist() == op.frequencies.tolist()


def test_tensors_elsewhere():
    with pytest.raises(_lib.BlocksparseLibraryError):
        tb.Rotation.of_base(64)(torch.zeros(1, 1, 1, 64))
    with pytest.raises(ValueError, match='one tensor or two'):
        tb.Rotation.of_base(64)()


class FakeGpu(torch.Tensor):
    is_cuda = True


def fake(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype).as_subclass(FakeGpu)


def test_shapes_types_and_positions():
    op = tb.Rotation.of_base(64)
    ids = lambda *s, dtype=torch.int32: torch.zeros(s, dtype=dtype)    # noqa: E731
    good = [((fake(2, 3, 5, 64), fake(2, 1, 5, 64)), ids(5)), ((fake(2, 3, 5, 64),), ids(2, 5)), ((fake(7, 3, 128),), ids(7)), ((fake(7, 3, 72),), None)]
    for tensors, positions in good:
        op._check(tensors, positions)
    bad = [((fake(64),), None), ((fake(3, 5, 64, dtype=torch.float64),), None), ((fake(3, 5, 64, dtype=torch.int32),), None), ((fake(3, 5, 60),), None), ((fake(3, 5, 32),), None),
           ((fake(2, 3, 5, 64), fake(2, 3, 6, 64)), None), ((fake(2, 3, 5, 64), fake(1, 3, 5, 64)), None), ((fake(2, 3, 5, 64), fake(2, 3, 5, 128)), None),
           ((fake(2, 3, 5, 64), fake(2, 3, 64)), None), ((fake(2, 3, 5, 64), fake(2, 3, 5, 64, dtype=torch.float32)), None), ((fake(2, 3, 5, 64),) * 3, None),
           ((fake(2, 3, 5, 64),), ids(2)), ((fake(2, 3, 5, 64),), ids(5, dtype=torch.int64)), ((fake(2, 3, 5, 64),), ids(1, 5)), ((fake(7, 3, 64),), ids(3)), ((fake(7, 3, 64),), ids(7, 1))]
    for tensors, positions in bad:
        with pytest.raises(ValueError):
            op._check(tensors, positions)
    with pytest.raises(ValueError, match='2\\^32'):
        op._check((fake(1, 1, 1, 64).expand(1 << 13, 1, 1 << 13, 64),), None)


def test_rotated_writes():
    op, cpu = tb.Rotation.of_base(64), torch.device('cpu')
    p = torch.zeros(5, dtype=torch.int32)
    assert cache.check_rotation(None, None, 5, 64, cpu) is None
    assert torch.equal(cache.check_rotation(op, p, 5, 64, cpu), p)
    for rotation_, positions, dim in ((None, p, 64), (op, None, 64), (op, p[:4], 64), (op, p.long(), 64), ('turn', p, 64), (tb.Rotation.of_base(128), p, 64)):
        with pytest.raises(ValueError):
            cache.check_rotation(rotation_, positions, 5, dim, cpu)


def test_c_entries_refuse():
    lib = _lib.load()
    held = torch.zeros(1 << 14, dtype=torch.uint8)
    at = held.data_ptr() + -held.data_ptr() % 16
    s = rotation._STRIDES.pack(*[64] * 6)
    call = lambda dtype=0, Z=1, L=1, D=64, pairs=32, f=at, x=at, y=at, H=1, s0=s, x1=None, y1=None, H1=0, s1=None: \
        lib.bsp_rotate(dtype, Z, L, D, pairs, 0, 0, f, None, 0, 0, x, y, H, s0, x1, y1, H1, s1, None)    # noqa: E731
    for bad in (dict(Z=0), dict(L=0), dict(D=60), dict(pairs=12), dict(pairs=40), dict(f=None), dict(f=at + 4), dict(x=at + 8), dict(y=None), dict(H=0), dict(s0=None),
                dict(s0=rotation._STRIDES.pack(4, *[64] * 5)), dict(H1=1), dict(H1=1, x1=at, y1=at), dict(H1=-1)):
        assert call(**bad) == ERR_ARG, bad
    assert call(dtype=3) == UNSUPPORTED and call(Z=1 << 16, L=1 << 16) == UNSUPPORTED
    write = lambda f=at, pairs=32, p=at: lib.bsp_cache_write_rotated(0, at, 4, 16, 1, 64, 4, at, 64, 64, at, 64, 64, at, 1, at, f, pairs, 0, p, None)    # noqa: E731
    for bad in (dict(f=None), dict(pairs=0), dict(pairs=36), dict(pairs=40), dict(p=None)):
        assert write(**bad) == ERR_ARG, bad
