"""CPU: derivatives of Rotation in forward mode, its launch replaced by the formula."""
import contextlib

import pytest
import torch
from torch.autograd import forward_ad

import torch_blocksparse as tb
from torch_blocksparse import rotation


def formula(op, tensors, positions, back):
    x = tensors[0]
    at = positions if positions is not None else torch.arange(x.size(2))
    angle = at.double()[..., None] * op.frequencies
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float() * (-1 if back else 1)
    n = op.pairs
    return tuple(torch.cat([t[..., :n] * cos - t[..., n:] * sin, t[..., :n] * sin + t[..., n:] * cos], -1).detach() for t in tensors)


@pytest.fixture
def op(monkeypatch):
    calls = []
    monkeypatch.setattr(rotation._lib, 'on_device', lambda device: contextlib.nullcontext())
    monkeypatch.setattr(tb.Rotation, '_check', lambda self, tensors, positions: None)
    monkeypatch.setattr(tb.Rotation, '_launch', lambda self, tensors, positions, back: (calls.append(len(tensors)), formula(self, tensors, positions, back))[1])
    op = tb.Rotation.of_base(16)
    op.calls = calls
    return op


def randn(seed):
    return torch.randn(2, 3, 5, 16, generator=torch.Generator().manual_seed(seed))


def test_tangents(op):
    x, y, dx, dy = [randn(i) for i in range(4)]
    positions = torch.tensor([3, 1, 4, 1, 5])
    with forward_ad.dual_level():
        one = forward_ad.unpack_dual(op(forward_ad.make_dual(x, dx), positions=positions))
        a, b = [forward_ad.unpack_dual(t) for t in op(forward_ad.make_dual(x, dx), forward_ad.make_dual(y, dy))]
        c, d = [forward_ad.unpack_dual(t) for t in op(x, forward_ad.make_dual(y, dy))]
        e = op(x)
        with torch.no_grad():
            f = forward_ad.unpack_dual(op(forward_ad.make_dual(x, dx)))
        assert forward_ad.unpack_dual(e).tangent is None
    assert torch.equal(one.primal, op(x, positions=positions)) and torch.equal(one.tangent, op(dx, positions=positions))
    assert torch.equal(a.tangent, op(dx)) and torch.equal(b.tangent, op(dy)) and torch.equal(d.tangent, op(dy)) and torch.equal(f.tangent, op(dx))
    assert c.tangent is None or not bool(c.tangent.any())
    assert torch.equal(c.primal, op(x)) and torch.equal(d.primal, op(y))


def test_forward_mode_through_a_backward_pass(op):
    """x -> sum(turned(x)^3): its second derivative along dx, in both orders"""
    x, dx = randn(1), randn(2)
    leaf = x.clone().requires_grad_(True)
    gradient, = torch.autograd.grad(op(leaf).pow(3).sum(), leaf, create_graph=True)
    want, = torch.autograd.grad((gradient * dx).sum(), leaf)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.clone().requires_grad_(True), dx)
        gradient, = torch.autograd.grad(op(dual).pow(3).sum(), dual)
        got = forward_ad.unpack_dual(gradient).tangent
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)
    with forward_ad.dual_level():                          # ... and a gradient of a tangent
        dual = forward_ad.make_dual(leaf, dx)
        tangent = forward_ad.unpack_dual(op(dual).pow(3).sum()).tangent
        got, = torch.autograd.grad(tangent, leaf)
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)


def test_without_a_derivative_nothing_is_recorded(op, monkeypatch):
    monkeypatch.setattr(rotation._turn, 'apply', None)
    op(randn(1), randn(2))
    with torch.no_grad():
        op(randn(1).requires_grad_(True))
    assert op.calls == [2, 1]
