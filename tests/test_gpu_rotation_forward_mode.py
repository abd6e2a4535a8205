"""GPU: derivatives of Rotation in forward mode: the turn is linear, so a tangent is turned as what it belongs to."""
import pytest
import torch
from torch.autograd import forward_ad

import torch_blocksparse as tb

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('neighbours', [False, True])
def test_tangents(dtype, neighbours):
    op = tb.Rotation.of_base(64, neighbours=neighbours)
    q, k, dq, dk = [randn((2, h, 33, 128), dtype, i) for i, h in enumerate((4, 2, 4, 2))]
    odd = dk.transpose(2, 3).contiguous().transpose(2, 3)
    with forward_ad.dual_level():
        y, z = [forward_ad.unpack_dual(t) for t in op(forward_ad.make_dual(q, dq), forward_ad.make_dual(k, odd))]
        same, alone = [forward_ad.unpack_dual(t) for t in op(q, forward_ad.make_dual(k, dk))]
    assert torch.equal(y.primal, op(q)) and torch.equal(z.primal, op(k))
    assert torch.equal(y.tangent, op(dq)) and torch.equal(z.tangent, op(dk)) and torch.equal(alone.tangent, op(dk))
    assert torch.equal(same.primal, op(q)) and (same.tangent is None or not bool(same.tangent.any()))
    leaf = q.clone().requires_grad_(True)
    with forward_ad.dual_level():                          # a gradient of what a tangent came to
        tangent = forward_ad.unpack_dual(op(forward_ad.make_dual(leaf, dq)).pow(2).sum()).tangent
        got, = torch.autograd.grad(tangent, leaf)
    assert got.shape == q.shape and bool(torch.isfinite(got).all())
    if dtype == torch.float32:                             # |turned x|^2 = |x|^2, whose derivative along dq is 2 x . dq and that one's gradient 2 dq
        assert torch.allclose(got, 2 * dq, rtol=1e-5, atol=1e-5)
