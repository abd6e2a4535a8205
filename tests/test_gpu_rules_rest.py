"""GPU: what the rounding of Attention's result to a 16-bit type leaves out reaches its gradients."""
import pytest
import torch

import torch_blocksparse as tb

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('softcap', [0., 5.])
def test_delta_is_that_of_the_result_before_it_was_rounded(dtype, D, softcap):
    """Scores of zero, so shares that are all 1 / n; values that are one number or its upper neighbour, half of the keys each, so a result that
    lies in the middle of the two and is rounded to the lower one; keys of ones and a gradient of ones.  Then dp is delta +- x with x = D / 2 steps,
    and dq = sum_j (dp_j - delta) / n is zero.  A delta of the rounded result is off by x, and dq with it."""
    Z, H, L = 2, 2, 128
    u = torch.finfo(dtype).eps / 2
    low, high = 1., 1. + 2 * u                           # (1 has an even last digit, so the middle is rounded down)
    q, k, do = [torch.full((Z, H, L, D), x, dtype=dtype, device=DEV) for x in (0., 1., 1.)]
    v = torch.full((Z, H, L, D), low, dtype=dtype, device=DEV)
    v[:, :, 1::2] = high
    q.requires_grad_(True)
    o = tb.Attention(torch.ones(H, 2, 2), 64)(q, k, v, softcap=softcap)
    assert bool((o == low).all())
    dq, = torch.autograd.grad(o, q, do)
    x, size = D * u, D * (1 + u)
    # sums in fp32 of terms whose sizes add up to `size`; the remainder u is kept in the type, exactly; a score gradient is rounded by u of
    # itself, where the two kinds need not cancel; the result once more
    c = 2. ** -24 * (2 * D + L + 32)
    bound = (c * size + u * (x + c * size)) * (1 + u) + 2. ** -25
    assert x > 10 * bound                                # (what it would be with the rounded result)
    assert float(dq.abs().max()) <= bound
