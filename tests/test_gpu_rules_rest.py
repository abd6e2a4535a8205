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


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('heads', [16, 640])
def test_the_gradient_of_a_query_is_made_of_score_gradients_as_they_are(dtype, D, heads):
    """Shares of 1 / 64; score gradients +-A / 64 and +-B / 64, A a little above the middle of two neighbours, B a little below it, such that
    dq = (A - B) / 2 is a quarter of what it would be with A and B rounded.  (Many heads: one pair of wavefronts a line; few: two.)"""
    L, H, u = 256, heads, torch.finfo(dtype).eps / 2
    a, b = [1., u, u / 4], [1., u, -u / 4]
    v, k, do, q = [torch.zeros(1, H, L, D) for _ in range(4)]
    for kind, (x, sign, key) in enumerate(((a, 1, 1), (a, -1, -1), (b, 1, -1), (b, -1, 1))):
        v[:, :, kind::4, :3] = sign * torch.tensor(x)
        k[:, :, kind::4] = key
    do[..., :3] = 1.
    # blocks of the diagonal: a row sees 64 keys
    q, k, v, do = [t.to(dtype).to(DEV) for t in (q, k, v, do)]
    q.requires_grad_(True)
    o = tb.Attention(torch.eye(L // 64).expand(H, -1, -1), 64)(q, k, v)
    assert not bool(o.any())
    dq, = torch.autograd.grad(o, q, do)
    exact, size = u / 4, 1 + 2 * u
    c = 2. ** -24 * (2 * D + 64 + 32)
    bound = (c + u * u) * size + u * exact               # sums in fp32; score gradients in two terms; the result
    assert 3 * exact > 10 * bound                        # (A and B rounded: four times as much)
    assert float((dq.double() - exact).abs().max()) <= bound


@pytest.mark.parametrize('dtype,score,tells', [(torch.float16, -497 / 1024, 1.7), (torch.bfloat16, -77 / 256, 8.)])
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('heads', [1, 640])
@pytest.mark.parametrize('softcap', [0., 5.])
def test_the_gradient_of_a_key_sees_no_rounded_shares(dtype, score, tells, D, heads, softcap):
    """Half of the keys have scores of zero and values that give dp = 1, the others dp one step above it and scores whose exponential is off by
    much of half a step when it is rounded.  dp - delta is below a step, so a delta of the rounded shares is off by a large part of it."""
    L, u = 256, torch.finfo(dtype).eps / 2
    q, k, v, do = [torch.zeros(1, heads, L, D) for _ in range(4)]
    q[..., 0], do[..., 1], v[..., 1] = 1., 1., 1.
    k[:, :, 1::2, 0], v[:, :, 1::2, 1] = score, 1. + 2 * u
    q, k, v, do = [t.to(dtype).to(DEV) for t in (q, k, v, do)]
    k.requires_grad_(True)
    o = tb.Attention(torch.eye(L // 64).expand(heads, -1, -1), 64)(q, k, v, softcap=softcap)
    dk, = torch.autograd.grad(o, k, do)
    s = torch.tensor(score, dtype=torch.float64)
    t = torch.tanh(s / softcap) if softcap else torch.zeros(())
    e = torch.exp(softcap * t if softcap else s)
    p0, p1 = 1 / (32 * (1 + e)), e / (32 * (1 + e))      # of a key of each kind
    delta = 1. + 32 * p1 * 2 * u
    want = 64 * torch.stack([p0 * (1. - delta), p1 * (1. + 2 * u - delta) * (1 - t * t)])
    c = 2. ** -24 * (2 * D + 64 + 8 * (0.31 + softcap) + 32)
    # per row: p and dp off by c, 1 - t^2 by 2^-21 of one; the score gradient rounded; a sum over 64 rows and the result
    bound = 64 * torch.stack([p0, p1]) * (3 * c + 2. ** -21 * 2 * u) + (2 * u + c) * want.abs()
    off = 64 * torch.stack([p0, p1]) * 32 * p1 * (e.to(dtype).double() / e - 1).abs()
    assert bool((off > tells * bound).all())             # (delta of the rounded shares)
    got = dk[..., 0].double().cpu().view(1, heads, L // 2, 2)
    assert bool(((got - want).abs() <= bound).all())
