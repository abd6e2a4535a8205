"""Attention with score rules in 64 bits on the CPU, with the bounds that its GPU results are held to.

What rounding may do to a result, with u half a step of the type (eps / 2), n the keys of the longest row, D the head dimension:
  * the operands are exact, their products are summed in fp32: a logit is off by c = 2^-24 (2 D + n + 8 max|y| + 32) relative to the sum of its
    terms' sizes at most (the tanh's 2^-23 cap among them), and so is a share p of the softmax, relative to itself;
  * shares and softmax gradients are rounded to the type where they become an operand: u of themselves, in fp16 not less than 2^-25;
  * a share is an exponential in fp32, which holds nothing between 0 and 2^-126 (numbers that are not normal count as 0 in these units), and
    bfloat16 has the same exponents: so a share is off by up to 2^-126, and a softmax gradient by that and by that times |dp - delta|;
  * delta = do . o takes o as stored: off by u sum_d |do_d o_d|;
  * the result is rounded once more."""
import math

import torch


def dense_layout(layout, block, L):
    return (layout != 0).repeat_interleave(block, 1).repeat_interleave(block, 2)[:, :L, :L]


def attention(q, k, v, layout, block, do=None, scale=1., softcap=0., slopes=None, causal=False, documents=None, prefix=None):
    """{name: (value, bound)} for o and, with do, dq, dk, dv"""
    dtype = q.dtype
    u = torch.finfo(dtype).eps / 2
    q, k, v = [t.detach().double().cpu() for t in (q, k, v)]
    Z, H, L, D = q.shape
    G = H // k.size(1)
    pos = torch.arange(L)
    seen = dense_layout(layout.cpu(), block, L)[None].expand(Z, H, L, L).clone()
    if causal:
        rule = (pos[None, :] <= pos[:, None]).expand(Z, 1, L, L)
        if prefix is not None:
            rule = rule | (pos < prefix.cpu()[:, None, None, None])
        seen &= rule
    if documents is not None:
        ids = documents.cpu()
        seen &= ((ids[:, :, None] == ids[:, None, :]) & (ids[:, :, None] >= 0) & (ids[:, None, :] >= 0))[:, None]
        pad = (ids < 0)[:, None, :, None]
        q, k, v = [t.masked_fill(pad, 0.) for t in (q, k, v)]                   # (they may hold anything)
    kx, vx = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = scale * (q @ kx.transpose(-1, -2))
    terms = abs(scale) * (q.abs() @ kx.abs().transpose(-1, -2))
    t = torch.tanh(s / softcap) if softcap else torch.zeros_like(s)
    y = softcap * t if softcap else s
    if slopes is not None:
        far = slopes.detach().double().cpu()[:, None, None] * (pos[:, None] - pos[None, :]).abs()
        y, terms = y - far, terms + far.abs()
    y = y.masked_fill(~seen, -math.inf)
    most = y.amax(-1, keepdim=True)
    p = torch.exp(y - torch.where(most == -math.inf, 0., most))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1., total)
    n = int(seen.sum(-1).max())
    big = float(torch.where(seen, terms, 0.).max()) if n else 0.
    c = 2. ** -24 * (2 * D + n + 8 * (big + softcap) + 32)
    tiny = 2. ** -25 if dtype == torch.float16 else 2. ** -126
    o = p @ vx
    out = {'o': (o, u * o.abs() + (u + c) * (p @ vx.abs()) + tiny * (1 + seen.double() @ vx.abs()))}
    if do is None:
        return out
    do = do.detach().double().cpu()
    if documents is not None:
        do = do.masked_fill(pad, 0.)
    dp = do @ vx.transpose(-1, -2)
    delta = (do * o).sum(-1, keepdim=True)
    size = (do.abs() * o.abs()).sum(-1, keepdim=True)
    through = 1 - t * t
    e = p * (dp - delta) * through
    # (1 - t^2 is off by 2 |t| 2^-23, so by 2^-22 of one, not of itself)
    off = u * e.abs() + through * p * ((u + c) * size + c * (do.abs() @ vx.abs().transpose(-1, -2)) + c * (dp - delta).abs()) + 2. ** -21 * p * (dp - delta).abs() * bool(softcap)
    off = off + (tiny + 2. ** -126 * (dp - delta).abs()) * seen
    per = lambda m: m.unflatten(1, (-1, G)).sum(2)    # noqa: E731  sums over the query heads that share a key head
    sc = abs(scale)
    dq, dk, dv = scale * (e @ kx), per(scale * (e.transpose(-1, -2) @ q)), per(p.transpose(-1, -2) @ do)
    sums = c * sc * (e.abs() @ kx.abs()), c * sc * per(e.abs().transpose(-1, -2) @ q.abs())
    out['dq'] = dq, u * dq.abs() + sc * (off @ kx.abs()) + sums[0] + tiny
    out['dk'] = dk, u * dk.abs() + sc * per(off.transpose(-1, -2) @ q.abs()) + sums[1] + tiny
    out['dv'] = dv, u * dv.abs() + per((u + c) * (p.transpose(-1, -2) @ do.abs()) + tiny * (seen.double().transpose(-1, -2) @ do.abs())) + tiny
    return out


def check(got, want, what):
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    assert bool(torch.isfinite(got).all()), '%s: not finite at %s' % (what, torch.nonzero(~torch.isfinite(got))[0].tolist())
    err = (got - value).abs()
    bad = err > bound
    if bool(bad.any()):
        i = tuple(torch.nonzero(bad)[0].tolist())
        raise AssertionError('%s: %d of %d outside their bound; first at %s: got %g, is %g, bound %g; worst %g of the bound'
                             % (what, int(bad.sum()), bad.numel(), i, got[i], value[i], bound[i], float((err / bound.clamp(min=1e-300)).max())))
    return float((err / bound.clamp(min=1e-300)).max())
