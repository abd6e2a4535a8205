"""Attention over latent vectors in 64 bits, with the bound that GPU results are held to.

With u half a step of the type, K = latent + 64 and n the positions of a sequence: the operands are exact and a score is summed in fp32, so it is off by (K + 8) 2^-24 of the sum of its terms' sizes, by
softcap * 2^-22 with a cap and by 4 * 2^-24 of the distance's part; a share (an exponential over a sum of n of them) by twice the largest of that and (n + 16) 2^-24 relative to itself. A share goes into
the product in two terms: u^2 of it, in fp16 not less than 2^-25 for shares that are relative to a maximum of 1 or less.  With more than 32 heads a workgroup (of at most 64, as evenly as can be) it goes
in one, rounded by u of itself, and the sum is that of the rounded ones: p_j (1 + d_j) / sum_k p_k (1 + d_k) with all |d| <= u is off by u sum_j p_j |c_j| in the one and by u |o| in the other. The product is summed in fp32 (n 2^-24 of the terms), the result rounded once."""
import math

import torch


def attention(q, q_r, c, r, table, lengths, block, layout=None, scale=1., softcap=0., slopes=None):
    """(value, bound) [B, H, latent] on the GPU; c, r: the cache's rows [positions, ..]"""
    dtype, (B, H, D) = q.dtype, q.shape
    u, tiny = torch.finfo(dtype).eps / 2, 2. ** -25 if dtype == torch.float16 else 2. ** -126
    pages = c.size(0) // block
    value, bound = torch.zeros(B, H, D, dtype=torch.float64, device=q.device), torch.zeros(B, H, D, dtype=torch.float64, device=q.device)
    if layout is not None:
        layout = (layout != 0).to(q.device)
    most = table.size(1) * block if layout is None else min(table.size(1), layout.size(1)) * block
    for b in range(B):
        n = min(int(lengths[b]), most)
        if n <= 0:
            continue
        page = table[b].long().repeat_interleave(block)[:n]
        at = page * block + torch.arange(n, device=q.device) % block
        held = (page >= 0) & (page < pages)
        at = torch.where(held, at, 0)
        cb, rb = [torch.where(held[:, None], t[at], 0.).double() for t in (c, r)]
        qb, qrb = q[b].double(), q_r[b].double()
        s, terms = scale * (qb @ cb.T + qrb @ rb.T), abs(scale) * (qb.abs() @ cb.abs().T + qrb.abs() @ rb.abs().T)
        off = (D + 72) * 2. ** -24 * terms
        if softcap:
            s, off = softcap * torch.tanh(s / softcap), off + softcap * 2. ** -22
        if slopes is not None:
            far = slopes.double()[:, None] * torch.arange(n - 1, -1, -1, device=q.device)
            s, off = s - far, off + 4 * 2. ** -24 * (far + s.abs())
        seen = held[None].expand(H, n)
        if layout is not None:
            seen = seen & layout[:, (n - 1) // block].repeat_interleave(block, 1)[:, :n]
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0., top))
        total = p.sum(1, keepdim=True)
        p = p / torch.where(total == 0, 1., total)
        off = 2 * torch.where(seen, off, 0.).amax(1, keepdim=True) + (2 * n + 24) * 2. ** -24 + u * u
        value[b] = p @ cb
        one_term = u if -(-H // -(-H // 64)) > 32 else 0.
        bound[b] = one_term * (p @ cb.abs() + value[b].abs()) * (1 + 2 * u) + u * value[b].abs() + off * (1 + u) * (p @ cb.abs()) + tiny * (1 + seen.double() @ cb.abs())
    return value, bound


def check(got, want, what):
    value, bound = want
    assert bool(torch.isfinite(got).all()), what
    err = (got.double() - value).abs()
    bad = err > bound
    assert not bool(bad.any()), '%s: %d of %d outside their bound, first at %s: got %g, is %g, bound %g' % (
        what, int(bad.sum()), bad.numel(), torch.nonzero(bad)[0].tolist(), got[bad][0], value[bad][0], bound[bad][0])
