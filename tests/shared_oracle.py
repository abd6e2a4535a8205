"""Attention with a key part that all heads share, in 64 bits on the CPU, over a causal layout without holes, with the bounds that results are held to where every operand that a kernel rounds itself goes
into its product in two terms.

With u half a step of the type (eps / 2), n the longest row's keys and D the elements of a head:
  * a logit is off by c = 2^-24 (2 (D + 64) + n + 8 max|y| + 32) relative to the sum of its terms' sizes at most, and so is a share p, relative to itself; sums of products take c too;
  * two terms leave out u of what the first leaves out: u^2 of a share or of a score gradient, in fp16 not less than 2^-25, in bfloat16 than 2^-126;
  * the result of the forward pass is kept in two terms too, for delta = do . o: off by u^2 |o| and by what o itself is off, (u^2 + c) p . |v|;
  * every result is rounded once: u of itself."""
import math

import torch


def attention(q, k, v, q_s, k_s, do, scale):
    """{name: (value, bound)}; q, k, v, do [Z, H, L, D], q_s [Z, H, L, 64], k_s [Z, L, 64]"""
    dtype = q.dtype
    u, tiny = torch.finfo(dtype).eps / 2, 2. ** -25 if dtype == torch.float16 else 2. ** -126
    q, k, v, q_s, k_s, do = [t.detach().double().cpu() for t in (q, k, v, q_s, k_s, do)]
    H, L, D = q.shape[1:]
    both_q, both_k = torch.cat([q, q_s], 3), torch.cat([k, k_s[:, None].expand(-1, H, -1, -1)], 3)
    seen = torch.ones(L, L, dtype=torch.bool).tril()
    s = scale * (both_q @ both_k.transpose(-1, -2))
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    big = float((scale * (both_q.abs() @ both_k.abs().transpose(-1, -2))).masked_fill(~seen, 0.).max())
    c, two = 2. ** -24 * (2 * (D + 64) + L + 8 * big + 32), u * u
    o, o_size, every = p @ v, p @ v.abs(), seen.double()
    dp = do @ v.transpose(-1, -2)
    delta = (do * o).sum(-1, keepdim=True)
    e = p * (dp - delta)
    # p is off by c of itself, dp by c |do| . |v|, delta by what o is off and c of its terms
    off = p * (c * (dp - delta).abs() + c * (do.abs() @ v.abs().transpose(-1, -2)) + (do.abs() * (two * o.abs() + (two + 2 * c) * o_size + tiny * (1 + every @ v.abs()))).sum(-1, keepdim=True))
    off = off * (1 + c) + (two + c) * e.abs() + (tiny + 2. ** -126 * (dp - delta).abs()) * every
    t = lambda x: x.transpose(-1, -2)    # noqa: E731
    dq, dk, dv = scale * (e @ both_k), scale * (t(e) @ both_q), t(p) @ do
    dq_b = u * dq.abs() + scale * (off @ both_k.abs()) + tiny
    dk_b = scale * (t(off) @ both_q.abs())
    out = dict(o=(o, u * o.abs() + (two + c) * o_size + tiny * (1 + every @ v.abs())), dv=(dv, u * dv.abs() + (two + c) * (t(p) @ do.abs()) + tiny * (1 + t(every) @ do.abs())))
    out['dq'], out['dq_s'] = [(dq[..., x], dq_b[..., x]) for x in (slice(0, D), slice(D, None))]
    out['dk'] = dk[..., :D], u * dk[..., :D].abs() + dk_b[..., :D] + tiny
    total = dk[..., D:].sum(1)
    out['dk_s'] = total, u * total.abs() + dk_b[..., D:].sum(1) + H * 2. ** -24 * dk[..., D:].abs().sum(1) + tiny
    return out
