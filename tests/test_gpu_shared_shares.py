"""GPU: attention with a shared key part, forward and gradients against 64 bits, under bounds that have no place for an operand that is rounded to the type in one term."""
import pytest
import torch

import rules_oracle
import shared_oracle as O
import torch_blocksparse as tb

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('Z,H,L,D', [(1, 1, 1, 64), (2, 3, 7, 64), (2, 2, 12, 128), (1, 4, 45, 64), (1, 3, 100, 128), (9, 16, 300, 64), (9, 16, 300, 128)])
def test_operands_in_two_terms(dtype, Z, H, L, D):
    """(the last two: launches of more lines, of 64 elements with two pairs of wavefronts each, of 128 with one)"""
    g = torch.Generator().manual_seed(L)
    x = {n: torch.randn(s, generator=g) for n, s in (('q', (Z, H, L, D)), ('k', (Z, H, L, D)), ('v', (Z, H, L, D)), ('q_s', (Z, H, L, 64)), ('k_s', (Z, L, 64)), ('do', (Z, H, L, D)))}
    for n in ('q', 'q_s'):
        x[n] *= 0.3                                       # (shares alike, so that their roundings are what counts)
    x = {n: t.to(dtype).to(DEV) for n, t in x.items()}
    leaves = {n: x[n].requires_grad_(True) for n in ('q', 'k', 'v', 'q_s', 'k_s')}
    block = 16 if L < 64 else 64
    blocks = -(-L // block)
    o = tb.Attention(torch.ones(H, blocks, blocks, dtype=torch.int64).tril(), block)(x['q'], x['k'], x['v'], scale=(D + 64) ** -0.5, causal=True, shared=(x['q_s'], x['k_s']))
    got = dict(zip(('dq', 'dk', 'dv', 'dq_s', 'dk_s'), torch.autograd.grad(o, list(leaves.values()), x['do'])), o=o)
    want = O.attention(*[x[n] for n in ('q', 'k', 'v', 'q_s', 'k_s', 'do')], (D + 64) ** -0.5)
    for n in want:
        rules_oracle.check(got[n], want[n], n)
