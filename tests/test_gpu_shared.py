"""GPU: attention whose keys have a part that all heads share, forward and gradients against 64 bits (the oracle of attention with score rules over the parts side by side), and latent attention in both
forms as a program uses them, one after the other."""
import pytest
import torch

import rules_oracle as O
import torch_blocksparse as tb
from helpers import random_layout

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def randn(shape, dtype, seed, scale=1.):
    return (scale * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dtype).to(DEV)


def inputs(dtype, Z, H, kv, L, D, seed=0):
    sizes = dict(q=(Z, H, L, D), k=(Z, kv, L, D), v=(Z, kv, L, D), q_s=(Z, H, L, 64), k_s=(Z, L, 64), do=(Z, H, L, D))
    return {n: randn(s, dtype, seed + i) for i, (n, s) in enumerate(sizes.items())}


def expected(x, layout, block, **rules):
    D, kv = x['q'].size(3), x['k'].size(1)
    q, k = torch.cat([x['q'], x['q_s']], 3), torch.cat([x['k'], x['k_s'][:, None].expand(-1, kv, -1, -1)], 3)
    want = O.attention(q.cpu(), k.cpu(), x['v'].cpu(), layout, block, do=x['do'].cpu(), **{n: t.cpu() if isinstance(t, torch.Tensor) else t for n, t in rules.items()})
    out = dict(o=want['o'], dv=want['dv'])
    for name, both in (('q', want['dq']), ('k', want['dk'])):
        out['d' + name] = both[0][..., :D], both[1][..., :D]
        out['d' + name + '_s'] = both[0][..., D:], both[1][..., D:]
    # the sum over the key heads, in fp32 (each one's bound has the rounding to the type in it, which the sum takes once)
    value, bound = out['dk_s']
    out['dk_s'] = value.sum(1), bound.sum(1) + kv * 2. ** -24 * value.abs().sum(1)
    return out


def run(op, x, **rules):
    leaves = {n: x[n].detach().requires_grad_(True) for n in ('q', 'k', 'v', 'q_s', 'k_s')}
    o = op(leaves['q'], leaves['k'], leaves['v'], shared=(leaves['q_s'], leaves['k_s']), **rules)
    grads = torch.autograd.grad(o, list(leaves.values()), x['do'])
    return dict({'d' + n: g for n, g in zip(leaves, grads)}, o=o.detach())


def check(op, x, layout, block, **rules):
    got, want = run(op, x, **rules), expected(x, layout, block, **rules)
    for name in want:
        O.check(got[name], want[name], name)
    with torch.no_grad():
        assert torch.equal(op(x['q'], x['k'], x['v'], shared=(x['q_s'], x['k_s']), **rules), got['o'])
    return got


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('Z,H,kv,L,D,block,causal', [(1, 1, 1, 1, 64, 16, True), (2, 3, 3, 33, 64, 16, True), (1, 4, 2, 200, 128, 32, True), (2, 4, 4, 130, 128, 64, False),
                                                     (1, 8, 1, 97, 64, 64, True), (1, 2, 2, 500, 64, 128, True), (1, 5, 5, 64, 128, 16, False)])
def test_forward_and_gradients(dtype, Z, H, kv, L, D, block, causal):
    blocks = -(-L // block)
    for layout in (torch.ones(H, blocks, blocks, dtype=torch.int64), random_layout((H, blocks, blocks), 0.5, L)):
        check(tb.Attention(layout, block), inputs(dtype, Z, H, kv, L, D, L), layout, block, scale=(D + 64) ** -0.5, causal=causal)


@pytest.mark.parametrize('dtype,D', [(torch.float16, 64), (torch.bfloat16, 128)])
def test_many_lines(dtype, D):
    """so many that a line is one pair of wavefronts', with several tiles"""
    Z, H, L = 9, 16, 500
    layout = torch.ones(H, 8, 8, dtype=torch.int64)
    check(tb.Attention(layout, 64), inputs(dtype, Z, H, H, L, D, 11), layout, 64, scale=0.08, causal=True)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('D', [64, 128])
def test_rules(dtype, D):
    Z, H, L, block = 2, 4, 150, 32
    layout = random_layout((H, 5, 5), 0.7, 1)
    layout[:, 3] = 0                                           # rows that see nothing
    x = inputs(dtype, Z, H, H, L, D, 3)
    documents = torch.tensor([[0] * 40 + [1] * 65 + [2] * 30 + [-1] * 15, [-1] * 3 + [5] * 147], dtype=torch.int32, device=DEV)
    slopes = torch.tensor([0.5 ** (h + 1) for h in range(H)], device=DEV)
    prefix = torch.tensor([20, 90], dtype=torch.int32, device=DEV)
    op = tb.Attention(layout, block)
    for rules in (dict(softcap=4.), dict(slopes=slopes), dict(documents=documents), dict(causal=True, prefix=prefix), dict(softcap=20., slopes=slopes, documents=documents, causal=True, prefix=prefix)):
        check(op, x, layout, block, scale=0.1, **rules)
    # what padding holds reaches nothing
    clean = run(op, x, scale=0.1, documents=documents)
    pad = (documents < 0)[:, None, :, None]
    dirty = {n: t.masked_fill(pad if t.dim() == 4 else pad[:, 0], float('nan')) for n, t in x.items()}
    got = run(op, dirty, scale=0.1, documents=documents)
    assert all(torch.equal(got[n], clean[n]) for n in clean)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_long_columns_in_parts(dtype):
    Z, H, L, D, block = 1, 2, 1500, 64, 64
    layout = torch.zeros(H, 24, 24, dtype=torch.int64)
    layout[:, :, 0] = 1
    layout[:, torch.arange(24), torch.arange(24)] = 1
    x = inputs(dtype, Z, H, H, L, D, 5)
    op = tb.Attention(layout, block)
    first = check(op, x, layout, block, scale=0.09, causal=True)
    again = run(op, x, scale=0.09, causal=True)
    assert all(torch.equal(first[n], again[n]) for n in first)


def test_many_lines_take_the_other_kernels():
    """Launches of more lines have one pair of wavefronts a line"""
    Z, H, L, D, block = 8, 16, 1100, 64, 64
    layout = torch.eye(18, dtype=torch.int64)[None].repeat(H, 1, 1)
    x = inputs(torch.bfloat16, Z, H, H, L, D, 5)
    got = run(tb.Attention(layout, block), x, scale=0.09, causal=True)
    for z in (0, 7):
        one = {n: t[z:z + 1] for n, t in x.items()}
        want = expected(one, layout, block, scale=0.09, causal=True)
        for n in want:
            O.check(got[n][z:z + 1], want[n], n)


def test_a_shared_part_of_zeros_is_none():
    layout, block = torch.ones(3, 4, 4, dtype=torch.int64), 32
    x = inputs(torch.float32, 2, 3, 3, 120, 64)
    op = tb.Attention(layout, block)
    x['q_s'].zero_()
    got = run(op, x, scale=0.1, causal=True)
    q, k, v = [x[n].detach().requires_grad_(True) for n in 'qkv']
    o = op(q, k, v, scale=0.1, causal=True)
    want = torch.autograd.grad(o, (q, k, v), x['do'])
    # (the same sums with products of zeros behind them)
    assert torch.equal(got['o'], o) and all(torch.equal(got[n], w) for n, w in zip(('dq', 'dk', 'dv'), want))
    assert not bool(got['dk_s'].any()) and bool(got['dq_s'].any())


def test_gradients_against_differences():
    layout, block = torch.ones(2, 2, 2, dtype=torch.int64), 16
    x = inputs(torch.float32, 1, 2, 2, 20, 64, 7)
    op = tb.Attention(layout, block)
    rules = dict(scale=0.1, causal=True)
    got = run(op, x, **rules)
    with torch.no_grad():
        for i, n in enumerate(('q', 'k', 'v', 'q_s', 'k_s')):
            d, h = randn(tuple(x[n].shape), torch.float32, 50 + i), 2. ** -5
            at = lambda s: {m: (t.double() + s * h * d.double() if m == n else t.double()).float() for m, t in x.items()}    # noqa: E731
            values = []
            for s in (1., -1.):
                y = at(s)
                values.append((op(y['q'], y['k'], y['v'], shared=(y['q_s'], y['k_s']), **rules).double() * x['do'].double()).sum())
            slope, exact = (values[0] - values[1]) / (2 * h), (got['d' + n].double() * d.double()).sum()
            # the third derivative's h^2 / 6 (scores move by 0.1 * 16 h at most a standard deviation, of sums of about 2560 terms of size one) and fp32's 2^-22 of the sums over 2 h
            assert abs(slope - exact) < 2560 ** 0.5 * ((1.6 * h) ** 2 + 2. ** -22 * 64 / h), (n, float(slope), float(exact))


def test_only_some_gradients():
    layout, block = torch.ones(3, 4, 4, dtype=torch.int64), 32
    x = inputs(torch.bfloat16, 2, 3, 3, 120, 64)
    op = tb.Attention(layout, block)
    full = run(op, x, scale=0.1)
    for wanted in (['q_s'], ['k_s'], ['q', 'k_s'], ['v']):
        leaves = {n: x[n].detach().clone().requires_grad_(n in wanted) for n in ('q', 'k', 'v', 'q_s', 'k_s')}
        o = op(leaves['q'], leaves['k'], leaves['v'], scale=0.1, shared=(leaves['q_s'], leaves['k_s']))
        o.backward(x['do'])
        for n, t in leaves.items():
            assert (t.grad is not None) == (n in wanted)
            if n in wanted:
                assert torch.equal(t.grad, full['d' + n])


def test_views_and_copies():
    layout, block = torch.ones(4, 4, 4, dtype=torch.int64), 32
    x = inputs(torch.bfloat16, 2, 4, 4, 100, 128)
    op = tb.Attention(layout, block)
    want = run(op, x, scale=0.1)
    q = torch.cat([x['q'], x['q_s']], 3).transpose(1, 2).contiguous().transpose(1, 2)           # one projection gives both parts
    latent = torch.cat([randn((2, 100, 512), torch.bfloat16, 9), x['k_s']], 2)
    odd = torch.empty(x['k_s'].numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].view(2, 100, 64).copy_(x['k_s'])
    for q_s, k_s in ((q[..., 128:], latent[..., 512:]), (q[..., 128:], odd)):
        got = run(op, dict(x, q=q[..., :128], q_s=q_s, k_s=k_s), scale=0.1)
        assert all(torch.equal(got[n], want[n]) for n in want)
    same_keys = x['k_s'][:1].expand(2, 100, 64)
    got, same = run(op, dict(x, k_s=same_keys), scale=0.1), run(op, dict(x, k_s=same_keys.contiguous()), scale=0.1)
    assert all(torch.equal(got[n], same[n]) for n in same)
    empty = {n: t[:0].requires_grad_(True) for n, t in x.items()}
    op(empty['q'], empty['k'], empty['v'], shared=(empty['q_s'], empty['k_s'])).sum().backward()
    assert empty['k_s'].grad.shape == (0, 100, 64)


def test_captured():
    layout, block = torch.ones(2, 4, 4, dtype=torch.int64), 32
    x = inputs(torch.bfloat16, 1, 2, 2, 120, 64)
    op = tb.Attention(layout, block)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(op, x, scale=0.1, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(op, x, scale=0.1, causal=True)
    for i in range(3):
        for n, t in inputs(torch.bfloat16, 1, 2, 2, 120, 64, 40 + 10 * i).items():
            x[n].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = run(op, x, scale=0.1, causal=True)
        assert all(torch.equal(got[n], want[n]) for n in want)


# ---- both forms of latent attention, one after the other ------------------------------------------------------------------------------


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('mode', ['dense', 'fixed'])
def test_a_prompt_and_then_an_answer(dtype, mode):
    """A prompt by the expanded form with rotated positions, its latent vectors appended to a cache, and its last position again by the absorbed form: the same up to what the matrices' products
    round between them"""
    Z, H, L, D, latent, block = 2, 4, 150, 128, 512, 32
    module = tb.SparseSelfAttention(tb.SparsityConfig(mode=mode, block=block, stride=64, attention='unidirectional'))
    rotation = tb.Rotation.of_base(64, neighbours=True)
    # numbers whose products with the matrices are exact in the type: each expanded element is a sum of two latent ones
    g = torch.Generator().manual_seed(1)
    c = (torch.randint(-8, 9, (Z, L, latent), generator=g) / 8.).to(dtype).to(DEV)
    pick = torch.randint(0, latent, (2, H, D, 2), generator=g)
    matrices = torch.zeros(2, H, D, latent).scatter_add_(3, pick, torch.ones(2, H, D, 2)).to(DEV)
    k, v = [torch.einsum('zlc,hdc->zhld', c.float(), w).to(dtype) for w in matrices]
    n, t, r = randn((Z, H, L, D), dtype, 2), randn((Z, H, L, 64), dtype, 3), randn((Z, L, 64), dtype, 4)
    positions = torch.arange(L, dtype=torch.int32, device=DEV) + 1000
    t_at, r_at = rotation(t, r[:, None], positions=positions)
    o = module(n, k, v, causal=True, shared=(t_at, r_at[:, 0]))
    cache = tb.LatentCache(20, block, latent, dtype=dtype)
    table = torch.randperm(20, generator=g)[:Z * 5].int().view(Z, 5).to(DEV)
    slots = (table.long().repeat_interleave(block, 1) * block + torch.arange(5 * block, device=DEV) % block)[:, :L].flatten().int()
    cache.write(c.flatten(0, 1), r.flatten(0, 1), slots, rotation=rotation, positions=positions.repeat(Z))
    lengths = torch.full((Z,), L, dtype=torch.int32, device=DEV)
    absorbed = torch.einsum('zhd,hdc->zhc', n[:, :, -1].float(), matrices[0]).to(dtype)
    y = module.decode(absorbed, cache, table, lengths, shared=t_at[:, :, -1].contiguous(), scale=(D + 64) ** -0.5)
    got = torch.einsum('zhc,hdc->zhd', y.float(), matrices[1])
    # absorbed queries are rounded once (u of up to four latent elements of size one each, 128 of them), the sums of the shares' c once more; so is o
    u = torch.finfo(dtype).eps / 2
    off = (D + 64) ** -0.5 * u * (n[:, :, -1].float().abs().sum(-1, keepdim=True) * 2)
    bound = 2 * off * 2 + 8 * u * 2
    assert bool(((got - o[:, :, -1].float()).abs() <= bound).all()), float(((got - o[:, :, -1].float()).abs() / bound).max())


def test_rotation_feeds_attention():
    """Gradients through the rotation, attention with a shared part and back"""
    layout, block = torch.ones(2, 3, 3, dtype=torch.int64), 32
    x = inputs(torch.float32, 1, 2, 2, 90, 64)
    op, rotation = tb.Attention(layout, block), tb.Rotation.of_base(64)
    leaves = {n: x[n].detach().requires_grad_(True) for n in ('q', 'k', 'v', 'q_s', 'k_s')}
    q_s, k_s = rotation(leaves['q_s'], leaves['k_s'][:, None])
    op(leaves['q'], leaves['k'], leaves['v'], scale=0.1, causal=True, shared=(q_s, k_s[:, 0])).backward(x['do'])
    ahead = [x['q_s'].detach().requires_grad_(True), x['k_s'].detach().requires_grad_(True)]
    turned = rotation(ahead[0], ahead[1][:, None])
    got = run(op, dict(x, q_s=turned[0].detach(), k_s=turned[1].detach()[:, 0]), scale=0.1, causal=True)
    back = torch.autograd.grad(turned, ahead, (got['dq_s'], got['dk_s'][:, None]))
    assert torch.equal(leaves['q_s'].grad, back[0]) and torch.equal(leaves['k_s'].grad, back[1])
    assert torch.equal(leaves['q'].grad, got['dq'])
