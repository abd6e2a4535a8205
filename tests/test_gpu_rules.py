"""GPU: torch_blocksparse.Attention (score rules) against the same in 64 bits, forward and gradients, bounds from rules_oracle."""
import itertools

import pytest
import torch

import torch_blocksparse as tb
from helpers import random_layout
import rules_oracle

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def inputs(Z, H, kv, L, D, dtype, seed, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    return [(spread * torch.randn(Z, h, L, D, generator=g)).to(dtype).to(DEV) for h in (H, kv, kv, H)]


def documents_of(Z, L, n, seed, pad=True):
    g = torch.Generator().manual_seed(seed)
    ids = torch.sort(torch.randint(0, max(n, 1), (Z, L), generator=g), 1).values
    if pad:
        for z in range(Z):
            ids[z, L - L // (z + 4):] = -1
            ids[z, :z * 3] = -7
    return ids.int().to(DEV)


def run(op, q, k, v, do, **rules):
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    o = op(*leaves, **rules)
    return (o.detach(),) + torch.autograd.grad(o, leaves, do)


def compare(op, layout, block, q, k, v, do, what, **rules):
    got = run(op, q, k, v, do, **rules)
    want = rules_oracle.attention(q, k, v, layout, block, do, **rules)
    worst = [rules_oracle.check(g, want[n], '%s %s' % (what, n)) for g, n in zip(got, ('o', 'dq', 'dk', 'dv'))]
    with torch.no_grad():
        assert torch.equal(op(q, k, v, **rules), got[0])
    print(what, 'worst share of the bounds: ' + ', '.join('%.2f' % w for w in worst))
    return got


def rules_of(name, Z, H, L, seed=3):
    slopes = torch.tensor([2. ** (-8. * (h + 1) / H) for h in range(H)], device=DEV)
    prefix = torch.tensor([(5 + 17 * z) % (L + 1) for z in range(Z)], dtype=torch.int32, device=DEV)
    return {'plain': dict(), 'causal': dict(causal=True), 'cap': dict(softcap=7.), 'slopes': dict(slopes=slopes), 'documents': dict(documents=documents_of(Z, L, 4, seed)),
            'prefix': dict(causal=True, prefix=prefix),
            'all': dict(causal=True, prefix=prefix, softcap=11., slopes=slopes, documents=documents_of(Z, L, 3, seed))}[name]


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('name', ['plain', 'causal', 'cap', 'slopes', 'documents', 'prefix', 'all'])
def test_each_rule(dtype, name):
    Z, H, kv, L, D, block = 2, 4, 2, 171, 64, 16
    lay = random_layout((H, 11, 11), 0.5, 5)
    q, k, v, do = inputs(Z, H, kv, L, D, dtype, 11)
    compare(tb.Attention(lay, block), lay, block, q, k, v, do, '%s %s' % (name, dtype), scale=D ** -0.5, **rules_of(name, Z, H, L))


@pytest.mark.parametrize('dtype,D', [(torch.float16, 64), (torch.bfloat16, 128), (torch.float32, 128)])
@pytest.mark.parametrize('L,block', [(1, 16), (2, 128), (15, 16), (16, 16), (17, 16), (33, 32), (63, 64), (64, 64), (65, 64), (129, 128), (200, 128), (300, 32), (449, 64)])
def test_lengths_and_blocks(dtype, D, L, block):
    Z, H, kv = 2, 3, 1
    blocks = -(-L // block)
    lay = random_layout((H, blocks, blocks), 0.6, L)
    q, k, v, do = inputs(Z, H, kv, L, D, dtype, L)
    compare(tb.Attention(lay, block), lay, block, q, k, v, do, 'L %d block %d' % (L, block), scale=0.3, **rules_of('all', Z, H, L, L))


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('H,kv', [(1, 1), (8, 8), (8, 1), (6, 3)])
def test_shared_heads_long_columns_and_parts(H, kv, D):
    # dense causal at 40 tiles a row: lines that take several rounds of the walk, columns that are cut into parts
    L, block = 2500, 64
    lay = torch.ones(H, 40, 40, dtype=torch.int64).tril()
    q, k, v, do = inputs(1, H, kv, L, D, torch.bfloat16, 1)
    op = tb.Attention(lay, block)
    compare(op, lay, block, q, k, v, do, 'H %d kv %d' % (H, kv), scale=D ** -0.5, causal=True, softcap=20.)
    assert op.tables(q.device).columns(kv, 1)[4] > 0


def test_many_documents_skip_tiles():
    Z, H, L, D, block = 3, 2, 1000, 64, 64
    lay = torch.ones(H, 16, 16, dtype=torch.int64)
    q, k, v, do = inputs(Z, H, H, L, D, torch.float16, 2)
    ids = documents_of(Z, L, 40, 9)
    ids[1] = -1                                             # a sequence of nothing
    ids[2] = ids[2].flip(0)                                 # descending numbers, padding in front
    got = compare(tb.Attention(lay, block), lay, block, q, k, v, do, 'documents', scale=0.125, documents=ids)
    assert all(not bool(t[1].any()) for t in got)
    # numbers in no order, and as large as they come
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 3, (Z, L), generator=g).int().to(DEV) * 1073741823
    compare(tb.Attention(lay, block), lay, block, q, k, v, do, 'mixed documents', scale=0.125, documents=ids, causal=True)


def test_rows_and_columns_without_blocks():
    H, block, D = 2, 32, 64
    lay = random_layout((H, 9, 9), 0.4, 8)
    lay[0, 2:5] = 0                                         # rows that see nothing: whole lines and halves of lines
    lay[1, :, 3] = 0
    lay[1, :, 6:8] = 0
    q, k, v, do = inputs(2, H, H, 9 * block, D, torch.float16, 3)
    got = compare(tb.Attention(lay, block), lay, block, q, k, v, do, 'holes', scale=0.2)
    assert not bool(got[0][:, 0, 64:160].any()) and not bool(got[1][:, 0, 64:160].any()) and not bool(got[2][:, 1, 96:128].any())


def test_an_empty_layout_and_an_empty_batch():
    lay = torch.zeros(2, 3, 3, dtype=torch.int64)
    q, k, v, do = inputs(1, 2, 2, 48, 64, torch.float16, 3)
    assert not any(bool(t.any()) for t in run(tb.Attention(lay, 16), q, k, v, do))
    out = run(tb.Attention(torch.ones(2, 3, 3), 16), q[:0], k[:0], v[:0], do[:0])
    assert all(t.shape == (0, 2, 48, 64) for t in out)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('causal', [False, True])
def test_padding_may_hold_anything(dtype, causal):
    Z, H, kv, L, D, block = 2, 2, 1, 150, 64, 16
    lay = torch.ones(H, 10, 10, dtype=torch.int64)
    op = tb.Attention(lay, block)
    q, k, v, do = inputs(Z, H, kv, L, D, dtype, 6)
    ids = documents_of(Z, L, 3, 1)
    rules = dict(scale=0.125, softcap=9., causal=causal, documents=ids)
    clean = compare(op, lay, block, q, k, v, do, 'padding', **rules)
    pad = (ids < 0)[:, None, :, None]
    assert bool(pad[1, 0, 0]) and bool(pad[1, 0, -1])
    for value in (float('nan'), float('inf'), torch.finfo(dtype).min):
        dirty = run(op, *[t.masked_fill(pad, value) for t in (q, k, v, do)], **rules)
        for a, b in zip(clean, dirty):
            assert torch.equal(a, b)


def test_scales_of_all_kinds():
    H, L, D, block = 2, 130, 64, 64
    lay = torch.ones(H, 3, 3, dtype=torch.int64)
    op = tb.Attention(lay, block)
    q, k, v, do = inputs(1, H, H, L, D, torch.bfloat16, 12)
    for scale, cap in ((-0.2, 0.), (0., 0.), (0., 5.), (-0.5, 3.), (1e-20, 0.), (4., 2.), (0.05, 1000.)):
        compare(op, lay, block, q, k, v, do, 'scale %g cap %g' % (scale, cap), scale=scale, softcap=cap, causal=True)
    # logits far from zero: what the rounding of a row's reference leaves out counts
    q, k = q.abs() + 4, k.abs() + 4
    compare(op, lay, block, q, k, v, do, 'large', scale=0.5)


def test_strides_and_addresses():
    Z, H, kv, L, D, block = 2, 4, 2, 100, 64, 32
    lay = torch.ones(H, 4, 4, dtype=torch.int64).tril()
    op = tb.Attention(lay, block)
    q, k, v, do = inputs(Z, H, kv, L, D, torch.float16, 13)
    rules = dict(scale=0.125, causal=True)
    want = run(op, q, k, v, do, **rules)
    packed = torch.cat([t.transpose(1, 2) for t in (q, k, v)], 2)                        # [Z, L, heads, D], as a projection gives them
    views = [t.transpose(1, 2) for t in packed.split((H, kv, kv), 2)]
    odd = [torch.empty(t.numel() + 3, dtype=t.dtype, device=DEV)[3:].view(t.shape).copy_(t) for t in (q, k, v)]
    wide = [torch.empty(t.shape[:3] + (D + 4,), dtype=t.dtype, device=DEV)[..., :D].copy_(t) for t in (q, k, v)]
    inner = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)]
    for name, (a, b, c) in dict(views=views, odd=odd, wide=wide, inner=inner).items():
        got = run_views(op, a, b, c, do, **rules)
        for x, y in zip(got, want):
            assert torch.equal(x, y), name
    # one key head for all, given as a view of stride 0, and a gradient that is one row for all
    k1, v1 = k[:, :1], v[:, :1]
    shared = run(op, q, k1, v1, do, **rules)
    o = op(q, k1.expand(Z, H, L, D), v1.expand(Z, H, L, D), **rules)
    assert torch.equal(o, shared[0])
    row = do[:, :, :1].expand(Z, H, L, D)
    for x, y in zip(run(op, q, k, v, row, **rules), run(op, q, k, v, row.contiguous(), **rules)):
        assert torch.equal(x, y)
    # documents as a slice and as a transposed tensor
    ids = torch.randint(0, 3, (Z, L + 5), dtype=torch.int32, device=DEV)[:, 2:L + 2]
    for view in (ids, ids.t().contiguous().t()):
        assert torch.equal(op(q, k, v, documents=view), op(q, k, v, documents=ids.contiguous()))


def run_views(op, q, k, v, do, **rules):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = op(*leaves, **rules)
    return (o.detach(),) + torch.autograd.grad(o, leaves, do)


@pytest.mark.parametrize('which', [c for n in (1, 2) for c in itertools.combinations(range(3), n)])
def test_some_of_the_gradients(which):
    lay = torch.ones(2, 3, 3, dtype=torch.int64)
    op = tb.Attention(lay, 32)
    q, k, v, do = inputs(1, 2, 2, 90, 64, torch.float16, 14)
    want = run(op, q, k, v, do, softcap=5.)[1:]
    leaves = [t.detach().clone().requires_grad_(i in which) for i, t in enumerate((q, k, v))]
    got = torch.autograd.grad(op(*leaves, softcap=5.), [leaves[i] for i in which], do)
    for i, g in zip(which, got):
        assert torch.equal(g, want[i])


def test_gradients_by_differences():
    # (f(x + h d) - f(x - h d)) / 2h in fp32, for f = sum(o * do): h = 2^-7 leaves h^2 / 6 times third derivatives of the order of the first (1e-5) and 2^-24 / h of rounding
    H, L, D, block = 2, 70, 64, 16
    lay = random_layout((H, 5, 5), 0.6, 3)
    op = tb.Attention(lay, block)
    q, k, v, do = inputs(1, H, 1, L, D, torch.float32, 15, spread=0.7)
    rules = dict(scale=0.125, softcap=3., slopes=torch.tensor([0.1, 0.02], device=DEV), causal=True, documents=documents_of(1, L, 2, 3))
    grads = run(op, q, k, v, do, **rules)[1:]
    g = torch.Generator().manual_seed(1)
    for i in range(3):
        d = torch.randn(grads[i].shape, generator=g).to(DEV)
        ends = []
        for sign in (1, -1):
            moved = [t + sign * 2. ** -7 * d if j == i else t for j, t in enumerate((q, k, v))]
            ends.append((op(*moved, **rules).double() * do.double()).sum())
        slope, want = (ends[0] - ends[1]) / 2. ** -6, (grads[i].double() * d.double()).sum()
        assert abs(float(slope - want)) <= 1e-3 * float((grads[i].double() * d.double()).abs().sum()) / grads[i].numel() ** 0.5 + 1e-3 * abs(float(want)), (i, float(slope), float(want))


def test_another_stream_and_the_same_bits():
    lay = torch.ones(4, 8, 8, dtype=torch.int64).tril()
    op = tb.Attention(lay, 64)
    q, k, v, do = inputs(2, 4, 2, 500, 64, torch.bfloat16, 16)
    ids = documents_of(2, 500, 5, 2)
    want = run(op, q, k, v, do, documents=ids, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(op, q, k, v, do, documents=ids, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_captured_and_replayed():
    lay = torch.ones(2, 6, 6, dtype=torch.int64).tril()
    op = tb.Attention(lay, 64)
    static = inputs(2, 2, 1, 370, 64, torch.float16, 17)
    ids = documents_of(2, 370, 3, 5)
    rules = dict(scale=0.125, softcap=15., causal=True, documents=ids)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(op, *static, **rules)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(op, *static, **rules)
    for seed in (21, 22, 23):
        for t, new in zip(static, inputs(2, 2, 1, 370, 64, torch.float16, seed)):
            t.copy_(new)
        ids.copy_(documents_of(2, 370, 3, seed))
        eager = run(op, *static, **rules)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)


def test_operands_changed_before_the_backward_pass_are_refused():
    lay = torch.ones(2, 2, 2, dtype=torch.int64)
    op = tb.Attention(lay, 16)
    q, k, v, do = inputs(1, 2, 2, 32, 64, torch.float16, 18)
    q.requires_grad_(True)
    ids = torch.zeros(1, 32, dtype=torch.int32, device=DEV)
    o = op(q, k, v, documents=ids)
    ids.fill_(1)
    with pytest.raises(RuntimeError, match='modified'):
        o.backward(do)


def test_far_positions():
    # positions past 16 bits, a bias by distance over all of them; one row of tiles a head
    H, block, L, D = 1, 128, 70000, 64
    blocks = -(-L // block)
    lay = torch.zeros(H, blocks, blocks, dtype=torch.int64)
    lay[:, -1, ::91] = 1
    lay[:, -1, -1] = 1
    q, k, v, do = inputs(1, H, 1, L, D, torch.float32, 19)
    op = tb.Attention(lay, block)
    slopes = torch.tensor([2. ** -14], device=DEV)
    got = run(op, q, k, v, do, scale=0.125, slopes=slopes, causal=True)
    first = (blocks - 1) * block
    keys = torch.nonzero(lay[0, -1].repeat_interleave(block)[:L])[:, 0]
    rows = torch.arange(first, L)
    s = 0.125 * (q[0, 0, rows].double().cpu() @ k[0, 0, keys].double().cpu().t()) - slopes.item() * (rows[:, None] - keys).abs()
    s = s.masked_fill(keys > rows[:, None], float('-inf'))
    p = s.softmax(1)
    vv = v[0, 0, keys].double().cpu()
    # logits of up to 12, a bias up to 4.3: 2^-24 * (128 + 1000 keys + 8 * 16 + 32) = 8e-5 of the terms
    assert bool(((got[0][0, 0, rows].double().cpu() - p @ vv).abs() <= 8e-5 * (p @ vv.abs())).all())
    dv = p.t() @ do[0, 0, rows].double().cpu()
    assert bool(((got[3][0, 0, keys].double().cpu() - dv).abs() <= 8e-5 * (p.t() @ do[0, 0, rows].double().cpu().abs())).all())
    assert not bool(got[0][0, 0, :first].any())


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('name', ['causal', 'all'])
def test_a_launch_of_few_lines_and_one_of_many(dtype, D, name):
    """Few lines have two pairs of wavefronts each, many one: the same sequence alone and 120 times over."""
    H, kv, L, block, times = 4, 2, 300, 32, 120
    lay = random_layout((H, 10, 10), 0.6, 9)
    lay[:, 3] = 0                                        # rows that see nothing, and a line of an odd number of halves
    op = tb.Attention(lay, block)
    q, k, v, do = inputs(1, H, kv, L, D, dtype, 21)
    rules = dict(rules_of(name, 1, H, L), scale=D ** -0.5)
    compare(op, lay, block, q, k, v, do, 'few %s %d %s' % (name, D, dtype), **rules)
    want = rules_oracle.attention(q, k, v, lay, block, do, **rules)
    many = {n: t.expand(times, *t.shape[1:]).contiguous() if n in ('documents', 'prefix') else t for n, t in rules.items()}
    got = run(op, *[t.expand(times, -1, -1, -1).contiguous() for t in (q, k, v, do)], **many)
    for z in (0, 57, times - 1):
        for g, n in zip(got, ('o', 'dq', 'dk', 'dv')):
            rules_oracle.check(g[z:z + 1], want[n], 'many %s' % n)
    for g in got:
        assert torch.equal(g[:1].expand_as(g), g)
