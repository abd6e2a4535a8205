"""GPU: calls of Attention, KeyValueCache and CacheAttention in ways that programs have: one tensor for several operands, expanded operands and
gradients, saved tensors that were moved, operators shared by two streams, pages shared by sequences."""
import pytest
import torch

import rules_oracle as R
import torch_blocksparse as tb
from helpers import random_layout

pytestmark = pytest.mark.gpu
DEV = 'cuda'
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def randn(*shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


@pytest.mark.parametrize('dtype', DTYPES)
def test_one_tensor_as_query_key_and_value(dtype):
    H, L, block = 2, 100, 16
    lay = random_layout((H, 7, 7), 0.6, 1)
    op = tb.Attention(lay, block)
    x, do = randn(2, H, L, 64, dtype=dtype, seed=1), randn(2, H, L, 64, dtype=dtype, seed=2)
    want = R.attention(x, x, x, lay, block, do, scale=0.125, causal=True)
    leaf = x.clone().requires_grad_(True)
    o = op(leaf, leaf, leaf, scale=0.125, causal=True)
    o.backward(do)
    R.check(o, want['o'], 'o')
    value = sum(want[n][0] for n in ('dq', 'dk', 'dv'))
    # each addition of two of them is rounded to the type once more
    u = torch.finfo(dtype).eps / 2
    bound = sum(want[n][1] for n in ('dq', 'dk', 'dv')) + 2.1 * u * sum(want[n][0].abs() + want[n][1] for n in ('dq', 'dk', 'dv'))
    R.check(leaf.grad, (value, bound), 'gradient')


@pytest.mark.parametrize('dtype', DTYPES)
def test_gradients_that_are_expanded_or_in_another_order(dtype):
    B, H, L, D, block = 2, 2, 70, 64, 32
    lay = torch.ones(H, 3, 3)
    op = tb.Attention(lay, block)
    q, k, v = [randn(B, H, L, D, dtype=dtype, seed=s).requires_grad_(True) for s in (3, 4, 5)]
    for do in (torch.ones((), dtype=dtype, device=DEV).expand(B, H, L, D), randn(L, D, dtype=dtype, seed=6).expand(B, H, L, D),
               randn(B, L, H, D, dtype=dtype, seed=7).transpose(1, 2), randn(B, H, D, L, dtype=dtype, seed=8).transpose(2, 3)):
        want = R.attention(q, k, v, lay, block, do, scale=0.125)
        for got, n in zip(torch.autograd.grad(op(q, k, v, scale=0.125), (q, k, v), do), ('dq', 'dk', 'dv')):
            R.check(got, want[n], n)


def test_saved_tensors_that_were_elsewhere():
    B, H, L, D, block = 2, 2, 70, 64, 32
    op = tb.Attention(torch.ones(H, 3, 3), block)
    x = [randn(B, L, H, D, dtype=torch.bfloat16, seed=s).transpose(1, 2).requires_grad_(True) for s in (3, 4, 5)]
    do = randn(B, H, L, D, dtype=torch.bfloat16, seed=6)
    ids = torch.tensor([0] * 30 + [1] * 35 + [-1] * 5, dtype=torch.int32, device=DEV).expand(B, L)
    rules = dict(scale=0.125, softcap=20., causal=True, documents=ids, slopes=torch.tensor([0.1, 0.], device=DEV))
    want = torch.autograd.grad(op(*x, **rules), x, do)
    with torch.autograd.graph.save_on_cpu():
        o = op(*x, **rules)
    for a, b in zip(torch.autograd.grad(o, x, do), want):
        assert torch.equal(a, b)


def test_documents_and_a_prefix_that_are_expanded():
    B, H, L, D, block = 3, 2, 50, 64, 16
    lay = random_layout((H, 4, 4), 0.7, 2)
    op = tb.Attention(lay, block)
    q, k, v, do = [randn(B, H, L, D, dtype=torch.float16, seed=s) for s in (1, 2, 3, 4)]
    ids = torch.tensor([4] * 20 + [2] * 25 + [-1] * 5, dtype=torch.int32, device=DEV)
    prefix = torch.tensor([23], dtype=torch.int32, device=DEV)
    wide = torch.stack([ids, ids], 1)                    # every other element
    for documents in (ids.expand(B, L), wide[:, 0].expand(B, L)):
        rules = dict(scale=0.125, causal=True, documents=documents, prefix=prefix.expand(B))
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        o = op(*leaves, **rules)
        o.backward(do)
        want = R.attention(q, k, v, lay, block, do, **rules)
        for got, n in zip([o] + [t.grad for t in leaves], ('o', 'dq', 'dk', 'dv')):
            R.check(got, want[n], n)
    # prefixes outside the positions: none of them, all of them
    for n in (-5, 2 ** 31 - 1):
        rules = dict(scale=0.125, causal=True, prefix=torch.full((B,), n, dtype=torch.int32, device=DEV))
        R.check(op(q, k, v, **rules), R.attention(q, k, v, lay, block, **rules)['o'], 'prefix %d' % n)


def test_two_streams_share_the_operators():
    B, H, L, D, block = 2, 4, 600, 64, 64
    lay = tb.fixed_layout(H, 10, 'dense', 1, 'unidirectional', 1, 1)
    op, cache = tb.Attention(lay, block), tb.KeyValueCache(40, block, H, D, bits=8)
    decode = tb.CacheAttention(block, lay)
    sets = [[randn(B, H, L, D, dtype=torch.float16, seed=10 * i + s).requires_grad_(True) for s in range(3)] for i in range(2)]
    do = randn(B, H, L, D, dtype=torch.float16, seed=99)
    pages = [torch.arange(20 * i, 20 * i + 20, dtype=torch.int32, device=DEV).view(B, 10) for i in range(2)]
    at = torch.arange(L, device=DEV)
    lengths = torch.full((B,), L, dtype=torch.int32, device=DEV)

    def work(i):
        q, k, v = sets[i]
        o = op(q, k, v, scale=0.125, causal=True)
        grads = torch.autograd.grad(o, (q, k, v), do)
        slots = (pages[i][:, at // block] * block + at % block).int().flatten()
        cache.write(k.detach().transpose(1, 2).flatten(0, 1), v.detach().transpose(1, 2).flatten(0, 1), slots)
        return (o.detach(),) + grads + (decode(q[:, :, -1].detach(), cache, pages[i], lengths, scale=0.125),)

    want = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(work(i))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert not bool(cache._owner.any())


@pytest.mark.parametrize('bits', [4, 8])
def test_pages_that_sequences_share(bits):
    """One prompt's pages in several sequences, a page twice in one, one table for all."""
    H, kv, D, block = 4, 2, 64, 16
    cache = tb.KeyValueCache(9, block, kv, D, bits=bits)
    k, v = [randn(9 * block, kv, D, dtype=torch.float16, seed=s) for s in (1, 2)]
    cache.write(k, v, torch.arange(9 * block, dtype=torch.int32, device=DEV))
    q = randn(3, H, D, dtype=torch.float16, seed=3)
    op = tb.CacheAttention(block)
    lengths = torch.tensor([40, 64, 33], dtype=torch.int32, device=DEV)
    table = torch.tensor([[0, 1, 2, 3], [0, 1, 5, 6], [0, 1, 1, 0]], dtype=torch.int32, device=DEV)
    got = op(q, cache, table, lengths, scale=0.125)
    for b in range(3):
        assert torch.equal(op(q[b:b + 1], cache, table[b:b + 1], lengths[b:b + 1], scale=0.125)[0], got[b])
    one = table[:1].expand(3, 4)
    assert torch.equal(op(q, cache, one, lengths, scale=0.125), op(q, cache, one.contiguous(), lengths, scale=0.125))
    # a page that is there twice is the same as a copy of it
    cache.data[7] = cache.data[1]
    cache.data[8] = cache.data[0]
    copy = torch.tensor([[0, 1, 7, 8]], dtype=torch.int32, device=DEV)
    assert torch.equal(op(q[2:], cache, copy, lengths[2:], scale=0.125)[0], got[2])
    # lengths below nothing and past the table
    bad = torch.tensor([-3, 10 ** 6, 0], dtype=torch.int32, device=DEV)
    o = op(q, cache, table, bad, scale=0.125)
    assert not bool(o[0].any()) and not bool(o[2].any())
    assert torch.equal(o[1], op(q, cache, table, torch.full_like(lengths, 64), scale=0.125)[1])


def test_a_prompt_as_it_comes_out_of_a_projection():
    """k and v as views of one projection [tokens, 3, heads, dim], written to the cache and attended to without a copy's help."""
    T, heads, D, block = 50, 4, 64, 16
    qkv = randn(T, 3, heads, D, dtype=torch.bfloat16, seed=5)
    cache = tb.KeyValueCache(4, block, heads, D, bits=8)
    slots = torch.arange(T, dtype=torch.int32, device=DEV)
    cache.write(qkv[:, 1], qkv[:, 2], slots)
    other = tb.KeyValueCache(4, block, heads, D, bits=8)
    other.write(qkv[:, 1].contiguous(), qkv[:, 2].contiguous(), slots)
    assert torch.equal(cache.data, other.data)
    lay = torch.ones(heads, 4, 4)
    x = qkv.detach().clone().requires_grad_(True)
    q, k, v = [x[:, i].transpose(0, 1)[None] for i in range(3)]
    do = randn(1, heads, T, D, dtype=torch.bfloat16, seed=6)
    o = tb.Attention(lay, block)(q, k, v, scale=0.125, causal=True)
    o.backward(do)
    want = R.attention(q, k, v, lay, block, do, scale=0.125, causal=True)
    for i, n in enumerate(('dq', 'dk', 'dv')):
        R.check(x.grad[:, i].transpose(0, 1)[None], want[n], n)
