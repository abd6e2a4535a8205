"""GPU: the operators that SparseSelfAttention keeps: a captured chain outlives what other calls make, and tables of dropped operators are not given away
while a stream reads them."""
import collections
import gc

import pytest
import torch

import torch_blocksparse as tb
from torch_blocksparse import _lib

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.mark.parametrize('dtype,masked', [(torch.float16, False), (torch.float16, True), (torch.float32, False)])
def test_a_captured_chain_outlives_the_operators_of_decoding_and_of_other_lengths(dtype, masked):
    cls = tb.DeepSpeedSparseSelfAttention
    B, H, L, D, block = 2, 2, 128, 64, 16
    mod = tb.SparseSelfAttention(tb.SparsityConfig(block=block, stride=32, numverts=2))
    g = torch.Generator().manual_seed(4)
    static = [torch.randn(B, H, L, D, generator=g).to(dtype).to(DEV) for _ in range(4)]
    mask = torch.ones(L, L, dtype=dtype, device=DEV).tril() if masked else None

    def step():
        leaves = [t.detach().clone().requires_grad_(True) for t in static[:3]]
        o = mod(*leaves, attn_mask=mask)
        return (o.detach(),) + torch.autograd.grad(o, leaves, static[3])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    kept = mod.get_ops(H, L, static[0].device)
    cache = tb.KeyValueCache(2 * cls.OPS_CACHE_SIZE, block, H, D)
    q, lengths = torch.zeros(1, H, D, dtype=torch.float16, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    for n in range(1, cls.OPS_CACHE_SIZE + 2):
        mod.decode(q, cache, torch.zeros(1, n, dtype=torch.int32, device=DEV), lengths)
        y = torch.zeros(1, H, L + 32 * n, D, dtype=dtype, device=DEV)
        mod(y, y, y)
    assert mod.get_ops(H, L, static[0].device) is kept
    filler = [torch.full((1 << 14,), 1, dtype=torch.int32, device=DEV) for _ in range(64)]   # (what a dropped table's memory would be given to)
    for seed in (5, 6, 7):
        g.manual_seed(seed)
        for t in static:
            t.copy_(torch.randn(t.shape, generator=g))
        eager = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)
    del filler


def round_up(n):
    return -(-n // 512) * 512                            # (the allocator's unit)


@pytest.mark.parametrize('block', [16, 32, 64])
def test_all_that_a_chain_holds_on_the_gpu_is_found(block, monkeypatch):
    """What stays allocated when a chain was used in all ways is what a drop tells of the streams."""
    monkeypatch.setattr(tb.DeepSpeedSparseSelfAttention, 'ops', collections.OrderedDict())    # (no operator of another test is dropped meanwhile)
    mod = tb.SparseSelfAttention(tb.SparsityConfig(block=block, stride=2 * block, numverts=2))
    B, H, L, D = 2, 4, 8 * block, 64
    x = {t: torch.randn(B, H, L, D, device=DEV).to(t) for t in (torch.float16, torch.bfloat16, torch.float32)}
    mask = {t: torch.ones(L, L, dtype=t, device=DEV) for t in x}

    def use(length):
        for t in x:
            for attn_mask in (None, mask[t][:length, :length].contiguous()):
                leaves = [x[t][:, :, :length].contiguous().requires_grad_(True) for _ in range(3)]
                mod(*leaves, attn_mask=attn_mask).sum().backward()

    use(4 * block)                                       # (what the libraries keep for themselves)
    torch.cuda.synchronize()
    gc.collect()
    before = torch.cuda.memory_allocated()
    use(8 * block)
    torch.cuda.synchronize()
    gc.collect()
    held = torch.cuda.memory_allocated() - before
    found = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in _lib.tensors_of(mod.get_ops(H, L, x[torch.float16].device)) if t.is_cuda}
    assert held == sum(round_up(n) for n in found.values()) > 0


def busy_stream(seconds=2.):
    """a stream with work of that length under way"""
    start, stop = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    start.record()
    torch.cuda._sleep(1 << 22)                           # (of a clock that differs between cards)
    stop.record()
    stop.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(int((1 << 22) * 1e3 * seconds / start.elapsed_time(stop)))
    return stream


def addresses(tensors):
    return [(t.untyped_storage().data_ptr(), t.untyped_storage().data_ptr() + t.untyped_storage().nbytes()) for t in tensors if t.is_cuda]


def test_tables_are_not_given_away_while_another_stream_reads_them():
    """Operators made on one stream, in use on another one when they are dropped: their memory stays theirs until that is done."""
    cls = tb.DeepSpeedSparseSelfAttention
    B, H, D, block, L = 2, 2, 64, 16, 256
    mod = tb.SparseSelfAttention(tb.SparsityConfig(block=block, stride=32))
    q, k, v = [torch.randn(B, H, L, D, device=DEV).half() for _ in range(3)]
    lay = tb.fixed_layout(H, L // block, 'fixed', 2, 'unidirectional', 1, 1)
    cache = tb.KeyValueCache(2 * L // block, block, H, D)
    cache.write(k.transpose(1, 2).flatten(0, 1), v.transpose(1, 2).flatten(0, 1), torch.arange(B * L, dtype=torch.int32, device=DEV))
    table, lengths = torch.arange(2 * L // block, dtype=torch.int32, device=DEV).view(B, -1), torch.full((B,), L, dtype=torch.int32, device=DEV)
    ops = dict(rules=tb.Attention(lay, block), decode=tb.CacheAttention(block, lay))
    work = dict(chain=lambda: mod(q, k, v), rules=lambda: ops['rules'](q, k, v, causal=True), decode=lambda: ops['decode'](q[:, :, -1].contiguous(), cache, table, lengths))
    want = {n: w() for n, w in work.items()}
    torch.cuda.synchronize()
    for name in work:
        held = _lib.tensors_of(mod.get_ops(H, L, q.device) if name == 'chain' else ops[name])
        places = addresses(held)
        sizes = sorted({b - a for a, b in places})
        assert places
        del held
        stream = busy_stream()
        with torch.cuda.stream(stream):
            got = work[name]()                           # behind the sleep
        if name == 'chain':
            for n in range(1, cls.OPS_CACHE_SIZE + 1):
                mod.get_ops(H, L + 32 * n, q.device)
        else:
            del ops[name]
        gc.collect()
        fresh = [torch.empty(n, dtype=torch.uint8, device=DEV) for _ in range(20) for n in sizes]
        new = addresses(fresh)
        assert not stream.query()                        # (still under way)
        assert not any(a < d and c < b for a, b in places for c, d in new), name
        stream.synchronize()
        assert torch.equal(got, want[name])


@pytest.mark.parametrize('mode,attention', [('fixed', 'unidirectional'), ('fixed', 'bidirectional'), ('dense', 'unidirectional')])
@pytest.mark.parametrize('width', [1, 3, 16, 17, 39, 130])
def test_decoding_over_tables_of_all_widths(mode, attention, width):
    """The same as CacheAttention over the layout of exactly so many blocks: for one direction bit by bit, and where later blocks count as
    work (that nobody sees) up to the order of sums: 2^-10 of a value for each of the two."""
    B, H, kv, D, block = 3, 4, 2, 64, 16
    mod = tb.SparseSelfAttention(tb.SparsityConfig(mode, block, 64, attention, numverts=2))
    g = torch.Generator().manual_seed(width)
    cache = tb.KeyValueCache(B * width, block, kv, D, bits=8)
    k, v = [torch.randn(B * width * block, kv, D, generator=g).half().to(DEV) for _ in range(2)]
    cache.write(k, v, torch.arange(B * width * block, dtype=torch.int32, device=DEV))
    table = torch.randperm(B * width, generator=g).int().view(B, width).to(DEV)
    q = torch.randn(B, H, D, generator=g).half().to(DEV)
    lengths = torch.tensor([width * block, 1 + width * block // 2, width * block + 99], dtype=torch.int32, device=DEV)
    lay = None if mode == 'dense' else tb.fixed_layout(H, -(-width // 4) * 4, mode, 4, attention, 2, 1)[:, :width, :width]
    want = tb.CacheAttention(block, lay)(q, cache, table, lengths, scale=D ** -0.5, softcap=9.)
    got = mod.decode(q, cache, table, lengths, softcap=9.)
    if attention == 'unidirectional':
        assert torch.equal(got, want)
    else:
        assert float((got.float() - want.float()).abs().max()) <= 2 * 2. ** -10 * float(v.abs().max())


def test_a_cache_is_not_given_away_while_another_stream_writes_it():
    H, D, block, pages = 2, 64, 16, 64
    T = pages * block
    k, v = [torch.randn(T, H, D, device=DEV).half() for _ in range(2)]
    slots = torch.arange(T, dtype=torch.int32, device=DEV)
    cache = tb.KeyValueCache(pages, block, H, D, bits=8)
    cache.write(k, v, slots)
    want = cache.read(slots)
    places = addresses([cache.data, cache._owner])
    torch.cuda.synchronize()
    stream = busy_stream()
    with torch.cuda.stream(stream):
        cache.write(v, k, slots)
        got = cache.read(slots)
    del cache
    gc.collect()
    fresh = [torch.empty(b - a, dtype=torch.uint8, device=DEV) for _ in range(20) for a, b in places]
    new = addresses(fresh)
    assert not stream.query()
    assert not any(a < d and c < b for a, b in places for c, d in new)
    stream.synchronize()
    assert torch.equal(got[0], want[1]) and torch.equal(got[1], want[0])
