"""GPU: the quantised cache bit by bit against its definition in 64 bits, and attention over it against the same in 64 bits."""
import math

import pytest
import torch

import torch_blocksparse as tb
from helpers import random_layout

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def quantised(x, bits):
    """(values, codes) in 64 bits: the values that the cache holds for x [.., d]"""
    x = x.double().cpu().unflatten(-1, (-1, 32))
    bad = torch.isnan(x).any(-1, keepdim=True)
    x = x.clamp(-65504., 65504.)
    least = x.nan_to_num().amin(-1, keepdim=True).float().half().double()
    step = ((x.nan_to_num().amax(-1, keepdim=True) - least) / (2 ** bits - 1)).float().half().double()
    code = torch.where(step > 0, ((x - least) / torch.where(step > 0, step, 1.)).round().clamp(0, 2 ** bits - 1), 0.)
    return torch.where(bad, math.nan, least + code * step).flatten(-2), step.expand_as(x).flatten(-2), least.expand_as(x).flatten(-2)


def same(got, want, dtype):
    """the definition's value, rounded once to the type (least + code * step has 24 bits or fewer beyond fp32 only where least is far from step: rounded twice)"""
    once, twice = want.to(dtype), want.float().to(dtype)
    got = got.cpu()
    return bool(((got == once) | (got == twice) | (torch.isnan(got) & torch.isnan(once))).all())


def random_kv(T, heads, D, dtype, seed, spread=1.):
    g = torch.Generator().manual_seed(seed)
    return [(spread * torch.randn(T, heads, D, generator=g)).to(dtype).to(DEV) for _ in range(2)]


def slots_of(T, capacity, seed):
    return torch.randperm(capacity, generator=torch.Generator().manual_seed(seed))[:T].int().to(DEV)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('bits,D,heads,block', [(4, 64, 1, 16), (4, 128, 3, 64), (8, 64, 5, 32), (8, 128, 2, 128)])
@pytest.mark.parametrize('T', [1, 7, 300, 1500])
def test_written_and_read_back(dtype, bits, D, heads, block, T):
    cache = tb.KeyValueCache(1600 // block + 3, block, heads, D, bits=bits)
    k, v = random_kv(T, heads, D, dtype, T, 3.)
    slots = slots_of(T, cache.pages * block, T + 1)
    before = cache.data.clone()
    cache.write(k, v, slots)
    for got, x in zip(cache.read(slots, dtype), (k, v)):
        assert same(got, quantised(x, bits)[0], dtype)
    # what was not written is as it was
    rest = torch.ones(cache.pages * block, dtype=torch.bool, device=DEV)
    rest[slots.long()] = False
    others = torch.nonzero(rest)[:, 0].int()
    assert not any(bool(t.any()) for t in cache.read(others, dtype)) and bool((before == 0).all())
    assert not bool(cache._owner.any())
    # all types read the same numbers
    for other in (torch.float16, torch.bfloat16, torch.float32):
        for got, x in zip(cache.read(slots, other), (k, v)):
            assert same(got, quantised(x, bits)[0], other)


@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
def test_groups_of_all_kinds(bits, dtype):
    D, most = 64, 2 ** bits - 1
    g = torch.Generator().manual_seed(1)
    rows = [torch.zeros(D), torch.full((D,), 3.), torch.full((D,), -65504.), torch.linspace(-1, 1, D), torch.randn(D, generator=g) * 1e-6, torch.randn(D, generator=g) * 1e4]
    # exact middles between two codes: least 0, step 1, and least -8, step 1 / 4
    ties = (torch.arange(D) % (2 * most)).float() / 2
    ties[::32], ties[31::32] = 0., float(most)
    rows += [ties, ties / 4 - 8]
    # a least value far from the rest, neighbours of middles
    far = torch.rand(D, generator=g)
    far[5], far[40] = -65504., 65504.
    rows += [far, (ties * (1 + 2. ** -7)).clamp(max=float(most)), ties + (torch.rand(D, generator=g) - 0.5) * 2. ** -9]
    # infinities and NaN: taken into fp16's range, and the group's
    inf = torch.randn(D, generator=g)
    inf[3], inf[50] = math.inf, -math.inf
    nan = torch.randn(D, generator=g)
    nan[7] = math.nan
    both = inf.clone()
    both[4] = math.nan
    rows += [inf, nan, both, torch.full((D,), math.nan)]
    if dtype != torch.float16:
        rows += [torch.randn(D, generator=g) * 1e30, torch.randn(D, generator=g) * 1e-30]
    if dtype == torch.float32:
        rows += [torch.randn(D, generator=g) * 1e-44]
    x = torch.stack(rows)[:, None].to(dtype).to(DEV)
    cache = tb.KeyValueCache(3, 16, 1, D, bits=bits)
    slots = torch.arange(x.size(0), dtype=torch.int32, device=DEV)
    cache.write(x, x.flip(0), slots)
    k, v = cache.read(slots, torch.float32)
    assert same(k, quantised(x, bits)[0], torch.float32)
    assert same(v, quantised(x.flip(0), bits)[0], torch.float32)


@pytest.mark.parametrize('bits', [4, 8])
def test_codes_are_those_of_exact_arithmetic(bits):
    # many values, and of those as many as can be close to the middle of two codes
    D, T = 128, 4000
    g = torch.Generator().manual_seed(2)
    k = torch.randn(T, 2, D, generator=g, dtype=torch.float64)
    _, step, least = quantised(k.half(), bits)
    near = least + step * ((k - least) / step).floor() + step * 0.5 * (1 + (torch.rand(k.shape, generator=g) - 0.5) * 2. ** -18)
    inside = (torch.rand(k.shape, generator=g) < 0.5) & (near < k.unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2))
    k = torch.where(inside, near, k).float().to(DEV)
    cache = tb.KeyValueCache(250, 16, 2, D, bits=bits)
    slots = torch.arange(T, dtype=torch.int32, device=DEV)
    cache.write(k, k, slots)
    got = cache.read(slots, torch.float32)[0]
    assert same(got, quantised(k, bits)[0], torch.float32)


@pytest.mark.parametrize('T', [2, 40, 512, 513, 3000])
def test_the_last_of_a_slot_is_written(T):
    cache = tb.KeyValueCache(20, 16, 2, 64, bits=8)
    k, v = random_kv(T, 2, 64, torch.float16, 5)
    slots = torch.randint(-3, min(320, T), (T,), generator=torch.Generator().manual_seed(T)).int().to(DEV)
    slots[T // 2] = 320                                      # one past the cache
    for _ in range(3):
        cache.write(k, v, slots)
        last = {s: t for t, s in enumerate(slots.tolist())}
        at = [s for s in last if 0 <= s < 320]
        if not at:
            continue
        got = cache.read(torch.tensor(at, dtype=torch.int32, device=DEV))
        rows = [last[s] for s in at]
        for x, y in zip(got, (k, v)):
            assert same(x, quantised(y[rows], 8)[0], torch.float16)
        assert not bool(cache._owner.any())
        k, v = k.flip(0), v.flip(0)
    outside = cache.read(torch.tensor([-1, 320, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV))
    assert not any(bool(t.any()) for t in outside)


def test_views_empty_calls_and_pages_beside():
    cache = tb.KeyValueCache(4, 32, 2, 64, bits=4)
    qkv = torch.randn(50, 6, 64, device=DEV, dtype=torch.bfloat16)       # a packed projection
    k, v = qkv[:, 2:4], qkv[:, 4:]
    slots = slots_of(50, 128, 3)
    cache.write(k, v, slots)
    odd = torch.empty(50 * 128 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(50, 2, 64).copy_(k)
    other = tb.KeyValueCache(4, 32, 2, 64, bits=4)
    other.write(odd, v.transpose(0, 1).contiguous().transpose(0, 1), slots[:, None].expand(-1, 2).contiguous()[:, 0])
    assert torch.equal(cache.data, other.data)
    cache.write(k[:0], v[:0], slots[:0])
    assert [t.shape for t in cache.read(slots[:0])] == [(0, 2, 64)] * 2
    cache.write(k, v, torch.full_like(slots, -1))
    assert torch.equal(cache.data, other.data)


# ---- attention -------------------------------------------------------------------------------------------------------------------------


def oracle(q, k, v, least, step, bits, lengths, layout, block, scale, softcap, slopes, held):
    """(o, bound) in 64 bits.  k, v, least, step [B, positions, kv heads, D]: the cache's values and, of the keys, the group's numbers.  Bound, with u half a step of
    the result's type: scores are sums in fp32 of least * q and step * code * q: c = 2^-24 (2 D + n + 8 max terms + 32) of a share; shares and values
    are rounded to fp16 for the second product (2^-11 of themselves each, not below 2^-25; the largest share is 1); the result once more."""
    u = torch.finfo(q.dtype).eps / 2
    q = q.double().cpu()
    B, H, D = q.shape
    G = H // k.size(2)
    out, bound = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    for b, n in enumerate(lengths.tolist()):
        n = min(n, held.size(1), layout.size(1) * block if layout is not None else n)
        if n <= 0:
            continue
        j = torch.arange(n)
        for h in range(H):
            seen = held[b, :n].clone()
            if layout is not None:
                seen &= (layout[h, (n - 1) // block] != 0).repeat_interleave(block)[:n]
            if not bool(seen.any()):
                continue
            kb, vb = k[b, :n, h // G], v[b, :n, h // G]
            y = scale * (kb @ q[b, h])
            terms = abs(scale) * ((least[b, :n, h // G].abs() + (2 ** bits - 1) * step[b, :n, h // G]) @ q[b, h].abs())
            if softcap:
                y = softcap * torch.tanh(y / softcap)
            if slopes is not None:
                far = float(slopes[h]) * (n - 1 - j)
                y, terms = y - far, terms + abs(far)
            p = torch.softmax(y.masked_fill(~seen, -math.inf), 0)
            vb = torch.where(seen[:, None], vb, 0.)
            out[b, h] = p @ vb
            c = 2. ** -24 * (2 * D + n + 8 * (float(terms[seen].max()) + softcap) + 32)
            bound[b, h] = u * out[b, h].abs() + (2. ** -10 + c) * (p @ vb.abs()) + 2. ** -25 * (1 + seen.double() @ vb.abs())
    return out, bound


def filled(B, H, kv, D, block, bits, width, dtype, seed, spare=3):
    """a cache whose every position is written, a table of pages in no order, and the keys and values by position"""
    g = torch.Generator().manual_seed(seed)
    cache = tb.KeyValueCache(B * width + spare, block, kv, D, bits=bits)
    k, v = random_kv(cache.pages * block, kv, D, dtype, seed, 1.5)
    cache.write(k, v, torch.arange(cache.pages * block, dtype=torch.int32, device=DEV))
    table = torch.randperm(cache.pages, generator=g)[:B * width].int().view(B, width)
    at = (table.long()[:, :, None] * block + torch.arange(block)).flatten(1)
    (kq, step, least), (vq, _, _) = quantised(k, bits), quantised(v, bits)
    q = (2 * torch.randn(B, H, D, generator=g)).to(dtype).to(DEV)
    return cache, q, table.to(DEV), [t[at] for t in (kq, vq, least, step)]


def check(got, want, what):
    out, bound = want
    err = (got.double().cpu() - out).abs()
    assert bool((err <= bound).all()), '%s: worst %g of the bound' % (what, float((err / bound.clamp(min=1e-300)).max()))
    return float((err / bound.clamp(min=1e-300)).max())


@pytest.mark.parametrize('bits,D', [(4, 64), (4, 128), (8, 64), (8, 128)])
@pytest.mark.parametrize('H,kv', [(2, 2), (8, 2), (7, 1), (16, 1), (40, 2)])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
def test_decoding(bits, D, H, kv, dtype):
    B, block, width = 5, 32, 9
    cache, q, table, held = filled(B, H, kv, D, block, bits, width, dtype, H + D)
    lengths = torch.tensor([1, 288, 33, 0, 170], dtype=torch.int32, device=DEV)
    slopes = torch.tensor([2. ** (-8. * (h + 1) / H) for h in range(H)], device=DEV)
    lay = random_layout((H, width, width), 0.5, 3)
    everything = torch.ones(B, width * block, dtype=torch.bool)
    for rules in (dict(), dict(softcap=8.), dict(slopes=slopes), dict(softcap=15., slopes=slopes, layout=lay), dict(layout=lay)):
        layout = rules.pop('layout', None)
        o = tb.CacheAttention(block, layout)(q, cache, table, lengths, scale=D ** -0.5, **rules)
        want = oracle(q, *held[:2], held[2], held[3], bits, lengths, layout, block, D ** -0.5, rules.get('softcap', 0.), rules.get('slopes'), everything)
        print(sorted(rules), layout is not None, 'worst share of the bound: %.2f' % check(o, want, str(rules)))
        assert not bool(o[3].any())


@pytest.mark.parametrize('block', [16, 32, 64, 128])
@pytest.mark.parametrize('bits', [4, 8])
def test_blocks_lengths_and_pages_that_are_not_held(block, bits):
    B, H, kv, D = 12, 4, 2, 64
    width = max(2, 260 // block)
    cache, q, table, held = filled(B, H, kv, D, block, bits, width, torch.float16, block)
    lengths = torch.tensor([1, 2, 15, 16, 17, 31, 32, 33, width * block - 1, width * block, width * block + 50, -4], dtype=torch.int32, device=DEV)
    lay = random_layout((H, width, width), 0.6, 9)
    lay[1] = 0                                                # a head that sees nothing
    gone = torch.rand(B, width, generator=torch.Generator().manual_seed(1)) < 0.3
    missing = torch.where(gone, torch.randint(0, 3, (B, width)) * 0 - 1, 0).int().to(DEV)
    holes = torch.where(missing < 0, missing, table)
    holes[0, 1:] = 2 ** 31 - 1                                # (no position there is asked for)
    holes[5, -1] = cache.pages                                # one past the cache
    for t, layout in ((table, None), (table, lay), (holes, None), (holes, lay)):
        there = ((t >= 0) & (t < cache.pages)).cpu().repeat_interleave(block, 1)
        o = tb.CacheAttention(block, layout)(q, cache, t, lengths, scale=0.3, softcap=20.)
        check(o, oracle(q, *held[:2], held[2], held[3], bits, lengths, layout, block, 0.3, 20., None, there), 'block %d' % block)
        assert layout is None or not bool(o[:, 1].any())


def test_long_sequences_are_split():
    B, H, kv, D, block = 2, 4, 1, 128, 64
    width = 160
    cache, q, table, held = filled(B, H, kv, D, block, 4, width, torch.bfloat16, 7)
    lengths = torch.tensor([width * block - 3, 100], dtype=torch.int32, device=DEV)
    from torch_blocksparse import _lib
    assert _lib.load().bsp_cache_attention_splits(B, H, kv, block, width) > 1
    everything = torch.ones(B, width * block, dtype=torch.bool)
    lay = torch.zeros(H, width, width, dtype=torch.int64)
    lay[:, :, ::3] = 1
    lay[2, :, 5] = 1
    for layout in (None, lay):
        o = tb.CacheAttention(block, layout)(q, cache, table, lengths, scale=D ** -0.5)
        check(o, oracle(q, *held[:2], held[2], held[3], 4, lengths, layout, block, D ** -0.5, 0., None, everything), 'long')
        assert torch.equal(o, tb.CacheAttention(block, layout)(q, cache, table, lengths, scale=D ** -0.5))


def test_what_lies_behind_the_end_reaches_nothing():
    B, H, kv, D, block, width = 2, 2, 2, 64, 32, 4
    cache, q, table, held = filled(B, H, kv, D, block, 8, width, torch.float16, 8)
    lengths = torch.tensor([70, 97], dtype=torch.int32, device=DEV)
    op = tb.CacheAttention(block)
    want = op(q, cache, table, lengths, scale=0.125)
    at = (table.long()[:, :, None] * block + torch.arange(block, device=DEV)).flatten(1)
    behind = torch.cat([at[b, n:] for b, n in enumerate(lengths.tolist())]).int()
    x = torch.full((behind.numel(), kv, D), math.nan, dtype=torch.float16, device=DEV)
    cache.write(x, x, behind)
    assert torch.equal(op(q, cache, table, lengths, scale=0.125), want)
    # ... a NaN that is seen comes out
    cache.write(x[:1], x[:1], at[1, 5:6].int())
    o = op(q, cache, table, lengths, scale=0.125)
    assert torch.equal(o[0], want[0]) and bool(torch.isnan(o[1]).all())


def test_queries_of_all_sizes_and_strides():
    B, H, kv, D, block, width = 3, 4, 4, 64, 16, 5
    cache, q, table, held = filled(B, H, kv, D, block, 8, width, torch.bfloat16, 9)
    lengths = torch.tensor([80, 41, 7], dtype=torch.int32, device=DEV)
    op = tb.CacheAttention(block)
    everything = torch.ones(B, width * block, dtype=torch.bool)
    for size, scale in ((1e30, 1e-30), (1e-30, 1e30), (0., 1.), (1e-38, 1.)):
        x = (q.float() * size).bfloat16()
        check(op(x, cache, table, lengths, scale=scale), oracle(x, *held[:2], held[2], held[3], 8, lengths, None, block, scale, 0., None, everything), str(size))
    want = op(q, cache, table, lengths)
    wide = torch.empty(B, H, D + 2, dtype=q.dtype, device=DEV)[..., :D].copy_(q)
    packed = torch.empty(B, 3 * H, D, dtype=q.dtype, device=DEV)
    packed[:, :H] = q
    for view in (wide, packed[:, :H], q.transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(op(view, cache, table.t().contiguous().t(), lengths), want)
    assert op(q[:0], cache, table[:0], lengths[:0]).shape == (0, H, D)


def test_a_prompt_then_tokens_one_by_one():
    """As a program answers: the prompt through Attention, its keys and values to the cache, then position after position."""
    B, H, kv, D, block, L, prompt, bits = 2, 4, 2, 64, 16, 75, 60, 8
    blocks = -(-L // block)
    lay = tb.fixed_layout(H, 6, 'fixed', 2, 'unidirectional', 1, 1)[:, :blocks, :blocks].contiguous()
    g = torch.Generator().manual_seed(3)
    q, k, v = [torch.randn(B, h, L, D, generator=g).half().to(DEV) for h in (H, kv, kv)]
    slopes = torch.tensor([0.5, 0.1, 0.02, 0.], device=DEV)
    rules = dict(scale=D ** -0.5, softcap=10., slopes=slopes)
    cache = tb.KeyValueCache(B * blocks, block, kv, D, bits=bits)
    table = torch.randperm(B * blocks, generator=g).int().view(B, blocks).to(DEV)
    pos = torch.arange(L, device=DEV)
    slots = table[:, pos // block] * block + pos % block                        # [B, L]
    cache.write(k[:, :, :prompt].transpose(1, 2).flatten(0, 1), v[:, :, :prompt].transpose(1, 2).flatten(0, 1), slots[:, :prompt].flatten().int())
    decode = tb.CacheAttention(block, lay)
    steps = []
    for t in range(prompt, L):
        cache.write(k[:, :, t], v[:, :, t], slots[:, t].int().contiguous())
        steps.append(decode(q[:, :, t], cache, table, torch.full((B,), t + 1, dtype=torch.int32, device=DEV), **rules))
    kc, vc = [x.view(B, L, kv, D).transpose(1, 2) for x in cache.read(slots.flatten().int(), torch.float32)]
    whole = tb.Attention(lay, block)(q.float(), kc, vc, causal=True, **rules)
    got = torch.stack(steps, 2).float()
    # fp16: result, share and value rounded (2^-11 each) of values up to 5
    assert float((got - whole[:, :, prompt:]).abs().max()) <= 3 * 2. ** -11 * float(vc.abs().max())


def test_captured_and_replayed():
    B, H, kv, D, block, width = 3, 4, 2, 64, 32, 40
    cache, q, table, _ = filled(B, H, kv, D, block, 4, width, torch.float16, 10)
    lay = random_layout((H, width, width), 0.5, 3)
    op = tb.CacheAttention(block, lay)
    lengths = torch.tensor([1200, 5, 640], dtype=torch.int32, device=DEV)
    k, v = random_kv(700, kv, D, torch.float16, 3)
    slots = slots_of(700, cache.pages * block, 4)
    big = tb.CacheAttention(block)

    def step():
        cache.write(k, v, slots)
        return op(q, cache, table, lengths, scale=0.125), big(q, cache, table, lengths, scale=0.125)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2, 3):
        for x, y in zip((k, v), random_kv(700, kv, D, torch.float16, seed + 20)):
            x.copy_(y)
        slots.copy_(slots_of(700, cache.pages * block, seed + 30))
        slots[100:110] = slots[99]
        lengths.copy_(torch.randint(0, 1280, (B,), generator=torch.Generator().manual_seed(seed)).int())
        eager = step()
        torch.cuda.synchronize()
        cache.data.random_(0, 16)                             # (small codes; the replay writes its positions again)
        kept = cache.data.clone()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in out]
        cache.data.copy_(kept)
        eager = step()
        for a, b in zip(replayed, eager):
            assert torch.equal(a, b)
        assert not bool(cache._owner.any())


def test_a_cache_past_four_gigabytes():
    # page numbers whose bytes lie past 32 bits
    block, kv, D = 128, 8, 128
    pages = 2 ** 32 // (2 * block * kv * (D + D // 8)) + 40
    cache = tb.KeyValueCache(pages, block, kv, D, bits=8)
    assert cache.data.numel() > 2 ** 32
    k, v = random_kv(block, kv, D, torch.float16, 1)
    first = (pages - 2) * block
    cache.write(k, v, torch.arange(first, first + block, dtype=torch.int32, device=DEV))
    got = cache.read(torch.arange(first, first + block, dtype=torch.int32, device=DEV))
    for x, y in zip(got, (k, v)):
        assert same(x, quantised(y, 8)[0], torch.float16)
    small = tb.KeyValueCache(1, block, kv, D, bits=8)
    small.data.copy_(cache.data[pages - 2:pages - 1])
    q = torch.randn(1, 16, D, device=DEV).half()
    op, n = tb.CacheAttention(block), torch.tensor([block], dtype=torch.int32, device=DEV)
    at = lambda p: torch.tensor([[p]], dtype=torch.int32, device=DEV)    # noqa: E731
    assert torch.equal(op(q, cache, at(pages - 2), n), op(q, small, at(0), n))
    assert not bool(cache.data[:pages - 2].any()) and not bool(cache.data[pages - 1].any())
