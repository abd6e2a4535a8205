"""GPU: the cache of latent vectors element by element, and attention over it against 64 bits."""
import math

import pytest
import torch

import latent_oracle as O
import rotation_oracle as R
import torch_blocksparse as tb
from helpers import random_layout
from torch_blocksparse import _lib

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def randn(shape, dtype, seed, scale=1.):
    return (scale * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dtype).to(DEV)


def order(n, seed):
    return torch.randperm(n, generator=torch.Generator().manual_seed(seed)).int()


# ---- the cache ------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('latent,block', [(128, 16), (256, 128), (512, 64)])
@pytest.mark.parametrize('T', [1, 7, 8, 300, 700])
def test_written_and_read_back(dtype, latent, block, T):
    cache = tb.LatentCache(1024 // block, block, latent, dtype=dtype)
    cache.data.fill_(math.nan)
    c, r, slots = randn((T, latent), dtype, 1), randn((T, 64), dtype, 2), order(1024, 3)[:T].to(DEV)
    cache.write(c, r, slots)
    got = cache.read(slots)
    assert torch.equal(got[0], c) and torch.equal(got[1], r)
    rows = cache.data.view(1024, latent + 64)
    assert torch.equal(rows[slots.long()], torch.cat([c, r], 1))
    rest = torch.ones(1024, dtype=torch.bool, device=DEV)
    rest[slots.long()] = False
    assert bool(torch.isnan(rows[rest]).all()) and not bool(cache._owner.any())
    outside = cache.read(torch.tensor([-1, 1024, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV))
    assert not any(bool(t.any()) for t in outside)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('neighbours', [False, True])
@pytest.mark.parametrize('T,pairs', [(1, 32), (13, 24), (40, 8), (600, 32)])
def test_written_rotated(dtype, neighbours, T, pairs):
    f = [10000. ** (-p / pairs) for p in range(pairs)]
    cache = tb.LatentCache(20, 32, 128, dtype=dtype)
    c, r, slots = randn((T, 128), dtype, 1), randn((T, 64), dtype, 2, 2.), order(640, 3)[:T].to(DEV)
    positions = torch.randint(0, 131072, (T,), generator=torch.Generator().manual_seed(5)).int()
    rotation = tb.Rotation(f, neighbours=neighbours)
    cache.write(c, r, slots, rotation=rotation, positions=positions.to(DEV))
    got = cache.read(slots)
    assert torch.equal(got[0], c)
    R.check(got[1], R.turned(r, R.angles(positions, f), neighbours), 'r')
    assert torch.equal(got[1], rotation(r[:, None], positions=positions.to(DEV))[:, 0])     # the same numbers as ahead of the call


@pytest.mark.parametrize('T', [2, 40, 512, 513, 3000])
def test_the_last_of_a_slot_is_written(T):
    cache = tb.LatentCache(20, 16, 128)
    c, r = randn((T, 128), torch.bfloat16, 1), randn((T, 64), torch.bfloat16, 2)
    slots = torch.randint(-3, min(320, T), (T,), generator=torch.Generator().manual_seed(T)).int()
    slots[T // 2] = 320                                      # one past the cache
    for _ in range(3):
        cache.write(c, r, slots.to(DEV))
        last = {s: t for t, s in enumerate(slots.tolist()) if 0 <= s < 320}
        if last:
            got = cache.read(torch.tensor(list(last), dtype=torch.int32, device=DEV))
            rows = list(last.values())
            assert torch.equal(got[0], c[rows]) and torch.equal(got[1], r[rows])
        assert not bool(cache._owner.any())
        c, r = c.flip(0), r.flip(0)


def test_views_and_empty_writes():
    cache, other = tb.LatentCache(4, 32, 128), tb.LatentCache(4, 32, 128)
    both = randn((50, 192), torch.bfloat16, 1)               # one projection gives both
    slots = order(128, 3)[:50].to(DEV)
    cache.write(both[:, :128], both[:, 128:], slots)
    odd = torch.empty(50 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(50, 64).copy_(both[:, 128:])
    other.write(both[:, :128].T.contiguous().T, odd, slots.repeat_interleave(2)[::2])
    assert torch.equal(cache.data, other.data)
    cache.write(both[:0, :128], both[:0, 128:], slots[:0])
    assert [tuple(t.shape) for t in cache.read(slots[:0])] == [(0, 128), (0, 64)]
    one = both[:1, :128].expand(50, 128)
    cache.write(one, both[:1, 128:].expand(50, 64), slots)
    assert torch.equal(cache.read(slots)[0], one)


# ---- attention ------------------------------------------------------------------------------------------------------------------------


def setting(dtype, B, H, latent, block, lengths, seed=0, width=None, spare=3):
    """a cache whose rows that no sequence holds are NaN, and what a call takes"""
    lengths = torch.tensor(lengths, dtype=torch.int32)
    width = width or max(1, -(-int(lengths.max()) // block))
    need = [-(-int(n) // block) for n in lengths.clamp(min=0, max=width * block)]
    cache = tb.LatentCache(sum(need) + spare, block, latent, dtype=dtype)
    cache.data.fill_(math.nan)
    pages, table, at = order(cache.pages, seed), torch.full((B, width), -1, dtype=torch.int32), 0
    rows = cache.data.view(-1, latent + 64)
    for b in range(B):
        table[b, :need[b]] = pages[at:at + need[b]]
        at += need[b]
    for b in range(B):
        n = min(max(int(lengths[b]), 0), width * block)
        where = (table[b].long().repeat_interleave(block) * block + torch.arange(width * block) % block)[:n].to(DEV)
        rows[where] = randn((n, latent + 64), dtype, seed + 10 + b)
    return cache, randn((B, H, latent), dtype, seed + 1), randn((B, H, 64), dtype, seed + 2), table.to(DEV), lengths.to(DEV)


def expected(cache, q, q_r, table, lengths, **options):
    rows = cache.data.view(-1, cache.latent + 64)
    return O.attention(q, q_r, rows[:, :cache.latent], rows[:, cache.latent:], table, lengths, cache.block, **options)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('latent', [128, 256, 512])
@pytest.mark.parametrize('H,block', [(1, 16), (5, 64), (16, 128), (17, 32), (32, 16), (33, 64), (64, 128), (65, 16), (128, 64)])
def test_lengths(dtype, latent, H, block):
    lengths = [1, 0, 15, 16, 17, 63, 64, 65, 128, 200, 1000, -3]
    cache, q, q_r, table, lengths = setting(dtype, len(lengths), H, latent, block, lengths, H)
    op, scale = tb.LatentAttention(block), latent ** -0.5
    o = op(q, q_r, cache, table, lengths, scale=scale)
    O.check(o, expected(cache, q, q_r, table, lengths, scale=scale), 'o')
    assert not bool(o[1].any()) and not bool(o[-1].any())
    assert torch.equal(o, op(q, q_r, cache, table, lengths, scale=scale))


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('H,latent', [(16, 512), (64, 512), (7, 128)])
def test_one_long_sequence(dtype, H, latent):
    cache, q, q_r, table, lengths = setting(dtype, 1, H, latent, 64, [20011], 3)
    o = tb.LatentAttention(64)(q, q_r, cache, table, lengths, scale=0.05)
    O.check(o, expected(cache, q, q_r, table, lengths, scale=0.05), 'o')


@pytest.mark.parametrize('H,B,longest', [(65, 300, 150), (16, 700, 150), (40, 259, 900), (9, 270, 1500)])
def test_many_sequences(H, B, longest):
    """more of them than a workgroup looks at together"""
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, longest, (B,), generator=g).tolist()
    lengths[B // 2] = 3000
    cache, q, q_r, table, lengths = setting(torch.bfloat16, B, H, 128, 16, lengths, 5)
    o = tb.LatentAttention(16)(q, q_r, cache, table, lengths, scale=0.08)
    O.check(o, expected(cache, q, q_r, table, lengths, scale=0.08), 'o')


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('H,block', [(3, 16), (20, 32), (48, 64), (70, 128)])
def test_layouts_caps_slopes_and_pages_not_held(dtype, H, block):
    blocks = 9
    layout = random_layout((H, blocks, blocks), 0.4, H)
    layout[0], layout[-1, 5] = 0, 0                            # a head that sees nothing, a row of another
    lengths = [1, block, 3 * block + 1, blocks * block, blocks * block - 5, 6 * block, 2 * block + 7, blocks * block + 100]
    cache, q, q_r, table, lengths = setting(dtype, len(lengths), H, 256, block, lengths, H, width=blocks)
    table[3, 4] = -1
    table[4, ::2] = cache.pages
    table[5] = -7
    slopes = torch.tensor([2. ** (-4. * (h + 1) / H) for h in range(H)], device=DEV)
    for options in (dict(), dict(softcap=3.), dict(slopes=slopes), dict(softcap=20., slopes=slopes)):
        for lay in (layout, None):
            o = tb.LatentAttention(block, lay)(q, q_r, cache, table, lengths, scale=0.1, **options)
            O.check(o, expected(cache, q, q_r, table, lengths, layout=lay, scale=0.1, **options), str(options.keys()))
            assert not bool(o[5].any())


def test_a_layout_of_fewer_blocks_than_the_table():
    layout = torch.ones(4, 3, 3, dtype=torch.int64)
    cache, q, q_r, table, lengths = setting(torch.bfloat16, 3, 4, 128, 32, [200, 96, 50], 1)
    o = tb.LatentAttention(32, layout)(q, q_r, cache, table, lengths, scale=0.1)
    O.check(o, expected(cache, q, q_r, table, lengths, layout=layout, scale=0.1), 'o')


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('H,latent', [(16, 128), (16, 512), (32, 256), (70, 128), (64, 512)])
def test_scores_that_grow(dtype, H, latent):
    """the running maximum moves again and again, up and far down"""
    cache, q, q_r, table, lengths = setting(dtype, 2, H, latent, 16, [1500, 1500], 2)
    rows = cache.data.view(-1, latent + 64)
    for b, sign in ((0, 1.), (1, -1.)):
        at = (table[b].long().repeat_interleave(16) * 16 + torch.arange(table.size(1) * 16, device=DEV) % 16)[:1500]
        rows[at, :64] = (sign * torch.linspace(-3, 3, 1500, device=DEV)[:, None]).to(dtype)
    q[..., :64] = 1.5
    o = tb.LatentAttention(16)(q, q_r, cache, table, lengths, scale=1.)
    O.check(o, expected(cache, q, q_r, table, lengths, scale=1.), 'o')


def test_views_shared_pages_and_wide_tables():
    cache, q, q_r, table, lengths = setting(torch.bfloat16, 4, 16, 512, 32, [100, 70, 33, 90], 4)
    op = tb.LatentAttention(32)
    o = op(q, q_r, cache, table, lengths, scale=0.1)
    packed = torch.cat([q, q_r], 2)
    assert torch.equal(o, op(packed[..., :512], packed[..., 512:], cache, table, lengths, scale=0.1))
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(o, op(by_head, q_r, cache, table, lengths, scale=0.1))
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape).copy_(q)
    assert torch.equal(o, op(odd, q_r, cache, table.T.contiguous().T, lengths, scale=0.1))
    wide = torch.full((4, 500), 2 ** 30, dtype=torch.int32, device=DEV)
    wide[:, :table.size(1)] = table
    O.check(op(q, q_r, cache, wide, lengths, scale=0.1), expected(cache, q, q_r, table, lengths, scale=0.1), 'a wide table')
    # one prompt's pages in two sequences' tables
    table[1] = table[0]
    O.check(op(q, q_r, cache, table, lengths, scale=0.1), expected(cache, q, q_r, table, lengths, scale=0.1), 'shared pages')
    assert op(q[:0], q_r[:0], cache, table[:0], lengths[:0]).shape == (0, 16, 512)
    assert not op(q.requires_grad_(True), q_r, cache, table, lengths).requires_grad


def test_captured_while_lengths_grow():
    cache, q, q_r, table, lengths = setting(torch.bfloat16, 3, 16, 512, 16, [400, 300, 290], 4)
    op = tb.LatentAttention(16)
    lengths -= 250
    op(q, q_r, cache, table, lengths, scale=0.1)
    graph, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = op(q, q_r, cache, table, lengths, scale=0.1)
    with torch.cuda.graph(two):
        o2 = op(q, q_r, cache, table, lengths, scale=0.05)
    for i in range(4):
        q.copy_(randn(tuple(q.shape), q.dtype, 30 + i))
        graph.replay()
        two.replay()
        assert torch.equal(o, op(q, q_r, cache, table, lengths, scale=0.1))
        assert torch.equal(o2, op(q, q_r, cache, table, lengths, scale=0.05))
        lengths += 60


def test_on_other_streams():
    cache, q, q_r, table, lengths = setting(torch.float16, 5, 32, 256, 64, [3000, 100, 700, 64, 65], 4)
    op = tb.LatentAttention(64)
    want = op(q, q_r, cache, table, lengths, scale=0.1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                got.append(op(q, q_r, cache, table, lengths, scale=0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(want, x) for x in got)


def test_offsets_past_32_bits():
    cache = tb.LatentCache(70000, 64)                         # 5.2 GB
    table = torch.tensor([[69999, 3, 65536], [1, 69000, 58254]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([170, 131], dtype=torch.int32, device=DEV)
    q, q_r, want = randn((2, 20, 512), torch.bfloat16, 1), randn((2, 20, 64), torch.bfloat16, 2), []
    for b in range(2):
        n = int(lengths[b])
        c, r = randn((n, 512), torch.bfloat16, 3 + b), randn((n, 64), torch.bfloat16, 5 + b)
        j = torch.arange(n, device=DEV)
        slots = (table[b, j // 64] * 64 + j % 64).int()
        cache.write(c, r, slots)
        got = cache.read(slots)
        assert torch.equal(got[0], c) and torch.equal(got[1], r)
        c, r = [torch.nn.functional.pad(t, (0, 0, 0, 192 - n)) for t in (c, r)]       # (the oracle takes whole pages)
        small = torch.arange(3, dtype=torch.int32, device=DEV)[None]
        want.append(O.attention(q[b:b + 1], q_r[b:b + 1], c, r, small, lengths[b:b + 1], 64, scale=0.04))
    o = tb.LatentAttention(64)(q, q_r, cache, table, lengths, scale=0.04)
    O.check(o, tuple(torch.cat([w[i] for w in want]) for i in range(2)), 'o')


@pytest.mark.parametrize('layout', [False, True])
def test_no_more_blocks_than_the_workspace_is_for(layout):
    """A C caller's mistake stays in its workspace: the blocks past most_blocks are not seen"""
    block, most = 16, 4
    rows = None
    if layout:
        # a first block-row of eight entries, and seven of none
        rows = torch.tensor([0] + [8] * 8 + [x for j in range(8) for x in (j, 1, 0)] + [0] * 3, dtype=torch.int32, device=DEV)
    cache, q, q_r, table, lengths = setting(torch.float16, 3, 1, 128, block, [128, 100, 128], 1)
    lib = _lib.load()
    need = lib.bsp_latent_attention_workspace_bytes(3, 1, 128, block, most)
    guard = torch.full((need + 4096,), 77, dtype=torch.uint8, device=DEV)
    o = torch.empty_like(q)
    ask = lengths if rows is None else torch.full_like(lengths, block)
    rc = lib.bsp_latent_attention(0, q.data_ptr(), 128, 128, q_r.data_ptr(), 64, 64, o.data_ptr(), 128, 128, 3, 1, cache.data.data_ptr(), cache.pages, block, 128, table.data_ptr(),
                                  table.stride(0), table.size(1), ask.data_ptr(), None if rows is None else rows.data_ptr(), 8, most, 0.05, 0., None, guard.data_ptr(), need, _lib.raw_stream(q.device))
    assert rc == 0
    assert bool((guard[need:] == 77).all())
    seen = ask.clamp(max=most * block)
    O.check(o, expected(cache, q, q_r, table, seen, scale=0.05), 'o')
