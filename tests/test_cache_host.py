"""CPU: what KeyValueCache and CacheAttention refuse, the sizes of the C ABI, and the table that a layout becomes."""
import pytest
import torch

import torch_blocksparse as tb
from torch_blocksparse import _lib
from torch_blocksparse.cache import _rows_table
from helpers import random_layout


@pytest.mark.parametrize('shape,kv', [((1, 1, 1), 1), ((4, 7, 7), 2), ((32, 5, 5), 1), ((40, 6, 6), 2), ((8, 20, 20), 8)])
def test_rows_table_holds_the_layout(shape, kv):
    lay = random_layout(shape, 0.3, 4)
    rows, longest = _rows_table(lay, kv)
    H, R, C = shape
    G = H // kv
    per = -(-G // -(-G // 16))
    assert per <= 16
    got = torch.zeros_like(lay)
    units = kv * -(-G // per)
    for unit in range(units):
        first = unit // -(-G // per) * G + unit % -(-G // per) * per
        starts = rows[unit * (R + 1):][:R + 1].tolist()
        for r in range(R):
            assert starts[r + 1] - starts[r] <= longest
            for e in rows[starts[r]:starts[r + 1]].tolist():
                e &= 0xffffffff
                for i in range(16):
                    if e >> i & 1:
                        got[first + i, r, e >> 16] += 1
    assert torch.equal(got != 0, lay != 0) and int(got.max()) <= 1 and rows.numel() == units * (R + 1) + sum(
        int((lay[h:h + n] != 0).any(0).sum()) for h, n in [(g * G + u, min(per, G - u)) for g in range(kv) for u in range(0, G, per)])


def test_sizes_of_the_abi():
    lib = _lib.load()
    assert lib.bsp_cache_page_bytes(16, 1, 64, 4) == 2 * 16 * (32 + 8) and lib.bsp_cache_page_bytes(128, 3, 128, 8) == 2 * 128 * 3 * (128 + 16)
    for bad in ((8, 1, 64, 4), (16, 0, 64, 4), (16, 1, 96, 4), (16, 1, 64, 2)):
        assert lib.bsp_cache_page_bytes(*bad) < 0
    assert lib.bsp_cache_attention_splits(64, 32, 8, 64, 128) >= 1
    assert lib.bsp_cache_attention_splits(1, 8, 8, 64, 1) == 1 and lib.bsp_cache_attention_splits(1, 1, 1, 16, 1 << 19) == 64
    assert lib.bsp_cache_attention_splits(1, 6, 4, 64, 1) < 0
    assert lib.bsp_cache_attention_workspace_bytes(2, 8, 2, 64, 1) == 0 and lib.bsp_cache_attention_workspace_bytes(2, 8, 2, 64, 3) == 2 * 8 * 3 * 66 * 4


def test_abi_refuses_before_it_launches():
    lib = _lib.load()
    x = torch.zeros(1 << 14, dtype=torch.uint8)
    at = x.data_ptr() + -x.data_ptr() % 16
    write = lambda **k: lib.bsp_cache_write(*[k.get(n, d) for n, d in (                  # noqa: E731
        ('dtype', 0), ('pages', at), ('n', 1), ('block', 16), ('heads', 1), ('D', 64), ('bits', 4), ('k', at), ('kt', 64), ('kh', 64), ('v', at), ('vt', 64), ('vh', 64),
        ('slots', at), ('T', 1), ('owner', at), ('stream', 0))])
    for bad in (dict(dtype=3), dict(pages=0), dict(pages=at + 8), dict(n=0), dict(block=48), dict(heads=0), dict(D=32), dict(bits=3), dict(k=at + 2), dict(kt=4), dict(vh=12),
                dict(slots=0), dict(T=0), dict(owner=0), dict(n=1 << 28)):
        assert write(**bad) < 0, bad
    read = lambda **k: lib.bsp_cache_read(*[k.get(n, d) for n, d in (                    # noqa: E731
        ('dtype', 0), ('pages', at), ('n', 1), ('block', 16), ('heads', 1), ('D', 64), ('bits', 4), ('k', at), ('v', at), ('slots', at), ('T', 1), ('stream', 0))])
    for bad in (dict(dtype=-1), dict(k=0), dict(v=at + 4), dict(bits=16), dict(T=-1)):
        assert read(**bad) < 0, bad
    names = ('dtype q qb qh o ob oh B H pages n block kv D bits table ts width lengths rows n_rows most scale cap slopes ws bytes splits stream').split()
    good = dict(zip(names, (0, at, 64, 64, at, 64, 64, 1, 1, at, 1, 16, 1, 64, 4, at, 1, 1, at, 0, 0, 1, 1., 0., 0, 0, 0, 1, 0)))
    for bad in (dict(dtype=2), dict(q=0), dict(q=at + 2), dict(qb=4), dict(o=at + 2), dict(oh=1), dict(B=0), dict(H=3, kv=2), dict(n=0), dict(block=20), dict(width=0),
                dict(width=1 << 20), dict(lengths=0), dict(rows=at), dict(rows=at, n_rows=1 << 17), dict(most=0), dict(scale=float('nan')), dict(cap=-1.), dict(splits=0), dict(splits=65),
                dict(splits=2), dict(splits=2, ws=at, bytes=16)):
        assert lib.bsp_cache_attention(*dict(good, **bad).values()) < 0, bad


def test_refusals():
    for bad in (dict(pages=0), dict(block=8), dict(heads=0), dict(head_dim=96), dict(bits=2), dict(pages=1 << 28)):
        with pytest.raises(ValueError):
            tb.KeyValueCache(**dict(dict(pages=2, block=16, heads=2, head_dim=64, bits=4), **bad))
    with pytest.raises(RuntimeError, match='GPU'):
        tb.KeyValueCache(2, 16, 2, 64, device='cpu')
    for block, lay in ((48, None), (16, torch.ones(2, 3, 4)), (16, torch.ones(3, 3)), (16, torch.ones(2, 0, 0))):
        with pytest.raises(ValueError):
            tb.CacheAttention(block, lay)


def test_refusals_of_calls():
    cache = tb.KeyValueCache.__new__(tb.KeyValueCache)
    cache.pages, cache.block, cache.heads, cache.head_dim, cache.bits, cache.device = 4, 16, 2, 64, 4, torch.device('cpu')
    slots, k = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, 64)
    assert cache._check_slots(slots) is slots and cache._operand(k, 'k', 3)[1:] == (128, 64)
    for bad in (slots.long(), slots[None], slots.float()):
        with pytest.raises(ValueError):
            cache._check_slots(bad)
    for bad in (k[:2], k[:, :1], k[..., :32], k.double(), k[0]):
        with pytest.raises(ValueError):
            cache._operand(bad, 'k', 3)
    with pytest.raises(ValueError):
        cache.write(k, k.half(), slots)
    with pytest.raises(ValueError):
        cache.read(slots, torch.float64)
    op = tb.CacheAttention(16, torch.ones(4, 3, 3))
    q, table, lengths = torch.zeros(2, 4, 64, dtype=torch.float16), torch.zeros(2, 5, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    op._check(q, cache, table, lengths, 1., 0., torch.zeros(4))
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[0]), dict(table=table[:1]), dict(table=table.long()), dict(table=table[:, :0]),
                dict(lengths=lengths.long()), dict(lengths=lengths[:1]), dict(slopes=torch.zeros(2)), dict(slopes=torch.zeros(4).half()), dict(softcap=-1.), dict(scale=float('inf')),
                dict(q=torch.zeros(2, 2, 64, dtype=torch.float16))):
        args = dict(dict(q=q, cache=cache, table=table, lengths=lengths, scale=1., softcap=0., slopes=None), **bad)
        with pytest.raises(ValueError):
            op._check(**args)
    with pytest.raises(ValueError):
        tb.CacheAttention(32)._check(q, cache, table, lengths, 1., 0., None)
