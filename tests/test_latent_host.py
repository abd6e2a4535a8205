"""CPU: what LatentCache and LatentAttention refuse, and the table of a layout's rows."""
import copy

import pytest
import torch

import torch_blocksparse as tb
from torch_blocksparse import _lib, latent

ERR_ARG, UNSUPPORTED, CAPACITY = -1, -2, -3


def test_caches():
    for bad in (dict(block=48), dict(latent=96), dict(latent=1024), dict(shared=32), dict(dtype=torch.float32), dict(pages=0), dict(pages=1 << 28)):
        with pytest.raises(ValueError):
            tb.LatentCache(**dict(dict(pages=4, block=16, latent=512), **bad))
    with pytest.raises(_lib.BlocksparseLibraryError):
        tb.LatentCache(4, 16, device='cpu')


def host_cache(block=16, width=128, dtype=torch.bfloat16):
    cache = tb.LatentCache.__new__(tb.LatentCache)
    cache.pages, cache.block, cache.latent, cache.dtype, cache.device = 8, block, width, dtype, torch.device('cpu')
    return cache


def test_writes():
    cache = host_cache()
    c, r, slots = torch.zeros(5, 128, dtype=torch.bfloat16), torch.zeros(5, 64, dtype=torch.bfloat16), torch.zeros(5, dtype=torch.int32)
    p, rotation = torch.zeros(5, dtype=torch.int32), tb.Rotation.of_base(64)
    bad = [(c, r, slots.long()), (c, r, slots[None]), (c[:4], r, slots), (c, r[:4], slots), (c.half(), r, slots), (c, r.float(), slots), (c, r[:, :32], slots), (c[:, :64], r, slots),
           (c, r, slots, rotation), (c, r, slots, None, p), (c, r, slots, rotation, p[:4]), (c, r, slots, tb.Rotation.of_base(128), p), (c, r, slots, rotation, p.float())]
    for args in bad:
        with pytest.raises(ValueError):
            cache.write(*args)
    cache.write(c[:0], r[:0], slots[:0])
    with pytest.raises(ValueError, match='2\\^24'):
        cache._check_slots(torch.zeros(1, dtype=torch.int32).expand(1 << 24))


def test_attention():
    for args in ((48,), (16, torch.ones(2, 3)), (16, torch.ones(2, 3, 4)), (16, torch.ones(0, 3, 3))):
        with pytest.raises(ValueError):
            tb.LatentAttention(*args)
    op, cache = tb.LatentAttention(16, torch.ones(3, 4, 4)), host_cache()
    q, q_r = torch.zeros(2, 3, 128, dtype=torch.bfloat16), torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    table, lengths = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    good = dict(q=q, q_r=q_r, cache=cache, table=table, lengths=lengths, scale=1., softcap=0., slopes=None)
    op._check(**good)
    other = tb.KeyValueCache.__new__(tb.KeyValueCache)
    other.device = torch.device('cpu')
    for bad in (dict(cache=other), dict(cache=host_cache(32)), dict(cache=host_cache(16, 256)), dict(cache=host_cache(dtype=torch.float16)), dict(q=q.half()), dict(q_r=q_r[:, :2]), dict(q_r=q_r[:, :, :32]),
                dict(q=q[0]), dict(q=q[:, :2], q_r=q_r[:, :2]), dict(q=q[:1]), dict(table=table.long()), dict(table=table[:1]), dict(table=table[:, :0]), dict(table=table[0]),
                dict(table=table[:, :1].expand(2, 1 << 20)), dict(lengths=lengths.long()), dict(lengths=lengths[:1]), dict(slopes=torch.zeros(2)), dict(slopes=torch.zeros(3).half()),
                dict(softcap=2000.), dict(softcap=-1.), dict(scale=float('nan')), dict(scale=2. ** 101)):
        with pytest.raises(ValueError):
            op._check(**dict(good, **bad))
    with pytest.raises(ValueError, match='KeyValueCache'):
        cache.heads, cache.head_dim = 1, 128
        tb.CacheAttention(16)._check(torch.zeros(2, 3, 128, dtype=torch.float16), cache, table, lengths, 1., 0., None)
    assert copy.deepcopy(op)._rows == {}


@pytest.mark.parametrize('H,per', [(3, 3), (40, 40), (65, 33), (128, 64)])
def test_rows(H, per):
    assert _lib.load().bsp_latent_attention_heads(H) == per
    R = 5
    layout = (torch.rand(H, R, R, generator=torch.Generator().manual_seed(H)) < 0.3).long()
    layout[:, 2] = 0
    t = [x & 0xffffffff for x in latent._rows_table(layout, per).tolist()]
    units = -(-H // per)
    back, entries = torch.zeros_like(layout), t[units * (R + 1):]
    for u in range(units):
        for i in range(R):
            for e in range(t[u * (R + 1) + i], t[u * (R + 1) + i + 1]):
                col, heads = entries[3 * e], entries[3 * e + 1] | entries[3 * e + 2] << 32
                assert heads
                for h in range(64):
                    if heads >> h & 1:
                        back[u * per + h, i, col] = 1
    assert torch.equal(back, layout) and len(entries) == 3 * (t[units * (R + 1) - 1] + 1)


def test_rows_that_do_not_fit_32_bits(monkeypatch):
    monkeypatch.setattr(latent, 'MOST_ROWS', 24)
    with pytest.raises(ValueError, match='layout'):
        latent._rows_table(torch.ones(2, 5, 5), 2)


def test_c_entries_refuse():
    lib = _lib.load()
    held = torch.zeros(1 << 14, dtype=torch.uint8)
    at = held.data_ptr() + -held.data_ptr() % 16
    write = lambda dtype=0, pages=at, n=4, block=16, latent=128, c=at, st=128, r=at, slots=at, T=1, owner=at, f=None, pairs=0, p=None: \
        lib.bsp_latent_write(dtype, pages, n, block, latent, c, st, r, 64, slots, T, owner, f, pairs, 0, p, None)    # noqa: E731
    for bad in (dict(pages=None), dict(pages=at + 8), dict(n=0), dict(c=None), dict(c=at + 8), dict(st=4), dict(r=None), dict(r=at + 1), dict(slots=None), dict(T=0), dict(owner=None),
                dict(f=at, pairs=32), dict(f=at, pairs=12, p=at), dict(f=at, pairs=40, p=at)):
        assert write(**bad) == ERR_ARG, bad
    for bad in (dict(dtype=2), dict(block=48), dict(latent=64), dict(n=1 << 27), dict(T=1 << 24)):
        assert write(**bad) == UNSUPPORTED, bad
    read = lambda c=at, r=at, T=1: lib.bsp_latent_read(0, at, 4, 16, 128, c, r, at, T, None)    # noqa: E731
    assert read(c=None) == read(r=at + 4) == read(T=0) == ERR_ARG and read(T=1 << 24) == UNSUPPORTED

    def attention(dtype=0, q=at, q_sh=128, qr=at, o=at, B=1, H=1, n=4, block=16, width=4, rows=None, n_rows=0, most=4, scale=1., cap=0., ws=at, ws_bytes=1 << 40):
        return lib.bsp_latent_attention(dtype, q, 128, q_sh, qr, 64, 64, o, 128, 128, B, H, at, n, block, 128, at, width, width, at, rows, n_rows, most, scale, cap, None, ws, ws_bytes, None)
    for bad in (dict(q=None), dict(q=at + 8), dict(q_sh=4), dict(qr=at + 8), dict(o=None), dict(B=0), dict(H=0), dict(width=0), dict(most=0), dict(rows=at), dict(scale=2. ** 101), dict(cap=2000.), dict(ws=at + 8)):
        assert attention(**bad) == ERR_ARG, bad
    for bad in (dict(dtype=2), dict(block=48), dict(width=1 << 20), dict(n=1 << 27), dict(B=1 << 24), dict(rows=at, n_rows=65537)):
        assert attention(**bad) == UNSUPPORTED, bad
    need = lib.bsp_latent_attention_workspace_bytes(3, 65, 512, 64, 10)
    assert need == -(-3 * 2 * 8 // 16) * 16 + 60 * 2 * 33 * 514 * 4 and lib.bsp_latent_attention_workspace_bytes(3, 65, 512, 64, 1) == 48
    assert attention(ws=None) == attention(ws_bytes=8) == CAPACITY
    assert lib.bsp_latent_attention_workspace_bytes(3, 65, 96, 64, 10) == lib.bsp_latent_attention_workspace_bytes(0, 65, 512, 64, 10) == ERR_ARG
