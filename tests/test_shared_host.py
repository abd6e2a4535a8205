"""CPU: what attention with a shared key part refuses, and the module's calls of both forms."""
import pytest
import torch

import torch_blocksparse as tb
from test_rotation_host import fake
from torch_blocksparse import _lib, rules

ERR_ARG, UNSUPPORTED = -1, -2


def test_shared_parts():
    q, k, q_s, k_s = fake(2, 3, 40, 64), fake(2, 1, 40, 64), fake(2, 3, 40, 64), fake(2, 40, 64)
    check = tb.Attention._check_shared
    check(q, k, (q_s, k_s))
    check(q, k, [q_s, k_s])
    for bad in (q_s, (q_s,), (q_s, k_s, k_s), (q_s, k_s[:1]), (q_s, k_s[:, :39]), (q_s[:, :1], k_s), (q_s[..., :32], k_s[..., :32]), (q_s, fake(2, 3, 40, 64)), (q_s.float(), k_s), (q_s, k_s.float())):
        with pytest.raises(ValueError):
            check(q, k, bad)
    with pytest.raises(_lib.BlocksparseLibraryError):
        check(q, k, (torch.zeros(2, 3, 40, 64).half(), k_s))
    with pytest.raises(ValueError, match='65535'):
        check(fake(1, 1, 1, 64).expand(65536, 1, 1, 64), k, (fake(1, 1, 1, 64).expand(65536, 1, 1, 64), fake(1, 1, 64).expand(65536, 1, 64)))


def test_shared_does_not_go_with_masks():
    module, x = tb.SparseSelfAttention(tb.SparsityConfig(block=16)), torch.zeros(1, 2, 64, 64)
    with pytest.raises(ValueError, match='key_padding_mask'):
        module(x, x, x, key_padding_mask=torch.zeros(1, 64), shared=(x, x[:, 0]))


def test_decoding_goes_by_the_cache():
    module = tb.SparseSelfAttention(tb.SparsityConfig(block=16))
    q, table, lengths = torch.zeros(1, 2, 128), torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    latent, heads = tb.LatentCache.__new__(tb.LatentCache), tb.KeyValueCache.__new__(tb.KeyValueCache)
    for cache, options in ((latent, dict()), (latent, dict(scale=1.)), (latent, dict(shared=q)), (heads, dict(scale=1.)), (heads, dict(shared=q)), (heads, dict(shared=q, scale=1.))):
        with pytest.raises(ValueError, match='LatentCache'):
            module.decode(q, cache, table, lengths, **options)


def test_c_entries_refuse():
    lib = _lib.load()
    held = torch.zeros(1 << 14, dtype=torch.uint8)
    at = held.data_ptr() + -held.data_ptr() % 16

    def call(entry, q=at, k=at, strides=(64,) * 10, dq=at, dk=at, heads=at, Z=1, part=True, **call):
        c = rules._CALL.pack(call.get('dtype', 0), Z, 1, 1, 1, call.get('D', 64), 64, *([64] * 24), 1., 0., 0, 0, 0, 0, 0, 0, at, at, at)
        p = rules._PART.pack(q, k, *strides, dq, dk, heads) if part else None
        if entry == 'fwd':
            return lib.bsp_attention_shared_fwd(c, p, at, at, at, at, None)
        return lib.bsp_attention_shared_bwd(c, p, at, at, at, at, at, at, at if dk else None, at if dk else None, at, at, 1, None, 0, None, 0, None)
    for entry in ('fwd', 'bwd'):
        for bad in (dict(part=False), dict(q=0), dict(k=0), dict(q=at + 8), dict(k=at + 2), dict(strides=(4,) + (64,) * 9), dict(strides=(64, 64, 56) + (64,) * 7), dict(strides=(64,) * 4 + (0,) + (64,) * 5),
                    dict(strides=(64, 64, 1 << 40) + (64,) * 7)):
            assert call(entry, **bad) == ERR_ARG, (entry, bad)
        assert call(entry, D=96) == UNSUPPORTED and call(entry, dtype=3) == UNSUPPORTED
    for bad in (dict(dq=0), dict(dq=at + 4), dict(heads=0), dict(strides=(64,) * 7 + (56, 64, 64)), dict(strides=(64,) * 9 + (0,))):
        assert call('bwd', **bad) == ERR_ARG, bad
    assert call('bwd', Z=65536) == UNSUPPORTED
