"""SparseSelfAttention with score rules and its decode, on the host: what is refused, which layout a length gets, what is kept."""
import collections

import pytest
import torch

import torch_blocksparse as tb


@pytest.fixture
def empty(monkeypatch):
    monkeypatch.setattr(tb.DeepSpeedSparseSelfAttention, 'ops', collections.OrderedDict())
    monkeypatch.setattr(tb.DeepSpeedSparseSelfAttention, 'captured', dict())


@pytest.mark.parametrize('mode,attention', [('fixed', 'unidirectional'), ('fixed', 'bidirectional'), ('dense', 'unidirectional')])
@pytest.mark.parametrize('blocks', [1, 3, 4, 7, 13])
def test_a_length_has_the_first_blocks_of_the_next_whole_layout(empty, mode, attention, blocks):
    mod = tb.SparseSelfAttention(tb.SparsityConfig(mode, 16, 64, attention, numverts=2))
    op = mod._kept('rules', 4, blocks, lambda layout: tb.Attention(layout, 16))
    whole = tb.fixed_layout(4, -(-blocks // 4) * 4, mode, 4, attention, 2, 1)
    assert torch.equal(op.layout.long(), whole[:, :blocks, :blocks])
    assert mod._kept('rules', 4, blocks, None) is op
    # one direction: a block-row is the same in a longer layout, so a longer table of pages changes nothing
    if attention == 'unidirectional':
        longer = tb.fixed_layout(4, 16, mode, 4, attention, 2, 1)
        seen = torch.ones(blocks, blocks, dtype=torch.long).tril()
        assert torch.equal(op.layout.long() * seen, longer[:, :blocks, :blocks] * seen)


def test_the_operators_are_bounded_and_those_of_graphs_stay(empty, monkeypatch):
    cls = tb.DeepSpeedSparseSelfAttention
    mod = tb.SparseSelfAttention(tb.SparsityConfig(block=16, stride=64))
    make = lambda layout: tb.Attention(layout, 16)       # noqa: E731
    monkeypatch.setattr(torch.cuda, 'is_available', lambda: True)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    first = mod._kept('rules', 2, 1, make)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    for blocks in range(2, 2 * cls.OPS_CACHE_SIZE):
        mod._kept('rules', 2, blocks, make)
    assert len(cls.ops) == cls.OPS_CACHE_SIZE and list(cls.captured.values()) == [first]
    assert mod._kept('rules', 2, 1, None) is first
    with pytest.raises(TypeError):
        mod._kept('rules', 2, 2, None)                   # gone: made again


def test_refusals(empty):
    mod = tb.SparseSelfAttention(tb.SparsityConfig(block=16, stride=64))
    q, mask = torch.zeros(1, 2, 40, 64, dtype=torch.float16), torch.zeros(1, 40)
    for rules in (dict(softcap=5.), dict(slopes=torch.zeros(2)), dict(causal=True), dict(documents=torch.zeros(1, 40, dtype=torch.int32)), dict(prefix=torch.zeros(1, dtype=torch.int32))):
        for masks in (dict(rpe=mask), dict(key_padding_mask=mask), dict(attn_mask=mask)):
            with pytest.raises(ValueError, match='do not go with'):
                mod(q, q, q, **rules, **masks)
        with pytest.raises(ValueError):
            mod(q[0], q[0], q[0], **rules)
        with pytest.raises(RuntimeError, match='GPU'):
            mod(q, q, q, **rules)
    with pytest.raises(ValueError, match='do not go with'):
        mod(q, q[:, :1], q[:, :1], key_padding_mask=mask)
    with pytest.raises(ValueError, match='dividable'):
        mod(q, q, q)                                     # no rule: a length of whole blocks, as before
    with pytest.raises(ValueError):
        tb.SparseSelfAttention(tb.SparsityConfig(block=16, stride=56))(q, q, q, causal=True)
    with pytest.raises(ValueError):
        mod.decode(q, None, torch.zeros(1, 3, dtype=torch.int32), torch.ones(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        mod.decode(q[:, :, 0], None, torch.zeros(3, dtype=torch.int32), torch.ones(1, dtype=torch.int32))


@pytest.mark.parametrize('bad', [dict(softcap=1e-4), dict(softcap=2000.), dict(softcap=1e30), dict(softcap=-1.), dict(softcap=float('nan')), dict(scale=1e35), dict(scale=float('-inf'))])
def test_caps_and_scales_that_fp32_cannot_keep(bad, monkeypatch):
    from torch_blocksparse import _lib, rules
    numbers = dict(dict(scale=1., softcap=0.), **bad)
    with pytest.raises(ValueError):
        rules.check_scores(**numbers)
    lib = _lib.load()
    import ctypes
    at = 1 << 20
    call = rules._CALL.pack(0, 1, 1, 1, 1, 64, 16, *([64] * 12 + [0] * 12), numbers['scale'] if abs(numbers['scale']) < 1e38 else float('inf'), numbers['softcap'], 0, 0, 0, 0, 0, 0, at, 0, 0)
    assert lib.bsp_attention_rules_fwd(call, at, at, at, at, 0) < 0
    names = ('dtype q qb qh o ob oh B H pages n block kv D bits table ts width lengths rows n_rows most scale softcap slopes ws bytes splits stream').split()
    good = dict(zip(names, (0, at, 64, 64, at, 64, 64, 1, 1, at, 1, 16, 1, 64, 4, at, 1, 1, at, 0, 0, 1, 1., 0., 0, 0, 0, 1, 0)))
    assert lib.bsp_cache_attention(*[ctypes.c_float(v) if n in ('scale', 'softcap') else v for n, v in dict(good, **numbers).items()]) < 0


def test_good_caps_and_scales():
    from torch_blocksparse import rules
    for scale, softcap in ((1., 0.), (0., 1024.), (-3., 2. ** -10), (2. ** 100, 30.)):
        rules.check_scores(scale, softcap)
