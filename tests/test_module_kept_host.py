"""CPU: which operators SparseSelfAttention keeps: each kind has places of its own, and what a captured graph has in it stays."""
import collections
import copy
import threading

import pytest
import torch

import torch_blocksparse as tb
from torch_blocksparse import _lib

CLS = tb.DeepSpeedSparseSelfAttention


@pytest.fixture
def empty(monkeypatch):
    monkeypatch.setattr(CLS, 'ops', collections.OrderedDict())
    monkeypatch.setattr(CLS, 'captured', dict())


def capturing(monkeypatch, yes):
    monkeypatch.setattr(torch.cuda, 'is_available', lambda: True)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: yes)


def module():
    return tb.SparseSelfAttention(tb.SparsityConfig(block=16, stride=64))


def test_a_kind_of_operators_takes_no_place_of_another(empty):
    mod = module()
    chain = mod.get_ops(2, 64)
    rules = mod._kept('rules', 2, 4, lambda layout: tb.Attention(layout, 16))
    for blocks in range(1, 2 * CLS.OPS_CACHE_SIZE):
        mod._kept('decode', 2, blocks, lambda layout: tb.CacheAttention(16, layout))
    assert mod.get_ops(2, 64) is chain and mod._kept('rules', 2, 4, None) is rules
    for blocks in range(1, 2 * CLS.OPS_CACHE_SIZE):
        mod.get_ops(2, 64 * blocks + 64)
    assert mod._kept('rules', 2, 4, None) is rules
    assert mod.get_ops(2, 64) is not chain               # (its own kind has as many places as ever)
    assert len(CLS.ops) == 2 * CLS.OPS_CACHE_SIZE + 1


def test_the_chain_of_a_graph_stays(empty, monkeypatch):
    mod = module()
    capturing(monkeypatch, False)
    mod.get_ops(2, 128)
    capturing(monkeypatch, True)
    chain = mod.get_ops(2, 64)
    capturing(monkeypatch, False)
    for blocks in range(2, 2 * CLS.OPS_CACHE_SIZE):
        mod.get_ops(2, 64 * blocks)
    assert [c for c in CLS.captured.values()] == [chain]
    assert mod.get_ops(2, 64) is chain


@pytest.mark.parametrize('kind', ['chain', 'rules'])
def test_another_thread_may_drop_operators(empty, monkeypatch, kind):
    """While a call has found its operators and not yet returned them, a second thread makes as many others as there are places."""
    mod, made, workers = module(), [], []

    def call(n):
        return mod.get_ops(2, 64 * n) if kind == 'chain' else mod._kept('rules', 2, n, lambda layout: tb.Attention(layout, 16))

    def others():
        for n in range(2, 3 + CLS.OPS_CACHE_SIZE):
            made.append(call(n))

    class Racing(collections.OrderedDict):
        def move_to_end(self, key):
            if not workers:
                workers.append(threading.Thread(target=others))
                workers[0].start()
                workers[0].join(0.5)                     # (as long as it takes, or waiting for this call)
            super().move_to_end(key)

    monkeypatch.setattr(CLS, 'ops', Racing())
    assert call(1) is not None
    workers[0].join(30)
    assert len(made) == 1 + CLS.OPS_CACHE_SIZE and len(CLS.ops) == CLS.OPS_CACHE_SIZE


class Table:
    """a device tensor that says which streams it was told of"""
    is_cuda = True

    def __init__(self):
        self.told = []

    def record_stream(self, stream):
        self.told.append(stream)

    def data_ptr(self):
        return 0


def test_tables_are_told_of_every_stream_that_reads_them(monkeypatch):
    now = [1]
    monkeypatch.setattr(_lib, 'raw_stream', lambda device: now[0])
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda device=None: 'stream %d' % now[0])
    early, late, readers = Table(), Table(), _lib.Readers()
    readers.table(early, None, torch.zeros(1))           # (one that is on the host needs nothing)
    for now[0] in (1, 2, 1):
        readers.read('device')
    readers.table(late)
    now[0] = 3
    readers.read('device')
    assert early.told == ['stream 1', 'stream 2', 'stream 3'] and sorted(late.told) == ['stream 1', 'stream 2', 'stream 3']


def test_the_tensors_of_an_operator_are_found_wherever_they_are():
    op, plan, t = tb.MatMul(torch.ones(1, 1, 1), 16, 'dsd'), tb.Softmax(torch.ones(1, 1, 1), 16), [torch.zeros(i + 1) for i in range(6)]
    plan.table, t[1].gplan, inside = t[0], plan, t[5]
    op.lut_cache['key'] = ([t[1], (t[2], None)], dict(a=t[3], b=op))
    op.build = lambda: inside
    op._products[0] = [t[4]]
    found = {id(x) for x in _lib.tensors_of((op, 3, 'text'))}
    assert found == {id(x) for x in t + [op.layout, plan.layout]}


def test_a_dropped_chain_tells_its_tables(empty, monkeypatch):
    told, now = [], [7]
    capturing(monkeypatch, False)
    monkeypatch.setattr(CLS, '_readers', dict())
    monkeypatch.setattr(_lib, 'raw_stream', lambda device: now[0])
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda device=None: now[0])
    monkeypatch.setattr(_lib.Readers, 'table', lambda self, *tensors: told.append((sorted(self.streams), len(tensors))))
    monkeypatch.setattr(CLS, '_chain', lambda self, H, L, device: (torch.zeros(H), torch.zeros(L)))
    mod, device = module(), torch.device('cuda', 0)
    for now[0] in (7, 8, 7):
        mod.get_ops(2, 64, device)
    for n in range(2, 2 + CLS.OPS_CACHE_SIZE):
        mod.get_ops(2, 64 * n, device)
    assert told == [([7, 8], 2)] and len(CLS._readers) == CLS.OPS_CACHE_SIZE


@pytest.mark.parametrize('attention', ['unidirectional', 'bidirectional'])
@pytest.mark.parametrize('stride,numverts,vertsize', [(64, 1, 1), (64, 2, 2), (112, 7, 1)])
def test_a_table_of_pages_that_grows_finds_its_operator(empty, monkeypatch, attention, stride, numverts, vertsize):
    mod = tb.SparseSelfAttention(tb.SparsityConfig(block=16, stride=stride, attention=attention, numverts=numverts, vertsize=vertsize))
    used = []
    monkeypatch.setattr(tb.CacheAttention, '__call__', lambda self, q, cache, table, lengths, **rules: used.append(self) or q)
    H, window = 9, stride // 16
    q, lengths = torch.zeros(1, H, 64, dtype=torch.float16), torch.ones(1, dtype=torch.int32)
    for width in range(1, 257):
        mod.decode(q, None, torch.zeros(1, width, dtype=torch.int32), lengths)
        lay = used[-1].layout
        # ... at most a quarter longer (short ones: sixteen blocks), with what each position of the table sees
        assert tuple(lay.shape) == (H,) + (lay.size(1),) * 2 and width <= lay.size(1) <= max(width + 15, 1.25 * width)
        if width % 37 == 0:
            exact = tb.fixed_layout(H, -(-width // window) * window, 'fixed', window, attention, numverts, vertsize)[:, :width, :width]
            assert torch.equal(lay[:, :width, :width].long(), exact)
    assert len({id(op) for op in used}) <= 16


def test_decoding_without_a_layout_makes_none(empty, monkeypatch):
    mod = tb.SparseSelfAttention(tb.SparsityConfig('dense', block=16, stride=64))
    sizes, used = [], []
    make = CLS._make_layout
    monkeypatch.setattr(CLS, '_make_layout', staticmethod(lambda H, blocks, *args, **k: sizes.append(blocks) or make(H, blocks, *args, **k)))
    monkeypatch.setattr(tb.CacheAttention, '__call__', lambda self, q, cache, table, lengths, **rules: used.append(self) or q)
    q, lengths = torch.zeros(1, 16, 64, dtype=torch.float16), torch.ones(1, dtype=torch.int32)
    for width in (1, 7, 300, 1 << 19):
        mod.decode(q, None, torch.zeros(1, 1, dtype=torch.int32).expand(1, width), lengths)
    assert used == [used[0]] * 4 and used[0].layout is None and not any(sizes)


def test_the_widest_layout_of_pages_is_made(empty, monkeypatch):
    mod = tb.SparseSelfAttention(tb.SparsityConfig(block=16, stride=16))
    widths = []
    monkeypatch.setattr(CLS, '_kept', lambda self, kind, H, blocks, make: widths.append(blocks) or (lambda *a, **k: None))
    q, lengths = torch.zeros(1, 1, 64, dtype=torch.float16), torch.ones(1, dtype=torch.int32)
    for width in (40000, 57344, 57345, 65535, 65536):
        mod.decode(q, None, torch.zeros(1, 1, dtype=torch.int32).expand(1, width), lengths)
    assert widths == [40960, 57344, 65535, 65535, 65536]


def bare_cache(monkeypatch):
    cache = tb.KeyValueCache.__new__(tb.KeyValueCache)
    cache.__setstate__(dict(pages=4, block=16, heads=2, head_dim=64, bits=4, device=torch.device('cpu'), data=Table(), _owner=Table()))
    return cache


def test_a_cache_tells_its_memory_of_the_streams_that_use_it(monkeypatch):
    now = [1]
    monkeypatch.setattr(_lib, 'raw_stream', lambda device: now[0])
    monkeypatch.setattr(_lib, 'on_device', lambda device: _lib._nothing)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda device=None: now[0])

    class Library:
        def __getattr__(self, name):
            return lambda *args: 0
    monkeypatch.setattr(_lib, 'load', lambda: Library())
    cache, slots, k = bare_cache(monkeypatch), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, 64)
    cache.write(k, k, slots)
    now[0] = 2
    cache.read(slots)
    now[0] = 3
    q, table, lengths = torch.zeros(1, 2, 64, dtype=torch.float16), torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    tb.CacheAttention(16)(q, cache, table, lengths)
    assert cache.data.told == cache._owner.told == [1, 2, 3]


def test_a_cache_can_be_copied(monkeypatch):
    monkeypatch.setattr(_lib, 'raw_stream', lambda device: 1)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda device=None: object())
    cache = bare_cache(monkeypatch)
    cache._users.read(cache.device)
    for other in (copy.deepcopy(cache), copy.copy(cache)):
        assert other.pages == 4 and other._users is not cache._users and not other._users.streams and other._users.tables == [other.data, other._owner]
