"""CPU: launches of more threads than a grid holds (2^32) are refused before anything is launched."""
import pytest
import torch

import torch_blocksparse as tb
from torch_blocksparse import _lib, cache, rules

UNSUPPORTED = -2


def aligned():
    x = torch.zeros(1 << 14, dtype=torch.uint8)
    return x, x.data_ptr() + -x.data_ptr() % 16


def test_a_cache_call_of_many_positions():
    """... of which the first of two launches would have left marks that later calls take for their own."""
    lib, (held, at) = _lib.load(), aligned()
    for T in (1 << 24, (1 << 31) - 1):
        assert lib.bsp_cache_write(0, at, 1 << 20, 16, 1, 64, 4, at, 64, 64, at, 64, 64, at, T, at, 0) == UNSUPPORTED
        assert lib.bsp_cache_read(0, at, 1 << 20, 16, 1, 64, 4, at, at, at, T, 0) == UNSUPPORTED


def test_attention_over_a_cache_of_many_sequences():
    lib, (held, at) = _lib.load(), aligned()
    for B, kv in ((1 << 24, 1), (1 << 20, 16)):
        assert lib.bsp_cache_attention(0, at, 64, 64, at, 64, 64, B, kv, at, 1, 16, kv, 64, 4, at, 1, 1, at, 0, 0, 1, 1., 0., 0, 0, 0, 1, 0) == UNSUPPORTED


def test_attention_of_many_lines():
    lib, (held, at) = _lib.load(), aligned()
    for Z, H, length in ((1 << 25, 1, 64), (1 << 20, 32, 1), (1 << 12, 8, 1 << 16)):
        lines = (length + 63) // 64
        call = rules._CALL.pack(0, Z, H, H, lines, 64, length, *([64] * 24), 1., 0., 0, 0, 0, 0, 0, 0, at, 0, 0)
        assert lib.bsp_attention_rules_fwd(call, at, at, at, at, 0) == UNSUPPORTED


def test_too_many_tokens_are_refused_by_name():
    held = tb.KeyValueCache.__new__(tb.KeyValueCache)
    held.device = torch.device('cpu')
    with pytest.raises(ValueError, match='tokens'):
        held._check_slots(torch.zeros(1, dtype=torch.int32).expand(1 << 24))
    held._check_slots(torch.zeros(5, dtype=torch.int32))


def test_a_layout_whose_rows_do_not_fit_32_bits(monkeypatch):
    """Places in the table of a layout's rows are 32 bits wide: a longer table is refused."""
    lay = torch.ones(2, 5, 5)
    whole = cache._rows_table(lay, 2)[0].numel()
    monkeypatch.setattr(cache, 'MOST_ROWS', whole)
    assert cache._rows_table(lay, 2)[0].numel() == whole
    monkeypatch.setattr(cache, 'MOST_ROWS', whole - 1)
    with pytest.raises(ValueError, match='layout'):
        cache._rows_table(lay, 2)


def test_a_layout_whose_tables_do_not_fit_32_bits(monkeypatch):
    lay = torch.ones(2, 8, 8)
    made = rules._Tables(lay, 64, torch.device('cpu'))
    rows, columns = made.rows.numel(), made.columns(2, 1)[0].numel()
    assert columns > rows
    monkeypatch.setattr(rules, 'MOST_PLACES', columns)
    assert rules._Tables(lay, 64, torch.device('cpu')).columns(2, 1)[0].numel() == columns
    monkeypatch.setattr(rules, 'MOST_PLACES', columns - 1)
    made = rules._Tables(lay, 64, torch.device('cpu'))
    with pytest.raises(ValueError, match='layout'):
        made.columns(2, 1)
    monkeypatch.setattr(rules, 'MOST_PLACES', rows - 1)
    with pytest.raises(ValueError, match='layout'):
        rules._Tables(lay, 64, torch.device('cpu'))
