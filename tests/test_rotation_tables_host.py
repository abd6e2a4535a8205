"""CPU: what Rotation computes of its frequencies is computed once, when it is made."""
import copy
import pickle

import torch

import torch_blocksparse as tb
from torch_blocksparse import _lib, rotation


def test_a_first_call_computes_no_fractions(monkeypatch):
    op = tb.Rotation.of_base(64)
    others = [copy.deepcopy(op), pickle.loads(pickle.dumps(op)), copy.copy(op)]
    want = [rotation._fraction_of_a_turn(f) for f in op.frequencies.tolist()]
    monkeypatch.setattr(rotation, '_fraction_of_a_turn', None)
    monkeypatch.setattr(_lib, 'raw_stream', lambda device: 0)
    monkeypatch.setattr(_lib.Readers, 'read', lambda self, device: None)
    for x in [op] + others:
        for device in (torch.device('cpu'), torch.device('cpu', 0)):
            assert x.fractions(device).tolist() == want


def test_states_without_them():
    """as objects that were stored by an earlier version have"""
    state = tb.Rotation.of_base(32).__getstate__()
    assert set(state) == {'frequencies', 'pairs', 'neighbours', '_fractions'}
    op = tb.Rotation.__new__(tb.Rotation)
    op.__setstate__(state)
    assert op._turns.tolist() == tb.Rotation.of_base(32)._turns.tolist()


def test_two_threads_make_one_table(monkeypatch):
    """a table that was given to a call stays: nothing else holds it until the launch"""
    op, device, inner = tb.Rotation.of_base(64), torch.device('cpu', 0), []
    monkeypatch.setattr(_lib, 'raw_stream', lambda device: 0)
    monkeypatch.setattr(_lib.Readers, 'read', lambda self, device: None)
    turns = op._turns

    class Turns:
        def to(self, device):                              # (the other thread's call, while this one copies its table)
            if not inner:
                inner.append(None)
                inner[0] = op.fractions(device)
            return turns.clone()

    op._turns = Turns()
    outer = op.fractions(device)
    assert outer is inner[0] and op.fractions(device) is outer
