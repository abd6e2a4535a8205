"""CPU: tables that the library writes in host memory are made there whatever torch's default device is (written through the address of a
device tensor, they would end the process)."""
import pytest
import torch

from helpers import random_layout
from torch_blocksparse import attention_core
from torch_blocksparse.cache import _rows_table
from torch_blocksparse.matmul import GroupPlan
from torch_blocksparse.rules import _Tables

HOST = torch.device('cpu')
SMALL, TALL, LARGE = random_layout((4, 20, 20), 0.4, 1), random_layout((2, 8, 8), 0.9, 3), random_layout((2, 64, 64), 0.9, 4)


def rules():
    t = _Tables(SMALL, 16, HOST)
    items, n_items, splits, n_splits, slots = t.columns(2, 1)
    return [t.rows, items] + ([] if splits is None else [splits])


MADE = dict(rules=rules, decode=lambda: [_rows_table(SMALL, 2)[0]],
            stored=lambda: [attention_core._stored_tables(TALL, 16)[0]], quad=lambda: [attention_core._QuadTables(TALL, 16, HOST).rows],
            tiles=lambda: [GroupPlan.build_sdd_tiles(TALL, HOST).table], chunks=lambda: [GroupPlan.build_xsd_chunks(LARGE, True, HOST, always=True).table])


@pytest.mark.parametrize('what', sorted(MADE))
def test_tables_are_made_on_the_host(what):
    want = MADE[what]()
    with torch.device('meta'):
        got = MADE[what]()
    assert len(got) == len(want)
    for a, b in zip(want, got):
        assert b.device.type == 'cpu' and torch.equal(a, b)
