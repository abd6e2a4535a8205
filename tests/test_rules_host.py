"""CPU: the tables of torch_blocksparse.Attention against the layouts that they stand for, and what its calls refuse."""
import pytest
import torch

import torch_blocksparse as tb
from torch_blocksparse.rules import _Tables
from helpers import random_layout

CASES = [((2, 5, 5), 16, 2, 0.4), ((4, 3, 3), 32, 2, 0.5), ((4, 9, 9), 64, 1, 0.3), ((6, 2, 2), 128, 3, 0.7), ((1, 1, 1), 16, 1, 1.0), ((8, 21, 21), 16, 2, 0.2),
         ((2, 40, 40), 64, 1, 0.9)]


def blocks_of_16(layout, block, rows):
    lay = (layout != 0).repeat_interleave(block // 16, 1).repeat_interleave(block // 16, 2)
    return torch.nn.functional.pad(lay, (0, rows // 16 - lay.size(2), 0, rows // 16 - lay.size(1)))


def pieces(entry, fixed, by_rows):
    """(row, column) in groups of sixteen of the pieces that an entry of a tile holds"""
    bits = int(entry[4])
    for a in range(4):
        for b in range(4):
            if bits >> (4 * a + b) & 1:
                yield (fixed[a], int(entry[b])) if by_rows else (int(entry[a]), fixed[b])


@pytest.mark.parametrize('shape,block,kv,density', CASES)
def test_tables_hold_every_block_once(shape, block, kv, density):
    lay = random_layout(shape, density, 7)
    lay[:, :, 0] = 1                                        # one long column
    t = _Tables(lay, block, torch.device('cpu'))
    H, rows = shape[0], 64 * t.lines
    assert rows >= shape[1] * block
    want = blocks_of_16(lay, block, rows)
    got = torch.zeros_like(want, dtype=torch.int32)
    for h in range(H):
        for line in range(t.lines):
            n, at = t.rows[2 * (h * t.lines + line):][:2].tolist()
            for e in t.rows[at:at + 8 * n].view(-1, 8):
                for r, c in pieces(e, [64 * line + 16 * g for g in range(4)], True):
                    got[h, r // 16, c // 16] += 1
    assert torch.equal(got, want.int())
    for batches in (1, 3, 1000):
        items, n_items, splits, n_splits, slots = t.columns(kv, batches)
        got = torch.zeros_like(want, dtype=torch.int32)
        heads, used, keys = items[:12 * kv * n_items].view(kv, n_items, 12), [], dict()
        assert bool((heads[:, 1:, 0] <= heads[:, :-1, 0]).all())
        for at, i in enumerate(heads.flatten(0, 1).tolist()):
            assert i[1] >= 12 * kv * n_items and (i[1] - 12 * kv * n_items) % 8 == 0 and i[1] + 8 * i[0] <= items.numel()
            if i[3] < 0:
                assert i[0] == 0 and i[4] == -1
                continue
            assert i[2] == at // n_items
            used += [i[4]] if i[4] >= 0 else []
            keys.setdefault((i[2], i[3]), []).append(i)
            for e in items[i[1]:i[1] + 8 * i[0]].view(-1, 8):
                for at, c in pieces(e, i[8:], False):
                    h, r = i[2] * (H // kv) + (at >> 24), at & (1 << 24) - 1
                    got[h, r // 16, c // 16] += 1
        assert torch.equal(got, want.int())
        assert sorted(used) == list(range(slots))
        assert len(keys) == kv * t.lines                    # every column of tiles has an item, and so its gradients
        assert sorted(p for (g, _), items_of in keys.items() if g == 0 for p in items_of[0][8:]) == list(range(0, rows, 16))
        cut = {key: v for key, v in keys.items() if len(v) > 1}
        assert n_splits == len(cut) and (splits is None) == (not cut)
        for s in ([] if splits is None else splits.tolist()):
            parts = cut[s[0], s[1]]
            assert sorted(i[4] for i in parts) == list(range(s[2], s[2] + s[3])) and s[4:] == parts[0][8:]


def test_every_item_has_one_workgroup():
    # the order of workgroups in the kernels (rules_place): each item of each head once, and the XCDs (every eighth workgroup) get equal shares of them
    for units in (1, 2, 7, 8, 9, 12, 16, 40, 100):
        for n in (1, 3, 8, 65):
            rest, spread = units % 8, (units % 8 * n + 7) // 8 * 8
            got, share = set(), [0] * 8
            for wg in range(spread + units // 8 * 8 * n):
                if wg < spread:
                    unit, item = (units // 8 * 8 + wg % rest if wg // rest < n else -1), wg // rest
                else:
                    per, x, i = units // 8, wg - spread & 7, wg - spread >> 3
                    first = i // (4 * n) * 4
                    heads = min(4, per - first)
                    unit, item = x * per + first + i % (4 * n) % heads, i % (4 * n) // heads
                if unit >= 0:
                    assert 0 <= unit < units and 0 <= item < n and (unit, item) not in got
                    got.add((unit, item))
                    share[wg % 8] += 1
            assert len(got) == units * n and max(share) - min(share) <= 1


def test_refusals_of_the_constructor():
    lay = torch.ones(2, 3, 3)
    for layout, block in ((lay, 8), (lay, 24), (lay, 256), (torch.ones(2, 3, 4), 16), (torch.ones(3, 3), 16)):
        with pytest.raises(ValueError):
            tb.Attention(layout, block)
    with pytest.raises(ValueError):
        tb.Attention(torch.ones(1, 1 << 17, 1).expand(1, 1 << 17, 1 << 17), 128)


def test_calls_need_a_gpu():
    q = torch.zeros(1, 2, 40, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match='GPU'):
        tb.Attention(torch.ones(2, 3, 3), 16)(q, q, q)


def test_refusals_of_a_call(monkeypatch):
    monkeypatch.setattr(tb.rules._lib, 'require_gpu_tensor', lambda t, what: None)
    op = tb.Attention(torch.ones(4, 3, 3), 16)
    half = lambda *shape: torch.zeros(*shape, dtype=torch.float16)       # noqa: E731
    q, k = half(2, 4, 40, 64), half(2, 2, 40, 64)
    good = dict(softcap=0., scale=1., slopes=None, causal=True, documents=None, prefix=None)
    op._check(q, k, k, **good)
    ids = torch.zeros(2, 40, dtype=torch.int32)
    op._check(q, k, k, **dict(good, documents=ids, prefix=ids[:, 0], slopes=torch.zeros(4)))
    for args in ((q[0], k, k), (q, k.float(), k), (q, k, half(2, 2, 40, 128)), (half(2, 4, 40, 32),) * 3, (q, half(2, 3, 40, 64), half(2, 3, 40, 64)),
                 (half(2, 4, 32, 64), half(2, 2, 32, 64), half(2, 2, 32, 64)), (half(2, 4, 49, 64),) * 3, (half(2, 2, 40, 64),) * 3, (q, half(2, 4, 41, 64), half(2, 4, 41, 64)),
                 (q.double(), k.double(), k.double()), (half(2, 4, 0, 64),) * 3, (half(1, 4, 40, 64), k, k)):
        with pytest.raises(ValueError):
            op._check(*args, **good)
    for bad in (dict(softcap=-1.), dict(softcap=float('inf')), dict(softcap=float('nan')), dict(scale=float('nan')), dict(slopes=torch.zeros(2)), dict(slopes=half(4)),
                dict(slopes=torch.zeros(4, requires_grad=True)), dict(documents=ids.long()), dict(documents=ids[:, :39]), dict(documents=ids[0]),
                dict(prefix=torch.zeros(2)), dict(prefix=torch.zeros(1, dtype=torch.int32)), dict(causal=False, prefix=ids[:, 0])):
        with pytest.raises(ValueError):
            op._check(q, k, k, **dict(good, **bad))
