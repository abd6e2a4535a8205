"""GPU: the codes themselves of turned keys, where 32 of them lie so close together, far from zero, that fp32 does not tell them apart."""
import pytest
import torch

import rotation_oracle as R
import torch_blocksparse as tb

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def held(cache, T, D, bits):
    """(codes [T, D], steps and least values [T, D / 32]) of the keys of a cache of one head, whose first T positions are written.  A page has the codes of `block` keys, then their steps and least
    values; of a key, eight elements that follow each other (a chunk) are `bits` bytes, chunk c of group g at c * (D / 32) + g; in four bits element 2 i of a chunk is nibble i, element 2 i + 1 nibble 4 + i"""
    groups, row, block = D // 32, D * bits // 8, cache.block
    pages = cache.data.cpu()
    codes = pages[:, :block * row].reshape(-1, 4, groups, bits)[:T]
    meta = pages[:, block * row:block * (row + 4 * groups)].reshape(-1, groups, 4)[:T].contiguous().view(torch.float16).double()
    if bits == 4:
        low = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)                     # nibbles 0 .. 7
        codes = torch.stack([low[..., :4], low[..., 4:]], -1).flatten(-2)
    return codes.transpose(1, 2).reshape(T, D).long(), meta[..., 0], meta[..., 1]


def definition(x, bits):
    """the same of x [T, D] in 64 bits; and how far each is from a border between two codes"""
    g = x.unflatten(-1, (-1, 32)).clamp(-65504., 65504.)
    least = g.amin(-1).float().half().double()
    step = ((g.amax(-1) - least) / (2 ** bits - 1)).float().half().double()
    at = (g - least[..., None]) / torch.where(step == 0, 1., step)[..., None]
    codes = torch.where((step == 0)[..., None], 0., at.round().clamp(0, 2 ** bits - 1))
    return codes.flatten(-2).long(), step, least, ((at - at.floor()) - 0.5).abs().flatten(-2)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('neighbours', [False, True])
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('a,b', [(1000., -1.), (16384., -8.), (-2048., 0.5), (32768., 4.), (3., 1.), (65280., -16.)])
def test_turned_elements_close_together(dtype, bits, neighbours, D, a, b):
    T, pairs = 9, D // 2
    f = [500000. ** (-p / pairs) for p in range(pairs)]
    cache = tb.KeyValueCache(1, 16, 1, D, bits=bits)
    k = torch.empty(T, 1, D)
    one, two = (slice(0, None, 2), slice(1, None, 2)) if neighbours else (slice(0, pairs), slice(pairs, None))
    k[..., one], k[..., two] = a, b
    k = k.to(dtype)
    positions = torch.tensor([0, 1, 2, 3, 5, 8, 100, 4000, 131071], dtype=torch.int32)
    cache.write(k.to(DEV), k.to(DEV), torch.arange(T, dtype=torch.int32, device=DEV), rotation=tb.Rotation(f, neighbours=neighbours), positions=positions.to(DEV))
    turned = R.turned(k[:, 0].double(), R.angles(positions, f), neighbours)[0]
    codes, step, least, border = definition(turned, bits)
    got = held(cache, T, D, bits)
    assert torch.equal(got[2], least) and torch.equal(got[1], step)
    # (a frequency is off by 2^-65 of a turn, an angle by that for each position, 2^-62 of an element's size; sines, products and sums in 64 bits leave 2^-49 of it: what lies nearer a border may fall either way)
    off = (2. ** -49 + positions.double().abs()[:, None] * 2. ** -62) * (abs(a) + abs(b))
    near = border <= off / step.abs().clamp(min=2. ** -24).repeat_interleave(32, 1)
    assert float(near.double().mean()) < 0.01
    wrong = (got[0] != codes) & ~near
    assert not bool(wrong.any()), '%d of %d codes, by up to %d' % (int(wrong.sum()), wrong.numel(), int((got[0] - codes).abs().max()))
