"""GPU: the quantised cache and attention over it at the ends of float16's range."""
import math

import pytest
import torch

import torch_blocksparse as tb
from test_gpu_cache import check, oracle, quantised

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def saturated(T, kv, D, dtype, seed):
    """keys, and values of which every position has a group at an end of float16's range or past it"""
    g = torch.Generator().manual_seed(seed)
    k, v = [torch.randn(T, kv, D, generator=g) for _ in range(2)]
    big = 65504. if dtype == torch.float16 else 1e6
    v[0::4, :, 0::32] = big
    v[1::4, :, 1::32], v[1::4, :, 2::32] = big, -big
    v[2::4, :, 3::32] = -big
    v[3::4] = v[3::4].abs() * 3e4
    return [t.clamp(-big, big).to(dtype).to(DEV) for t in (k, v)]


@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
def test_what_is_finite_reads_back_finite(bits, dtype):
    """The step of such a group may be rounded up, and with it the greatest element past 65504: float16 has it as 65504."""
    k, v = saturated(64, 2, 64, dtype, 1)
    v[5, 0, 40] = math.nan
    cache = tb.KeyValueCache(4, 16, 2, 64, bits=bits)
    slots = torch.arange(64, dtype=torch.int32, device=DEV)
    cache.write(k, v, slots)
    want = quantised(v, bits)[0]
    assert float(want.nan_to_num().max()) > 65504        # (there is something to see)
    for other in (torch.float16, torch.bfloat16, torch.float32):
        got = cache.read(slots, other)[1].cpu()
        once = (want.clamp(max=65504.) if other == torch.float16 else want).float().to(other)
        assert bool(torch.isnan(got[5, 0, 32:]).all()) and int(torch.isnan(got).sum()) == 32
        assert bool(((got == once) | (torch.isnan(got) & torch.isnan(once))).all()) and not bool(torch.isinf(got).any())


@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('H,kv', [(2, 2), (7, 1), (16, 1)])
def test_decoding_over_values_at_the_ends(bits, D, dtype, H, kv):
    """... and attention takes them as 65504 too: where a head's share is nothing, or its layout hides the block that another head of the
    workgroup sees, nothing comes of them."""
    B, block, width = 2, 16, 4
    T = B * width * block
    k, v = saturated(T, kv, D, dtype, 3)
    cache = tb.KeyValueCache(B * width, block, kv, D, bits=bits)
    cache.write(k, v, torch.arange(T, dtype=torch.int32, device=DEV))
    table = torch.arange(B * width, dtype=torch.int32, device=DEV).view(B, width)
    g = torch.Generator().manual_seed(7)
    q = (40 * torch.randn(B, H, D, generator=g)).to(dtype).to(DEV)            # (most shares are below 2^-24)
    lengths = torch.tensor([64, 51], dtype=torch.int32, device=DEV)
    lay = torch.ones(H, width, width, dtype=torch.int64)
    lay[::2, :, 1] = 0
    lay[1::2, :, 2] = 0
    (kq, step, least), vq = quantised(k, bits), quantised(v, bits)[0].clamp(max=65504.)
    held = [t.view(B, -1, kv, D) for t in (kq, vq, least, step)]
    everything = torch.ones(B, width * block, dtype=torch.bool)
    for layout in (None, lay):
        for scale in (1., 1e-4):
            o = tb.CacheAttention(block, layout)(q, cache, table, lengths, scale=scale)
            out, bound = oracle(q, *held[:2], held[2], held[3], bits, lengths, layout, block, scale, 0., None, everything)
            # a result in fp16 whose bound reaches past the type's range may be infinite: from above it is held to nothing, from below, as any
            # result, to |got| >= |out| - bound (sums of values of both signs may have a bound that is wide)
            fits = (out.abs() + bound <= 65504.) if dtype == torch.float16 else torch.ones_like(out, dtype=torch.bool)
            assert bool(fits.float().mean() > 0.5)
            got = o.double().cpu()
            assert not bool(torch.isnan(got).any())
            check(torch.where(fits, got, out), (out, bound), 'scale %g' % scale)
            assert bool((got.abs() >= out.abs() - bound)[~fits].all())


@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('softcap', [0., 9.])
@pytest.mark.parametrize('exponent', [-120, 100, 117, 118, 122, 126])
def test_queries_at_the_ends_of_bfloat16(bits, softcap, exponent):
    """Queries so large (or small) that only the scale makes scores of them, keys that are zero among the others."""
    B, H, kv, D, block, width = 2, 4, 2, 64, 16, 4
    T = B * width * block
    g = torch.Generator().manual_seed(exponent)
    k, v = [torch.randn(T, kv, D, generator=g).bfloat16().to(DEV) for _ in range(2)]
    k[::3] = 0.
    cache = tb.KeyValueCache(B * width, block, kv, D, bits=bits)
    cache.write(k, v, torch.arange(T, dtype=torch.int32, device=DEV))
    table = torch.arange(B * width, dtype=torch.int32, device=DEV).view(B, width)
    q = (torch.rand(B, H, D, generator=g) * 1.9 - 0.95).double().mul(2. ** exponent).bfloat16().to(DEV)
    q[1, :, 3] = 2. ** exponent
    lengths = torch.tensor([64, 51], dtype=torch.int32, device=DEV)
    (kq, step, least), vq = quantised(k, bits), quantised(v, bits)[0]
    held = [t.view(B, -1, kv, D) for t in (kq, vq, least, step)]
    everything = torch.ones(B, width * block, dtype=torch.bool)
    scale = max(2. ** -exponent, 2. ** -100) if exponent > 0 else 2. ** 100
    for scale in (scale, 2. ** -exponent if exponent > 0 else scale, -scale):
        o = tb.CacheAttention(block)(q, cache, table, lengths, scale=scale, softcap=softcap)
        check(o, oracle(q, *held[:2], held[2], held[3], bits, lengths, None, block, scale, softcap, None, everything), 'scale %g' % scale)


@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('D', [64, 128])
def test_groups_whose_least_value_is_rounded_up_past_them(bits, D):
    """Elements closer together than float16's numbers: the least value rounded to float16 may lie above all of them, and the step below zero."""
    g = torch.Generator().manual_seed(5)
    base = torch.tensor([1000.3, 1000.1, -1000.1, 0.1, 65500., -65490., 3e-8, 12.003, -7.7e-5, 1 / 3])
    spread = torch.tensor([0., 2. ** -15, 2. ** -13, 2. ** -12, 2. ** -11])
    x = (base[:, None, None] * (1 + spread[:, None] * torch.rand(len(base), len(spread), D, generator=g))).view(-1, 1, D)
    cache = tb.KeyValueCache(4, 16, 1, D, bits=bits)
    slots = torch.arange(x.size(0), dtype=torch.int32, device=DEV)
    cache.write(x.to(DEV), x.flip(0).to(DEV), slots)
    # from the definition (a code is 0 where the step is 0), in 64 bits
    groups, most = x.double().clamp(-65504., 65504.).unflatten(-1, (-1, 32)), 2 ** bits - 1
    least = groups.amin(-1, keepdim=True).float().half().double()
    step = ((groups.amax(-1, keepdim=True) - least) / most).float().half().double()
    assert 10 < int((step < 0).sum()) < step.numel() - 10
    code = torch.where(step != 0, ((groups - least) / torch.where(step != 0, step, 1.)).round().clamp(0, most), 0.)
    want = (least + code * step).flatten(-2)
    for got, value in zip(cache.read(slots, torch.float32), (want, want.flip(0))):
        assert torch.equal(got.double().cpu(), value.float().double())


@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('H', [1, 6, 16])
@pytest.mark.parametrize('length', [64, 4096])
def test_shares_of_a_float16_result_are_not_those_of_its_type(bits, D, H, length):
    """Half of the positions have scores of zero, the others scores whose exponential is off by 4e-4 of itself when it is rounded to float16, to
    what makes their values cancel.  (Groups of one value each: the cache holds them as they are.)"""
    block, score = 16, -497 / 1024
    k, v = [torch.zeros(length, 1, D) for _ in range(2)]
    e = math.exp(score)
    low = -float(torch.tensor(e).half())
    k[1::2], v[0::2], v[1::2] = score, low, 1.
    cache = tb.KeyValueCache(length // block, block, 1, D, bits=bits)
    cache.write(k.half().to(DEV), v.half().to(DEV), torch.arange(length, dtype=torch.int32, device=DEV))
    q = torch.zeros(1, H, D, dtype=torch.float16, device=DEV)
    q[..., 5] = 1.
    o = tb.CacheAttention(block)(q, cache, torch.arange(length // block, dtype=torch.int32, device=DEV)[None], torch.tensor([length], dtype=torch.int32, device=DEV))
    want, size = (low + e) / (1 + e), (abs(low) + e) / (1 + e)
    # sums in fp32 of terms of that size, shares in two terms of eleven bits each, the result
    c = 2. ** -24 * (2 * D + length / 8 + 8 + 32)         # (a lane's sum is of a sixteenth of the positions)
    bound = (c + 2. ** -22) * size + 2. ** -11 * abs(want) + 2. ** -25
    assert abs(want) > 4 * bound                         # (with shares rounded to float16 it is zero)
    assert float((o.double() - want).abs().max()) <= bound
