"""GPU: the quantised cache at the ends of float16's range."""
import math

import pytest
import torch

import torch_blocksparse as tb
from test_gpu_cache import quantised

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
