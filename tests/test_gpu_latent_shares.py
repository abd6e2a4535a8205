"""GPU: attention over latent vectors that cancel, or of which one has nearly all of the sum: what a share loses where it becomes an operand of a product is then all there is to see."""
import pytest
import torch

import latent_oracle as O
import torch_blocksparse as tb

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def expected(cache, q, q_r, table, lengths, **options):
    """The oracle's value and bound for shares in two terms, which it has up to 32 heads: no more than that at a time"""
    rows, slopes = cache.data.view(-1, cache.latent + 64), options.pop('slopes', None)
    c, r = rows[:, :cache.latent], rows[:, cache.latent:]
    parts = [O.attention(q[:, h:h + 32], q_r[:, h:h + 32], c, r, table, lengths, cache.block, slopes=None if slopes is None else slopes[h:h + 32], **options) for h in range(0, q.size(1), 32)]
    return tuple(torch.cat(x, 1) for x in zip(*parts))


def call(dtype, H, latent, n, values, weight, slopes=None):
    """B = 3 sequences of n, n - 1 and 1 positions whose latent vectors are `values(position, sequence)` times one vector, so that a score is q times it"""
    g = torch.Generator().manual_seed(n + H)
    block, B = 16, 3
    pages = -(-n // block)
    cache = tb.LatentCache(B * pages, block, latent, dtype=dtype)
    vector = torch.randn(latent, generator=g).sign() * (1 + torch.rand(latent, generator=g))
    rows = torch.stack([torch.cat([values(j, b) * vector, torch.zeros(64)]) for b in range(B) for j in range(pages * block)])
    rows[:, latent:] = 0.5 * torch.randn(rows.size(0), 64, generator=g)
    cache.data.copy_(rows.view(cache.data.shape).to(dtype))
    q = (weight * torch.randn(B, H, latent, generator=g) / latent).to(dtype).to(DEV)
    q_r = (0.3 * torch.randn(B, H, 64, generator=g)).to(dtype).to(DEV)
    table = torch.arange(B * pages, dtype=torch.int32, device=DEV).view(B, pages)
    lengths = torch.tensor([n, max(1, n - 1), 1], dtype=torch.int32, device=DEV)
    o = tb.LatentAttention(block)(q, q_r, cache, table, lengths, scale=0.25, slopes=slopes)
    O.check(o, expected(cache, q, q_r, table, lengths, scale=0.25, slopes=slopes), 'o')


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('latent', [128, 256, 512])
@pytest.mark.parametrize('H', [16, 32, 33, 64, 65, 128])
@pytest.mark.parametrize('n', [2, 5, 64, 70])
def test_vectors_that_cancel(dtype, latent, H, n):
    call(dtype, H, latent, n, lambda j, b: 1. - 2. * (j % 2), 1.)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('H', [16, 64, 128])
@pytest.mark.parametrize('n', [3, 64, 130])
def test_one_position_has_nearly_all(dtype, H, n):
    """The newest, by a bias that falls with the distance; shares are relative to a maximum that was found before it"""
    slopes = torch.linspace(1., 3., H, device=DEV)
    call(dtype, H, 512, n, lambda j, b: 1. + 0.125 * (j % 5), 1., slopes)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('H', [32, 64, 128])
def test_equal_vectors_come_out_as_they_are(dtype, H):
    """their mean, whatever the shares"""
    cache = tb.LatentCache(5, 16, 256, dtype=dtype)
    g = torch.Generator().manual_seed(1)
    row = torch.randn(256, generator=g).to(dtype)
    cache.data[:, :, :256] = row.to(DEV)
    cache.data[:, :, 256:] = torch.randn(5, 16, 64, generator=g).to(dtype).to(DEV)
    q, q_r = torch.zeros(1, H, 256, dtype=dtype, device=DEV), torch.randn(1, H, 64, generator=g).to(dtype).to(DEV)
    table, lengths = torch.arange(5, dtype=torch.int32, device=DEV)[None], torch.tensor([77], dtype=torch.int32, device=DEV)
    o = tb.LatentAttention(16)(q, q_r, cache, table, lengths, scale=0.3)
    # (a share's two terms are off by u^2 of it, the sums by (2 * 77 + 24) 2^-24: with what the last rounding adds less than one step, u and the rounding's own half of one)
    u = torch.finfo(dtype).eps / 2
    assert bool(((o[0].double() - row.to(DEV).double()).abs() <= (u + u * u + 178 * 2. ** -24) * row.to(DEV).double().abs()).all())
