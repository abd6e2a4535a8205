"""GPU: the operators that SparseSelfAttention keeps: a captured chain outlives what other calls make."""
import pytest
import torch

import torch_blocksparse as tb

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.mark.parametrize('dtype,masked', [(torch.float16, False), (torch.float16, True), (torch.float32, False)])
def test_a_captured_chain_outlives_the_operators_of_decoding_and_of_other_lengths(dtype, masked):
    cls = tb.DeepSpeedSparseSelfAttention
    B, H, L, D, block = 2, 2, 128, 64, 16
    mod = tb.SparseSelfAttention(tb.SparsityConfig(block=block, stride=32, numverts=2))
    g = torch.Generator().manual_seed(4)
    static = [torch.randn(B, H, L, D, generator=g).to(dtype).to(DEV) for _ in range(4)]
    mask = torch.ones(L, L, dtype=dtype, device=DEV).tril() if masked else None

    def step():
        leaves = [t.detach().clone().requires_grad_(True) for t in static[:3]]
        o = mod(*leaves, attn_mask=mask)
        return (o.detach(),) + torch.autograd.grad(o, leaves, static[3])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    kept = mod.get_ops(H, L, static[0].device)
    cache = tb.KeyValueCache(2 * cls.OPS_CACHE_SIZE, block, H, D)
    q, lengths = torch.zeros(1, H, D, dtype=torch.float16, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    for n in range(1, cls.OPS_CACHE_SIZE + 2):
        mod.decode(q, cache, torch.zeros(1, n, dtype=torch.int32, device=DEV), lengths)
        y = torch.zeros(1, H, L + 32 * n, D, dtype=dtype, device=DEV)
        mod(y, y, y)
    assert mod.get_ops(H, L, static[0].device) is kept
    filler = [torch.full((1 << 14,), 1, dtype=torch.int32, device=DEV) for _ in range(64)]   # (what a dropped table's memory would be given to)
    for seed in (5, 6, 7):
        g.manual_seed(seed)
        for t in static:
            t.copy_(torch.randn(t.shape, generator=g))
        eager = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)
    del filler
