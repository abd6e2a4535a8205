"""GPU: operators that are made and first called while the GPU is torch's default device, and those first called in inference mode."""
import collections

import pytest
import torch

import torch_blocksparse as tb

pytestmark = pytest.mark.gpu


def steps():
    B, H, kv, L, D, block = 2, 4, 2, 96, 64, 16
    g = torch.Generator(device='cuda').manual_seed(3)
    q, k, v = [torch.randn(B, h, L, D, generator=g, device='cuda').half() for h in (H, kv, kv)]
    mod = tb.SparseSelfAttention(tb.SparsityConfig(block=block, stride=32, numverts=2))
    with torch.device('cpu'):
        lay = tb.bigbird_layout(H, L // block, causal=True)
    cache = tb.KeyValueCache(B * L // block, block, kv, D, bits=8)
    cache.write(k.transpose(1, 2).flatten(0, 1), v.transpose(1, 2).flatten(0, 1), torch.arange(B * L, dtype=torch.int32, device='cuda'))
    table = torch.arange(B * L // block, dtype=torch.int32, device='cuda').view(B, -1)
    lengths = torch.full((B,), L, dtype=torch.int32, device='cuda')
    kx, vx = k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)
    rules, decode = tb.Attention(lay, block), tb.CacheAttention(block, lay)

    def step(grad):
        out = [mod(q, k, v, causal=True), mod(q, kx, vx), rules(q, k, v), mod.decode(q[:, :, -1].contiguous(), cache, table, lengths), decode(q[:, :, -1].contiguous(), cache, table, lengths)]
        if grad:
            leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
            out += torch.autograd.grad(rules(*leaves, causal=True), leaves, q)
        return out
    return step


def test_the_gpu_as_the_default_device(monkeypatch):
    want = steps()(True)
    monkeypatch.setattr(tb.DeepSpeedSparseSelfAttention, 'ops', collections.OrderedDict())
    with torch.device('cuda'):
        got = steps()(True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_first_calls_in_inference_mode(monkeypatch):
    want = steps()(True)
    monkeypatch.setattr(tb.DeepSpeedSparseSelfAttention, 'ops', collections.OrderedDict())
    step = steps()
    with torch.inference_mode():
        first = step(False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(True)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(first + got, want[:5] + want):
        assert torch.equal(a, b)
