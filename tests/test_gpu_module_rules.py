"""GPU: SparseSelfAttention with score rules, and a prompt and its answer through the module and a cache."""
import pytest
import torch

import rules_oracle as R
import torch_blocksparse as tb

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('kv,L,mode,attention', [(4, 256, 'fixed', 'unidirectional'), (2, 201, 'fixed', 'unidirectional'), (1, 77, 'fixed', 'bidirectional'), (4, 130, 'dense', 'unidirectional')])
def test_forward_and_backward_with_rules(dtype, kv, L, mode, attention):
    B, H, D, block = 2, 4, 64, 16
    g = torch.Generator().manual_seed(L)
    q, k, v, do = [torch.randn(B, h, L, D, generator=g).to(dtype) for h in (H, kv, kv, H)]
    ids = (torch.arange(L) * 3 // L).int().repeat(B, 1)
    ids[1, L - 9:] = -1
    rules = dict(softcap=12., slopes=torch.tensor([0.2, 0.05, 0.01, 0.]), causal=True, documents=ids, prefix=torch.tensor([5, 0], dtype=torch.int32))
    mod = tb.SparseSelfAttention(tb.SparsityConfig(mode, block, 64, attention, numverts=2))
    blocks = -(-L // block)
    lay = tb.fixed_layout(H, -(-blocks // 4) * 4, mode, 4, attention, 2, 1)[:, :blocks, :blocks]
    want = R.attention(q, k, v, lay, block, do=do, scale=D ** -0.5, **rules)
    qg, kg, vg = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    o = mod(qg, kg, vg, **{n: t.to(DEV) if torch.is_tensor(t) else t for n, t in rules.items()})
    o.backward(do.to(DEV))
    for name, got in (('o', o), ('dq', qg.grad), ('dk', kg.grad), ('dv', vg.grad)):
        R.check(got, want[name], name)
    # keys given transposed, as without rules
    with torch.no_grad():
        again = mod(qg, kg.transpose(2, 3), vg, **{n: t.to(DEV) if torch.is_tensor(t) else t for n, t in rules.items()})
    assert torch.equal(again, o)


def test_shared_key_heads_alone_take_the_rules_way():
    B, H, L, D = 1, 4, 64, 64
    g = torch.Generator().manual_seed(1)
    q, k, v = [torch.randn(B, h, L, D, generator=g).half() for h in (H, 2, 2)]
    mod = tb.SparseSelfAttention(tb.SparsityConfig())
    want = R.attention(q, k, v, tb.fixed_layout(H, 4, 'fixed', 4, 'unidirectional', 1, 1), 16, scale=D ** -0.5)
    R.check(mod(q.to(DEV), k.to(DEV), v.to(DEV)), want['o'], 'o')


@pytest.mark.parametrize('mode', ['fixed', 'dense'])
def test_a_prompt_and_its_answer(mode):
    B, H, kv, D, block, L, prompt = 2, 4, 2, 64, 16, 75, 61
    mod = tb.SparseSelfAttention(tb.SparsityConfig(mode, block, 32, numverts=2))
    g = torch.Generator().manual_seed(5)
    q, k, v = [torch.randn(B, h, L, D, generator=g).half().to(DEV) for h in (H, kv, kv)]
    rules = dict(softcap=10., slopes=torch.tensor([0.5, 0.1, 0.02, 0.], device=DEV))
    blocks = -(-L // block)
    cache = tb.KeyValueCache(B * blocks, block, kv, D, bits=8)
    table = torch.randperm(B * blocks, generator=g).int().view(B, blocks).to(DEV)
    pos = torch.arange(L, device=DEV)
    slots = (table[:, pos // block] * block + pos % block).int()
    cache.write(k[:, :, :prompt].transpose(1, 2).flatten(0, 1), v[:, :, :prompt].transpose(1, 2).flatten(0, 1), slots[:, :prompt].flatten())
    steps = []
    for t in range(prompt, L):
        cache.write(k[:, :, t], v[:, :, t], slots[:, t].contiguous())
        steps.append(mod.decode(q[:, :, t], cache, table, torch.full((B,), t + 1, dtype=torch.int32, device=DEV), **rules))
    kc, vc = [x.view(B, L, kv, D).transpose(1, 2) for x in cache.read(slots.flatten(), torch.float32)]
    whole = mod(q.float(), kc, vc, causal=True, **rules)
    # fp16: result, share and value rounded (2^-11 each) of values up to the largest
    assert float((torch.stack(steps, 2).float() - whole[:, :, prompt:]).abs().max()) <= 3 * 2. ** -11 * float(vc.abs().max())


def test_a_captured_step_outlives_the_operators_kept():
    cls = tb.DeepSpeedSparseSelfAttention
    B, H, D, block, width = 2, 2, 64, 16, 6
    mod = tb.SparseSelfAttention(tb.SparsityConfig(block=block, stride=32))
    cache = tb.KeyValueCache(B * width, block, H, D)
    g = torch.Generator().manual_seed(2)
    k, v = [torch.randn(B * width * block, H, D, generator=g).half().to(DEV) for _ in range(2)]
    cache.write(k, v, torch.arange(B * width * block, dtype=torch.int32, device=DEV))
    table = torch.arange(B * width, dtype=torch.int32, device=DEV).view(B, width)
    q, lengths = torch.randn(B, H, D, generator=g).half().to(DEV), torch.tensor([90, 33], dtype=torch.int32, device=DEV)
    x = torch.randn(1, H, 40, D, generator=g).half().to(DEV)
    step = lambda: (mod.decode(q, cache, table, lengths), mod(x, x, x, causal=True))       # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for blocks in range(3, 4 + cls.OPS_CACHE_SIZE):
        y = torch.randn(1, H, 16 * blocks, D, generator=g).half().to(DEV)
        mod(y, y, y, causal=True)
    filler = [torch.full((1 << 16,), 7, dtype=torch.int32, device=DEV) for _ in range(64)]   # (what a freed table's memory could be given to)
    for n in (90, 17, 64):
        lengths.fill_(n)
        q.copy_(torch.randn(B, H, D, generator=g))
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)
    del filler
