"""GPU: rotated positions against 64 bits, forward and gradients, and keys rotated on their way into a quantised cache."""
import pytest
import torch

import rotation_oracle as R
import torch_blocksparse as tb
from test_gpu_cache import quantised, same

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def frequencies(pairs, base=10000.):
    return [base ** (-p / pairs) for p in range(pairs)]


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('neighbours', [False, True])
@pytest.mark.parametrize('Z,H,kv,L,D,pairs', [(1, 1, 1, 1, 64, 32), (2, 4, 2, 37, 128, 64), (3, 5, 1, 130, 64, 8), (1, 2, 2, 19, 128, 24), (2, 1, 3, 5, 40, 16), (1, 33, 7, 300, 64, 32)])
def test_forward_and_gradients(dtype, neighbours, Z, H, kv, L, D, pairs):
    f = frequencies(pairs)
    op = tb.Rotation(f, neighbours=neighbours)
    q, k, gq, gk = randn((Z, H, L, D), dtype, 1), randn((Z, kv, L, D), dtype, 2), randn((Z, H, L, D), dtype, 3), randn((Z, kv, L, D), dtype, 4)
    positions = torch.randint(0, 5000, (Z, L), generator=torch.Generator().manual_seed(5)).int()
    q.requires_grad_(True), k.requires_grad_(True)
    y, z = op(q, k, positions=positions.to(DEV))
    dq, dk = torch.autograd.grad((y, z), (q, k), (gq, gk))
    angle = R.angles(positions, f)[:, None]
    for got, x, back in ((y, q, False), (z, k, False), (dq, gq, True), (dk, gk, True)):
        assert got.dtype == dtype and got.is_contiguous()
        R.check(got, R.turned(x, angle, neighbours, back), (back, tuple(x.shape)))
    with torch.no_grad():
        a, b = op(q, k, positions=positions.to(DEV))
    assert torch.equal(a, y) and torch.equal(b, z)
    # one tensor, positions of all sequences, and those that count from zero
    one = op(k.detach(), positions=positions[0].contiguous().to(DEV))
    R.check(one, R.turned(k, R.angles(positions[:1], f)[:, None], neighbours), 'shared positions')
    R.check(op(k.detach()), R.turned(k, R.angles(torch.arange(L), f), neighbours), 'no positions')


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('T,H,kv,D', [(1, 1, 1, 64), (7, 12, 3, 128), (1000, 3, 3, 64)])
def test_tokens(dtype, T, H, kv, D):
    f = frequencies(D // 2, 500000.)
    op = tb.Rotation(f)
    q, k = randn((T, H, D), dtype, 1), randn((T, kv, D), dtype, 2)
    positions = torch.randint(0, 131072, (T,), generator=torch.Generator().manual_seed(5)).int()
    angle = R.angles(positions, f)[:, None]
    for got, x in zip(op(q, k, positions=positions.to(DEV)), (q, k)):
        R.check(got, R.turned(x, angle, False), 'tokens')


def test_far_and_negative_positions_and_frequencies_of_all_kinds():
    f = [1., -1., 0., 2 * 3.141592653589793, 1e-9, 1e9, 3.5e18, 0.75] * 2
    op = tb.Rotation(f, neighbours=True)
    positions = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1, 12345678], dtype=torch.int32)
    x = randn((7, 2, 32), torch.float32, 6)
    # (an angle is off by 2^-34 of a turn for the farthest ones: 4e-10 beside the bound's 5e-7 of the elements)
    R.check(op(x, positions=positions.to(DEV)), R.turned(x, R.angles(positions, f)[:, None], True), 'far')
    assert torch.equal(op(x, positions=torch.zeros(7, dtype=torch.int32, device=DEV)), x)


def test_gradient_against_differences():
    op = tb.Rotation.of_base(64)
    x, g = randn((1, 2, 9, 64), torch.float32, 1).requires_grad_(True), randn((1, 2, 9, 64), torch.float32, 2)
    dx, = torch.autograd.grad(op(x), x, g)
    d = randn((1, 2, 9, 64), torch.float32, 3)
    with torch.no_grad():
        ahead, behind = [(op(x + s * d).double() * g.double()).sum() for s in (1., -1.)]
    # linear, so a difference of any width is the derivative; 1152 products whose factors are off by 8 * 2^-24 of sizes up to 4.5
    assert abs((ahead - behind) / 2 - (dx.double() * d.double()).sum()) < 1152 * 2 * 4.5 * 4.5 * 8 * 2. ** -24


def test_gradients_of_some_and_of_gradients():
    op = tb.Rotation.of_base(64, neighbours=True)
    q, k = randn((1, 2, 9, 64), torch.float32, 1).requires_grad_(True), randn((1, 1, 9, 64), torch.float32, 2)
    y, z = op(q, k)
    (y * y).sum().backward()
    angle = R.angles(torch.arange(9), op.frequencies.tolist())
    R.check(q.grad, (2 * q.detach().double().cpu(), 6 * R.turned(q, angle, True)[1]), 'a turn keeps lengths')
    # one output unused, and the gradient's gradient: turned back and forth
    q2, k2 = q.detach().clone().requires_grad_(True), k.clone().requires_grad_(True)
    y, z = op(q2, k2)
    gz = randn((1, 1, 9, 64), torch.float32, 3).requires_grad_(True)
    dk, = torch.autograd.grad(z, k2, gz, create_graph=True)
    w = randn((1, 1, 9, 64), torch.float32, 4)
    dgz, = torch.autograd.grad(dk, gz, w)
    R.check(dgz, R.turned(w, angle, True), 'second derivative')


def test_views_copies_and_empty_tensors():
    op = tb.Rotation.of_base(128)
    qkv = randn((2, 50, 3, 4, 128), torch.bfloat16, 1)                       # a packed projection
    q, k = qkv[:, :, 0].transpose(1, 2), qkv[:, :, 1].transpose(1, 2)
    want = op(q.contiguous(), k.contiguous())
    for got, x in zip(op(q, k), want):
        assert torch.equal(got, x)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape).copy_(q)
    assert torch.equal(op(odd), want[0])
    wide = q.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(op(wide), want[0])
    same_head = q[:, :1].expand(2, 4, 50, 128)
    assert torch.equal(op(same_head), op(same_head.contiguous()))
    positions = torch.arange(100, dtype=torch.int32, device=DEV)
    assert torch.equal(op(q, positions=positions[::2]), op(q, positions=positions[::2].contiguous()))
    assert torch.equal(op(q, positions=positions[:50].expand(2, 50)), want[0])
    assert op(q[:0], k[:0])[1].shape == (0, 4, 50, 128) and op(q[:, :, :0]).shape == (2, 4, 0, 128)
    a, b = op(q[:, :0], k)
    assert a.shape == (2, 0, 50, 128) and torch.equal(b, want[1])
    empty = q[:0].detach().requires_grad_(True)
    op(empty).sum().backward()
    assert empty.grad.shape == empty.shape


def test_offsets_past_32_bits():
    held = torch.empty((1 << 32) + (1 << 20), dtype=torch.bfloat16, device=DEV)           # 8.6 GB
    for shape, stride in (((2, 3, 5, 64), (1 << 32, 64 * 5, 64, 1)), ((1, 2, 5, 64), (0, 1 << 32, 64, 1)), ((1, 1, 3, 64), (0, 0, 1 << 31, 1))):
        x = held.as_strided(shape, stride)
        x.copy_(randn(shape, torch.bfloat16, 1))
        assert torch.equal(tb.Rotation.of_base(64)(x), tb.Rotation.of_base(64)(x.contiguous()))


def test_changed_positions_are_noticed():
    op = tb.Rotation.of_base(64)
    x, positions = randn((4, 2, 64), torch.float32, 1).requires_grad_(True), torch.arange(4, dtype=torch.int32, device=DEV)
    y = op(x, positions=positions)
    positions += 1
    with pytest.raises(RuntimeError, match='modified'):
        y.sum().backward()


def test_captured_and_on_another_stream():
    op = tb.Rotation.of_base(64)
    x, positions = randn((30, 8, 64), torch.float16, 1), torch.arange(30, dtype=torch.int32, device=DEV)
    op(x, positions=positions)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = op(x, positions=positions)
    for i in range(3):
        x.copy_(randn((30, 8, 64), torch.float16, 10 + i))
        positions += 7
        graph.replay()
        assert torch.equal(y, op(x, positions=positions))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        z = op(x, positions=positions)
    stream.synchronize()
    assert torch.equal(z, y)


# ---- keys rotated on their way into the cache ----------------------------------------------------------------------------------------


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('neighbours', [False, True])
@pytest.mark.parametrize('T,heads,D,pairs,bits,block', [(1, 1, 64, 32, 4, 16), (9, 16, 64, 32, 8, 64), (70, 3, 128, 64, 4, 32), (130, 5, 128, 24, 8, 16), (700, 2, 64, 8, 4, 128)])
def test_written_rotated(dtype, neighbours, T, heads, D, pairs, bits, block):
    f = frequencies(pairs)
    cache = tb.KeyValueCache(1024 // block, block, heads, D, bits=bits)
    k, v = 3 * randn((T, heads, D), dtype, 1), randn((T, heads, D), dtype, 2)
    positions = torch.randint(0, 131072, (T,), generator=torch.Generator().manual_seed(5)).int()
    slots = torch.randperm(1024, generator=torch.Generator().manual_seed(6))[:T].int().to(DEV)
    cache.write(k, v, slots, rotation=tb.Rotation(f, neighbours=neighbours), positions=positions.to(DEV))
    got = cache.read(slots, torch.float32)
    want = R.turned(k.double(), R.angles(positions, f)[:, None], neighbours)[0]
    assert same(got[0], quantised(want, bits)[0], torch.float32)
    assert same(got[1], quantised(v, bits)[0], torch.float32)
    assert not bool(cache._owner.any())


@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
def test_position_zero_is_no_rotation(bits, dtype):
    """The same bits as without one, middles between codes and values past float16's range among them"""
    most, D = 2 ** bits - 1, 64
    ties = (torch.arange(D) % (2 * most)).float() / 2
    ties[::32], ties[31::32] = 0., float(most)
    rows = [torch.zeros(D), torch.full((D,), -65504.), ties, ties / 4 - 8, ties * 0.3, torch.linspace(-1, 1, D)]
    if dtype != torch.float16:
        rows.append(torch.linspace(-1e30, 1e20, D))
    x = torch.stack(rows)[:, None].to(dtype).to(DEV)
    slots, zero = torch.arange(len(rows), dtype=torch.int32, device=DEV), torch.zeros(len(rows), dtype=torch.int32, device=DEV)
    for rotation in (tb.Rotation.of_base(64), tb.Rotation.of_base(32, neighbours=True)):
        a, b = tb.KeyValueCache(3, 16, 1, D, bits=bits), tb.KeyValueCache(3, 16, 1, D, bits=bits)
        a.write(x, x.flip(0), slots)
        b.write(x, x.flip(0), slots, rotation=rotation, positions=zero)
        assert torch.equal(a.data, b.data)


def test_rotated_nan_stays_in_its_pairs_groups():
    cache = tb.KeyValueCache(2, 16, 1, 128, bits=8)
    k = randn((3, 1, 128), torch.bfloat16, 1)
    k[0, 0, 5] = float('nan')
    k[1, 0, 70] = float('inf')
    slots = torch.arange(3, dtype=torch.int32, device=DEV)
    cache.write(k, k, slots, rotation=tb.Rotation.of_base(128), positions=slots + 1)
    got = cache.read(slots, torch.float32)[0][:, 0]
    assert bool(torch.isnan(got[0, :32]).all()) and bool(torch.isnan(got[0, 64:96]).all()) and bool(torch.isfinite(got[0, 32:64]).all()) and bool(torch.isfinite(got[0, 96:]).all())
    # (an infinity: the one with the sign of its sine or cosine, as the type's largest value)
    assert not bool(torch.isnan(got[1]).any()) and bool((got[1].abs() > 60000.).any())
    assert bool(torch.isfinite(got[2]).all())


@pytest.mark.parametrize('T', [40, 700])
def test_the_last_of_a_slot_is_written_rotated(T):
    cache, rotation = tb.KeyValueCache(20, 16, 2, 64, bits=8), tb.Rotation.of_base(64)
    k, v = randn((T, 2, 64), torch.float16, 1), randn((T, 2, 64), torch.float16, 2)
    slots = torch.randint(-3, min(320, T), (T,), generator=torch.Generator().manual_seed(T)).int().to(DEV)
    positions = torch.arange(T, dtype=torch.int32, device=DEV)
    cache.write(k, v, slots, rotation=rotation, positions=positions)
    last = {s: t for t, s in enumerate(slots.tolist()) if s >= 0}
    other = tb.KeyValueCache(20, 16, 2, 64, bits=8)
    rows = torch.tensor(list(last.values()), device=DEV)
    other.write(k[rows], v[rows], slots[rows], rotation=rotation, positions=positions[rows])
    assert torch.equal(cache.data, other.data)


def test_rotated_write_captured():
    cache, other, rotation = tb.KeyValueCache(4, 16, 2, 64, bits=4), tb.KeyValueCache(4, 16, 2, 64, bits=4), tb.Rotation.of_base(64)
    k, v = randn((6, 2, 64), torch.bfloat16, 1), randn((6, 2, 64), torch.bfloat16, 2)
    slots, positions = torch.arange(6, dtype=torch.int32, device=DEV), torch.arange(6, dtype=torch.int32, device=DEV)
    cache.write(k, v, slots, rotation=rotation, positions=positions)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.write(k, v, slots, rotation=rotation, positions=positions)
    for i in range(3):
        k.copy_(randn((6, 2, 64), torch.bfloat16, 20 + i))
        slots += 6
        positions += 6
        graph.replay()
        other.write(k, v, slots, rotation=rotation, positions=positions)
        for a, b in zip(cache.read(slots), other.read(slots)):
            assert torch.equal(a, b)
