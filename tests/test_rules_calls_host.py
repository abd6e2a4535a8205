"""CPU: calls of Attention that launch nothing, and slopes that are a parameter of the model."""
import pytest
import torch

import torch_blocksparse as tb


def check(slopes, q_grad=False):
    q = torch.zeros(2, 4, 40, 64, dtype=torch.float16, requires_grad=q_grad)
    tb.Attention(torch.ones(4, 3, 3), 16)._check(q, q, q, 0., 1., slopes, True, None, None)


def test_slopes_that_are_a_parameter(monkeypatch):
    monkeypatch.setattr(tb.rules._lib, 'require_gpu_tensor', lambda t, what: None)
    slopes = torch.nn.Parameter(torch.zeros(4))
    for q_grad in (False, True):
        with pytest.raises(ValueError, match='gradient'):
            check(slopes, q_grad)
        with torch.no_grad():
            check(slopes, q_grad)
        with torch.inference_mode():
            check(slopes, q_grad)
        check(slopes.detach(), q_grad)


@pytest.mark.parametrize('Z,L', [(0, 40), (2, 0), (0, 0)])
def test_no_positions_or_no_sequences(monkeypatch, Z, L):
    monkeypatch.setattr(tb.rules._lib, 'require_gpu_tensor', lambda t, what: None)
    q, k, v = [torch.zeros(Z, h, L, 64, dtype=torch.float16, requires_grad=True) for h in (4, 2, 2)]
    blocks = -(-L // 16)
    o = tb.Attention(torch.ones(4, blocks, blocks), 16)(q, k, v, causal=True, documents=torch.zeros(Z, L, dtype=torch.int32))
    assert o.shape == q.shape and o.dtype == q.dtype
    grads = torch.autograd.grad(o, (q, k, v), torch.zeros_like(o))
    assert [g.shape for g in grads] == [q.shape, k.shape, v.shape]


def test_gradients_that_the_backward_pass_cannot_address_are_refused_in_the_forward_pass(monkeypatch):
    monkeypatch.setattr(tb.rules._lib, 'require_gpu_tensor', lambda t, what: None)
    G, block = 127, 128
    length = -(-(1 << 29) // G)                          # G * length is just past 2^29
    for L, refused in ((length, True), (length - block, False)):
        blocks = -(-L // block)
        op = tb.Attention(torch.ones(1, 1, 1, dtype=torch.uint8).expand(G, blocks, blocks), block)
        q = torch.zeros(1, 1, 1, 64, dtype=torch.float16).expand(1, G, L, 64)
        k, leaf = q[:, :1], torch.zeros(1, 1, 1, 64, dtype=torch.float16, requires_grad=True).expand(1, 1, L, 64)
        args = (0., 1., None, True, None, None)
        op._check(q, k, k, *args)
        with torch.no_grad():
            op._check(q, leaf, leaf, *args)
        for keys, values in ((leaf, k), (k, leaf)):
            if refused:
                with pytest.raises(ValueError, match='gradient'):
                    op._check(q, keys, values, *args)
            else:
                op._check(q, keys, values, *args)
