"""CPU: slopes that are a parameter of the model: refused where a gradient would be expected of them, taken where none is."""
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
