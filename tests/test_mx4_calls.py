"""4-bit storage without a GPU: which calls the products take and which they refuse, beyond types and sizes."""
import pytest
import torch

import neuzip
from tests.test_mx4_host import manager_with

BF16 = torch.bfloat16


class Launched(Exception):
    pass


@pytest.fixture
def at_launch(monkeypatch):
    """A product that is let through ends where its kernels would be launched."""
    from neuzip_b200.mx4 import MX4Backend
    calls = []

    def launch(self, entry, x, n_rows, per_input, ids, bias, y):
        calls.append((x, bias, y))
        return y.zero_()
    monkeypatch.setattr(MX4Backend, "_launch", launch)
    return calls


def test_a_bias_may_need_a_gradient(at_launch):
    m = manager_with((32, 64))
    x, bias = torch.zeros(2, 3, 64, dtype=BF16), torch.zeros(32, dtype=BF16, requires_grad=True)
    y = m.linear("w", x, bias)
    assert y.requires_grad and y.shape == (2, 3, 32)
    y.backward(torch.ones_like(y))
    assert torch.equal(bias.grad, torch.full((32,), 6, dtype=BF16))
    with torch.no_grad():
        assert not m.linear("w", x, bias).requires_grad
    with pytest.raises(RuntimeError, match="nn.Linear"):
        m.linear("w", x.clone().requires_grad_(), bias)


def test_the_bias_of_a_stack_has_no_gradient(at_launch):
    m = manager_with((4, 32, 64))
    x, ids = torch.zeros(5, 64, dtype=BF16), torch.zeros(5, 2, dtype=torch.int64)
    bias = torch.zeros(4, 32, dtype=BF16, requires_grad=True)
    with pytest.raises(RuntimeError, match="gradient for its bias"):
        m.grouped_linear("w", x, ids, bias)
    with torch.no_grad():
        assert m.grouped_linear("w", x, ids, bias).shape == (5, 2, 32)
    assert m.grouped_linear("w", x, ids, bias.detach()).shape == (5, 2, 32)
