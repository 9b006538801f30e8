"""The autograd function of the compressed Linear where inputs and weight have different types."""
import pytest
import torch

from neuzip_b200.ops import CompressedLinear


class Weight(torch.nn.Parameter):
    """A parameter whose product takes any type, as one on 4-bit storage does."""

    def __new__(cls, w):
        self = super().__new__(cls, torch.zeros(0, dtype=w.dtype), True)
        self.w, self._gradient = w, None
        return self

    def __call__(self):
        return self.w

    def linear(self, inputs, bias=None):
        return (inputs.float() @ self.w.float().t()).to(inputs.dtype)


@pytest.mark.parametrize("x_type,w_type", [(torch.float16, torch.bfloat16), (torch.bfloat16, torch.float16)])
def test_gradients_have_the_inputs_type(x_type, w_type):
    g = torch.Generator().manual_seed(1)
    # whole numbers: every product and sum is exact
    w, x, up = (torch.randint(-3, 4, s, generator=g) for s in ((5, 8), (2, 3, 8), (2, 3, 5)))
    p, xd = Weight(w.to(w_type)), x.to(x_type).requires_grad_()
    CompressedLinear.apply(xd, p, None).backward(up.to(x_type))
    assert xd.grad.dtype == x_type and torch.equal(xd.grad.long(), up @ w)
    assert p._gradient.dtype == x_type
    assert torch.equal(p._gradient.long(), up.reshape(6, 5).t() @ x.reshape(6, 8))


def test_a_weight_beyond_the_range_of_the_inputs_type():
    p, x = Weight(torch.full((2, 4), 2.0 ** 20, dtype=torch.bfloat16)), torch.zeros(1, 4, dtype=torch.float16)
    x.requires_grad_()
    CompressedLinear.apply(x, p, None).backward(torch.full((1, 2), 2.0 ** -12, dtype=torch.float16))
    assert torch.equal(x.grad, torch.full((1, 4), 512.0, dtype=torch.float16))
