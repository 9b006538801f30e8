"""CompressedAdamW's kernel reads a weight's bits as bf16: every other type is refused, where the optimiser is
made, and at a step whose handle holds another type by then."""
import pytest
import torch

import neuzip
from neuzip_b200.optim import CompressedAdamW
from tests.fakes import cpu_manager


def layer(manager, dtype):
    return neuzip.nn.Linear(manager, torch.nn.Linear(8, 4, bias=False).to(dtype))


class KeepsAnything:
    """A manager whose tensors keep their type, as MX4Manager's fp16 ones do."""

    def __init__(self):
        self.held = {}

    def write(self, tensor, handle=None, operand=None):
        handle = handle or str(len(self.held))
        self.held[handle] = tensor.detach().clone()
        return handle

    def read(self, handle):
        return self.held[handle].clone()


@pytest.mark.parametrize("dtype", (torch.float16, torch.float32))
def test_weights_of_another_type_are_refused(dtype):
    with pytest.raises(TypeError, match="bf16"):
        CompressedAdamW(layer(KeepsAnything(), dtype).parameters())


def test_bf16_weights_are_taken():
    CompressedAdamW(layer(cpu_manager(7), torch.bfloat16).parameters())
    CompressedAdamW(layer(KeepsAnything(), torch.bfloat16).parameters())


def test_a_handle_that_changed_its_type_is_refused_at_the_step(monkeypatch):
    m = KeepsAnything()
    lin = layer(m, torch.bfloat16)
    opt = CompressedAdamW(lin.parameters())
    m.write(m.read(lin._p._handle).half(), lin._p._handle)
    before = m.read(lin._p._handle)
    lin._p._gradient = torch.ones(4, 8, dtype=torch.bfloat16)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: type("S", (), {"cuda_stream": 0})())
    monkeypatch.setattr(opt, "_lib", None)                    # the kernel is not to be reached
    with pytest.raises(TypeError, match="bf16"):
        opt.step()
    assert torch.equal(m.read(lin._p._handle), before)
