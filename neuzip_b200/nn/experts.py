"""The matrices of a mixture-of-experts layer, held in 4 bits (not in the reference, whose
conversion only knows ``nn.Linear``, neuzip/utils.py:57-68)."""
import torch

from .module import Parameter


class Experts(torch.nn.Module):
    """``weight`` is a stack ``[experts, out_features, in_features]``, ``bias`` ``[experts,
    out_features]`` or None.  ``forward(x, experts)`` multiplies every row by the matrix of its
    expert (`MX4Manager.grouped_linear`): with ``[T, k]`` expert numbers and ``[T, in]`` or
    ``[T, k, in]`` inputs it gives ``[T, k, out]``.  For serving: the weights are frozen and
    inputs that need a gradient are refused."""

    def __init__(self, manager, weight: torch.Tensor, bias=None) -> None:
        super().__init__()
        if not hasattr(manager, "grouped_linear"):
            raise TypeError("Experts needs a manager with grouped_linear (MX4Manager)")
        if weight.dim() != 3:
            raise ValueError(f"weight must be [experts, out, in], got shape {tuple(weight.shape)}")
        self.manager = manager
        self.num_experts, self.out_features, self.in_features = (int(d) for d in weight.shape)
        if bias is not None and tuple(bias.shape) != (self.num_experts, self.out_features):
            raise ValueError(f"bias must be [{self.num_experts}, {self.out_features}], "
                             f"got shape {tuple(bias.shape)}")
        self._p = Parameter(manager, weight.detach(), requires_grad=False)
        if bias is None:
            self.register_parameter("bias", None)
        else:
            self.bias = torch.nn.Parameter(bias.detach(), requires_grad=False)

    @property
    def weight(self) -> Parameter:
        return self._p

    def forward(self, x: torch.Tensor, experts: torch.Tensor) -> torch.Tensor:
        return self.manager.grouped_linear(self._p._handle, x, experts, self.bias)

    def get_extra_state(self):
        return self._p._manager.export_entry(self._p._handle)

    def set_extra_state(self, state):
        if state is None:
            return
        if tuple(state["shape"]) != (self.num_experts, self.out_features, self.in_features):
            raise ValueError(f"checkpoint holds a stack of shape {tuple(state['shape'])}, not "
                             f"{(self.num_experts, self.out_features, self.in_features)}")
        self._p._manager.import_entry(state, self._p._handle)

    def extra_repr(self) -> str:
        return (f"! experts={self.num_experts}, in_features={self.in_features}, "
                f"out_features={self.out_features}, bias={self.bias is not None}")
