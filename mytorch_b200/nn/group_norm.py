"""GroupNorm (no counterpart in the reference): affine weight=1 / bias=0, the same in training and evaluation."""
from mytorch_b200.dtype import float32
from mytorch_b200.nn.functional.group_norm import group_norm
from mytorch_b200.nn.module import Module
from mytorch_b200.nn.parameter import Parameter
from mytorch_b200.tensor import Tensor


class GroupNorm(Module):
    """``activation``: None, "relu" or "silu", in the same pass (see ``functional.group_norm``)."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, activation=None, device="cpu", dtype=float32):
        super().__init__()
        if num_groups < 1 or num_channels % num_groups:
            raise RuntimeError(f"GroupNorm: {num_channels} channels are no {num_groups} groups")
        self.num_groups, self.num_channels, self.eps, self.affine, self.activation = num_groups, num_channels, eps, affine, activation
        for name in ("weight", "bias"):
            self.register_parameter(name, Parameter(Tensor(shape=(num_channels,), dtype=dtype, device=device)) if affine else None)
        self.reset_parameters()

    def reset_parameters(self):
        if self.affine:
            self.weight.fill_(1)
            self.bias.fill_(0)

    def forward(self, x):
        return group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.activation)
