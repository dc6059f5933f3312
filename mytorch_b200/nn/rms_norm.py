"""RMSNorm, and the norms around a residual block with its gate (no counterpart in the reference); the same in training and evaluation."""
from mytorch_b200.dtype import float32
from mytorch_b200.nn.functional.rms_norm import add_rms_norm, rms_norm
from mytorch_b200.nn.module import Module
from mytorch_b200.nn.parameter import Parameter
from mytorch_b200.tensor import Tensor


class RMSNorm(Module):
    """``functional.rms_norm`` with a weight of ones (``affine``)."""

    def __init__(self, num_channels, eps=1e-6, affine=True, device="cpu", dtype=float32):
        super().__init__()
        self.num_channels, self.eps = num_channels, eps
        self.register_parameter("weight", Parameter(Tensor(shape=(num_channels,), dtype=dtype, device=device)) if affine else None)
        self.reset_parameters()

    def reset_parameters(self):
        if self.weight is not None:
            self.weight.fill_(1)

    def forward(self, x):
        return rms_norm(x, self.weight, self.eps)


class AddRMSNorm(Module):
    """``functional.add_rms_norm``: (residual, block) -> (new residual, its norm).  ``post_norm``: the block is normed first; ``gate``: what the gate, one value a
    channel, begins with (None: there is none, though one may be given to the call); ``scale`` that of the residual."""

    def __init__(self, num_channels, eps=1e-6, post_norm=True, gate=None, scale=1.0, device="cpu", dtype=float32):
        super().__init__()
        self.num_channels, self.eps, self.scale, self.first_gate = num_channels, eps, scale, gate
        for name, there in (("weight", True), ("post_weight", post_norm), ("gate", gate is not None)):
            self.register_parameter(name, Parameter(Tensor(shape=(num_channels,), dtype=dtype, device=device)) if there else None)
        self.reset_parameters()

    def reset_parameters(self):
        for t, value in ((self.weight, 1), (self.post_weight, 1), (self.gate, self.first_gate)):
            if t is not None:
                t.fill_(value)

    def forward(self, residual, block, gate=None):
        if gate is not None and self.gate is not None:
            raise RuntimeError("AddRMSNorm: a gate of its own and another one")
        return add_rms_norm(residual, block, self.weight, self.post_weight, self.gate if gate is None else gate, self.scale, self.eps)
