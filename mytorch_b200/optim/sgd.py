"""SGD (``mytorch/optim/sgd.py:6-56``): same constructor, same per-parameter
``state[param]["momentum_buffer"]``.  When every parameter of a group lives on one CUDA device
the whole group is updated by one multi-tensor launch; otherwise (and through the registry's
``sgd`` entry) one launch per parameter, as in the reference.  ``max_grad_norm`` (no counterpart there):
the gradients of all groups together, times ``grad_scale``, are clipped to that norm on their way into the
update, which leaves ``param.grad`` as it is; ``grad_norm`` is then their norm, a tensor of one element on the device."""
from mytorch_b200.backends.backend_dispatcher import BackendDispatcher
from mytorch_b200.optim.optimizer import Optimizer
from mytorch_b200.tensor import Tensor


class SGD(Optimizer):
    def __init__(self, params, lr=0.001, momentum=0, dampening=0, weight_decay=0, nesterov=False, maximize=False, max_grad_norm=None):
        super().__init__(params, dict(lr=lr, momentum=momentum, dampening=dampening, weight_decay=weight_decay,
                                      nesterov=nesterov, maximize=maximize))
        self.grad_scale = 1.0  # set to 1/world_size by the data-parallel wrapper
        if max_grad_norm is not None and not max_grad_norm >= 0:
            raise RuntimeError(f"max_grad_norm is a number from 0 up: {max_grad_norm}")
        self.max_grad_norm = max_grad_norm
        self.grad_norm = None  # of the last step with max_grad_norm

    def step(self):
        dispatcher = BackendDispatcher.instance()
        clipped = []
        if self.max_grad_norm is not None:  # before anything is made for the first step
            devices = {p.device for group in self.param_groups for p in group["params"]}
            if len(devices) != 1 or next(iter(devices)).type != "cuda":
                raise RuntimeError(f"max_grad_norm needs all parameters on one CUDA device: {devices}")
        for group in self.param_groups:
            entries, states = [], self.state
            devices = set()
            for param in group["params"]:
                if param.shape != param.grad.shape:
                    raise RuntimeError(f"Mismatched shape between param and param.grad: {param}, {param.grad}")
                state = states.get(param)
                if state is None:
                    state = states[param] = {}
                buffer = state.get("momentum_buffer")
                first = buffer is None
                if first:
                    buffer = state["momentum_buffer"] = Tensor(shape=param.shape, device=param.device, dtype=param.dtype)
                entries.append((param, buffer, first))
                devices.add(param.device)
            hyper = (group["lr"], group["weight_decay"], group["momentum"], group["dampening"], group["nesterov"], group["maximize"])
            if self.max_grad_norm is not None:
                if entries:
                    clipped.append((entries, *hyper))
            elif len(devices) == 1 and next(iter(devices)).type == "cuda":
                dispatcher.dispatch("cuda", "sgd_multi")(entries, *hyper, self.grad_scale)
            else:
                for param, buf, first in entries:
                    dispatcher.dispatch(param.device.type, "sgd")(param, buf, first, *hyper)
        if clipped:
            self.grad_norm = dispatcher.dispatch("cuda", "sgd_multi_clipped")(clipped, float(self.max_grad_norm), self.grad_scale)
