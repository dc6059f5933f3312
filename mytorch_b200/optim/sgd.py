"""SGD (``mytorch/optim/sgd.py:6-56``): same constructor, same per-parameter
``state[param]["momentum_buffer"]``.  When every parameter of a group lives on one CUDA device
the whole group is updated by one multi-tensor launch; otherwise (and through the registry's
``sgd`` entry) one launch per parameter, as in the reference.  ``max_grad_norm`` (no counterpart there):
the gradients of all groups together, times ``grad_scale``, are clipped to that norm on their way into the
update, which leaves ``param.grad`` as it is; ``grad_norm`` is then their norm, a tensor of one element on the device.  Every
parameter needs a gradient, with clipping as without."""
from mytorch_b200.backends.backend_dispatcher import BackendDispatcher
from mytorch_b200.dtype import float32
from mytorch_b200.optim.optimizer import Optimizer
from mytorch_b200.tensor import InvalidDataTypeError, Tensor


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
        if self.max_grad_norm is not None:
            self._step_clipped()
            return
        dispatcher = BackendDispatcher.instance()
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
            if len(devices) == 1 and next(iter(devices)).type == "cuda":
                dispatcher.dispatch("cuda", "sgd_multi")(entries, *hyper, self.grad_scale)
            else:
                for param, buf, first in entries:
                    dispatcher.dispatch(param.device.type, "sgd")(param, buf, first, *hyper)

    def _step_clipped(self):
        some = next((p for group in self.param_groups for p in group["params"]), None)
        if some is not None and some.device.type == "cuda":
            self.grad_norm = self._clipped(self.state, [()] * len(self.param_groups))
            if self.grad_norm is not None:
                return
        # the first update of some parameters, or something is wrong: found before anything is made
        devices = {p.device for group in self.param_groups for p in group["params"]}
        if len(devices) != 1 or some.device.type != "cuda":
            raise RuntimeError(f"max_grad_norm needs all parameters on one CUDA device: {devices}")
        first, seen = [], set()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    raise RuntimeError(f"max_grad_norm: there is no gradient of a parameter of shape {p.shape}")
                if p.shape != p.grad.shape or p.grad.device is not p.device:
                    raise RuntimeError(f"Mismatched shape or device between param and param.grad: {p}, {p.grad}")
                if p.dtype is not float32 or p.grad.dtype is not float32:
                    raise InvalidDataTypeError([p.dtype, p.grad.dtype])
            first.append({p for p in group["params"] if self.state.get(p, {}).get("momentum_buffer") is None} - seen)
            seen |= first[-1]
        states = dict(self.state)
        for p in seen:
            states[p] = {**states.get(p, {}), "momentum_buffer": Tensor(shape=p.shape, device=p.device, dtype=p.dtype)}
        self.grad_norm = self._clipped(states, first)
        if self.grad_norm is None:
            raise RuntimeError("a momentum buffer is not of its parameter's shape, dtype or device")
        for p in seen:
            self.state[p] = states[p]

    def _clipped(self, states, first):
        groups = [(g["params"], g["lr"], g["weight_decay"], g["momentum"], g["dampening"], g["nesterov"], g["maximize"], set(fresh))
                  for g, fresh in zip(self.param_groups, first)]
        return BackendDispatcher.instance().dispatch("cuda", "sgd_multi_clipped")(groups, states, float(self.max_grad_norm), self.grad_scale)
