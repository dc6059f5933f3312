"""AdamW (no counterpart in the reference): all parameters of a group in one launch, the step counted on the device, so that a captured update counts on
when it is replayed.  ``state_bits=8`` holds both moments in a byte each.  Every parameter needs a gradient, as in ``SGD``, and occurs
once in its group."""
import ctypes

from mytorch_b200.backends.backend_dispatcher import BackendDispatcher
from mytorch_b200.dtype import float32, int64, uint8
from mytorch_b200.optim.optimizer import Optimizer
from mytorch_b200.tensor import InvalidDataTypeError, Tensor, shape_size

BLOCK = 256  # values in 8 bits that share a scale


class AdamW(Optimizer):
    """m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2, p = p (1 - lr weight_decay) - lr m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps).

    ``max_grad_norm``, ``grad_scale`` and ``grad_norm`` as in ``SGD``.  State of a parameter: ``step`` (an int64 tensor of one element, which the parameters of a group
    share), and ``exp_avg`` and ``exp_avg_sq`` like the parameter.  With ``state_bits=8`` these are ``moments`` and ``scales``: blocks of 256 values in the order of the
    parameter's memory share a scale, a first moment keeps 3 bits behind its leading one and a second one as many over a wider range, rounded at random (by ``seed``, the
    parameter's place, the step and the value's place: the same every time) so that small steps add up; ``moments()`` says what they stand for.  The betas then count
    with 20 bits.  Where a gradient is not finite, its whole block of moments reads NaN from then on, and the block's parameters do after the
    next step.  Like ``lr`` and the betas, ``seed`` is not part of a checkpoint: a resumed run rounds as the first one would have if it is given again."""

    def __init__(self, params, lr=0.001, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, maximize=False, max_grad_norm=None, state_bits=32, seed=0):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, maximize=maximize))
        if state_bits not in (8, 32):
            raise RuntimeError(f"AdamW: state_bits is 8 or 32: {state_bits}")
        if max_grad_norm is not None and not max_grad_norm >= 0:
            raise RuntimeError(f"max_grad_norm is a number from 0 up: {max_grad_norm}")
        for g in self.param_groups:
            if len({id(p) for p in g["params"]}) != len(g["params"]):  # the updates of a group run side by side
                raise RuntimeError("AdamW: a parameter occurs twice in a group")
            if len(g["betas"]) != 2 or not all(0 <= b < 1 for b in g["betas"]) or not all(g[k] >= 0 for k in ("lr", "eps", "weight_decay")):
                raise RuntimeError(f"AdamW: betas are two numbers from 0 to below 1, lr, eps and weight_decay numbers from 0 up: {[g[k] for k in self.defaults]}")
        self.grad_scale = 1.0  # set to 1/world_size by the data-parallel wrapper
        self.max_grad_norm, self.state_bits, self.seed = max_grad_norm, state_bits, seed
        self.grad_norm = None  # of the last step with max_grad_norm

    def step(self):
        for group in self.param_groups:
            for p in group["params"]:
                if p.device.type != "cuda":
                    raise RuntimeError(f"AdamW needs all parameters on one CUDA device, not on {p.device}")
                break
        done = self._update(self.state)
        if done is None:  # the first update of some parameters, or something is wrong
            states = self._with_new_states()
            done = self._update(states)
            if done is None:
                raise RuntimeError(f"AdamW: a parameter's state is not of its size, dtype or device, or not of {self.state_bits} bits")
            self.state.update(states)
        if self.max_grad_norm is not None:
            self.grad_norm = done

    def _update(self, states):
        groups = [(g["params"], g["lr"], *g["betas"], g["eps"], g["weight_decay"], g["maximize"]) for g in self.param_groups]
        limit = None if self.max_grad_norm is None else float(self.max_grad_norm)
        return BackendDispatcher.instance().dispatch("cuda", "adamw_multi")(groups, states, self.state_bits, self.grad_scale, limit, self.seed & 0xFFFFFFFF)

    def _with_new_states(self):
        devices = {p.device for group in self.param_groups for p in group["params"]}
        if len(devices) != 1 or next(iter(devices)).type != "cuda":
            raise RuntimeError(f"AdamW needs all parameters on one CUDA device: {devices}")
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    raise RuntimeError(f"AdamW: there is no gradient of a parameter of shape {p.shape}")
                if p.shape != p.grad.shape or p.grad.device is not p.device:
                    raise RuntimeError(f"Mismatched shape or device between param and param.grad: {p}, {p.grad}")
                if p.dtype is not float32 or p.grad.dtype is not float32:
                    raise InvalidDataTypeError([p.dtype, p.grad.dtype])
        states = {}
        for group in self.param_groups:
            step = None
            for p in group["params"]:
                state = self.state.get(p)
                if not state:
                    if step is None:
                        step = _zeros((1,), int64, p)
                    if self.state_bits == 8:
                        blocks = -(-shape_size(p.shape) // BLOCK)
                        state = {"step": step, "moments": _zeros((blocks, 2 * BLOCK), uint8, p), "scales": _zeros((blocks, 2), uint8, p)}
                    else:
                        state = {"step": step, "exp_avg": _zeros(p.shape, float32, p), "exp_avg_sq": _zeros(p.shape, float32, p)}
                states[p] = state
        return states

    def moments(self, param=None):
        """(first, second moments) as float32 tensors: of one parameter in its shape, or of all, one behind the other in the order of their memory, as vectors."""
        params = [p for g in self.param_groups for p in g["params"]] if param is None else [param]
        if self.state_bits == 8:
            found = BackendDispatcher.instance().dispatch("cuda", "adamw8_moments")(params, self.state)
            if found is None:
                raise RuntimeError("AdamW: a parameter has no moments yet, or they are not of its size or device")
            return found if param is None else tuple(Tensor._on_device(param.shape, float32, param.device, t._native_array) for t in found)
        if any(not self.state.get(p) for p in params):
            raise RuntimeError("AdamW: a parameter has no moments yet")
        held = [[self.state[p][name] for p in params] for name in ("exp_avg", "exp_avg_sq")]
        return tuple(h[0] for h in held) if param is not None else tuple(_side_by_side(h) for h in held)


def _zeros(shape, dtype, like):
    from mytorch_b200.backends.cuda.env import CudaEnv

    env = CudaEnv.instance()
    if env.capturing():
        raise RuntimeError("optimizer state does not exist yet: run one eager optimizer step before capturing the step in a CUDA graph")
    t = Tensor(shape=shape, dtype=dtype, device=like.device)
    env.lib.memset_async(t, 0, shape_size(shape) * dtype.itemsize(), env.stream())
    return t


def _side_by_side(tensors):
    from mytorch_b200.backends.cuda.env import CudaEnv

    env, sizes = CudaEnv.instance(), [shape_size(t.shape) for t in tensors]
    out = Tensor(shape=(sum(sizes),), dtype=float32, device=tensors[0].device)
    count, offsets = len(sizes), [sum(sizes[:i]) for i in range(len(sizes))]
    env.lib.pack_scale_f32(count, (ctypes.c_void_p * count)(*[t._native_array.ptr for t in tensors]), (ctypes.c_longlong * count)(*offsets),
                           (ctypes.c_longlong * count)(*sizes), out, 1.0, env.stream())
    return out
