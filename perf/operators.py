"""Operators around a convolutional network that learns from tokens: group normalisation with an activation (channels last),
embedding lookup with its gradient, the global gradient norm with clipping.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` builds what a program has in hand before
the call, ``run`` is one pass (in plain PyTorch operations, or, where ``own`` is true, by the calls a user of this package makes),
``exact`` the same from the definitions in 64 bits, ``work`` the bytes and operations that a pass cannot do without.  Storage is
float32, images are channels-last ([N, H, W, C] in memory), tokens int32 or int64.
"""
import math
import random

import numpy as np
import torch

own = False
DEVICE = "cuda:0"
EPS = 1e-5  # of the normalisation
LR, MOMENTUM, DECAY = 0.1, 0.9, 5e-4  # of the update
LARGEST_IMAGE = 256 * 128 * 56 * 56  # elements
LARGEST_TOKENS = (131072 + 50000) * 512  # rows of gradient and table, times their width
LARGEST_MODEL = 25557032  # parameters


# ------------------------------------------------------------------------------ which cases

def listed():
    return [
        # classifying one image: the activations are a few KB, the call is latency
        {"name": "gn_forward_one_image", "op": "group_norm", "mode": "forward", "n": 1, "c": 64, "h": 8, "w": 8, "groups": 8, "act": "silu"},
        # the first stage of a small residual network at one rank's batch of 64
        {"name": "gn_forward_64x64x32x32", "op": "group_norm", "mode": "forward", "n": 64, "c": 64, "h": 32, "w": 32, "groups": 32, "act": "relu"},
        # large images and batches: nothing but memory traffic
        {"name": "gn_forward_256x128x56x56", "op": "group_norm", "mode": "forward", "n": 256, "c": 128, "h": 56, "w": 56, "groups": 32, "act": "silu"},
        # channels in groups of ten, an image of odd size: no vector of four stays within a group
        {"name": "gn_backward_30x150x37x41", "op": "group_norm", "mode": "backward", "n": 30, "c": 150, "h": 37, "w": 41, "groups": 15, "act": "silu"},
        # the gradient of the large one
        {"name": "gn_backward_256x128x56x56", "op": "group_norm", "mode": "backward", "n": 256, "c": 128, "h": 56, "w": 56, "groups": 32, "act": "silu"},
        # one new token for each of 8 sequences
        {"name": "embed_8_tokens", "op": "embedding", "mode": "forward", "tokens": 8, "rows": 10000, "width": 256, "index": "int64", "padding": -1},
        # a long batch over a large table
        {"name": "embed_131072_tokens", "op": "embedding", "mode": "forward", "tokens": 131072, "rows": 50000, "width": 512, "index": "int64", "padding": -1},
        # training on 64 sequences of 128 tokens, frequent tokens far more frequent than the rest, one of them padding; ragged sizes
        {"name": "embed_grad_8191_tokens", "op": "embedding", "mode": "backward", "tokens": 8191, "rows": 10007, "width": 300, "index": "int32", "padding": 0},
        # the gradient of the long batch
        {"name": "embed_grad_131072_tokens", "op": "embedding", "mode": "backward", "tokens": 131072, "rows": 50000, "width": 512, "index": "int64", "padding": -1},
        # a small network's gradients, under the limit as in most steps: twenty tensors of odd sizes packed side by side
        {"name": "clip_20_tensors", "op": "clip", "mode": "in_place", "tensors": 20, "elements": 190001, "align": 1},
        # update with clipping of an 18-layer residual network
        {"name": "clipped_update_62_tensors", "op": "clip", "mode": "update", "tensors": 62, "elements": 11173962, "align": 64},
        # and of a 50-layer one
        {"name": "clipped_update_161_tensors", "op": "clip", "mode": "update", "tensors": 161, "elements": LARGEST_MODEL, "align": 64},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["group_norm", "group_norm", "embedding", "embedding", "clip"])
    if op == "group_norm":
        while True:
            groups, each = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
            case = {"op": op, "mode": rng.choice(["forward", "backward"]), "n": _log_int(rng, 1, 256), "c": groups * each, "h": rng.randint(1, 80),
                    "w": rng.randint(1, 80), "groups": groups, "act": "silu"}
            # behind a ReLU a gradient jumps where a value crosses zero: one bit there is a whole value in the answer
            case["act"] = rng.choice(["none", "silu"] + (["relu"] if case["mode"] == "forward" else []))
            # of a group of two or three values nothing but rounding is left in the gradient
            if 4 <= case["c"] <= 1024 and each * case["h"] * case["w"] >= 16 and case["n"] * case["c"] * case["h"] * case["w"] <= LARGEST_IMAGE // 2:
                return case
    if op == "embedding":
        while True:
            rows = _log_int(rng, 100, 50000)
            case = {"op": op, "mode": rng.choice(["forward", "backward"]), "tokens": _log_int(rng, 1, 131072), "rows": rows, "width": _log_int(rng, 8, 1024),
                    "index": rng.choice(["int32", "int64"]), "padding": rng.choice([-1, -1, rng.randrange(rows)])}
            if case["mode"] == "forward":  # padding is a matter of the gradient
                case["padding"] = -1
            if (case["tokens"] + rows) * case["width"] <= LARGEST_TOKENS:
                return case
    tensors = _log_int(rng, 1, 200)
    return {"op": op, "mode": rng.choice(["in_place", "update"]), "tensors": tensors, "elements": max(40 * tensors, _log_int(rng, 2000, LARGEST_MODEL)),
            "align": rng.choice([1, 64])}


# ------------------------------------------------------------------------------ what a program holds

def prepare(case, seed):
    state = {"case": case}
    g = torch.Generator(DEVICE).manual_seed(seed)

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(*shape, generator=g, device=DEVICE).mul_(std).add_(mean)

    if case["op"] == "group_norm":
        n, c, h, w, groups = (case[k] for k in ("n", "c", "h", "w", "groups"))
        state.update(x=normal(n, h, w, c, mean=0.5, std=2.0), gamma=torch.rand(c, generator=g, device=DEVICE) + 0.5, beta=normal(c, std=0.1))
        if case["mode"] == "backward":  # what forward kept
            var, mean = torch.var_mean(state["x"].view(n, h * w, groups, c // groups).double(), dim=(1, 3), correction=0)
            state.update(dy=normal(n, h, w, c), mean=mean.float(), rstd=(var + EPS).rsqrt().float())
    elif case["op"] == "embedding":
        rows, width, count = case["rows"], case["width"], case["tokens"]
        # the k-th most frequent token comes up about 1/k times as often as the first
        u = torch.rand(count, generator=g, device=DEVICE, dtype=torch.float64)
        rank = (u * math.log(rows + 1)).exp().long().sub_(1).clamp_(0, rows - 1)
        token = torch.randperm(rows, generator=g, device=DEVICE)[rank]
        state.update(tokens=token.to(getattr(torch, case["index"])), scale=math.sqrt(width))
        if case["mode"] == "forward":
            state.update(table=normal(rows, width, std=1 / math.sqrt(width)))
        else:
            state.update(dy=normal(count, width))
    else:
        sizes = _tensor_sizes(case)
        offsets, total = [], 0
        for size in sizes:
            offsets.append(total)
            total += -(-size // case["align"]) * case["align"]
        used = torch.zeros(total, device=DEVICE)
        for at, size in zip(offsets, sizes):
            used[at:at + size] = 1
        state.update(sizes=sizes, offsets=offsets, grads=normal(total, std=1e-2) * used)
        # a limit that a third of the norm reaches, or, in place, one that the norm stays under (a second pass then finds what the first found)
        state.update(max_norm=1e-2 * math.sqrt(case["elements"]) * (3.0 if case["mode"] == "in_place" else 1 / 3))
        if case["mode"] == "update":
            state.update(params=normal(total, std=0.05) * used, momenta=normal(total, std=1e-2) * used)
    return state


def _tensor_sizes(case):
    """Sizes as networks have them: one tensor in three holds nearly all elements (weights), the others a few hundred (vectors)."""
    rng = random.Random(case["tensors"] * 1000003 + case["elements"])
    count, left = case["tensors"], case["elements"]
    small = {k: min(rng.randint(10, 2048), max(1, left // (4 * count))) for k in range(count) if k % 3}
    share = {k: math.exp(rng.uniform(0, 4)) for k in range(count) if k % 3 == 0}
    left -= sum(small.values())
    sizes = [small[k] if k in small else max(1, int(left * share[k] / sum(share.values()))) for k in range(count)]
    sizes[0] += case["elements"] - sum(sizes)
    return sizes


# ------------------------------------------------------------------------------ one pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_plain(state):
    case = state["case"]
    if case["op"] == "group_norm":
        return (_plain_norm if case["mode"] == "forward" else _plain_norm_gradient)(state)
    if case["op"] == "embedding":
        if case["mode"] == "forward":
            return state["table"][state["tokens"]] * state["scale"]
        scaled = state["dy"] * state["scale"]
        if case["padding"] >= 0:
            scaled = scaled * (state["tokens"] != case["padding"]).unsqueeze(1)
        return torch.zeros(case["rows"], case["width"], device=DEVICE).index_add_(0, state["tokens"], scaled)
    grads = state["grads"]
    norm = (grads * grads).sum().sqrt()
    coefficient = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    if case["mode"] == "in_place":
        grads.mul_(coefficient)
        return {"norm": norm.reshape(1), "grads": grads}
    params, momenta = state["params"], state["momenta"]
    step = grads * coefficient + params * DECAY
    momenta.mul_(MOMENTUM).add_(step)
    params.sub_(momenta * LR)
    return {"norm": norm.reshape(1), "params": params, "momenta": momenta}


def _plain_norm(state):
    case, x = state["case"], state["x"]
    n, c, groups = case["n"], case["c"], case["groups"]
    v = x.view(n, -1, groups, c // groups)
    d = v - v.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / ((d * d).mean(dim=(1, 3), keepdim=True) + EPS).sqrt()
    z = (d * rstd).view(n, -1, c) * state["gamma"] + state["beta"]
    if case["act"] == "relu":
        z = z.clamp(min=0)
    elif case["act"] == "silu":
        z = z / (1 + (-z).exp())
    return z.view(x.shape)


def _plain_norm_gradient(state):
    case, x = state["case"], state["x"]
    n, c, groups = case["n"], case["c"], case["groups"]
    of_group = (n, 1, groups, 1)
    rstd = state["rstd"].view(of_group)
    hat = ((x.view(n, -1, groups, c // groups) - state["mean"].view(of_group)) * rstd).view(n, -1, c)
    dz = state["dy"].view(n, -1, c)
    if case["act"] == "silu":
        z = hat * state["gamma"] + state["beta"]
        s = 1 / (1 + (-z).exp())
        dz = dz * (s * (1 + z * (1 - s)))
    weighted = (dz * state["gamma"]).view(n, -1, groups, c // groups)
    grouped = hat.view(weighted.shape)
    dx = rstd * (weighted - weighted.mean(dim=(1, 3), keepdim=True) - grouped * (weighted * grouped).mean(dim=(1, 3), keepdim=True))
    return {"dx": dx.reshape(x.shape), "dgamma": (dz * hat).sum(dim=(0, 1)), "dbeta": dz.sum(dim=(0, 1))}


def _run_own(state):
    import mytorch_b200 as mt
    import mytorch_b200.nn.functional as F
    import mytorch_b200.optim as optim
    from mytorch_b200.backends.backend_dispatcher import BackendDispatcher

    case = state["case"]
    held = state.get("own")
    if held is None:
        held = state["own"] = _tensors_of(state)
    if case["op"] == "group_norm":
        if case["mode"] == "forward":
            with mt.no_grad():
                return _torch(F.group_norm(held["x"], case["groups"], held["gamma"], held["beta"], EPS, _activation(case)), state["x"].shape)
        backward = BackendDispatcher.instance().dispatch("cuda", "group_norm_backward")
        dx, dgamma, dbeta = backward(held["dy"], held["mean"], held["rstd"], held["x"], held["gamma"], held["beta"], case["groups"], _activation(case))
        return {"dx": _torch(dx, state["x"].shape), "dgamma": _torch(dgamma, dgamma.shape), "dbeta": _torch(dbeta, dbeta.shape)}
    if case["op"] == "embedding":
        if case["mode"] == "forward":
            with mt.no_grad():
                out = F.embedding(held["tokens"], held["table"], scale=state["scale"])
            return _torch(out, out.shape)
        backward = BackendDispatcher.instance().dispatch("cuda", "embedding_backward")
        dtable = backward(held["dy"], held["tokens"], held["table"], state["scale"], case["padding"] if case["padding"] >= 0 else None)[0]
        return _torch(dtable, dtable.shape)
    if case["mode"] == "in_place":
        norm = optim.clip_grad_norm_(held["params"], state["max_norm"])
        return {"norm": _torch(norm, (1,)), "grads": state["grads"]}
    held["optimizer"].step()
    return {"norm": _torch(held["optimizer"].grad_norm, (1,)), "params": state["params"], "momenta": state["momenta"]}


def _activation(case):
    return None if case["act"] == "none" else case["act"]


def _tensors_of(state):
    """This package's tensors over the memory that the program holds, and its optimizer."""
    import mytorch_b200 as mt
    from mytorch_b200.backends.cuda.env import CudaEnv, CudaMemoryView
    from mytorch_b200.optim import SGD

    CudaEnv.instance()
    device = mt.Device(DEVICE)

    class Memory:
        def __init__(self, t):
            self.ptr, self.device_index, self.held = t.data_ptr(), t.device.index, t

    def over(t, shape=None, first=0, count=None):
        count = t.numel() if count is None else count
        memory = CudaMemoryView(Memory(t), first * t.element_size(), count * t.element_size(), None)
        return mt.Tensor._on_device(tuple(t.shape) if shape is None else shape, mt.DType.from_name(str(t.dtype).split(".")[1]), device, memory)

    case, held = state["case"], {}
    if case["op"] == "group_norm":
        image = (case["n"], case["c"], case["h"], case["w"])
        return {k: over(state[k], image if k in ("x", "dy") else None) for k in ("x", "gamma", "beta", "dy", "mean", "rstd") if k in state}
    if case["op"] == "embedding":
        held = {k: over(state[k]) for k in ("tokens", "table", "dy") if k in state}
        if "table" not in held:  # the backward asks the table for its shape, not for its values
            held["table"] = mt.Tensor(shape=(case["rows"], case["width"]), dtype=mt.float32, device=DEVICE)
        return held
    held["params"] = []
    for size, first in zip(state["sizes"], state["offsets"]):
        p = over(state["params" if "params" in state else "grads"], (size,), first, size)
        p.requires_grad, p.grad = True, over(state["grads"], (size,), first, size)
        held["params"].append(p)
    if case["mode"] == "update":
        held["optimizer"] = SGD(held["params"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY, max_grad_norm=state["max_norm"])
        for p, size, first in zip(held["params"], state["sizes"], state["offsets"]):
            held["optimizer"].state[p] = {"momentum_buffer": over(state["momenta"], (size,), first, size)}
    return held


def _torch(tensor, shape):
    """A PyTorch view of a result; it keeps the result's memory."""
    from mytorch_b200.parallel import torch_view

    view = torch_view(tensor._native_array, math.prod(shape)).view(shape)
    view._of = tensor
    return view


# ------------------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in prepare(case, seed).items()}
    if case["op"] == "group_norm":
        return _exact_norm(case, s) if case["mode"] == "forward" else _exact_norm_gradient(case, s)
    if case["op"] == "embedding":
        t = s["tokens"].long()
        if case["mode"] == "forward":
            return torch.index_select(s["table"], 0, t).mul_(s["scale"])
        if case["padding"] >= 0:
            kept = t != case["padding"]
            t, s["dy"] = t[kept], s["dy"][kept]
        out = torch.zeros(case["rows"], case["width"], device=DEVICE, dtype=torch.float64)
        return out.index_put_((t,), s["dy"], accumulate=True).mul_(s["scale"])
    norm = torch.linalg.vector_norm(s["grads"])
    factor = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    if case["mode"] == "in_place":
        return {"norm": norm.reshape(1), "grads": s["grads"] * factor}
    momenta = MOMENTUM * s["momenta"] + (factor * s["grads"] + DECAY * s["params"])
    return {"norm": norm.reshape(1), "params": s["params"] - LR * momenta, "momenta": momenta}


def _exact_norm(case, s):
    x = s["x"]
    y = torch.empty_like(x)
    each = case["c"] // case["groups"]
    for i in range(case["groups"]):
        at = slice(i * each, (i + 1) * each)
        var, mean = torch.var_mean(x[..., at], dim=(1, 2, 3), correction=0, keepdim=True)
        y[..., at] = (x[..., at] - mean) * torch.rsqrt(var + EPS) * s["gamma"][at] + s["beta"][at]
    return {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu}[case["act"]](y)


def _exact_norm_gradient(case, s):
    each, m = case["c"] // case["groups"], case["c"] // case["groups"] * case["h"] * case["w"]
    mean, rstd = (s[k].repeat_interleave(each, dim=1)[:, None, None, :] for k in ("mean", "rstd"))
    hat = (s["x"] - mean) * rstd
    dz = s["dy"]
    if case["act"] == "silu":
        z = hat * s["gamma"] + s["beta"]
        sig = torch.sigmoid(z)
        dz = dz * (sig + z * sig * (1 - sig))
    per_channel, with_hat = dz.sum(dim=(1, 2)), (dz * hat).sum(dim=(1, 2))
    a, b = ((t * s["gamma"]).view(case["n"], case["groups"], each).sum(2).repeat_interleave(each, dim=1)[:, None, None, :] / m for t in (per_channel, with_hat))
    return {"dx": (dz * s["gamma"] - a - hat * b) * rstd, "dgamma": with_hat.sum(0), "dbeta": per_channel.sum(0)}


# ------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if case["op"] == "group_norm":
        elements, vectors = case["n"] * case["c"] * case["h"] * case["w"], 2 * 4 * case["c"]
        if case["mode"] == "forward":  # x; y
            return {"bytes": 8 * elements + vectors, "flops": 12 * elements}
        return {"bytes": 12 * elements + 2 * vectors + 8 * case["n"] * case["groups"], "flops": 25 * elements}  # x, dy; dx
    if case["op"] == "embedding":
        count, width = case["tokens"], case["width"]
        index = count * (8 if case["index"] == "int64" else 4)
        if case["mode"] == "forward":  # the distinct rows; one row a token
            k = np.arange(1, case["rows"] + 1, dtype=np.float64)
            distinct = float((1 - (1 - np.log1p(1 / k) / math.log(case["rows"] + 1)) ** count).sum())
            return {"bytes": index + 4 * width * (distinct + count), "flops": count * width}
        return {"bytes": index + 4 * width * (count + case["rows"]), "flops": 2 * count * width}  # a row a token; the table's gradient
    if case["mode"] == "in_place":  # the gradients, which stay as they are
        return {"bytes": 4 * case["elements"], "flops": 2 * case["elements"]}
    return {"bytes": 20 * case["elements"], "flops": 10 * case["elements"]}  # gradients, parameters, momenta; the last two written
