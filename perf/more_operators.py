"""Operators of a model that learns and answers with tokens: log probabilities of given tokens with entropy and top alternatives, the norms around a
residual block with its gate, AdamW over many tensors with states in 32 or in 8 bits.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` builds what a program has in hand before
the call, ``run`` is one pass (in plain PyTorch operations, or, where ``own`` is true, by the calls a user of this package makes),
``exact`` the same from the definitions in 64 bits, ``work`` the bytes and operations that a pass cannot do without.  Storage is
float32, tokens int32 or int64.  Moments in 8 bits come back as the values that they stand for.
"""
import math
import random

import torch

own = False
DEVICE = "cuda:0"
EPS = 1e-6  # of the norms
IGNORED = -100  # a row without a token
LR, BETAS, ADAM_EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.01
SEED = 7  # of the roundings to 8 bits
BLOCK = 256  # values that share a scale
LARGEST_LOGITS = 4096 * 50000
LARGEST_ROWS = 32768 * 1024
LARGEST_MODEL = 25557032  # parameters


# ------------------------------------------------------------------------------ which cases

def listed():
    return [
        # what one new token could have been: the row is read by the whole card, the call is latency
        {"name": "log_probs_one_row", "op": "log_probs", "mode": "forward", "n": 1, "v": 50000, "top": 20, "index": "int64", "masked": False, "ignored": False},
        # a batch under a grammar that forbids two tokens in three, sequences of unequal length padded; ragged sizes
        {"name": "log_probs_509x10007", "op": "log_probs", "mode": "forward", "n": 509, "v": 10007, "top": 5, "index": "int32", "masked": True, "ignored": True},
        # scoring a long batch over a large table
        {"name": "log_probs_4096x50000", "op": "log_probs", "mode": "forward", "n": 4096, "v": 50000, "top": 8, "index": "int64", "masked": False, "ignored": False},
        # the gradient of that batch through log probabilities, entropies and alternatives
        {"name": "log_probs_grad_4096x50000", "op": "log_probs", "mode": "backward", "n": 4096, "v": 50000, "top": 8, "index": "int64", "masked": False, "ignored": False},
        # between two blocks, for one new token
        {"name": "norms_one_row", "op": "norms", "mode": "forward", "batch": 1, "positions": 1, "c": 1024, "post": True, "gate": "channel", "scale": 1.0},
        # a long batch, gated by sample
        {"name": "norms_32768x1024", "op": "norms", "mode": "forward", "batch": 64, "positions": 512, "c": 1024, "post": True, "gate": "sample", "scale": 1.0},
        # the gradient where no vector of four fits a row
        {"name": "norms_grad_1110x750", "op": "norms", "mode": "backward", "batch": 30, "positions": 37, "c": 750, "post": False, "gate": "channel", "scale": 0.5},
        # the gradient of a long batch, gated by channel
        {"name": "norms_grad_32768x1024", "op": "norms", "mode": "backward", "batch": 64, "positions": 512, "c": 1024, "post": True, "gate": "channel", "scale": 1.0},
        # a small network: twenty tensors of odd sizes packed side by side
        {"name": "adamw_20_tensors", "op": "adamw", "bits": 32, "tensors": 20, "elements": 190001, "align": 1, "clip": True},
        # an 18-layer residual network
        {"name": "adamw_62_tensors", "op": "adamw", "bits": 32, "tensors": 62, "elements": 11173962, "align": 64, "clip": True},
        # the small one with its states in 8 bits
        {"name": "adamw8_20_tensors", "op": "adamw", "bits": 8, "tensors": 20, "elements": 190001, "align": 1, "clip": False},
        # a 50-layer residual network, states in 8 bits
        {"name": "adamw8_161_tensors", "op": "adamw", "bits": 8, "tensors": 161, "elements": LARGEST_MODEL, "align": 64, "clip": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["log_probs", "log_probs", "norms", "norms", "adamw", "adamw"])
    if op == "log_probs":
        while True:
            case = {"op": op, "mode": rng.choice(["forward", "backward"]), "n": _log_int(rng, 1, 16384), "v": _log_int(rng, 8, 200000), "top": rng.choice([0, 1, rng.randint(2, 32)]),
                    "index": rng.choice(["int32", "int64"]), "masked": rng.random() < 0.3, "ignored": rng.random() < 0.3}
            case["top"] = min(case["top"], case["v"])
            if case["n"] * case["v"] <= LARGEST_LOGITS // 2 and (case["n"] >= 4 or not case["ignored"]):
                return case
    if op == "norms":
        while True:
            case = {"op": op, "mode": rng.choice(["forward", "backward"]), "batch": _log_int(rng, 1, 256), "positions": _log_int(rng, 1, 4096), "c": _log_int(rng, 8, 8192),
                    "post": rng.random() < 0.5, "gate": rng.choice(["none", "channel", "sample", "full"]), "scale": rng.choice([1.0, 0.5, math.sqrt(0.5)])}
            if case["batch"] * case["positions"] * case["c"] <= LARGEST_ROWS // 2:
                return case
    tensors = _log_int(rng, 1, 200)
    return {"op": op, "bits": rng.choice([32, 8]), "tensors": tensors, "elements": max(40 * tensors, _log_int(rng, 2000, LARGEST_MODEL)), "align": rng.choice([1, 64]),
            "clip": rng.random() < 0.5}


# ------------------------------------------------------------------------------ what a program holds

def prepare(case, seed):
    state = {"case": case}
    g = torch.Generator(DEVICE).manual_seed(seed)

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(*shape, generator=g, device=DEVICE).mul_(std).add_(mean)

    if case["op"] == "log_probs":
        n, v = case["n"], case["v"]
        state["logits"] = normal(n, v, std=2.0)
        if case["masked"]:
            state["logits"].masked_fill_(torch.rand(n, v, generator=g, device=DEVICE) < 0.67, -math.inf)
            state["logits"][:, v // 2] = 0.25  # something is allowed in every row
        tokens = (torch.rand(n, generator=g, device=DEVICE) * v).long().clamp_(max=v - 1)
        if case["masked"]:
            tokens[:] = v // 2
        if case["ignored"]:
            tokens[torch.arange(n, device=DEVICE) % 4 == 3] = IGNORED
        state["tokens"] = tokens.to(getattr(torch, case["index"]))
        if case["mode"] == "backward":  # what forward kept
            z = state["logits"].double()
            top = z.max(dim=1, keepdim=True)[0]
            d = (z - top).clamp_(min=-1e30)
            e = d.exp()
            total = e.sum(dim=1, keepdim=True)
            entropy = total.log() - (e * d).sum(dim=1, keepdim=True) / total
            state["stats"] = torch.cat([top, total, entropy], dim=1).float()
            del z, d, e
            state.update(dlog_probs=normal(n), dentropy=normal(n, std=0.1), dtop=normal(n, case["top"], std=0.1))
            # the alternatives: in earnest the largest; any distinct tokens do for the gradient
            first = (torch.rand(n, 1, generator=g, device=DEVICE) * v).long().clamp_(max=v - 1)
            state["top_tokens"] = (first + torch.arange(case["top"], device=DEVICE) * max(1, v // max(1, case["top"]))) % v
    elif case["op"] == "norms":
        shape, c = (case["batch"], case["positions"], case["c"]), case["c"]
        state.update(residual=normal(*shape, std=2.0), block=normal(*shape, std=0.5), weight=normal(c, mean=1.0, std=0.2))
        if case["post"]:
            state["post_weight"] = normal(c, mean=1.0, std=0.2)
        if case["gate"] != "none":
            state["gate"] = normal(*{"channel": (c,), "sample": (case["batch"], c), "full": shape}[case["gate"]], std=0.5)
        if case["mode"] == "backward":  # what forward kept
            state["new"] = state.pop("residual")
            state["rstd"] = (state["new"].double().square().mean(dim=2) + EPS).rsqrt().float()
            if case["post"]:
                state["block_rstd"] = (state["block"].double().square().mean(dim=2) + EPS).rsqrt().float()
            state.update(dnew=normal(*shape), dy=normal(*shape))
    else:
        sizes = _tensor_sizes(case)
        offsets, blocks, total, count = [], [], 0, 0
        for size in sizes:
            offsets.append(total)
            blocks.append(count)
            total += -(-size // case["align"]) * case["align"]
            count += -(-size // BLOCK)
        sized = torch.tensor(sizes, device=DEVICE)
        tensor = torch.repeat_interleave(torch.arange(len(sizes), device=DEVICE), sized, output_size=case["elements"])
        within = torch.arange(case["elements"], device=DEVICE) - (sized.cumsum(0) - sized)[tensor]
        at = torch.tensor(offsets, device=DEVICE)[tensor] + within  # where in the flat buffers an element lies
        state.update(sizes=sizes, offsets=offsets, blocks=blocks, at=at, step=torch.full((1,), 100, dtype=torch.int64, device=DEVICE))

        def spread(values):
            out = torch.zeros(total, device=DEVICE)
            out[at] = values
            return out

        # gradients of unequal size from element to element, moments as they are after many of them
        size = 1e-3 * normal(case["elements"]).exp()
        state.update(params=spread(normal(case["elements"], std=0.05)), grads=spread(size * normal(case["elements"])))
        m, v = 0.23 * size * normal(case["elements"]), size.square() * (0.9 + 0.2 * torch.rand(case["elements"], generator=g, device=DEVICE))
        # a limit that a third of the norm reaches
        state["max_norm"] = 1e-3 * math.e * math.sqrt(case["elements"]) / 3 if case["clip"] else None
        if case["bits"] == 32:
            state.update(exp_avg=spread(m), exp_avg_sq=spread(v))
        else:
            state.update(tensor=tensor, within=within, slot=torch.tensor(blocks, device=DEVICE)[tensor] * BLOCK + within, count=count)
            state["moments"] = torch.zeros(count, 2 * BLOCK, dtype=torch.uint8, device=DEVICE)
            state["scales"] = torch.zeros(count, 2, dtype=torch.uint8, device=DEVICE)
            random16 = torch.full((2, case["elements"]), 1 << 15, device=DEVICE)
            for k, (values, fields, low) in enumerate(((m, 15, 0), (v, 31, 1))):
                _plain_encode(state, k, values, fields, low, random16[k])
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
    if case["op"] == "log_probs":
        return (_plain_log_probs if case["mode"] == "forward" else _plain_log_probs_gradient)(state)
    if case["op"] == "norms":
        return (_plain_norms if case["mode"] == "forward" else _plain_norms_gradient)(state)
    return _plain_adamw(state)


def _plain_log_probs(state):
    case, z, tokens = state["case"], state["logits"], state["tokens"].long()
    d = z - z.max(dim=1, keepdim=True)[0]
    e = d.exp()
    total = e.sum(dim=1)
    log_total = total.log()
    entropy = log_total - torch.where(e > 0, e * d, 0.0).sum(dim=1) / total
    known = tokens != IGNORED
    given = d.gather(1, torch.where(known, tokens, 0)[:, None])[:, 0] - log_total
    out = {"log_probs": torch.where(known, given, 0.0), "entropy": entropy}
    if case["top"]:
        # one whole number for value and place: in the order of the values, and of equal ones the first place is the largest
        bits = (z + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * (1 << 32) + (0xFFFFFFFF - torch.arange(case["v"], device=z.device))
        best = torch.topk(key, case["top"], dim=1)[0]
        out["top_tokens"] = 0xFFFFFFFF - (best & 0xFFFFFFFF)
        out["top_log_probs"] = d.gather(1, out["top_tokens"]) - log_total[:, None]
    return out


def _plain_log_probs_gradient(state):
    case, z, tokens = state["case"], state["logits"], state["tokens"].long()
    top, total, entropy = state["stats"].split(1, dim=1)
    d = z - top
    p = d.exp() / total
    known = tokens != IGNORED
    of_token = torch.where(known, state["dlog_probs"], 0.0)[:, None]
    dz = -p * (of_token + state["dtop"].sum(dim=1, keepdim=True)) - torch.where(p > 0, p * (d - total.log() + entropy), 0.0) * state["dentropy"][:, None]
    dz.scatter_add_(1, torch.where(known, tokens, 0)[:, None], of_token)
    return dz.scatter_add_(1, state["top_tokens"], state["dtop"])


def _plain_norms(state):
    case, n = state["case"], state["block"]
    if case["post"]:
        n = n / (n.square().mean(dim=2, keepdim=True) + EPS).sqrt() * state["post_weight"]
    if case["gate"] != "none":
        n = n * _spread_gate(state)
    new = state["residual"] * case["scale"] + n
    return {"new": new, "y": new / (new.square().mean(dim=2, keepdim=True) + EPS).sqrt() * state["weight"]}


def _spread_gate(state):
    gate = state["gate"]
    return gate[:, None, :] if state["case"]["gate"] == "sample" else gate


def _plain_norms_gradient(state):
    case, dy, rstd = state["case"], state["dy"], state["rstd"][:, :, None]
    hat = state["new"] * rstd
    u = dy * state["weight"]
    total = state["dnew"] + rstd * (u - hat * (u * hat).mean(dim=2, keepdim=True))
    out = {"dresidual": total * case["scale"], "dweight": (dy * hat).sum(dim=(0, 1))}
    normed = block_hat = state["block"]
    if case["post"]:
        block_hat = block_hat * state["block_rstd"][:, :, None]
        normed = block_hat * state["post_weight"]
    dn = total
    if case["gate"] != "none":
        dgate = total * normed
        out["dgate"] = {"channel": lambda: dgate.sum(dim=(0, 1)), "sample": lambda: dgate.sum(dim=1), "full": lambda: dgate}[case["gate"]]()
        dn = total * _spread_gate(state)
    if case["post"]:
        out["dpost_weight"] = (dn * block_hat).sum(dim=(0, 1))
        t = dn * state["post_weight"]
        dn = state["block_rstd"][:, :, None] * (t - block_hat * (t * block_hat).mean(dim=2, keepdim=True))
    out["dblock"] = dn
    return out


def _plain_adamw(state):
    """In 64 bits: a value in 8 bits is a whole step off where the value before rounding is one bit off."""
    case, at = state["case"], state["at"]
    b1, b2 = _betas(case)
    state["step"] += 1
    t = state["step"].double()
    g = state["grads"][at]
    out = {}
    if case["clip"]:
        norm = g.double().square().sum().sqrt()
        g = g * (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
        out["norm"] = norm.float().reshape(1)
    g64 = g.double()
    if case["bits"] == 32:
        m = b1 * state["exp_avg"][at].double() + (1 - b1) * g64
        v = b2 * state["exp_avg_sq"][at].double() + (1 - b2) * g64 * g64
        state["exp_avg"][at], state["exp_avg_sq"][at] = m.float(), v.float()
        out.update(exp_avg=state["exp_avg"], exp_avg_sq=state["exp_avg_sq"])
    else:
        h = (g * _f32(math.sqrt(1 - b2))).double()
        m = (b1 * _plain_decode(state, 0) + (1 - b1) * g64).float().double()
        v = (b2 * _plain_decode(state, 1) + h * h).float().double()
        r = _plain_random(state)
        _plain_encode(state, 0, m, 15, 0, r >> 16)
        _plain_encode(state, 1, v, 31, 1, r & 0xFFFF)
        out.update(exp_avg=_plain_decode(state, 0).float(), exp_avg_sq=_plain_decode(state, 1).float())
    params = state["params"][at].double()
    state["params"][at] = (params * (1 - LR * DECAY) - LR / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + ADAM_EPS)).float()
    out["params"] = state["params"]
    return out


def _betas(case):
    """For states in 8 bits of 20 bits: their product with a state then fits a float32."""
    return tuple(round(b * (1 << 20)) / (1 << 20) for b in BETAS) if case["bits"] == 8 else BETAS


def _f32(value):
    return torch.tensor(value, dtype=torch.float32).item()


def _mix(x):
    """32 bits to 32 bits, each of which depends on all."""
    x = (x ^ (x >> 16)) * 0x6A09E667 & 0xFFFFFFFF
    x = (x ^ (x >> 15)) * 0xBB67AE85 & 0xFFFFFFFF
    return x ^ (x >> 16)


def _plain_random(state):
    """32 bits for each element, by seed, tensor, step and place."""
    of_tensor = _mix((SEED + 0x9E3779B1 * (torch.arange(len(state["sizes"]), device=DEVICE) + 1)) & 0xFFFFFFFF)
    key = _mix((of_tensor + state["step"]) & 0xFFFFFFFF)
    return _mix((key[state["tensor"]] + state["within"] * 0x9E3779B1) & 0xFFFFFFFF)


def _plain_decode(state, k):
    """The first or second moments, in 64 bits.  A code is the exponent and three bits of a float; its block's scale says what the largest exponent stands for."""
    code = state["moments"][:, k * BLOCK:(k + 1) * BLOCK].reshape(-1)[state["slot"]].long()
    scale = state["scales"][:, k][state["slot"] // BLOCK].double()
    sign = torch.where(code >= 128, -1.0, 1.0).double() if k == 0 else 1.0
    code, highest = (code & 127, 15) if k == 0 else (code, 31)
    e, f = code >> 3, (code & 7).double()
    value = torch.where(e > 0, f + 8, f) * torch.exp2((e.clamp(min=1) - highest + 1 - 3).double() + scale - 127)
    return torch.where(scale > 0, sign * value, 0.0)


def _plain_encode(state, k, values, highest, low, random16):
    """Rounds to a neighbouring code, up as often as the value is near the upper one; what is not zero stays at least `low`."""
    x = torch.zeros(state["count"] * BLOCK, dtype=torch.float64, device=DEVICE)
    x[state["slot"]] = values.double()
    x = x.view(-1, BLOCK)
    r = torch.zeros(state["count"] * BLOCK, dtype=torch.int64, device=DEVICE)
    r[state["slot"]] = random16
    largest = x.abs().max(dim=1)[0]
    scale = torch.where(largest > 0, (torch.frexp(largest)[1] + 126).clamp(min=1), 0)
    # the exponent `highest` for twice the largest value's, and everything under exponent 1 in equal steps, as in a float32
    y = (x.abs() * torch.exp2((127 - scale).double())[:, None] * 2.0 ** (highest - 128)).float().view(torch.int32).long()
    code = (y + r.view(-1, BLOCK) * 16 + 8) >> 20
    code = torch.where(x == 0, 0, code.clamp(min=low))
    if k == 0:
        code = code + torch.where(x < 0, 128, 0)
    state["moments"][:, k * BLOCK:(k + 1) * BLOCK] = code.to(torch.uint8)
    state["scales"][:, k] = scale.to(torch.uint8)


def _run_own(state):
    import mytorch_b200 as mt
    import mytorch_b200.nn.functional as F
    from mytorch_b200.backends.backend_dispatcher import BackendDispatcher

    case = state["case"]
    held = state.get("own")
    if held is None:
        held = state["own"] = _tensors_of(state)
    if case["op"] == "log_probs":
        if case["mode"] == "forward":
            with mt.no_grad():
                got = F.token_log_probs(held["logits"], held["tokens"], top=case["top"], ignore_index=IGNORED)
            return {k: _torch(v) for k, v in got._asdict().items() if v is not None}
        backward = BackendDispatcher.instance().dispatch("cuda", "token_log_probs_backward")
        grads = [held[k] for k in ("dlog_probs", "dentropy")] + [held["dtop"] if case["top"] else None]
        return _torch(backward(*grads, held["stats"], held["top_tokens"] if case["top"] else None, held["logits"], held["tokens"], IGNORED)[0])
    if case["op"] == "norms":
        weights = [held.get(k) for k in ("weight", "post_weight", "gate")]
        if case["mode"] == "forward":
            with mt.no_grad():
                new, y = F.add_rms_norm(held["residual"], held["block"], *weights, scale=case["scale"], eps=EPS)
            return {"new": _torch(new), "y": _torch(y)}
        backward = BackendDispatcher.instance().dispatch("cuda", "add_rms_norm_backward")
        got = backward(held["dnew"], held["dy"], held["new"], held["rstd"], held.get("block_rstd"), held["new"], held["block"], *weights, case["scale"])
        return {k: _torch(t) for k, t in zip(("dresidual", "dblock", "dweight", "dpost_weight", "dgate"), got) if t is not None}
    optimizer = held["optimizer"]
    optimizer.step()
    out = {"params": state["params"]}
    if case["clip"]:
        out["norm"] = _torch(optimizer.grad_norm)
    if case["bits"] == 32:
        out.update(exp_avg=state["exp_avg"], exp_avg_sq=state["exp_avg_sq"])
    else:
        out.update(zip(("exp_avg", "exp_avg_sq"), map(_torch, optimizer.moments())))
    return out


def _tensors_of(state):
    """This package's tensors over the memory that the program holds, and its optimizer."""
    import mytorch_b200 as mt
    from mytorch_b200.backends.cuda.env import CudaEnv, CudaMemoryView
    from mytorch_b200.optim import AdamW

    CudaEnv.instance()
    device = mt.Device(DEVICE)

    class Memory:
        def __init__(self, t):
            self.ptr, self.device_index, self.held = t.data_ptr(), t.device.index, t

    def over(t, shape=None, first=0):
        shape = tuple(t.shape) if shape is None else shape
        memory = CudaMemoryView(Memory(t), first * t.element_size(), math.prod(shape) * t.element_size(), None)
        return mt.Tensor._on_device(shape, mt.DType.from_name(str(t.dtype).split(".")[1]), device, memory)

    case = state["case"]
    if case["op"] != "adamw":
        return {k: over(t) for k, t in state.items() if isinstance(t, torch.Tensor) and t.numel() and (t.dim() < 4)}
    params, states, step = [], {}, over(state["step"])
    for size, first, block in zip(state["sizes"], state["offsets"], state["blocks"]):
        p = over(state["params"], (size,), first)
        p.requires_grad, p.grad = True, over(state["grads"], (size,), first)
        params.append(p)
        if case["bits"] == 32:
            states[p] = {"step": step, **{k: over(state[k], (size,), first) for k in ("exp_avg", "exp_avg_sq")}}
        else:
            count = -(-size // BLOCK)
            states[p] = {"step": step, "moments": over(state["moments"], (count, 2 * BLOCK), block * 2 * BLOCK), "scales": over(state["scales"], (count, 2), block * 2)}
    optimizer = AdamW(params, lr=LR, betas=BETAS, eps=ADAM_EPS, weight_decay=DECAY, max_grad_norm=state["max_norm"], state_bits=case["bits"], seed=SEED)
    optimizer.state.update(states)
    return {"optimizer": optimizer}


def _torch(tensor):
    """A PyTorch view of a result; it keeps the result's memory."""
    memory = tensor._native_array

    class Values:
        __cuda_array_interface__ = {"shape": tuple(tensor.shape), "typestr": {"float32": "<f4", "int64": "<i8"}[tensor.dtype.name], "data": (memory.ptr, False), "version": 3}

    view = torch.as_tensor(Values(), device=DEVICE)
    view._of = tensor
    return view


# ------------------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(case, s)
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    if case["op"] == "norms":
        return _exact_norms(case, s) if case["mode"] == "forward" else _exact_norms_gradient(case, s)
    log_p = torch.log_softmax(s["logits"], dim=1)
    p = log_p.exp()
    rows = torch.arange(case["n"], device=DEVICE)
    tokens = s["tokens"].long()
    known = tokens != IGNORED
    entropy = -torch.special.xlogy(p, p).sum(dim=1)
    if case["mode"] == "forward":
        out = {"log_probs": torch.where(known, log_p[rows, tokens.clamp(min=0)], 0.0), "entropy": entropy}
        if case["top"]:
            out.update(top_tokens=None, top_log_probs=log_p.sort(dim=1, descending=True)[0][:, :case["top"]].clone())
        return out
    # d log p_t / d z_j = [j = t] - p_j, d entropy / d z_j = -p_j (log p_j + entropy)
    dz = -s["dentropy"][:, None] * (torch.special.xlogy(p, p) + p * entropy[:, None])
    for t, d in [(tokens.clamp(min=0), s["dlog_probs"] * known)] + [(s["top_tokens"][:, k], s["dtop"][:, k]) for k in range(case["top"])]:
        dz[rows, t] += d
    return dz.sub_(p * (s["dlog_probs"] * known + s["dtop"].sum(dim=1))[:, None])


def _exact_norms(case, s):
    inner = s["block"]
    if case["post"]:
        inner = inner * torch.rsqrt((inner * inner).sum(-1, keepdim=True) / case["c"] + EPS) * s["post_weight"]
    if case["gate"] != "none":
        inner = inner * (s["gate"].unsqueeze(1) if case["gate"] == "sample" else s["gate"])
    new = case["scale"] * s["residual"] + inner
    # what follows sees the sum as it is stored
    return {"new": new, "y": new * torch.rsqrt((new * new).sum(-1, keepdim=True) / case["c"] + EPS) * s["weight"]}


def _exact_norms_gradient(case, s):
    """By autograd on the formulas, where the statistics are functions of the values."""
    with torch.enable_grad():
        new = s["new"].requires_grad_()
        y = new * torch.rsqrt(new.pow(2).mean(-1, keepdim=True) + EPS) * s["weight"].requires_grad_()
        dnew, dweight = torch.autograd.grad(y, (new, s["weight"]), s["dy"])
        dnew = dnew + s["dnew"]
        inner = s["block"].requires_grad_()
        wanted = {"dblock": inner}
        if case["post"]:
            wanted["dpost_weight"] = s["post_weight"].requires_grad_()
            inner = inner * torch.rsqrt(inner.pow(2).mean(-1, keepdim=True) + EPS) * s["post_weight"]
        if case["gate"] != "none":
            wanted["dgate"] = s["gate"].requires_grad_()
            inner = inner * (s["gate"].unsqueeze(1) if case["gate"] == "sample" else s["gate"])
        inner = inner * 1.0
        grads = torch.autograd.grad(inner, list(wanted.values()), dnew)
    return {"dresidual": case["scale"] * dnew, "dweight": dweight, **dict(zip(wanted, grads))}


def _exact_adamw(case, s):
    at = s["at"]
    t = int(s["step"]) + 1
    (b1, b2), g = _betas(case), s["grads"][at].double()
    out = {}
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        factor = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
        # with states in 8 bits the factor and the gradient that the moments see are float32 by definition
        g = (g.float() * _f32(factor)).double() if case["bits"] == 8 else g * factor
        out["norm"] = norm.reshape(1)
    if case["bits"] == 32:
        m, v = torch.lerp(g, s["exp_avg"][at].double(), b1), torch.lerp(g * g, s["exp_avg_sq"][at].double(), b2)
        for name, x in (("exp_avg", m), ("exp_avg_sq", v)):
            out[name] = torch.zeros_like(s[name], dtype=torch.float64).index_put_((at,), x)
    else:
        old = [_exact_decode(s, k) for k in range(2)]
        m = (old[0] * b1 + g * (1 - b1)).float().double()
        v = (old[1] * b2 + (g.float() * _f32(math.sqrt(1 - b2))).double().square()).float().double()
        s["step"] += 1
        bits = _plain_random(s)  # random numbers are given
        out["exp_avg"] = _exact_round(s, m, 13, (bits >> 16) * 16 + 8)
        out["exp_avg_sq"] = _exact_round(s, v, 29, (bits & 0xFFFF) * 16 + 8, True)
    step = LR * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + ADAM_EPS)
    new = s["params"][at].double() * (1 - LR * DECAY) - step
    out["params"] = torch.zeros_like(s["params"], dtype=torch.float64).index_put_((at,), new)
    return out


def _exact_decode(s, k):
    """By a table of what the codes stand for, relative to a scale of 1."""
    if k == 0:
        table = [(1 - 2 * (c >> 7)) * math.ldexp((c & 7) + (8 if c & 120 else 0), max(c >> 3 & 15, 1) - 17) for c in range(256)]
    else:
        table = [math.ldexp((c & 7) + (8 if c >> 3 else 0), max(c >> 3, 1) - 33) for c in range(256)]
    values = torch.tensor(table, dtype=torch.float64, device=DEVICE)[s["moments"].view(-1, 2, BLOCK)[:, k].long()]
    return (values * (2.0 ** (s["scales"][:, k].double() - 127))[:, None]).view(-1)[s["slot"]] * (s["scales"][:, k] > 0)[s["slot"] // BLOCK]


def _exact_round(s, x, below, random20, keep=False):
    """Eighths of the value's power of two, none smaller than those `below` powers under the largest of its block."""
    largest = torch.zeros(s["count"], dtype=torch.float64, device=DEVICE).scatter_reduce_(0, s["slot"] // BLOCK, x.abs(), "amax")
    power = torch.log2(largest.clamp(min=2.0 ** -126)).floor()[s["slot"] // BLOCK]
    own_power = torch.log2(x.abs().clamp(min=2.0 ** -200)).floor()
    eighth = torch.exp2(torch.maximum(own_power, power - below) - 3)
    n = torch.floor((torch.round(x.abs() / eighth * 2 ** 20) + random20) / 2 ** 20)
    if keep:
        n = n.clamp(min=1)
    return torch.where(x == 0, 0.0, torch.sign(x) * n * eighth)


# ------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if case["op"] == "log_probs":
        n, v, top = case["n"], case["v"], case["top"]
        rows = n * ((8 if case["index"] == "int64" else 4) + 8 + 12 * top)
        if case["mode"] == "forward":  # logits
            return {"bytes": 4 * n * v + rows, "flops": 6 * n * v}
        return {"bytes": 8 * n * v + rows + 12 * n, "flops": 10 * n * v}  # logits; their gradient
    if case["op"] == "norms":
        rows, c = case["batch"] * case["positions"], case["c"]
        gate = {"none": 0, "channel": c, "sample": case["batch"] * c, "full": rows * c}[case["gate"]]
        vectors = c * (2 if case["post"] else 1) + gate
        if case["mode"] == "forward":  # residual, block; their sum and its norm
            return {"bytes": 4 * (4 * rows * c + vectors), "flops": 10 * rows * c}
        return {"bytes": 4 * (6 * rows * c + 2 * vectors + 2 * rows), "flops": 22 * rows * c}  # both gradients, sum, block; two gradients
    if case["bits"] == 32:  # gradients, parameters, two moments; the last three written
        return {"bytes": 28 * case["elements"], "flops": 14 * case["elements"]}
    # gradients, parameters, moments of a byte; the last two written, and the moments as what they stand for
    return {"bytes": (12 + 4 * (1 + 1 / BLOCK) + 8) * case["elements"], "flops": 40 * case["elements"]}
