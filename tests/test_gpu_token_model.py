"""The operators of a token model in a row: embedding, norms around a block, log probabilities, their gradients and the update, against PyTorch in 64 bits on the CPU; the
example that uses them; and a whole step of it in a graph.

Tolerances: a product's sums go through at most 96 additions, a norm's and a softmax's through as many, one behind the other through six operators and back: under
2000 roundings of 2^-24 of the largest terms, 1.2e-4 of a gradient's 2-norm."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def blocks_of_these_sizes_go_back_to_the_driver():
    """A later module's test of the memory pool counts on sizes that no earlier one left there."""
    yield
    from mytorch_b200.backends.cuda.env import CudaEnv

    CudaEnv.instance().lib.pool_trim()


ROWS, WIDTH, N, L = 96, 48, 5, 7
NAMES = {"table": (ROWS, WIDTH), "first": (WIDTH,), "block": (WIDTH, WIDTH), "weight": (WIDTH,), "post": (WIDTH,), "gate": (N, WIDTH), "head": (ROWS, WIDTH)}


def _arrays(seed=0):
    rng = np.random.default_rng(seed)
    made = {k: (rng.standard_normal(s) * 0.5).astype(np.float32) for k, s in NAMES.items()}
    tokens, target = rng.integers(0, ROWS, (N, L)), rng.integers(0, ROWS, (N, L))
    target[1::2, 4:] = -100
    return made, tokens, target, rng.standard_normal((N, L)).astype(np.float32)


def _ours(p, tokens, target, advantage):
    import mytorch_b200.nn.functional as F

    residual = F.embedding(tokens, p["table"])
    y = F.rms_norm(residual, p["first"])
    block = F.linear(y.reshape((N * L, WIDTH)), p["block"]).reshape((N, L, WIDTH))
    new, y = F.add_rms_norm(residual, block, p["weight"], p["post"], p["gate"], scale=0.75)
    logits = F.linear(y.reshape((N * L, WIDTH)), p["head"]).reshape((N, L, ROWS))
    scores = F.token_log_probs(logits, target, top=4, ignore_index=-100)
    return (scores.log_probs * advantage).sum() * -1.0 - scores.entropy.sum() * 0.1 + scores.top_log_probs.sum() * 0.01 + (new * new).sum() * 0.001


def _theirs(p, tokens, target, advantage):
    import torch

    norm = lambda x: x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    residual = p["table"][tokens]
    block = (norm(residual) * p["first"]) @ p["block"].T
    new = 0.75 * residual + p["gate"][:, None, :] * (norm(block) * p["post"])
    log_p = torch.log_softmax((norm(new) * p["weight"]) @ p["head"].T, -1)
    known = target != -100
    given = log_p.gather(-1, torch.where(known, target, 0)[..., None])[..., 0] * known
    entropy = -(log_p.exp() * log_p).sum(-1)
    return -(given * advantage).sum() - 0.1 * entropy.sum() + 0.01 * log_p.topk(4, dim=-1)[0].sum() + 0.001 * new.square().sum()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_of_all_of_them(bits, monkeypatch):
    monkeypatch.setenv("MTB_DISABLE_TC", "1")  # Linear's products in float32: rounded to TF32 their factors would be 2^-11 off
    import gpu_util as g
    import mytorch_b200.nn as nn
    import torch
    from mytorch_b200.optim import AdamW

    made, tokens, target, advantage = _arrays()
    ours = {k: nn.Parameter(g.dev(a)) for k, a in made.items()}
    opt = AdamW(ours.values(), lr=0.01, weight_decay=0.1, max_grad_norm=0.5, state_bits=bits)
    theirs = {k: torch.tensor(a, dtype=torch.float64, requires_grad=True) for k, a in made.items()}
    m, v, factors = {}, {}, (0.9, 0.999) if bits == 32 else tuple(round(b * 2 ** 20) / 2 ** 20 for b in (0.9, 0.999))
    loss = _ours(ours, g.dev(tokens), g.dev(target), g.dev(advantage))
    opt.zero_grad()
    loss.backward()
    want = _theirs(theirs, torch.tensor(tokens), torch.tensor(target), torch.tensor(advantage, dtype=torch.float64))
    want.backward()
    assert abs(loss.item() - want.item()) <= 1.2e-4 * abs(want.item())
    for k, p in ours.items():
        w = theirs[k].grad.numpy()
        assert np.linalg.norm(g.host(p.grad) - w) <= 1.2e-4 * np.linalg.norm(w), k
    grads = {k: g.host(p.grad).astype(np.float64) for k, p in ours.items()}
    opt.step()
    norm = np.sqrt(sum((x * x).sum() for x in grads.values()))
    assert abs(g.host(opt.grad_norm)[0] - norm) <= 2.0 ** -23 * norm and norm > 0.5
    for k, p in ours.items():
        x = grads[k] * (0.5 / (norm + 1e-6))
        m[k], v[k] = (1 - factors[0]) * x, (1 - factors[1]) * x * x
        step = 0.01 * (m[k] / (1 - factors[0])) / (np.sqrt(v[k] / (1 - factors[1])) + 1e-8)
        want = made[k] * (1 - 0.001) - step
        assert (np.abs(g.host(p) - want) <= 2.0 ** -24 * (4 * np.abs(made[k]) + 20 * np.abs(step))).all(), k
        first, second = (g.host(t).astype(np.float64) for t in opt.moments(p))
        tol = 2.0 ** -21 if bits == 32 else 2.0 ** -3  # a step of an eighth either way
        big = np.abs(m[k]) > np.abs(m[k]).max() * 2.0 ** -10
        assert (np.abs(first - m[k])[big] <= tol * np.abs(m[k])[big]).all() and (np.abs(second - v[k])[big] <= tol * v[k][big]).all(), k


@pytest.mark.parametrize("bits", [32, 8])
def test_the_example_runs(bits):
    from mytorch_b200.examples.masked_tokens import train_masked_tokens

    losses, shares = train_masked_tokens(steps=4, batch=8, length=16, state_bits=bits, log=lambda text: None)
    assert len(losses) == 4 and np.isfinite(losses).all() and 0 <= shares[0] <= shares[1] <= 1


def test_the_example_in_a_graph():
    """Steps replayed from a graph are those of a model beside it."""
    import gpu_util as g
    import mytorch_b200 as mt
    from mytorch_b200.cuda_graph import StepGraph
    from mytorch_b200.examples.masked_tokens import IGNORED, MaskedTokenModel, batch_of, loss_of
    from mytorch_b200.optim import AdamW

    rng = np.random.default_rng(3)
    batches = [batch_of(rng, 8, 16) for _ in range(4)]
    count = 20
    results = []
    for captured in (False, True):
        mt.manual_seed(3)
        model = MaskedTokenModel(blocks=1)
        model.to("cuda:0")
        opt = AdamW(model.parameters(), max_grad_norm=1.0, state_bits=8)
        tokens, target = (g.dev(a) for a in batches[0])

        def step():
            loss = loss_of(model, tokens, target, count, 0.01)
            opt.zero_grad()
            loss.backward()
            opt.step()
            return loss

        step()
        graph = StepGraph(step, [tokens, target])
        if captured:
            graph.capture()
        losses = []
        for b in batches[1:]:
            if captured:
                losses.append(g.host(graph.replay(b)))
            else:
                for t, a in zip((tokens, target), b):
                    t._native_array.write(a)
                losses.append(g.host(step()))
        results.append(losses + [g.host(p) for p in model.parameters()])
        if captured:
            graph.destroy()
    assert all(np.array_equal(a, b) for a, b in zip(*results))


def test_two_threads_share_scratch():
    """The gradient of the norms hands sums on in scratch: two host threads get the bits that one alone gets."""
    import threading

    import gpu_util as g

    rng = np.random.default_rng(4)

    def case(rows, c):
        a = [rng.standard_normal(s).astype(np.float32) for s in ((rows, c),) * 4 + ((c,),) * 3]
        rstd = np.abs(rng.standard_normal((2, rows))).astype(np.float32)

        def run():
            dnew, dy, new, block, weight, post, gate = (g.dev(x) for x in a)
            return g.op("add_rms_norm_backward")(dnew, dy, new, g.dev(rstd[0]), g.dev(rstd[1]), new, block, weight, post, gate, 1.0)

        return run

    cases = [case(300, 96), case(2000, 64), case(100, 1500), case(40, 9000)]
    alone = [[g.host(t) for t in run()] for run in cases]
    wrong = []

    def worker(order):
        for _ in range(10):
            for i, tensors in [(i, cases[i]()) for i in order]:
                if not all(np.array_equal(g.host(t), want) for t, want in zip(tensors, alone[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=worker, args=(order,)) for order in ((0, 1, 2, 3), (2, 0, 3, 1))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
