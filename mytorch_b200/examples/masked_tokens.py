"""A model that fills in masked tokens, on synthetic data: an embedding whose rows are the channels of a channels-last image of one line, residual blocks of
Conv2d, ReLU and Conv2d with the norms around them (RMSNorm, AddRMSNorm), a Linear head, log probabilities of the masked tokens with an entropy term, AdamW with clipping
and its states in 8 bits.

A sequence counts through the tokens in steps of its own, so that a masked token follows from its neighbours; sequences of unequal length are padded (token 0).

    python -m mytorch_b200.examples.masked_tokens [--device cuda:0] [--steps 300] [--batch 64] [--length 64] [--state-bits 8]
"""
import argparse

import numpy as np

import mytorch_b200 as mytorch
import mytorch_b200.nn as nn
import mytorch_b200.nn.functional as F
from mytorch_b200.optim import AdamW

PADDING, MASK, FIRST = 0, 1, 2  # the tokens that count begin at FIRST
IGNORED = -100


class MaskedTokenModel(nn.Module):
    def __init__(self, vocabulary=200, width=64, blocks=2):
        super().__init__()
        self.vocabulary, self.width, self.depth = vocabulary, width, blocks
        self.embed = nn.Embedding(vocabulary, width, padding_idx=PADDING, channels_first=True)
        self.norm = nn.RMSNorm(width)
        for i in range(blocks):
            setattr(self, f"wide{i}", nn.Conv2d(width, 2 * width, (1, 3), padding=(0, 1)))
            setattr(self, f"relu{i}", nn.ReLU())
            setattr(self, f"narrow{i}", nn.Conv2d(2 * width, width, (1, 1)))
            setattr(self, f"between{i}", nn.AddRMSNorm(width, post_norm=True, gate=0.5))
        self.head = nn.Linear(width, vocabulary)

    def forward(self, tokens):
        """``tokens``: [N, 1, L]; logits [N, L, vocabulary]"""
        residual = self.embed(tokens)
        y = self.norm(residual)
        for i in range(self.depth):
            block = getattr(self, f"narrow{i}")(getattr(self, f"relu{i}")(getattr(self, f"wide{i}")(y)))
            residual, y = getattr(self, f"between{i}")(residual, block)
        n, _, length = tokens.shape
        return self.head(y.permute((0, 2, 3, 1)).reshape((n, length, self.width)))


def batch_of(rng, batch, length, vocabulary=200, masked=0.15):
    """(tokens with masks [batch, 1, length], what the masks hide, IGNORED elsewhere [batch, length]), both int64 arrays."""
    used = rng.integers(length // 2, length + 1, (batch, 1))
    place = np.arange(length)[None, :]
    step = rng.integers(1, 8, (batch, 1))
    tokens = (rng.integers(0, vocabulary, (batch, 1)) + step * place) % (vocabulary - FIRST) + FIRST
    hidden = (rng.random((batch, length)) < masked) & (place < used)
    hidden[:, 1] = True  # one at least
    target = np.where(hidden, tokens, IGNORED)
    tokens = np.where(hidden, MASK, np.where(place < used, tokens, PADDING))
    return tokens.reshape(batch, 1, length).astype(np.int64), target.astype(np.int64)


def loss_of(model, tokens, target, count, entropy_weight=0.0):
    """The mean of -log p over the ``count`` hidden tokens, less ``entropy_weight`` times the mean entropy."""
    scores = F.token_log_probs(model(tokens), target, ignore_index=IGNORED)
    loss = scores.log_probs.sum() * (-1.0 / count)
    return loss - scores.entropy.sum() * (entropy_weight / target.shape[0] / target.shape[1]) if entropy_weight else loss


def train_masked_tokens(device="cuda:0", steps=300, batch=64, length=64, lr=3e-3, max_grad_norm=1.0, state_bits=8, entropy_weight=0.01, seed=0, log=print):
    """Trains on fresh batches; returns (loss of each step, share of 512 new sequences' hidden tokens that are the first alternative, or among the first five)."""
    rng = np.random.default_rng(seed)
    mytorch.manual_seed(seed)
    model = MaskedTokenModel()
    model.to(device)
    optimizer = AdamW(model.parameters(), lr=lr, max_grad_norm=max_grad_norm, state_bits=state_bits, seed=seed)
    losses = []
    for i in range(steps):
        tokens, target = batch_of(rng, batch, length)
        count = int((target != IGNORED).sum())
        loss = loss_of(model, mytorch.tensor(tokens, device=device), mytorch.tensor(target, device=device), count, entropy_weight)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
        if (i + 1) % 50 == 0:
            log(f"Step #{i}, loss: {losses[-1]:0.4f}, norm of the gradients: {optimizer.grad_norm.item():0.4f}")
    tokens, target = batch_of(rng, 512, length)
    with mytorch.no_grad():
        found = F.token_log_probs(model(mytorch.tensor(tokens, device=device)), mytorch.tensor(target, device=device), top=5, ignore_index=IGNORED)
    hit = found.top_tokens.to("cpu").numpy() == target[:, :, None]
    shares = tuple(float(hit[target != IGNORED][:, :k].any(axis=1).mean()) for k in (1, 5))
    log(f"Hidden tokens found: {shares[0] * 100:0.2f}%, among the first five: {shares[1] * 100:0.2f}%")
    return losses, shares


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--device", default="cuda:0")
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--batch", type=int, default=64)
    ap.add_argument("--length", type=int, default=64)
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    a = ap.parse_args()
    train_masked_tokens(a.device, a.steps, a.batch, a.length, state_bits=a.state_bits)
