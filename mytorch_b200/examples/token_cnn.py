"""A convolutional classifier of token sequences, on synthetic data: an embedding whose rows are the channels of a channels-last image of one line, two
stages of Conv2d and GroupNorm with SiLU, the mean over positions and a Linear layer; gradients clipped on their way into the SGD update.

A sequence's class is the token that its marker is followed by; the rest is noise whose tokens are as unevenly frequent as those of text, with padding
(token 0) behind the end.

    python -m mytorch_b200.examples.token_cnn [--device cuda:0] [--steps 300] [--batch 64] [--length 64]
"""
import argparse

import numpy as np

import mytorch_b200 as mytorch
import mytorch_b200.nn as nn
import mytorch_b200.nn.functional as F
from mytorch_b200.optim import SGD

CLASSES, MARKER = 8, 1


class TokenCNN(nn.Module):
    def __init__(self, vocabulary=1000, width=64, classes=CLASSES, groups=8):
        super().__init__()
        self.embed = nn.Embedding(vocabulary, width, padding_idx=0, scale=width ** 0.5, channels_first=True)
        self.embed.reset_parameters(width ** -0.5)
        self.conv1 = nn.Conv2d(width, width, (1, 3), padding=(0, 1), bias=False)
        self.norm1 = nn.GroupNorm(groups, width, activation="silu")
        self.conv2 = nn.Conv2d(width, 2 * width, (1, 3), padding=(0, 1), bias=False)
        self.norm2 = nn.GroupNorm(groups, 2 * width, activation="silu")
        self.head = nn.Linear(2 * width, classes)

    def forward(self, tokens):
        """``tokens``: [N, 1, L]"""
        x = self.norm1(self.conv1(self.embed(tokens)))
        x = self.norm2(self.conv2(x))
        return self.head(x.mean(dim=(2, 3)))


def batch_of(rng, batch, length, vocabulary=1000):
    """(tokens [batch, 1, length], classes [batch]), both int64 arrays."""
    first = 2 + CLASSES
    noise = np.exp(rng.random((batch, length)) * np.log(vocabulary - first + 1)).astype(np.int64) - 1 + first
    tokens = np.minimum(noise, vocabulary - 1)
    used = rng.integers(length // 2, length + 1, batch)
    tokens[np.arange(length)[None, :] >= used[:, None]] = 0
    label = rng.integers(0, CLASSES, batch)
    at = (rng.random(batch) * (used - 1)).astype(np.int64)
    tokens[np.arange(batch), at] = MARKER
    tokens[np.arange(batch), at + 1] = 2 + label
    return tokens.reshape(batch, 1, length), label


def train_token_cnn(device="cuda:0", steps=300, batch=64, length=64, lr=0.1, max_grad_norm=1.0, seed=0, log=print):
    """Trains on fresh batches; returns (loss of each step, accuracy on 512 new sequences)."""
    rng = np.random.default_rng(seed)
    mytorch.manual_seed(seed)
    model = TokenCNN()
    model.to(device)
    optimizer = SGD(model.parameters(), lr=lr, momentum=0.9, max_grad_norm=max_grad_norm)
    losses = []
    for i in range(steps):
        tokens, label = (mytorch.tensor(a, device=device) for a in batch_of(rng, batch, length))
        loss = F.cross_entropy(model(tokens), label)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
        if (i + 1) % 50 == 0:
            log(f"Step #{i}, loss: {losses[-1]:0.4f}, norm of the gradients: {optimizer.grad_norm.item():0.4f}")
    tokens, label = batch_of(rng, 512, length)
    with mytorch.no_grad():
        found = model(mytorch.tensor(tokens, device=device)).max(dim=1)[1]
    accuracy = float((found.to("cpu").numpy() == label).mean())
    log(f"Accuracy: {accuracy * 100:0.2f}%")
    return losses, accuracy


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--device", default="cuda:0")
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--batch", type=int, default=64)
    ap.add_argument("--length", type=int, default=64)
    a = ap.parse_args()
    train_token_cnn(a.device, a.steps, a.batch, a.length)
