"""Train a small next-token model with this package's operators alone, in mixed
precision: float32 weights that the optimizer steps, bf16 copies that the
products read.

    h = E[token] @ W1.T          tilec.ext.matrix_mul (bf16 in, float32 out)
    y = layer_norm(h) w + b      tilec.ext.layer_norm (float32 in, bf16 out)
    loss = CE(y @ W2.T, next)    tilec.ext.linear_cross_entropy_grad

and back: dy and dW2 come with the loss, dh, dw and db from
tilec.ext.layer_norm_backward, dW1 = dh.T @ x from matrix_mul, and
tilec.ext.adamw_step moves all of them in one call.  (The embedding E is fixed.)

    python examples/train_classifier.py [--steps 60] [--bits 8]

The data are sequences of a fixed random permutation: the next token follows
from the last one, one in ten is noise, and one in ten is not to be learned
from (ignored).
"""

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import tilec  # noqa: E402

IGNORE = -100


class Model:
    """The trained tensors, their bf16 copies and their AdamW states."""

    def __init__(self, vocab, width, hidden, bits, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape, std):
            return torch.randn(shape, generator=g, device="cuda") * std

        self.embedding = normal(vocab, width, std=1.0).bfloat16()
        self.params = [normal(hidden, width, std=1 / math.sqrt(width)), torch.ones(hidden, device="cuda"),
                       torch.zeros(hidden, device="cuda"), normal(vocab, hidden, std=1 / math.sqrt(hidden))]
        self.copies = [p.bfloat16() for p in self.params]
        states = [tilec.ext.adamw_state(p, bits) for p in self.params]
        self.exp_avg, self.exp_avg_sq = [s[0] for s in states], [s[1] for s in states]
        self.steps = 0

    def forward(self, tokens):
        w1, w, b, w2 = self.copies
        x = self.embedding[tokens]
        h = tilec.ext.matrix_mul(x, w1.t())
        y, mean, rstd = tilec.ext.layer_norm(h, w, b, dtype=torch.bfloat16)
        return x, h, y, mean, rstd

    def losses(self, tokens, targets):
        """One loss per token; no logits are kept."""
        return tilec.ext.linear_cross_entropy(self.forward(tokens)[2], self.copies[3], targets, reduction="none",
                                              ignore_index=IGNORE)

    def step(self, tokens, targets, lr):
        w = self.copies[1]
        x, h, y, mean, rstd = self.forward(tokens)
        loss, dy, dw2 = tilec.ext.linear_cross_entropy_grad(y, self.copies[3], targets, ignore_index=IGNORE)
        dh, dw, db = tilec.ext.layer_norm_backward(dy, h, mean, rstd, w)
        dw1 = tilec.ext.matrix_mul(dh.t(), x)
        self.steps += 1
        tilec.ext.adamw_step(self.params, [dw1, dw, db, dw2], self.exp_avg, self.exp_avg_sq, step=self.steps, lr=lr,
                             weight_decay=1e-2, copies=self.copies)
        return loss


def batch(follow, count, seed):
    """Tokens, and as targets the ones that follow them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = torch.randint(len(follow), (count,), generator=g, device="cuda")
    targets = follow[tokens]
    draw = torch.rand(count, generator=g, device="cuda")
    noise = torch.randint(len(follow), (count,), generator=g, device="cuda")
    targets = torch.where(draw < 0.1, noise, targets)
    return tokens, torch.where(draw > 0.9, IGNORE, targets)


def train(steps=60, tokens=2048, vocab=4000, width=128, hidden=256, bits=32, lr=1e-2, log=print):
    """The mean loss of every step, on the host."""
    follow = torch.randperm(vocab, generator=torch.Generator().manual_seed(1)).cuda()
    model = Model(vocab, width, hidden, bits)
    losses = []
    for i in range(steps):
        losses.append(model.step(*batch(follow, tokens, seed=i), lr=lr))
        if log and (i % 10 == 0 or i + 1 == steps):
            log(f"step {i + 1}: loss {losses[-1].item():.3f}")
    x, t = batch(follow, tokens, seed=steps)
    held_out = model.losses(x, t).sum() / (t != IGNORE).sum()
    if log:
        log(f"held out: loss {held_out.item():.3f} (uniform guess {math.log(vocab):.3f})")
    return [v.item() for v in losses], held_out.item()


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--bits", type=int, choices=(32, 8), default=32, help="of the optimizer's states")
    a = ap.parse_args()
    train(steps=a.steps, bits=a.bits)
