"""A small torch policy learns from a network's priors and then picks moves itself.

The teacher is the Connect4 graph-attention network: its priors on random
positions are the targets.  The student is a torch MLP whose weights are kept
in 32 bits and used in bfloat16.  Each step takes the loss and its gradient
over the legal moves (policy_loss), continues the backward pass in torch, and
updates all tensors, clipped, with 8-bit optimiser states and the bfloat16
copies (AdamW).  Then the student draws legal moves (policy_sample).

Usage: python examples/distill_policy.py [--steps 300] [--batch 2048]
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import graphzero_b200 as gz  # noqa: E402

GAME = gz.CONNECT4


def legal_moves(boards):
    """[n][7]: columns whose top cell is empty."""
    return boards.view(-1, 6, 7)[:, 0] == 0


def features(boards, side):
    """Own and other stones of every cell, bfloat16 [n][84]."""
    own = boards * side[:, None]
    return torch.cat([own == 1, own == -1], 1).to(torch.bfloat16)


class Student:
    """Layers of weights and biases in 32 bits with bfloat16 copies to compute with."""

    def __init__(self, sizes=(84, 256, 256, 7), seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.params = []
        for a, b in zip(sizes, sizes[1:]):
            self.params += [torch.randn(a, b, device="cuda", generator=g) * (2 / a) ** 0.5, torch.zeros(b, device="cuda")]
        self.copies = [p.to(torch.bfloat16).requires_grad_() for p in self.params]

    def logits(self, x):
        for w, b in zip(self.copies[:-2:2], self.copies[1:-2:2]):
            x = torch.relu(x @ w + b)
        return x @ self.copies[-2] + self.copies[-1]


def draw(student, boards, side, seed, **filters):
    """A legal move for every position, drawn from the student's policy."""
    with torch.no_grad():
        logits = student.logits(features(boards, side))
    g = torch.Generator(device="cuda").manual_seed(seed)
    noise = -torch.empty(logits.shape, device="cuda").exponential_(generator=g).log()
    return gz.policy_sample(logits, noise, mask=legal_moves(boards), **filters)


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--batch", type=int, default=2048)
    a = ap.parse_args(argv)

    teacher = gz.Net(GAME, max_batch=a.batch)
    weights = gz.synth_weights(GAME, seed=1, bias_scale=0.3)
    shape = gz.game_shape(GAME)
    heads, _ = gz.train_bucket_range(GAME, shape.layers)  # the policy head comes first
    weights[heads:heads + 256 * max(1, shape.policy_per_node)] *= 30  # a teacher with opinions
    teacher.load_weights(weights)
    student = Student()
    opt = gz.AdamW(student.params, lr=2e-3, weight_decay=1e-4, state_bits=8, copies=[c.detach() for c in student.copies],
                   max_norm=1.0)

    def batch(seed):
        boards, side = gz.synth_positions_device(GAME, a.batch, seed=seed)
        pi, v = torch.empty(a.batch, 7, device="cuda"), torch.empty(a.batch, device="cuda")
        teacher.predict_batch(boards, side, a.batch, pi, v)
        return boards, side, pi

    def agreement(seed):
        """The teacher's mean probability, among the legal moves, of drawn ones."""
        boards, side, pi = batch(seed)
        move, _ = draw(student, boards, side, seed, temperature=0.8, top_p=0.95)
        pi = pi * legal_moves(boards)
        return float((pi.gather(1, move.long()[:, None])[:, 0] / pi.sum(1)).mean())

    before, losses = agreement(10**6), []
    for step in range(a.steps):
        boards, side, pi = batch(step)
        logits = student.logits(features(boards, side))
        loss, grad = gz.policy_loss(logits.detach(), target=pi, mask=legal_moves(boards), grad_scale=1.0 / a.batch)
        logits.backward(grad)
        opt.step([c.grad for c in student.copies])
        for c in student.copies:
            c.grad = None
        losses.append(loss.mean())
    after = agreement(10**6)
    teacher.check()
    losses = torch.stack(losses).tolist() if losses else [float("nan")]
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}; the teacher's probability of the moves drawn {before:.4f} -> {after:.4f}")
    return losses, before, after


if __name__ == "__main__":
    main()
