"""A double-pass training step on one B200, from tokens to NF4 weights.

The model is a stack of residual blocks x <- x + norm(x) W^T with NF4 weights and
a language model's head.  As AethelStream's doublepass runs it, the first pass
keeps only each norm's input, in 8 bits; the second walks the blocks backwards,
takes each gradient from those checkpoints and hands it to the GaLore optimizer,
which updates the NF4 weight in place:

    first pass   rms_norm_checkpoint (norm, residual add and checkpoint in one read)
    head         cut_cross_entropy and its backward, no logits kept
    second pass  checkpoint_weight_grad -> project_layer,
                 rms_norm_checkpoint_backward (joined with the residual's gradient)
    update       finish_step over all blocks, notify_step

    python examples/double_pass_step.py [--steps 8]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import aethelstream_b200 as A  # noqa: E402


class Model:
    """Residual blocks with NF4 weights, fp32 norm gains and a frozen head."""

    def __init__(self, d: int, blocks: int, vocab: int, rank: int, lr: float, seed: int = 0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
        self.d, self.blocks = d, blocks
        self.embed = rand(vocab, d).bfloat16()
        self.head = (rand(vocab, d) * d ** -0.5).bfloat16()
        self.weights = [A.nf4_quantize(rand(d, d) * 0.3 * d ** -0.5) for _ in range(blocks)]
        self.gains = [torch.ones(d, device="cuda") for _ in range(blocks + 1)]  # one per block, one for the head
        self.lr = lr
        self.keys = [(b, "d_wo") for b in range(blocks)]
        cfg = A.GaLoreConfig(mode="b200", state_codec="dynamic", adam=A.AdamWConfig(lr=lr), svd_refresh=False)
        self.opt = A.GaLoreOptimizer(cfg, [(b, "d_wo", d, d, rank) for b in range(blocks)])

    def step(self, tokens: torch.Tensor, labels: torch.Tensor, number: int) -> torch.Tensor:
        """One training step; the mean loss (on the device)."""
        # first pass: every norm's input is kept in 8 bits, nothing else
        x = self.embed[tokens]
        kept = []
        y, ckpt = A.rms_norm_checkpoint(x, self.gains[0])
        for b in range(self.blocks):
            kept.append(ckpt)
            branch = y @ A.nf4_dequantize(self.weights[b], torch.bfloat16).view(self.d, self.d).T
            y, ckpt, x = A.rms_norm_checkpoint(x, self.gains[b + 1], residual=branch)
        # the head: loss and the gradient of its input
        ce = A.cut_cross_entropy(y, self.head, labels)
        dy, _ = A.cut_cross_entropy_backward(y, self.head, labels, ce, need_weight=False)
        # second pass, from the last block to the first
        dx, dg = A.rms_norm_checkpoint_backward(dy, ckpt, self.gains[-1])
        d_gains = [dg]
        for b in reversed(range(self.blocks)):
            grad = A.checkpoint_weight_grad(dx, kept[b], norm_weight=self.gains[b])
            self.opt.project_layer([self.keys[b]], [grad])
            dy = dx @ A.nf4_dequantize(self.weights[b], torch.bfloat16).view(self.d, self.d)
            dx, dg = A.rms_norm_checkpoint_backward(dy, kept[b], self.gains[b], d_residual=dx)
            d_gains.append(dg)
        # the update: global clip, INT8 Adam, NF4 write; plain steps for the gains
        self.opt.finish_step(self.keys, self.weights)
        self.opt.notify_step(number)
        for g, dg in zip(self.gains, reversed(d_gains)):
            g.sub_(dg, alpha=self.lr)
        return ce.loss


def train(steps: int = 8, d: int = 512, blocks: int = 2, vocab: int = 4099, tokens: int = 1000, rank: int = 64,
          lr: float = 3e-3, seed: int = 0) -> list[float]:
    """Losses of `steps` steps on one batch of a synthetic next-token task."""
    model = Model(d, blocks, vocab, rank, lr, seed)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    ids = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    labels = (ids * 7 + 3) % vocab
    labels[torch.rand(tokens, generator=gen, device="cuda") < 0.2] = -100  # a prompt's tokens
    losses = [model.step(ids, labels, i + 1) for i in range(steps)]
    model.opt.close()
    return [float(x) for x in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=8)
    for i, loss in enumerate(train(ap.parse_args().steps)):
        print(f"step {i + 1}: loss {loss:.4f}")
