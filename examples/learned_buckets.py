"""LayerStack buckets that are learned instead of fixed by the king ranks.

A gate looks at the feature transformer's output of a position and chooses the stack of hidden layers that evaluates it:

    rows of the trainer's feature transformer -> layer norm -> gate logits -> choice of 2 of 9 buckets with gates

The first choice is the bucket the trainer trains the position in.  The gate itself learns from a linear head per bucket: the heads of
the chosen buckets, weighted by the gates, predict the game's outcome, and a balance loss keeps the buckets in use.  Its matrices take the Muon
step, the layer norm's vectors plain gradient steps.

    python examples/learned_buckets.py [--steps 20] [--batch 4096]
"""
from __future__ import annotations

import argparse
import os
import sys
from dataclasses import dataclass

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import tatara_b200 as tb  # noqa: E402
from tatara_b200 import ops  # noqa: E402


@dataclass
class GateConfig:
    buckets: int = 9
    chosen: int = 2
    lr: float = 0.02
    vector_lr: float = 1e-3
    balance: float = 0.05   # weight of the balance loss
    z: float = 1e-4         # weight of the z loss
    eps: float = 1e-12      # a fresh net's rows are small: their variance is 1e-9


class BucketGate:
    """The gate and its heads, with the forward and backward pass written out."""

    def __init__(self, width: int, cfg: GateConfig, seed: int = 1, device: str = "cuda"):
        g = torch.Generator("cpu").manual_seed(seed)
        self.cfg = cfg
        make = lambda: (torch.randn(cfg.buckets, width, generator=g) / width ** 0.5).to(device)  # noqa: E731
        self.gate, self.heads = make(), make()
        self.weight, self.bias = torch.ones(width, device=device), torch.zeros(width, device=device)
        self.momentum = {"gate": torch.zeros_like(self.gate), "heads": torch.zeros_like(self.heads)}
        self.dlosses = torch.tensor([cfg.balance, cfg.z], device=device)

    def forward(self, rows: torch.Tensor):
        x, mean, rstd = ops.layer_norm_forward(rows, self.weight, self.bias, eps=self.cfg.eps)
        logits = x @ self.gate.t()
        routing = ops.route_forward(logits, self.cfg.chosen)
        values = (x @ self.heads.t()).gather(1, routing.index.long())  # [rows, chosen]: every position has that many buckets
        return (routing.gate * values).sum(1), (x, mean, rstd, logits, routing, values)

    def gradients(self, rows: torch.Tensor, dout: torch.Tensor, saved):
        """Gradients of sum(dout * output) + balance and z losses."""
        x, mean, rstd, logits, routing, values = saved
        dvalues = torch.zeros_like(logits).scatter_(1, routing.index.long(), dout[:, None] * routing.gate)
        dlogits = ops.route_backward(logits, routing, dout[:, None] * values, self.dlosses)
        dx = dvalues @ self.heads + dlogits @ self.gate
        _, dweight, dbias = ops.layer_norm_backward(dx, rows, mean, rstd, self.weight)
        return {"gate": dlogits.t() @ x, "heads": dvalues.t() @ x, "weight": dweight, "bias": dbias}

    def step(self, rows: torch.Tensor, target: torch.Tensor):
        """One training step; the routing it chose and the losses (mean squared error, balance, z)."""
        out, saved = self.forward(rows)
        error = out - target
        grads = self.gradients(rows, error * (2.0 / max(1, len(rows))), saved)
        for name in ("gate", "heads"):
            ops.muon_step(getattr(self, name), self.momentum[name], grads[name], lr=self.cfg.lr)
        self.weight -= self.cfg.vector_lr * grads["weight"]
        self.bias -= self.cfg.vector_lr * grads["bias"]
        routing = saved[4]
        return routing, torch.cat([error.square().mean().reshape(1), routing.losses])


def run(steps: int = 20, batch_size: int = 4096, ft_out: int = 256, seed: int = 0, verbose: bool = True):
    fs, loss = tb.FEATURE_SETS["halfka-hm-merged"], tb.LossKind.sigmoid()
    cfg = GateConfig()
    trainer = tb.GpuTrainer(batch_size, ft_out, 16, 32, cfg.buckets, fs, optimizer="ranger", init=tb.layerstack_default_init(fs, ft_out, 16, 32, cfg.buckets))
    gate = BucketGate(ft_out, cfg)
    history = []
    for k in range(steps):
        batch = tb.synthetic_batch(tb.SYNTH_SEED + seed + k, batch_size, fs)
        # the feature transformer's output does not depend on the bucket; a validation pass leaves it in a buffer
        trainer.validate_step(batch, 0.0, loss)
        rows = torch.from_numpy(trainer.read_buffer("combined", batch_size * ft_out).reshape(batch_size, ft_out)).cuda()
        routing, losses = gate.step(rows, torch.from_numpy(batch.wdl).cuda() - 0.5)
        batch.bucket_idx = np.ascontiguousarray(routing.index[:, 0].cpu().numpy())
        trainer.train_step(batch, 8.75e-4, 0.0, loss)
        history.append((losses.tolist(), trainer.flush_pending_loss() / batch_size, routing.counts.tolist()))
        if verbose:
            (mse, balance, z), net, counts = history[-1]
            print("step %3d  gate: mse %.4f  balance %.4f  z %.3f  counts %s  net: loss %.5f" % (k, mse, balance, z, counts, net))
    trainer.close()
    return history


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--batch", type=int, default=4096)
    a = ap.parse_args()
    run(a.steps, a.batch)
