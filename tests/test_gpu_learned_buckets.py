"""The example that runs the operators together: its gradients against automatic differentiation in 64 bits, and a short training run."""
import importlib.util
import os
import sys

import pytest

from helpers import ROOT

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def example():
    spec = importlib.util.spec_from_file_location("learned_buckets", os.path.join(ROOT, "examples", "learned_buckets.py"))
    m = sys.modules[spec.name] = importlib.util.module_from_spec(spec)  # where its dataclass looks for it
    spec.loader.exec_module(m)
    return m


def test_gradients():
    m = example()
    gate = m.BucketGate(96, m.GateConfig(balance=0.3, z=0.01, eps=1e-5))
    g = torch.Generator("cuda").manual_seed(2)
    rows, dout = torch.rand(700, 96, generator=g, device="cuda"), torch.randn(700, generator=g, device="cuda")
    out, saved = gate.forward(rows)
    got = gate.gradients(rows, dout, saved)
    p = {n: getattr(gate, n).double().requires_grad_() for n in ("gate", "heads", "weight", "bias")}
    x = rows.double()
    x = (x - x.mean(1, keepdim=True)) / (x.var(1, correction=0, keepdim=True) + 1e-5).sqrt() * p["weight"] + p["bias"]
    logits = x @ p["gate"].t()
    index, counts = saved[4].index.long(), saved[4].counts.double()
    chosen = torch.softmax(logits.gather(1, index), 1)
    want_out = (chosen * (x @ p["heads"].t()).gather(1, index)).sum(1)
    balance = 9 / (700 * 2) * (counts * torch.softmax(logits, 1).mean(0)).sum()
    z = torch.logsumexp(logits, 1).square().mean()
    ((want_out * dout.double()).sum() + 0.3 * balance + 0.01 * z).backward()
    # fp32 throughout: sums of 700 and 96 terms, a few of them in a row: (700 + 3 * 96) 2^-24 = 6e-5 of the norm at worst
    assert (out.double() - want_out).norm() <= 6e-5 * want_out.norm()
    for name, t in p.items():
        assert (got[name].double() - t.grad).norm() <= 6e-5 * t.grad.norm(), name


def test_short_run():
    history = example().run(steps=6, batch_size=1024, verbose=False)
    assert len(history) == 6
    for (mse, balance, z), net, counts in history:
        assert 0 < mse < 10 and balance >= 0.9 and z >= 0 and 0 < net < 1 and sum(counts) == 2 * 1024
    assert history[-1][0][0] < history[0][0][0]    # the heads learn something of the outcome
