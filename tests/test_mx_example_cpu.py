"""examples/mx_lm.py: every mx_linear of every step has a seed of its own.  A seed names the random bits by an
element's place, so two layers of one seed round their gradients alike."""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_seeds_differ_between_layers_and_steps(monkeypatch):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import mx_lm
    finally:
        sys.path.pop(0)
    seeds = []

    def linear(x, weight, seed=None, **_):
        seeds.append(seed)
        return x @ weight.T

    def norm(x, weight, residual):
        h = x + residual
        return h * weight, h

    monkeypatch.setattr(mx_lm, "mx_linear", linear)
    monkeypatch.setattr(mx_lm, "rms_norm", norm)
    monkeypatch.setattr(mx_lm, "Adafactor8Bit", lambda params, **_: torch.optim.SGD(params, lr=0.0))
    mx_lm.train(3, device="cpu")
    assert len(seeds) == 3 * (2 * mx_lm.BLOCKS + 1) and None not in seeds
    assert len(set(seeds)) == len(seeds), seeds
