"""Muon's adamw groups with held moments: refused steps, and checkpoints of groups held otherwise."""

from __future__ import annotations

import pytest
import torch

from gram_newton_schulz_ampere_b200 import Muon

pytestmark = pytest.mark.gpu


def make(device, bits, sizes=(700, 33, 256), dtype=torch.bfloat16):
    params = [torch.nn.Parameter(torch.linspace(-1, 1, n, device=device).to(dtype)) for n in sizes]
    group = {"params": params, "algorithm": "adamw"}
    if bits is not None:
        group["state_bits"] = bits
    return params, Muon([group], lr=1e-2, weight_decay=0.1)


def give(params, seed):
    gen = torch.Generator(device=params[0].device).manual_seed(seed)
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen, device=p.device).to(p.dtype)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_refused_step_counts_for_nothing(cuda_device, bits):
    params, optimizer = make(cuda_device, bits)
    twin, untouched = make(cuda_device, bits)
    for number in (1, 2):
        for ps, opt in ((params, optimizer), (twin, untouched)):
            give(ps, number)
            opt.step()
    held = optimizer.state[params[1]]["exp_avg"]
    optimizer.state[params[1]]["exp_avg"] = held.double()
    before = [p.detach().clone() for p in params]
    give(params, 3)
    for _ in range(2):
        with pytest.raises(TypeError, match="AdamW moments must be"):
            optimizer.step()
    assert all(torch.equal(p, b) for p, b in zip(params, before))
    assert [optimizer.state[p]["step"].item() for p in params] == [2.0, 2.0, 2.0]
    optimizer.state[params[1]]["exp_avg"] = held
    for number in (3, 4):
        for ps, opt in ((params, optimizer), (twin, untouched)):
            give(ps, number)
            opt.step()
    assert all(torch.equal(p, q) for p, q in zip(params, twin))
    assert [optimizer.state[p]["step"].item() for p in params] == [4.0, 4.0, 4.0]
