"""Muon's adamw groups with held moments: refused steps, and checkpoints of groups held otherwise."""

from __future__ import annotations

import math

import pytest
import torch

from gram_newton_schulz_ampere_b200 import Muon

pytestmark = pytest.mark.gpu


def make(device, bits, dtype=torch.bfloat16):
    shapes = ((700,), (33,), (16, 16))
    params = [torch.nn.Parameter(torch.linspace(-1, 1, math.prod(s), device=device).to(dtype).view(s)) for s in shapes]
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


def values(state):
    """The moments of a parameter in 64 bits, however they are held."""
    found = []
    for name in ("exp_avg", "exp_avg_sq"):
        moment = state[name].double().reshape(-1)
        if f"{name}_scale" in state:
            moment = moment * state[f"{name}_scale"].double().repeat_interleave(256)[:moment.numel()]
        found.append(moment)
    return found


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("source,target", [(None, 8), (8, None), (32, 8), (8, 32), (None, 32), (32, None), (8, 8), (32, 32)])
def test_a_checkpoint_is_brought_into_the_configured_form(cuda_device, source, target, dtype):
    """A value's e4m3 code is within 2^-4 of it or half the smallest code step (2^-10 of the
    scale; a second moment is raised by up to 2^-9), an fp32 value is the product of code and
    scale rounded once, one in the parameters' type rounded once more."""
    params, saved = make(cuda_device, source, dtype=dtype)
    for number in (1, 2, 3):
        give(params, number)
        saved.step()
    twin, loaded = make(cuda_device, target, dtype=dtype)
    checkpoint = saved.state_dict()
    loaded.load_state_dict(checkpoint)
    assert loaded.param_groups[0].get("state_bits") == target
    kind = {8: torch.float8_e4m3fn, 32: torch.float32, None: dtype}[target]
    for p, q in zip(params, twin):
        state = loaded.state[q]
        assert state["step"].item() == 3.0
        assert set(state) == {"step", "exp_avg", "exp_avg_sq"} | ({"exp_avg_scale", "exp_avg_sq_scale"} if target == 8 else set())
        for name, was, now in zip(("exp_avg", "exp_avg_sq"), values(saved.state[p]), values(state)):
            assert state[name].dtype == kind and state[name].shape == q.shape
            assert state[name].data_ptr() != saved.state[p][name].data_ptr()
            error = torch.finfo(kind if target != 8 else torch.float32).eps * was.abs()
            if target == 8 and source != 8:
                scale = state[f"{name}_scale"].double().repeat_interleave(256)[:now.numel()]
                smallest = scale * (2.0**-10 if name == "exp_avg" else 2.0**-9)
                error = torch.maximum(was.abs() * 2.0**-4, smallest) * (1 + 2.0**-20)
                top = torch.nn.functional.pad(was.abs(), (0, -was.numel() % 256)).view(-1, 256).amax(1)
                assert ((state[f"{name}_scale"].double() - top / 448).abs() <= 2.0**-22 * top / 448).all()
            elif source == target:
                error = 0.0
            assert ((now - was).abs() <= error).all()
            if name == "exp_avg_sq":
                assert (now[was > 0] > 0).all()
    give(twin, 4)
    loaded.step()
    assert all(q.isfinite().all() for q in twin) and loaded.state[twin[0]]["step"].item() == 4.0
    assert saved.state[params[0]]["step"].item() == 3.0
