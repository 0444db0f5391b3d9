"""What an AdamW step over held moments hands to the native call, with that call replaced: no GPU."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from gram_newton_schulz_ampere_b200 import _native, ops

HYPER = (1e-3, 0.9, 0.95, 1e-8, 0.1)


class Place:
    """Stands for the CUDA device that the CPU tensors of these tests are not on."""

    index = -1

    def __eq__(self, other):
        return isinstance(other, Place) or other.type == "cpu"


class OnDevice:
    def __init__(self, index):
        pass

    def __enter__(self):
        return 0

    def __exit__(self, *error):
        pass


@pytest.fixture
def calls(monkeypatch):
    """The address lists (parameters, gradients, moments, scales) of each native call."""
    seen = []

    def step(count, *rest):
        seen.append([None if row is None else [place or 0 for place in row[:count]] for row in rest[:6]])
        return 0

    monkeypatch.setattr(ops, "_require_cuda", lambda *tensors: Place())
    monkeypatch.setattr(_native, "load", lambda: SimpleNamespace(gns_adamw_states_step=step))
    monkeypatch.setattr(_native, "on_device", OnDevice)
    return seen


def make(bits, sizes=(300, 40, 256)):
    return ops.AdamWStates([torch.ones(n) for n in sizes], bits), [torch.ones(n) for n in sizes]


def places(states):
    roles = [states.parameters, None, states.exp_avgs, states.exp_avg_sqs]
    roles += [states.exp_avg_scales, states.exp_avg_sq_scales] if states.bits == 8 else []
    return [role and [t.data_ptr() for t in role] for role in roles]


def same_places(call, states):
    return all(want is None or got == want for got, want in zip(call, places(states)))


@pytest.mark.parametrize("bits", [8, 32])
def test_tensors_that_are_replaced_or_moved_are_the_ones_stepped(calls, bits):
    states, grads = make(bits)
    states.step(grads, *HYPER, 1)
    assert same_places(calls[-1], states)
    first = places(states)
    states.exp_avgs[0] = states.exp_avgs[0].clone()
    states.exp_avg_sqs[2].data = states.exp_avg_sqs[2].data.clone()
    states.parameters[1].data = states.parameters[1].data.clone()
    if bits == 8:
        states.exp_avg_scales[1] = states.exp_avg_scales[1].clone()
        states.exp_avg_sq_scales[0].data = states.exp_avg_sq_scales[0].data.clone()
    assert places(states) != first
    states.step(grads, *HYPER, 2)
    assert same_places(calls[-1], states)
    # A step without some of the gradients takes the same tensors.
    states.exp_avgs[2] = states.exp_avgs[2].clone()
    states.step([grads[0], None, grads[2]], *HYPER, 3)
    now = places(states)
    assert all(want is None or got == [want[0], want[2]] for got, want in zip(calls[-1], now))


@pytest.mark.parametrize("bits", [8, 32])
def test_what_is_put_in_place_is_checked(calls, bits):
    dtype = torch.float8_e4m3fn if bits == 8 else torch.float32
    for role in ("exp_avgs", "exp_avg_sqs"):
        for wrong, error, match in (
            (torch.zeros(299).to(dtype), ValueError, "sizes differ"),
            (torch.zeros(300, dtype=torch.float16), TypeError, "must be"),
            (torch.zeros(600).to(dtype)[::2], ValueError, "contiguous"),
        ):
            for partly in (False, True):
                states, grads = make(bits)
                states.step(grads, *HYPER, 1)
                getattr(states, role)[0] = wrong
                before = len(calls)
                with pytest.raises(error, match=match):
                    states.step([grads[0], None, grads[2]] if partly else grads, *HYPER, 2)
                assert len(calls) == before
    states, grads = make(bits)
    states.exp_avgs[0].data = states.exp_avgs[0].data[:100]  # the same address, fewer elements behind it
    with pytest.raises(ValueError, match="sizes differ"):
        states.step(grads, *HYPER, 1)
    states, grads = make(bits)
    states.parameters[2].data = states.parameters[2].data[:100]
    with pytest.raises(ValueError, match="not that of its moments"):
        states.step(grads, *HYPER, 1)
    states, grads = make(bits)
    states.parameters[2].data = states.parameters[2].data.half()
    with pytest.raises(TypeError, match="share a dtype"):
        states.step(grads, *HYPER, 1)
    if bits == 8:
        states, grads = make(bits)
        states.exp_avg_scales[0] = torch.zeros(1)
        with pytest.raises(ValueError, match="sizes differ"):
            states.step(grads, *HYPER, 1)
    states, grads = make(bits)
    states.exp_avgs.pop()
    with pytest.raises(ValueError, match="equal lengths"):
        states.step(grads, *HYPER, 1)


def test_empty_lists_and_tensors(calls):
    ops.AdamWStates([]).step([], *HYPER, 1)
    states, grads = make(8, (0, 5))
    states.step(grads, *HYPER, 1)
    assert len(calls) == 1 and same_places(calls[-1], states)
