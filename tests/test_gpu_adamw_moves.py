"""AdamW states that are moved or replaced between steps go on as untouched ones do."""

from __future__ import annotations

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops

pytestmark = pytest.mark.gpu

HYPER = (1e-2, 0.9, 0.95, 1e-8, 0.1)


@pytest.mark.parametrize("bits", [8, 32])
def test_moved_out_and_back(cuda_device, bits):
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    sizes = [5000, 33, 300]
    params = [torch.randn(n, generator=gen, device=cuda_device) for n in sizes]
    twin = [p.clone() for p in params]
    ours, untouched = ops.AdamWStates(params, bits), ops.AdamWStates(twin, bits)
    for step in range(1, 5):
        grads = [torch.randn(n, generator=gen, device=cuda_device) for n in sizes]
        for role in (ours.exp_avgs, ours.exp_avg_sqs, ours.exp_avg_scales, ours.exp_avg_sq_scales):
            for i, t in enumerate(role):
                if step % 2:
                    role[i] = t.clone()  # another tensor
                else:
                    host = t.cpu()
                    t.data = torch.empty(0, dtype=t.dtype, device=cuda_device)
                    t.data = host.to(cuda_device)  # the same one, elsewhere
        if step == 3:
            params[0].data = params[0].data.clone()
        given = [grads[0], None, grads[2]] if step == 2 else grads
        ours.step(given, *HYPER, step)
        untouched.step(given, *HYPER, step)
    for a, b in zip(ours.parameters + ours.exp_avg_scales, twin + untouched.exp_avg_scales):
        assert torch.equal(a, b)
    for a, b in zip(ours.exp_avgs + ours.exp_avg_sqs, untouched.exp_avgs + untouched.exp_avg_sqs):
        assert torch.equal(a.float(), b.float())
    # While a state is away, a step is refused.
    host = ours.exp_avgs[0].cpu()
    ours.exp_avgs[0].data = host
    with pytest.raises(ValueError, match="device"):
        ours.step(grads, *HYPER, 5)
