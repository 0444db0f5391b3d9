"""AdamW over many tensors with 8- and 32-bit states, against 64-bit arithmetic.

Bounds: a moment is formed with at most four fp32 roundings; the update m / (sqrt(v)
c + eps) with the approximate square root and division errs by less than 2^-20 of
itself; the parameter is rounded once to its type. An e4m3 value is within 2^-4 of
the exact one, or within half of its smallest step (2^-10 of a block's scale)."""

from __future__ import annotations

import math

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops

pytestmark = pytest.mark.gpu

ROUNDING = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}  # unit roundoff
HYPER = {"learning_rate": 3e-3, "beta1": 0.9, "beta2": 0.95, "epsilon": 1e-8, "weight_decay": 0.1}


def blocks(t):
    flat = t.reshape(-1).double()
    return torch.nn.functional.pad(flat, (0, -flat.numel() % ops.STATE_BLOCK)).view(-1, ops.STATE_BLOCK)


def value(codes, scales):
    return (blocks(codes) * scales.double()[:, None]).reshape(-1)[:codes.numel()].view(codes.shape)


def moments(states, i):
    if states.bits == 32:
        return states.exp_avgs[i].double(), states.exp_avg_sqs[i].double()
    return (value(states.exp_avgs[i], states.exp_avg_scales[i]),
            value(states.exp_avg_sqs[i], states.exp_avg_sq_scales[i]))


def check_step(states, gradients, step, scale=None, hyper=HYPER):
    """One step of `states`, checked against the formula in 64 bits from the moments before it."""
    before = [p.double() for p in states.parameters]
    old = [moments(states, i) for i in range(len(before))]
    states.step(gradients, step=step, gradient_scale=scale, **hyper)
    lr, b1, b2 = hyper["learning_rate"], hyper["beta1"], hyper["beta2"]
    for i, g in enumerate(gradients):
        p = states.parameters[i]
        if g is None:
            assert torch.equal(p.double(), before[i])
            assert torch.equal(torch.stack(moments(states, i)), torch.stack(old[i]))
            continue
        g = g.double() * (1.0 if scale is None else scale.item())
        m = b1 * old[i][0] + (1 - b1) * g
        v = b2 * old[i][1] + (1 - b2) * g * g
        m_error = 2.0**-22 * (b1 * old[i][0].abs() + (1 - b1) * g.abs())
        denominator = (v / (1 - b2**step)).sqrt() + hyper["epsilon"]
        update = lr / (1 - b1**step) * m / denominator
        error = lr / (1 - b1**step) * m_error / denominator + 2.0**-20 * update.abs() + 2.0**-22 * before[i].abs()
        want = before[i] * (1 - lr * hyper["weight_decay"]) - update
        bound = error + ROUNDING[p.dtype] * (want.abs() + error) + (2.0**-25 if p.dtype == torch.float16 else 0.0)
        assert ((p.double() - want).abs() <= bound).all()
        new_m, new_v = moments(states, i)
        if states.bits == 32:
            assert ((new_m - m).abs() <= m_error + 1e-45).all()
            assert ((new_v - v).abs() <= 2.0**-22 * v + 1e-45).all()
            continue
        for new, exact, scales in ((new_m, m, states.exp_avg_scales[i]), (new_v, v, states.exp_avg_sq_scales[i])):
            top = blocks(exact).abs().amax(1)
            assert ((scales.double() - top / 448).abs() <= 2.0**-21 * top / 448 + 1e-45).all()
            smallest = scales.double()[:, None] * 2.0**-10
            floor = 2 * smallest if exact is v else smallest  # a second moment is raised to the smallest code
            spare = 2.0**-20 * blocks(exact).abs() + blocks(m_error if exact is m else exact * 2.0**-22)
            off = (blocks(new) - blocks(exact)).abs()
            assert (off <= torch.maximum(blocks(exact).abs() * 2.0**-4, floor) * (1 + 2.0**-18) + spare).all()
        assert (new_v[v > 0] > 0).all()


def tensors(gen, sizes, p_dtype, g_dtype, device, g_scale=1e-2):
    params = [(torch.randn(n, generator=gen, device=device) * 0.05).to(p_dtype) for n in sizes]
    grads = [(torch.randn(n, generator=gen, device=device) * g_scale).to(g_dtype) for n in sizes]
    return params, grads


SIZES = [[1], [255, 256, 257], [0, 8, 16383, 16384, 16385, 3], [100000, 1, 77], [64] * 300]


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("p_dtype,g_dtype", [
    (torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
    (torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16), (torch.float32, torch.bfloat16),
])
def test_steps(cuda_device, bits, sizes, p_dtype, g_dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    params, grads = tensors(gen, sizes, p_dtype, g_dtype, cuda_device)
    states = ops.AdamWStates(params, bits)
    for step in (1, 2, 3):
        check_step(states, grads, step)
        grads = [torch.randn(g.shape, generator=gen, device=cuda_device).mul(1e-2).to(g_dtype) for g in grads]


@pytest.mark.parametrize("bits", [8, 32])
def test_unaligned_slices(cuda_device, bits):
    """Tensors packed one behind the other, starting anywhere."""
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    sizes = [1, 300, 7, 5000, 2, 513]
    total = sum(sizes)
    for dtype in (torch.bfloat16, torch.float32):
        (flat_p,), (flat_g,) = tensors(gen, [total], dtype, dtype, cuda_device)
        states = ops.AdamWStates(list(flat_p.split(sizes)), bits)
        check_step(states, list(flat_g.split(sizes)), 1)
        check_step(states, list(flat_g.split(sizes)), 2)
    if bits == 8:  # the states too
        held = torch.zeros((2, total + 1), device=cuda_device).to(torch.float8_e4m3fn)
        counts = [(n + 255) // 256 for n in sizes]
        scales = torch.zeros((2, sum(counts)), device=cuda_device)
        states = ops.AdamWStates(
            list(flat_p.split(sizes)), 8, list(held[0, 1:].split(sizes)), list(held[1, 1:].split(sizes)),
            list(scales[0].split(counts)), list(scales[1].split(counts)))
        check_step(states, list(flat_g.split(sizes)), 1)
        check_step(states, list(flat_g.split(sizes)), 2)


@pytest.mark.parametrize("bits", [8, 32])
def test_wide_range_of_gradients(cuda_device, bits):
    """Magnitudes from 1e-12 to 1e3 inside a block, exact zeros among them."""
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    params, _ = tensors(gen, [4096], torch.float32, torch.float32, cuda_device)
    exponent = torch.rand(4096, generator=gen, device=cuda_device) * 15 - 12
    grad = torch.randn(4096, generator=gen, device=cuda_device) * 10**exponent
    grad[::7] = 0.0
    states = ops.AdamWStates(params, bits)
    for step in (1, 2):
        check_step(states, [grad], step)


@pytest.mark.parametrize("bits", [8, 32])
def test_zero_gradients(cuda_device, bits):
    params = [torch.ones(1000, device=cuda_device)]
    states = ops.AdamWStates(params, bits)
    states.step([torch.zeros(1000, device=cuda_device)], step=1, **HYPER)
    assert torch.allclose(params[0], torch.full_like(params[0], 1 - 3e-4), rtol=2.0**-22)
    assert not any(t.float().any() for t in moments(states, 0))


@pytest.mark.parametrize("bits", [8, 32])
def test_missing_gradients_scale_and_steps(cuda_device, bits):
    gen = torch.Generator(device=cuda_device).manual_seed(4)
    params, grads = tensors(gen, [300, 40, 5000], torch.bfloat16, torch.bfloat16, cuda_device)
    states = ops.AdamWStates(params, bits)
    check_step(states, [grads[0], None, grads[2]], 1, torch.tensor(0.25, device=cuda_device))
    check_step(states, grads, 2, torch.tensor([1.0 / 65536], device=cuda_device))
    # One step number for each parameter: the bias corrections are the parameter's own.
    twin = [p.clone() for p in params]
    alone = [ops.AdamWStates([p], bits) for p in twin]
    fresh = ops.AdamWStates(params, bits)
    fresh.step(grads, step=[1, 5, 9], **HYPER)
    for s, g, t in zip(alone, grads, (1, 5, 9)):
        s.step([g], step=t, **HYPER)
    assert all(torch.equal(a, b) for a, b in zip(params, twin))


def test_nonfinite_gradients(cuda_device):
    """A gradient that is not finite reaches its own block and no other; with 32-bit states
    its own element."""
    for bad in (float("nan"), float("inf")):
        for bits in (8, 32):
            params = [torch.ones(1024, device=cuda_device)]
            grad = torch.full((1024,), 0.5, device=cuda_device)
            grad[300] = bad
            states = ops.AdamWStates(params, bits)
            states.step([grad], step=1, **HYPER)
            assert not params[0][300].isfinite()
            states.step([grad], step=2, **HYPER)
            reached = torch.zeros(1024, dtype=torch.bool, device=cuda_device)
            reached[256:512] = bits == 8
            reached[300] = True
            assert params[0][~reached].isfinite().all()
            assert not moments(states, 0)[0][300].isfinite()


def test_repeats_bit_for_bit_on_another_stream(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(5)
    params, grads = tensors(gen, [70000, 33], torch.bfloat16, torch.bfloat16, cuda_device)
    twin = [p.clone() for p in params]
    first, second = ops.AdamWStates(params, 8), ops.AdamWStates(twin, 8)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    for step in (1, 2, 3):
        first.step(grads, step=step, **HYPER)
        with torch.cuda.stream(stream):
            second.step(grads, step=step, **HYPER)
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(params + first.exp_avg_scales, twin + second.exp_avg_scales):
        assert torch.equal(a, b)


def test_trains_like_32_bits(cuda_device):
    """A least-squares fit reaches the neighbourhood of the 32-bit run's loss."""
    gen = torch.Generator(device=cuda_device).manual_seed(6)
    a = torch.randn(512, 256, generator=gen, device=cuda_device)
    target = a @ torch.randn(256, generator=gen, device=cuda_device)
    losses = {}
    for bits in (8, 32):
        w = torch.zeros(256, device=cuda_device)
        states = ops.AdamWStates([w], bits)
        for step in range(1, 401):
            grad = a.T @ (a @ w - target) / 512
            states.step([grad], 2e-2, 0.9, 0.95, 1e-8, 0.0, step)
        losses[bits] = (a @ w - target).square().mean().item()
    start = target.square().mean().item()
    assert losses[32] < 1e-2 * start and losses[8] < 1e-2 * start


def test_refusals(cuda_device):
    p = [torch.ones(300, device=cuda_device)]
    with pytest.raises(ValueError, match="8 or 32"):
        ops.AdamWStates(p, 16)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.AdamWStates([torch.ones(3)])
    with pytest.raises(ValueError, match="contiguous"):
        ops.AdamWStates([torch.ones(4, 4, device=cuda_device).T])
    with pytest.raises(TypeError, match="share a dtype"):
        ops.AdamWStates([p[0], p[0].half()])
    with pytest.raises(TypeError, match="unsupported dtype"):
        ops.AdamWStates([p[0].double()])
    with pytest.raises(ValueError, match="need their scales"):
        ops.AdamWStates(p, 8, [p[0].to(torch.float8_e4m3fn)], [p[0].to(torch.float8_e4m3fn)])
    with pytest.raises(TypeError, match="must be torch.float32"):
        ops.AdamWStates(p, 32, [p[0].half()], [p[0].half()])
    states = ops.AdamWStates(p)
    for gradients, hyper, error, match in (
        ([], {}, ValueError, "equal lengths"),
        ([p[0][:200]], {}, ValueError, "sizes differ"),
        ([p[0].cpu()], {}, ValueError, "device"),
        (p, {"epsilon": 0.0}, ValueError, "epsilon"),
        (p, {"beta1": 1.0}, ValueError, "betas"),
        (p, {"step": 0}, ValueError, "from 1"),
        (p, {"step": [1, 2]}, ValueError, "one for each"),
        (p, {"gradient_scale": torch.ones(2, device=cuda_device)}, ValueError, "gradient_scale"),
        ([p[0].double()], {}, TypeError, "unsupported dtype"),
    ):
        with pytest.raises(error, match=match):
            states.step(gradients, **{**HYPER, "step": 1, **hyper})
    assert math.isclose(p[0].sum().item(), 300.0)
