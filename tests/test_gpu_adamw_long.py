"""AdamW over tensors long enough that a warp steps many blocks, with the bounds of test_gpu_adamw_states.py.

A CTA's chunk grows from 2048 to 32768 elements where a call has more than 8 of the
shorter ones for each of 148 SMs (32 with 32-bit states): above 2.4, 4.8, 9.7 and
19.4 million elements with 8-bit states, 9.7 to 77.6 with 32-bit ones. A warp of the
8-bit kernel then steps 2 to 16 blocks of 256 through a ring of four."""

from __future__ import annotations

import pytest
import torch

from gram_newton_schulz_ampere_b200 import ops
from test_gpu_adamw_states import check_step, tensors

pytestmark = pytest.mark.gpu

TYPES = [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32), (torch.bfloat16, torch.float32),
         (torch.float16, torch.bfloat16)]
# Not multiples of a chunk, a block or 8; one tensor a whole number of chunks; small ones beside them.
SIZES = [[2_500_011, 300, 7], [5_000_001, 32768, 1], [9_000_000, 999_999], [77, 21_000_123, 2048 * 16 + 5, 256]]


def run(states, grads, gen):
    for step in (1, 2):
        check_step(states, grads, step)
        for g in grads:
            g.copy_(torch.randn(g.shape, generator=gen, device=g.device) * 1e-2)


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("p_dtype,g_dtype", TYPES)
def test_8_bit_states(cuda_device, sizes, p_dtype, g_dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    params, grads = tensors(gen, sizes, p_dtype, g_dtype, cuda_device)
    run(ops.AdamWStates(params, 8), grads, gen)


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("p_dtype,g_dtype", TYPES)
def test_8_bit_states_that_start_anywhere(cuda_device, sizes, p_dtype, g_dtype):
    """Parameters, gradients and codes packed into flat buffers, at offsets of their own."""
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    total = sum(sizes)
    (p,), (g,) = tensors(gen, [total + 3], p_dtype, g_dtype, cuda_device)
    held = torch.zeros((2, total + 9), dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn)
    counts = [(n + 255) // 256 for n in sizes]
    scales = torch.zeros((2, sum(counts)), device=cuda_device)
    states = ops.AdamWStates(
        list(p[1:-2].split(sizes)), 8, list(held[0, 5:-4].split(sizes)), list(held[1, 2:-7].split(sizes)),
        list(scales[0].split(counts)), list(scales[1].split(counts)))
    ends = p[[0, -2, -1]].clone()
    run(states, list(g[3:].split(sizes)), gen)
    assert torch.equal(p[[0, -2, -1]], ends)  # what lies around them is as it was
    for row, a in ((held[0], 5), (held[1], 2)):
        bytes_ = row.view(torch.uint8)
        assert not bytes_[:a].any() and not bytes_[a + total:].any()


@pytest.mark.parametrize("sizes", [[12_000_011, 40], [80_000_003, 9]])
@pytest.mark.parametrize("p_dtype,g_dtype", TYPES[:2])
@pytest.mark.parametrize("offset", [0, 1])
def test_32_bit_states(cuda_device, sizes, p_dtype, g_dtype, offset):
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    params, grads = tensors(gen, [n + offset for n in sizes], p_dtype, g_dtype, cuda_device)
    states = ops.AdamWStates([p[offset:] for p in params], 32)
    run(states, [g[offset:] for g in grads], gen)
