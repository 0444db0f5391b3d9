"""Where the statistics of a distillation loss may lie: the kernels read and write a row's two at once."""

from __future__ import annotations

import ctypes

import pytest
import torch

from gram_newton_schulz_ampere_b200 import _native, ops


def test_native_call_refuses_statistics_off_eight_bytes(native_lib):
    place = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)

    def call(loss, grad, dlogits, stats):
        return native_lib.gns_distillation_loss(1, 4, 100, 3, place, 100, place, 64, 3, place, 2, 3, 1.0, grad, loss, stats,
                                                dlogits, 100, None)

    # Never reaches a launch: refused before the device is looked up.
    for arguments in ((place, None, None), (None, place, place), (place, place, place)):
        assert call(*arguments, ctypes.c_void_p(4100)) < 0
        assert b"8 bytes" in _native.load().gns_last_error()


@pytest.mark.gpu
def test_gradient_from_statistics_at_an_odd_offset(cuda_device):
    rows, vocabulary, top = 37, 501, 6
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    logits = torch.randn(rows, vocabulary, generator=gen, device=cuda_device)
    indices = torch.randint(-1, vocabulary, (rows, top), generator=gen, device=cuda_device)
    teacher = torch.randn(rows, top, generator=gen, device=cuda_device)
    grad = torch.rand(rows, generator=gen, device=cuda_device)
    _, statistics = ops.distillation_loss(logits, indices, teacher, 2.0)
    want = ops.distillation_loss_backward(grad, logits, indices, teacher, statistics, 2.0)
    kept = torch.zeros(1 + 2 * rows, device=cuda_device)
    odd = kept[1:].view(rows, 2).copy_(statistics)
    assert odd.data_ptr() % 8 == 4 and odd.is_contiguous()
    assert torch.equal(ops.distillation_loss_backward(grad, logits, indices, teacher, odd, 2.0), want)
