"""Argument checks of the training operators that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from gram_newton_schulz_ampere_b200 import _native, build, ops


@pytest.fixture(scope="module")
def library() -> ctypes.CDLL:
    if build.is_stale():
        build.build()
    return _native.load()


def test_no_cpu_path():
    x, w = torch.ones(4, 8), torch.ones(8)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.layer_norm(x, w, None, 1e-5)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.grouped_gemm(x.bfloat16(), torch.ones(2, 8, 4, dtype=torch.bfloat16), torch.tensor([2, 4]))
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.grouped_gemm_reduce(x.bfloat16(), x.bfloat16(), torch.tensor([2, 4]))
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.AdamWStates([w])


def test_empty_list_of_parameters():
    states = ops.AdamWStates([])
    states.step([], 1e-3, 0.9, 0.95, 1e-8, 0.0, 1)
    with pytest.raises(ValueError, match="epsilon"):
        states.step([], 1e-3, 0.9, 0.95, 0.0, 0.0, 1)


def failure(library, rc: int) -> str:
    assert rc < 0
    return library.gns_last_error().decode()


def test_native_calls_check_their_arguments(library):
    """Bad arguments are refused with a message before any CUDA call."""
    none = [None] * 6
    step = library.gns_adamw_states_step
    assert step(0, *none, None, 1, 1, 8, None, None, 0.9, 0.1, 0.9, 0.1, 1e-8, 1.0, None, None) == 0
    assert "state_bits" in failure(library, step(0, *none, None, 1, 1, 4, None, None, 0.9, 0.1, 0.9, 0.1, 1e-8, 1.0, None, None))
    assert "dtype" in failure(library, step(0, *none, None, 3, 1, 8, None, None, 0.9, 0.1, 0.9, 0.1, 1e-8, 1.0, None, None))
    assert "list" in failure(library, step(1, *none, None, 1, 1, 8, None, None, 0.9, 0.1, 0.9, 0.1, 1e-8, 1.0, None, None))

    rows = library.gns_grouped_gemm
    assert "F16 or BF16" in failure(library, rows(2, 8, 8, 8, 2, None, 8, None, 64, 8, 1, None, 32, None, 1, 8, None))
    assert "32 or 64" in failure(library, rows(1, 8, 8, 8, 2, None, 8, None, 64, 8, 1, None, 16, None, 1, 8, None))
    assert "1024" in failure(library, rows(1, 8, 8, 8, 1025, None, 8, None, 64, 8, 1, None, 32, None, 1, 8, None))
    assert "negative" in failure(library, rows(1, -1, 8, 8, 2, None, 8, None, 64, 8, 1, None, 32, None, 1, 8, None))
    assert "null" in failure(library, rows(1, 8, 8, 8, 2, None, 8, None, 64, 8, 1, None, 32, None, 1, 8, None))
    assert rows(1, 0, 8, 8, 2, None, 8, None, 64, 8, 1, None, 32, None, 1, 8, None) == 0
    place = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)
    assert "unit stride" in failure(library, rows(1, 8, 8, 8, 2, place, 8, place, 64, 16, 2, place, 32, place, 1, 8, None))

    reduce = library.gns_grouped_gemm_reduce
    assert "output dtype" in failure(library, reduce(1, 8, 8, 8, 2, None, 8, None, 8, None, 32, None, 7, 64, 8, None))
    assert reduce(1, 8, 8, 8, 0, None, 8, None, 8, None, 32, None, 1, 64, 8, None) == 0

    forward = library.gns_layer_norm_forward
    assert "cols" in failure(library, forward(1, 1, 4, 0, None, 8, None, None, 1e-5, None, None, None, None))
    assert "stride" in failure(library, forward(1, 1, 4, 8, None, 4, None, None, 1e-5, None, None, None, None))
    assert "null" in failure(library, forward(1, 1, 4, 8, None, 8, None, None, 1e-5, None, None, None, None))
    assert forward(1, 1, 0, 8, None, 8, None, None, 1e-5, None, None, None, None) == 0
    backward = library.gns_layer_norm_backward
    assert "dtype" in failure(library, backward(1, 5, 4, 8, None, 8, None, 8, None, None, None, None, None, None, None, 0, None))
    assert library.gns_layer_norm_backward_workspace_size(0, 8) == 0
    assert library.gns_layer_norm_backward_workspace_size(100, 8) >= 2 * 8 * 4
