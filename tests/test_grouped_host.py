"""Output strides of the grouped products, checked before any CUDA call."""

from __future__ import annotations

import ctypes

import pytest

from gram_newton_schulz_ampere_b200 import _native, build

LAYOUT = "overlap"


@pytest.fixture(scope="module")
def library() -> ctypes.CDLL:
    if build.is_stale():
        build.build()
    return _native.load()


@pytest.mark.parametrize("stride", [7, 1, 0, -8])
def test_rows_of_the_output_may_not_overlap(library, stride):
    place = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)
    rc = library.gns_grouped_gemm(1, 8, 8, 8, 2, place, 8, place, 64, 8, 1, place, 32, place, 1, stride, None)
    assert rc < 0 and LAYOUT in library.gns_last_error().decode()
    rc = library.gns_grouped_gemm_reduce(1, 8, 8, 8, 2, place, 8, place, 8, place, 32, place, 1, 64, stride, None)
    assert rc < 0 and LAYOUT in library.gns_last_error().decode()


@pytest.mark.parametrize("stride", [63, 8, 0, -64])
def test_groups_of_the_output_may_not_overlap(library, stride):
    place = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)
    rc = library.gns_grouped_gemm_reduce(1, 8, 8, 8, 2, place, 8, place, 8, place, 32, place, 1, stride, 8, None)
    assert rc < 0 and LAYOUT in library.gns_last_error().decode()
