"""Argument checks of the 8-bit products, the RMS norm and the distillation loss that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from gram_newton_schulz_ampere_b200 import _native, build, ops, training


@pytest.fixture(scope="module")
def library() -> ctypes.CDLL:
    if build.is_stale():
        build.build()
    return _native.load()


def failure(library, rc: int) -> str:
    assert rc < 0
    return library.gns_last_error().decode()


def test_no_cpu_path():
    x, w = torch.ones(4, 128), torch.ones(128)
    codes, scales = torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.ones(4, 1)
    index, teacher = torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2)
    for call in (
        lambda: ops.quantize_8bit(x),
        lambda: ops.gemm_8bit(codes, scales, codes.t(), torch.ones(1, 1)),
        lambda: ops.rms_norm(x, w),
        lambda: ops.rms_norm_8bit(x, w),
        lambda: ops.rms_norm_backward(x, x, w, torch.ones(4)),
        lambda: ops.distillation_loss(x, index, teacher),
        lambda: ops.distillation_loss_gradient(torch.ones(4), x, index, teacher),
        lambda: ops.distillation_loss_backward(torch.ones(4), x, index, teacher, torch.ones(4, 2)),
        lambda: training.rms_norm(x, w),
        lambda: training.linear_8bit(x.bfloat16(), x.bfloat16()),
        lambda: training.rms_norm_linear_8bit(x.bfloat16(), w, x.bfloat16()),
        lambda: training.distillation_loss(x, index, teacher),
    ):
        with pytest.raises(ValueError, match="CUDA tensors"):
            call()


def test_layers_check_their_arguments():
    x = torch.ones(4, 128)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        training.linear_8bit(x, x)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        training.rms_norm_linear_8bit(x.half(), x[0], x.bfloat16())
    with pytest.raises(ValueError, match="out, in"):
        training.linear_8bit(x.half(), x[:, :64].half())
    with pytest.raises(ValueError, match="size zero"):
        training.linear_8bit(x[:, :0].half(), x[:, :0].half())
    index, teacher = torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2)
    with pytest.raises(ValueError, match="no gradient"):
        training.distillation_loss(x, index, teacher.requires_grad_())
    with pytest.raises(ValueError, match="top"):
        training.distillation_loss(x, index[:3], teacher.detach())


def test_native_products_check_their_arguments(library):
    place = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)

    def gemm(m=4, n=4, k=128, left=place, lr=128, ls=place, right=place, rr=1, rc=128, rs=place, out=place, dt=1, ldd=4):
        return library.gns_gemm_8bit(m, n, k, left, lr, ls, 1, 4, right, rr, rc, rs, 1, 1, out, dt, ldd, None)

    assert "dtype" in failure(library, gemm(dt=3))
    assert "negative" in failure(library, gemm(m=-1))
    assert "k > 0" in failure(library, gemm(k=0))
    assert "limits" in failure(library, gemm(n=1 << 23, ldd=1 << 23))
    assert "limits" in failure(library, gemm(k=1 << 25))
    assert "limits" in failure(library, gemm(m=1 << 30, n=1 << 20, ldd=1 << 20))
    for name in ("left", "ls", "right", "rs", "out"):
        assert "null" in failure(library, gemm(**{name: None}))
    assert "overlap" in failure(library, gemm(ldd=3))
    assert "unit stride" in failure(library, gemm(rr=2, rc=128))
    assert "unit stride" in failure(library, gemm(rr=1, rc=130))
    assert gemm(m=0) == 0 and gemm(n=0) == 0

    def quantize(dt=1, block=1, rows=4, cols=130, x=place, xr=130, codes=place, ld=144, scales=place):
        return library.gns_quantize_8bit(dt, block, rows, cols, x, xr, codes, ld, scales, 1, 4, None)

    assert "dtype" in failure(library, quantize(dt=7))
    assert "1 or 128" in failure(library, quantize(block=2))
    assert "negative" in failure(library, quantize(rows=-1))
    assert "null" in failure(library, quantize(x=None))
    assert "16 bytes" in failure(library, quantize(ld=130))
    assert "16 bytes" in failure(library, quantize(ld=128))
    assert "stride" in failure(library, quantize(xr=100))
    assert quantize(rows=0) == 0 and quantize(cols=0) == 0


def test_native_norm_checks_its_arguments(library):
    place = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)

    def forward(dt=1, rows=4, cols=8, x=place, xr=8, residual=None, rr=0, weight=place, y=place, total=None, rstd=place):
        return library.gns_rms_norm_forward(dt, 1, rows, cols, x, xr, residual, rr, weight, 1e-5, y, total, rstd, None)

    assert "dtype" in failure(library, forward(dt=4))
    assert "cols" in failure(library, forward(cols=0))
    assert "stride" in failure(library, forward(xr=4))
    assert "stride" in failure(library, forward(residual=place, rr=4, total=place))
    for name in ("x", "weight", "y", "rstd"):
        assert "null" in failure(library, forward(**{name: None}))
    assert "null" in failure(library, forward(residual=place, rr=8))  # nowhere for the sum
    assert forward(rows=0) == 0

    def eight(cols=8, codes=place, ld=16, scales=place):
        return library.gns_rms_norm_forward_8bit(1, 1, 4, cols, place, 8, None, 0, place, 1e-5, codes, ld, scales, 1, 4, None, place, None)

    assert "null" in failure(library, eight(codes=None))
    assert "16 bytes" in failure(library, eight(ld=8))

    def backward(rows=4, grad=place, dw=place, workspace=None, nbytes=0, gr=8):
        return library.gns_rms_norm_backward(1, 1, rows, 8, grad, gr, place, 8, place, place, None, 0, place, dw, workspace, nbytes, None)

    assert "null" in failure(library, backward(grad=None))
    assert "null" in failure(library, backward(dw=None))
    assert "stride" in failure(library, backward(gr=7))
    assert "workspace" in failure(library, backward())
    assert library.gns_rms_norm_backward_workspace_size(0, 8) == 0
    assert library.gns_rms_norm_backward_workspace_size(100, 8) >= 8 * 4


def test_native_loss_checks_its_arguments(library):
    place = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)

    def loss(dt=1, rows=4, v=100, top=3, z=place, zr=100, index=place, bits=64, teacher=place, t=1.0, grad=None, out=place,
             stats=None, dz=None):
        return library.gns_distillation_loss(dt, rows, v, top, z, zr, index, bits, 3, teacher, 2, 3, t, grad, out, stats, dz, 100, None)

    assert "dtype" in failure(library, loss(dt=5))
    assert "32 or 64" in failure(library, loss(bits=16))
    assert "vocabulary" in failure(library, loss(v=0))
    assert "1024" in failure(library, loss(top=1025))
    assert "too large" in failure(library, loss(v=1 << 29))
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-5):
        assert "temperature" in failure(library, loss(t=t))
    assert "null" in failure(library, loss(z=None))
    assert "null" in failure(library, loss(index=None))
    assert "earlier call" in failure(library, loss(out=None))
    assert "earlier call" in failure(library, loss(out=None, grad=place, dz=place))
    assert "together" in failure(library, loss(grad=place))
    assert "stride" in failure(library, loss(zr=99))
    assert loss(rows=0) == 0
