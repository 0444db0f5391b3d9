"""Tensor-level wrappers of the sm_100a kernels (C ABI in include/gns_b200.h).

Each function validates its tensors, allocates outputs and workspaces with
torch (so the caching allocator owns all memory), and launches on the current
CUDA stream of the tensors' device. There is no CPU path: non-CUDA tensors are
rejected and a missing native library raises.
"""

from __future__ import annotations

import array
import contextlib
import ctypes
import os
from collections.abc import Iterator, Sequence
from typing import cast

import torch
from torch import Tensor

from gram_newton_schulz_ampere_b200 import _native as nat


# ----------------------------------------------------- bounded-wait status
class DeviceWaitError(nat.NativeError):
    """A kernel's bounded wait ran out; its results are invalid (NaN where the
    normalisation gave up)."""


_status = {"enabled": os.environ.get("GNS_B200_CHECK_STATUS", "") not in ("", "0"), "depth": 0}


def set_status_checks(enabled: bool) -> bool:
    """Opt in (or out) of a device-status check after every public call
    (``GramNewtonSchulz.__call__``, ``Muon.step``, ``Dion3.step``; also set by the
    environment variable GNS_B200_CHECK_STATUS=1). Each check synchronises the
    device once per outermost call. Returns the previous setting."""
    previous = bool(_status["enabled"])
    _status["enabled"] = bool(enabled)
    return previous


def check_device_status() -> None:
    """Reads and clears the device status word; raises DeviceWaitError if a
    kernel's bounded wait ran out since the last read."""
    code = nat.device_status(clear=True)
    if code != 0:
        raise DeviceWaitError(f"a kernel's bounded wait ran out (device status {code}); results are invalid")


@contextlib.contextmanager
def status_checked() -> Iterator[None]:
    """Runs the body and, when checks are enabled, checks the device status once
    at the end of the outermost such block."""
    _status["depth"] += 1
    try:
        yield
    finally:
        _status["depth"] -= 1
    if _status["depth"] == 0 and _status["enabled"]:
        check_device_status()


def _require_cuda(*tensors: Tensor | None) -> torch.device:
    device = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("gram_newton_schulz_ampere_b200 kernels require CUDA tensors")
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError("all tensors must be on the same CUDA device")
    if device is None:
        raise ValueError("no tensor given")
    return device


def _device_index(*tensors: Tensor | None) -> int:
    """``_require_cuda`` for the calls whose host time counts: the device's index."""
    index = -1
    for t in tensors:
        if t is None:
            continue
        here = t.get_device()
        if here < 0:
            raise ValueError("gram_newton_schulz_ampere_b200 kernels require CUDA tensors")
        if index < 0:
            index = here
        elif here != index:
            raise ValueError("all tensors must be on the same CUDA device")
    if index < 0:
        raise ValueError("no tensor given")
    return index


def _workspace(nbytes: int, device: torch.device) -> Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


def _as_batched(t: Tensor) -> Tensor:
    if t.ndim == 2:
        return t.unsqueeze(0)
    if t.ndim == 3:
        return t
    raise ValueError("expected a matrix or a batch of matrices")


def _aligned_operand(t: Tensor) -> Tensor:
    """Returns `t` if a TMA tile load can read it (unit stride on one matrix axis,
    16-byte aligned base and strides), else a copy whose row pitch is padded to a
    multiple of 8 elements. The copy is layout plumbing only."""
    es = t.element_size()
    b, r, c = t.shape
    sb, sr, sc = t.stride()
    base_ok = t.data_ptr() % 16 == 0

    def ok_stride(s: int, extent: int) -> bool:
        return extent == 1 or (s * es) % 16 == 0

    if base_ok and (sc == 1 or c == 1) and ok_stride(sr, r) and ok_stride(sb, b):
        return t
    if base_ok and (sr == 1 or r == 1) and ok_stride(sc, c) and ok_stride(sb, b):
        return t
    pitch = (c + 7) // 8 * 8
    padded = torch.empty((b, r, pitch), dtype=t.dtype, device=t.device)
    view = padded[:, :, :c]
    view.copy_(t)
    return view


def gemm(
    left: Tensor,
    right: Tensor,
    accumulator: Tensor | None = None,
    alpha: float = 1.0,
    beta: float = 0.0,
    symmetric: bool = False,
    out_dtype: torch.dtype | None = None,
) -> Tensor:
    """``alpha * left @ right + beta * accumulator`` on tcgen05 tensor cores.

    left [B, m, k] and right [B, k, n] share dtype float16 or bfloat16; either may
    be a transposed view. With ``symmetric=True`` the caller asserts the result is
    symmetric: only its upper triangle is computed and mirrored (exactly symmetric
    output), as the reference's symmetric CUTLASS kernels do
    (kernels/cutlass_ns.cu:167-223 + mirror_lower_triangle :127-165).
    When beta == 0 the accumulator is never read (NaNs in it do not propagate,
    matching torch.baddbmm). Inside a region that torch.compile traces, the call
    is the custom op ``torch.ops.gns_b200.gemm``.
    """
    if torch.compiler.is_compiling():
        return torch.ops.gns_b200.gemm(left, right, accumulator, float(alpha), float(beta), bool(symmetric),
                                       out_dtype)
    return _gemm_eager(left, right, accumulator, alpha, beta, symmetric, out_dtype)


def _gemm_eager(
    left: Tensor,
    right: Tensor,
    accumulator: Tensor | None = None,
    alpha: float = 1.0,
    beta: float = 0.0,
    symmetric: bool = False,
    out_dtype: torch.dtype | None = None,
) -> Tensor:
    index = _device_index(left, right, accumulator)
    squeeze = left.ndim == 2
    a = _as_batched(left)
    b = _as_batched(right)
    if a.dtype != b.dtype or a.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("left and right must share dtype float16 or bfloat16")
    if a.shape[0] != b.shape[0] or a.shape[2] != b.shape[1]:
        raise ValueError(f"incompatible shapes {tuple(left.shape)} @ {tuple(right.shape)}")
    batch, m, k = a.shape
    n = b.shape[2]
    if symmetric and m != n:
        raise ValueError("a symmetric product must be square")
    dtype = out_dtype or a.dtype
    out = left.new_empty((batch, m, n), dtype=dtype)
    if batch == 0 or m == 0 or n == 0:
        return out[0] if squeeze else out
    if k == 0:
        out.zero_()
        if accumulator is not None and beta != 0.0:
            out.add_(_as_batched(accumulator).expand(batch, m, n), alpha=beta)
        return out[0] if squeeze else out
    a = _aligned_operand(a)
    b = _aligned_operand(b)
    c = None
    if accumulator is not None and beta != 0.0:
        c = _as_batched(accumulator)
        if c.shape != (batch, m, n):
            c = c.expand(batch, m, n)
        if c.dtype != dtype:
            c = c.to(dtype)
        if c.stride(-1) != 1 or (batch > 1 and c.stride(0) == 0):
            c = c.contiguous()
    lib = nat.load()
    with nat.on_device(index) as stream:
        rc = lib.gns_gemm(
            nat.dtype_code(a.dtype), batch, m, n, k,
            a.data_ptr(), a.stride(0), a.stride(1), a.stride(2),
            b.data_ptr(), b.stride(0), b.stride(1), b.stride(2),
            nat.ptr(c), nat.dtype_code(c.dtype) if c is not None else 0,
            c.stride(0) if c is not None else 0, c.stride(1) if c is not None else 0,
            out.data_ptr(), nat.dtype_code(dtype), out.stride(0), out.stride(1),
            float(alpha), float(beta) if c is not None else 0.0, 1 if symmetric else 0,
            stream,
        )
    nat.check(rc, "gns_gemm")
    return out[0] if squeeze else out


@torch.library.custom_op("gns_b200::gemm", mutates_args=())
def _gemm_op(
    left: Tensor, right: Tensor, accumulator: Tensor | None, alpha: float, beta: float, symmetric: bool,
    out_dtype: torch.dtype | None,
) -> Tensor:
    return _gemm_eager(left, right, accumulator, alpha, beta, symmetric, out_dtype)


@_gemm_op.register_fake
def _(left, right, accumulator, alpha, beta, symmetric, out_dtype):  # type: ignore[no-untyped-def]
    shape = (left.shape[-2], right.shape[-1]) if left.ndim == 2 else (left.shape[0], left.shape[-2], right.shape[-1])
    return torch.empty(shape, dtype=out_dtype or left.dtype, device=left.device)


def frobenius_normalize(matrix: Tensor, epsilon: float) -> Tensor:
    """fp16(X / (||X||_F + eps)) per matrix, norm in fp32 (newton_schulz.py:141-144)."""
    device = _require_cuda(matrix)
    x = _as_batched(matrix)
    if x.stride(-1) != 1:
        x = x.contiguous()
    batch, rows, cols = x.shape
    ld = (cols + 7) // 8 * 8
    out = torch.empty((batch, rows, ld), dtype=torch.float16, device=device)[:, :, :cols]
    lib = nat.load()
    ws = _workspace(lib.gns_normalize_workspace_size(batch, rows, cols), device)
    with torch.cuda.device(device):
        rc = lib.gns_frobenius_normalize(
            nat.dtype_code(x.dtype), batch, rows, cols, x.data_ptr(), x.stride(0), x.stride(1),
            out.data_ptr(), ld, float(epsilon), ws.data_ptr(), ws.numel(), nat.stream_handle(device),
        )
    nat.check(rc, "gns_frobenius_normalize")
    return out if matrix.ndim == 3 else out[0]


def _coefficient_array(coefficients: Sequence[Sequence[float]]) -> ctypes.Array:
    flat = [float(v) for triple in coefficients for v in triple]
    if len(flat) != 3 * len(coefficients):
        raise ValueError("each coefficient entry must be an (a, b, c) triple")
    return (ctypes.c_double * max(len(flat), 1))(*flat)


def _chain_input(matrix: Tensor) -> Tensor:
    x = _as_batched(matrix)
    if x.stride(-1) != 1:
        x = x.contiguous()
    return x


def newton_schulz_chain(
    matrix: Tensor,
    coefficients: Sequence[Sequence[float]],
    epsilon: float,
    gram: bool,
    reset_iterations: Sequence[int] = (),
    out_dtype: torch.dtype | None = None,
) -> Tensor:
    """Whole (Gram) Newton-Schulz orthogonalisation of [B, r, c] in one native call.

    Follows build_gram_newton_schulz_operation / build_standard_newton_schulz_operation
    (newton_schulz.py:66-223): fp32 Frobenius normalisation, fp16 products with fp32
    accumulation, output cast to ``out_dtype`` (default: the input dtype). Inside a
    region that torch.compile traces, the call is the custom op
    ``torch.ops.gns_b200.newton_schulz_chain`` (same kernels, no graph break).
    """
    if torch.compiler.is_compiling():
        return torch.ops.gns_b200.newton_schulz_chain(
            matrix, [float(v) for triple in coefficients for v in triple], float(epsilon), bool(gram),
            [int(i) for i in reset_iterations], out_dtype or matrix.dtype,
        )
    return _newton_schulz_chain_eager(matrix, coefficients, epsilon, gram, reset_iterations, out_dtype)


def _newton_schulz_chain_eager(
    matrix: Tensor,
    coefficients: Sequence[Sequence[float]],
    epsilon: float,
    gram: bool,
    reset_iterations: Sequence[int] = (),
    out_dtype: torch.dtype | None = None,
) -> Tensor:
    device = _require_cuda(matrix)
    x = _chain_input(matrix)
    batch, rows, cols = x.shape
    dtype = out_dtype or matrix.dtype
    out = torch.empty((batch, rows, cols), dtype=dtype, device=device)
    if len(coefficients) > 32:
        raise ValueError("at most 32 Newton-Schulz iterations are supported")
    mask = 0
    for it in reset_iterations:
        if it < 0:
            raise ValueError("reset iterations must be non-negative")
        if it < 32:
            mask |= 1 << int(it)
    coeffs = _coefficient_array(coefficients)
    lib = nat.load()
    ws = _workspace(lib.gns_newton_schulz_workspace_size(batch, rows, cols), device)
    with torch.cuda.device(device):
        if gram:
            rc = lib.gns_gram_newton_schulz(
                nat.dtype_code(x.dtype), batch, rows, cols, x.data_ptr(), x.stride(0), x.stride(1),
                out.data_ptr(), nat.dtype_code(dtype), out.stride(0), out.stride(1),
                coeffs, len(coefficients), mask, float(epsilon), ws.data_ptr(), ws.numel(),
                nat.stream_handle(device),
            )
        else:
            rc = lib.gns_standard_newton_schulz(
                nat.dtype_code(x.dtype), batch, rows, cols, x.data_ptr(), x.stride(0), x.stride(1),
                out.data_ptr(), nat.dtype_code(dtype), out.stride(0), out.stride(1),
                coeffs, len(coefficients), float(epsilon), ws.data_ptr(), ws.numel(),
                nat.stream_handle(device),
            )
    if rc != 0:
        msg = nat.last_error()
        if "requires coefficients" in msg or "no accumulated update" in msg:
            raise RuntimeError(msg)
        nat.check(rc, "Newton-Schulz chain")
    return out if matrix.ndim == 3 else out[0]


@torch.library.custom_op("gns_b200::newton_schulz_chain", mutates_args=())
def _newton_schulz_chain_op(
    matrix: Tensor, coefficients: list[float], epsilon: float, gram: bool, reset_iterations: list[int],
    out_dtype: torch.dtype,
) -> Tensor:
    triples = [coefficients[i:i + 3] for i in range(0, len(coefficients), 3)]
    return _newton_schulz_chain_eager(matrix, triples, epsilon, gram, reset_iterations, out_dtype)


@_newton_schulz_chain_op.register_fake
def _(matrix, coefficients, epsilon, gram, reset_iterations, out_dtype):  # type: ignore[no-untyped-def]
    # The output has the input's shape and is contiguous, like the native call's.
    return torch.empty(matrix.shape, dtype=out_dtype, device=matrix.device)


# ------------------------------------------------ sharded-chain pieces
@contextlib.contextmanager
def small_chain_tactic(enabled: bool) -> Iterator[None]:
    """Within the block, Gram Newton-Schulz calls on matrices with a short side of
    at most 128 run as one fused kernel (``enabled``, the default) or as one GEMM
    launch per product; the previous setting is restored on exit. The switch is
    process-wide (``gns_set_small_chain``)."""
    lib = nat.load()
    previous = lib.gns_set_small_chain(1 if enabled else 0)
    try:
        yield
    finally:
        lib.gns_set_small_chain(previous)


def gemm_sm_limit(sms: int) -> int:
    """Caps the SMs each GEMM launch occupies (0: all), process-wide; returns the
    previous cap (``gns_set_gemm_sm_limit``)."""
    return int(nat.load().gns_set_gemm_sm_limit(int(sms)))


def _padded(batch: int, rows: int, cols: int, dtype: torch.dtype, device: torch.device) -> Tensor:
    """[batch, rows, cols] view of a buffer whose row pitch is a multiple of 8 elements."""
    pitch = (cols + 7) // 8 * 8
    return torch.empty((batch, rows, pitch), dtype=dtype, device=device)[:, :, :cols]


def frobenius_sumsq(matrix: Tensor) -> Tensor:
    """Per-matrix sum of squares in fp32 (fixed summation order), shape [batch]."""
    device = _require_cuda(matrix)
    x = _chain_input(matrix)
    batch, rows, cols = x.shape
    out = torch.empty(batch, dtype=torch.float32, device=device)
    lib = nat.load()
    ws = _workspace(lib.gns_normalize_workspace_size(batch, rows, cols), device)
    with torch.cuda.device(device):
        rc = lib.gns_frobenius_sumsq(
            nat.dtype_code(x.dtype), batch, rows, cols, x.data_ptr(), x.stride(0), x.stride(1), out.data_ptr(),
            ws.data_ptr(), ws.numel(), nat.stream_handle(device),
        )
    nat.check(rc, "gns_frobenius_sumsq")
    return out


def frobenius_scale(matrix: Tensor, sumsq: Tensor, epsilon: float) -> Tensor:
    """fp16(X / (sqrt(sumsq) + eps)) per matrix, for a sum of squares computed elsewhere."""
    device = _require_cuda(matrix, sumsq)
    x = _chain_input(matrix)
    batch, rows, cols = x.shape
    if sumsq.dtype != torch.float32 or sumsq.numel() != batch:
        raise ValueError("sumsq must hold one fp32 value per matrix")
    out = _padded(batch, rows, cols, torch.float16, device)
    lib = nat.load()
    with torch.cuda.device(device):
        rc = lib.gns_frobenius_scale(
            nat.dtype_code(x.dtype), batch, rows, cols, x.data_ptr(), x.stride(0), x.stride(1),
            sumsq.contiguous().data_ptr(), float(epsilon), out.data_ptr(), out.stride(1), nat.stream_handle(device),
        )
    nat.check(rc, "gns_frobenius_scale")
    return out


def gram_iterations(
    gram: Tensor,
    coefficients: Sequence[Sequence[float]],
    it_begin: int,
    it_end: int,
) -> Tensor:
    """Runs Gram iterations [it_begin, it_end) between two restarts from G (fp32 or
    fp16 [B, m, m], rounded to fp16); returns the accumulated polynomial Q in fp16."""
    device = _require_cuda(gram)
    g = _as_batched(gram)
    if g.dtype not in (torch.float32, torch.float16) or g.stride(-1) != 1:
        g = g.float().contiguous()
    batch, m, _ = g.shape
    q = _padded(batch, m, m, torch.float16, device)
    coeffs = _coefficient_array(coefficients)
    lib = nat.load()
    ws = _workspace(lib.gns_gram_iterations_workspace_size(batch, m), device)
    with torch.cuda.device(device):
        rc = lib.gns_gram_iterations(
            batch, m, g.data_ptr(), 1 if g.dtype == torch.float32 else 0, g.stride(0), g.stride(1), coeffs,
            len(coefficients), int(it_begin), int(it_end), q.data_ptr(), q.stride(0), q.stride(1),
            ws.data_ptr(), ws.numel(), nat.stream_handle(device),
        )
    nat.check(rc, "gns_gram_iterations")
    return q if gram.ndim == 3 else q[0]


# ------------------------------------------------------------------- Muon
def _ptr_array(tensors: Sequence[Tensor | None]) -> ctypes.Array:
    return (ctypes.c_void_p * max(len(tensors), 1))(*[0 if t is None else t.data_ptr() for t in tensors])


def muon_momentum(
    gradients: Sequence[Tensor],
    momenta: Sequence[Tensor],
    momentum: float,
    nesterov: bool,
    wanted: Sequence[bool] | None = None,
) -> list[Tensor | None] | None:
    """Fused multi-tensor Muon momentum (muon.py:423-438).

    Updates every momentum buffer in place (m <- g + mu m) and, for Nesterov,
    returns new update tensors u = g + mu m. Returns None when the caller should
    use the gradient (mu == 0) or the momentum buffer itself (no Nesterov).
    ``wanted`` (Nesterov only) limits the update outputs to the marked tensors;
    the others advance their momentum and get None.
    """
    if len(gradients) != len(momenta):
        raise ValueError("gradients and momenta must have equal lengths")
    if not gradients:
        return [] if nesterov and momentum != 0.0 else None
    device = _require_cuda(*gradients, *momenta)
    g_dtype = gradients[0].dtype
    m_dtype = momenta[0].dtype
    for g, m in zip(gradients, momenta, strict=True):
        if g.dtype != g_dtype or m.dtype != m_dtype:
            raise TypeError("all gradients (and all momenta) of one call must share a dtype")
        if g.shape != m.shape:
            raise ValueError("gradient and momentum shapes differ")
        if not (g.is_contiguous() and m.is_contiguous()):
            raise ValueError("gradients and momenta must be contiguous")
    write_update = nesterov and momentum != 0.0
    u_dtype = torch.promote_types(g_dtype, m_dtype)
    if wanted is not None and len(wanted) != len(gradients):
        raise ValueError("wanted must have one flag per gradient")
    updates: list[Tensor | None] | None = None
    if write_update:
        # Updates of one shape are consecutive slices of one buffer, in order, so a
        # bucket of them is already the batch an orthogonaliser takes (no stacking copy).
        by_shape: dict[tuple[int, ...], list[int]] = {}
        for index, g in enumerate(gradients):
            if wanted is None or wanted[index]:
                by_shape.setdefault(tuple(g.shape), []).append(index)
        slots: list[Tensor | None] = [None] * len(gradients)
        for shape, indices in by_shape.items():
            block = torch.empty((len(indices), *shape), dtype=u_dtype, device=device)
            for position, index in enumerate(indices):
                slots[index] = block[position]
        updates = slots
    numel = (ctypes.c_int64 * len(gradients))(*[g.numel() for g in gradients])
    lib = nat.load()
    with torch.cuda.device(device):
        rc = lib.gns_muon_momentum(
            len(gradients), _ptr_array(gradients), _ptr_array(momenta),
            _ptr_array(updates) if updates is not None else None, numel,
            nat.dtype_code(g_dtype), nat.dtype_code(m_dtype), nat.dtype_code(u_dtype),
            float(momentum), 1 if write_update else 0, nat.stream_handle(device),
        )
    nat.check(rc, "gns_muon_momentum")
    return updates


def muon_apply(
    parameters: Sequence[Tensor],
    updates: Sequence[Tensor],
    decay: float | None,
    adjusted_learning_rates: Sequence[float],
) -> None:
    """Fused multi-tensor ``p <- p * decay; p <- p - lr_adj * update`` (muon.py:471-476)."""
    if not parameters:
        return
    if not (len(parameters) == len(updates) == len(adjusted_learning_rates)):
        raise ValueError("parameters, updates and learning rates must have equal lengths")
    device = _require_cuda(*parameters, *updates)
    p_dtype, o_dtype = parameters[0].dtype, updates[0].dtype
    for p, o in zip(parameters, updates, strict=True):
        if p.dtype != p_dtype or o.dtype != o_dtype:
            raise TypeError("all parameters (and all updates) of one call must share a dtype")
        if p.numel() != o.numel():
            raise ValueError("parameter and update sizes differ")
        if not (p.is_contiguous() and o.is_contiguous()):
            raise ValueError("parameters and updates must be contiguous")
    numel = (ctypes.c_int64 * len(parameters))(*[p.numel() for p in parameters])
    lrs = (ctypes.c_float * len(parameters))(*[float(v) for v in adjusted_learning_rates])
    lib = nat.load()
    with torch.cuda.device(device):
        rc = lib.gns_muon_apply(
            len(parameters), _ptr_array(parameters), _ptr_array(updates), numel,
            nat.dtype_code(p_dtype), nat.dtype_code(o_dtype),
            float(decay if decay is not None else 1.0), 0 if decay is None else 1, lrs,
            nat.stream_handle(device),
        )
    nat.check(rc, "gns_muon_apply")


# ------------------------------------------------------------------- Dion3
def _leading(t: Tensor) -> int:
    b = 1
    for s in t.shape[:-2]:
        b *= s
    return b


def dion3_select_rows(
    momentum: Tensor,
    gradient: Tensor,
    parameter: Tensor | None,
    selected_count: int,
    decay: float,
    parameter_decay: float,
) -> tuple[Tensor, Tensor]:
    """Fused momentum + decay + L1 row norm, top-k rows, gather + error-feedback decay.

    Returns (bf16 selected rows [..., k, cols], int64 indices [..., k] ascending).
    Mirrors select_rows (kernels/dion3_cuda.cu:336-351) / select_dion3_rows
    (dion3_update.py:14-70); k == rows selects every row.
    """
    device = _require_cuda(momentum, gradient, parameter)
    if momentum.ndim < 2:
        raise ValueError("momentum must have at least two dimensions")
    if gradient.shape != momentum.shape:
        raise ValueError("momentum and gradient shapes must match")
    if parameter is not None and parameter.shape != momentum.shape:
        raise ValueError("momentum and parameter shapes must match")
    if not momentum.is_contiguous():
        raise ValueError("momentum must be C contiguous")
    grad = gradient.to(dtype=momentum.dtype).contiguous()
    if parameter is not None:
        if parameter.dtype != momentum.dtype or not parameter.is_contiguous():
            raise ValueError("parameter must be contiguous with the momentum dtype")
    rows, cols = momentum.shape[-2], momentum.shape[-1]
    batch = _leading(momentum)
    lead = tuple(momentum.shape[:-2])
    k = int(selected_count)
    if rows == 0:
        momentum.add_(grad)
        if parameter is not None and parameter_decay != 1.0:
            parameter.mul_(parameter_decay)
        return momentum.to(torch.bfloat16), torch.empty((*lead, 0), dtype=torch.long, device=device)
    k = min(k, rows)
    if k < 1:
        raise ValueError("selected_count must be positive")
    selected = torch.empty((*lead, k, cols), dtype=torch.bfloat16, device=device)
    indices = torch.empty((*lead, k), dtype=torch.long, device=device)
    lib = nat.load()
    ws = _workspace(lib.gns_dion3_select_workspace_size(batch, rows), device)
    with torch.cuda.device(device):
        rc = lib.gns_dion3_select_rows(
            nat.dtype_code(momentum.dtype), batch, rows, cols, momentum.data_ptr(), grad.data_ptr(),
            nat.ptr(parameter), k, float(decay),
            float(parameter_decay) if parameter is not None else 1.0,
            selected.data_ptr(), indices.data_ptr(), ws.data_ptr(), ws.numel(), nat.stream_handle(device),
        )
    nat.check(rc, "gns_dion3_select_rows")
    return selected, indices


def dion3_select_rows_multi(
    momenta: Sequence[Tensor],
    gradients: Sequence[Tensor],
    parameters: Sequence[Tensor] | None,
    selected_count: int,
    decay: float,
    parameter_decay: float,
) -> tuple[Tensor, Tensor]:
    """dion3_select_rows over separate same-shape matrices in one set of launches.

    Returns one bf16 stack [n, k, cols] of the selected rows and one int64 stack
    [n, k] of ascending indices (row i is matrix i's selection). Mirrors
    select_dion3_rows_cuda_batch (kernels/dion3_cuda.py:111-149) for a bucket of
    equal shapes and counts.
    """
    count = len(momenta)
    if len(gradients) != count or (parameters is not None and len(parameters) != count):
        raise ValueError("batched selection inputs must have equal lengths")
    if count == 0:
        raise ValueError("batched selection needs at least one matrix")
    device = _require_cuda(*momenta, *gradients, *(parameters or []))
    first = momenta[0]
    if first.ndim != 2:
        raise ValueError("batched selection takes 2-D matrices")
    rows, cols = first.shape
    dtype = first.dtype
    grads = []
    for i, m in enumerate(momenta):
        if m.shape != first.shape or m.dtype != dtype or not m.is_contiguous():
            raise ValueError("batched selection needs contiguous momenta of one shape and dtype")
        if gradients[i].shape != first.shape:
            raise ValueError("momentum and gradient shapes must match")
        grads.append(gradients[i].to(dtype=dtype).contiguous())
        if parameters is not None:
            p = parameters[i]
            if p.shape != first.shape or p.dtype != dtype or not p.is_contiguous():
                raise ValueError("parameters must be contiguous with the momentum shape and dtype")
    k = min(int(selected_count), rows)
    if k < 1 or rows == 0:
        raise ValueError("batched selection requires 1 <= selected_count and rows > 0")
    selected = torch.empty((count, k, cols), dtype=torch.bfloat16, device=device)
    indices = torch.empty((count, k), dtype=torch.long, device=device)
    lib = nat.load()
    ws = _workspace(lib.gns_dion3_select_workspace_size(count, rows), device)
    with torch.cuda.device(device):
        rc = lib.gns_dion3_select_rows_multi(
            nat.dtype_code(dtype), count, rows, cols, _ptr_array(momenta), _ptr_array(grads),
            _ptr_array(parameters) if parameters is not None else None, k, float(decay),
            float(parameter_decay) if parameters is not None else 1.0,
            selected.data_ptr(), indices.data_ptr(), ws.data_ptr(), ws.numel(), nat.stream_handle(device),
        )
    nat.check(rc, "gns_dion3_select_rows_multi")
    return selected, indices


def dion3_normalize_apply_multi(
    parameters: Sequence[Tensor],
    selected_updates: Tensor,
    variances: Sequence[Tensor],
    indices: Tensor,
    beta_two: float,
    epsilon: float,
    learning_rate: float,
    weight_decay: float,
    adjusted_learning_rate: float,
) -> None:
    """dion3_normalize_apply over separate same-shape parameters: ``selected_updates``
    is one [n, k, cols] stack and ``indices`` one [n, k] stack (row i belongs to
    parameter i). Mirrors normalize_apply_rows_cuda_batch (kernels/dion3_cuda.py:220-253)
    for a bucket of equal shapes, counts and adjusted learning rates."""
    count = len(parameters)
    if len(variances) != count or selected_updates.shape[0] != count or indices.shape[0] != count:
        raise ValueError("batched normalization inputs must have equal lengths")
    if count == 0:
        return
    device = _require_cuda(*parameters, *variances, selected_updates, indices)
    first = parameters[0]
    rows, cols = first.shape[-2], first.shape[-1]
    for p, v in zip(parameters, variances, strict=True):
        if p.shape != first.shape or p.dtype != first.dtype or not p.is_contiguous():
            raise ValueError("parameters must be contiguous and share one shape and dtype")
        if v.dtype != torch.float32 or not v.is_contiguous() or v.numel() != rows:
            raise ValueError("variances must be contiguous float32 with one entry per row")
    if indices.dtype != torch.long:
        raise ValueError("indices must be int64")
    k = selected_updates.shape[-2]
    if selected_updates.shape != (count, k, cols) or indices.shape != (count, k):
        raise ValueError("selected_updates must be [n, k, cols] and indices [n, k]")
    u = selected_updates if selected_updates.stride(-1) == 1 else selected_updates.contiguous()
    idx = indices.contiguous()
    lib = nat.load()
    ws = _workspace(lib.gns_dion3_normalize_workspace_size(count, max(k, 1)), device)
    with torch.cuda.device(device):
        rc = lib.gns_dion3_normalize_apply_multi(
            nat.dtype_code(first.dtype), nat.dtype_code(u.dtype), count, rows, cols, k,
            _ptr_array(parameters), u.data_ptr() if k > 0 else None, u.stride(0), u.stride(1),
            _ptr_array(variances), idx.data_ptr() if k > 0 else None,
            float(beta_two), float(epsilon), float(learning_rate), float(weight_decay),
            float(adjusted_learning_rate), ws.data_ptr(), ws.numel(), nat.stream_handle(device),
        )
    nat.check(rc, "gns_dion3_normalize_apply_multi")


def dion3_normalize_apply(
    parameter: Tensor,
    selected_update: Tensor,
    variance: Tensor,
    indices: Tensor,
    beta_two: float,
    epsilon: float,
    learning_rate: float,
    weight_decay: float,
    adjusted_learning_rate: float,
) -> None:
    """NorMuon per-neuron normalisation + norm-preserving rescale + row scatter update
    (kernels/dion3_cuda.cu:353-503; dion3_update.py:73-148)."""
    device = _require_cuda(parameter, selected_update, variance, indices)
    if not parameter.is_contiguous():
        raise ValueError("parameter must be C contiguous")
    if variance.dtype != torch.float32 or not variance.is_contiguous():
        raise ValueError("variance must be contiguous float32")
    if indices.dtype != torch.long:
        raise ValueError("indices must be int64")
    rows, cols = parameter.shape[-2], parameter.shape[-1]
    batch = _leading(parameter)
    k = selected_update.shape[-2]
    if variance.numel() != batch * rows:
        raise ValueError("variance and parameter batch dimensions must match")
    if indices.numel() != batch * k:
        raise ValueError("indices and selected_update shapes must match")
    if selected_update.numel() != batch * k * cols:
        raise ValueError("parameter and selected_update batch dimensions must match")
    u = selected_update.reshape(batch, k, cols)
    if u.stride(-1) != 1:
        u = u.contiguous()
    idx = indices.reshape(batch * k).contiguous() if k > 0 else indices
    lib = nat.load()
    ws = _workspace(lib.gns_dion3_normalize_workspace_size(batch, max(k, 1)), device)
    with torch.cuda.device(device):
        rc = lib.gns_dion3_normalize_apply(
            nat.dtype_code(parameter.dtype), nat.dtype_code(u.dtype), batch, rows, cols, k,
            parameter.data_ptr(), u.data_ptr() if k > 0 else None, u.stride(0), u.stride(1),
            variance.data_ptr(), idx.data_ptr() if k > 0 else None,
            float(beta_two), float(epsilon), float(learning_rate), float(weight_decay),
            float(adjusted_learning_rate), ws.data_ptr(), ws.numel(), nat.stream_handle(device),
        )
    nat.check(rc, "gns_dion3_normalize_apply")


def dion3_normalize_rows(
    selected_update: Tensor,
    variance: Tensor,
    indices: Tensor,
    beta_two: float,
    epsilon: float,
) -> tuple[Tensor, Tensor]:
    """The normalisation half of dion3_normalize_apply (reference kernels/dion3_cuda.cu:353-400):
    updates ``variance`` in place and returns (normalized fp32 [*, k, cols], squared_norms fp32 [batch, 2])."""
    device = _require_cuda(selected_update, variance, indices)
    if variance.dtype != torch.float32 or not variance.is_contiguous():
        raise ValueError("variance must be contiguous float32")
    if indices.dtype != torch.long:
        raise ValueError("indices must be int64")
    k, cols = selected_update.shape[-2], selected_update.shape[-1]
    batch = _leading(selected_update)
    rows = variance.shape[-2]
    if indices.numel() != batch * k:
        raise ValueError("indices and selected_update shapes must match")
    if variance.numel() != batch * rows:
        raise ValueError("variance and selected_update batch dimensions must match")
    normalized = torch.empty(selected_update.shape, dtype=torch.float32, device=device)
    squared_norms = torch.empty((batch, 2), dtype=torch.float32, device=device)
    u = selected_update.reshape(batch, k, cols)
    if u.stride(-1) != 1:
        u = u.contiguous()
    idx = indices.reshape(batch * k).contiguous() if k > 0 else indices
    lib = nat.load()
    ws = _workspace(lib.gns_dion3_normalize_workspace_size(batch, max(k, 1)), device)
    with torch.cuda.device(device):
        rc = lib.gns_dion3_normalize_rows(
            nat.dtype_code(u.dtype), batch, rows, cols, k, u.data_ptr() if k > 0 else None, u.stride(0), u.stride(1),
            variance.data_ptr(), idx.data_ptr() if k > 0 else None, float(beta_two), float(epsilon),
            normalized.data_ptr() if normalized.numel() else None, squared_norms.data_ptr(), ws.data_ptr(),
            ws.numel(), nat.stream_handle(device),
        )
    nat.check(rc, "gns_dion3_normalize_rows")
    return normalized, squared_norms


def dion3_apply_rows(
    parameter: Tensor,
    normalized_update: Tensor,
    indices: Tensor,
    squared_norms: Tensor,
    learning_rate: float,
    weight_decay: float,
    adjusted_learning_rate: float,
    epsilon: float,
) -> None:
    """The update half of dion3_normalize_apply (reference kernels/dion3_cuda.cu:402-470): decays the
    parameter and adds the norm-preserving rescaled ``normalized_update`` to the selected rows."""
    device = _require_cuda(parameter, normalized_update, indices, squared_norms)
    if not parameter.is_contiguous():
        raise ValueError("parameter must be C contiguous")
    if normalized_update.dtype != torch.float32:
        raise ValueError("normalized_update must be float32")
    if indices.dtype != torch.long:
        raise ValueError("indices must be int64")
    if squared_norms.dtype != torch.float32:
        raise ValueError("squared_norms must be float32")
    rows, cols = parameter.shape[-2], parameter.shape[-1]
    batch = _leading(parameter)
    k = normalized_update.shape[-2]
    if normalized_update.numel() != batch * k * cols:
        raise ValueError("parameter and normalized_update batch dimensions must match")
    if indices.numel() != batch * k:
        raise ValueError("indices and normalized_update shapes must match")
    if squared_norms.numel() != batch * 2:
        raise ValueError("squared_norms must contain two values per batch")
    if k == 0 and parameter.numel() != 0:
        raise ValueError("an empty selected update requires an empty parameter shard")
    n = normalized_update.contiguous()
    idx = indices.reshape(batch * k).contiguous() if k > 0 else indices
    sq = squared_norms.contiguous()
    lib = nat.load()
    with torch.cuda.device(device):
        rc = lib.gns_dion3_apply_rows(
            nat.dtype_code(parameter.dtype), batch, rows, cols, k, parameter.data_ptr(),
            n.data_ptr() if n.numel() else None, idx.data_ptr() if k > 0 else None, sq.data_ptr(),
            float(learning_rate), float(weight_decay), float(adjusted_learning_rate), float(epsilon),
            nat.stream_handle(device),
        )
    nat.check(rc, "gns_dion3_apply_rows")


# ------------------------------------------------------------ AdamW / Lion
def _group_check(tensors_by_role: Sequence[Sequence[Tensor]]) -> torch.device:
    first = tensors_by_role[0]
    for role in tensors_by_role:
        if len(role) != len(first):
            raise ValueError("tensor lists must have equal lengths")
        for t, ref in zip(role, first, strict=True):
            if t.numel() != ref.numel():
                raise ValueError("tensor sizes differ within one parameter")
            if not t.is_contiguous():
                raise ValueError("tensors must be contiguous")
        if len({t.dtype for t in role}) > 1:
            raise TypeError("tensors of one role must share a dtype")
    return _require_cuda(*[t for role in tensors_by_role for t in role])


def adamw_step(
    parameters: Sequence[Tensor],
    gradients: Sequence[Tensor],
    exp_avgs: Sequence[Tensor],
    exp_avg_sqs: Sequence[Tensor],
    lr_over_bias_correction1: Sequence[float],
    inverse_sqrt_bias_correction2: Sequence[float],
    beta1: float,
    beta2: float,
    epsilon: float,
    decay: float | None,
) -> None:
    """One multi-tensor AdamW step over a group (muon.py:516-553), in place."""
    if not parameters:
        return
    device = _group_check([parameters, gradients, exp_avgs, exp_avg_sqs])
    count = len(parameters)
    numel = (ctypes.c_int64 * count)(*[t.numel() for t in parameters])
    lr_bc1 = (ctypes.c_float * count)(*[float(v) for v in lr_over_bias_correction1])
    inv_bc2 = (ctypes.c_float * count)(*[float(v) for v in inverse_sqrt_bias_correction2])
    lib = nat.load()
    with torch.cuda.device(device):
        rc = lib.gns_adamw_step(
            count, _ptr_array(parameters), _ptr_array(gradients), _ptr_array(exp_avgs), _ptr_array(exp_avg_sqs),
            numel, nat.dtype_code(parameters[0].dtype), nat.dtype_code(gradients[0].dtype),
            nat.dtype_code(exp_avgs[0].dtype), lr_bc1, inv_bc2, float(beta1), float(beta2), float(1 - beta1),
            float(1 - beta2), float(epsilon),
            float(decay) if decay is not None else 1.0, 1 if decay is not None else 0, nat.stream_handle(device),
        )
    nat.check(rc, "gns_adamw_step")


def lion_step(
    parameters: Sequence[Tensor],
    gradients: Sequence[Tensor],
    buffers: Sequence[Tensor],
    learning_rate: float,
    beta1: float,
    beta2: float,
    decay: float | None,
) -> None:
    """One multi-tensor Lion step over a group (muon.py:555-583), in place."""
    if not parameters:
        return
    device = _group_check([parameters, gradients, buffers])
    count = len(parameters)
    numel = (ctypes.c_int64 * count)(*[t.numel() for t in parameters])
    lib = nat.load()
    with torch.cuda.device(device):
        rc = lib.gns_lion_step(
            count, _ptr_array(parameters), _ptr_array(gradients), _ptr_array(buffers), numel,
            nat.dtype_code(parameters[0].dtype), nat.dtype_code(gradients[0].dtype), nat.dtype_code(buffers[0].dtype),
            float(learning_rate), float(beta1), float(beta2), float(1 - beta1), float(1 - beta2),
            float(decay) if decay is not None else 1.0,
            1 if decay is not None else 0, nat.stream_handle(device),
        )
    nat.check(rc, "gns_lion_step")


# ------------------------------------------------- AdamW states in 8 or 32 bits
STATE_ROUNDINGS = ("nearest", "unbiased")  # of the 8-bit states
STATE_BLOCK = 256  # consecutive elements of a tensor that share a scale of the 8-bit states


def _pointers(tensors: Sequence[Tensor]) -> ctypes.Array:
    """``_ptr_array`` of many tensors, at a quarter of its cost for each."""
    places = array.array("Q", map(Tensor.data_ptr, tensors))
    return (ctypes.c_void_p * len(places)).from_buffer(places)


def moment_in_8_bits(moment: Tensor, second: bool) -> tuple[Tensor, Tensor]:
    """A moment as ``AdamWStates`` holds it in 8 bits: e4m3 values of its shape and one fp32 scale
    for each ``STATE_BLOCK`` elements. ``second``: values above zero stay above it."""
    flat = moment.detach().reshape(-1).float()
    blocks = torch.nn.functional.pad(flat, (0, -flat.numel() % STATE_BLOCK)).view(-1, STATE_BLOCK)
    top = blocks.abs().amax(1) if blocks.numel() else blocks.new_zeros(0)
    codes = blocks * torch.where(top > 1e-30, 448.0 / top, 0.0)[:, None]
    if second:
        codes = torch.where(blocks > 0, codes.clamp_min(2.0**-9), codes)
    held = codes.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).reshape(-1)[:flat.numel()]
    return held.clone().view(moment.shape), top * (1 / 448)


def moment_from_8_bits(codes: Tensor, scales: Tensor) -> Tensor:
    """The fp32 values of a moment that ``AdamWStates`` holds in 8 bits."""
    each = scales.repeat_interleave(STATE_BLOCK)[:codes.numel()]
    return (codes.reshape(-1).float() * each).view(codes.shape)


class AdamWStates:
    """The AdamW moments of a list of parameters, in 32 bits or in 8, and the step over them.

    With ``bits=8`` the moments are ``float8_e4m3fn`` tensors of the parameters' shapes
    with one fp32 scale for each 256 consecutive elements (``exp_avg_scales``,
    ``exp_avg_sq_scales``: 1-D, ``ceil(numel / 256)`` entries): an element's value is its
    e4m3 value times its block's scale. With ``bits=32`` they are fp32 tensors. Moments
    that are not given start at zero. Parameters are contiguous CUDA tensors of one
    16- or 32-bit floating type; they and the moments are updated in place.

    Unlike ``adamw_step``, which rounds after every operation as the torch sequence it
    replaces does, the arithmetic is fp32 throughout with one rounding at the end.

    ``rounding`` says how 8-bit moments round. ``"nearest"``: each step's values are as near
    as they can be, but a value that decays by less than half a code a step stays where it
    is. With a ``beta2`` of 0.95 that is 1.125 or 1.25 times a power of two, with 0.999 every
    code, so an element's second moment may stay above its exact value (and its steps too
    small) until its block's scale comes down: over 3000 steps at 0.95 the root of the second
    moment grew to 1.45 times the exact one where elements were a tenth of their block's
    largest (1.41 at 0.99, 1.19 at 0.999), and an element whose gradient stopped kept
    it. ``"unbiased"`` rounds up or down with the probabilities that make the mean right
    (0.994 to 0.998 of the exact root in all of these), for any ``beta2`` and long runs;
    single values are then up to a whole code off. The random bits follow from the step
    number, the tensor's place in the call and the element's place in the tensor, so equal
    runs give equal bits. Unbiased second moments still never round to zero.
    """

    def __init__(
        self,
        parameters: Sequence[Tensor],
        bits: int = 8,
        exp_avgs: Sequence[Tensor] | None = None,
        exp_avg_sqs: Sequence[Tensor] | None = None,
        exp_avg_scales: Sequence[Tensor] | None = None,
        exp_avg_sq_scales: Sequence[Tensor] | None = None,
        rounding: str = "nearest",
    ) -> None:
        if bits not in (8, 32):
            raise ValueError(f"bits must be 8 or 32, got {bits}")
        if rounding not in STATE_ROUNDINGS:
            raise ValueError(f"rounding must be one of {STATE_ROUNDINGS}, got {rounding!r}")
        if rounding != "nearest" and bits != 8:
            raise ValueError("rounding is a setting of 8-bit moments")
        self.bits = bits
        self.rounding = rounding
        self.parameters = list(parameters)
        if (exp_avgs is None) != (exp_avg_sqs is None):
            raise ValueError("give both moments or neither")
        if bits == 8 and exp_avgs is not None and (exp_avg_scales is None or exp_avg_sq_scales is None):
            raise ValueError("8-bit moments need their scales")
        if exp_avg_scales is not None and exp_avgs is None:
            raise ValueError("scales without moments")
        if bits == 32 and (exp_avg_scales is not None or exp_avg_sq_scales is not None):
            raise ValueError("32-bit moments have no scales")
        dtype = torch.float8_e4m3fn if bits == 8 else torch.float32
        for p in self.parameters:
            if not p.is_contiguous():
                raise ValueError("parameters must be contiguous")
            if p.dtype != self.parameters[0].dtype:
                raise TypeError("all parameters of one call must share a dtype")
        self.device = _require_cuda(*self.parameters) if self.parameters else None
        if self.parameters:
            nat.dtype_code(self.parameters[0].dtype)

        def moments(given: Sequence[Tensor] | None) -> list[Tensor]:
            if given is None:
                return [torch.zeros(p.shape, dtype=dtype, device=p.device) for p in self.parameters]
            return self._checked(given, dtype, [p.numel() for p in self.parameters], "moments")

        def scales(given: Sequence[Tensor] | None) -> list[Tensor]:
            counts = [(p.numel() + STATE_BLOCK - 1) // STATE_BLOCK for p in self.parameters]
            if given is None:
                return [torch.zeros(n, dtype=torch.float32, device=p.device) for n, p in zip(counts, self.parameters)]
            return self._checked(given, torch.float32, counts, "scales")

        self.exp_avgs = moments(exp_avgs)
        self.exp_avg_sqs = moments(exp_avg_sqs)
        self.exp_avg_scales = scales(exp_avg_scales) if bits == 8 else []
        self.exp_avg_sq_scales = scales(exp_avg_sq_scales) if bits == 8 else []
        self._numel = [p.numel() for p in self.parameters]
        self._sizes = (ctypes.c_int64 * max(len(self._numel), 1))(*self._numel)
        self._note(*self._tensors_now())

    def _checked(self, given: Sequence[Tensor], dtype: torch.dtype, counts: list[int], what: str) -> list[Tensor]:
        if len(given) != len(counts):
            raise ValueError("tensor lists must have equal lengths")
        if self.device is not None and (
            list(map(Tensor.numel, given)) == counts and all(map(Tensor.is_contiguous, given))
            and {t.dtype for t in given} == {dtype} and set(map(Tensor.get_device, given)) == {self.device.index}
        ):
            return list(given)
        for t, n in zip(given, counts, strict=True):  # which of them it is
            if t.dtype != dtype:
                raise TypeError(f"{self.bits}-bit AdamW {what} must be {dtype}, got {t.dtype}")
            if t.numel() != n:
                raise ValueError("tensor sizes differ within one parameter")
            if not t.is_contiguous():
                raise ValueError("tensors must be contiguous")
            if t.device != self.device:
                raise ValueError("all tensors must be on the same CUDA device")
        return list(given)

    def _tensors_now(self) -> tuple[array.array, list[int]]:
        """Addresses and bytes of the parameters, moments and scales."""
        held = [*self.parameters, *self.exp_avgs, *self.exp_avg_sqs, *self.exp_avg_scales, *self.exp_avg_sq_scales]
        return array.array("Q", map(Tensor.data_ptr, held)), [t.nbytes for t in held]

    def _note(self, places: array.array, extents: list[int]) -> None:
        """Keeps what was checked, and each list's addresses as the native call takes them."""
        self._places, self._bytes = places, extents
        row = ctypes.c_void_p * len(self._numel)
        self._rows = tuple(
            row.from_buffer(places, i * ctypes.sizeof(row)) if row._length_ and (i < 3 or self.bits == 8) else None
            for i in range(5)
        )

    def _look_at_tensors(self) -> None:
        """Brings ``_rows`` up to date with the tensors in the lists. Between two steps any of
        them may be replaced, or moved by an assignment to its ``.data``, so their addresses are
        read on every step. All else is checked again only where an address or the bytes behind
        it are new (checked on every step it would cost twice the rest of a small step)."""
        places, extents = self._tensors_now()
        if places == self._places and extents == self._bytes:
            return
        for p, n in zip(self.parameters, self._numel, strict=True):
            if p.numel() != n:
                raise ValueError("a parameter's size is not that of its moments")
            if p.dtype != self.parameters[0].dtype:
                raise TypeError("all parameters of one call must share a dtype")
            if p.device != self.device:
                raise ValueError("parameters must stay on the device of their moments")
        dtype = torch.float8_e4m3fn if self.bits == 8 else torch.float32
        self._checked(self.exp_avgs, dtype, self._numel, "moments")
        self._checked(self.exp_avg_sqs, dtype, self._numel, "moments")
        if self.bits == 8:
            counts = [(n + STATE_BLOCK - 1) // STATE_BLOCK for n in self._numel]
            self._checked(self.exp_avg_scales, torch.float32, counts, "scales")
            self._checked(self.exp_avg_sq_scales, torch.float32, counts, "scales")
        self._note(places, extents)

    def step(
        self,
        gradients: Sequence[Tensor | None],
        learning_rate: float,
        beta1: float,
        beta2: float,
        epsilon: float,
        weight_decay: float,
        step: int | Sequence[float],
        gradient_scale: Tensor | None = None,
    ) -> None:
        """One AdamW step in place. ``step`` is the number of this step, from 1 on (one value,
        or one for each parameter); a gradient of None leaves its parameter and moments as
        they are; ``gradient_scale`` is one fp32 value on the device that every gradient is
        multiplied by (a clipping factor, or the inverse of a loss scale)."""
        count = len(self.parameters)
        if len(gradients) != count:
            raise ValueError("gradients and parameters must have equal lengths")
        if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
            raise ValueError(f"betas must be in [0, 1), got {(beta1, beta2)}")
        if not epsilon > 0.0:
            raise ValueError(f"epsilon must be positive, got {epsilon}")
        try:
            dtypes = {g.dtype for g in gradients}  # type: ignore[union-attr]
            whole = True
        except AttributeError:  # None among them
            whole = False
            dtypes = {g.dtype for g in gradients if g is not None}
        present = range(count) if whole else [i for i, g in enumerate(gradients) if g is not None]
        if not present:
            return
        given = cast(Sequence[Tensor], gradients) if whole else [cast(Tensor, gradients[i]) for i in present]
        places = self.parameters if whole else [self.parameters[i] for i in present]
        g_dtype = given[0].dtype
        if len(dtypes) > 1:
            raise TypeError("all gradients of one call must share a dtype")
        numel = list(map(Tensor.numel, given))
        if numel != (self._numel if whole else [self._numel[i] for i in present]):
            raise ValueError("gradient and parameter sizes differ")
        if not (all(map(Tensor.is_contiguous, given)) and all(map(Tensor.is_contiguous, places))):
            raise ValueError("gradients and parameters must be contiguous")
        index = cast(torch.device, self.device).index
        if set(map(Tensor.get_device, given)) != {index}:
            raise ValueError("gradients must be on the parameters' device")
        self._look_at_tensors()
        if gradient_scale is not None:
            if gradient_scale.dtype != torch.float32 or gradient_scale.numel() != 1:
                raise ValueError("gradient_scale must be one float32 value")
            if gradient_scale.get_device() != index:
                raise ValueError("gradient_scale must be on the parameters' device")
        floats = ctypes.c_float * len(given)
        if isinstance(step, (int, float)):
            lr_bc1, inv_bc2 = self._bias_corrections(step, learning_rate, beta1, beta2)
            corrections = tuple(
                floats.from_buffer(array.array("f", [value]) * len(given)) for value in (lr_bc1, inv_bc2)
            )
        else:
            if len(step) != count:
                raise ValueError("step must be one value or one for each parameter")
            pairs = [self._bias_corrections(step[i], learning_rate, beta1, beta2) for i in present]
            corrections = tuple(floats.from_buffer(array.array("f", values)) for values in zip(*pairs))
        rows, sizes = self._rows, self._sizes
        if not whole:
            sizes = (ctypes.c_int64 * len(given))(*numel)
            roles = (self.parameters, self.exp_avgs, self.exp_avg_sqs, self.exp_avg_scales, self.exp_avg_sq_scales)
            rows = tuple(_ptr_array([role[i] for i in present]) if role else None for role in roles)
        call, form = nat.load().gns_adamw_states_step, (self.bits,)
        if self.rounding == "unbiased":
            numbers = [step] * len(given) if isinstance(step, (int, float)) else [step[i] for i in present]
            seeds = array.array("I", [int(number) & 0xFFFFFFFF for number in numbers])
            call, form = nat.load().gns_adamw_states_step_unbiased, ((ctypes.c_uint32 * len(seeds)).from_buffer(seeds),)
        with nat.on_device(index) as stream:
            rc = call(
                len(given), rows[0], _pointers(given), *rows[1:], sizes,
                nat.dtype_code(places[0].dtype), nat.dtype_code(g_dtype), *form, *corrections,
                beta1, 1 - beta1, beta2, 1 - beta2, epsilon, 1 - learning_rate * weight_decay,
                nat.ptr(gradient_scale), stream,
            )
        nat.check(rc, "gns_adamw_states_step")

    @staticmethod
    def _bias_corrections(step: float, learning_rate: float, beta1: float, beta2: float) -> tuple[float, float]:
        if step < 1:
            raise ValueError(f"steps count from 1, got {step}")
        return learning_rate / (1 - beta1**step), (1 - beta2**step) ** -0.5


# ------------------------------------------------- products grouped by expert
def _aligned_copy(
    t: Tensor, batch: int, rows: int, cols: int, batch_stride: int, row_stride: int, ends: Tensor | None = None
) -> tuple[Tensor, int]:
    """A buffer with a copy of the rows [batch, rows, cols] that start at `t`'s first element, with
    unit column stride, and its row pitch, a multiple of 8 elements. With ``ends``, without
    the matrices of groups that have no rows."""
    pitch = (cols + 7) // 8 * 8
    buffer = torch.empty(batch * rows * pitch, dtype=t.dtype, device=t.device)
    lib = nat.load()
    with nat.on_device(t.get_device()) as stream:
        rc = lib.gns_align_rows(batch, rows, cols, t.data_ptr(), batch_stride, row_stride, nat.ptr(ends),
                                0 if ends is None else 8 * ends.element_size(), buffer.data_ptr(), rows * pitch,
                                pitch, stream)
    nat.check(rc, "gns_align_rows")
    return buffer, pitch


def row_operand(t: Tensor) -> Tensor:
    """Returns the matrix `t` if a TMA tile load can read its rows (unit column stride,
    16-byte aligned base and row stride), else a copy whose row pitch is padded to a
    multiple of 8 elements. The grouped products make such a copy themselves; a caller
    that passes a matrix to several of them saves the others with this."""
    rows, cols = t.shape
    held, _, pitch = _row_layout(t)
    return t if held is t else held.as_strided((rows, cols), (pitch, 1))


def _row_layout(t: Tensor) -> tuple[Tensor, int, int]:
    """(owner, address, row stride) of the matrix `t` or of a copy of it that TMA can read."""
    rows, cols = t.shape
    sr, sc = t.stride()
    place = t.data_ptr()
    if place % 16 == 0 and (sc == 1 or cols == 1) and ((sr % 8 == 0 and sr >= cols) or rows == 1):
        return t, place, sr
    if sc != 1 and cols > 1:
        t, sr = t.contiguous(), cols
    copy, pitch = _aligned_copy(t, 1, rows, cols, 0, sr)
    return copy, copy.data_ptr(), pitch


def _group_layout(t: Tensor, ends: Tensor | None = None) -> tuple[Tensor, int, int, int, int]:
    """(owner, address, strides) of one matrix per group [groups, k, n], stored by rows or by
    columns, or of a copy of it, in the same order, that TMA can read."""
    groups, k, n = t.shape
    sg, sk, sn = t.stride()
    place = t.data_ptr()
    sound = place % 16 == 0 and ((sg % 8 == 0 and sg != 0) or groups == 1)
    by_rows, by_columns = sn == 1 or n == 1, sk == 1 or k == 1
    if sound and by_rows and ((sk % 8 == 0 and sk >= n) or k == 1):
        return t, place, sg, sk, 1
    if sound and by_columns and ((sn % 8 == 0 and sn >= k) or n == 1):
        return t, place, sg, 1, sn
    if not (by_rows or by_columns):
        t = t.contiguous()
        sg, sk, sn, by_rows = k * n, n, 1, True
    if by_rows:
        copy, pitch = _aligned_copy(t, groups, k, n, sg, sk, ends)
        return copy, copy.data_ptr(), k * pitch, pitch, 1
    copy, pitch = _aligned_copy(t, groups, n, k, sg, sn, ends)
    return copy, copy.data_ptr(), n * pitch, 1, pitch


def _group_ends(ends: Tensor, groups: int | None = None) -> Tensor:
    if ends.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ends must be int32 or int64, got {ends.dtype}")
    if ends.ndim != 1 or (groups is not None and ends.numel() != groups):
        raise ValueError("ends must hold one row number for each group")
    return ends.contiguous()


def grouped_gemm(left: Tensor, right: Tensor, ends: Tensor, out_dtype: torch.dtype | None = None) -> Tensor:
    """``out[r] = left[r] @ right[e]`` for the rows r of each group e, on tcgen05 tensor cores.

    left [T, k] holds rows sorted by group, right [E, k, n] one matrix for each group (either
    may have its last two dimensions transposed in memory), both float16 or both bfloat16.
    ``ends`` [E] (int32 or int64, on the device) are the row numbers where the groups end:
    group e owns the rows ``ends[e - 1] <= r < ends[e]``. They are read on the device, without
    a synchronisation, and are clamped to [0, T] and to ascending order. Rows that no group
    owns (from ``ends[-1]`` on) come out zero. Sums are fp32, rounded once to ``out_dtype``
    (default: the inputs' type); their order depends on the sizes of the call (few rows with
    a long k are summed in parts), never on the run.

    With an expert layer's weights W [E, n, k], the layer is
    ``grouped_gemm(x, W.transpose(1, 2), ends)``, its gradient for the rows
    ``grouped_gemm(dy, W, ends)`` and for the weights ``grouped_gemm_reduce(dy, x, ends)``.
    """
    index = _device_index(left, right, ends)
    if left.ndim != 2 or right.ndim != 3:
        raise ValueError("expected left [rows, k] and right [groups, k, n]")
    if left.dtype != right.dtype or left.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("left and right must share dtype float16 or bfloat16")
    if left.shape[1] != right.shape[1]:
        raise ValueError(f"incompatible shapes {tuple(left.shape)} @ {tuple(right.shape)}")
    groups, k, n = right.shape
    rows = left.shape[0]
    ends = _group_ends(ends, groups)
    dtype = out_dtype or left.dtype
    code = nat.dtype_code(dtype)
    if rows == 0 or n == 0 or k == 0 or groups == 0:
        return torch.zeros((rows, n), dtype=dtype, device=left.device)
    out = left.new_empty((rows, n), dtype=dtype)
    left_held, left_at, left_pitch = _row_layout(left)
    right_held, *right_layout = _group_layout(right, ends)
    lib = nat.load()
    with nat.on_device(index) as stream:
        rc = lib.gns_grouped_gemm(
            nat.dtype_code(left.dtype), rows, n, k, groups, left_at, left_pitch, *right_layout,
            ends.data_ptr(), 8 * ends.element_size(), out.data_ptr(), code, n, stream,
        )
    nat.check(rc, "gns_grouped_gemm")
    return out


def grouped_gemm_plan(rows: int, n: int, k: int, groups: int) -> tuple[int, int]:
    """How ``grouped_gemm`` runs [rows, k] by [groups, k, n] on the current device: the rows of a
    tile, and the CTAs that share a tile's contraction."""
    tile, split = ctypes.c_int(), ctypes.c_int()
    rc = nat.load().gns_grouped_gemm_plan(rows, n, k, groups, ctypes.byref(tile), ctypes.byref(split))
    nat.check(rc, "gns_grouped_gemm_plan")
    return tile.value, split.value


def grouped_gemm_reduce(left: Tensor, right: Tensor, ends: Tensor, out_dtype: torch.dtype | None = None) -> Tensor:
    """``out[e] = left[rows of e].T @ right[rows of e]`` for each group of rows, on tcgen05
    tensor cores: [E, m, n] from left [T, m] and right [T, n], zero for a group without rows.
    ``ends`` as for ``grouped_gemm``; rows that no group owns have no part in any sum."""
    index = _device_index(left, right, ends)
    if left.ndim != 2 or right.ndim != 2:
        raise ValueError("expected left [rows, m] and right [rows, n]")
    if left.dtype != right.dtype or left.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("left and right must share dtype float16 or bfloat16")
    if left.shape[0] != right.shape[0]:
        raise ValueError(f"left and right have {left.shape[0]} and {right.shape[0]} rows")
    ends = _group_ends(ends)
    rows, m = left.shape
    n = right.shape[1]
    groups = ends.numel()
    dtype = out_dtype or left.dtype
    code = nat.dtype_code(dtype)
    if rows == 0 or m == 0 or n == 0 or groups == 0:
        return torch.zeros((groups, m, n), dtype=dtype, device=left.device)
    out = left.new_empty((groups, m, n), dtype=dtype)
    left_held, left_at, left_pitch = _row_layout(left)
    right_held, right_at, right_pitch = _row_layout(right)
    lib = nat.load()
    with nat.on_device(index) as stream:
        rc = lib.gns_grouped_gemm_reduce(
            nat.dtype_code(left.dtype), rows, m, n, groups, left_at, left_pitch, right_at, right_pitch,
            ends.data_ptr(), 8 * ends.element_size(), out.data_ptr(), code, m * n, n, stream,
        )
    nat.check(rc, "gns_grouped_gemm_reduce")
    return out


# ------------------------------------------------------------------ layer norm
def _norm_rows(t: Tensor, columns: int) -> Tensor:
    """[rows, columns] view of `t` with unit column stride and rows that do not overlap."""
    flat = t if t.ndim == 2 else t.reshape(-1, columns)
    if columns > 1 and flat.stride(1) != 1 or flat.shape[0] > 1 and flat.stride(0) < columns:
        flat = flat.contiguous()
    return flat


def _norm_check(x: Tensor, weight: Tensor, bias: Tensor | None) -> int:
    if x.ndim < 1 or weight.ndim != 1 or x.shape[-1] != weight.numel() or weight.numel() == 0:
        raise ValueError("weight must have one entry for each element of x's last dimension")
    nat.dtype_code(x.dtype)
    nat.dtype_code(weight.dtype)
    if bias is not None:
        if bias.shape != weight.shape:
            raise ValueError("weight and bias shapes differ")
        if bias.dtype != weight.dtype:
            raise TypeError("weight and bias must share a dtype")
    return weight.numel()


def layer_norm(x: Tensor, weight: Tensor, bias: Tensor | None, epsilon: float) -> tuple[Tensor, Tensor, Tensor]:
    """Layer norm over the last dimension: ``y = (x - mean) * rstd * weight + bias``.

    Returns y (x's type, contiguous) and the fp32 mean and rstd of each row (x's shape
    without the last dimension), which ``layer_norm_backward`` takes. The variance is the
    biased one; all arithmetic is fp32. weight and bias share a floating type of their own;
    bias may be None."""
    index = _device_index(x, weight, bias)
    columns = _norm_check(x, weight, bias)
    flat = _norm_rows(x, columns)
    rows = flat.shape[0]
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    w = weight.contiguous()
    b = bias.contiguous() if bias is not None else None
    lib = nat.load()
    with nat.on_device(index) as stream:
        rc = lib.gns_layer_norm_forward(
            nat.dtype_code(x.dtype), nat.dtype_code(w.dtype), rows, columns, flat.data_ptr(), flat.stride(0),
            w.data_ptr(), nat.ptr(b), float(epsilon), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
            stream,
        )
    nat.check(rc, "gns_layer_norm_forward")
    return y, mean, rstd


def layer_norm_backward(
    grad: Tensor, x: Tensor, weight: Tensor, mean: Tensor, rstd: Tensor
) -> tuple[Tensor, Tensor, Tensor]:
    """Gradients (dx, dweight, dbias) of ``layer_norm`` from the gradient of y and the mean and
    rstd that the forward pass returned. dx has x's type, dweight and dbias the weight's;
    their sums over the rows are fp32, in a fixed order."""
    index = _device_index(grad, x, weight, mean, rstd)
    columns = _norm_check(x, weight, None)
    if grad.shape != x.shape:
        raise ValueError("grad and x shapes differ")
    if grad.dtype != x.dtype:
        raise TypeError("grad and x must share a dtype")
    rows = x.numel() // columns
    for t in (mean, rstd):
        if t.dtype != torch.float32 or t.numel() != rows or not t.is_contiguous():
            raise ValueError("mean and rstd must be contiguous float32 with one entry per row")
    flat, g = _norm_rows(x, columns), _norm_rows(grad, columns)
    w = weight.contiguous()
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dweight, dbias = torch.empty_like(w), torch.empty_like(w)
    lib = nat.load()
    nbytes = lib.gns_layer_norm_backward_workspace_size(rows, columns)
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    with nat.on_device(index) as stream:
        rc = lib.gns_layer_norm_backward(
            nat.dtype_code(x.dtype), nat.dtype_code(w.dtype), rows, columns, g.data_ptr(), g.stride(0),
            flat.data_ptr(), flat.stride(0), w.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(),
            dweight.data_ptr(), dbias.data_ptr(), nat.ptr(ws), nbytes, stream,
        )
    nat.check(rc, "gns_layer_norm_backward")
    return dx, dweight, dbias


# ------------------------------------------------------ 8 bits, blocks of 128
_BLOCK = 128


def _code_buffers(like: Tensor, rows: int, columns: int, block_rows: int = 1) -> tuple[Tensor, Tensor]:
    """Buffers for the codes [rows, columns] and scales of a matrix: rows of codes start on 16
    bytes, the scales of one block column follow one another."""
    pitch = (columns + 15) // 16 * 16
    codes = like.new_empty((rows, pitch), dtype=torch.float8_e4m3fn)
    scales = like.new_empty(((columns + _BLOCK - 1) // _BLOCK, (rows + block_rows - 1) // block_rows), dtype=torch.float32)
    return codes if pitch == columns else codes[:, :columns], scales.t()


def quantize_8bit(x: Tensor, block_rows: int = 1) -> tuple[Tensor, Tensor]:
    """A matrix [rows, columns] as e4m3 codes with an fp32 scale for each block of ``block_rows``
    (1 or 128) rows and 128 columns: ``scale = top / 448`` and ``code = e4m3(x * (448 / top))``,
    rounded to nearest even, with top the block's largest magnitude (at least 448 * 2^-126).

    Returns the codes (``float8_e4m3fn``, x's shape, rows starting on multiples of 16 bytes) and
    the scales [ceil(rows / block_rows), ceil(columns / 128)]. ``gemm_8bit`` takes activations
    and gradients in blocks of 1 x 128, weights in blocks of 128 x 128. x is float16, bfloat16 or
    float32. A NaN keeps a code of NaN; an infinity makes its block's scale infinite and the
    block's products NaN."""
    index = _device_index(x)
    if x.ndim != 2:
        raise ValueError("expected a matrix")
    if block_rows not in (1, _BLOCK):
        raise ValueError(f"a block has 1 or 128 rows, got {block_rows}")
    code = nat.dtype_code(x.dtype)
    rows, columns = x.shape
    codes, scales = _code_buffers(x, rows, columns, block_rows)
    if rows == 0 or columns == 0:
        return codes, scales
    held = _norm_rows(x, columns)
    with nat.on_device(index) as stream:
        rc = nat.load().gns_quantize_8bit(
            code, block_rows, rows, columns, held.data_ptr(), held.stride(0), codes.data_ptr(), codes.stride(0),
            scales.data_ptr(), *scales.stride(), stream,
        )
    nat.check(rc, "gns_quantize_8bit")
    return codes, scales


def _byte_rows(t: Tensor) -> Tensor:
    """A copy of the 8-bit matrix `t` whose rows start on multiples of 16 bytes."""
    rows, columns = t.shape
    copy = t.new_empty((rows, (columns + 15) // 16 * 16))
    copy.view(torch.uint8)[:, :columns].copy_(t.view(torch.uint8))
    return copy


def _byte_layout(t: Tensor) -> tuple[Tensor, int, int]:
    """(owner, row stride, column stride) of the 8-bit matrix `t` or of a copy of it, in the same
    order, that TMA can read: a unit stride, the other one a multiple of 16 bytes."""
    rows, columns = t.shape
    sr, sc = t.stride()
    sound = t.data_ptr() % 16 == 0
    if sound and (sc == 1 or columns == 1) and ((sr % 16 == 0 and sr >= columns) or rows == 1):
        return t, sr if rows > 1 else 0, 1
    if sound and (sr == 1 or rows == 1) and ((sc % 16 == 0 and sc >= rows) or columns == 1):
        return t, 1, sc if columns > 1 else 0
    if sr == 1 and sc != 1:
        held, stride, _ = _byte_layout(t.t())
        return held, 1, stride
    copy = _byte_rows(t)
    return copy, copy.stride(0), 1


def gemm_8bit(
    left: Tensor, left_scales: Tensor, right: Tensor, right_scales: Tensor, out_dtype: torch.dtype = torch.bfloat16
) -> Tensor:
    """``left @ right`` of e4m3 matrices with fp32 scales, on tcgen05 tensor cores.

    left [m, k] has a scale for each row and each 128 of k: left_scales [m, ceil(k / 128)].
    right [k, n] has one for each 128 x 128 block: right_scales [ceil(k / 128), ceil(n / 128)];
    it may be stored by rows or by columns. Both come from ``quantize_8bit`` (left also from
    ``rms_norm_8bit``). With a layer's weights W [n, k] in blocks of 128 x 128, codes w and
    scales s, the layer is ``gemm_8bit(x, xs, w.T, s.T)`` and the gradient of its input
    ``gemm_8bit(dy, dys, w, s)``.

    The sum over a block of 128 is the tensor cores' with fp32 accumulators; it is scaled by the
    fp32 product of its two scales and added up in fp32, and rounded once to ``out_dtype``
    (float16, bfloat16 or float32). The order of the sums depends on the sizes of the call (few
    rows with a long k are summed in parts), never on the run. Operands that TMA cannot read (rows
    that do not start on 16 bytes) are copied first."""
    index = _device_index(left, left_scales, right, right_scales)
    if left.ndim != 2 or right.ndim != 2 or left.shape[1] != right.shape[0]:
        raise ValueError(f"incompatible shapes {tuple(left.shape)} @ {tuple(right.shape)}")
    if left.dtype != torch.float8_e4m3fn or right.dtype != torch.float8_e4m3fn:
        raise TypeError("left and right must be float8_e4m3fn")
    if left_scales.dtype != torch.float32 or right_scales.dtype != torch.float32:
        raise TypeError("scales must be float32")
    m, k = left.shape
    n = right.shape[1]
    blocks = (k + _BLOCK - 1) // _BLOCK
    if tuple(left_scales.shape) != (m, blocks):
        raise ValueError(f"left_scales must be {(m, blocks)}, got {tuple(left_scales.shape)}")
    if tuple(right_scales.shape) != (blocks, (n + _BLOCK - 1) // _BLOCK):
        raise ValueError(f"right_scales must be {(blocks, (n + _BLOCK - 1) // _BLOCK)}, got {tuple(right_scales.shape)}")
    code = nat.dtype_code(out_dtype)
    if m == 0 or n == 0 or k == 0:
        return torch.zeros((m, n), dtype=out_dtype, device=left.device)
    left_held, left_pitch, unit = _byte_layout(left)
    if unit != 1:  # held by columns
        left_held = _byte_rows(left)
        left_pitch = left_held.stride(0)
    right_held, *right_strides = _byte_layout(right)
    out = left.new_empty((m, n), dtype=out_dtype)
    with nat.on_device(index) as stream:
        rc = nat.load().gns_gemm_8bit(
            m, n, k, left_held.data_ptr(), left_pitch, left_scales.data_ptr(), *left_scales.stride(),
            right_held.data_ptr(), *right_strides, right_scales.data_ptr(), *right_scales.stride(),
            out.data_ptr(), code, n, stream,
        )
    nat.check(rc, "gns_gemm_8bit")
    return out


def gemm_8bit_plan(m: int, n: int, k: int) -> tuple[int, int]:
    """How ``gemm_8bit`` runs [m, k] by [k, n] on the current device: the rows of a tile, and the
    CTAs that share a tile's contraction."""
    tile, parts = ctypes.c_int(), ctypes.c_int()
    rc = nat.load().gns_gemm_8bit_plan(m, n, k, ctypes.byref(tile), ctypes.byref(parts))
    nat.check(rc, "gns_gemm_8bit_plan")
    return tile.value, parts.value


def _quantized(lib, x: Tensor, block_rows: int, stream: int) -> tuple[Tensor, int, int, int, int]:  # type: ignore[no-untyped-def]
    """``quantize_8bit`` of a 16-bit matrix into one buffer, scales behind the codes, for the calls
    below, whose host time counts: (buffer, and of codes and scales address and stride)."""
    rows, columns = x.shape
    pitch, tall = (columns + 15) // 16 * 16, (rows + block_rows - 1) // block_rows
    buffer = x.new_empty(rows * pitch + 4 * tall * ((columns + _BLOCK - 1) // _BLOCK), dtype=torch.uint8)
    codes = buffer.data_ptr()
    scales = codes + rows * pitch
    rc = lib.gns_quantize_8bit(
        nat.DTYPE_CODES[x.dtype], block_rows, rows, columns, x.data_ptr(), x.stride(0), codes, pitch, scales, 1, tall,
        stream,
    )
    nat.check(rc, "gns_quantize_8bit")
    return buffer, codes, pitch, scales, tall


def _linear_8bit(x: Tensor, weight: Tensor) -> tuple[Tensor, Tensor]:
    """``x @ weight.T`` with both in 8 bits, and the weight's codes and scales for the gradient: the
    same calls as ``quantize_8bit`` and ``gemm_8bit`` make, with a look at the device and the
    arguments (16-bit matrices of one type) for all of them."""
    index = _device_index(x, weight)
    n, k = weight.shape
    x, weight = _norm_rows(x, k), _norm_rows(weight, k)
    m = x.shape[0]
    y = x.new_empty((m, n))
    lib = nat.load()
    with nat.on_device(index) as stream:
        kept, right, pitch, right_scales, tall = _quantized(lib, weight, _BLOCK, stream)
        if m > 0:
            held, left, left_pitch, left_scales, left_tall = _quantized(lib, x, 1, stream)
            rc = lib.gns_gemm_8bit(
                m, n, k, left, left_pitch, left_scales, 1, left_tall, right, 1, pitch, right_scales, tall, 1,
                y.data_ptr(), nat.DTYPE_CODES[x.dtype], n, stream,
            )
            nat.check(rc, "gns_gemm_8bit")
    return y, kept


def _linear_8bit_gradient(grad: Tensor, kept: Tensor, n: int, k: int) -> Tensor:
    """The gradient [m, k] of x in ``_linear_8bit`` from that of its output [m, n]."""
    index = _device_index(grad, kept)
    grad = _norm_rows(grad, n)
    m = grad.shape[0]
    dx = grad.new_empty((m, k))
    if m == 0:
        return dx
    pitch = (k + 15) // 16 * 16
    right = kept.data_ptr()
    lib = nat.load()
    with nat.on_device(index) as stream:
        held, left, left_pitch, left_scales, left_tall = _quantized(lib, grad, 1, stream)
        rc = lib.gns_gemm_8bit(
            m, k, n, left, left_pitch, left_scales, 1, left_tall, right, pitch, 1, right + n * pitch, 1,
            (n + _BLOCK - 1) // _BLOCK, dx.data_ptr(), nat.DTYPE_CODES[grad.dtype], k, stream,
        )
        nat.check(rc, "gns_gemm_8bit")
    return dx


def _rows_product(left: Tensor, right: Tensor) -> Tensor:
    """``gemm(left.t(), right)`` of 16-bit matrices [rows, a] and [rows, b], rows > 0, as the
    gradients of linear layers have them."""
    index = _device_index(left, right)
    (rows, a), b = left.shape, right.shape[1]
    left, left_place, left_pitch = _row_layout(left)
    right, right_place, right_pitch = _row_layout(right)
    out = left.new_empty((a, b))
    code = nat.DTYPE_CODES[left.dtype]
    with nat.on_device(index) as stream:
        rc = nat.load().gns_gemm(
            code, 1, a, b, rows, left_place, rows * left_pitch, 1, left_pitch, right_place, rows * right_pitch,
            right_pitch, 1, None, 0, 0, 0, out.data_ptr(), code, a * b, b, 1.0, 0.0, 0, stream,
        )
    nat.check(rc, "gns_gemm")
    return out


# --------------------------------------------------------------------- RMS norm
def _rms_check(x: Tensor, weight: Tensor, residual: Tensor | None) -> int:
    columns = _norm_check(x, weight, None)
    if residual is not None and residual.shape != x.shape:
        raise ValueError("x and residual shapes differ")
    if residual is not None and residual.dtype != x.dtype:
        raise TypeError("x and residual must share a dtype")
    return columns


def rms_norm(
    x: Tensor, weight: Tensor, residual: Tensor | None = None, epsilon: float = 1e-5
) -> tuple[Tensor, Tensor, Tensor]:
    """Root-mean-square norm of a residual stream: ``total = x + residual`` and
    ``y = total * rstd * weight`` with ``rstd = 1 / sqrt(mean(total^2) + epsilon)`` over the last
    dimension.

    Returns y and total (x's type, contiguous; total is x itself without a residual) and the
    fp32 rstd of each row. total is rounded to x's type before the norm; all arithmetic is fp32.
    weight has a floating type of its own."""
    index = _device_index(x, weight, residual)
    columns = _rms_check(x, weight, residual)
    flat = _norm_rows(x, columns)
    other = _norm_rows(residual, columns) if residual is not None else None
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    total = torch.empty_like(y) if other is not None else x
    rstd = x.new_empty(x.shape[:-1], dtype=torch.float32)
    w = weight.contiguous()
    with nat.on_device(index) as stream:
        rc = nat.load().gns_rms_norm_forward(
            nat.dtype_code(x.dtype), nat.dtype_code(w.dtype), flat.shape[0], columns, flat.data_ptr(), flat.stride(0),
            nat.ptr(other), other.stride(0) if other is not None else 0, w.data_ptr(), float(epsilon), y.data_ptr(),
            total.data_ptr(), rstd.data_ptr(), stream,
        )
    nat.check(rc, "gns_rms_norm_forward")
    return y, total, rstd


def rms_norm_8bit(
    x: Tensor, weight: Tensor, residual: Tensor | None = None, epsilon: float = 1e-5
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """``rms_norm`` whose y comes as e4m3 codes with a scale for each 128 columns of a row, as
    ``quantize_8bit`` makes them of the unrounded y: the left factor of ``gemm_8bit``.

    Returns the codes [rows, columns] and scales [rows, ceil(columns / 128)] (rows: all dimensions
    of x but the last), total and rstd as ``rms_norm``."""
    index = _device_index(x, weight, residual)
    columns = _rms_check(x, weight, residual)
    flat = _norm_rows(x, columns)
    other = _norm_rows(residual, columns) if residual is not None else None
    rows = flat.shape[0]
    codes, scales = _code_buffers(x, rows, columns)
    total = torch.empty_like(x, memory_format=torch.contiguous_format) if other is not None else x
    rstd = x.new_empty(x.shape[:-1], dtype=torch.float32)
    w = weight.contiguous()
    with nat.on_device(index) as stream:
        rc = nat.load().gns_rms_norm_forward_8bit(
            nat.dtype_code(x.dtype), nat.dtype_code(w.dtype), rows, columns, flat.data_ptr(), flat.stride(0),
            nat.ptr(other), other.stride(0) if other is not None else 0, w.data_ptr(), float(epsilon), codes.data_ptr(),
            codes.stride(0), scales.data_ptr(), *scales.stride(), total.data_ptr(), rstd.data_ptr(), stream,
        )
    nat.check(rc, "gns_rms_norm_forward_8bit")
    return codes, scales, total, rstd


def rms_norm_backward(
    grad: Tensor, total: Tensor, weight: Tensor, rstd: Tensor, grad_total: Tensor | None = None
) -> tuple[Tensor, Tensor]:
    """Gradients (dx, dweight) of ``rms_norm`` from the gradients of y and of total (which may be
    None). dx is the gradient of x and of the residual alike, of total's type; dweight has the
    weight's type, its sum over the rows is fp32 in a fixed order."""
    index = _device_index(grad, total, weight, rstd, grad_total)
    columns = _rms_check(total, weight, grad_total)
    if grad.shape != total.shape:
        raise ValueError("grad and total shapes differ")
    if grad.dtype != total.dtype:
        raise TypeError("grad and total must share a dtype")
    rows = total.numel() // columns
    if rstd.dtype != torch.float32 or rstd.numel() != rows or not rstd.is_contiguous():
        raise ValueError("rstd must be contiguous float32 with one entry per row")
    flat, g = _norm_rows(total, columns), _norm_rows(grad, columns)
    more = _norm_rows(grad_total, columns) if grad_total is not None else None
    w = weight.contiguous()
    dx = torch.empty_like(total, memory_format=torch.contiguous_format)
    dweight = torch.empty_like(w)
    lib = nat.load()
    nbytes = lib.gns_rms_norm_backward_workspace_size(rows, columns)
    ws = total.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    with nat.on_device(index) as stream:
        rc = lib.gns_rms_norm_backward(
            nat.dtype_code(total.dtype), nat.dtype_code(w.dtype), rows, columns, g.data_ptr(), g.stride(0),
            flat.data_ptr(), flat.stride(0), w.data_ptr(), rstd.data_ptr(), nat.ptr(more),
            more.stride(0) if more is not None else 0, dx.data_ptr(), dweight.data_ptr(), nat.ptr(ws), nbytes, stream,
        )
    nat.check(rc, "gns_rms_norm_backward")
    return dx, dweight


# ---------------------------------------------------- distillation from top logits
def _distillation_rows(logits: Tensor, indices: Tensor, teacher: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    if logits.ndim != 2 or logits.shape[1] == 0:
        raise ValueError("expected logits [rows, vocabulary]")
    if indices.ndim != 2 or indices.shape != teacher.shape or indices.shape[0] != logits.shape[0]:
        raise ValueError("expected indices and teacher [rows, top], a row for each row of the logits")
    if indices.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"indices must be int32 or int64, got {indices.dtype}")
    nat.dtype_code(logits.dtype)
    nat.dtype_code(teacher.dtype)
    top = indices.shape[1]

    def rows(t: Tensor) -> Tensor:
        return t if t.stride(1) == 1 or top <= 1 else t.contiguous()

    return _norm_rows(logits, logits.shape[1]), rows(indices), rows(teacher)


def _row_values(t: Tensor, rows: int, name: str) -> Tensor:
    if t.dtype != torch.float32 or t.shape != (rows,):
        raise ValueError(f"{name} must be float32 with one value for each row")
    return t.contiguous()


def _distillation(
    z: Tensor, indices: Tensor, teacher: Tensor, temperature: float, grad: Tensor | None, loss: Tensor | None,
    stats: Tensor | None, dlogits: Tensor | None,
) -> None:
    rows, vocabulary = z.shape
    with nat.on_device(z.get_device()) as stream:
        rc = nat.load().gns_distillation_loss(
            nat.dtype_code(z.dtype), rows, vocabulary, indices.shape[1], z.data_ptr(), z.stride(0), indices.data_ptr(),
            8 * indices.element_size(), indices.stride(0), teacher.data_ptr(), nat.dtype_code(teacher.dtype),
            teacher.stride(0), float(temperature), nat.ptr(grad), nat.ptr(loss), nat.ptr(stats), nat.ptr(dlogits),
            vocabulary, stream,
        )
    nat.check(rc, "gns_distillation_loss")


def distillation_loss(
    logits: Tensor, indices: Tensor, teacher: Tensor, temperature: float = 1.0
) -> tuple[Tensor, Tensor]:
    """The loss of each row against a teacher's top logits:
    ``T^2 * sum_j p_j (log p_j - log q[i_j])`` with p the softmax over the row's entries of
    ``teacher / T`` and q that of ``logits / T`` over the whole vocabulary.

    logits [rows, vocabulary] and teacher [rows, top] are float16, bfloat16 or float32, indices
    [rows, top] int32 or int64; top is at most 1024. An entry whose index is outside the vocabulary
    (-1) has no part in its row; an index may come more than once. A row without entries, or
    whose entries' logits are all -inf, has a loss of zero whatever its logits hold. Where they
    count, logits of -inf have a q of zero, and a NaN, a +inf or a row of -inf alone makes
    the row's loss and gradient NaN.

    Returns the fp32 loss [rows] and the statistics [rows, 2] that
    ``distillation_loss_backward`` takes."""
    _device_index(logits, indices, teacher)
    z, index, t = _distillation_rows(logits, indices, teacher)
    loss = z.new_empty(z.shape[0], dtype=torch.float32)
    stats = z.new_empty((z.shape[0], 2), dtype=torch.float32)
    _distillation(z, index, t, temperature, None, loss, stats, None)
    return loss, stats


def distillation_loss_backward(
    grad: Tensor, logits: Tensor, indices: Tensor, teacher: Tensor, statistics: Tensor, temperature: float = 1.0
) -> Tensor:
    """The gradient of the logits, ``grad * T * (q - p)``, from the gradient of each row's loss
    (fp32) and the statistics that ``distillation_loss`` returned. Of the logits' type; rows
    without entries get zeros."""
    _device_index(grad, logits, indices, teacher, statistics)
    z, index, t = _distillation_rows(logits, indices, teacher)
    g = _row_values(grad, z.shape[0], "grad")
    if statistics.dtype != torch.float32 or statistics.shape != (z.shape[0], 2) or not statistics.is_contiguous():
        raise ValueError("statistics must be contiguous float32 [rows, 2]")
    if statistics.data_ptr() % 8 != 0:  # the kernel reads a row's pair at once
        statistics = statistics.clone()
    dlogits = torch.empty_like(z, memory_format=torch.contiguous_format)
    _distillation(z, index, t, temperature, g, None, statistics, dlogits)
    return dlogits


def distillation_loss_gradient(
    grad: Tensor, logits: Tensor, indices: Tensor, teacher: Tensor, temperature: float = 1.0
) -> tuple[Tensor, Tensor]:
    """``distillation_loss`` and the gradient of the logits in one call, which reads the logits from
    memory once: for a loop that knows each row's weight in its loss beforehand (``grad``, fp32, a
    mask over the number of tokens for a mean) and goes on with ``logits.backward(dlogits)``.

    Returns the loss [rows] and dlogits."""
    _device_index(grad, logits, indices, teacher)
    z, index, t = _distillation_rows(logits, indices, teacher)
    g = _row_values(grad, z.shape[0], "grad")
    loss = z.new_empty(z.shape[0], dtype=torch.float32)
    dlogits = torch.empty_like(z, memory_format=torch.contiguous_format)
    _distillation(z, index, t, temperature, g, loss, None, dlogits)
    return loss, dlogits
