"""The residual's addition and the root-mean-square norm of its rows in one pass, on gfx950.

``sum = x + residual`` (rounded to the residual's type), ``y = sum * f * weight`` with ``f = 1 / sqrt(mean(sum^2) +
epsilon)`` of the rounded sum; without a residual, of x.  ``f`` is computed in 64 bits, it and both products are rounded
to float32, and that y becomes

* ``add_rms_norm`` -- a float type;
* ``add_rms_norm_int8`` -- int8 rows and scales, as ``quantize_rows_int8`` makes them, for the W8A8 linears;
* ``add_rms_norm_q8_0`` -- Q8_0 blocks, as ``quantize_q8_0`` makes them, for the Q4_0 and Q8_0 linears;
* ``add_rms_norm_mxfp8``, ``add_rms_norm_mxfp4`` -- microscaling blocks, as ``quantize_mxfp8`` and ``quantize_mxfp4``
  make them, for ``mxfp4_gemm`` and ``mxfp4_gated_gemm``.

Each returns its outputs and the sum (None without a residual).  ``residual_out`` may be the residual itself, and a float
``out`` of x's type x itself.  The reference's norm programs (``src/qpu_xla/kernels``) are separate fp32 launches; no
counterpart of the fused form exists there.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Any

import torch

from qpu_xla_amd import _lib
from qpu_xla_amd._paged import TYPES
from qpu_xla_amd._rows import MX_BLOCK, float_rows, mx_outputs, new_rows, require_current_gpu, vector
from qpu_xla_amd._tensors import rows_are_dense, stream_handle
from qpu_xla_amd.errors import KernelError
from qpu_xla_amd.kernel import Kernel
from qpu_xla_amd.kernels.quantize import Q8_0_BLOCK_BYTES


def _run(name: str, kind: int, x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None, epsilon: float,
         out: torch.Tensor, out_stride: int, scales: torch.Tensor | None, scales_stride: int,
         residual_out: torch.Tensor | None, stream: Any) -> torch.Tensor | None:
    """The checks and the call that every form shares; the sum."""
    rows, columns, x_code, x_stride = float_rows(name, "x", x)
    if columns == 0:
        raise ValueError(f"{name}: rows must not be empty")
    if not epsilon >= 0.0:
        raise ValueError(f"{name}: epsilon must not be negative")
    weight_at = vector(name, "weight", weight, columns)
    residual_at = sum_at = None
    code = stride = sum_stride = 0
    if residual is None:
        if residual_out is not None:
            raise ValueError(f"{name}: residual_out without a residual")
        require_current_gpu(name, x, weight, out, scales)
    else:
        r_rows, r_columns, code, stride = float_rows(name, "residual", residual)
        if r_rows != rows or r_columns != columns:
            raise ValueError(f"{name}: residual must have x's shape")
        if residual_out is None:
            residual_out, sum_stride = new_rows(stream, residual, (rows, columns), residual.dtype), columns * (2 if code else 4)
        else:
            if residual_out.dtype is not residual.dtype:
                raise ValueError(f"{name}: residual_out must have the residual's type")
            s_rows, s_columns, _, sum_stride = float_rows(name, "residual_out", residual_out)
            if s_rows != rows or s_columns != columns:
                raise ValueError(f"{name}: residual_out must have x's shape")
        residual_at, sum_at = residual.data_ptr(), residual_out.data_ptr()
        require_current_gpu(name, x, weight, residual, residual_out, out, scales)
    _lib.call("qxt_add_rms_norm", x.data_ptr(), x_stride, x_code, residual_at, stride, code, sum_at, sum_stride, weight_at,
              epsilon, out.data_ptr(), out_stride, None if scales is None else scales.data_ptr(), scales_stride, kind, rows,
              columns, stream_handle(stream))
    return residual_out


def _shape(name: str, x: torch.Tensor) -> tuple[int, int]:
    if x.dim() != 2:
        raise ValueError(f"{name}: x must be float32, bfloat16 or float16 [rows, columns] with dense rows")
    return tuple(x.shape)


def add_rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: torch.Tensor | None = None,
    *,
    epsilon: float = 1e-6,
    out: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
    stream: Any = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(y, sum) of float rows x [T, D], fp32 weight [D] and residual [T, D]; y in x's type unless ``out`` is given."""
    shape = _shape("add_rms_norm", x)
    if out is None:
        out = new_rows(stream, x, shape, x.dtype)
    rows, columns, code, stride = float_rows("add_rms_norm", "out", out)
    if (rows, columns) != shape:
        raise ValueError("add_rms_norm: out must have x's shape")
    return out, _run("add_rms_norm", code, x, weight, residual, epsilon, out, stride, None, 0, residual_out, stream)


def add_rms_norm_int8(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: torch.Tensor | None = None,
    *,
    epsilon: float = 1e-6,
    out: torch.Tensor | None = None,
    scales: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
    stream: Any = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """(int8 [T, D], fp32 scales [T], sum): y through ``quantize_rows_int8``'s rule."""
    name = "add_rms_norm_int8"
    shape = _shape(name, x)
    if out is None:
        out, stride = new_rows(stream, x, shape, torch.int8), shape[1]
    else:
        if out.dtype is not torch.int8 or tuple(out.shape) != shape or (shape[1] > 1 and out.stride(1) != 1) or (
                shape[0] > 1 and out.stride(0) < shape[1]):
            raise ValueError(f"{name}: out must be int8 {list(shape)} with dense rows")
        stride = out.stride(0) if shape[0] > 1 else 0
    if scales is None:
        scales = new_rows(stream, x, shape[:1], torch.float32)
    else:
        vector(name, "scales", scales, shape[0])
    total = _run(name, _lib.ROWS_INT8, x, weight, residual, epsilon, out, stride, scales, 0, residual_out, stream)
    return out, scales, total


def add_rms_norm_q8_0(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: torch.Tensor | None = None,
    *,
    epsilon: float = 1e-6,
    out: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
    stream: Any = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(Q8_0 blocks uint8 [T, D/32, 34], sum): y through ``quantize_q8_0``'s rule."""
    name = "add_rms_norm_q8_0"
    rows, columns = _shape(name, x)
    if columns == 0 or columns % MX_BLOCK:
        raise ValueError(f"{name}: columns must be a positive multiple of 32")
    shape = (rows, columns // MX_BLOCK, Q8_0_BLOCK_BYTES)
    if out is None:
        out = new_rows(stream, x, shape, torch.uint8)
    elif out.dtype is not torch.uint8 or tuple(out.shape) != shape or (rows and not rows_are_dense(out)) or (
            rows > 1 and out.stride(0) < shape[1] * Q8_0_BLOCK_BYTES):
        raise ValueError(f"{name}: out must be uint8 {list(shape)} with dense rows")
    stride = out.stride(0) if rows > 1 else 0
    return out, _run(name, _lib.ROWS_Q8_0, x, weight, residual, epsilon, out, stride, None, 0, residual_out, stream)


def _mx(name: str, kind: int, x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None, epsilon: float,
        values: torch.Tensor | None, scales: torch.Tensor | None, residual_out: torch.Tensor | None,
        stream: Any) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    rows, columns = _shape(name, x)
    values, stride, scales, scales_stride = mx_outputs(name, x, rows, columns, kind == _lib.ROWS_MXFP8, values, scales, stream)
    total = _run(name, kind, x, weight, residual, epsilon, values, stride, scales, scales_stride, residual_out, stream)
    return values, scales, total


def add_rms_norm_mxfp8(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: torch.Tensor | None = None,
    *,
    epsilon: float = 1e-6,
    values: torch.Tensor | None = None,
    scales: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
    stream: Any = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """(values float8_e4m3fn [T, D], scales uint8 [T, D/32], sum): y through ``quantize_mxfp8``'s rule."""
    return _mx("add_rms_norm_mxfp8", _lib.ROWS_MXFP8, x, weight, residual, epsilon, values, scales, residual_out, stream)


def add_rms_norm_mxfp4(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: torch.Tensor | None = None,
    *,
    epsilon: float = 1e-6,
    values: torch.Tensor | None = None,
    scales: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
    stream: Any = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """(packed 4-bit values uint8 [T, D/2], scales uint8 [T, D/32], sum): y through ``quantize_mxfp4``'s rule."""
    return _mx("add_rms_norm_mxfp4", _lib.ROWS_MXFP4, x, weight, residual, epsilon, values, scales, residual_out, stream)


@dataclass(frozen=True, slots=True)
class AddRmsNormOptions:
    """Last argument of ``ADD_RMS_NORM_KERNEL``."""

    epsilon: float = 1e-6


def add_rms_norm_grid(x: torch.Tensor) -> tuple[int, int, int]:
    """Grid of ``ADD_RMS_NORM_KERNEL``: (rows, 1, 1)."""
    return (x.shape[0], 1, 1)


_FORMS = {torch.int8: add_rms_norm_int8, torch.float8_e4m3fn: add_rms_norm_mxfp8, torch.uint8: add_rms_norm_mxfp4}


def _execute_add_rms_norm(stream: Any, args: tuple[Any, ...], grid: tuple[int, int, int]) -> None:
    if (len(args) != 7 or not isinstance(args[0], torch.Tensor) or not isinstance(args[1], torch.Tensor)
            or not isinstance(args[3], torch.Tensor) or not all(a is None or isinstance(a, torch.Tensor) for a in args[2:6])
            or not isinstance(args[6], AddRmsNormOptions)):
        raise KernelError("add rms norm expects (x, weight, residual or None, destination, its scales or None, "
                          "residual_out or None, AddRmsNormOptions)")
    x, weight, residual, out, scales, residual_out, options = args
    if x.dim() != 2 or tuple(grid) != add_rms_norm_grid(x):
        raise KernelError(f"add rms norm grid must be (rows, 1, 1), got {tuple(grid)}")
    if (residual is None) != (residual_out is None):
        raise KernelError("add rms norm takes residual and residual_out together")
    shared = {"epsilon": options.epsilon, "residual_out": residual_out, "stream": stream}
    if out.dtype in TYPES or out.dim() == 3:
        if scales is not None:
            raise KernelError("add rms norm: floats and Q8_0 blocks have no scales of their own")
        (add_rms_norm if out.dtype in TYPES else add_rms_norm_q8_0)(x, weight, residual, out=out, **shared)
        return
    if out.dtype not in _FORMS or scales is None:
        raise KernelError("add rms norm: the destination must be floats, int8 rows, Q8_0 or microscaling blocks, quantised rows with scales")
    first = "out" if out.dtype is torch.int8 else "values"
    _FORMS[out.dtype](x, weight, residual, scales=scales, **{first: out}, **shared)


ADD_RMS_NORM_KERNEL = Kernel("gfx950.add_rms_norm", _execute_add_rms_norm)

__all__ = ["ADD_RMS_NORM_KERNEL", "AddRmsNormOptions", "add_rms_norm", "add_rms_norm_grid", "add_rms_norm_int8",
           "add_rms_norm_mxfp4", "add_rms_norm_mxfp8", "add_rms_norm_q8_0"]
