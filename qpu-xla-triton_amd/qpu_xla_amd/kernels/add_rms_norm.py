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
from qpu_xla_amd._paged import TYPES, empty_for
from qpu_xla_amd._rows import MX_BLOCK, float_rows, mx_outputs, require_current_gpu, vector
from qpu_xla_amd._tensors import row_stride, rows_are_dense, stream_handle
from qpu_xla_amd.errors import KernelError
from qpu_xla_amd.kernel import Kernel
from qpu_xla_amd.kernels.quantize import Q8_0_BLOCK_BYTES


class _Call:
    """The arguments that every form shares."""

    def __init__(self, name: str, x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None,
                 residual_out: torch.Tensor | None, epsilon: float, stream: Any) -> None:
        self.name, self.stream, self.device = name, stream, x.device
        self.rows, self.columns, x_code, x_stride = float_rows(name, "x", x)
        if self.columns == 0:
            raise ValueError(f"{name}: rows must not be empty")
        if not epsilon >= 0.0:
            raise ValueError(f"{name}: epsilon must not be negative")
        weight_at = vector(name, "weight", weight, self.columns)
        self.tensors = [weight, residual]
        head = [x.data_ptr(), x_stride, x_code]
        if residual is None:
            if residual_out is not None:
                raise ValueError(f"{name}: residual_out without a residual")
            head += [None, 0, 0, None, 0]
        else:
            rows, columns, code, stride = float_rows(name, "residual", residual)
            if residual_out is None:
                residual_out = self.empty((rows, columns), residual.dtype)
            elif residual_out.dtype is not residual.dtype:
                raise ValueError(f"{name}: residual_out must have the residual's type")
            out_rows, out_columns, _, out_stride = float_rows(name, "residual_out", residual_out)
            if (rows, columns) != (self.rows, self.columns) or (out_rows, out_columns) != (rows, columns):
                raise ValueError(f"{name}: residual and residual_out must have x's shape")
            head += [residual.data_ptr(), stride, code, residual_out.data_ptr(), out_stride]
        self.sum = residual_out
        self.head = [*head, weight_at, epsilon]
        self.x = x

    def empty(self, shape: tuple[int, ...], dtype: torch.dtype) -> torch.Tensor:
        return empty_for(self.stream, shape, dtype, self.device)

    def run(self, out: torch.Tensor, out_stride: int, scales: torch.Tensor | None, scales_stride: int, kind: int) -> None:
        require_current_gpu(self.name, self.x, *self.tensors, self.sum, out, scales)
        _lib.call("qxt_add_rms_norm", *self.head, out.data_ptr(), out_stride, None if scales is None else scales.data_ptr(),
                  scales_stride, kind, self.rows, self.columns, stream_handle(self.stream))


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
    call = _Call("add_rms_norm", x, weight, residual, residual_out, epsilon, stream)
    if out is None:
        out = call.empty((call.rows, call.columns), x.dtype)
    rows, columns, code, stride = float_rows(call.name, "out", out)
    if (rows, columns) != (call.rows, call.columns):
        raise ValueError("add_rms_norm: out must have x's shape")
    call.run(out, stride, None, 0, code)
    return out, call.sum


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
    call = _Call(name, x, weight, residual, residual_out, epsilon, stream)
    shape = (call.rows, call.columns)
    out = call.empty(shape, torch.int8) if out is None else out
    scales = call.empty(shape[:1], torch.float32) if scales is None else scales
    if out.dtype is not torch.int8 or tuple(out.shape) != shape or (call.rows and not rows_are_dense(out)) or (
            call.rows > 1 and out.stride(0) < call.columns):
        raise ValueError(f"{name}: out must be int8 {list(shape)} with dense rows")
    vector(name, "scales", scales, call.rows)
    call.run(out, out.stride(0) if call.rows > 1 else 0, scales, 0, _lib.ROWS_INT8)
    return out, scales, call.sum


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
    call = _Call(name, x, weight, residual, residual_out, epsilon, stream)
    if call.columns % MX_BLOCK:
        raise ValueError(f"{name}: columns must be a multiple of 32")
    shape = (call.rows, call.columns // MX_BLOCK, Q8_0_BLOCK_BYTES)
    out = call.empty(shape, torch.uint8) if out is None else out
    if out.dtype is not torch.uint8 or tuple(out.shape) != shape or (call.rows and not rows_are_dense(out)) or (
            call.rows > 1 and out.stride(0) < shape[1] * Q8_0_BLOCK_BYTES):
        raise ValueError(f"{name}: out must be uint8 {list(shape)} with dense rows")
    call.run(out, row_stride(out) if call.rows > 1 else 0, None, 0, _lib.ROWS_Q8_0)
    return out, call.sum


def _mx(name: str, kind: int, x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None, epsilon: float,
        values: torch.Tensor | None, scales: torch.Tensor | None, residual_out: torch.Tensor | None,
        stream: Any) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    call = _Call(name, x, weight, residual, residual_out, epsilon, stream)
    values, stride, scales, scales_stride = mx_outputs(name, call.rows, call.columns, kind == _lib.ROWS_MXFP8, values, scales, call.empty)
    call.run(values, stride, scales, scales_stride, kind)
    return values, scales, call.sum


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
