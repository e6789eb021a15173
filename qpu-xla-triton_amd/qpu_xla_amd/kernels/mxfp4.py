"""Microscaling blocks and linears over weights of 4-bit ones, on gfx950.

A block is 32 elements of a row under one shared power of two (OCP Microscaling Formats): 4-bit e2m1 elements
(``mxfp4``) or 8-bit e4m3 ones (``mxfp8``).  Stored as values and scales of their own: mxfp4 values uint8 [R, K/2] with
the lower index in a byte's low half (``torch.float4_e2m1fn_x2``'s layout), mxfp8 values float8_e4m3fn [R, K], scales
uint8 [R, K/32] (bytes of ``torch.float8_e8m0fnu``).

* ``quantize_mxfp4``, ``quantize_mxfp8`` -- float rows to blocks; ``dequantize_mxfp4``, ``dequantize_mxfp8`` back.  A
  block with an infinity or a NaN becomes NaN as a whole.
* ``mxfp4_gemm`` -- ``a @ w.T (+ bias)`` over activations in either format; ``mxfp4_linear`` takes them as floats and
  quantises them first.
* ``mxfp4_gated_gemm``, ``mxfp4_gated_linear`` -- ``f(a @ gate.T) * (a @ up.T)``, the inner product of a feed-forward
  block, as floats or as the blocks that the next linear takes.

Sums are fp32, each result is rounded once.  An output shares no memory with the operands.  There are no gradients: the weights are quantised ones, for serving.  No
counterpart in the reference, whose block formats are ggml's.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Any

import torch

from qpu_xla_amd import _lib
from qpu_xla_amd._paged import TYPES, workspace_for
from qpu_xla_amd._rows import (
    FP8,
    MX_BLOCK,
    float_rows,
    mx_format,
    mx_outputs,
    mx_rows,
    new_rows,
    require_current_gpu,
    share_memory,
    vector,
)
from qpu_xla_amd._tensors import stream_handle
from qpu_xla_amd.errors import KernelError
from qpu_xla_amd.kernel import Kernel
from qpu_xla_amd.kernels.add_rms_norm import add_rms_norm_mxfp4, add_rms_norm_mxfp8

_GATES = {"silu": _lib.GATE_SILU, "gelu": _lib.GATE_GELU}
_BLOCK_KINDS = {"mxfp8": _lib.ROWS_MXFP8, "mxfp4": _lib.ROWS_MXFP4}


def _quantize(name: str, fp8: bool, x: torch.Tensor, values: torch.Tensor | None, scales: torch.Tensor | None,
              stream: Any) -> tuple[torch.Tensor, torch.Tensor]:
    rows, columns, code, stride = float_rows(name, "x", x)
    values, v_stride, scales, s_stride = mx_outputs(name, x, rows, columns, fp8, values, scales, stream)
    require_current_gpu(name, x, values, scales)
    _lib.call("qxt_quantize_mx", x.data_ptr(), stride, code, values.data_ptr(), v_stride, scales.data_ptr(), s_stride, rows,
              columns, _lib.MX_FP8 if fp8 else _lib.MX_FP4, stream_handle(stream))
    return values, scales


def quantize_mxfp4(x: torch.Tensor, values: torch.Tensor | None = None, scales: torch.Tensor | None = None, *,
                   stream: Any = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Float rows [R, K] (K a multiple of 32) -> (packed 4-bit values uint8 [R, K/2], scales uint8 [R, K/32])."""
    return _quantize("quantize_mxfp4", False, x, values, scales, stream)


def quantize_mxfp8(x: torch.Tensor, values: torch.Tensor | None = None, scales: torch.Tensor | None = None, *,
                   stream: Any = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Float rows [R, K] (K a multiple of 32) -> (values float8_e4m3fn [R, K], scales uint8 [R, K/32])."""
    return _quantize("quantize_mxfp8", True, x, values, scales, stream)


def _dequantize(name: str, fmt: int, values: torch.Tensor, scales: torch.Tensor, out: torch.Tensor | None,
                dtype: torch.dtype | None, stream: Any) -> torch.Tensor:
    rows, columns, found, _ = mx_rows(name, "the rows", values, scales, (fmt,))
    if found != fmt:
        raise ValueError(f"{name}: the values are of another block format")
    if out is None:
        out = new_rows(stream, values, (rows, columns), torch.float32 if dtype is None else dtype)
    elif dtype is not None and out.dtype is not dtype:
        raise ValueError(f"{name}: out is not of the given dtype")
    out_rows, out_columns, code, stride = float_rows(name, "out", out)
    if (out_rows, out_columns) != (rows, columns):
        raise ValueError(f"{name}: out must be [{rows}, {columns}]")
    require_current_gpu(name, values, scales, out)
    _lib.call("qxt_dequantize_mx", values.data_ptr(), 0 if rows <= 1 else values.stride(0), scales.data_ptr(),
              0 if rows <= 1 else scales.stride(0), out.data_ptr(), stride, code, rows, columns, fmt, stream_handle(stream))
    return out


def dequantize_mxfp4(values: torch.Tensor, scales: torch.Tensor, out: torch.Tensor | None = None, *,
                     dtype: torch.dtype | None = None, stream: Any = None) -> torch.Tensor:
    """What 4-bit blocks stand for, float32 unless ``out`` or ``dtype`` says otherwise."""
    return _dequantize("dequantize_mxfp4", _lib.MX_FP4, values, scales, out, dtype, stream)


def dequantize_mxfp8(values: torch.Tensor, scales: torch.Tensor, out: torch.Tensor | None = None, *,
                     dtype: torch.dtype | None = None, stream: Any = None) -> torch.Tensor:
    """What 8-bit blocks stand for, float32 unless ``out`` or ``dtype`` says otherwise."""
    return _dequantize("dequantize_mxfp8", _lib.MX_FP8, values, scales, out, dtype, stream)


# -------------------------------------------------------------------- linears


def _float_out(name: str, like: torch.Tensor, out: torch.Tensor | None, dtype: torch.dtype, rows: int, columns: int,
               stream: Any) -> tuple[torch.Tensor, int, int]:
    """(out, type code, byte stride)."""
    if out is None:
        code = TYPES.get(dtype)
        if code is None:
            raise ValueError(f"{name}: the output must be float32, bfloat16 or float16")
        return new_rows(stream, like, (rows, columns), dtype), code, columns * (2 if code else 4)
    if out.dtype is not dtype:
        raise ValueError(f"{name}: out is not of the output's type")
    got_rows, got_columns, code, stride = float_rows(name, "out", out)
    if (got_rows, got_columns) != (rows, columns):
        raise ValueError(f"{name}: out must be [{rows}, {columns}]")
    return out, code, stride


def _workspace(rows: int, columns: int, depth: int, weights: int, fmt: int, x_kind: int, kind: int, stream: Any,
               device: torch.device) -> tuple[torch.Tensor | None, int | None, int]:
    """(the workspace, its address, its size)."""
    size = (_lib._lib or _lib.load()).qxt_mxfp4_linear_workspace(rows, columns, depth, weights, fmt, x_kind, kind)
    if not size:
        return None, None, 0
    workspace = workspace_for(stream, size, device)
    return workspace, workspace.data_ptr(), size


def _x_kind(x: torch.Tensor, code: int, stride: int) -> int:
    return 1 + code if (x.data_ptr() | stride) % 16 else 1 + code + _lib.ROWS_ALIGNED


def mxfp4_gemm(
    a_values: torch.Tensor,
    a_scales: torch.Tensor,
    w_values: torch.Tensor,
    w_scales: torch.Tensor,
    bias: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    *,
    dtype: torch.dtype | None = None,
    stream: Any = None,
) -> torch.Tensor:
    """``a @ w.T (+ bias)`` [M, N] of blocks a [M, K] (either format) and w [N, K] (mxfp4), float32 unless said otherwise."""
    name = "mxfp4_gemm"
    m, k, fmt, a = mx_rows(name, "a", a_values, a_scales)
    n, w_k, _, w = mx_rows(name, "w", w_values, w_scales, (_lib.MX_FP4,))
    if k != w_k:
        raise ValueError(f"{name}: a and w differ in K")
    bias_at = vector(name, "bias", bias, n)
    dtype = dtype if dtype is not None else torch.float32 if out is None else out.dtype
    out, code, stride = _float_out(name, a_values, out, dtype, m, n, stream)
    require_current_gpu(name, a_values, a_scales, w_values, w_scales, bias, out)
    workspace, at, size = _workspace(m, n, k, 1, fmt, 0, code, stream, a_values.device)
    _lib.call("qxt_mxfp4_gemm", a, fmt, w, bias_at, out.data_ptr(), stride, code, m, n, k, at, size,
              stream_handle(stream))
    return out


def mxfp4_linear(
    x: torch.Tensor,
    w_values: torch.Tensor,
    w_scales: torch.Tensor,
    bias: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    *,
    activations: str = "mxfp8",
    dtype: torch.dtype | None = None,
    stream: Any = None,
) -> torch.Tensor:
    """``mxfp4_gemm`` of float activations [M, K], quantised to ``activations`` first; x's type unless said otherwise."""
    name = "mxfp4_linear"
    m, k, x_code, x_stride = float_rows(name, "x", x)
    fmt = mx_format(name, activations)
    n, w_k, _, w = mx_rows(name, "w", w_values, w_scales, (_lib.MX_FP4,))
    if k != w_k:
        raise ValueError(f"{name}: x and w differ in K")
    bias_at = vector(name, "bias", bias, n)
    dtype = dtype if dtype is not None else x.dtype if out is None else out.dtype
    out, code, stride = _float_out(name, x, out, dtype, m, n, stream)
    require_current_gpu(name, x, w_values, w_scales, bias, out)
    workspace, at, size = _workspace(m, n, k, 1, fmt, _x_kind(x, x_code, x_stride), code, stream, x.device)
    _lib.call("qxt_mxfp4_linear", x.data_ptr(), x_stride, x_code, fmt, w, bias_at, out.data_ptr(), stride, code, m, n, k, at, size,
              stream_handle(stream))
    return out


def _gated_out(name: str, like: torch.Tensor, output: Any, out: Any, m: int, n: int, stream: Any) -> tuple[Any, list, int, list]:
    """(what is returned, its tensors, kind, [address, stride, scales' address, stride])."""
    if isinstance(output, str):
        kind = _BLOCK_KINDS.get(output)
        if kind is None:
            raise ValueError(f"{name}: the output must be a float type, 'mxfp8' or 'mxfp4', got {output!r}")
        if out is not None and not (isinstance(out, tuple) and len(out) == 2):
            raise ValueError(f"{name}: out must be (values, scales)")
        values, scales = (None, None) if out is None else out
        values, stride, scales, scale_stride = mx_outputs(name, like, m, n, output == "mxfp8", values, scales, stream)
        return (values, scales), [values, scales], kind, [values.data_ptr(), stride, scales.data_ptr(), scale_stride]
    if out is not None and not isinstance(out, torch.Tensor):
        raise ValueError(f"{name}: out must be a tensor")
    out, kind, stride = _float_out(name, like, out, output, m, n, stream)
    return out, [out], kind, [out.data_ptr(), stride, None, 0]


def _gate_weights(name: str, k: int, gate_values: torch.Tensor, gate_scales: torch.Tensor, up_values: torch.Tensor,
                  up_scales: torch.Tensor) -> tuple[int, bytes, bytes]:
    n, gate_k, _, gate = mx_rows(name, "gate", gate_values, gate_scales, (_lib.MX_FP4,))
    up_n, up_k, _, up = mx_rows(name, "up", up_values, up_scales, (_lib.MX_FP4,))
    if gate_k != k or up_k != k or n != up_n:
        raise ValueError(f"{name}: gate and up must have one shape, and the activations' K")
    return n, gate, up


def _gate_function(name: str, gate: str) -> int:
    if gate not in _GATES:
        raise ValueError(f"{name}: the gate function must be 'silu' or 'gelu', got {gate!r}")
    return _GATES[gate]


def mxfp4_gated_gemm(
    a_values: torch.Tensor,
    a_scales: torch.Tensor,
    gate_values: torch.Tensor,
    gate_scales: torch.Tensor,
    up_values: torch.Tensor,
    up_scales: torch.Tensor,
    out: Any = None,
    *,
    gate: str = "silu",
    output: Any = None,
    stream: Any = None,
) -> Any:
    """``f(a @ gate.T) * (a @ up.T)`` [M, N] of blocks, f ``gate`` ("silu", or "gelu" by erf) of the fp32 sums.

    ``output``: a float type (float32, or ``out``'s, where it is not given), or "mxfp8" / "mxfp4" for (values, scales), N a
    multiple of 32, and then ``out`` is such a pair.
    """
    name = "mxfp4_gated_gemm"
    m, k, fmt, a = mx_rows(name, "a", a_values, a_scales)
    n, gate_at, up_at = _gate_weights(name, k, gate_values, gate_scales, up_values, up_scales)
    function = _gate_function(name, gate)
    if output is None:
        output = out.dtype if isinstance(out, torch.Tensor) else torch.float32
    result, tensors, kind, places = _gated_out(name, a_values, output, out, m, n, stream)
    require_current_gpu(name, a_values, a_scales, gate_values, gate_scales, up_values, up_scales, *tensors)
    workspace, at, size = _workspace(m, n, k, 2, fmt, 0, kind, stream, a_values.device)
    _lib.call("qxt_mxfp4_gated_gemm", a, fmt, gate_at, up_at, function, *places, kind, m, n, k, at, size,
              stream_handle(stream))
    return result


def mxfp4_gated_linear(
    x: torch.Tensor,
    gate_values: torch.Tensor,
    gate_scales: torch.Tensor,
    up_values: torch.Tensor,
    up_scales: torch.Tensor,
    out: Any = None,
    *,
    activations: str = "mxfp8",
    gate: str = "silu",
    output: Any = None,
    stream: Any = None,
) -> Any:
    """``mxfp4_gated_gemm`` of float activations [M, K], quantised to ``activations`` first; x's type unless said otherwise."""
    name = "mxfp4_gated_linear"
    m, k, x_code, x_stride = float_rows(name, "x", x)
    fmt = mx_format(name, activations)
    n, gate_at, up_at = _gate_weights(name, k, gate_values, gate_scales, up_values, up_scales)
    function = _gate_function(name, gate)
    if output is None:
        output = out.dtype if isinstance(out, torch.Tensor) else x.dtype
    result, tensors, kind, places = _gated_out(name, x, output, out, m, n, stream)
    require_current_gpu(name, x, gate_values, gate_scales, up_values, up_scales, *tensors)
    workspace, at, size = _workspace(m, n, k, 2, fmt, _x_kind(x, x_code, x_stride), kind, stream, x.device)
    _lib.call("qxt_mxfp4_gated_linear", x.data_ptr(), x_stride, x_code, fmt, gate_at, up_at, function, *places, kind, m, n, k, at, size,
              stream_handle(stream))
    return result


# What the C entries take: rows or columns, and K.
_MOST_ROWS, _MOST_K = (2**31 - 1) // 32, 2**22


def feed_forward(
    x: torch.Tensor, residual: torch.Tensor | None, norm_weight: torch.Tensor, gate: Any, up: Any, down: Any, epsilon: float,
    activations: str, function: str, residual_out: torch.Tensor | None, out: torch.Tensor | None, dtype: torch.dtype | None,
    stream: Any,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``quantization.mxfp4_feed_forward``: the norm, ``mxfp4_gated_gemm`` and ``mxfp4_gemm`` in a row.

    The norm may write the sum over the residual, so that nothing may be refused after it: the checks of all three come
    first, and so do the outputs and the workspace.
    """
    name = "mxfp4_feed_forward"
    m, k, _, _ = float_rows(name, "x", x)
    fmt, kind = mx_format(name, activations), _BLOCK_KINDS[activations]
    gate_function = _gate_function(name, function)
    n, gate_at, up_at = _gate_weights(name, k, gate.values, gate.scales, up.values, up.scales)
    columns, down_k, _, down_at = mx_rows(name, "down", down.values, down.scales, (_lib.MX_FP4,))
    if down_k != n:
        raise ValueError(f"{name}: the gated rows and down differ in K")
    if max(m, n, columns) > _MOST_ROWS or max(k, n) >= _MOST_K:
        raise ValueError(f"{name}: too many rows or columns")
    weights = (gate.values, up.values, down.values, gate.scales, up.scales, down.scales)
    ranges = [(w.data_ptr(), w.numel()) for w in weights]
    if any(at % 16 for at, _ in ranges[:3]):
        raise ValueError(f"{name}: weights must be in rows aligned to 16 bytes")
    if dtype is None:
        dtype = x.dtype if out is None else out.dtype
    given = out
    out, code, stride = _float_out(name, x, out, dtype, m, columns, stream)
    h, h_stride, h_scales, h_scale_stride = mx_outputs(name, x, m, n, fmt == _lib.MX_FP8, None, None, stream)
    require_current_gpu(name, x, *weights, out)
    for written in (given, residual_out):
        # (A residual_out that is not rows is refused by the norm, before its launch.)
        if written is not None and m and written.dim() == 2:
            first = written.data_ptr()
            last = first + ((m - 1) * written.stride(0) + written.shape[1]) * written.element_size()
            if any(first < at + size and at < last for at, size in ranges):
                raise ValueError(f"{name}: an output shares memory with another operand")
    if given is not None and any(t is not None and t.dim() == d and share_memory(out, t) for t, d in ((norm_weight, 1), (residual_out, 2))):
        raise ValueError(f"{name}: an output shares memory with another operand")
    query = (_lib._lib or _lib.load()).qxt_mxfp4_linear_workspace
    size = max(query(m, n, k, 2, fmt, 0, kind), query(m, columns, n, 1, fmt, 0, code))
    workspace = workspace_for(stream, size, x.device)
    at = None if workspace is None else workspace.data_ptr()

    norm = add_rms_norm_mxfp8 if fmt == _lib.MX_FP8 else add_rms_norm_mxfp4
    values, scales, total = norm(x, norm_weight, residual, epsilon=epsilon, residual_out=residual_out, stream=stream)
    handle = stream_handle(stream)
    rows = _lib.MX_MATRIX.pack(values.data_ptr(), values.shape[1], scales.data_ptr(), scales.shape[1])
    _lib.call("qxt_mxfp4_gated_gemm", rows, fmt, gate_at, up_at, gate_function, h.data_ptr(), h_stride, h_scales.data_ptr(),
              h_scale_stride, kind, m, n, k, at, size, handle)
    rows = _lib.MX_MATRIX.pack(h.data_ptr(), h_stride, h_scales.data_ptr(), h_scale_stride)
    _lib.call("qxt_mxfp4_gemm", rows, fmt, down_at, None, out.data_ptr(), stride, code, m, columns, n, at, size, handle)
    return out, total


# -------------------------------------------------------------- queue kernels


@dataclass(frozen=True, slots=True)
class Mxfp4GatedOptions:
    """Last argument of ``MXFP4_GATED_GEMM_KERNEL``."""

    gate: str = "silu"


def mxfp4_gemm_grid(rows: int, columns: int) -> tuple[int, int, int]:
    """Grid of ``MXFP4_GEMM_KERNEL`` and ``MXFP4_GATED_GEMM_KERNEL``: 16 x 16 tiles (columns, rows) of the result."""
    return ((columns + 15) // 16, (rows + 15) // 16, 1)


def _execute_mxfp4_gemm(stream: Any, args: tuple[Any, ...], grid: tuple[int, int, int]) -> None:
    if len(args) != 6 or not all(isinstance(a, torch.Tensor) for a in args[:5]) or not (args[5] is None or isinstance(args[5], torch.Tensor)):
        raise KernelError("mxfp4 gemm expects (a_values, a_scales, w_values, w_scales, destination, bias or None)")
    *operands, out, bias = args
    if out.dim() != 2 or tuple(grid) != mxfp4_gemm_grid(*out.shape):
        raise KernelError(f"mxfp4 gemm grid must be 16 x 16 tiles of the destination, got {tuple(grid)}")
    mxfp4_gemm(*operands, bias, out, stream=stream)


MXFP4_GEMM_KERNEL = Kernel("gfx950.mxfp4_gemm", _execute_mxfp4_gemm)


def _execute_mxfp4_gated_gemm(stream: Any, args: tuple[Any, ...], grid: tuple[int, int, int]) -> None:
    if (len(args) != 9 or not all(isinstance(a, torch.Tensor) for a in args[:7])
            or not (args[7] is None or isinstance(args[7], torch.Tensor)) or not isinstance(args[8], Mxfp4GatedOptions)):
        raise KernelError("mxfp4 gated gemm expects (a_values, a_scales, gate_values, gate_scales, up_values, up_scales, "
                          "destination, its scales or None, Mxfp4GatedOptions)")
    *operands, out, scales, options = args
    columns = 0
    if out.dim() == 2:
        columns = out.shape[1] * (2 if scales is not None and out.dtype is not FP8 else 1)
    if out.dim() != 2 or tuple(grid) != mxfp4_gemm_grid(out.shape[0], columns):
        raise KernelError(f"mxfp4 gated gemm grid must be 16 x 16 tiles of the destination, got {tuple(grid)}")
    if scales is None:
        mxfp4_gated_gemm(*operands, out, gate=options.gate, output=out.dtype, stream=stream)
    else:
        mxfp4_gated_gemm(*operands, (out, scales), gate=options.gate, output="mxfp8" if out.dtype is FP8 else "mxfp4", stream=stream)


MXFP4_GATED_GEMM_KERNEL = Kernel("gfx950.mxfp4_gated_gemm", _execute_mxfp4_gated_gemm)

__all__ = [
    "MXFP4_GATED_GEMM_KERNEL", "MXFP4_GEMM_KERNEL", "MX_BLOCK", "Mxfp4GatedOptions", "dequantize_mxfp4", "dequantize_mxfp8",
    "mxfp4_gated_gemm", "mxfp4_gated_linear", "mxfp4_gemm", "mxfp4_gemm_grid", "mxfp4_linear", "quantize_mxfp4", "quantize_mxfp8",
]
