"""Refusals of the norms, the microscaling blocks and their linears (no GPU: checks return before any HIP call), and the
64-bit definitions themselves."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import mx_reference as reference
from qpu_xla_amd import KernelError, LaunchConfig, _lib
from qpu_xla_amd import kernels as k
from qpu_xla_amd.quantization import QuantizedMatrixMxfp4

FAKE, FAR = 1 << 20, 1 << 28  # 16-byte aligned, never dereferenced; operands of one call lie FAR apart
BF16 = torch.bfloat16


def _u8(*shape):
    return torch.zeros(shape, dtype=torch.uint8)


# ------------------------------------------------------------------- Python


@pytest.mark.parametrize("call", [k.quantize_mxfp4, k.quantize_mxfp8])
@pytest.mark.parametrize("args,fragment", [
    ((torch.zeros((2, 64)),), "HIP device"),
    ((torch.zeros((2, 48)),), "multiple of 32"),
    ((torch.zeros((2, 0)),), "multiple of 32"),
    ((torch.zeros((2, 64), dtype=torch.float64),), "x must be"),
    ((torch.zeros(64),), "x must be"),
    ((torch.zeros((2, 128))[:, ::2],), "dense rows"),
    ((torch.zeros((1, 64)).expand(3, 64),), "dense rows"),
    ((torch.zeros((2, 64)), torch.zeros((2, 16), dtype=torch.uint8)), "values must be"),
    ((torch.zeros((2, 64)), None, torch.zeros((2, 3), dtype=torch.uint8)), "scales must be"),
    ((torch.zeros((2, 64)), None, torch.zeros((2, 2), dtype=torch.int8)), "scales must be"),
])
def test_quantise_refuses(call, args, fragment) -> None:
    with pytest.raises(ValueError, match=fragment):
        call(*args)


@pytest.mark.parametrize("call,values,scales,options,fragment", [
    (k.dequantize_mxfp4, _u8(2, 32), _u8(2, 2), {}, "HIP device"),
    (k.dequantize_mxfp4, _u8(2, 32), _u8(2, 3), {}, "scales must be"),
    (k.dequantize_mxfp4, _u8(2, 24), _u8(2, 1), {}, "multiples of 32"),
    (k.dequantize_mxfp4, torch.zeros((2, 64), dtype=torch.float8_e4m3fn), _u8(2, 2), {}, "4-bit"),
    (k.dequantize_mxfp8, _u8(2, 32), _u8(2, 2), {}, "values"),
    (k.dequantize_mxfp4, _u8(2, 32), _u8(2, 2), {"dtype": torch.float64}, "out must be"),
    (k.dequantize_mxfp4, _u8(2, 32), _u8(2, 2), {"out": torch.zeros((2, 32))}, "out must be"),
    (k.dequantize_mxfp4, _u8(2, 32), _u8(2, 2), {"out": torch.zeros((2, 64)), "dtype": BF16}, "dtype"),
])
def test_dequantise_refuses(call, values, scales, options, fragment) -> None:
    with pytest.raises(ValueError, match=fragment):
        call(values, scales, **options)


NORMS = [k.add_rms_norm, k.add_rms_norm_int8, k.add_rms_norm_q8_0, k.add_rms_norm_mxfp8, k.add_rms_norm_mxfp4]


@pytest.mark.parametrize("call", NORMS)
@pytest.mark.parametrize("changes,fragment", [
    ({}, "HIP device"),
    ({"x": torch.zeros((2, 64), dtype=torch.float64)}, "x must be|must be float32"),
    ({"x": torch.zeros(64)}, "x must be"),
    ({"x": torch.zeros((2, 128))[:, ::2]}, "dense rows"),
    ({"x": torch.zeros((2, 0)), "weight": torch.zeros(0), "residual": None}, "empty|multiple"),
    ({"weight": torch.zeros(63)}, "weight"),
    ({"weight": torch.zeros(64, dtype=BF16)}, "weight"),
    ({"weight": torch.zeros(128)[::2]}, "weight"),
    ({"residual": torch.zeros((3, 64))}, "x's shape"),
    ({"residual": torch.zeros((2, 64), dtype=torch.int32)}, "residual must be"),
    ({"residual": None, "residual_out": torch.zeros((2, 64))}, "without a residual"),
    ({"residual_out": torch.zeros((2, 64), dtype=BF16)}, "residual's type"),
    ({"residual_out": torch.zeros((2, 32))}, "x's shape"),
    ({"epsilon": -1.0}, "epsilon"),
    ({"epsilon": math.nan}, "epsilon"),
])
def test_norms_refuse(call, changes, fragment) -> None:
    args = {"x": torch.zeros((2, 64)), "weight": torch.zeros(64), "residual": torch.zeros((2, 64)), **changes}
    with pytest.raises(ValueError, match=fragment):
        call(**args)


@pytest.mark.parametrize("call,options,fragment", [
    (k.add_rms_norm, {"out": torch.zeros((2, 32))}, "out must"),
    (k.add_rms_norm, {"out": torch.zeros((2, 64), dtype=torch.int8)}, "out must"),
    (k.add_rms_norm_int8, {"out": torch.zeros((2, 64))}, "out must be int8"),
    (k.add_rms_norm_int8, {"out": torch.zeros((2, 128), dtype=torch.int8)[:, ::2]}, "out must be int8"),
    (k.add_rms_norm_int8, {"scales": torch.zeros(3)}, "scales"),
    (k.add_rms_norm_q8_0, {"out": _u8(2, 2, 33)}, "out must be uint8"),
    (k.add_rms_norm_mxfp8, {"values": _u8(2, 64)}, "values must be"),
    (k.add_rms_norm_mxfp4, {"values": _u8(2, 64)}, "values must be"),
    (k.add_rms_norm_mxfp4, {"scales": _u8(2, 1)}, "scales must be"),
])
def test_norm_outputs_refuse(call, options, fragment) -> None:
    with pytest.raises(ValueError, match=fragment):
        call(torch.zeros((2, 64)), torch.zeros(64), **options)


@pytest.mark.parametrize("call", [k.add_rms_norm_q8_0, k.add_rms_norm_mxfp8, k.add_rms_norm_mxfp4])
def test_block_norms_refuse_odd_rows(call) -> None:
    with pytest.raises(ValueError, match="multiple of 32"):
        call(torch.zeros((2, 48)), torch.zeros(48))


def _gemm(**changes):
    args = {"a_values": torch.zeros((3, 64), dtype=torch.float8_e4m3fn), "a_scales": _u8(3, 2), "w_values": _u8(5, 32), "w_scales": _u8(5, 2)}
    args.update(changes)
    return args


@pytest.mark.parametrize("changes,fragment", [
    ({}, "HIP device"),
    ({"a_values": torch.zeros((3, 64))}, "a values"),
    ({"a_values": _u8(3, 64)}, "scales must be"),
    ({"a_scales": _u8(3, 3)}, "scales must be"),
    ({"w_values": torch.zeros((5, 64), dtype=torch.float8_e4m3fn)}, "4-bit"),
    ({"w_values": _u8(5, 64), "w_scales": _u8(5, 4)}, "differ in K"),
    ({"w_values": _u8(5, 64)[:, ::2]}, "dense rows"),
    ({"bias": torch.zeros(4)}, "bias"),
    ({"bias": torch.zeros(5, dtype=BF16)}, "bias"),
    ({"dtype": torch.int32}, "output must be"),
    ({"out": torch.zeros((3, 4))}, "out must be"),
    ({"out": torch.zeros((3, 5)), "dtype": BF16}, "output's type"),
])
def test_gemm_refuses(changes, fragment) -> None:
    with pytest.raises(ValueError, match=fragment):
        k.mxfp4_gemm(**_gemm(**changes))


@pytest.mark.parametrize("changes,fragment", [
    ({}, "HIP device"),
    ({"x": torch.zeros((3, 32))}, "differ in K"),
    ({"x": torch.zeros((3, 64), dtype=torch.float64)}, "x must be"),
    ({"activations": "int8"}, "block format"),
])
def test_linear_refuses(changes, fragment) -> None:
    args = {"x": torch.zeros((3, 64)), "w_values": _u8(5, 32), "w_scales": _u8(5, 2), **changes}
    with pytest.raises(ValueError, match=fragment):
        k.mxfp4_linear(**args)


@pytest.mark.parametrize("call", [k.mxfp4_gated_gemm, k.mxfp4_gated_linear])
@pytest.mark.parametrize("changes,fragment", [
    ({}, "HIP device"),
    ({"gate": "relu"}, "gate function"),
    ({"up_values": _u8(32, 32), "up_scales": _u8(32, 2)}, "one shape"),
    ({"output": "int8"}, "output must be"),
    ({"output": torch.int8}, "output must be"),
    ({"output": "mxfp8", "out": torch.zeros((3, 64))}, "values, scales"),
    ({"out": (_u8(3, 64), _u8(3, 2)), "output": BF16}, "out must be a tensor"),
    ({"output": "mxfp8", "gate_values": _u8(48, 32), "gate_scales": _u8(48, 2), "up_values": _u8(48, 32), "up_scales": _u8(48, 2)}, "multiple of 32"),
])
def test_gated_refuses(call, changes, fragment) -> None:
    args = {"gate_values": _u8(64, 32), "gate_scales": _u8(64, 2), "up_values": _u8(64, 32), "up_scales": _u8(64, 2), **changes}
    first = (torch.zeros((3, 64)),) if call is k.mxfp4_gated_linear else (torch.zeros((3, 64), dtype=torch.float8_e4m3fn), _u8(3, 2))
    with pytest.raises(ValueError, match=fragment):
        call(*first, **args)


@pytest.mark.parametrize("values,scales", [
    (_u8(4, 32), _u8(3, 2)), (_u8(4, 32), _u8(4, 3)), (_u8(4), _u8(4, 2)), (_u8(4, 0), _u8(4, 0)),
    (torch.zeros((4, 32)), _u8(4, 2)), (_u8(4, 64)[:, ::2], _u8(4, 2)),
])
def test_matrix_refuses(values, scales) -> None:
    with pytest.raises(ValueError, match="microscaling matrix"):
        QuantizedMatrixMxfp4(values, scales)


def test_matrix_shape() -> None:
    assert QuantizedMatrixMxfp4(_u8(4, 32), _u8(4, 2)).shape == (4, 64)


def test_queue_kernels_refuse() -> None:
    a, w = (torch.zeros((3, 64), dtype=torch.float8_e4m3fn), _u8(3, 2)), (_u8(32, 32), _u8(32, 2))
    run = lambda kernel, args, grid: kernel.execute(None, args, LaunchConfig(grid))  # noqa: E731
    with pytest.raises(KernelError, match="expects"):
        run(k.MXFP4_GEMM_KERNEL, (*a, *w), (2, 1, 1))
    with pytest.raises(KernelError, match="grid"):
        run(k.MXFP4_GEMM_KERNEL, (*a, *w, torch.zeros((3, 32)), None), (1, 1, 1))
    with pytest.raises(KernelError, match="expects"):
        run(k.MXFP4_GATED_GEMM_KERNEL, (*a, *w, *w, torch.zeros((3, 32)), None, None), (2, 1, 1))
    with pytest.raises(KernelError, match="grid"):
        run(k.MXFP4_GATED_GEMM_KERNEL, (*a, *w, *w, _u8(3, 16), _u8(3, 1), k.Mxfp4GatedOptions()), (1, 1, 1))
    x, options = torch.zeros((3, 64)), k.AddRmsNormOptions()
    for args, grid, fragment in [
        ((x, torch.zeros(64), None, x), (3, 1, 1), "expects"),
        ((x, torch.zeros(64), None, x, None, None, options), (2, 1, 1), "grid"),
        ((x, torch.zeros(64), x, x, None, None, options), (3, 1, 1), "together"),
        ((x, torch.zeros(64), None, x, torch.zeros(3), None, options), (3, 1, 1), "scales of their own"),
        ((x, torch.zeros(64), None, torch.zeros((3, 64), dtype=torch.int8), None, None, options), (3, 1, 1), "destination"),
        ((x, torch.zeros(64), None, torch.zeros((3, 64), dtype=torch.int16), torch.zeros(3), None, options), (3, 1, 1), "destination"),
    ]:
        with pytest.raises(KernelError, match=fragment):
            run(k.ADD_RMS_NORM_KERNEL, args, grid)


# --------------------------------------------------------------------- C ABI


def _c(name, *args):
    return getattr(_lib.load(), name)(*args)


def _norm_call(x=FAKE, x_stride=256, x_type=0, residual=FAKE + FAR, residual_stride=256, residual_type=0, total=FAKE + 2 * FAR, sum_stride=256,
               weight=FAKE + 3 * FAR, epsilon=1e-6, out=FAKE + 4 * FAR, out_stride=256, scales=FAKE + 5 * FAR, scales_stride=2, kind=0,
               rows=2, columns=64):
    return _c("qxt_add_rms_norm", x, x_stride, x_type, residual, residual_stride, residual_type, total, sum_stride, weight,
              epsilon, out, out_stride, scales, scales_stride, kind, rows, columns, None)


@pytest.mark.parametrize("changes", [
    {"x": None}, {"weight": None}, {"out": None}, {"total": None}, {"x_type": 3}, {"residual_type": 7}, {"kind": 7}, {"columns": 0},
    {"x_stride": 252}, {"x": FAKE + 2}, {"x_stride": 258}, {"out_stride": 128}, {"weight": FAKE + 2}, {"epsilon": -1.0},
    {"epsilon": math.nan}, {"residual_stride": 128}, {"sum_stride": 130}, {"kind": 3, "scales": None}, {"kind": 3, "scales": FAKE + 1},
    {"kind": 4, "columns": 48}, {"kind": 4, "out_stride": 67}, {"kind": 4, "out": FAKE + 1}, {"kind": 5, "columns": 48},
    {"kind": 5, "scales_stride": 1}, {"kind": 6, "scales": None}, {"kind": 6, "out_stride": 31}, {"rows": 2**31},
])
def test_norm_entry_refuses(changes) -> None:
    assert _norm_call(**changes) == _lib.INVALID_ARGUMENT


def test_entries_return_at_once_without_rows() -> None:
    assert _norm_call(rows=0) == _lib.OK
    assert _c("qxt_quantize_mx", None, 0, 0, None, 0, None, 0, 0, 64, 0, None) == _lib.OK


@pytest.mark.parametrize("name", ["qxt_quantize_mx", "qxt_dequantize_mx"])
@pytest.mark.parametrize("changes", [
    {"x": None}, {"values": None}, {"scales": None}, {"type": 3}, {"format": 2}, {"columns": 48}, {"columns": 0}, {"x": FAKE + 1},
    {"x_stride": 100}, {"v_stride": 28}, {"values": FAKE + 2}, {"s_stride": 1}, {"format": 1, "values": FAKE + 4},
    {"rows": 2**31 - 1, "columns": 2**20}, {"values": FAKE}, {"values": FAKE + 700}, {"scales": FAKE + 256}, {"scales": FAKE + FAR + 20},
])
def test_quantise_entries_refuse(name, changes) -> None:
    a = {"x": FAKE, "x_stride": 256, "type": 0, "values": FAKE + FAR, "v_stride": 64, "scales": FAKE + 2 * FAR, "s_stride": 2, "rows": 3,
         "columns": 64, "format": 0, **changes}
    x, values = (a["x"], a["x_stride"], a["type"]), (a["values"], a["v_stride"], a["scales"], a["s_stride"])
    args = (*x, *values) if name == "qxt_quantize_mx" else (*values, *x)
    assert _c(name, *args, a["rows"], a["columns"], a["format"], None) == _lib.INVALID_ARGUMENT


def _matrix(values=FAKE, stride=32, scales=FAKE, scale_stride=2):
    return _lib.MX_MATRIX.pack(values or 0, stride, scales or 0, scale_stride)


def _linear_call(floats=False, gated=False, a=None, w=None, up=None, fmt=0, gate=0, bias=None, y=FAKE + 2 * FAR, ldy=256, scales=FAKE + 3 * FAR,
                 lds=2, kind=0, m=3, n=64, k=64, x=FAKE + FAR, ldx=256, x_type=0, workspace=FAKE + 4 * FAR, size=1 << 30):
    first = (x, ldx, x_type, fmt) if floats else (a or _matrix(), fmt)
    tail = (m, n, k, workspace, size, None)
    if gated:
        return _c("qxt_mxfp4_gated_linear" if floats else "qxt_mxfp4_gated_gemm", *first, w or _matrix(), up or _matrix(), gate, y, ldy, scales, lds,
                  kind, *tail)
    return _c("qxt_mxfp4_linear" if floats else "qxt_mxfp4_gemm", *first, w or _matrix(), bias, y, ldy, kind, *tail)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("floats", [False, True])
@pytest.mark.parametrize("changes", [
    {"fmt": 2}, {"k": 48}, {"k": 0}, {"k": 2**22}, {"kind": 3}, {"y": None}, {"y": FAKE + 2}, {"ldy": 252}, {"ldy": 258}, {"m": 2**31},
    {"w": _matrix(values=None)}, {"w": _matrix(scales=None)}, {"w": _matrix(values=FAKE + 8)}, {"w": _matrix(stride=16)},
    {"w": _matrix(stride=40)}, {"w": _matrix(stride=1 << 23)}, {"w": _matrix(scale_stride=1)},
])
def test_linear_entries_refuse(gated, floats, changes) -> None:
    assert _linear_call(floats, gated, **changes) == _lib.INVALID_ARGUMENT


@pytest.mark.parametrize("changes", [
    {"a": _matrix(values=None)}, {"a": _matrix(stride=24)}, {"a": _matrix(scale_stride=1)}, {"kind": 5}, {"kind": 6}, {"bias": FAKE + 2},
    {"m": 40, "workspace": None, "k": 4096, "a": _matrix(stride=2048, scale_stride=128), "w": _matrix(stride=2048, scale_stride=128)},
    {"m": 40, "size": 16, "k": 4096, "a": _matrix(stride=2048, scale_stride=128), "w": _matrix(stride=2048, scale_stride=128)},
    {"m": 40, "workspace": FAKE + 8, "k": 4096, "a": _matrix(stride=2048, scale_stride=128), "w": _matrix(stride=2048, scale_stride=128)},
])
def test_gemm_entry_refuses(changes) -> None:
    assert _linear_call(**changes) == _lib.INVALID_ARGUMENT


@pytest.mark.parametrize("changes", [
    {"x": None}, {"x": FAKE + 2}, {"ldx": 128}, {"ldx": 258}, {"x_type": 3},
    {"m": 40, "workspace": None}, {"x": FAKE + 4, "workspace": None}, {"x": FAKE + 4, "size": 8},
])
def test_float_entry_refuses(changes) -> None:
    assert _linear_call(True, **changes) == _lib.INVALID_ARGUMENT


@pytest.mark.parametrize("changes", [
    {"gate": 2}, {"up": _matrix(values=None)}, {"up": _matrix(stride=24)}, {"kind": 5, "scales": None}, {"kind": 5, "lds": 1},
    {"kind": 5, "n": 48, "ldy": 64}, {"kind": 6, "y": FAKE + 2}, {"kind": 5, "ldy": 60}, {"kind": 4},
])
def test_gated_entry_refuses(changes) -> None:
    assert _linear_call(gated=True, **changes) == _lib.INVALID_ARGUMENT


@pytest.mark.parametrize("changes", [
    {"out": FAKE + 4, "out_stride": 256}, {"out": FAKE, "out_stride": 512}, {"out": FAKE, "kind": 1}, {"total": FAKE + FAR + 4},
    {"total": FAKE, "sum_stride": 512}, {"total": FAKE + 4 * FAR}, {"out": FAKE + 3 * FAR}, {"kind": 3, "scales": FAKE + 4 * FAR + 60},
    {"kind": 5, "scales": FAKE + FAR + 2}, {"kind": 5, "out": FAKE}, {"kind": 3, "scales": FAKE + 2 * FAR + 4},
])
def test_norm_entry_refuses_shared_memory(changes) -> None:
    assert _norm_call(**changes) == _lib.INVALID_ARGUMENT


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("floats", [False, True])
@pytest.mark.parametrize("changes", [
    {"y": FAKE}, {"y": FAKE + FAR, "w": _matrix(FAKE + FAR)}, {"y": FAKE + 1024, "w": _matrix(scales=FAKE + 1536)},
    {"y": FAKE + 64, "ldy": 512}, {"y": FAKE + FAR + 256, "x": FAKE + FAR, "a": _matrix(FAKE + FAR + 512)},
])
def test_linear_entries_refuse_shared_memory(gated, floats, changes) -> None:
    assert _linear_call(floats, gated, **changes) == _lib.INVALID_ARGUMENT


def test_linear_outputs_refuse_shared_memory() -> None:
    assert _linear_call(bias=FAKE + 2 * FAR) == _lib.INVALID_ARGUMENT
    assert _linear_call(gated=True, up=_matrix(FAKE + 2 * FAR)) == _lib.INVALID_ARGUMENT
    assert _linear_call(gated=True, kind=5, scales=FAKE + 2 * FAR + 32) == _lib.INVALID_ARGUMENT
    assert _linear_call(gated=True, kind=5, scales=FAKE) == _lib.INVALID_ARGUMENT


def test_rows_between_rows_of_one_buffer_are_taken() -> None:
    """Columns of one wide tensor: the injected failure tells that the checks are passed."""
    _lib.set_failure_mask(_lib.FAIL_SUBMISSION)
    try:
        for changes in ({"out": FAKE, "residual": None}, {"total": FAKE + FAR}, {"total": FAKE}, {"out": FAKE}, {"out": FAKE + FAR},
                        {"x_stride": 512, "out": FAKE + 256, "out_stride": 512}, {"x_stride": 768, "out": FAKE + 256, "out_stride": 768, "total": FAKE + 512, "sum_stride": 768},
                        {"kind": 5, "out_stride": 66, "scales": FAKE + 4 * FAR + 64, "scales_stride": 66}, {"kind": 3, "out": FAKE + 8 * FAR}):
            assert _norm_call(**changes) == _lib.SUBMISSION_FAILED, changes
        assert _linear_call(True, ldx=512, y=FAKE + FAR + 256, ldy=512) == _lib.SUBMISSION_FAILED
        assert _linear_call(True, ldx=512, x=FAKE + FAR + 256, y=FAKE + FAR, ldy=512) == _lib.SUBMISSION_FAILED
        assert _linear_call(True, ldx=512, y=FAKE + FAR + 252, ldy=512) == _lib.INVALID_ARGUMENT
    finally:
        _lib.set_failure_mask(_lib.FAIL_NONE)


def test_null_matrices() -> None:
    assert _c("qxt_mxfp4_gemm", None, 0, _matrix(), None, FAKE, 256, 0, 3, 64, 64, None, 0, None) == _lib.INVALID_ARGUMENT
    assert _c("qxt_mxfp4_linear", FAKE, 256, 0, 0, None, None, FAKE, 256, 0, 3, 64, 64, None, 0, None) == _lib.INVALID_ARGUMENT
    assert _c("qxt_mxfp4_gated_gemm", _matrix(), 0, _matrix(), None, 0, FAKE, 256, None, 0, 0, 3, 64, 64, None, 0, None) == _lib.INVALID_ARGUMENT


def test_failure_injection_comes_before_any_launch() -> None:
    _lib.set_failure_mask(_lib.FAIL_SUBMISSION)
    try:
        assert _norm_call() == _lib.SUBMISSION_FAILED
        assert _c("qxt_quantize_mx", FAKE, 256, 0, FAKE + FAR, 64, FAKE + 2 * FAR, 2, 3, 64, 0, None) == _lib.SUBMISSION_FAILED
        for floats in (False, True):
            for gated in (False, True):
                assert _linear_call(floats, gated) == _lib.SUBMISSION_FAILED
                assert _linear_call(floats, gated, m=100) == _lib.SUBMISSION_FAILED
    finally:
        _lib.set_failure_mask(_lib.FAIL_NONE)


def _workspace(m, n, k, weights=1, fmt=1, x_kind=0, kind=1):
    return _c("qxt_mxfp4_linear_workspace", m, n, k, weights, fmt, x_kind, kind)


def test_workspace() -> None:
    # Few rows need none, but for floats that are too many or not aligned for every workgroup to quantise them.
    assert _workspace(1, 4096, 4096) == _workspace(8, 4096, 4096) == 0
    assert _workspace(1, 4096, 4096, x_kind=2 + _lib.ROWS_ALIGNED) == 0
    assert _workspace(1, 4096, 4096, x_kind=2) == 4096 + 128
    assert _workspace(8, 4096, 4096, x_kind=1 + _lib.ROWS_ALIGNED) == 8 * (4096 + 128)
    assert _workspace(4, 4096, 14336) == _workspace(8, 4096, 14336) == 0 and _workspace(4, 4097, 14336) > 0 and _workspace(4, 1024, 14336) > 0
    assert _workspace(8, 4096, 14336, weights=2) > 0 and _workspace(16, 4096, 14336) > 0
    # Many rows: quantised rows, scales in words, and the sums of the parts of K.
    plain = _workspace(4096, 4096, 4096)
    assert plain == 4096 * 128 * 2
    assert _workspace(4096, 4096, 4096, x_kind=1) == plain + 4096 * 4096
    assert _workspace(4096, 4096, 4096, weights=2) == plain + 4096 * 128
    few = _workspace(32, 256, 8192)
    parts = (few - 32 * 256 - 256 * 256) / (32 * 256 * 4)
    assert parts == int(parts) and 2 <= parts <= 16
    assert _workspace(32, 0, 8192) == _workspace(0, 32, 8192) == _workspace(3, 3, 33) == _workspace(3, 3, 32, weights=3) == _workspace(3, 3, 32, x_kind=4) == 0


# --------------------------------------------------------------- definitions


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_reference_values_survive_their_own_quantisation(fmt) -> None:
    grid = reference.FP4 if fmt == "mxfp4" else reference.FP8
    x = torch.cat([grid, -grid])
    x = torch.cat([x, torch.zeros(-len(x) % 32, dtype=torch.float64)]).view(-1, 32)
    x[:, 0] = grid[-1]
    for shift in (-100, -3, 0, 40):
        scaled = x * 2.0**shift
        codes, scales = reference.quantize(scaled, fmt)
        assert torch.equal(reference.values(codes, scales, fmt), scaled)
        assert torch.equal(reference.read(*reference.stored(scaled, fmt), fmt), scaled)


def test_reference_rounds_ties_to_even_and_cuts() -> None:
    x = torch.zeros((1, 32), dtype=torch.float64)
    x[0, :8] = torch.tensor([6.0, 0.25, 0.75, 1.25, 2.5, 5.0, 7.9, -3.5])
    codes, scales = reference.quantize(x, "mxfp4")
    assert int(scales[0, 0]) == 127
    assert reference.values(codes, scales, "mxfp4")[0, :8].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 4.0, 6.0, -4.0]


def test_reference_agrees_with_torch_eight_bit_rounding() -> None:
    x = torch.randn((64, 32), generator=torch.Generator().manual_seed(1)) * 100
    codes, scales = reference.quantize(x, "mxfp8")
    scaled = (x.double() / 2.0 ** (scales.double() - 127)).clamp(-448, 448)
    assert torch.equal(codes.view(torch.float8_e4m3fn).double(), scaled.float().to(torch.float8_e4m3fn).double())


def test_large_bytes_of_a_word() -> None:
    """The mask that splits 8-bit elements: 0xFF in each byte whose bit 6 is set."""
    for word in (0, 0x40, 0x7F80C03F, 0xFFFFFFFF, 0x41424344, 0x3F3F3F3F):
        bit = (word >> 6) & 0x01010101
        mask = ((bit << 8) - bit) & 0xFFFFFFFF
        assert [(mask >> 8 * i) & 0xFF for i in range(4)] == [0xFF if (word >> (8 * i)) & 0x40 else 0 for i in range(4)]
    # Within either part no product with a 4-bit element has a bit more than 13 below another product's power of two.
    values = reference.FP8[1:]
    for part in (values[values >= 2], values[values < 2]):
        top = math.floor(math.log2(float(part.max()))) + 2  # times 2^2, the largest power of a 4-bit element
        last = min(max(math.floor(math.log2(float(v))), -6) - 3 for v in part) - 1  # times 0.5
        assert top - last <= 13


def test_ctypes_struct_is_the_headers() -> None:
    assert _lib.MX_MATRIX.size == ctypes.sizeof(ctypes.c_void_p) * 4
