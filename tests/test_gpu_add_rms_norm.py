"""The residual norm against its 64-bit definition: sums and codes bit for bit, floats within their roundings.

y errs by the roundings of the factor and of two products (3 units of 2^-24), and by half a step of its own type.
"""

from __future__ import annotations

import math

import pytest
import torch

import mx_reference as reference
from qpu_xla_amd import Queue
from qpu_xla_amd.kernels import (
    ADD_RMS_NORM_KERNEL,
    AddRmsNormOptions,
    add_rms_norm,
    add_rms_norm_grid,
    add_rms_norm_int8,
    add_rms_norm_mxfp4,
    add_rms_norm_mxfp8,
    add_rms_norm_q8_0,
    quantize_mxfp8,
    quantize_q8_0,
    quantize_rows_int8,
)

pytestmark = pytest.mark.gpu

EPSILON = 1e-5
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _inputs(rows, columns, x_type, residual_type, seed=0):
    gen = torch.Generator().manual_seed(seed + columns)
    x = torch.randn((rows, columns), generator=gen).to(x_type)
    weight = 1 + 0.3 * torch.randn((columns,), generator=gen)
    residual = None if residual_type is None else (torch.randn((rows, columns), generator=gen) * 3).to(residual_type)
    return x, weight, residual


def _cuda(*tensors):
    return [None if t is None else t.cuda() for t in tensors]


def _check_floats(got, want):
    reference.check(got, want, reference.rounded(want, 3 * 2.0**-24 * want.abs(), got.dtype))


def _check_sum(got, want):
    assert (got is None) == (want is None)
    if want is not None:
        assert got.dtype is want.dtype and torch.equal(got.cpu(), want)


# Lone rows, widths of one to several pieces a thread, the wide workgroups, rows past the held ones, no multiple of anything.
WIDTHS = [(1, 2048), (3, 32), (2, 8), (5, 4096), (600, 4096), (3, 11008), (2, 16384), (2, 24576), (700, 20480), (2, 32768), (2, 40960),
          (4, 1), (3, 33), (2, 4100), (5, 1000), (513, 2056)]


@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                   (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, None),
                                   (torch.float32, None)])
@pytest.mark.parametrize("size", WIDTHS)
def test_floats(size, types) -> None:
    x, weight, residual = _inputs(*size, *types)
    want, _, total = reference.norm(x, weight, residual, EPSILON)
    got, added = add_rms_norm(*_cuda(x, weight, residual), epsilon=EPSILON)
    assert got.dtype is x.dtype
    _check_floats(got, want)
    _check_sum(added, total)


@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, None)])
@pytest.mark.parametrize("size", [(1, 2048), (3, 32), (5, 4096), (600, 4096), (3, 11008), (2, 24576), (2, 40960), (2, 96)])
def test_quantised_rows(size, types) -> None:
    x, weight, residual = _inputs(*size, *types)
    _, y, total = reference.norm(x, weight, residual, EPSILON)
    args = _cuda(x, weight, residual)
    values, scales, added = add_rms_norm_int8(*args, epsilon=EPSILON)
    want_values, want_scales = reference.int8_rows(y)
    assert torch.equal(values.cpu(), want_values) and torch.equal(scales.cpu(), want_scales)
    _check_sum(added, total)
    blocks, added = add_rms_norm_q8_0(*args, epsilon=EPSILON)
    assert torch.equal(blocks.cpu(), reference.q8_0(y))
    _check_sum(added, total)
    for fmt, call in (("mxfp8", add_rms_norm_mxfp8), ("mxfp4", add_rms_norm_mxfp4)):
        values, scales, added = call(*args, epsilon=EPSILON)
        codes, want_scales = reference.quantize(y, fmt)
        assert torch.equal(scales.cpu(), want_scales) and torch.equal(reference.unpack(values, fmt), codes)
        _check_sum(added, total)


def test_codes_are_those_of_the_quantisers() -> None:
    x, weight, residual = _cuda(*_inputs(37, 4096, torch.float32, torch.float32))
    y, _ = add_rms_norm(x, weight, residual, epsilon=EPSILON)
    values, scales, _ = add_rms_norm_int8(x, weight, residual, epsilon=EPSILON)
    want_values, want_scales = quantize_rows_int8(y)
    assert torch.equal(values, want_values) and torch.equal(scales, want_scales)
    assert torch.equal(add_rms_norm_q8_0(x, weight, residual, epsilon=EPSILON)[0], quantize_q8_0(y))
    values, scales, _ = add_rms_norm_mxfp8(x, weight, residual, epsilon=EPSILON)
    want_values, want_scales = quantize_mxfp8(y)
    assert torch.equal(values.view(torch.uint8), want_values.view(torch.uint8)) and torch.equal(scales, want_scales)


@pytest.mark.parametrize("offset", [0, 1, 2, 8])
def test_strided_and_unaligned_rows(offset) -> None:
    x, weight, residual = _inputs(11, 320, torch.bfloat16, torch.bfloat16)
    place = lambda t: torch.zeros((11, 360), dtype=t.dtype, device="cuda")[:, offset:offset + 320].copy_(t)  # noqa: E731
    stores = [torch.full((11, 360), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    out, total_out = (s[:, offset:offset + 320] for s in stores)
    want, y, total = reference.norm(x, weight, residual, EPSILON)
    xs, rs, ws = place(x), place(residual), weight.cuda()
    add_rms_norm(xs, ws, rs, epsilon=EPSILON, out=out, residual_out=total_out)
    _check_floats(out, want)
    _check_sum(total_out, total)
    for store in stores:
        assert bool((store[:, :offset] == 7).all()) and bool((store[:, offset + 320:] == 7).all())
    values, scales, _ = add_rms_norm_mxfp4(xs, ws, rs, epsilon=EPSILON)
    codes, want_scales = reference.quantize(y, "mxfp4")
    assert torch.equal(scales.cpu(), want_scales) and torch.equal(reference.unpack(values, "mxfp4"), codes)
    values, scales, _ = add_rms_norm_mxfp8(xs, ws, rs, epsilon=EPSILON)
    codes, want_scales = reference.quantize(y, "mxfp8")
    assert torch.equal(scales.cpu(), want_scales) and torch.equal(reference.unpack(values, "mxfp8"), codes)
    values, scales, _ = add_rms_norm_int8(xs, ws, rs, epsilon=EPSILON)
    want_values, want_scales = reference.int8_rows(y)
    assert torch.equal(values.cpu(), want_values) and torch.equal(scales.cpu(), want_scales)
    assert torch.equal(add_rms_norm_q8_0(xs, ws, rs, epsilon=EPSILON)[0].cpu(), reference.q8_0(y))


@pytest.mark.parametrize("width", [4096, 1001])
def test_in_place(width) -> None:
    x, weight, residual = _inputs(6, width, torch.bfloat16, torch.bfloat16)
    want, _, total = reference.norm(x, weight, residual, EPSILON)
    xs, ws, rs = _cuda(x, weight, residual)
    out, added = add_rms_norm(xs, ws, rs, epsilon=EPSILON, out=xs, residual_out=rs)
    assert out is xs and added is rs
    _check_floats(xs, want)
    _check_sum(rs, total)
    want, _, _ = reference.norm(x, weight, None, EPSILON)
    xs = x.cuda()
    add_rms_norm(xs, ws, epsilon=EPSILON, out=xs)
    _check_floats(xs, want)


@pytest.mark.parametrize("width", [2048, 96, 1001])
def test_rows_of_zeros_large_values_and_no_numbers(width) -> None:
    x, weight, residual = _inputs(6, width, torch.float32, torch.float32)
    x[0], residual[0] = 0.0, 0.0
    x[1] *= 1e30  # squares past fp32
    x[2] *= 1e-30
    residual[2] *= 1e-30
    x[3, width // 2] = math.nan
    residual[4, 7] = math.inf
    want, y, total = reference.norm(x, weight, residual, EPSILON)
    args = _cuda(x, weight, residual)
    got, added = add_rms_norm(*args, epsilon=EPSILON)
    _check_floats(got, want)
    assert torch.equal(added.cpu().nan_to_num(0.5), total.nan_to_num(0.5))
    if width % 32 == 0:
        values, scales, _ = add_rms_norm_mxfp8(*args, epsilon=EPSILON)
        codes, want_scales = reference.quantize(y, "mxfp8")
        assert torch.equal(scales.cpu(), want_scales) and torch.equal(reference.unpack(values, "mxfp8"), codes)
        assert bool((scales[3] == 255).all())


def test_no_rows() -> None:
    empty, weight = torch.zeros((0, 64), device="cuda"), torch.ones(64, device="cuda")
    y, total = add_rms_norm(empty, weight, empty)
    assert y.shape == total.shape == (0, 64)
    values, scales, _ = add_rms_norm_int8(empty, weight)
    assert values.shape == (0, 64) and scales.shape == (0,)
    assert add_rms_norm_q8_0(empty, weight)[0].shape == (0, 2, 34)
    assert add_rms_norm_mxfp4(empty, weight)[1].shape == (0, 2)


def test_queue_kernel_and_captured() -> None:
    x, weight, residual = _cuda(*_inputs(12, 512, torch.float32, torch.float32))
    want = add_rms_norm_mxfp8(x, weight, residual, epsilon=EPSILON)
    values, scales, total = torch.empty((12, 512), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((12, 16), dtype=torch.uint8, device="cuda"), torch.empty_like(x)
    int8, int8_scales, blocks = torch.empty((12, 512), dtype=torch.int8, device="cuda"), torch.empty(12, device="cuda"), torch.empty((12, 16, 34), dtype=torch.uint8, device="cuda")
    with Queue() as queue:
        grid, options = add_rms_norm_grid(x), AddRmsNormOptions(EPSILON)
        queue.submit(ADD_RMS_NORM_KERNEL, (x, weight, residual, values, scales, total, options), grid=grid).wait()
        queue.submit(ADD_RMS_NORM_KERNEL, (x, weight, residual, int8, int8_scales, total, options), grid=grid).wait()
        queue.submit(ADD_RMS_NORM_KERNEL, (x, weight, None, blocks, None, None, options), grid=grid).wait()
    assert torch.equal(values.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales, want[1]) and torch.equal(total, want[2])
    assert torch.equal(int8, add_rms_norm_int8(x, weight, residual, epsilon=EPSILON)[0])
    assert torch.equal(blocks, add_rms_norm_q8_0(x, weight, epsilon=EPSILON)[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = add_rms_norm(x, weight, residual, epsilon=EPSILON)
    for step in range(3):
        x.mul_(-1.5)
        graph.replay()
        torch.cuda.synchronize()
        eager = add_rms_norm(x, weight, residual, epsilon=EPSILON)
        assert torch.equal(captured[0], eager[0]) and torch.equal(captured[1], eager[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("columns", [520, 1096, 4104, 8200, 9000])
def test_quantised_rows_with_the_sum_in_place(columns, dtype) -> None:
    """Widths that leave threads past the row: they re-read a place whose sum may be stored by then."""
    x, weight, residual = _inputs(2048, columns, dtype, dtype)
    xs, ws, rs = _cuda(x, weight, residual)
    want = add_rms_norm_int8(xs, ws, rs, epsilon=EPSILON)
    got = add_rms_norm_int8(xs, ws, rs, epsilon=EPSILON, residual_out=rs)
    assert got[2] is rs
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    _, rounded, total = reference.norm(x[:64], weight, residual[:64], EPSILON)
    codes, scale = reference.int8_rows(rounded)
    assert torch.equal(want[0][:64].cpu(), codes) and torch.equal(want[1][:64].cpu(), scale) and torch.equal(want[2][:64].cpu(), total)
