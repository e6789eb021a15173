"""Microscaling blocks: codes and scales are those of the 64-bit definition, bit for bit, and read back exactly."""

from __future__ import annotations

import math

import pytest
import torch

import mx_reference as reference
from qpu_xla_amd import Queue
from qpu_xla_amd.kernels import dequantize_mxfp4, dequantize_mxfp8, quantize_mxfp4, quantize_mxfp8

pytestmark = pytest.mark.gpu

QUANTIZE = {"mxfp4": quantize_mxfp4, "mxfp8": quantize_mxfp8}
DEQUANTIZE = {"mxfp4": dequantize_mxfp4, "mxfp8": dequantize_mxfp8}
FORMATS = ("mxfp4", "mxfp8")
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _rows(shape, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen, dtype=torch.float32)
    spread = torch.randint(-12, 12, (shape[0], shape[1] // 32, 1), generator=gen)
    return (x.unflatten(1, (-1, 32)) * 2.0**spread).flatten(1).to(dtype)


def _check(values, scales, x, fmt):
    codes, want = reference.quantize(x, fmt)
    assert torch.equal(scales.cpu(), want)
    assert torch.equal(reference.unpack(values, fmt), codes)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 32), (3, 64), (5, 96), (1, 4096), (33, 2048), (7, 11008)])
def test_codes_and_values(shape, dtype, fmt) -> None:
    x = _rows(shape, dtype, 1 + shape[0])
    values, scales = QUANTIZE[fmt](x.cuda())
    _check(values, scales, x, fmt)
    want = reference.read(values, scales, fmt)
    for out in DTYPES:
        got = DEQUANTIZE[fmt](values, scales, dtype=out)
        assert got.dtype is out and torch.equal(got.cpu(), want.float().to(out))  # float32 holds every value


@pytest.mark.parametrize("fmt", FORMATS)
def test_borders_ties_and_ends(fmt) -> None:
    grid = reference.FP4 if fmt == "mxfp4" else reference.FP8
    middle = ((grid[1:] + grid[:-1]) / 2).float()
    around = torch.cat([middle, torch.nextafter(middle, torch.tensor(math.inf)), torch.nextafter(middle, torch.tensor(0.0)), grid.float()])
    top = float(grid[-1])
    around = torch.cat([around, -around, torch.tensor([top * 1.05, top * 1.14, 0.0, -0.0])])
    padded = torch.zeros(-(-around.numel() // 31) * 31)
    padded[: around.numel()] = around
    blocks = torch.cat([torch.full((padded.numel() // 31, 1), top), padded.view(-1, 31)], 1)  # the first element fixes the scale
    for shift in (-140, -126, -125, -100, -20, 0, 20, 100, 118):
        x = (blocks.double() * 2.0**shift).float().flatten()[None]
        values, scales = QUANTIZE[fmt](x.cuda())
        _check(values, scales, x, fmt)
        assert torch.equal(DEQUANTIZE[fmt](values, scales).cpu().double(), reference.read(values, scales, fmt))


@pytest.mark.parametrize("fmt", FORMATS)
def test_every_power_of_two(fmt) -> None:
    exponents = torch.arange(-149, 128, dtype=torch.float64)
    x = torch.zeros((len(exponents), 32))
    x[:, 5] = (2.0**exponents).float()
    x[:, 6] = -(2.0**exponents * 1.75).float()
    values, scales = QUANTIZE[fmt](x.cuda())
    _check(values, scales, x, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_that_hold_no_number_become_nan(fmt, dtype) -> None:
    x = torch.randn((4, 128), generator=torch.Generator().manual_seed(2)).to(dtype)
    x[0, 3], x[1, 40], x[2, 127], x[3, 64:96] = math.nan, math.inf, -math.inf, 0.0
    values, scales = QUANTIZE[fmt](x.cuda())
    _check(values, scales, x, fmt)
    bad = torch.zeros((4, 4), dtype=torch.bool)
    bad[0, 0] = bad[1, 1] = bad[2, 3] = True
    assert torch.equal(torch.isnan(DEQUANTIZE[fmt](values, scales).cpu()), bad.repeat_interleave(32, 1))
    assert int(scales[3, 2]) == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("offset", [0, 1, 2, 4])
def test_strided_rows_in_and_out(fmt, offset) -> None:
    x = _rows((9, 256), torch.bfloat16, 3)
    wide = torch.zeros((9, 300), dtype=torch.bfloat16)
    wide[:, offset:offset + 256] = x
    size = 256 if fmt == "mxfp8" else 128
    store = torch.full((9, size + 16), 0x55, dtype=torch.uint8).cuda()
    scale_store = torch.full((9, 11), 0x66, dtype=torch.uint8).cuda()
    values = store[:, 8:8 + size]
    values = values.view(torch.float8_e4m3fn) if fmt == "mxfp8" else values
    QUANTIZE[fmt](wide.cuda()[:, offset:offset + 256], values, scale_store[:, 1:9])
    _check(values, scale_store[:, 1:9], x, fmt)
    assert bool((store[:, :8] == 0x55).all()) and bool((store[:, 8 + size:] == 0x55).all())  # nothing beside the rows
    assert bool((scale_store[:, 0] == 0x66).all()) and bool((scale_store[:, 9:] == 0x66).all())
    out = torch.zeros((9, 300), dtype=torch.bfloat16, device="cuda")
    DEQUANTIZE[fmt](values, scale_store[:, 1:9], out[:, offset:offset + 256])
    assert torch.equal(out[:, offset:offset + 256].cpu().double(), reference.read(values, scale_store[:, 1:9], fmt).bfloat16().double())
    assert bool((out[:, :offset] == 0).all()) and bool((out[:, offset + 256:] == 0).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_no_rows_and_torch_types(fmt) -> None:
    values, scales = QUANTIZE[fmt](torch.zeros((0, 64), device="cuda"))
    assert scales.shape == (0, 2) and DEQUANTIZE[fmt](values, scales).shape == (0, 64)
    x = _rows((3, 64), torch.float32, 4)
    values, scales = QUANTIZE[fmt](x.cuda())
    stored = values if fmt == "mxfp8" else values.view(torch.float4_e2m1fn_x2)
    got = DEQUANTIZE[fmt](stored, scales.view(torch.float8_e8m0fnu))
    assert torch.equal(got.cpu().double(), reference.read(values, scales, fmt))


def test_on_a_queue_and_captured() -> None:
    x = _rows((64, 512), torch.float32, 5).cuda()
    with Queue() as queue:
        values, scales = quantize_mxfp4(x, stream=queue)
        queue.stream.synchronize()
    _check(values, scales, x, "mxfp4")
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    source, out = x.clone(), torch.empty_like(x)
    with torch.cuda.stream(side):
        dequantize_mxfp8(*quantize_mxfp8(source), out)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        dequantize_mxfp8(*quantize_mxfp8(source), out)
    for seed in range(4):
        source.copy_(_rows((64, 512), torch.float32, 10 + seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, dequantize_mxfp8(*quantize_mxfp8(source)))
