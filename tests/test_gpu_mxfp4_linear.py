"""Linears over 4-bit microscaling weights and the gated product, against the 64-bit definition (mx_reference has the bounds)."""

from __future__ import annotations

import pytest
import torch

import mx_reference as reference
from qpu_xla_amd import Queue
from qpu_xla_amd.kernels import (
    MXFP4_GATED_GEMM_KERNEL,
    MXFP4_GEMM_KERNEL,
    Mxfp4GatedOptions,
    mxfp4_gated_gemm,
    mxfp4_gated_linear,
    mxfp4_gemm,
    mxfp4_gemm_grid,
    mxfp4_linear,
    quantize_mxfp4,
    quantize_mxfp8,
)

pytestmark = pytest.mark.gpu

FORMATS = ("mxfp8", "mxfp4")
QUANTIZE = {"mxfp4": quantize_mxfp4, "mxfp8": quantize_mxfp8}
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _operands(m, n, k, fmt, seed=0, weights=1, spread=True):
    gen = torch.Generator().manual_seed(seed + m + 7 * n + 13 * k)
    a = torch.randn((m, k), generator=gen)
    if spread:  # blocks of very different sizes, and loud channels
        a *= torch.where(torch.rand((k,), generator=gen) < 0.02, 20.0, 1.0)
        a = (a.unflatten(1, (-1, 32)) * 2.0 ** torch.randint(-3, 3, (m, k // 32, 1), generator=gen)).flatten(1)
    return (a, *(torch.randn((n, k), generator=gen) * k**-0.5 for _ in range(weights)))


def _stored(x, fmt):
    values, scales = reference.stored(x, fmt)
    return values.cuda(), scales.cuda()


# One token, tiles with one row or column too many, K of one block, blocks that do not fill an instruction, long K, many rows.
SHAPES = [(1, 32, 32), (1, 5632, 2048), (1, 17, 96), (2, 64, 128), (3, 100, 160), (8, 257, 512), (15, 48, 1056), (16, 96, 2048),
          (17, 33, 544), (31, 130, 4096), (33, 200, 352), (64, 512, 1024), (77, 300, 3008), (128, 256, 2048), (130, 129, 640),
          (200, 1030, 96), (257, 260, 1152), (300, 520, 4096), (515, 777, 256),
          # K in many parts (whole groups of 512 elements or not), every tile.
          (20, 96, 9248), (70, 200, 8192), (150, 130, 6176), (260, 300, 12288), (1030, 2060, 544), (2050, 2310, 256), (700, 1500, 1024)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", SHAPES)
def test_gemm_against_the_definition(shape, fmt) -> None:
    m, n, k = shape
    a, w = _operands(m, n, k, fmt)
    a_stored, w_stored = _stored(a, fmt), _stored(w, "mxfp4")
    want, size = reference.product(reference.read(*a_stored, fmt), reference.read(*w_stored, "mxfp4"))
    bias = torch.randn((n,), generator=torch.Generator().manual_seed(1))
    for dtype in DTYPES:
        error = reference.sum_error(size, k, fmt, dtype is torch.float32)
        got = mxfp4_gemm(*a_stored, *w_stored, dtype=dtype)
        assert got.dtype is dtype
        reference.check(got, want, reference.rounded(want, error, dtype))
        with_bias = want + bias.double()
        got = mxfp4_gemm(*a_stored, *w_stored, bias.cuda(), dtype=dtype)
        reference.check(got, with_bias, reference.rounded(with_bias, error + 2.0**-24 * (with_bias.abs() + error), dtype))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 96, 2048), (4, 40, 352), (16, 300, 1024), (33, 64, 4096), (150, 300, 512)])
def test_linear_quantises_as_the_quantiser_does(shape, dtype, fmt) -> None:
    m, n, k = shape
    a, w = _operands(m, n, k, fmt)
    x = a.to(dtype).cuda()
    w_stored = _stored(w, "mxfp4")
    got = mxfp4_linear(x, *w_stored, activations=fmt)
    assert got.dtype is dtype
    assert torch.equal(got, mxfp4_gemm(*QUANTIZE[fmt](x), *w_stored, dtype=dtype))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("gate", ["silu", "gelu"])
@pytest.mark.parametrize("shape", [(1, 64, 2048), (1, 5632, 512), (5, 96, 160), (16, 160, 1024), (20, 33, 96), (40, 96, 4096), (130, 352, 640),
                                   (260, 288, 1024), (24, 64, 8224), (100, 160, 6144), (1100, 1312, 256), (600, 1440, 512)])
def test_gated_against_the_definition(shape, gate, fmt) -> None:
    m, n, k = shape
    a, g, u = _operands(m, n, k, fmt, weights=2)
    a_stored, g_stored, u_stored = _stored(a, fmt), _stored(g, "mxfp4"), _stored(u, "mxfp4")
    operands = [reference.read(*a_stored, fmt), reference.read(*g_stored, "mxfp4"), reference.read(*u_stored, "mxfp4")]
    for dtype in DTYPES:
        want, error = reference.gated(*operands, gate, fmt, dtype is torch.float32)
        got = mxfp4_gated_gemm(*a_stored, *g_stored, *u_stored, gate=gate, output=dtype)
        assert got.dtype is dtype
        reference.check(got, want, reference.rounded(want, error, dtype))
    if n % 32 == 0:
        want, error = reference.gated(*operands, gate, fmt, False)
        for kind in FORMATS:
            values, scales = mxfp4_gated_gemm(*a_stored, *g_stored, *u_stored, gate=gate, output=kind)
            reference.check_blocks(values, scales, kind, want, error)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", [(1, 64, 2048), (7, 96, 352), (40, 64, 512)])
def test_gated_linear_quantises_as_the_quantiser_does(shape, fmt) -> None:
    m, n, k = shape
    a, g, u = _operands(m, n, k, fmt, weights=2)
    x = a.bfloat16().cuda()
    weights = (*_stored(g, "mxfp4"), *_stored(u, "mxfp4"))
    got = mxfp4_gated_linear(x, *weights, activations=fmt)
    assert got.dtype is torch.bfloat16
    assert torch.equal(got, mxfp4_gated_gemm(*QUANTIZE[fmt](x), *weights, output=torch.bfloat16))
    values, scales = mxfp4_gated_linear(x, *weights, activations=fmt, output="mxfp8")
    want = mxfp4_gated_gemm(*QUANTIZE[fmt](x), *weights, output="mxfp8")
    assert torch.equal(values.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales, want[1])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 16, 40, 200])
def test_strided_operands_and_neighbours_left_alone(m, fmt) -> None:
    n, k = 100, 352
    a, w = _operands(m, n, k, fmt)
    a_stored, w_stored = _stored(a, fmt), _stored(w, "mxfp4")
    want = mxfp4_gemm(*a_stored, *w_stored, dtype=torch.bfloat16)

    def spread(t, pad, at, fill):
        raw = t.view(torch.uint8)
        wide = torch.full((raw.shape[0], raw.shape[1] + pad), fill, dtype=torch.uint8, device="cuda")
        wide[:, at:at + raw.shape[1]] = raw
        return wide[:, at:at + raw.shape[1]].view(t.dtype)

    # What lies between the rows is NaN bytes: none of it may reach a result.
    strided = (spread(a_stored[0], 48, 16, 0x7F), spread(a_stored[1], 5, 1, 0xFF), spread(w_stored[0], 32, 32, 0x77), spread(w_stored[1], 3, 2, 0xFF))
    for pad, at in ((28, 0), (29, 1), (36, 4)):
        store = torch.full((m, n + pad), 5.0, dtype=torch.bfloat16, device="cuda")
        got = mxfp4_gemm(*strided, out=store[:, at:at + n])
        assert torch.equal(got, want)
        assert bool((store[:, :at] == 5).all()) and bool((store[:, at + n:] == 5).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [3, 70])
def test_nan_blocks_reach_their_rows_and_columns_only(m, fmt) -> None:
    n, k = 70, 256
    a, w = _operands(m, n, k, fmt)
    a_stored, w_stored = _stored(a, fmt), _stored(w, "mxfp4")
    clean = mxfp4_gemm(*a_stored, *w_stored)
    a_stored[1][1, 3] = 255
    w_stored[1][66, 0] = 255
    got = mxfp4_gemm(*a_stored, *w_stored)
    bad = torch.zeros((m, n), dtype=torch.bool, device="cuda")
    bad[1], bad[:, 66] = True, True
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[~bad], clean[~bad])


def test_no_rows_and_no_columns() -> None:
    a = quantize_mxfp8(torch.zeros((0, 64), device="cuda"))
    w = quantize_mxfp4(torch.ones((48, 64), device="cuda"))
    assert mxfp4_gemm(*a, *w).shape == (0, 48)
    values, scales = mxfp4_gated_linear(torch.zeros((0, 64), device="cuda"), *(t[:32] for t in w), *(t[:32] for t in w), output="mxfp8")
    assert values.shape == (0, 32) and scales.shape == (0, 1)


def test_queue_kernels() -> None:
    m, n, k = 5, 64, 256
    a, g, u = _operands(m, n, k, "mxfp8", weights=2)
    a, g, u = _stored(a, "mxfp8"), _stored(g, "mxfp4"), _stored(u, "mxfp4")
    bias = torch.randn(n, device="cuda")
    y, h = torch.empty((m, n), device="cuda"), torch.empty((m, n // 2), dtype=torch.uint8, device="cuda")
    h_scales, floats = torch.empty((m, n // 32), dtype=torch.uint8, device="cuda"), torch.empty((m, n), dtype=torch.float16, device="cuda")
    with Queue() as queue:
        queue.submit(MXFP4_GEMM_KERNEL, (*a, *g, y, bias), grid=mxfp4_gemm_grid(m, n)).wait()
        queue.submit(MXFP4_GATED_GEMM_KERNEL, (*a, *g, *u, h, h_scales, Mxfp4GatedOptions()), grid=mxfp4_gemm_grid(m, n)).wait()
        queue.submit(MXFP4_GATED_GEMM_KERNEL, (*a, *g, *u, floats, None, Mxfp4GatedOptions("gelu")), grid=mxfp4_gemm_grid(m, n)).wait()
    assert torch.equal(y, mxfp4_gemm(*a, *g, bias))
    want = mxfp4_gated_gemm(*a, *g, *u, output="mxfp4")
    assert torch.equal(h, want[0]) and torch.equal(h_scales, want[1])
    assert torch.equal(floats, mxfp4_gated_gemm(*a, *g, *u, gate="gelu", output=torch.float16))


@pytest.mark.parametrize("m", [1, 20, 200])
def test_repeats_give_the_same_bits(m) -> None:
    a, w = _operands(m, 512, 2048, "mxfp8")
    x, w_stored = a.bfloat16().cuda(), _stored(w, "mxfp4")
    first = mxfp4_linear(x, *w_stored, dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(first, mxfp4_linear(x, *w_stored, dtype=torch.float32))
