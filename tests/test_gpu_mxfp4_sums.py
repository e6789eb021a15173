"""Linears and gated products over 8-bit activations keep every bit of their products, whatever the rows and the output.

Of each eight neighbouring products two are large and cancel, and six are more than 13 bits below them.  All are multiples of
2^-7, and what one matrix instruction adds up (16 groups of eight, at most 16 * 2 * 2688 < 2^17 in magnitude) and the sums of
the small ones (at most K * 0.75 * 0.75 < 2^10) are multiples of it below 2^24 times as large: exact in float32 in any order.  So results are those of
the definition rounded once, and codes those of the definition, bit for bit.
"""

from __future__ import annotations

import pytest
import torch

import mx_reference as reference
from qpu_xla_amd.kernels import mxfp4_gated_gemm, mxfp4_gemm

pytestmark = pytest.mark.gpu

# Few rows, and rows for tiles of every size.
SHAPES = [(3, 96, 288), (17, 96, 288), (40, 224, 1120), (130, 160, 1056), (333, 4128, 288), (2050, 4128, 160)]


def _rows(gen, rows, k):
    """Activations: 448, 448, 2 and five multiples of 2^-6 up to 2^-3 of either sign, in each eight."""
    x = torch.randint(-8, 9, (rows, k // 8, 8), generator=gen).double() * 2.0**-6
    x[..., 0] = x[..., 1] = 448.0
    x[..., 2] = 2.0
    return x.flatten(1)


def _up(gen, rows, k):
    """6 and -6 in either order, then any 4-bit values."""
    w = reference.FP4[torch.randint(0, 8, (rows, k // 8, 8), generator=gen)] * (1 - 2 * torch.randint(0, 2, (rows, k // 8, 8), generator=gen))
    w[..., 0] = 6.0 - 12.0 * torch.randint(0, 2, (rows, k // 8), generator=gen)
    w[..., 1] = -w[..., 0]
    return w.flatten(1)


def _gate(rows, k):
    """6 and -6, then 4 times the activations' 2: 8 for each eight, K in all, of which both gate functions are K itself."""
    return torch.tensor([6.0, -6.0, 4.0, 0.0, 0.0, 0.0, 0.0, 0.0], dtype=torch.float64).repeat(rows, k // 8)


def _stored(x, fmt, powers=None):
    """Blocks of elements as they are, under scales of the rows' powers of two."""
    values = reference.pack(_codes(x, fmt), fmt).cuda()
    scales = torch.full((x.shape[0], x.shape[1] // 32), 127, dtype=torch.uint8)
    if powers is not None:
        scales += powers.to(torch.uint8)[:, None]
    return values, scales.cuda()


def _codes(x, fmt):
    grid = reference.FP4 if fmt == "mxfp4" else reference.FP8
    code = torch.searchsorted(grid, x.abs())
    assert torch.equal(grid[code], x.abs())
    return (code + torch.signbit(x) * (8 if fmt == "mxfp4" else 128)).to(torch.uint8)


@pytest.mark.parametrize("shape", SHAPES)
def test_small_products_beside_large_ones_that_cancel(shape) -> None:
    m, n, k = shape
    gen = torch.Generator().manual_seed(m + n)
    x, w = _rows(gen, m, k), _up(gen, n, k)
    powers = torch.randint(0, 4, (n,), generator=gen)
    want = (x.cuda() @ w.t().contiguous().cuda()).cpu() * 2.0**powers
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        got = mxfp4_gemm(*_stored(x, "mxfp8"), *_stored(w, "mxfp4", powers), dtype=dtype)
        assert torch.equal(got.cpu(), want.to(dtype)), (dtype, float((got.cpu().double() - want).abs().max()))


@pytest.mark.parametrize("gate", ["silu", "gelu"])
@pytest.mark.parametrize("shape", SHAPES)
def test_gated_small_products_beside_large_ones_that_cancel(shape, gate) -> None:
    m, n, k = shape
    gen = torch.Generator().manual_seed(m + n)
    x, w = _rows(gen, m, k), _up(gen, n, k)
    want = (x.cuda() @ w.t().contiguous().cuda()).cpu() * k
    operands = (*_stored(x, "mxfp8"), *_stored(_gate(n, k), "mxfp4"), *_stored(w, "mxfp4"))
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        got = mxfp4_gated_gemm(*operands, gate=gate, output=dtype)
        assert torch.equal(got.cpu(), want.to(dtype)), (dtype, float((got.cpu().double() - want).abs().max()))
    for fmt in ("mxfp8", "mxfp4"):
        values, scales = mxfp4_gated_gemm(*operands, gate=gate, output=fmt)
        codes, want_scales = reference.quantize(want, fmt)
        # (A result of zero may have either sign.)
        assert torch.equal(scales.cpu(), want_scales)
        assert torch.equal(reference.read(values, scales, fmt), reference.values(codes, want_scales, fmt))
