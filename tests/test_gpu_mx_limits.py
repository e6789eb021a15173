"""Norms, blocks and 4-bit linears at the ends of their ranges: long K, LDS at its fullest, rows gigabytes apart, many columns."""

from __future__ import annotations

import pytest
import torch

import mx_reference as reference
from qpu_xla_amd.kernels import (
    add_rms_norm_int8,
    add_rms_norm_mxfp4,
    dequantize_mxfp4,
    dequantize_mxfp8,
    mxfp4_gated_gemm,
    mxfp4_gated_linear,
    mxfp4_gemm,
    mxfp4_linear,
    quantize_mxfp4,
    quantize_mxfp8,
    quantize_rows_int8,
)

pytestmark = pytest.mark.gpu

QUANTIZE = {"mxfp4": quantize_mxfp4, "mxfp8": quantize_mxfp8}
READ = {"mxfp4": dequantize_mxfp4, "mxfp8": dequantize_mxfp8}


def _product(a, fmt, w):
    """(a w^T, |a| |w|^T) of stored blocks in 64 bits: what they read back as is exact in float32."""
    a, w = READ[fmt](*a).double(), dequantize_mxfp4(*w).double()
    return ((a[:, None] * w[None]).sum(-1).cpu(), (a.abs()[:, None] * w.abs()[None]).sum(-1).cpu())


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(1, 40, 65536), (3, 7, 2**20), (1, 4, 2**22 - 32), (20, 5, 2**18 + 96)])
def test_long_k(m, n, k, fmt) -> None:
    gen = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn((m, k), generator=gen, device="cuda")
    w = quantize_mxfp4(torch.randn((n, k), generator=gen, device="cuda"))
    a = QUANTIZE[fmt](x)
    want, size = _product(a, fmt, w)
    got = mxfp4_gemm(*a, *w)
    reference.check(got, want, reference.rounded(want, reference.sum_error(size, k, fmt, True), torch.float32))
    assert torch.equal(got, mxfp4_linear(x, *w, activations=fmt))


@pytest.mark.parametrize("m,k,fmt", [(11, 4096, "mxfp8"), (16, 2816, "mxfp8"), (1, 45056, "mxfp8"), (16, 5504, "mxfp4"), (2, 4096, "mxfp8"), (4, 4096, "mxfp4")])
def test_fullest_lds(m, k, fmt) -> None:
    """The most rows that lie in LDS beside the weights, and the most floats quantised there."""
    gen = torch.Generator().manual_seed(k)
    x = torch.randn((m, k), generator=gen).cuda()
    g, u = (quantize_mxfp4(torch.randn((96, k), generator=gen).cuda()) for _ in range(2))
    a = QUANTIZE[fmt](x)
    operands = [READ[fmt](*a).cpu().double(), dequantize_mxfp4(*g).cpu().double(), dequantize_mxfp4(*u).cpu().double()]
    want, error = reference.gated(*operands, "silu", fmt, True)
    reference.check(mxfp4_gated_gemm(*a, *g, *u), want, reference.rounded(want, error, torch.float32))
    for dtype in (torch.float32, torch.bfloat16):
        rows = x.to(dtype)
        assert torch.equal(mxfp4_gated_linear(rows, *g, *u, activations=fmt, output=torch.float32), mxfp4_gated_gemm(*QUANTIZE[fmt](rows), *g, *u))
        assert torch.equal(mxfp4_linear(rows, *g, activations=fmt, dtype=torch.float32), mxfp4_gemm(*QUANTIZE[fmt](rows), *g))


@pytest.mark.parametrize("fmt,m,k", [("mxfp8", 16, 8192), ("mxfp8", 9, 14336), ("mxfp8", 10, 14336), ("mxfp4", 16, 16384), ("mxfp8", 12, 4128)])
@pytest.mark.parametrize("n", [1030, 4096])
def test_rows_that_fill_the_lds_of_a_lone_workgroup(n, m, k, fmt) -> None:
    gen = torch.Generator(device="cuda").manual_seed(k + m)
    x = torch.randn((m, k), generator=gen, device="cuda")
    w = quantize_mxfp4(torch.randn((n, k), generator=gen, device="cuda"))
    a = QUANTIZE[fmt](x)
    want, size = reference.product(READ[fmt](*a).cpu().double(), dequantize_mxfp4(*w).cpu().double())
    got = mxfp4_gemm(*a, *w)
    reference.check(got, want, reference.rounded(want, reference.sum_error(size, k, fmt, True), torch.float32))
    assert torch.equal(got, mxfp4_linear(x, *w, activations=fmt))


@pytest.mark.parametrize("m", [3, 40])
def test_rows_gigabytes_apart(m) -> None:
    """Offsets past 32 bits, in elements' and in bytes."""
    k, n, apart = 512, 96, 2**32 // (m - 1) // 16 * 8 + 4096  # elements of two bytes: the last row begins past 2^32 bytes
    gen = torch.Generator().manual_seed(m)
    x = torch.randn((m, k), generator=gen).bfloat16().cuda()
    w = quantize_mxfp4(torch.randn((n, k), generator=gen).cuda())
    wide = torch.empty((m * apart,), dtype=torch.bfloat16, device="cuda")
    far, out = wide.as_strided((m, k), (apart, 1)), wide.as_strided((m, n), (apart, 1), 1024)
    far.copy_(x)
    assert (m - 1) * apart * 2 > 2**32
    assert torch.equal(mxfp4_linear(far, *w, out=out), mxfp4_linear(x, *w)) and torch.equal(far, x)
    for got, want in zip(quantize_mxfp8(far), quantize_mxfp8(x)):
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
    weight, residual = torch.ones(k, device="cuda"), wide.as_strided((m, k), (apart, 1), 2048)
    residual.copy_(x.flip(0))
    for norm in (add_rms_norm_int8, add_rms_norm_mxfp4):
        for got, want in zip(norm(far, weight, residual), norm(x, weight, x.flip(0).contiguous())):
            assert torch.equal(got, want)
    read = wide.as_strided((m, k), (apart, 1), 2816)
    dequantize_mxfp4(*quantize_mxfp4(x), read)
    assert torch.equal(read, dequantize_mxfp4(*quantize_mxfp4(x), dtype=torch.bfloat16))


@pytest.mark.parametrize("m", [1, 17])
def test_many_columns(m) -> None:
    k, n = 64, 300_007
    gen = torch.Generator(device="cuda").manual_seed(m)
    a = quantize_mxfp8(torch.randn((m, k), generator=gen, device="cuda"))
    w = quantize_mxfp4(torch.randn((n, k), generator=gen, device="cuda"))
    want, size = reference.product(dequantize_mxfp8(*a).cpu().double(), dequantize_mxfp4(*w).cpu().double())
    reference.check(mxfp4_gemm(*a, *w), want, reference.rounded(want, reference.sum_error(size, k, "mxfp8", True), torch.float32))


def test_int8_rows_are_the_quantisers_at_every_width() -> None:
    """Widths from one piece to several a thread: the norm of rows with unit mean square and a weight of ones is a rescaling."""
    for columns in (8, 264, 8192, 8200, 12288, 32768, 32776):
        x = torch.randn((5, columns), generator=torch.Generator().manual_seed(columns)).cuda()
        codes, scales, _ = add_rms_norm_int8(x, torch.ones(columns, device="cuda"), epsilon=0.0)
        _, rounded, _ = reference.norm(x, torch.ones(columns), None, 0.0)
        want = quantize_rows_int8(rounded.cuda())
        assert torch.equal(codes, want[0]) and torch.equal(scales.flatten(), want[1].flatten())
