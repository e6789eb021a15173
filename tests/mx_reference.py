"""Definitions in 64 bits, on the CPU, of the microscaling blocks, the residual norm, the linears and the gated product."""

from __future__ import annotations

import math

import torch

BLOCK = 32
FP4 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
FP8 = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()  # 0 .. 448
LARGEST = {"mxfp4": 2, "mxfp8": 8}  # floor(log2) of the largest element
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}  # half a step, relative


def quantize(x: torch.Tensor, fmt: str) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes [R, K] one a byte, scale bytes [R, K/32]) of rows, by searching the format's values for the nearest one."""
    grid = FP4 if fmt == "mxfp4" else FP8
    blocks = x.double().cpu().unflatten(-1, (-1, BLOCK))
    amax = blocks.abs().amax(-1)
    bad = ~torch.isfinite(blocks).all(-1)
    exponent = torch.where(amax > 0, torch.frexp(amax.nan_to_num(0, 0, 0)).exponent - 1, -1000) - LARGEST[fmt]
    scale = torch.where(bad, 255, exponent.clamp(min=-127) + 127).to(torch.uint8)
    size = blocks.nan_to_num(0, 0, 0).abs() / 2.0 ** (scale.double() - 127)[..., None]
    index = (size[..., None] - grid).abs().argmin(-1) if x.numel() < 200_000 else None
    borders = (grid[1:] + grid[:-1]) / 2  # ties go to the even code
    below, above = torch.bucketize(size, borders), torch.bucketize(size, borders, right=True)
    code = torch.where(below % 2 == 0, below, above)
    if index is not None:  # where there is no tie, the nearest value
        assert bool(((code == index) | (below != above)).all())
    code = code + torch.signbit(blocks) * (8 if fmt == "mxfp4" else 128)
    return torch.where(bad[..., None], 0, code).flatten(-2).to(torch.uint8), scale


def values(codes: torch.Tensor, scales: torch.Tensor, fmt: str) -> torch.Tensor:
    """What codes (one a byte) stand for."""
    half = 8 if fmt == "mxfp4" else 128
    grid = FP4 if fmt == "mxfp4" else torch.cat([FP8, torch.tensor([math.nan], dtype=torch.float64)])
    codes = codes.cpu().long()
    signed = grid[codes % half] * (1 - 2 * (codes // half))
    scale = torch.where(scales.cpu() == 255, math.nan, 2.0 ** (scales.cpu().double() - 127))
    return signed * scale.repeat_interleave(BLOCK, -1)


def unpack(stored: torch.Tensor, fmt: str) -> torch.Tensor:
    """Stored values -> codes, one a byte."""
    raw = stored.cpu().view(torch.uint8)
    return raw if fmt == "mxfp8" else torch.stack((raw & 15, raw >> 4), -1).flatten(-2)


def pack(codes: torch.Tensor, fmt: str) -> torch.Tensor:
    return codes.view(torch.float8_e4m3fn) if fmt == "mxfp8" else codes[..., 0::2] | codes[..., 1::2] << 4


def stored(x: torch.Tensor, fmt: str) -> tuple[torch.Tensor, torch.Tensor]:
    codes, scales = quantize(x, fmt)
    return pack(codes, fmt), scales


def read(stored_values: torch.Tensor, scales: torch.Tensor, fmt: str) -> torch.Tensor:
    return values(unpack(stored_values, fmt), scales, fmt)


def norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None, epsilon: float):
    """(y in 64 bits, y after its roundings to 32 bits, stored sum)."""
    total = None
    h = x.cpu()
    if residual is not None:
        total = (h.float() + residual.cpu().float()).to(residual.dtype)
        h = total
    h, weight = h.double(), weight.cpu().double()
    factor = 1 / torch.sqrt(h.square().sum(-1, keepdim=True) / h.shape[-1] + epsilon)
    rounded = ((h * factor.float().double()).float().double() * weight).float()
    return h * factor * weight, rounded, total


def int8_rows(y: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    scale = torch.maximum(y.abs().amax(-1).double() / 127, torch.tensor(0.0)).float()
    scale = torch.maximum(scale, torch.tensor(1.0 / 127.0, dtype=torch.float64).float())
    return torch.round((y.double() / scale[:, None].double()).float()).clamp(-127, 127).to(torch.int8), scale


def q8_0(y: torch.Tensor) -> torch.Tensor:
    blocks = y.unflatten(-1, (-1, BLOCK))
    d = (blocks.abs().amax(-1).double() / 127).float()
    inverse = torch.where(d > 0, (1 / d.double()).float(), 0.0)
    codes = torch.round((blocks.double() * inverse[..., None].double()).float()).clamp(-127, 127).to(torch.int8)
    return torch.cat([d.half()[..., None].view(torch.uint8), codes.view(torch.uint8)], -1)


def product(a: torch.Tensor, w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(a w^T, |a| |w|^T)."""
    return a @ w.t(), a.abs() @ w.abs().t()


def sum_error(size: torch.Tensor, k: int, fmt: str, exact: bool) -> torch.Tensor:
    """What the fp32 sums may be off by, given the sums of the products' magnitudes.

    A product of blocks is exact; each of the additions along K (at most K / 8 + 16: eight products a step, partial sums
    of waves and splits) loses at most a unit of 2^-23 of what it adds up.  The matrix instruction also drops, from each
    product of an 8-bit element, what lies more than 13 bits below the largest of its eight neighbours' exponents: at most
    2^-13 of that product's power of two, eight times, so 2^-10 of their sum.  Results in float32 are computed from parts
    for which nothing is dropped.
    """
    error = (k / 8 + 16) * 2.0**-23 * size
    return error if exact or fmt == "mxfp4" else error + 2.0**-10 * size


def gate_of(name: str, g: torch.Tensor) -> torch.Tensor:
    return g * torch.sigmoid(g) if name == "silu" else g * 0.5 * torch.erfc(-g / math.sqrt(2.0))


def gated(a: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, name: str, fmt: str, exact: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(f(a gate^T) (a up^T), what the kernel's fp32 value may be off by).

    Both gate functions have slopes below 1.13; the functions themselves err by at most 2^-20 relative to |g| (sums of
    1 + erf near zero cancel) and the products by a few units of 2^-24.
    """
    k = a.shape[1]
    g, g_size = product(a, gate)
    u, u_size = product(a, up)
    f = gate_of(name, g)
    dg, du = sum_error(g_size, k, fmt, exact), sum_error(u_size, k, fmt, exact)
    return f * u, 1.13 * dg * (u.abs() + du) + (f.abs() + 2.0**-20 * g.abs()) * du + (2.0**-20 * g.abs()) * u.abs() + 2.0**-22 * (f * u).abs()


def rounded(want: torch.Tensor, error: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The bound of a result stored in ``dtype``: half a step more, and half the least step below float16's range."""
    return error + HALF[dtype] * (want.abs() + error) + (2.0**-25 if dtype is torch.float16 else 1e-37)


def check(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor) -> None:
    got = got.cpu().double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    over = ((got - want).abs() - bound).nan_to_num(0.0)
    assert bool((over <= 0).all()), (float(over.max()), [int(i) for i in (over == over.max()).nonzero()[0]])


def check_blocks(stored_values: torch.Tensor, scales: torch.Tensor, fmt: str, want: torch.Tensor, error: torch.Tensor) -> None:
    """Blocks quantised from results that are ``error`` off at most: the scale is the one of a largest magnitude within
    the error, and each element is half a step off at most, or cut to the largest element."""
    blocks, off = want.unflatten(-1, (-1, BLOCK)), error.unflatten(-1, (-1, BLOCK))
    scales = scales.cpu()
    for sign in (-1, 1):
        amax = (blocks.abs() + sign * off).clamp(min=0).amax(-1)
        byte = (torch.where(amax > 0, torch.frexp(amax).exponent - 1, -1000) - LARGEST[fmt]).clamp(min=-127) + 127
        assert bool(((scales.int() - byte) * sign <= 0).all())
    scale = 2.0 ** (scales.double() - 127)[..., None]
    got = read(stored_values, scales, fmt).unflatten(-1, (-1, BLOCK))
    if fmt == "mxfp8":
        step = torch.maximum(2.0**-4 * (blocks.abs() + off), 2.0**-10 * scale)  # half a step of three bits, or of the least
        most = 448.0
    else:
        step, most = torch.maximum(0.25 * (blocks.abs() + off), 0.25 * scale), 6.0  # 1.5 of 6, 0.5 of 2 apart at most
    cut = (blocks.abs() + off - most * scale).clamp(min=0)
    assert bool(((got - blocks).abs() <= off + torch.maximum(step, cut) + 1e-37).all())
