"""The gate functions far from zero: float32 results relative to their own size, from sums that are exact.

Gates are sums of two elements, ups are one element each, so that both are exact in float32.

SiLU: a power of two and a reciprocal (2 units of 2^-24 each), the power's correction (2), the sum in the denominator (1) and
four products at most: 11 units.  GELU: the argument is off by 1.5 units (its product and its constant), which erfc takes
times 2 x^2 + 1 at most, x^2 = g^2 / 2; erfc itself is good for 16 units in the last place (32), and there are two products.
Below float32's normal numbers a result is off by one of its least steps.
"""

from __future__ import annotations

import math

import pytest
import torch

import mx_reference as reference
from qpu_xla_amd.kernels import mxfp4_gated_gemm, quantize_mxfp4

pytestmark = pytest.mark.gpu

UNIT = 2.0**-24


def _operands(g_high, g_low, up_power):
    """(activations, gate weights, up weights): 32 columns of g = g_high + g_low and u = 2^up_power a row."""
    m = len(g_high)
    a = torch.zeros((m, 64), dtype=torch.float8_e4m3fn)
    a[:, 0], a[:, 1], a[:, 32] = g_high.to(torch.float8_e4m3fn), g_low.to(torch.float8_e4m3fn), 1.0
    scales = torch.full((m, 2), 127, dtype=torch.uint8)
    scales[:, 1] = 127 + up_power
    gate, up = torch.zeros((32, 64)), torch.zeros((32, 64))
    gate[:, 0] = gate[:, 1] = 1.0
    up[:, 32] = 1.0
    return (a.cuda(), scales.cuda()), quantize_mxfp4(gate.cuda()), quantize_mxfp4(up.cuda())


def _gates(low, high):
    """About 400 sums of two 8-bit elements between `low` and `high`, of either sign, spread over their logarithms."""
    gen = torch.Generator().manual_seed(3)
    size = torch.exp(torch.rand((200,), generator=gen, dtype=torch.float64) * math.log(high / low) + math.log(low))
    first = reference.FP8[torch.searchsorted(reference.FP8, size.clamp(max=440.0)) - 1]
    second = reference.FP8[(torch.searchsorted(reference.FP8, size - first) - 1).clamp(min=0)]
    return torch.cat([first, -first]), torch.cat([second, -second])


@pytest.mark.parametrize("m", [8, 400])
@pytest.mark.parametrize("up_power", [0, 90])
@pytest.mark.parametrize("gate,low,high", [("silu", 0.05, 104.0), ("gelu", 0.05, 12.8)])
def test_gate_functions_to_a_few_units(gate, low, high, up_power, m) -> None:
    g_high, g_low = _gates(low, high)
    g = g_high + g_low
    assert torch.equal(g, g.float().double()) and float(g.min()) < -0.9 * high
    want = reference.gate_of(gate, g) * 2.0**up_power
    units = 11.0 if gate == "silu" else 1.5 * (g.square() + 1) + 34
    bound = units * UNIT * want.abs() + 2.0**-149
    for start in range(0, len(g), m):  # few rows a call, and many
        part = slice(start, start + m)
        a, gates, ups = _operands(g_high[part], g_low[part], up_power)
        got = mxfp4_gated_gemm(*a, *gates, *ups, gate=gate)
        reference.check(got, want[part, None].expand(-1, 32), bound[part, None].expand(-1, 32))


@pytest.mark.parametrize("gate", ["silu", "gelu"])
@pytest.mark.parametrize("m", [2, 40])
def test_gate_functions_at_their_ends(gate, m) -> None:
    """Large gates: themselves, or zero; no gate: zero.  A gate that is no number: no number."""
    g = torch.tensor([448.0, -448.0, 0.0, math.nan], dtype=torch.float64)
    for value, want in zip(g.tolist(), (448.0, 0.0, 0.0, math.nan)):
        a, gates, ups = _operands(torch.full((m,), value, dtype=torch.float64), torch.zeros(m, dtype=torch.float64), 0)
        got = mxfp4_gated_gemm(*a, *gates, *ups, gate=gate).cpu()
        assert torch.equal(got.nan_to_num(7.0), torch.full((m, 32), want).nan_to_num(7.0))
    a, gates, ups = _operands(torch.full((m,), 448.0), torch.zeros(m), 0)
    far = a[1].clone()
    far[:, 0] = 254  # 448 * 2^127: infinite as a sum
    got = mxfp4_gated_gemm(a[0], far, *gates, *ups, gate=gate)
    assert bool((got == math.inf).all())
