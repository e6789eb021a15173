"""Rows that hold no numbers go through the norms' quantising as through the quantisers: a block of NaN stays one."""

from __future__ import annotations

import math

import pytest
import torch

from qpu_xla_amd.kernels import (
    add_rms_norm,
    add_rms_norm_int8,
    add_rms_norm_mxfp4,
    add_rms_norm_mxfp8,
    add_rms_norm_q8_0,
    quantize_mxfp4,
    quantize_mxfp8,
    quantize_q8_0,
    quantize_rows_int8,
)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offset", [0, 1])  # rows held in registers, and those of any alignment
@pytest.mark.parametrize("width", [64, 96, 4096, 11008])
def test_codes_are_those_of_the_quantisers(width, offset) -> None:
    store = torch.randn((9, width + offset), generator=torch.Generator().manual_seed(width)).cuda()
    x, weight = store[:, offset:], torch.ones(width, device="cuda")
    x[1, 3], x[2, 5], x[3], x[4], x[5, 0] = math.nan, math.inf, math.nan, 0.0, -math.inf
    weight[33] = math.inf
    weight[width - 32:] = math.nan  # a block of NaN in rows of numbers
    x[6] *= 1e30
    x[7, 40] = 0.0  # no number where the weight is infinite
    y, _ = add_rms_norm(x, weight)
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(y[:, -32:]).all()) and bool(torch.isfinite(y[0, :32]).all())
    assert torch.equal(add_rms_norm_q8_0(x, weight)[0], quantize_q8_0(y))
    values, scales, _ = add_rms_norm_int8(x, weight)
    want, want_scales = quantize_rows_int8(y)
    assert torch.equal(values, want.view_as(values)) and torch.equal(scales.view(torch.int32), want_scales.flatten().view(torch.int32))
    for norm, quantise in ((add_rms_norm_mxfp8, quantize_mxfp8), (add_rms_norm_mxfp4, quantize_mxfp4)):
        values, scales, _ = norm(x, weight)
        want, want_scales = quantise(y)
        assert torch.equal(values.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales, want_scales)
