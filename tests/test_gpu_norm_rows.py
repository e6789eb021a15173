"""Residual norms over more rows than one launch takes: a launch has fewer than 2^32 threads, a workgroup for each row."""

from __future__ import annotations

import pytest
import torch

from qpu_xla_amd.kernels import add_rms_norm, add_rms_norm_int8, add_rms_norm_mxfp4

pytestmark = pytest.mark.gpu


def _rows(rows, columns, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((rows, columns), generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _joined(call, x, weight, residual):
    """The same rows by two calls of half as many."""
    half = x.shape[0] // 2
    parts = [call(x[s], weight, None if residual is None else residual[s]) for s in (slice(0, half), slice(half, None))]
    return [None if a is None else torch.cat([a, b]) for a, b in zip(*parts)]


@pytest.mark.parametrize("call,rows,columns,dtype,adds", [
    (add_rms_norm, 2**24 + 3, 4, torch.float32, True),  # 256 threads a row
    (add_rms_norm_int8, 2**24 + 3, 5, torch.bfloat16, True),
    (add_rms_norm, 2**26 + 5, 8, torch.bfloat16, False),  # 64
    (add_rms_norm_int8, 2**26 + 5, 8, torch.bfloat16, False),
    (add_rms_norm_mxfp4, 2**26 + 5, 32, torch.bfloat16, False),
])
def test_more_rows_than_a_launch_takes(call, rows, columns, dtype, adds) -> None:
    x, residual = _rows(rows, columns, dtype, 1), _rows(rows, columns, dtype, 2) if adds else None
    weight = torch.linspace(0.5, 1.5, columns, device="cuda")
    got = call(x, weight, residual)
    for a, b in zip(got, _joined(call, x, weight, residual)):
        assert (a is None) == (b is None)
        if a is not None:
            assert torch.equal(a, b)
