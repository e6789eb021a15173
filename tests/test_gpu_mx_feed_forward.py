"""A refused feed-forward block leaves the stream as it was, and no output of one is written over another operand."""

from __future__ import annotations

import pytest
import torch

from qpu_xla_amd import quantization
from qpu_xla_amd.errors import DependencyError
from qpu_xla_amd.quantization import QuantizedMatrixMxfp4, mxfp4_feed_forward, quantize_matrix_mxfp4

pytestmark = pytest.mark.gpu

D, HIDDEN, M = 128, 192, 5


def _layer():
    gen = torch.Generator().manual_seed(0)
    draw = lambda n, k: quantize_matrix_mxfp4(torch.randn((n, k), generator=gen).cuda())  # noqa: E731
    rows = lambda: torch.randn((M, D), generator=gen).cuda()  # noqa: E731
    return rows(), rows(), torch.ones(D, device="cuda"), draw(HIDDEN, D), draw(HIDDEN, D), draw(D, HIDDEN)


def _moved(matrix, offset):
    """The same matrix with its values `offset` bytes past an aligned address."""
    store = torch.empty(matrix.values.numel() + offset, dtype=torch.uint8, device="cuda")
    values = store[offset:].view(matrix.values.shape)
    values.copy_(matrix.values)
    return QuantizedMatrixMxfp4(values, matrix.scales)


def _cpu(matrix):
    return QuantizedMatrixMxfp4(matrix.values.cpu(), matrix.scales)


@pytest.mark.parametrize("changes", [
    lambda g, u, d: {"function": "relu"},
    lambda g, u, d: {"activations": "int8"},
    lambda g, u, d: {"dtype": torch.int32},
    lambda g, u, d: {"out": torch.empty((M, D), device="cuda"), "dtype": torch.bfloat16},
    lambda g, u, d: {"out": torch.empty((M, HIDDEN), device="cuda")},
    lambda g, u, d: {"out": torch.empty((M, D))},
    lambda g, u, d: {"out": torch.empty((M, 2 * D), device="cuda")[:, ::2]},
    lambda g, u, d: {"gate": d},
    lambda g, u, d: {"up": quantize_matrix_mxfp4(torch.ones((HIDDEN + 32, D), device="cuda"))},
    lambda g, u, d: {"down": g},
    lambda g, u, d: {"gate": quantize_matrix_mxfp4(torch.ones((48, D), device="cuda")),
                     "up": quantize_matrix_mxfp4(torch.ones((48, D), device="cuda"))},
    lambda g, u, d: {"gate": _moved(g, 8)},
    lambda g, u, d: {"down": _moved(d, 1)},
    lambda g, u, d: {"up": _cpu(u)},
    lambda g, u, d: {"down": _cpu(d)},
    lambda g, u, d: {"epsilon": -1.0},
])
def test_refused_calls_leave_the_stream(changes) -> None:
    x, residual, weight, gate, up, down = _layer()
    kept = residual.clone()
    options = {"gate": gate, "up": up, "down": down, **changes(gate, up, down)}
    with pytest.raises((ValueError, RuntimeError, DependencyError)):
        mxfp4_feed_forward(x, residual, weight, **options, residual_out=residual)
    assert torch.equal(residual, kept)
    y, total = mxfp4_feed_forward(x, residual, weight, gate, up, down, residual_out=residual)
    assert total is residual and torch.equal(residual, x + kept)
    want, _ = mxfp4_feed_forward(x, kept, weight, gate, up, down)
    assert torch.equal(y, want)


def test_outputs_over_other_operands_are_refused() -> None:
    x, residual, weight, gate, up, down = _layer()
    kept = [t.clone() for t in (x, residual, weight, gate.values, up.values, down.values, gate.scales, up.scales, down.scales)]
    over = lambda t, rows, columns: t.view(torch.float32).flatten()[: rows * columns].view(rows, columns)  # noqa: E731
    for options in ({"out": residual, "residual_out": residual}, {"out": x, "residual_out": x},
                    {"out": over(gate.values, M, D)}, {"out": over(up.values, M, D)}, {"out": over(down.values, M, D)},
                    {"residual_out": over(gate.values, M, D)}, {"residual_out": over(down.values, M, D)}):
        with pytest.raises(ValueError, match="shares memory"):
            mxfp4_feed_forward(x, residual, weight, gate, up, down, **options)
    for t, was in zip((x, residual, weight, gate.values, up.values, down.values, gate.scales, up.scales, down.scales), kept):
        assert torch.equal(t, was)


def test_outputs_over_what_is_no_longer_read() -> None:
    x, residual, weight, gate, up, down = _layer()
    want, total = mxfp4_feed_forward(x, residual, weight, gate, up, down)
    for place in (0, 1):  # over x, over the residual
        rows = [x.clone(), residual.clone()]
        y, again = mxfp4_feed_forward(*rows, weight, gate, up, down, out=rows[place])
        assert y is rows[place] and torch.equal(y, want) and torch.equal(again, total)
    wide = torch.zeros((M, 2 * D), device="cuda")  # y and the sum side by side
    y, again = mxfp4_feed_forward(x, residual, weight, gate, up, down, out=wide[:, :D], residual_out=wide[:, D:])
    assert torch.equal(y, want) and torch.equal(again, total)
    assert quantization.mxfp4_feed_forward(x[:0], residual[:0], weight, gate, up, down)[0].shape == (0, D)
