"""A launch of 2^32 threads or more is refused before it reaches the runtime, which runs it modulo that without an error.

No test here launches GPU work: the refusal comes first, and addresses are never dereferenced.
"""

from __future__ import annotations

import pytest

from qpu_xla_amd import _lib

FAKE, FAR = 1 << 20, 1 << 40  # 16-byte aligned; operands of one call lie FAR apart


def _refused(name, *args) -> None:
    assert getattr(_lib.load(), name)(*args) == _lib.INVALID_ARGUMENT
    assert "2^32" in _lib.last_error()


def test_rows_of_a_workgroup_each() -> None:
    _refused("qxt_quantize_rows_int8", FAKE, 32, FAKE + FAR, 8, FAKE + 2 * FAR, 2**24, 8, 8, 0, None)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("fmt", [_lib.MX_FP4, _lib.MX_FP8])
def test_results_of_more_tiles_than_a_launch_takes(fmt, kind) -> None:
    m, n, k = 2**26 - 1, 2**14, 128  # at least 2^24 tiles, of 256 threads at least
    blocks = lambda at, row: _lib.MX_MATRIX.pack(at, row, at + FAR // 2, 4)  # noqa: E731
    _refused("qxt_mxfp4_gemm", blocks(FAKE, 128 if fmt else 64), fmt, blocks(FAKE + FAR, 64), None, FAKE + 4 * FAR, 4 * n, kind, m, n, k,
             FAKE + 2 * FAR, 2**62, None)


@pytest.mark.parametrize("stride", [1 << 23, 1 << 40, 1 << 63, 2**64 - 16])
@pytest.mark.parametrize("rows", [3, 40])
def test_weights_that_lie_far_apart(rows, stride) -> None:
    """Strides are unsigned: those past 2^63 are as far apart as any."""
    blocks = lambda at, row: _lib.MX_MATRIX.pack(at, row, at + FAR // 2, 4)  # noqa: E731
    _lib.set_failure_mask(_lib.FAIL_SUBMISSION)
    try:
        for a_stride, w_stride in ((stride, 64), (64, stride)):
            assert _lib.load().qxt_mxfp4_gemm(blocks(FAKE, a_stride), _lib.MX_FP4, blocks(FAKE + FAR, w_stride), None, FAKE + 4 * FAR,
                                              256, 0, rows, 64, 128, FAKE + 2 * FAR, 2**40, None) == _lib.INVALID_ARGUMENT
    finally:
        _lib.set_failure_mask(_lib.FAIL_NONE)
