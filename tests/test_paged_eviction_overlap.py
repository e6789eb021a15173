"""Eviction refuses outputs whose rows share memory with other rows, and takes those in place or apart (no GPU: an
injected failure returns after the checks and before any launch)."""

from __future__ import annotations

import itertools
import random

import pytest

from qpu_xla_amd import _lib

BASE = 1 << 30  # never dereferenced
SLOTS = 32
ROW = 4 * SLOTS


def _evict(sequences, heads, scores, out, lens_out=1 << 29, which="scores"):
    """Status with rows (address, sequence stride, head stride) of `which` in and out, the other array in place."""
    lib = _lib.load()
    lens = 1 << 28
    cache = _lib.PAGED_CACHE.pack(BASE, 16 * heads * 128, heads * 128, 128, BASE, 16 * heads * 128, heads * 128, 128, BASE, 8, lens,
                                  8, 16, heads, 64, _lib.TYPE_BF16, SLOTS // 16, sequences)
    plain = (1 << 31, heads * ROW, ROW)
    rows = (*scores, *out, *plain, *plain) if which == "scores" else (*plain, *plain, *scores, *out)
    size = lib.qxt_paged_cache_evict_workspace(heads, sequences, SLOTS, 8)
    _lib.set_failure_mask(_lib.FAIL_SUBMISSION)
    try:
        return lib.qxt_paged_cache_evict(cache, *rows, lens_out, 8, 4, SLOTS, BASE, size, None)
    finally:
        _lib.set_failure_mask(_lib.FAIL_NONE)


@pytest.mark.parametrize("which", ["scores", "positions"])
@pytest.mark.parametrize("sequences,heads,rows,out,fine", [
    (3, 2, (BASE, 2 * ROW, ROW), (BASE, 2 * ROW, ROW), True),                        # in place
    (3, 2, (BASE, ROW, 3 * ROW), (BASE, ROW, 3 * ROW), True),                        # in place, heads first
    (3, 2, (BASE, 2 * ROW, ROW), (BASE + 6 * ROW, 2 * ROW, ROW), True),              # apart
    (3, 2, (BASE, 2 * ROW, ROW), (BASE + 6 * ROW, ROW, 3 * ROW), True),
    (3, 2, (BASE, 4 * ROW, ROW), (BASE + 2 * ROW, 4 * ROW, ROW), True),              # turn by turn in one buffer
    (3, 2, (BASE, 4 * ROW, 2 * ROW), (BASE + ROW, 4 * ROW, 2 * ROW), True),
    (1, 1, (BASE, 0, 0), (BASE, 4, 8), True),                                        # strides of single rows do not matter
    (1, 2, (BASE, 0, ROW), (BASE, 64, ROW), True),
    (3, 2, (BASE, 0, 0), (BASE + ROW, 2 * ROW, ROW), True),                          # expanded inputs are only read
    (3, 2, (BASE, 2 * ROW, ROW), (BASE + ROW, 2 * ROW, ROW), False),                 # one head on
    (3, 2, (BASE, 2 * ROW, ROW), (BASE + 2 * ROW, 2 * ROW, ROW), False),             # one sequence on
    (3, 2, (BASE, 2 * ROW, ROW), (BASE + 4, 2 * ROW, ROW), False),                   # one slot on
    (1, 1, (BASE, 0, 0), (BASE - 4, 0, 0), False),
    (3, 2, (BASE, 2 * ROW, ROW), (BASE, ROW, 3 * ROW), False),                       # the same memory in another order
    (3, 2, (BASE, 0, ROW), (BASE, 0, ROW), False),                                   # expanded outputs
    (3, 2, (BASE, 2 * ROW, ROW), (BASE + 99 * ROW, ROW, 0), False),
    (3, 2, (BASE, 2 * ROW, ROW), (BASE + 99 * ROW, 2 * ROW, ROW - 4), False),
    (3, 2, (BASE, 2 * ROW, ROW), (BASE + 99 * ROW, ROW, ROW), False),
])
def test_rows_of_outputs(sequences, heads, rows, out, fine, which) -> None:
    status = _evict(sequences, heads, rows, out, which=which)
    assert status == (_lib.SUBMISSION_FAILED if fine else _lib.INVALID_ARGUMENT)
    if not fine:
        assert "share memory" in _lib.last_error()


def test_rows_of_outputs_against_their_definition() -> None:
    rng = random.Random(0)
    seen = set()
    for _ in range(3000):
        sequences, heads = rng.randint(1, 4), rng.randint(1, 4)
        strides = [ROW // 4 * rng.randint(0, 24) for _ in range(2)]
        apart = ROW // 4 * rng.randint(-40, 40) * rng.randint(0, 1)

        def starts(base):
            return [base + i * strides[0] + j * strides[1] for i in range(sequences) for j in range(heads)]

        a, b = starts(0), starts(apart)
        overlap = any(abs(x - y) < ROW for x, y in itertools.combinations(b, 2)) or any(
            abs(x - y) < ROW for (i, x), (j, y) in itertools.product(enumerate(a), enumerate(b)) if apart or i != j)
        status = _evict(sequences, heads, (BASE, *strides), (BASE + apart, *strides))
        assert status == (_lib.INVALID_ARGUMENT if overlap else _lib.SUBMISSION_FAILED), (sequences, heads, strides, apart)
        seen.add((overlap, apart != 0))
    assert len(seen) == 4


@pytest.mark.parametrize("step,fine", [(-12, True), (-8, False), (-4, False), (0, False), (4, False), (8, False), (12, True)])
def test_new_lengths_lie_apart_from_the_old(step, fine) -> None:
    rows = (BASE, 2 * ROW, ROW)
    status = _evict(3, 2, rows, rows, lens_out=(1 << 28) + step)
    assert status == (_lib.SUBMISSION_FAILED if fine else _lib.INVALID_ARGUMENT)
    if not fine:
        assert "in place" in _lib.last_error()
