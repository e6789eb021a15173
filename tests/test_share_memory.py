"""Whether rows share memory, told for every pair of places in a small buffer and compared with the bytes themselves."""

from __future__ import annotations

import itertools

import torch

from qpu_xla_amd._rows import share_memory


def _bytes(t):
    return {t.data_ptr() + t.element_size() * sum(i * s for i, s in zip(index, t.stride())) + b
            for index in itertools.product(*map(range, t.shape)) for b in range(t.element_size())}


def test_rows_of_one_buffer() -> None:
    buffer = torch.zeros(60, dtype=torch.uint8)
    places = [buffer.as_strided((rows, columns), (stride, 1), offset)
              for rows in (1, 2, 3) for columns in (1, 3, 7) for stride in (7, 10) for offset in (0, 2, 5, 9, 17, 30)]
    places += [buffer[offset:offset + length] for offset in (0, 11, 24) for length in (1, 8)]
    taken = [_bytes(t) for t in places]
    for (a, mine), (b, others) in itertools.product(zip(places, taken), repeat=2):
        met = bool(mine & others)
        told = share_memory(a, b)
        assert told or not met
        strides = {t.stride(0) for t in (a, b) if t.dim() > 1 and t.shape[0] > 1}
        last = max(mine) < min(others) or max(others) < min(mine)
        if last or len(strides) == 0:
            assert told == met
    assert not share_memory(buffer[:0], buffer) and not share_memory(buffer.view(6, 10)[:, :4], buffer.view(6, 10)[:, 4:])


def test_types_of_more_bytes() -> None:
    wide = torch.zeros((4, 8), dtype=torch.float32)
    assert share_memory(wide[:, :4], wide[:, 3:5]) and not share_memory(wide[:, :4], wide[:, 4:])
    assert share_memory(wide, wide.view(torch.uint8)[2:3]) and not share_memory(wide[:2], wide.view(torch.bfloat16)[2:])
