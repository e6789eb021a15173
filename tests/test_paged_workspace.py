"""A call of the C ABI takes the workspace that ``*_workspace()`` names for its arguments (no GPU: an injected failure
returns after the checks and before any launch)."""

from __future__ import annotations

import pytest

from qpu_xla_amd import _lib

FAKE = 1 << 20  # 16-byte aligned, never dereferenced
HEADS, KV_HEADS, DIM, PAGE = 32, 8, 128, 64


@pytest.fixture
def stopped():
    _lib.load()
    _lib.set_failure_mask(_lib.FAIL_SUBMISSION)
    yield
    _lib.set_failure_mask(_lib.FAIL_NONE)


def _cache(slots, sequences):
    row = 2 * DIM
    strides = (PAGE * KV_HEADS * row, KV_HEADS * row, row)
    return _lib.PAGED_CACHE.pack(FAKE, *strides, FAKE, *strides, FAKE, 4 * (slots // PAGE), FAKE, slots // PAGE, PAGE, KV_HEADS, DIM,
                                 _lib.TYPE_BF16, slots // PAGE, sequences)


def _scores(slots, sequences, tokens, starts, max_query, max_context):
    lib = _lib.load()
    size = lib.qxt_paged_attention_scores_workspace(HEADS, KV_HEADS, sequences, tokens, slots, max_query, max_context)
    return lib.qxt_paged_attention_scores(
        FAKE, 2 * HEADS * DIM, 2 * DIM, _cache(slots, sequences), starts, FAKE, 4 * HEADS, None, 0, 0, FAKE, 4 * KV_HEADS * slots,
        4 * slots, tokens, HEADS, 0.1, 1, 0, max_query, max_context, FAKE if size else None, size, None)


def _attention(slots, sequences, tokens, starts, max_query, max_context):
    lib = _lib.load()
    size = lib.qxt_paged_attention_workspace(HEADS, KV_HEADS, DIM, sequences, tokens, max_query, max_context)
    return lib.qxt_paged_attention(
        FAKE, 2 * HEADS * DIM, 2 * DIM, _cache(slots, sequences), starts, FAKE, 2 * HEADS * DIM, 2 * DIM, _lib.TYPE_BF16, None, 0,
        tokens, HEADS, 0.1, 1, 0, max_query, max_context, FAKE if size else None, size, None)


@pytest.mark.parametrize("call", [_scores, _attention])
@pytest.mark.parametrize("max_context", [0, 1, 100, 4096, 4097, 8192, 1 << 20, 2**32 - 1])
@pytest.mark.parametrize("tokens", [1, 9, 300, 4096])
@pytest.mark.parametrize("sequences", [1, 3])
def test_contexts_up_to_and_past_the_slots(stopped, call, max_context, tokens, sequences) -> None:
    for max_query in {1, 7, tokens, 2 * tokens}:
        assert call(4096, sequences, tokens, FAKE, max_query, max_context) == _lib.SUBMISSION_FAILED, _lib.last_error()


@pytest.mark.parametrize("call", [_scores, _attention])
@pytest.mark.parametrize("sequences", [1, 2, 7, 64, 300])
@pytest.mark.parametrize("max_query", [0, 1, 2, 9, 64, 2**32 - 1])
def test_one_token_a_sequence_whatever_max_query_says(stopped, call, sequences, max_query) -> None:
    for max_context in (1, 700, 4096, 65536):
        assert call(65536, sequences, sequences, None, max_query, max_context) == _lib.SUBMISSION_FAILED, _lib.last_error()
        assert call(65536, sequences, sequences, FAKE, max_query, max_context) == _lib.SUBMISSION_FAILED, _lib.last_error()
