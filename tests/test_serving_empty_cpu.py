"""The paged operators' C entries on nothing: no sequences, no tokens, and the NULL
pointers that empty tensors have."""

from __future__ import annotations

import ctypes as C

import pytest

from tensorshrink_b200 import _C
from test_serving_cpu import INVALID, WORKSPACE, cache

THREE = (C.c_int64 * 3)(64, 64, 64)
EMPTY = dict(batch=0, k_pages=None, v_pages=None, page_table=None, seq_lens=None, num_pages=0, max_pages=0)


@pytest.mark.parametrize("kw", [dict(batch=0), EMPTY])
def test_no_sequences(kw):
    lib, c = _C.load(), cache(**kw)
    assert lib.ts_paged_append(None, THREE, None, THREE, 3, None, c, None, None, None, 0, None, None, None) == 0
    assert lib.ts_paged_decode_attention(None, 192, 1, c, None, None, None, 0, 0.1, 0, None, 64, None, 0, None) == 0
    assert lib.ts_paged_decode_attention(None, 192, 1, c, None, None, None, 0, 0.1, 1, None, 64, None, 0, None) == 0
    assert lib.ts_paged_evict(c, 4, 0, None, 0, None) == 0
    assert lib.ts_paged_decode_attention(None, 192, 1, c, None, None, None, 0, -1.0, 0, None, 64, None, 0, None) == INVALID
    assert lib.ts_paged_evict(c, 0, 0, None, 0, None) == INVALID


def test_no_tokens():
    lib, c = _C.load(), cache()
    assert lib.ts_paged_append(None, THREE, None, THREE, 0, None, c, None, None, None, 0, None, None, None) == 0
    assert lib.ts_paged_append(None, THREE, None, THREE, 1, None, c, None, None, None, 0, None, None, None) == INVALID
    assert lib.ts_paged_append(4096, THREE, 4096, THREE, -1, None, c, None, None, None, 0, None, None, None) == INVALID


def test_memory_is_asked_for_where_there_are_sequences():
    lib = _C.load()
    for kw in (dict(EMPTY, batch=1), dict(num_pages=0), dict(max_pages=0), dict(seq_lens=None)):
        assert lib.ts_paged_evict(cache(scores=4096, slot_pos=4096, **kw), 4, 0, None, 0, None) == INVALID
    assert lib.ts_paged_evict(cache(scores=4096, slot_pos=4096), 4, 0, None, 0, None) == WORKSPACE
