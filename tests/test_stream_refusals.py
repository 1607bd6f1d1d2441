"""Calls of the 8-bit cache, the shared prefix and cross attention that are refused, each
before anything is launched."""

from __future__ import annotations

import ctypes

import pytest

from gki import _lib

P, NULL = 16, ctypes.c_void_p(0)          # an aligned address that nothing reads


@pytest.mark.parametrize("sink,ring", [(0, 2**30), (2**30, 8), (2**31 - 1, 2**31 - 1), (5, 2**30 - 5)])
def test_caches_of_2_30_rows_or_more(sink, ring):
    """As gki_rolling8_append refuses them: a row index past 31 bits."""
    lib = _lib.load()
    where = (2, 1, 2, 1, 1, 64, sink, 8, ring, 5, 0.1, 0)
    assert lib.gki_rolling8_append(*[P] * 6, 2, 1, 1, 64, sink, ring, 0, 1, NULL) == 1
    assert lib.gki_rolling8_decode(*[P] * 7, *where, 1, NULL) == 1
    assert b"2^30" in lib.gki_last_error()
    assert lib.gki_rolling_step(*[P] * 7, 0, 0, 0, P, P, *where, 0, 1, NULL) == 1
    assert b"2^30" in lib.gki_last_error()
    prefix = (2, 1, 2, 1, 1, 64, sink, 8, ring, 5, 0.1, P)
    assert lib.gki_rolling_prefix_decode(P, P, P, 0, 0, P, P, 9, P, P, *prefix, 1, 1, NULL) == 1
    assert b"2^30" in lib.gki_last_error()
