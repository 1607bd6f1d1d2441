"""Slices of streams: the launch rules that choose their number, and steps whose own
tokens the launch that attends them writes, at several slices.
"""

from __future__ import annotations

import ctypes

import pytest

from gki import _lib


@pytest.mark.parametrize("B,H,H_kv,n_q,n_kv,D", [
    (1, 8, 8, 64, 8192, 128), (1, 8, 8, 64, 8192, 64), (1, 8, 8, 200, 8000, 128), (8, 32, 8, 16, 8192, 64),
    (2, 8, 1, 37, 3000, 128), (1, 4, 4, 17, 5000, 32), (4, 8, 2, 4, 6000, 128),
])
def test_both_16_bit_types_take_the_same_slices(B, H, H_kv, n_q, n_kv, D):
    """They run the same row tiles: 32 rows a workgroup for more than 16."""
    lib = _lib.load()
    bf16, fp16 = (lib.gki_cross_splits(dtype, B, H, H_kv, n_q, n_kv, D) for dtype in (2, 1))
    assert bf16 >= 1 and fp16 == bf16


@pytest.mark.parametrize("B,H,H_kv,n_q,n_tokens,D", [(2, 64, 2, 4, 3000, 128), (1, 32, 1, 2, 9000, 64), (4, 20, 1, 1, 5000, 128),
                                                     (3, 12, 12, 2, 700, 64), (16, 64, 2, 2, 8192, 128)])
def test_both_types_take_the_same_slices_behind_a_prefix(B, H, H_kv, n_q, n_tokens, D):
    lib, own = _lib.load(), ctypes.c_int32()

    def splits(dtype):
        return lib.gki_prefix_splits(dtype, B, H, H_kv, n_q, D, 4000, n_tokens, ctypes.byref(own)), own.value

    assert splits(1) == splits(2)
