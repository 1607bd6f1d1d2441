"""Slices of streams: the launch rules that choose their number, and steps whose own
tokens the launch that attends them writes, at several slices.
"""

from __future__ import annotations

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
