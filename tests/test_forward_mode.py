"""Tensors with a forward-mode tangent are refused, not answered without a tangent."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from gki import (MultiAxisRotary, PagedKVCache, PageTable, StreamingMaskSpec, block_sparse_attention, cross_attention,
                 make_streaming_mask)
from gki.ops import _refuse_tangents


def test_only_tangents_are_refused():
    x, y = torch.randn(3), torch.randn(3)
    _refuse_tangents(x, y)
    with forward_ad.dual_level():
        _refuse_tangents(x, y)
        dual = forward_ad.make_dual(x, torch.ones(3))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _refuse_tangents(y, dual)
        with torch.no_grad(), pytest.raises(NotImplementedError):      # tangents flow there too
            _refuse_tangents(y, dual)
        _refuse_tangents(forward_ad.unpack_dual(dual).primal)
    _refuse_tangents(x)


def _inputs(n_q):
    gen = torch.Generator(device="cuda").manual_seed(n_q)
    return [torch.randn((1, 2, n, 64), generator=gen, device="cuda") for n in (n_q, 128, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("n_q", [1, 128])
def test_cross_attention(which, n_q):
    qkv = _inputs(n_q)
    want = cross_attention(*qkv)
    with forward_ad.dual_level():
        assert torch.equal(cross_attention(*qkv), want)
        qkv[which] = forward_ad.make_dual(qkv[which], torch.ones_like(qkv[which]))
        with pytest.raises(NotImplementedError):
            cross_attention(*qkv)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            cross_attention(*qkv)
        qkv[0].requires_grad_(True)
        with pytest.raises(NotImplementedError):
            cross_attention(*qkv)


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("n_q", [1, 128])
def test_block_sparse_attention(which, n_q):
    qkv = _inputs(n_q)
    mask = make_streaming_mask(n_q, 128, StreamingMaskSpec(4, 64), 64, 64, device="cuda")
    call = dict(is_causal=True, sink_size=4, window_size=64)
    want = block_sparse_attention(*qkv, mask, **call)
    with forward_ad.dual_level():
        assert torch.equal(block_sparse_attention(*qkv, mask, **call), want)
        qkv[which] = forward_ad.make_dual(qkv[which], torch.ones_like(qkv[which]))
        with pytest.raises(NotImplementedError):
            block_sparse_attention(*qkv, mask, **call)


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("counts", [[1, 1], [3, 70]])
def test_paged_cache(which, counts):
    """Refused before anything is written."""
    table = PageTable(2, 8, StreamingMaskSpec(4, 100), device="cuda")
    cache, rope, rows = PagedKVCache(table, 2, 64), MultiAxisRotary(64, (32,)), sum(counts)
    gen = torch.Generator(device="cuda").manual_seed(rows)
    q, k, v = ((torch.randn((rows, h, 64), generator=gen, device="cuda")).bfloat16() for h in (4, 2, 2))
    batch = table.extend(torch.tensor(counts, device="cuda"), rows)
    cache.append(k, v, batch)
    want = cache.attend(q, batch)
    held = cache.k_pages.clone(), cache.v_pages.clone()
    qkv = [q, k, v]
    with forward_ad.dual_level():
        assert torch.equal(cache.attend(q, batch), want)
        qkv[which] = forward_ad.make_dual(2 * qkv[which], torch.ones_like(qkv[which]))
        calls = [lambda: cache.append_rotated(*qkv, batch, rope),
                 (lambda: cache.attend(qkv[0], batch)) if which == 0 else (lambda: cache.append(*qkv[1:], batch))]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
    assert torch.equal(cache.k_pages, held[0]) and torch.equal(cache.v_pages, held[1])
